// kvq8.h — the 8-bit KV cache (kvq8.cu): RoPE + quantizing append, read-back and attention.
//
// Cache of one layer: codes int8 [B][S_max][Hkv][128] for keys and for values, and one f32
// scale for each (sequence, block of kQ8Block positions, KV head): [B][ceil(S_max / 16)][Hkv].
// The row at position p stands for codes * scale of block p / 16. Scales are powers of two
// (or 0 for a block of zeros, NaN for a block that took a non-finite value).
#pragma once

#include <atomic>
#include <cstddef>
#include <cstdint>

#include <cuda_runtime.h>

namespace obn {

constexpr int kQ8HeadDim = 128;  // head_dim the kernels are built for
constexpr int kQ8Block = 16;     // positions that share a scale

struct Q8Cache {
  int8_t* k;       // [B][S_max][Hkv][128]
  int8_t* v;
  float* k_scale;  // [B][ceil(S_max / 16)][Hkv]
  float* v_scale;
  int B, S_max, Hkv;
};

inline int q8_blocks(int S_max) { return (S_max + kQ8Block - 1) / kQ8Block; }

// Rotates q and k of token t of sequence b at position pos + t (pos_dev[b] + t when pos_dev
// is given), writes q_out [B*n, H*128] and stores k and v into the cache.
cudaError_t launch_rope_append_q8(const float* qkv, const Q8Cache& c, int n, int H, int pos,
                                  const int* pos_dev, float theta_base, float* q_out,
                                  cudaStream_t s);

// Rows [first, first + count) of every sequence (first_dev[b] when given) as f32
// [B][count][Hkv][128]; rows outside the cache are zero. k_out / v_out may be null.
cudaError_t launch_read_q8(const Q8Cache& c, int first, const int* first_dev, int count,
                           float* k_out, float* v_out, cudaStream_t s);

// Causal GQA attention of the n newest tokens; sequence b holds seq_len positions, or
// min(max(lens_dev[b], 0), seq_len) when lens_dev is given.
size_t attention_q8_workspace_bytes(int B, int n, int H, int Hkv, int S_max);
cudaError_t launch_attention_q8(const float* q, const Q8Cache& c, int n, int H, int seq_len,
                                const int* lens_dev, float scale, float* out, void* workspace,
                                cudaStream_t s);

// Its pass for tiles of 256 query rows (kvq8_many.cu), and what that pass needs.
size_t attention_q8_many_workspace_bytes();
cudaError_t launch_attention_q8_many(const float* q, const Q8Cache& c, int n, int H, int seq_len,
                                     const int* lens_dev, float scale_log2, float* out, void* ws,
                                     cudaStream_t s);

// Raises a kernel's dynamic shared memory limit on the current device, once for each.
template <auto kKernel>
cudaError_t allow_smem(size_t bytes) {
  static std::atomic<uint64_t> done{0};  // one bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kKernel),
                           cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// How many clusters of `size` CTAs of a kernel (along x, up to 16, which is beyond the portable
// size) find room on the current device at once. Asked once for each device and size.
template <auto kKernel>
int active_clusters(int size, int threads, size_t smem) {
  static std::atomic<int> known[64][17];  // the answer + 1, 0: not known yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64 || size < 1 || size > 16) return 0;
  int n = known[dev][size].load(std::memory_order_relaxed) - 1;
  if (n >= 0) return n;
  const void* kernel = reinterpret_cast<const void*>(kKernel);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size, 1);
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess)
    n = 0;
  cudaGetLastError();
  known[dev][size].store(n + 1, std::memory_order_relaxed);
  return n;
}

// launch_pdl with clusters along x.
template <typename... Args, typename... Given>
cudaError_t launch_cluster(void (*kernel)(Args...), dim3 grid, int cluster, int threads, size_t smem,
                           cudaStream_t s, Given&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Args>(args)...);
}

}  // namespace obn
