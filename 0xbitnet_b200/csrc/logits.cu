// logits.cu — the rules that a server lays on each row of logits before a token is picked:
// penalties for the ids of a history, biases, a grammar's bit mask, and the greedy choice.
//
//   n = occurrences of v in the history, x = logit v
//   n > 0:  x > 0 ? x / rep^n : x * rep^n, then - (freq * n + pres)
//   + the biases listed for v;  -inf where the mask's bit is 0;  token = argmax, lowest v
//
// The pass reads and writes 4 bytes a logit and should wait for nothing else. A cluster of
// CTAs takes a row; each CTA copies its slice of it to shared memory and meanwhile counts the
// occurrences of the slice's ids, by shared-memory atomics on whole numbers (16 bits an id),
// so every order of arrival gives the same counts; every CTA of a row scans the whole
// history, which lies in L2. In a second scan the first thread to claim an id (a bit in shared
// memory) rewrites its logit there: the f64 work is spread over the threads as the history is, not as
// the ids lie (histories crowd in a few slices: 123 us for 64 rows of 128256 with 4096 ids
// when the threads that stream the logits did it in passing). Biases are compacted in list
// order; the first entry of an id owns it and adds up the others in that order. A rewritten
// logit is rounded once. Then the slice streams out, with the mask and the row's maximum, which
// goes through shuffles, shared memory and the first CTA of the cluster.
#include "logits.h"

#include <cmath>

#include "kvq8.h"
#include "obn_common.cuh"

namespace obn {
namespace {

constexpr int kThreads = 512;
constexpr int kQuads = 8;                           // float4 per thread
constexpr int kSliceIds = 4 * kQuads * kThreads;    // 16384
constexpr int kMaxCluster = 8;
constexpr int kMaxBias = 1024;

struct LogitSmem {
  float x[kSliceIds];
  uint32_t count[kSliceIds / 2];  // 16 bits an id
  uint32_t taken[kSliceIds / 32];  // ids whose logit has an owner
  int hit_id[kMaxBias];
  float hit_value[kMaxBias];
  int warp_hits[kThreads / 32];
  uint32_t best_key[kThreads / 32];
  uint32_t best_at[kThreads / 32];
  uint2 cluster_best[kMaxCluster];  // of the cluster's CTAs, in the first one
  uint64_t full;
};

// base^n for n >= 1 in f64.
OBN_DEVINL double ipow(double base, unsigned n) {
  double r = 1.0;
  for (; n; n >>= 1, base *= base)
    if (n & 1) r *= base;
  return r;
}

// Order-preserving key of a float above -inf (0 stands for none; -0 counts as +0).
OBN_DEVINL uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  if ((u << 1) == 0) return 0x80000000u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ __launch_bounds__(kThreads) void k_logits(const float* __restrict__ logits, int V,
                                                     obn_logit_rules u, int cluster,
                                                     float* out, int32_t* __restrict__ token) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  LogitSmem& sm = *reinterpret_cast<LogitSmem*>(smem_raw);
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x;
  const size_t r = blockIdx.y;
  const float* x_row = logits + r * V;
  float* y_row = out + r * V;
  // Quad q holds ids 4 q - mis .. + 3: aligned 16 bytes of the row, whose ends may be cut.
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(x_row) >> 2) & 3);
  const bool vec_out = (reinterpret_cast<uintptr_t>(y_row) & 15) == (reinterpret_cast<uintptr_t>(x_row) & 15);
  const int quads = (V + mis + 3) / 4;
  const int per = min((quads + cluster - 1) / cluster, kQuads * kThreads);  // quads of a slice
  const uint32_t* mask = u.mask ? u.mask + r * u.mask_ld : nullptr;
  const int hist = !u.history ? 0 : u.history_lens ? min(max(u.history_lens[r], 0), u.history_cap)
                                                   : u.history_cap;
  const int nbias = !u.bias_ids ? 0 : u.bias_lens ? min(max(u.bias_lens[r], 0), u.bias_cap)
                                                  : u.bias_cap;
  const double rep = u.repetition ? u.repetition[r] : 1.0f;
  const double freq = u.frequency ? u.frequency[r] : 0.0f;
  const double pres = u.presence ? u.presence[r] : 0.0f;
  const double inv_rep = 1.0 / rep;
  uint32_t best = 0, best_at = 0, phase = 0;
  bool dead = false;  // a copy did not come in time: no more of them
  if (tid == 0) {
    mbar_init(&sm.full, 1);
    fence_mbar_init();
  }
  __syncthreads();

  // The logit of an id with n occurrences. 1 / rep in f64 serves for the division: quotients
  // of two f32 lie at least 2^-49 (relative) from the middle between two f32, the product is
  // off by 2^-52, so a single occurrence gives the correctly rounded quotient.
  auto penalised = [&](double x, unsigned n) {
    if (n) x = x * ipow(x > 0.0 ? inv_rep : rep, n) - (freq * n + pres);
    return x;
  };

  for (int q0 = rank * per; q0 < quads; q0 += cluster * per) {
    const int nq = min(per, quads - q0);
    const int v0 = 4 * q0 - mis;  // the first id (may be below 0)
    // 1. request the slice: whole quads by one bulk copy, cut ones by their elements
    const int head = v0 < 0 ? 1 : 0, tail = v0 + 4 * nq > V && nq > head ? 1 : 0;
    const int whole = nq - head - tail;
    if (tid == 0 && whole > 0 && !dead) {
      fence_proxy_async_smem();  // the slice before was read and written by threads
      mbar_arrive_expect_tx(&sm.full, whole * 16);
      bulk_g2s(&sm.x[4 * head], x_row + v0 + 4 * head, whole * 16, &sm.full);
    }
    if (tid < 8) {
      const int q = tid < 4 ? 0 : nq - 1, i = 4 * q + (tid & 3), v = v0 + i;
      if ((tid < 4 ? head : tail) && v >= 0 && v < V) sm.x[i] = x_row[v];
    }
    uint32_t allow[kQuads];
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      const int q = tid + k * kThreads, v = v0 + 4 * q;
      allow[k] = 15u;
      if (mask && q < nq) {
        const int lo = max(v, 0) >> 5, hi = min(v + 3, V - 1) >> 5;
        const uint32_t a = __ldg(mask + lo), b = hi != lo ? __ldg(mask + hi) : a;
        allow[k] = v < 0 ? a << -v : __funnelshift_r(a, b, v & 31);
      }
    }
    // 2. occurrences and biases of the slice's ids
    const int32_t* h = u.history + r * u.history_ld;
    auto local = [&](int id) {  // index in the slice, or -1
      const unsigned at = static_cast<unsigned>(id - v0);
      return id >= 0 && id < V && at < static_cast<unsigned>(4 * nq) ? static_cast<int>(at) : -1;
    };
    if (hist) {
      for (int i = tid; i < (nq + 1) / 2; i += kThreads)
        reinterpret_cast<uint4*>(sm.count)[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    if (hist || nbias) {
      for (int i = tid; i < (4 * nq + 31) / 32; i += kThreads) sm.taken[i] = 0;
      __syncthreads();
    }
    for (int i = tid; i < hist; i += kThreads) {
      const int at = local(__ldg(h + i));
      if (at >= 0) atomicAdd(&sm.count[at >> 1], 1u << (16 * (at & 1)));
    }
    int hits = 0;
    for (int j0 = 0; j0 < nbias; j0 += kThreads) {
      const int j = j0 + tid;
      const int id = j < nbias ? __ldg(u.bias_ids + r * u.bias_ld + j) : -1;
      const int at = local(id);
      const uint32_t votes = __ballot_sync(0xffffffffu, at >= 0);
      if (lane == 0) sm.warp_hits[warp] = __popc(votes);
      __syncthreads();
      int before = hits;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        const int n = sm.warp_hits[w];
        if (w < warp) before += n;
        hits += n;
      }
      if (at >= 0) {
        const int place = before + __popc(votes & ((1u << lane) - 1u));
        sm.hit_id[place] = at;
        sm.hit_value[place] = __ldg(u.bias_values + r * u.bias_ld + j);
        atomicOr(&sm.taken[at >> 5], 1u << (at & 31));
      }
      __syncthreads();
    }
    if (whole > 0 && !dead) {
      dead = !mbar_wait(&sm.full, phase);
      phase ^= 1;
    }
    __syncthreads();
    // 3. rewrite the logits of ids that occur (those with a bias are taken already) ...
    auto count_of = [&](int at) { return (sm.count[at >> 1] >> (16 * (at & 1))) & 0xFFFFu; };
    for (int i = tid; i < hist; i += kThreads) {
      const int at = local(__ldg(h + i));
      if (at < 0) continue;
      const uint32_t bit = 1u << (at & 31);
      if (atomicOr(&sm.taken[at >> 5], bit) & bit) continue;
      sm.x[at] = static_cast<float>(penalised(sm.x[at], count_of(at)));
    }
    // ... and of ids with biases, each by the first of its entries
    for (int j = tid; j < hits; j += kThreads) {
      const int at = sm.hit_id[j];
      bool first = true;
      for (int i = 0; i < j; ++i) first &= sm.hit_id[i] != at;
      if (!first) continue;
      double t = penalised(sm.x[at], hist ? count_of(at) : 0);
      for (int i = j; i < hits; ++i)
        if (sm.hit_id[i] == at) t += sm.hit_value[i];
      sm.x[at] = static_cast<float>(t);
    }
    if (hist || hits) __syncthreads();
    // 4. out
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      const int q = tid + k * kThreads, v = v0 + 4 * q;
      if (q >= nq) break;
      const float4 x = *reinterpret_cast<const float4*>(&sm.x[4 * q]);
      float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!((allow[k] >> e) & 1u)) y[e] = -INFINITY;
        // ids before the row's start and behind its end are no candidates
        if (y[e] > -INFINITY && v + e >= 0 && v + e < V) {
          const uint32_t key = key_of(y[e]);
          if (key > best) {
            best = key;
            best_at = v + e;
          }
        }
      }
      if (vec_out && v >= 0 && v + 3 < V) {
        *reinterpret_cast<float4*>(y_row + v) = make_float4(y[0], y[1], y[2], y[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (v + e >= 0 && v + e < V) y_row[v + e] = y[e];
      }
    }
    __syncthreads();  // the next slice reuses the shared memory
  }

  if (!token) return;
  // the largest key, and the lowest id that has it
  const uint32_t wk = __reduce_max_sync(0xffffffffu, best);
  const uint32_t wa = __reduce_min_sync(0xffffffffu, best == wk ? best_at : 0xFFFFFFFFu);
  if (lane == 0) {
    sm.best_key[warp] = wk;
    sm.best_at[warp] = wa;
  }
  __syncthreads();
  if (warp == 0) {
    const uint32_t k = lane < kThreads / 32 ? sm.best_key[lane] : 0u;
    const uint32_t a = lane < kThreads / 32 ? sm.best_at[lane] : 0xFFFFFFFFu;
    const uint32_t ck = __reduce_max_sync(0xffffffffu, k);
    const uint32_t ca = __reduce_min_sync(0xffffffffu, k == ck ? a : 0xFFFFFFFFu);
    if (lane == 0) {
      uint32_t dst;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(smem_u32(&sm.cluster_best[rank])), "r"(0));
      asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(dst), "r"(ck), "r"(ca) : "memory");
    }
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank == 0 && tid == 0) {
    uint32_t k = 0, a = 0;
    for (int i = 0; i < cluster; ++i) {
      const uint2 o = sm.cluster_best[i];
      if (o.x > k || (o.x == k && o.x && o.y < a)) {
        k = o.x;
        a = o.y;
      }
    }
    token[r] = k ? static_cast<int32_t>(a) : -1;
  }
}

}  // namespace

cudaError_t launch_logits_process(const float* logits, int rows, int vocab,
                                  const obn_logit_rules& rules, float* out, int32_t* token,
                                  cudaStream_t s) {
  // CTAs of a row: one per 16384 ids, and more while they would leave SMs idle.
  int cluster = 1;
  while (cluster < kMaxCluster &&
         (static_cast<long long>(cluster) * kSliceIds < vocab ||
          (static_cast<long long>(rows) * cluster < 148 && cluster * 2048 < vocab)))
    cluster *= 2;
  cudaError_t e = allow_smem<&k_logits>(sizeof(LogitSmem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster, rows);
  cfg.blockDim = kThreads;
  cfg.dynamicSmemBytes = sizeof(LogitSmem);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, k_logits, logits, vocab, rules, cluster, out, token);
}

}  // namespace obn
