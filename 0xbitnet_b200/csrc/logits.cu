// logits.cu — the rules that a server lays on each row of logits before a token is picked.
#include "logits.h"

#include <cmath>

#include "obn_common.cuh"

namespace obn {
namespace {

constexpr int kLogitThreads = 256;
constexpr int kLogitSlice = 4096;

// base^n for a count n >= 1, in f64.
OBN_DEVINL double ipow(double base, unsigned n) {
  double r = 1.0;
  for (; n; n >>= 1, base *= base)
    if (n & 1) r *= base;
  return r;
}

__global__ __launch_bounds__(kLogitThreads) void k_logits_slice(const float* __restrict__ logits,
                                                                int V, obn_logit_rules u,
                                                                float* __restrict__ out) {
  __shared__ unsigned s_count[kLogitSlice];
  pdl_wait();
  const int tid = threadIdx.x, v0 = blockIdx.x * kLogitSlice, nv = min(kLogitSlice, V - v0);
  const size_t r = blockIdx.y;
  for (int i = tid; i < nv; i += kLogitThreads) s_count[i] = 0;
  __syncthreads();
  if (u.history) {
    const int hl = u.history_lens ? min(max(u.history_lens[r], 0), u.history_cap) : u.history_cap;
    const int32_t* h = u.history + r * u.history_ld;
    for (int i = tid; i < hl; i += kLogitThreads) {
      const unsigned d = static_cast<unsigned>(h[i]) - v0;
      if (h[i] >= 0 && d < static_cast<unsigned>(nv)) atomicAdd(&s_count[d], 1u);
    }
    __syncthreads();
  }
  const double rep = u.repetition ? u.repetition[r] : 1.0, freq = u.frequency ? u.frequency[r] : 0.0,
               pres = u.presence ? u.presence[r] : 0.0;
  const int bl = !u.bias_ids ? 0 : u.bias_lens ? min(max(u.bias_lens[r], 0), u.bias_cap) : u.bias_cap;
  for (int i = tid; i < nv; i += kLogitThreads) {
    const int v = v0 + i;
    double x = logits[r * V + v];
    const unsigned n = s_count[i];
    if (n) {
      const double f = ipow(rep, n);
      x = x > 0.0 ? x / f : x * f;
      x -= freq * n + pres;
    }
    for (int j = 0; j < bl; ++j)
      if (u.bias_ids[r * u.bias_ld + j] == v) x += u.bias_values[r * u.bias_ld + j];
    if (u.mask && !((u.mask[r * u.mask_ld + (v >> 5)] >> (v & 31)) & 1u)) x = -INFINITY;
    out[r * V + v] = static_cast<float>(x);
  }
}

__global__ __launch_bounds__(kLogitThreads) void k_row_token(const float* __restrict__ out, int V,
                                                             int32_t* __restrict__ token) {
  __shared__ float s_x[kLogitThreads];
  __shared__ int s_i[kLogitThreads];
  pdl_wait();
  const int tid = threadIdx.x;
  const size_t r = blockIdx.x;
  float best = -INFINITY;
  int at = -1;
  for (int v = tid; v < V; v += kLogitThreads)
    if (out[r * V + v] > best) {
      best = out[r * V + v];
      at = v;
    }
  s_x[tid] = best;
  s_i[tid] = at;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kLogitThreads; ++i)
      if (s_i[i] >= 0 && (at < 0 || s_x[i] > best || (s_x[i] == best && s_i[i] < at))) {
        best = s_x[i];
        at = s_i[i];
      }
    token[r] = at;
  }
}

}  // namespace

cudaError_t launch_logits_process(const float* logits, int rows, int vocab,
                                  const obn_logit_rules& rules, float* out, int32_t* token,
                                  cudaStream_t s) {
  k_logits_slice<<<dim3((vocab + kLogitSlice - 1) / kLogitSlice, rows), kLogitThreads, 0, s>>>(
      logits, vocab, rules, out);
  if (token) k_row_token<<<rows, kLogitThreads, 0, s>>>(out, vocab, token);
  return cudaGetLastError();
}

}  // namespace obn
