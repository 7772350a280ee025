// logits.cu — the rules that a server lays on each row of logits before a token is picked:
// penalties for the ids of a history, biases, a grammar's bit mask, and the greedy choice.
//
//   n = occurrences of v in the history, x = logit v
//   n > 0:  x > 0 ? x / rep^n : x * rep^n, then - (freq * n + pres)
//   + the biases listed for v;  -inf where the mask's bit is 0;  token = argmax, lowest v
//
// The pass reads and writes 4 bytes a logit and should wait for nothing else. A row is cut
// into slices of 8192 ids, which a cluster of CTAs (one to sixteen, as many as fit on the GPU at
// once) takes in turn; a CTA has the next slice's logits on the way (one bulk copy) while it works
// on one in shared memory, and the lists, read once, in registers:
//   1. count the occurrences of the slice's ids (16 bits an id, shared-memory atomics on
//      whole numbers: any order gives the same counts); an atomic that finds a zero puts
//      the id on the slice's list of distinct ids
//   2. the list's logits are rewritten in place, in f64, rounded once; an id with a bias is left
//      to the first of its bias entries, which has the sum of all of them in list order
//   3. the slice streams out, with the mask and the row's maximum
// With the list the f64 work falls on full warps. Histories crowd in a few slices and are sparse in
// the others: 64 rows of 128256 with 4096 ids took 123 us when the threads that stream the logits
// rewrote them in passing, 38 us when the threads that count an id rewrote it, 58 us with the
// history spread over the cluster and remote counters, 40 us when the marked ids were gathered and
// the others streamed through registers past them, without staging; 30 us as it is, 14 without any
// rule (the kernel from cold caches). Three smaller slices on their way took 37 us, twice the CTAs
// 35 us.
#include "logits.h"

#include <cmath>
#include <type_traits>

#include "kvq8.h"
#include "obn_common.cuh"

namespace obn {

int num_sms_cached();  // kernels.cu

namespace {

constexpr int kThreads = 512;
constexpr int kQuads = 4;                         // float4 of a slice per thread
constexpr int kSliceIds = 4 * kQuads * kThreads;  // 8192
constexpr int kMaxCluster = 16;
constexpr int kMaxBias = 1024, kBiasPer = kMaxBias / kThreads;
constexpr int kHistRegs = 8;    // history entries of a thread in registers

struct LogitSmem {
  float x[2][kSliceIds];
  uint16_t count[kSliceIds];
  uint16_t found[kSliceIds];  // distinct ids of the history in the slice
  uint32_t founds;
  uint32_t biased[kSliceIds / 32];  // ids with a bias, and with several
  uint32_t twice[kSliceIds / 32];
  int bias_id[kMaxBias];
  float bias_value[kMaxBias];
  uint32_t best_key[kThreads / 32];
  uint32_t best_at[kThreads / 32];
  uint2 cluster_best[kMaxCluster];  // of the cluster's CTAs, in the first one
  uint64_t full[2];
};

// base^n for n >= 1 in f64.
OBN_DEVINL double ipow(double base, unsigned n) {
  if (n == 1) return base;
  double r = 1.0;
  for (; n; n >>= 1, base *= base)
    if (n & 1) r *= base;
  return r;
}

constexpr int kNowhere = 0x7FFFFFFF;  // position of an id outside the row

// Order-preserving key of a float that is no NaN (-0 counts as +0).
OBN_DEVINL uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Ids count from the 16-byte boundary at or before the row's start: position p = v + mis.
__global__ __launch_bounds__(kThreads, 2) void k_logits(const float* logits, int V,
                                                        obn_logit_rules u, float* out,
                                                        int32_t* __restrict__ token) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  LogitSmem& sm = *reinterpret_cast<LogitSmem*>(smem_raw);
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x, cluster = gridDim.x;
  const size_t r = blockIdx.y;
  if (tid == 0) {
    mbar_init(&sm.full[0], 1);
    mbar_init(&sm.full[1], 1);
    fence_mbar_init();
  }
  for (int i = tid; i < kSliceIds / 8; i += kThreads)
    reinterpret_cast<uint4*>(sm.count)[i] = make_uint4(0u, 0u, 0u, 0u);
  for (int i = tid; i < kSliceIds / 32; i += kThreads) sm.biased[i] = sm.twice[i] = 0;
  if (tid == 0) sm.founds = 0;
  __syncthreads();
  // waited for at the end: no store to a CTA that has not started
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  pdl_wait();
  const float* x_row = logits + r * V;
  float* y_row = out + r * V;
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(x_row) >> 2) & 3);
  const bool vec_out = (reinterpret_cast<uintptr_t>(y_row) & 15) == (reinterpret_cast<uintptr_t>(x_row) & 15);
  const int end = V + mis;  // positions of the row: [mis, end)
  const int step = cluster * kSliceIds;
  const int own = 4 * tid - mis;  // the thread's first id in a slice, from the slice's position
  const int sh = own & 31;        // its bit in a mask word: slices are whole words
  bool dead = false;  // a copy did not come in time

  // Quads [q_head, q_end) of the slice at p0 lie in the row; one before them and one behind may
  // be cut by the row's ends.
  auto q_head = [&](int p0) { return p0 < mis ? 1 : 0; };
  auto q_end = [&](int p0) {
    const int cnt = min(kSliceIds, end - p0);
    return max(cnt / 4, q_head(p0));
  };
  // The whole quads of the slice at p0 by one bulk copy, the cut ones at the row's ends by their
  // elements (threads 0 to 7). Returns whether there is a copy to wait for.
  auto request = [&](int p0, int buf) {
    const int cnt = min(kSliceIds, end - p0), nq = (cnt + 3) / 4;
    const int head = q_head(p0), whole = q_end(p0) - head;
    if (tid == 0 && whole > 0) {
      fence_proxy_async_smem();  // threads read and wrote the buffer before
      mbar_arrive_expect_tx(&sm.full[buf], whole * 16);
      bulk_g2s(&sm.x[buf][4 * head], x_row + (p0 + 4 * head - mis), whole * 16, &sm.full[buf]);
    }
    if (tid < 8) {
      const int i = 4 * (tid < 4 ? 0 : nq - 1) + (tid & 3), p = p0 + i;
      if ((tid < 4 ? head : q_end(p0) < nq) && p >= mis && p < end) sm.x[buf][i] = x_row[p - mis];
    }
    return whole > 0;
  };
  const int p_first = rank * kSliceIds;
  bool copied = p_first < end ? request(p_first, 0) : false;

  // The lists, requested before their lengths are known.
  const int32_t* h = u.history + r * u.history_ld;
  int hid[kHistRegs], bid[kBiasPer];
  float bval[kBiasPer];
#pragma unroll
  for (int i = 0; i < kHistRegs; ++i)
    hid[i] = u.history && tid + i * kThreads < u.history_cap ? __ldg(h + tid + i * kThreads) : -1;
#pragma unroll
  for (int i = 0; i < kBiasPer; ++i) {
    const int j = tid + i * kThreads;
    const bool in = u.bias_ids && j < u.bias_cap;
    bid[i] = in ? __ldg(u.bias_ids + r * u.bias_ld + j) : -1;
    bval[i] = in ? __ldg(u.bias_values + r * u.bias_ld + j) : 0.0f;
  }
  const int hist = !u.history ? 0 : u.history_lens ? min(max(u.history_lens[r], 0), u.history_cap)
                                                   : u.history_cap;
  const int nbias = !u.bias_ids ? 0 : u.bias_lens ? min(max(u.bias_lens[r], 0), u.bias_cap)
                                                  : u.bias_cap;
  const double rep = u.repetition ? u.repetition[r] : 1.0f;
  const double freq = u.frequency ? u.frequency[r] : 0.0f;
  const double pres = u.presence ? u.presence[r] : 0.0f;
  const double inv_rep = 1.0 / rep;
  // From here on the lists hold positions.
  auto position = [&](int id) { return static_cast<unsigned>(id) < static_cast<unsigned>(V) ? id + mis : kNowhere; };
#pragma unroll
  for (int i = 0; i < kHistRegs; ++i)
    hid[i] = tid + i * kThreads < hist ? position(hid[i]) : kNowhere;
#pragma unroll
  for (int i = 0; i < kBiasPer; ++i) {
    const int j = tid + i * kThreads;
    bid[i] = j < nbias ? position(bid[i]) : kNowhere;
    if (nbias) {
      sm.bias_id[j] = bid[i];
      sm.bias_value[j] = bval[i];
    }
  }
  // The logit of an id with n occurrences. 1 / rep in f64 serves for the division: quotients
  // of two f32 lie at least 2^-49 (relative) from the middle between two f32, the product is
  // off by 2^-52, so a single occurrence gives the correctly rounded quotient.
  // A zero or an infinity stays what it is, also where the power leaves f64's range.
  auto penalised = [&](double x, unsigned n) {
    if (n) {
      if (x != 0.0 && fabs(x) < INFINITY) x *= ipow(x > 0.0 ? inv_rep : rep, n);
      x -= freq * n + pres;
    }
    return x;
  };

  const uint32_t* mask = u.mask ? u.mask + r * u.mask_ld : nullptr;
  float best = -INFINITY;
  int best_at = 0;
  uint32_t phase = 0;
  int buf = 0, p0 = p_first;
  for (; p0 < end; p0 += step, buf ^= 1) {
    const int cnt = min(kSliceIds, end - p0), nq = (cnt + 3) / 4;
    const bool wait = copied;
    if (p0 + step < end) copied = request(p0 + step, buf ^ 1);
    const int q0 = q_head(p0), q1 = q_end(p0);
    // mask words of the thread's whole quads, used when they have come: quad k begins at bit sh
    // of word kThreads / 8 * k behind the first one's
    uint32_t m_lo[kQuads], m_hi[kQuads];
    if (mask) {
      const uint32_t* words = mask + ((p0 + own) >> 5);
#pragma unroll
      for (int k = 0; k < kQuads; ++k) {
        const int q = tid + k * kThreads;
        m_lo[k] = m_hi[k] = 0;
        if (q >= q0 && q < q1) {
          m_lo[k] = __ldg(words + k * (kThreads / 8));
          if (sh > 28) m_hi[k] = __ldg(words + k * (kThreads / 8) + 1);
        }
      }
    }
    auto in = [&](int at) { return static_cast<unsigned>(at) < static_cast<unsigned>(cnt); };
    // 1. occurrences, distinct ids, biased ids
    if (hist) {
      auto occurs = [&](int at) {
        const int sh = 16 * (at & 1);
        const uint32_t was = atomicAdd(reinterpret_cast<uint32_t*>(sm.count) + (at >> 1), 1u << sh);
        if (((was >> sh) & 0xFFFFu) == 0)
          sm.found[atomicAdd(&sm.founds, 1u)] = static_cast<uint16_t>(at);
      };
#pragma unroll
      for (int i = 0; i < kHistRegs; ++i)
        if (in(hid[i] - p0)) occurs(hid[i] - p0);
      for (int j = tid + kHistRegs * kThreads; j < hist; j += kThreads) {
        const int at = position(__ldg(h + j)) - p0;
        if (in(at)) occurs(at);
      }
    }
    int bat[kBiasPer];
    if (nbias) {
#pragma unroll
      for (int i = 0; i < kBiasPer; ++i) {
        bat[i] = bid[i] - p0;
        if (!in(bat[i])) {
          bat[i] = -1;
          continue;
        }
        const uint32_t bit = 1u << (bat[i] & 31);
        if (atomicOr(&sm.biased[bat[i] >> 5], bit) & bit) atomicOr(&sm.twice[bat[i] >> 5], bit);
      }
    }
    float* x = sm.x[buf];
    dead = __syncthreads_or(wait && !mbar_wait(&sm.full[buf], (phase >> buf) & 1));
    if (dead) break;
    if (wait) phase ^= 1u << buf;
    // 2. rewrite
    const int founds = hist ? sm.founds : 0;
    for (int i = tid; i < founds; i += kThreads) {
      const int at = sm.found[i];
      if ((sm.biased[at >> 5] >> (at & 31)) & 1u) continue;
      x[at] = static_cast<float>(penalised(x[at], sm.count[at]));
    }
    if (nbias) {
#pragma unroll
      for (int i = 0; i < kBiasPer; ++i)
        if (bat[i] >= 0) {
          double sum = bval[i];
          if ((sm.twice[bat[i] >> 5] >> (bat[i] & 31)) & 1u) {
            // the first entry of the id takes all of them, in list order
            const int j = tid + i * kThreads;
            bool first = true;
            sum = 0.0;
            for (int e = 0; e < nbias; ++e)
              if (sm.bias_id[e] == bid[i]) {
                first &= e >= j;
                sum += sm.bias_value[e];
              }
            if (!first) continue;
          }
          x[bat[i]] = static_cast<float>(penalised(x[bat[i]], sm.count[bat[i]]) + sum);
        }
    }
    if (hist || nbias) __syncthreads();
    // 3. out
    const float* xs = x + 4 * tid;
    float* ys = y_row + (p0 + own);
    auto stream = [&](auto masked) {
#pragma unroll
      for (int k = 0; k < kQuads; ++k) {
        const int q = tid + k * kThreads;
        if (q < q0 || q >= q1) continue;
        float4 y = *reinterpret_cast<const float4*>(xs + 4 * k * kThreads);
        if constexpr (decltype(masked)::value) {
          const uint32_t allow = __funnelshift_r(m_lo[k], m_hi[k], sh);  // bits 0 to 3
          if (!(allow & 1u)) y.x = -INFINITY;
          if (!(allow & 2u)) y.y = -INFINITY;
          if (!(allow & 4u)) y.z = -INFINITY;
          if (!(allow & 8u)) y.w = -INFINITY;
        }
        // the quad of the largest logit so far (a NaN is in no maximum and above nothing)
        const float m = fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w));
        if (m > best) {
          best = m;
          best_at = p0 + own + 4 * k * kThreads;
        }
        float* dst = ys + 4 * k * kThreads;
        if (vec_out) {
          *reinterpret_cast<float4*>(dst) = y;
        } else {
          dst[0] = y.x;
          dst[1] = y.y;
          dst[2] = y.z;
          dst[3] = y.w;
        }
      }
    };
    if (mask)
      stream(std::true_type{});
    else
      stream(std::false_type{});
    if (tid < 8 && (tid < 4 ? q0 > 0 : q1 < nq)) {  // the cut quads, an id a thread
      const int i = 4 * (tid < 4 ? 0 : nq - 1) + (tid & 3), v = p0 + i - mis;
      if (v >= 0 && v < V) {
        const bool ok = !mask || ((__ldg(mask + (v >> 5)) >> (v & 31)) & 1u);
        const float y = ok ? x[i] : -INFINITY;
        y_row[v] = y;
        if (y > best || (y == best && y > -INFINITY && v < best_at)) {
          best = y;
          best_at = v;
        }
      }
    }
    if (p0 + step < end) {  // counters and bits back to zero
      for (int i = tid; i < founds; i += kThreads) sm.count[sm.found[i]] = 0;
      if (tid == 0) sm.founds = 0;
      if (nbias) {
#pragma unroll
        for (int i = 0; i < kBiasPer; ++i)
          if (bat[i] >= 0) sm.biased[bat[i] >> 5] = sm.twice[bat[i] >> 5] = 0;
      }
      __syncthreads();
    }
  }

  if (dead) {  // nothing of the slice was used: NaN for the rest of the CTA's ids, and no token
    if (tid == 0) {  // the copies may still be on their way into this CTA's shared memory
      mbar_wait(&sm.full[buf], (phase >> buf) & 1);
      if (copied && p0 + step < end) mbar_wait(&sm.full[buf ^ 1], (phase >> (buf ^ 1)) & 1);
    }
    for (; p0 < end; p0 += step)
      for (int p = max(p0, mis) + tid; p < min(p0 + kSliceIds, end); p += kThreads)
        y_row[p - mis] = __int_as_float(0x7FC00000);
  }

  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (!token) return;
  // the largest key, and the lowest id that has it
  uint32_t at = 0xFFFFFFFFu;
  if (best > -INFINITY) {  // which of the quad, as this thread wrote it
#pragma unroll
    for (int e = 3; e >= 0; --e) {
      const int v = best_at + e;
      if (v >= 0 && v < V && y_row[v] == best) at = v;
    }
  }
  // 0: nothing above -inf; no float has all bits of a key set, and the token is -1 with that one
  if (dead) at = 0xFFFFFFFFu;
  const uint32_t mine = dead ? 0xFFFFFFFFu : best > -INFINITY ? key_of(best) : 0u;
  const uint32_t wk = __reduce_max_sync(0xffffffffu, mine);
  const uint32_t wa = __reduce_min_sync(0xffffffffu, mine == wk ? at : 0xFFFFFFFFu);
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
      asm("mapa.shared::cluster.u32 %0, %1, %2;"
          : "=r"(dst)
          : "r"(smem_u32(&sm.cluster_best[rank])), "r"(0));
      asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(dst), "r"(ck), "r"(ca)
                   : "memory");
    }
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  if (rank != 0) return;
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (tid == 0) {
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
  cudaError_t e = allow_smem<&k_logits>(sizeof(LogitSmem));
  if (e != cudaSuccess) return e;
  const int most =
      active_clusters<&k_logits>(kMaxCluster, kThreads, sizeof(LogitSmem)) > 0 ? kMaxCluster : 8;
  // As many CTAs to a row as find room at once, two on an SM.
  const int slices = (vocab + kSliceIds - 1) / kSliceIds;
  int cluster = 1;
  while (cluster < most && cluster < slices && rows * cluster * 2ll <= 2 * num_sms_cached())
    cluster *= 2;
  return launch_cluster(&k_logits, dim3(cluster, rows), cluster, kThreads, sizeof(LogitSmem), s,
                        logits, vocab, rules, out, token);
}

}  // namespace obn
