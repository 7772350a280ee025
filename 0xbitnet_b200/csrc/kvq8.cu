// kvq8.cu — the KV cache held in 8 bits, sm_100a: append and read-back
// (attention over it: kvq8_attn.cu).
//
// Format. A row x of 128 values (a rotated key or a value) at position p is held as int8
// codes c with x ~ c * s, where s = 2^e is shared by the 16 positions of a block and one KV
// head. The block's scale is the smallest power of two that keeps every appended |x| at or
// below 127 * s. A block fills up token by token, so its scale can only be fixed later: when
// a new row needs a larger one, the rows already there are requantized, c' = rint(c * s / s').
// With powers of two s / s' is exact and a scale at least doubles when it grows, so the
// roundings of a row add up to at most s/2 (1 + 1/2 + 1/4 + ...) <= s of its last scale.
#include "kvq8.h"

#include <cmath>

#include "obn_common.cuh"

namespace obn {

namespace {

constexpr int D = kQ8HeadDim;
constexpr int kNoExp = -100000;   // exponent of an all-zero block
constexpr int kBadExp = 100000;   // a non-finite value was seen
constexpr int kMinExp = -126;     // smallest normal scale, so that 1 / s is finite

// |x| as 32 bits that order like it, as far as need_exp asks: the upper word of the f64, then
// whether the lower one is zero.
OBN_DEVINL uint32_t mag(double x) {
  return 2u * (static_cast<uint32_t>(__double2hiint(x)) & 0x7FFFFFFFu) + (__double2loint(x) != 0);
}
// Smallest e with |x| <= 127 * 2^e (clamped at kMinExp), of mag(x).
OBN_DEVINL int need_exp(uint32_t m) {
  if (m == 0) return kNoExp;
  const int ex = static_cast<int>(m >> 21);
  if (ex == 0x7FF) return kBadExp;
  // 127 = 1.984375 * 2^6, whose upper mantissa bits are 0xFC000
  const bool above = (m & 0x1FFFFFu) > 2u * 0xFC000u;
  return max(ex - 1023 - 6 + (above ? 1 : 0), kMinExp);
}

OBN_DEVINL float exp_scale(int e) {  // 2^e for a normal exponent
  return __int_as_float((e + 127) << 23);
}

// One CTA takes a block of 16 positions of one sequence and KV head, with the query heads of
// its group; a warp takes one row of one head (a lane four dims) at a time.
//  * Angles are p * base^(-2i/128) in turns, reduced in f64 (an f32 angle is off by 6e-3 at
//    position 1e5); their sines and cosines, about 50 f64 operations each, are shared by
//    the CTA's heads. k is rotated in f64, so that a code is off only where f64 is. q is
//    rotated in f32 with rounded sines and cosines (3.7e-8 from the exact one, rounded once 2.5e-8):
//    it is f32 in any case, attention holds it in 22 bits or more, and f64 would rotate four times
//    as many rows of q as of k. v times a power of two is exact in f32.
//  * A block's scale has to be known before its first code: the raw k and v rows stay in
//    registers (kKeep per warp) from one pass over memory.
// 2048 tokens of 20 + 2 x 5 heads (31 MB in, 24 MB out): 17.4 us from cold caches, 3.2 TB/s; it
// issues in 57% of the cycles, most of them angles and f64 rotations of k, and the
// rest is the start and end of 1.5 waves of CTAs. Several heads to a CTA, which share the angles,
// took 35 us (fewer loads on their way); three passes over k and v, without kept rows, 40 us.
// One token: 5.3 us, 64 sequences: 6.1 us, the latency of four dependent steps.
constexpr int kAppThreads = 256, kAppWarps = kAppThreads / 32;
constexpr int kKeep = kQ8Block / kAppWarps;  // k rows, and v rows, of a warp

struct RopeTurns {
  double f[D / 2];  // turns per position
};

struct AppendSmem {
  double c[kQ8Block][D / 2], s[kQ8Block][D / 2];
  float2 cs[kQ8Block][D / 2];
  uint32_t m[2];
};

__global__ __launch_bounds__(kAppThreads, 3) void k_append_q8(
    const float* __restrict__ qkv, Q8Cache c, int n, int H, int pos_host,
    const int* __restrict__ pos_dev, const __grid_constant__ RopeTurns turns,
    float* __restrict__ q_out, int window) {
  __shared__ AppendSmem sm;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < 2) sm.m[tid] = 0;
  // Dependents start only when this kernel is done: a decode pass reads older rows early.
  pdl_wait();
  const int b = blockIdx.x / window, h = blockIdx.y;
  const int G = H / c.Hkv, slots = H + 2 * c.Hkv;
  const long long pos = pos_dev ? pos_dev[b] : pos_host;
  const long long blk = (pos >= 0 ? pos / kQ8Block : -((-pos + kQ8Block - 1) / kQ8Block)) +
                        blockIdx.x % window;
  const long long p0 = blk * kQ8Block;
  const int r0 = static_cast<int>(max(pos - p0, 0ll));                 // first new row
  const int r1 = static_cast<int>(min(pos + n - p0, (long long)kQ8Block));  // past the last
  if (r0 >= r1) return;
  const int rs = p0 >= 0 && p0 < c.S_max  // past the last one with a place
                     ? static_cast<int>(min((long long)r1, c.S_max - p0)) : r0;
  const int nr = rs - r0;
  const float* rows = qkv + (static_cast<size_t>(b) * n + (p0 + r0 - pos)) * slots * D + 4 * lane;
  float4 kept[2][kKeep];
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    const int r = warp + i * kAppWarps;
    if (r < nr)
      for (int side = 0; side < 2; ++side)
        kept[side][i] = __ldg(reinterpret_cast<const float4*>(
            rows + (static_cast<size_t>(r) * slots + H + side * c.Hkv + h) * D));
  }
  const size_t scale_at =
      (static_cast<size_t>(b) * ((c.S_max + kQ8Block - 1) / kQ8Block) + blk) * c.Hkv + h;
  float was[2] = {0.0f, 0.0f};  // the scales of the block's earlier rows
  if (r0 > 0 && nr > 0) {
    was[0] = __ldcg(c.k_scale + scale_at);
    was[1] = __ldcg(c.v_scale + scale_at);
  }
  for (int i = tid; i < nr * (D / 2); i += kAppThreads) {
    const int r = i / (D / 2), j = i % (D / 2);
    const double t = static_cast<double>(p0 + r0 + r) * turns.f[j];
    double sn, cs;
    sincospi(2.0 * (t - rint(t)), &sn, &cs);
    sm.s[r][j] = sn;
    sm.c[r][j] = cs;
    sm.cs[r][j] = make_float2(static_cast<float>(cs), static_cast<float>(sn));
  }
  __syncthreads();
  // q heads of the group; a token without a place gets zeros. Four rows on their way at a time.
  const int q_units = G * (r1 - r0);
  for (int u0 = warp; u0 < q_units; u0 += 4 * kAppWarps) {
    float4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = u0 + i * kAppWarps;
      if (u < q_units)
        x[i] = __ldg(reinterpret_cast<const float4*>(
            rows + (static_cast<size_t>(u / G) * slots + h * G + u % G) * D));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = u0 + i * kAppWarps;
      if (u >= q_units) break;
      const int r = u / G;
      float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (r < nr) {
        const float2 a = sm.cs[r][2 * lane], d = sm.cs[r][2 * lane + 1];
        y = make_float4(x[i].x * a.x - x[i].y * a.y, x[i].x * a.y + x[i].y * a.x,
                        x[i].z * d.x - x[i].w * d.y, x[i].z * d.y + x[i].w * d.x);
      }
      const size_t tok = static_cast<size_t>(b) * n + (p0 + r0 - pos) + r;
      *reinterpret_cast<float4*>(q_out + (tok * H + h * G + u % G) * D + 4 * lane) = y;
    }
  }
  if (nr == 0) return;
  // k rotated, and the largest magnitudes
  double k[kKeep][4];
  uint32_t m[2] = {0, 0};
  float vmax = 0.0f;
  bool vnan = false;
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    const int r = warp + i * kAppWarps;
    if (r >= nr) break;
    const double2 cc = *reinterpret_cast<const double2*>(&sm.c[r][2 * lane]);
    const double2 ss = *reinterpret_cast<const double2*>(&sm.s[r][2 * lane]);
    const float4 x = kept[0][i], v = kept[1][i];
    k[i][0] = x.x * cc.x - x.y * ss.x, k[i][1] = x.x * ss.x + x.y * cc.x;
    k[i][2] = x.z * cc.y - x.w * ss.y, k[i][3] = x.z * ss.y + x.w * cc.y;
    m[0] = max(max(m[0], max(mag(k[i][0]), mag(k[i][1]))), max(mag(k[i][2]), mag(k[i][3])));
    vmax = fmaxf(fmaxf(vmax, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
    vnan |= v.x != v.x || v.y != v.y || v.z != v.z || v.w != v.w;
  }
  m[1] = mag(vnan ? INFINITY : vmax);
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    m[side] = __reduce_max_sync(0xffffffffu, m[side]);
    if (lane == 0) atomicMax(&sm.m[side], m[side]);
  }
  __syncthreads();
  const size_t ld = static_cast<size_t>(c.Hkv) * D;
  const size_t code0 = ((static_cast<size_t>(b) * c.S_max + p0) * c.Hkv + h) * D + 4 * lane;
  const float nan = __int_as_float(0x7FC00000);
  float now[2];  // the block's scales after this
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int x = need_exp(sm.m[side]);
    const float need = x == kNoExp ? 0.0f : x == kBadExp ? nan : exp_scale(x);
    now[side] = was[side] != was[side] || need != need ? nan : fmaxf(was[side], need);
  }
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    signed char* codes = side ? c.v : c.k;
    // the earlier rows of a block whose scale grows; not of a NaN
    if (was[side] > 0.0f && was[side] < now[side]) {
      const float ratio = was[side] / now[side];
      for (int r = warp; r < r0; r += kAppWarps) {
        char4* p = reinterpret_cast<char4*>(codes + code0 + r * ld);
        const char4 q = *p;
        *p = make_char4(static_cast<signed char>(__float2int_rn(q.x * ratio)),
                        static_cast<signed char>(__float2int_rn(q.y * ratio)),
                        static_cast<signed char>(__float2int_rn(q.z * ratio)),
                        static_cast<signed char>(__float2int_rn(q.w * ratio)));
      }
    }
    const float inv = now[side] > 0.0f ? 1.0f / now[side] : 0.0f;  // a power of two, or zero
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
      const int r = warp + i * kAppWarps;
      if (r >= nr) break;
      int q[4] = {0, 0, 0, 0};
      if (inv > 0.0f) {
        if (side == 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) q[j] = __double2int_rn(k[i][j] * inv);
        } else {
          const float4 v = kept[1][i];
          q[0] = __float2int_rn(v.x * inv), q[1] = __float2int_rn(v.y * inv);
          q[2] = __float2int_rn(v.z * inv), q[3] = __float2int_rn(v.w * inv);
        }
      }
      *reinterpret_cast<char4*>(codes + code0 + (r0 + r) * ld) =
          make_char4(static_cast<signed char>(q[0]), static_cast<signed char>(q[1]),
                     static_cast<signed char>(q[2]), static_cast<signed char>(q[3]));
    }
  }
  __syncthreads();  // every thread has read the old scales
  if (tid < 2) (tid ? c.v_scale : c.k_scale)[scale_at] = now[tid];
}

__global__ __launch_bounds__(256) void k_read_q8(Q8Cache c, int first, const int* __restrict__ first_dev,
                                                 int count, float* __restrict__ k_out,
                                                 float* __restrict__ v_out, size_t total) {
  pdl_wait();
  const size_t i = static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const int d4 = static_cast<int>(i % (D / 4));
  size_t rest = i / (D / 4);
  const int h = static_cast<int>(rest % c.Hkv);
  rest /= c.Hkv;
  const int r = static_cast<int>(rest % count);
  const size_t b = rest / count;
  const long long p = static_cast<long long>(first_dev ? first_dev[b] : first) + r;
  const bool in = p >= 0 && p < c.S_max;
  const size_t src = ((b * c.S_max + (in ? p : 0)) * c.Hkv + h) * D + 4 * d4;
  const size_t sc = (b * ((c.S_max + kQ8Block - 1) / kQ8Block) + (in ? p : 0) / kQ8Block) * c.Hkv + h;
  for (int side = 0; side < 2; ++side) {
    float* out = side ? v_out : k_out;
    if (!out) continue;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (in) {
      const char4 q = *reinterpret_cast<const char4*>((side ? c.v : c.k) + src);
      const float s = (side ? c.v_scale : c.k_scale)[sc];
      y = make_float4(q.x * s, q.y * s, q.z * s, q.w * s);
    }
    *reinterpret_cast<float4*>(out + 4 * i) = y;
  }
}

}  // namespace

cudaError_t launch_rope_append_q8(const float* qkv, const Q8Cache& c, int n, int H, int pos,
                                  const int* pos_dev, float theta_base, float* q_out,
                                  cudaStream_t s) {
  // The frequencies in turns as powers of base^(-2 / 128): after i products f_i is off by i 2^-53
  // (relative), i base^(-i / 64) 2^-53 of the first one, which is at most 2 to 10 roundings of
  // p f_0 for the bases in use (500000 to 10).
  RopeTurns turns;
  const double ratio = std::pow(static_cast<double>(theta_base), -2.0 / D);
  turns.f[0] = 1.0 / 6.283185307179586;
  for (int i = 1; i < D / 2; ++i) turns.f[i] = turns.f[i - 1] * ratio;
  // blocks that n rows from anywhere inside a block can touch
  const int window = static_cast<int>((static_cast<long long>(n) + 2 * (kQ8Block - 1)) / kQ8Block);
  const long long blocks = static_cast<long long>(window) * c.B;
  return launch_pdl(&k_append_q8, dim3(static_cast<unsigned>(blocks), c.Hkv), kAppThreads, 0, s,
                    qkv, c, n, H, pos, pos_dev, turns, q_out, window);
}

cudaError_t launch_read_q8(const Q8Cache& c, int first, const int* first_dev, int count,
                           float* k_out, float* v_out, cudaStream_t s) {
  const size_t total = static_cast<size_t>(c.B) * count * c.Hkv * (D / 4);
  return launch_pdl(k_read_q8, dim3(static_cast<unsigned>((total + 255) / 256)), 256, 0, s, c, first,
                    first_dev, count, k_out, v_out, total);
}

}  // namespace obn
