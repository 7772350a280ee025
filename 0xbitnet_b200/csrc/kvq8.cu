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

#include "obn_common.cuh"

namespace obn {
namespace {

constexpr int D = kQ8HeadDim;
constexpr int kNoExp = -100000;   // exponent of an all-zero block
constexpr int kBadExp = 100000;   // a non-finite value was seen
constexpr int kMinExp = -126;     // smallest normal scale, so that 1 / s is finite

// Smallest e with |x| <= 127 * 2^e (clamped at kMinExp).
OBN_DEVINL int need_exp(double x) {
  const long long bits = __double_as_longlong(x) & 0x7FFFFFFFFFFFFFFFll;
  if (bits == 0) return kNoExp;
  const int ex = static_cast<int>(bits >> 52);
  if (ex == 0x7FF) return kBadExp;
  // 127 = 1.984375 * 2^6, whose mantissa bits are 0xFC00000000000
  const bool above = (bits & 0xFFFFFFFFFFFFFll) > 0xFC00000000000ll;
  return max(ex - 1023 - 6 + (above ? 1 : 0), kMinExp);
}

OBN_DEVINL float exp_scale(int e) {  // 2^e for a normal exponent
  return __int_as_float((e + 127) << 23);
}

// Angle of pair i at position p: p * base^(-2i/128), in turns, reduced in f64 (an f32 angle is
// off by 6e-3 at position 1e5), then the sine and cosine of the rest.
OBN_DEVINL void rope_turn(int p, double turns_per_pos, double* sn, double* cs) {
  const double t = static_cast<double>(p) * turns_per_pos;
  sincospi(2.0 * (t - rint(t)), sn, cs);
}

constexpr int kAppThreads = 256;

__global__ __launch_bounds__(kAppThreads) void k_append_q8(
    const float* __restrict__ qkv, Q8Cache c, int n, int H, int pos_host,
    const int* __restrict__ pos_dev, float theta_base, float* __restrict__ q_out, int window) {
  __shared__ double s_c[kQ8Block][D / 2], s_s[kQ8Block][D / 2];
  __shared__ int s_e[2];
  // Dependents start only when this kernel is done: a decode pass reads older rows early.
  pdl_wait();
  const int tid = threadIdx.x;
  const int b = blockIdx.x / window, kvh = blockIdx.y;
  const int G = H / c.Hkv;
  const long long pos = pos_dev ? pos_dev[b] : pos_host;
  const long long blk = (pos >= 0 ? pos / kQ8Block : -((-pos + kQ8Block - 1) / kQ8Block)) +
                        blockIdx.x % window;
  const long long p0 = blk * kQ8Block;
  const int r0 = static_cast<int>(max(pos - p0, 0ll));                 // first new row
  const int r1 = static_cast<int>(min(pos + n - p0, (long long)kQ8Block));  // past the last
  if (r0 >= r1) return;
  const bool in_low = p0 >= 0, any = in_low && p0 < c.S_max;
  const int rs = any ? static_cast<int>(min((long long)r1, c.S_max - p0)) : r0;  // stored rows
  const size_t row0 = (static_cast<size_t>(b) * n + (p0 + r0 - pos));  // token row of row r0
  const int slots = H + 2 * c.Hkv;
  if (tid < 2) s_e[tid] = kNoExp;
  for (int i = tid; i < (rs - r0) * (D / 2); i += kAppThreads) {
    const int r = r0 + i / (D / 2), j = i % (D / 2);
    const double f = pow(static_cast<double>(theta_base), -2.0 * j / D) * 0.15915494309189535;
    rope_turn(static_cast<int>(p0) + r, f, &s_s[r][j], &s_c[r][j]);
  }
  __syncthreads();
  // q heads of the group; a token without a place gets zeros
  for (int i = tid; i < G * (r1 - r0) * (D / 2); i += kAppThreads) {
    const int j = i % (D / 2), r = r0 + (i / (D / 2)) % (r1 - r0), g = i / (D / 2) / (r1 - r0);
    const size_t tok = row0 + (r - r0);
    const float2 x = *reinterpret_cast<const float2*>(
        qkv + (tok * slots + kvh * G + g) * D + 2 * j);
    float2 y = make_float2(0.0f, 0.0f);
    if (r < rs) {
      y.x = static_cast<float>(x.x * s_c[r][j] - x.y * s_s[r][j]);
      y.y = static_cast<float>(x.x * s_s[r][j] + x.y * s_c[r][j]);
    }
    *reinterpret_cast<float2*>(q_out + (tok * H + kvh * G + g) * D + 2 * j) = y;
  }
  if (rs <= r0) return;
  // k (side 0) and v (side 1): the exponent that the new rows need, then the codes
  for (int side = 0; side < 2; ++side) {
    int e = kNoExp;
    for (int i = tid; i < (rs - r0) * (D / 2); i += kAppThreads) {
      const int j = i % (D / 2), r = r0 + i / (D / 2);
      const float2 x = *reinterpret_cast<const float2*>(
          qkv + ((row0 + (r - r0)) * slots + H + side * c.Hkv + kvh) * D + 2 * j);
      double y0 = x.x, y1 = x.y;
      if (side == 0) {
        y0 = x.x * s_c[r][j] - x.y * s_s[r][j];
        y1 = x.x * s_s[r][j] + x.y * s_c[r][j];
      }
      e = max(e, max(need_exp(y0), need_exp(y1)));
    }
    e = __reduce_max_sync(0xffffffffu, e);
    if (tid % 32 == 0) atomicMax(&s_e[side], e);
    __syncthreads();
    float* sp = (side ? c.v_scale : c.k_scale) +
                (static_cast<size_t>(b) * ((c.S_max + kQ8Block - 1) / kQ8Block) + blk) * c.Hkv +
                kvh;
    int8_t* codes = (side ? c.v : c.k) + ((static_cast<size_t>(b) * c.S_max + p0) * c.Hkv + kvh) * D;
    const size_t ld = static_cast<size_t>(c.Hkv) * D;
    const float was = r0 > 0 ? *sp : 0.0f;
    const int en = s_e[side];
    const float need = en == kNoExp ? 0.0f : en == kBadExp ? __int_as_float(0x7FC00000) : exp_scale(en);
    const float now = (was != was || need != need) ? __int_as_float(0x7FC00000) : fmaxf(was, need);
    __syncthreads();
    if (tid == 0) *sp = now;
    const bool fine = now > 0.0f;  // neither zero nor NaN
    if (r0 > 0 && fine && was > 0.0f && was < now) {
      const float ratio = was / now;
      for (int i = tid; i < r0 * D; i += kAppThreads) {
        int8_t* p = codes + (i / D) * ld + i % D;
        *p = static_cast<int8_t>(__float2int_rn(*p * ratio));
      }
    }
    const double inv = fine ? 1.0 / static_cast<double>(now) : 0.0;
    for (int i = tid; i < (rs - r0) * (D / 2); i += kAppThreads) {
      const int j = i % (D / 2), r = r0 + i / (D / 2);
      const float2 x = *reinterpret_cast<const float2*>(
          qkv + ((row0 + (r - r0)) * slots + H + side * c.Hkv + kvh) * D + 2 * j);
      double y0 = x.x, y1 = x.y;
      if (side == 0) {
        y0 = x.x * s_c[r][j] - x.y * s_s[r][j];
        y1 = x.x * s_s[r][j] + x.y * s_c[r][j];
      }
      char2 q = make_char2(0, 0);
      if (fine)
        q = make_char2(static_cast<signed char>(__double2int_rn(y0 * inv)),
                       static_cast<signed char>(__double2int_rn(y1 * inv)));
      *reinterpret_cast<char2*>(codes + r * ld + 2 * j) = q;
    }
  }
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
  // blocks that n rows from anywhere inside a block can touch
  const int window = static_cast<int>((static_cast<long long>(n) + 2 * (kQ8Block - 1)) / kQ8Block);
  return launch_pdl(k_append_q8, dim3(static_cast<unsigned>(window) * c.B, c.Hkv), kAppThreads, 0, s,
                    qkv, c, n, H, pos, pos_dev, theta_base, q_out, window);
}

cudaError_t launch_read_q8(const Q8Cache& c, int first, const int* first_dev, int count,
                           float* k_out, float* v_out, cudaStream_t s) {
  const size_t total = static_cast<size_t>(c.B) * count * c.Hkv * (D / 4);
  return launch_pdl(k_read_q8, dim3(static_cast<unsigned>((total + 255) / 256)), 256, 0, s, c, first,
                    first_dev, count, k_out, v_out, total);
}

}  // namespace obn
