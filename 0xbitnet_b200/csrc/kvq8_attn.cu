// kvq8_attn.cu — attention over the 8-bit KV cache for few query rows (decode, drafted tokens).
//
// softmax(q . k s_k * scale) v s_v with int8 codes k, v and a power-of-two scale per 16 keys.
// The pass has to read 2 * 128 bytes a key and KV head; everything else is arranged so that
// the HBM is what it waits for:
//
//  * Both products run on the int8 tensor cores (mma.sync m16n8k32, exact s32 sums) with the
//    codes as they lie in memory. The f32 side is cut into four 8-bit digits, which are rows
//    of the same MMA: 4 query rows x 4 digits fill its M = 16. q is a 31-bit fixed point
//    number against its row's largest element (balanced digits, s8); a weight
//    p = 2^(s - M) <= 1 is one of 31 bits against M >= the running maximum (u8 digits). So
//    nothing is rounded between q and the output to fewer than 24 bits, and an int8 MMA does
//    the work that two f16 MMAs (hi and lo halves) and a conversion of every code would.
//  * A weight's digits are an A fragment and the scores of the same keys an accumulator: the
//    reduction over digits leaves lane (quad q, digit j) the score of key 4q + j, and a 4 x 4
//    byte transpose over the four digit lanes (two shuffles) turns weights into digits.
//    K needs no rearrangement (dims may be contracted in any order), V a 4 x 4 byte transpose
//    in registers (8 byte permutes for 16 keys x 4 dims).
//  * The s32 sums are carried along the keys and only turned into f32 (and rescaled) when
//    the reference M has to grow, when a larger value scale comes, or after 2^15 keys (255 *
//    128 * 2^15 < 2^31). M is a whole number above the maximum, so that is rare.
//  * Each warp takes its own 32 keys of a 128-key unit, with its own cp.async ring and its own
//    softmax state; there is no barrier in the loop (more than 4 query rows: MT warps share a
//    ring, one named barrier a step). Four states are merged per pair in shared memory.
#include "kvq8.h"

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "kvq8_sched.cuh"

namespace obn {

int num_sms_cached();                                  // kernels.cu
cudaError_t ensure_smem(const void* fn, size_t bytes);  // kernels.cu

namespace {

constexpr int D = kQ8HeadDim;
constexpr int kKw = 4;                     // key slices of a unit, one warp (group) each
constexpr int kSliceKeys = kUnitKeys / kKw;  // 32: the PV MMA's K
constexpr int kStages = 2;
constexpr int kStageBytes = 2 * kSliceKeys * D + 64;  // K, V, four scales (padded)
constexpr int kFlushUnits = 1024;          // 2^15 keys of a slice: 255 * 128 * 2^15 < 2^31

template <int MT>
struct DecSmem {
  alignas(16) uint8_t ring[kKw][kStages][kStageBytes];
  float o[kKw][4 * MT][D];
  float m[kKw][4 * MT], l[kKw][4 * MT];
  long long sh[128 * MT + 4];
};

OBN_DEVINL void cp16(uint32_t dst, const void* src, bool full) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(full ? 16 : 0)
               : "memory");
}
OBN_DEVINL void cp4(uint32_t dst, const void* src, bool full) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
               "r"(full ? 4 : 0)
               : "memory");
}
OBN_DEVINL void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
OBN_DEVINL void mma_u8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
OBN_DEVINL float shx(float v, int m) { return __shfl_xor_sync(0xffffffffu, v, m); }
OBN_DEVINL uint32_t shxu(uint32_t v, int m) { return __shfl_xor_sync(0xffffffffu, v, m); }

// Codes of 4 keys (rows r) x 4 dims -> 4 dims x 4 keys.
OBN_DEVINL void transpose4(uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3, uint32_t (&o)[4]) {
  const uint32_t a = __byte_perm(r0, r1, 0x5140), b = __byte_perm(r0, r1, 0x7362);
  const uint32_t c = __byte_perm(r2, r3, 0x5140), d = __byte_perm(r2, r3, 0x7362);
  o[0] = __byte_perm(a, c, 0x5410);
  o[1] = __byte_perm(a, c, 0x7632);
  o[2] = __byte_perm(b, d, 0x5410);
  o[3] = __byte_perm(b, d, 0x7632);
}

template <int MT>
__global__ __launch_bounds__(128 * MT, MT == 1 ? 3 : MT == 2 ? 2 : 1) void k_attn_q8_few(
    const float* __restrict__ q, Q8Cache c, Q8Sched sc, float scale_log2, float* __restrict__ out,
    float* __restrict__ ws) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  DecSmem<MT>& sm = *reinterpret_cast<DecSmem<MT>*>(smem_raw);
  constexpr int kThreads = 128 * MT, kRows = 4 * MT;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kw = warp / MT, mt = warp % MT;
  const int grp = lane >> 2, qd = lane & 3, dig = grp & 3, qb = grp >> 2;
  const int H = sc.G * c.Hkv, rows_seq = sc.n * sc.G;

  long long front;
  const long long total = q8_total<kThreads>(sc, 0, &front, sm.sh);
  const int ctas = q8_ctas(sc, total);
  if (static_cast<int>(blockIdx.x) >= ctas) return;
  const long long u0 = q8_begin(total, ctas, blockIdx.x);
  const int mine = static_cast<int>(q8_begin(total, ctas, blockIdx.x + 1) - u0);
  Q8Cursor cur = q8_find<kThreads>(sc, u0, sm.sh);
  Q8Cursor pre = cur;

  const size_t ld = static_cast<size_t>(c.Hkv) * D;
  const int nblk = (c.S_max + kQ8Block - 1) / kQ8Block;
  uint8_t* ring = sm.ring[kw][0];
  // Requests slice kw of the unit at `pre` into stage st: rows of 128 bytes as 16-byte pieces,
  // swizzled so that the fragment loads below meet no bank conflicts.
  auto request = [&](int st) {
    const int b = pre.item / sc.tiles;
    const int len = q8_len(sc, b);
    const int k0 = pre.unit * kUnitKeys + kw * kSliceKeys;
    if (k0 < len) {
      const size_t base = (static_cast<size_t>(b) * c.S_max * c.Hkv + pre.kvh) * D;
      const uint32_t dst = smem_u32(ring + st * kStageBytes);
#pragma unroll
      for (int j = 0; j < 8 / MT; ++j) {
        const int i = mt * 32 + lane + j * 32 * MT;
        const int row = i >> 3, ch = i & 7;
        const bool in = k0 + row < len;
        const size_t off = base + static_cast<size_t>(in ? k0 + row : 0) * ld + ch * 16;
        cp16(dst + row * D + ((ch ^ ((row & 1) << 2)) << 4), c.k + off, in);
        cp16(dst + kSliceKeys * D + row * D + ((ch ^ (((row >> 2) & 3) << 1)) << 4), c.v + off,
             in);
      }
      if (mt == 0 && lane < 4) {  // scales of the slice's two blocks: k, k, v, v
        const int blk = k0 / kQ8Block + (lane & 1);
        const bool in = blk * kQ8Block < len;
        const size_t off = (static_cast<size_t>(b) * nblk + (in ? blk : 0)) * c.Hkv + pre.kvh;
        cp4(dst + 2 * kSliceKeys * D + lane * 4, (lane < 2 ? c.k_scale : c.v_scale) + off, in);
      }
    }
    q8_next(sc, pre);
  };

  int issued = 0;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    if (issued < mine) request(s);
    ++issued;
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // byte selectors of the digit transpose
  const uint32_t sel1 = (dig & 2) ? 0x3276u : 0x5410u;  // (own, other)
  const uint32_t sel2 = (dig & 1) ? 0x3715u : 0x6240u;
  const float dig_w = __int_as_float((127 + 8 * dig) << 23);       // 256^digit
  const float dig_v = __int_as_float((127 - 31 + 8 * dig) << 23);  // 256^digit / 2^31
  int acc[16][4];
  float o[4][4];
  float M[2], l[2], Vr = 0.0f, sq[2];
  int lim[2], since = 0;
  uint32_t aq[4][4];
  bool fresh = true;

  // The s32 sums into f32: value = sum over digits of 256^digit * sum, each lane keeping the
  // dims of its own digit number. Then everything moves to the reference Mn.
  auto flush = [&](float mn0, float mn1, float vn) {
    const float c0 = M[0] == mn0 ? 1.0f : exp2f(M[0] - mn0);
    const float c1 = M[1] == mn1 ? 1.0f : exp2f(M[1] - mn1);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float h[2][4];
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float lo = static_cast<float>(acc[4 * w + e][i]) * dig_v;
          const float hi = static_cast<float>(acc[4 * w + 2 + e][i]) * dig_v;
          const float keep = (dig & 2) ? hi : lo, send = (dig & 2) ? lo : hi;
          h[e][i] = keep + shx(send, 8);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float keep = (dig & 1) ? h[1][i] : h[0][i], send = (dig & 1) ? h[0][i] : h[1][i];
        const float v = keep + shx(send, 4);
        o[w][i] = fmaf(v, Vr, o[w][i]) * (i < 2 ? c0 : c1);
      }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0;
    l[0] *= c0;
    l[1] *= c1;
    M[0] = mn0;
    M[1] = mn1;
    Vr = vn;
    since = 0;
  };

  int u_first = cur.unit;
  for (int it = 0; it < mine; ++it) {
    if (fresh) {  // a new pair: its query rows as digits
      fresh = false;
      u_first = cur.unit;
      const int b = cur.item / sc.tiles, tile = cur.item - b * sc.tiles;
      const int len = q8_len(sc, b);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = tile * kRows + mt * 4 + qb + 2 * h;
        const bool real = row < rows_seq;
        const int t = real ? row / sc.G : 0, g = real ? row - t * sc.G : 0;
        const float* src =
            q + ((static_cast<size_t>(b) * sc.n + t) * H + cur.kvh * sc.G + g) * D + 16 * qd;
        float4 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[i] = real ? *reinterpret_cast<const float4*>(src + (i >= 4 ? 48 : 0) + 4 * i)
                      : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        // the largest magnitude's bits: an infinity or NaN shows as exponent 255
        uint32_t big = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          big = max(big, max(max(__float_as_uint(x[i].x) & 0x7FFFFFFFu,
                                 __float_as_uint(x[i].y) & 0x7FFFFFFFu),
                             max(__float_as_uint(x[i].z) & 0x7FFFFFFFu,
                                 __float_as_uint(x[i].w) & 0x7FFFFFFFu)));
        }
        big = max(big, shxu(big, 1));
        big = max(big, shxu(big, 2));
        const bool bad = big >= 0x7F800000u;
        const int ex = max(static_cast<int>(big >> 23) - 126, -90);  // |x| < 2^ex
        const float up = bad ? 0.0f : __int_as_float((127 + 30 - ex) << 23);
        sq[h] = bad ? __int_as_float(0x7FC00000) : __int_as_float((127 + ex - 30) << 23);
        sq[h] *= scale_log2;
        lim[h] = real ? min(len, q8_limit(sc, len, row)) : 0;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const float4 y = x[ks + 4 * s];
            auto digits = [&](float v) {
              return (static_cast<uint32_t>(bad ? 0 : __float2int_rn(v * up)) + 0x00808080u) ^
                     0x00808080u;
            };
            const uint32_t pick = dig | ((4 + dig) << 4);
            const uint32_t xy = __byte_perm(digits(y.x), digits(y.y), pick);
            const uint32_t zw = __byte_perm(digits(y.z), digits(y.w), pick);
            aq[ks][h + 2 * s] = __byte_perm(xy, zw, 0x5410);
          }
        M[h] = -INFINITY;
        l[h] = 0.0f;
      }
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[w][i] = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0;
      Vr = 0.0f;
      since = 0;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    if (MT == 1)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(1 + kw), "r"(32 * MT) : "memory");
    if (issued < mine) request(issued % kStages);
    ++issued;
    asm volatile("cp.async.commit_group;" ::: "memory");

    const uint8_t* st = ring + (it % kStages) * kStageBytes;
    const int k0 = cur.unit * kUnitKeys + kw * kSliceKeys;
    const int most = __reduce_max_sync(0xffffffffu, max(lim[0], lim[1]));
    if (k0 < most) {
      const float* scl = reinterpret_cast<const float*>(st + 2 * kSliceKeys * D);
      float s[2][2];  // [16-key block][query half]
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        int cc[2][4] = {};
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          // column grp of tile t is key 4 (grp / 2) + 2 t + grp % 2 of the block
          const int row = kb * 16 + 4 * (grp >> 1) + 2 * t + (grp & 1);
          const uint4 ka = *reinterpret_cast<const uint4*>(st + row * D + ((qd ^ ((row & 1) << 2)) << 4));
          const uint4 kc =
              *reinterpret_cast<const uint4*>(st + row * D + (((qd + 4) ^ ((row & 1) << 2)) << 4));
          mma_s8(cc[t], aq[0], ka.x, kc.x);
          mma_s8(cc[t], aq[1], ka.y, kc.y);
          mma_s8(cc[t], aq[2], ka.z, kc.z);
          mma_s8(cc[t], aq[3], ka.w, kc.w);
        }
        float h4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = static_cast<float>(cc[0][i]) * dig_w, b = static_cast<float>(cc[1][i]) * dig_w;
          h4[i] = ((dig & 2) ? b : a) + shx((dig & 2) ? a : b, 8);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float a = h4[2 * h], b = h4[2 * h + 1];
          s[kb][h] = ((dig & 1) ? b : a) + shx((dig & 1) ? a : b, 4);
        }
      }
      const float sk[2] = {scl[0], scl[1]}, sv[2] = {scl[2], scl[3]};
      const int key0 = k0 + 4 * qd + dig;  // of block 0; block 1: + 16
      bool seen[2][2], grow = since >= kFlushUnits;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          seen[kb][h] = key0 + 16 * kb < lim[h];
          // an overflowed score stays the largest or smallest number, a NaN stays one
          const float x = s[kb][h] * (sq[h] * sk[kb]);
          s[kb][h] = !seen[kb][h] ? -INFINITY : x > FLT_MAX ? FLT_MAX : x < -FLT_MAX ? -FLT_MAX : x;
          grow |= s[kb][h] > M[h];
        }
        grow |= k0 + 16 * kb < most && sv[kb] > Vr;
      }
      if (__any_sync(0xffffffffu, grow)) {
        float mn[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float m = fmaxf(s[0][h], s[1][h]);
#pragma unroll
          for (int d = 1; d <= 8; d <<= 1) m = fmaxf(m, shx(m, d));
          mn[h] = m > M[h] ? ceilf(m) + 1.0f : M[h];
        }
        float vn = Vr;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
          if (k0 + 16 * kb < most) vn = fmaxf(vn, sv[kb]);
        flush(mn[0], mn[1], vn);
      }
      const float inv_vr = Vr > 0.0f ? 1.0f / Vr : 0.0f;
      uint32_t ap[4];  // A fragment: [query half + 2 * block]
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        // a finite scale adds 0, a NaN one poisons the total
        const float poison = sv[kb] - sv[kb], f = sv[kb] * inv_vr * 2147483648.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float p = 0.0f;
          if (seen[kb][h]) {
            p = exp2f(s[kb][h] - M[h]);
            l[h] += p + poison;
          }
          const uint32_t w = __float2uint_rn(p * f);
          const uint32_t x = __byte_perm(w, shxu(w, 8), sel1);
          ap[h + 2 * kb] = __byte_perm(x, shxu(x, 4), sel2);
        }
      }
      const uint8_t* sv_rows = st + kSliceKeys * D;
      uint4 vr[2][4];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          vr[kb][i] = *reinterpret_cast<const uint4*>(sv_rows + (kb * 16 + 4 * qd + i) * D +
                                                      ((grp ^ (qd << 1)) << 4));
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        auto word = [&](const uint4& v) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; };
        uint32_t b0[4], b1[4];
        transpose4(word(vr[0][0]), word(vr[0][1]), word(vr[0][2]), word(vr[0][3]), b0);
        transpose4(word(vr[1][0]), word(vr[1][1]), word(vr[1][2]), word(vr[1][3]), b1);
#pragma unroll
        for (int e = 0; e < 4; ++e) mma_u8(acc[4 * w + e], ap, b0[e], b1[e]);
      }
      ++since;
    }

    const bool pair_ends = cur.unit + 1 == cur.units;
    if (pair_ends || it + 1 == mine) {  // merge the four slices, write the pair or its part
      flush(M[0], M[1], Vr);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int d = 1; d <= 8; d <<= 1) l[h] += shx(l[h], d);
        const int row = mt * 4 + qb + 2 * h;
        if ((lane & 15) == 0) {
          sm.m[kw][row] = M[h];
          sm.l[kw][row] = l[h];
        }
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            sm.o[kw][row][32 * qd + 16 * i + 4 * w + dig] = o[w][2 * h + i];
      }
      __syncthreads();
      const bool whole = pair_ends && u_first == 0;
      const int b = cur.item / sc.tiles, tile = cur.item - b * sc.tiles;
      const int slot = 2 * blockIdx.x + (u_first == 0 ? 1 : 0);
      float* po = whole ? nullptr : q8_part_o(ws, kRows, slot);
      float* pml = whole ? nullptr : q8_part_ml(ws, kRows, slot);
      for (int i = tid; i < kRows * (D / 4); i += kThreads) {
        const int row = i / (D / 4), d4 = i % (D / 4) * 4;
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < kKw; ++k) m = fmaxf(m, sm.m[k][row]);
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float lt = 0.0f;
#pragma unroll
        for (int k = 0; k < kKw; ++k) {
          // a slice that saw nothing has l = 0 and o = 0; its M is -inf or (NaN scores) kept
          const float e = sm.m[k][row] == m ? 1.0f : exp2f(sm.m[k][row] - m);
          const float4 x = *reinterpret_cast<const float4*>(&sm.o[k][row][d4]);
          lt = fmaf(sm.l[k][row], e, lt);
          y.x = fmaf(x.x, e, y.x);
          y.y = fmaf(x.y, e, y.y);
          y.z = fmaf(x.z, e, y.z);
          y.w = fmaf(x.w, e, y.w);
        }
        const int r = tile * kRows + row;
        if (whole) {
          if (r < rows_seq) {
            const int t = r / sc.G, g = r - t * sc.G;
            const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;  // no key: zeros
            *reinterpret_cast<float4*>(
                out + ((static_cast<size_t>(b) * sc.n + t) * H + cur.kvh * sc.G + g) * D + d4) =
                make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
          }
        } else {
          *reinterpret_cast<float4*>(po + row * D + d4) = y;
          if (d4 == 0) {
            pml[row] = m;
            pml[kRows + row] = lt;
          }
        }
      }
      __syncthreads();
      fresh = true;
    }
    if (it + 1 < mine) q8_next(sc, cur);
  }
}

// Joins the parts of the pairs that span CTAs, and zeroes the pairs without keys. One CTA per
// pair and row: four warps take every fourth part, a lane four dims.
__global__ __launch_bounds__(128) void k_q8_join(Q8Sched sc, const float* __restrict__ ws_,
                                                 float* __restrict__ out) {
  __shared__ long long sh[128 + 4];
  __shared__ float s_m[4], s_l[4];
  __shared__ float4 s_o[4][32];
  float* ws = const_cast<float*>(ws_);
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x % sc.tile_rows, kvh = blockIdx.y;
  const int item = blockIdx.x / sc.tile_rows;
  const int b = item / sc.tiles, tile = item - b * sc.tiles;
  const int r = tile * sc.tile_rows + row;
  if (r >= sc.n * sc.G) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t = r / sc.G, g = r - t * sc.G;
  float* dst = out + ((static_cast<size_t>(b) * sc.n + t) * (sc.G * sc.Hkv) + kvh * sc.G + g) * D;
  const int units = q8_units(sc, item);
  if (units == 0) {
    if (warp == 0) *reinterpret_cast<float4*>(dst + 4 * lane) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    return;
  }
  long long front;
  const long long total = q8_total<128>(sc, item, &front, sh);
  const long long x0 = front + static_cast<long long>(kvh) * units;
  const int ctas = q8_ctas(sc, total);
  const int c0 = q8_owner(total, ctas, x0), c1 = q8_owner(total, ctas, x0 + units - 1);
  if (c0 == c1) return;  // written by its CTA
  float m = -INFINITY, l = 0.0f;
  float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int c = c0 + warp; c <= c1; c += 4) {
    const int slot = 2 * c + (c == c0 ? 1 : 0);
    const float* ml = q8_part_ml(ws, sc.tile_rows, slot);
    const float pm = ml[row], pl = ml[sc.tile_rows + row];
    const float4 x = *reinterpret_cast<const float4*>(q8_part_o(ws, sc.tile_rows, slot) + row * D + 4 * lane);
    const float mn = fmaxf(m, pm);
    const float e0 = m == mn ? 1.0f : exp2f(m - mn), e1 = pm == mn ? 1.0f : exp2f(pm - mn);
    l = l * e0 + pl * e1;
    y = make_float4(y.x * e0 + x.x * e1, y.y * e0 + x.y * e1, y.z * e0 + x.z * e1,
                    y.w * e0 + x.w * e1);
    m = mn;
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  s_o[warp][lane] = y;
  __syncthreads();
  if (warp) return;
  m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  l = 0.0f;
  y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float e = s_m[w] == m ? 1.0f : exp2f(s_m[w] - m);
    const float4 x = s_o[w][lane];
    l += s_l[w] * e;
    y = make_float4(y.x + x.x * e, y.y + x.y * e, y.z + x.z * e, y.w + x.w * e);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<float4*>(dst + 4 * lane) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
}

template <int MT>
cudaError_t launch_few(const float* q, const Q8Cache& c, Q8Sched sc, float scale_log2, float* out,
                       float* ws, cudaStream_t s) {
  const size_t smem = sizeof(DecSmem<MT>);
  cudaError_t e = ensure_smem(reinterpret_cast<const void*>(&k_attn_q8_few<MT>), smem);
  if (e != cudaSuccess) return e;
  const long long bound = static_cast<long long>(sc.B) * sc.tiles * sc.Hkv *
                          ((sc.seq_len + kUnitKeys - 1) / kUnitKeys);
  const long long fit = static_cast<long long>(num_sms_cached()) * (MT == 1 ? 3 : MT == 2 ? 2 : 1);
  sc.ctas = static_cast<int>(std::min<long long>(std::max<long long>(std::min(bound, fit), 1), kQ8MaxCtas));
  e = launch_pdl(&k_attn_q8_few<MT>, dim3(sc.ctas), 128 * MT, smem, s, q, c, sc, scale_log2, out, ws);
  if (e != cudaSuccess) return e;
  return launch_pdl(k_q8_join, dim3(sc.B * sc.tiles * sc.tile_rows, sc.Hkv), 128, 0, s, sc, ws, out);
}

}  // namespace

size_t attention_q8_workspace_bytes(int B, int n, int H, int Hkv, int S_max) {
  (void)B, (void)n, (void)H, (void)Hkv, (void)S_max;
  return q8_workspace(16);
}

cudaError_t launch_attention_q8(const float* q, const Q8Cache& c, int n, int H, int seq_len,
                                const int* lens_dev, float scale, float* out, void* workspace,
                                cudaStream_t s) {
  Q8Sched sc = {c.B, n, H / c.Hkv, c.Hkv, 0, 0, seq_len, lens_dev, 0};
  const long long rows = static_cast<long long>(n) * sc.G;
  const float scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  sc.tile_rows = rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
  sc.tiles = static_cast<int>((rows + sc.tile_rows - 1) / sc.tile_rows);
  float* ws = static_cast<float*>(workspace);
  if (sc.tile_rows == 4) return launch_few<1>(q, c, sc, scale_log2, out, ws, s);
  if (sc.tile_rows == 8) return launch_few<2>(q, c, sc, scale_log2, out, ws, s);
  return launch_few<4>(q, c, sc, scale_log2, out, ws, s);
}

}  // namespace obn
