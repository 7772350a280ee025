// kvq8_many.cu — attention over the 8-bit KV cache for many query rows (prefill chunks).
//
// Here the tensor cores bound the pass: 4 * 128 operations per query row and key. They run as
// tcgen05.mma kind::f16 with f32 accumulators in tensor memory. The codes are whole numbers up
// to 127 and exact in f16; q and the weights are f32, so each is an f16 high part and the f16 of
// what is left (x = hi + lo to 2^-22), two MMAs for one. (kind::i8 has twice the rate, but
// three digits and an s32 accumulator for each of them: more tensor memory than there is.)
//
// One CTA per SM works on a pair of tiles, 2 x 128 query rows (token, group head) of a sequence
// and KV head, so every converted key block serves 256 rows, and on units of 128 keys
// (kvq8_sched.cuh). Roles, 21 warps:
//   warps 0-7, 8-15  softmax of tile A, B: two threads a row, 64 keys (and 64 dims of O) each. S
//                    from tensor memory twice (maximum; weights), the weights back over S as the
//                    A operand of the second product.
//   warps 16-19      codes to f16: TMA staging -> registers -> shared memory in the MMA's layout;
//                    V is transposed on the way. The staging is requested again as soon as
//                    it is read.
//   warp 20          issues the MMAs, in the order  PV_A(u) QK_A(u+1) PV_B(u) QK_B(u+1): while
//                    one tile's softmax runs, the other tile's products do.
// Tensor memory: S (and P) of A and B, 2 x 128 columns, O of A and B, 2 x 128.
//
// Softmax. With s = q.k, f = scale of q, key block and log2 e, v's block scale 2^lv: a weight
// is w = 2^(s f + lv - R), so its f16 pair is as exact as the contribution it makes is large,
// whatever the scales of other blocks, and O adds w times codes. R moves only when a row's
// maximum of s f + lv exceeds it by 15 (w <= 2^15 fits f16); then O is rescaled in
// tensor memory. The total is the sum of w 2^(lv0 - lv), exact factors, lv0 fixed for a part, while
// every value scale of the part lies within 2^32 of 2^lv0: its reference is T = R - lv0 then, and no
// weight that counts is flushed (R <= max s f + lv0 + 26, so a score 60 below the largest still has
// w >= 2^-118). From the first unit with a scale farther off, or with a block of zeros (whose keys
// have weight but no product) or a scale that is no power of two, the rest of the part is `far`:
// the total has exponentials and a reference T of its own, moved like R but by the scores alone, R
// goes by the blocks that are not zero, and the weights are multiplied by the scale's mantissa.
// The tensor cores truncate when they add to an accumulator, a bias of 1.5e-7 of O for every
// unit: after kDrain units O moves to an f32 copy in the workspace (L2) and starts anew.
//
// 2048 tokens of 20/5 heads over 6144 keys (107 GFLOP, twice that with the low halves): 252 us from
// cold caches, the join among them, 0.43 PFLOP/s, 0.85 with the low halves (244 us before far scales
// had code). A unit takes about 9100 cycles (taken when a call took 222 us with a warm L2), its
// products 5200: a tile's scores and weights share tensor memory, so its softmax (maximum 900,
// exchange 600, weights 2700, copies 1100 cycles) and its products (2600) follow one another, and
// the other tile's products fill only half of the softmax. 512 rows over 2100 keys: 47 us; a pair's
// query rows and its output cost 8000 cycles each there, as much as two of a CTA's three units.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include <cuda_fp16.h>

#include "kvq8_sched.cuh"

namespace obn {

int num_sms_cached();  // kernels.cu

namespace {

constexpr int D = kQ8HeadDim;
constexpr int kRows = 256;       // query rows of a CTA's pair of tiles
constexpr int kThreads = 672;
// Units between O's moves to its copy. Error against 64 bits (512 rows over 2100 keys, 2048 over
// 6144) and time of the latter with a warm L2, when this was chosen: 2 units 1.3e-6, 1.4e-6, 236 us;
// 3: 1.5e-6, 1.6e-6, 227 us; 4: 1.7e-6, 1.9e-6, 219 us; 8: 2.9e-6. An f32 softmax and product of the
// same values: 1.3e-6, 1.7e-6, so 512 rows are a little above it and 2048 a little below.
constexpr int kDrain = 3;
constexpr float kNear = 32.0f;  // how far from lv0 a value scale's exponent may be
constexpr float kNoExp = -1000.0f;  // the exponent of a scale of zero
constexpr int kStart = 2;  // places that a pair's query rows and outputs are worth
constexpr int kManyMaxCtas = 160;
constexpr int kHalf = 128 * 128;  // bytes of 128 rows x 64 f16, the swizzle's width

struct ManySmem {
  uint8_t q[2][2][2 * kHalf];  // [tile][hi, lo][dims 0-63, 64-127]
  uint8_t k[2 * kHalf];        // 128 keys x 128 dims
  uint8_t v[2 * kHalf];        // 128 dims x 128 keys
  uint8_t k_in[kUnitKeys * D], v_in[kUnitKeys * D];
  uint64_t kin_full, vin_full, kin_read, vin_read;
  uint64_t k_full, k_free, v_full, v_free;
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
  uint64_t swap[2][4];         // two threads of a row exchange a value
  float swapped[2][2][128];    // [tile][half][row]
  int16_t q_exp[2][128];       // rows of q are scaled by 2^(14 - exponent)
  uint64_t staged[2];          // rows of O on their way out
  uint64_t drain;
  uint32_t tmem_base;
  volatile int abort_flag;
  long long sh[kThreads / 32 + 8];
};
static_assert(sizeof(ManySmem) <= 227 * 1024, "shared memory");

constexpr uint32_t kIdesc = (1u << 4) | (static_cast<uint32_t>(128 >> 3) << 17) |
                            (static_cast<uint32_t>(128 >> 4) << 24);  // f32 = f16 x f16, 128 x 128

// One MMA, issued by the lane with `one` set while the whole warp runs the same code: operands
// then stay in uniform registers. (512 MMAs of 128 x 128 x 16 back to back: 106 cycles each from
// one thread in a branch, 68 like this with A in shared memory and 93 with A in tensor memory.)
OBN_DEVINL void mma_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t accumulate,
                       uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(kIdesc), "r"(accumulate), "r"(one)
      : "memory");
}
OBN_DEVINL void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t accumulate,
                       uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(kIdesc), "r"(accumulate), "r"(one)
      : "memory");
}
OBN_DEVINL uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r;
}

// The key at position (row of K, k index of V) r of a unit: within a group of 8 keys a the
// order is rotated by a, which keeps the transposing loads of V free of bank conflicts.
OBN_DEVINL int key_at(int r) { return (r & ~7) | ((r + (r >> 3)) & 7); }

// The same for column i of the 32 columns from 32 c on, against their first key.
OBN_DEVINL int key_in_32(int i, int c) { return (i & ~7) | ((i + (i >> 3) + 4 * c) & 7); }

OBN_DEVINL void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// Four signed bytes -> f16: 1024 + (c + 128) in the low mantissa bits, minus 1152.
OBN_DEVINL void bytes_to_half(uint32_t w, uint32_t* h01, uint32_t* h23) {
  const uint32_t u = w ^ 0x80808080u;
  const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
  uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
  __half2 ha = __hsub2(*reinterpret_cast<__half2*>(&a), off);
  __half2 hb = __hsub2(*reinterpret_cast<__half2*>(&b), off);
  *h01 = *reinterpret_cast<uint32_t*>(&ha);
  *h23 = *reinterpret_cast<uint32_t*>(&hb);
}

// q8_wait of the MMA warp, without sleep: it is one warp, and every product waits for it (2048 tokens,
// warm, 227 -> 222 us; softmax warps that spin as well take the slots of those that work: 231 us).
OBN_DEVINL bool mma_wait(volatile int* abort_flag, uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < (1u << 24); ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((i & 63) == 63 && *abort_flag) return false;
  }
  record_error(DEVERR_MBAR_TIMEOUT);
  *abort_flag = 1;
  return false;
}

// The total of a far part, over the 64 scores of a thread's half of a unit: l counts in 2^T, and T
// moves like R. Each half has a T of its own.
OBN_DEVINL void add_far(uint32_t t_s, int hf, float sq, float scl, int seen, float* T, float* l) {
#pragma unroll 1
  for (int b = 4 * hf; b < 4 * hf + 4; ++b) {
    const float f = sq * __shfl_sync(0xffffffffu, scl, b);
    const float sv = __shfl_sync(0xffffffffu, scl, 8 + b);
    uint32_t s[16];
    tmem_ld16(t_s + 16 * (b & 3), s);
    tmem_ld_wait();
    float top = -INFINITY, block = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (32 * (b >> 1) + key_in_32(16 * (b & 1) + i, b >> 1) < seen)
        top = fmaxf(top, __uint_as_float(s[i]) * f);
    if (top > *T + 15.0f) {
      const float to = ceilf(top) - 7.0f;
      *l *= ex2(*T - to);
      *T = to;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (32 * (b >> 1) + key_in_32(16 * (b & 1) + i, b >> 1) < seen)
        block += ex2(fmaf(__uint_as_float(s[i]), f, -*T));
    if (16 * b < seen) *l += block + (sv - sv);  // a poisoned block makes it NaN
  }
}

__global__ __launch_bounds__(kThreads, 1) void k_attn_q8_many(
    const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
    const float* __restrict__ q, const float* __restrict__ k_scale,
    const float* __restrict__ v_scale, int nblk, Q8Sched sc, float scale_log2,
    float* __restrict__ out, float* __restrict__ ws) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  ManySmem* sm = reinterpret_cast<ManySmem*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    mbar_init(&sm->kin_full, 1);
    mbar_init(&sm->vin_full, 1);
    mbar_init(&sm->kin_read, 128);
    mbar_init(&sm->vin_read, 128);
    mbar_init(&sm->k_full, 128);
    mbar_init(&sm->k_free, 1);
    mbar_init(&sm->v_full, 128);
    mbar_init(&sm->v_free, 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(&sm->q_full[x], 256);
      mbar_init(&sm->s_full[x], 1);
      mbar_init(&sm->p_full[x], 256);
      mbar_init(&sm->o_full[x], 1);
      mbar_init(&sm->staged[x], 256);
      for (int i = 0; i < 4; ++i) mbar_init(&sm->swap[x][i], 64);
    }
    mbar_init(&sm->drain, 1);
    sm->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 20) {
    tmem_alloc(&sm->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm->tmem_base;
  pdl_wait();
  pdl_launch_dependents();
  int place;
  long long total;
  Q8Cursor cur = q8_share<kThreads>(sc, blockIdx.x, &place, &total, sm->sh);
  if (tid == 0) q8_note_split(sc, cur, place, total, ws);

  if (cur.left == 0) {
    // nothing for this CTA
  } else if (warp < 16) {
    // ---- softmax: thread = half hf of row `row` of tile x ---------------------------------
    const int x = warp >> 3, hf = (warp >> 2) & 1, row = tid & 127;
    const int H = sc.G * sc.Hkv, rows_seq = sc.n * sc.G;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lane_base + 128 * x + 64 * hf,
                   t_o = tmem + lane_base + 256 + 128 * x + 64 * hf;
    // the copy of O: [4 dims] of this half, row by row
    float4* copy = reinterpret_cast<float4*>(ws + q8_workspace(kRows, kManyMaxCtas) / sizeof(float)) +
                   ((static_cast<size_t>(blockIdx.x) * 2 + x) * 2 + hf) * (16 * 128) + row;
    float R = -INFINITY, l = 0.0f, lv0 = 0.0f /* T in a far part */, sq = 0.0f, scl = 0.0f, copy_R = 0.0f;
    int part_u = 0;  // units of the part so far
    uint32_t swaps = 0, stagings = 0;
    int lim = 0, u_first = 0, r = 0, pairs = 0;
    bool fresh = true, ok = true, far = false;
    // lanes 0-7: the unit's key scales, 8-15: its value scales
    auto load_scale = [&](const Q8Cursor& c) {
      const int blk = c.unit * (kUnitKeys / kQ8Block) + (lane & 7);
      return lane < 16 && blk * kQ8Block < c.len
                 ? __ldg((lane < 8 ? k_scale : v_scale) +
                         (static_cast<size_t>(c.b) * nblk + blk) * sc.Hkv + c.kvh)
                 : 0.0f;
    };
    // this half's value to the other one's thread, and back; false after an abort. The halves change
    // slots each time: a slot is next written by the thread that read it.
    auto exchange = [&](float mine, float* other) {
      sm->swapped[x][hf ^ (swaps & 1)][row] = mine;
      mbar_arrive(&sm->swap[x][warp & 3]);
      const bool came =
          __all_sync(0xffffffffu, q8_wait(&sm->abort_flag, &sm->swap[x][warp & 3], swaps & 1));
      *other = sm->swapped[x][hf ^ 1 ^ (swaps & 1)][row];
      ++swaps;
      return came;
    };
    scl = load_scale(cur);
    for (int u = 0; cur.left > 0; ++u) {
      const int k0 = cur.unit * kUnitKeys;
      Q8Cursor nxt = cur;
      q8_next(sc, nxt);
      if (fresh) {  // 16 rows of q a warp, as f16 hi and lo scaled to below 2^14
        u_first = cur.unit;
        const int row0 = 16 * (warp & 7), qr0 = cur.tile * kRows + 128 * x + row0;
        int t = qr0 / sc.G, g = qr0 - t * sc.G;
        const float* src = q + ((static_cast<size_t>(cur.b) * sc.n + t) * H + cur.kvh * sc.G + g) * D + 4 * lane;
        int exps = 0;  // of row `lane`
#pragma unroll 1
        for (int i0 = 0; i0 < 16; i0 += 8) {
          float4 y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            y[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (qr0 + i0 + i < rows_seq) y[i] = __ldg(reinterpret_cast<const float4*>(src));
            src += D;
            if (++g == sc.G) {  // the next token's
              g = 0;
              src += (H - sc.G) * D;
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            // An infinity or NaN makes the row's high or low halves NaN, hence its scores.
            const float big = fmaxf(fmaxf(fabsf(y[i].x), fabsf(y[i].y)), fmaxf(fabsf(y[i].z), fabsf(y[i].w)));
            const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(big));
            const int ex = max(static_cast<int>(top >> 23) - 126, -90);  // |q| < 2^ex
            const float up = __int_as_float((127 + 14 - ex) << 23);
            exps = lane == i0 + i ? ex : exps;
            const float e[4] = {y[i].x * up, y[i].y * up, y[i].z * up, y[i].w * up};
            uint32_t wh[2], wl[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const __half2 h = __floats2half2_rn(e[2 * j], e[2 * j + 1]);
              const float2 back = __half22float2(h);
              const __half2 m = __floats2half2_rn(e[2 * j] - back.x, e[2 * j + 1] - back.y);
              wh[j] = *reinterpret_cast<const uint32_t*>(&h);
              wl[j] = *reinterpret_cast<const uint32_t*>(&m);
            }
            // 8 bytes of 16-byte chunk (lane / 2) % 8 of the half lane / 16
            const int at = (lane >> 4) * kHalf + (row0 + i0 + i) * 128 +
                           ((((lane >> 1) & 7) ^ (i & 7)) << 4) + (lane & 1) * 8;
            *reinterpret_cast<uint2*>(sm->q[x][0] + at) = make_uint2(wh[0], wh[1]);
            *reinterpret_cast<uint2*>(sm->q[x][1] + at) = make_uint2(wl[0], wl[1]);
          }
        }
        if (lane < 16) sm->q_exp[x][row0 + lane] = static_cast<int16_t>(exps);
        fence_proxy_async_smem();
        mbar_arrive(&sm->q_full[x]);
        ok = __all_sync(0xffffffffu, q8_wait(&sm->abort_flag, &sm->q_full[x], pairs & 1));
        if (!ok) break;
        ++pairs;
        sq = __int_as_float((127 + sm->q_exp[x][row] - 14) << 23) * scale_log2;
        r = cur.tile * kRows + 128 * x + row;
        const bool real = r < rows_seq;
        lim = real ? min(cur.len, q8_limit(sc, cur.len, r)) : 0;
        R = -INFINITY;
        l = 0.0f;
        part_u = 0;
        far = false;
        // the reference of the value scales: the unit's largest exponent
        float top = lane >= 8 && lane < 16 && scl > 0.0f ? scl : 0.0f;
        top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
        lv0 = top > 0.0f ? static_cast<float>(static_cast<int>(__float_as_uint(top) >> 23) - 127) : 0.0f;
      }
      // exponents of the value scales (a poisoned block's: any, it makes the total NaN)
      const float lv_lane =
          scl > 0.0f ? static_cast<float>(static_cast<int>(__float_as_uint(scl) >> 23) - 127)
                     : scl == 0.0f ? kNoExp : lv0;
      const bool held = lane >= 8 && lane < 16 && k0 + kQ8Block * (lane & 7) < cur.len;
      const bool mantissa = scl > 0.0f && (__float_as_uint(scl) & 0x7FFFFFu);
      if (!far && __any_sync(0xffffffffu, held && (fabsf(lv_lane - lv0) > kNear || mantissa))) {
        far = true;
        lv0 = R == -INFINITY ? R : R - lv0;  // what l counts in
      }
      // a block's part of the total counts times this: 2^(lv0 - lv), NaN for a poisoned one
      const float lf_lane = ex2(lv0 - lv_lane) + (scl - scl);
      const float scl_now = scl;
      if (nxt.left > 0) scl = load_scale(nxt);

      const int seen = lim - k0;  // keys of the unit that this row sees
      const bool all = __all_sync(0xffffffffu, seen >= kUnitKeys);  // nothing masked
      ok = __all_sync(0xffffffffu, q8_wait(&sm->abort_flag, &sm->s_full[x], u & 1));
      if (!ok) break;
      tc_fence_after();
      if (__builtin_expect(far, false)) add_far(t_s, hf, sq, scl_now, seen, &lv0, &l);
      // 1. the largest s f + lv of the row. The loops over 16-key blocks stay loops: unrolled, the
      // softmax warps, the converters and the MMA warp evict each other's instructions (both
      // passes unrolled: 8600 cycles a unit; in halves: 5600).
      // Units where nothing is masked or far have code of their own: compiled as one, the masks
      // cost every element two selects and two compares. (With a third version for far parts, in
      // place of add_far, the others ran slower too: 2048 rows 251 -> 276 us, as it is 257.)
      float xr = -INFINITY;
      auto largest = [&](auto clean) {
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t s[32];
          tmem_ld32(t_s + 32 * c, s);
          const int b = 4 * hf + 2 * c;  // 16-key block
          const float f0 = sq * __shfl_sync(0xffffffffu, scl_now, b);
          const float f1 = sq * __shfl_sync(0xffffffffu, scl_now, b + 1);
          const float lv_0 = __shfl_sync(0xffffffffu, lv_lane, 8 + b);
          const float lv_1 = __shfl_sync(0xffffffffu, lv_lane, 9 + b);
          tmem_ld_wait();
          if constexpr (!decltype(clean)::value) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (16 * b + key_in_32(i, b >> 1) >= seen) s[i] = 0xFF800000u;  // -inf
          }
          float m[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            m[i] = __uint_as_float(s[8 * i]);
#pragma unroll
            for (int j = 1; j < 8; ++j) m[i] = fmaxf(m[i], __uint_as_float(s[8 * i + j]));
          }
          const float m0 = fmaxf(m[0], m[1]), m1 = fmaxf(m[2], m[3]);
          xr = fmaxf(xr, m0 == -INFINITY ? -INFINITY : fmaf(m0, f0, lv_0));
          xr = fmaxf(xr, m1 == -INFINITY ? -INFINITY : fmaf(m1, f1, lv_1));
        }
      };
      const bool is_clean = all && !far;
      if (is_clean)
        largest(std::true_type{});
      else
        largest(std::false_type{});
      float xo;
      if (!exchange(xr, &xo)) break;
      xr = fmaxf(xr, xo);
      const bool grow = xr > R + (far ? 14.0f : 15.0f);  // a mantissa is below 2
      const float Rn = grow ? ceilf(xr) - 7.0f : R;
      const float corr = grow ? ex2(R - Rn) : 1.0f;
      const bool drain = part_u > 0 && part_u % kDrain == 0;
      l *= far ? 1.0f : corr;
      if (part_u > 0 && (drain || __any_sync(0xffffffffu, grow))) {
        ok = __all_sync(0xffffffffu, q8_wait(&sm->abort_flag, &sm->o_full[x], (u - 1) & 1));
        if (!ok) break;
        tc_fence_after();
        const bool add = drain && part_u > kDrain;
        if (add && copy_R != R) {  // the copy to the reference R
          const float old = ex2(copy_R - R);
#pragma unroll 4
          for (int i = 0; i < 16; ++i) {
            const float4 z = __ldcg(copy + i * 128);
            __stcg(copy + i * 128, make_float4(z.x * old, z.y * old, z.z * old, z.w * old));
          }
        }
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[16];
          tmem_ld16(t_o + 16 * c, o);
          tmem_ld_wait();
          if (drain) {  // added by the L2, which nobody has to wait for
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float4* at = copy + (4 * c + i) * 128;
              const float4 y = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                           __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
              if (add)
                asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at),
                             "f"(y.x), "f"(y.y), "f"(y.z), "f"(y.w)
                             : "memory");
              else
                __stcg(at, y);
            }
          } else {  // to the new reference
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
            tmem_st16(t_o + 16 * c, o);
          }
        }
        if (drain)
          copy_R = R;
        else
          tmem_st_wait();
      }
      R = Rn;
      ++part_u;
      fresh = false;
      // 2. the weights, over the scores: 8 columns of high and 8 of low halves per 16 keys
      const float Rs = R == -INFINITY ? 0.0f : R;
      auto weights = [&](auto clean) {
#pragma unroll 1
        for (int b = 4 * hf; b < 4 * hf + 4; ++b) {
          uint32_t s[16];
          tmem_ld16(t_s + 16 * (b & 3), s);
          const float f = sq * __shfl_sync(0xffffffffu, scl_now, b);
          const float lv = __shfl_sync(0xffffffffu, lv_lane, 8 + b), base = lv - Rs;
          const float lf = __shfl_sync(0xffffffffu, lf_lane, 8 + b);
          tmem_ld_wait();
          float w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = ex2(fmaf(__uint_as_float(s[i]), f, base));
          if constexpr (!decltype(clean)::value) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (32 * (b >> 1) + key_in_32(16 * (b & 1) + i, b >> 1) >= seen) w[i] = 0.0f;
          }
          float sum[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] = (w[i] + w[i + 4]) + (w[i + 8] + w[i + 12]);
          const float block = (sum[0] + sum[1]) + (sum[2] + sum[3]);
          if (decltype(clean)::value || (!far && 16 * b < seen)) l = fmaf(block, lf, l);
          if constexpr (!decltype(clean)::value) {
            if (far) {
              const float sv = __shfl_sync(0xffffffffu, scl_now, 8 + b);
              const float mantissa =
                  sv > 0.0f ? __uint_as_float((__float_as_uint(sv) & 0x7FFFFFu) | 0x3F800000u) : 0.0f;
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i] = lv == kNoExp ? 0.0f : w[i] * mantissa;
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const __half2 h = __floats2half2_rn(w[2 * i], w[2 * i + 1]);
            const float2 back = __half22float2(h);
            const __half2 m = __floats2half2_rn(w[2 * i] - back.x, w[2 * i + 1] - back.y);
            s[i] = *reinterpret_cast<const uint32_t*>(&h);
            s[8 + i] = *reinterpret_cast<const uint32_t*>(&m);
          }
          tmem_st16(t_s + 16 * (b & 3), s);
        }
      };
      if (is_clean)
        weights(std::true_type{});
      else
        weights(std::false_type{});
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sm->p_full[x]);

      const bool pair_ends = cur.unit + 1 == cur.units;
      if (pair_ends || nxt.left == 0) {  // write the pair or its part
        ok = __all_sync(0xffffffffu, q8_wait(&sm->abort_flag, &sm->o_full[x], u & 1));
        if (!ok) break;
        tc_fence_after();
        float lo;
        if (far) {
          if (!exchange(lv0, &lo)) break;
          const float T = fmaxf(lv0, lo);
          if (lv0 != T) l *= ex2(lv0 - T);
          lv0 = T;
        }
        if (!exchange(l, &lo)) break;
        l = hf ? lo + l : l + lo;
        const bool whole = pair_ends && u_first == 0;
        const int slot = 2 * blockIdx.x + (u_first == 0 ? 1 : 0);
        // O counts in 2^R and the total in 2^T. A total goes on as 1 <= l < 2 times 2^e, and the sums
        // of a part as that much less, so that neither leaves f32's range before the result does.
        const float T = far ? lv0 : R == -INFINITY ? R : R - lv0;
        const int e = l > 0.0f && l <= FLT_MAX ? static_cast<int>(__float_as_uint(l) >> 23) - 127 : 0;
        l *= ex2(static_cast<float>(-e));
        const float up = (R == -INFINITY ? 0.0f : R - T) - static_cast<float>(e);
        const float near_up = fminf(fmaxf(up, -100.0f), 100.0f), rest_up = ex2(up - near_up);
        const float unit = ex2(near_up) * (whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f);
        if (!whole && hf == 0) {
          float* ml = q8_part_ml(ws, kRows, slot);
          ml[128 * x + row] = T + static_cast<float>(e);
          ml[kRows + 128 * x + row] = l;
        }
        const bool copied = part_u > kDrain;
        const float old = copy_R == R ? 1.0f : ex2(copy_R - R);
        // through the query rows' shared memory (nobody needs them any more), so that rows go
        // out whole: [row][dim], 16-byte pieces swizzled
        float* stage = reinterpret_cast<float*>(sm->q[x][0]);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[16];
          tmem_ld16(t_o + 16 * c, o);
          float4 z[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            z[i] = copied ? __ldcg(copy + (4 * c + i) * 128) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 y = copied ? make_float4(fmaf(z[i].x, old, __uint_as_float(o[4 * i])),
                                                  fmaf(z[i].y, old, __uint_as_float(o[4 * i + 1])),
                                                  fmaf(z[i].z, old, __uint_as_float(o[4 * i + 2])),
                                                  fmaf(z[i].w, old, __uint_as_float(o[4 * i + 3])))
                                    : make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                                  __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
            const int piece = 16 * hf + 4 * c + i;
            *reinterpret_cast<float4*>(stage + row * D + 4 * (piece ^ (row & 31))) =
                make_float4(y.x * unit * rest_up, y.y * unit * rest_up, y.z * unit * rest_up,
                            y.w * unit * rest_up);
          }
        }
        mbar_arrive(&sm->staged[x]);
        ok = __all_sync(0xffffffffu, q8_wait(&sm->abort_flag, &sm->staged[x], stagings & 1));
        ++stagings;
        if (!ok) break;
        const int row0 = 16 * (warp & 7), qr0 = cur.tile * kRows + 128 * x + row0;
        const int t0 = qr0 / sc.G;
        int g = qr0 - t0 * sc.G;
        float* dst = 4 * lane + (whole ? out + ((static_cast<size_t>(cur.b) * sc.n + t0) * H +
                                                cur.kvh * sc.G + g) * D
                                       : q8_part_o(ws, kRows, slot) + (128 * x + row0) * D);
        const int to_next = whole ? (H - sc.G) * D : 0;  // from a token's last row
#pragma unroll 4
        for (int i = 0; i < 16; ++i) {
          if (qr0 + i >= rows_seq) break;
          *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(
              stage + (row0 + i) * D + 4 * (lane ^ ((row0 + i) & 31)));
          dst += D;
          if (++g == sc.G) {
            g = 0;
            dst += to_next;
          }
        }
        mbar_arrive(&sm->staged[x]);  // the stage becomes query rows again
        ok = __all_sync(0xffffffffu, q8_wait(&sm->abort_flag, &sm->staged[x], stagings & 1));
        ++stagings;
        if (!ok) break;
        tc_fence_before();
        fresh = true;
      }
      cur = nxt;
    }
    // After an abort: NaN for the rows that this warp would have written (a part's sums, or outputs),
    // of this pair and of the share's others, so that nothing stale passes for a result.
    while (cur.left > 0) {
      Q8Cursor nxt = cur;
      q8_next(sc, nxt);
      const bool pair_ends = cur.unit + 1 == cur.units;
      if (pair_ends || nxt.left == 0) {
        const float nan = __int_as_float(0x7FC00000);
        const int slot = 2 * blockIdx.x + (u_first == 0 ? 1 : 0);
        const int row0 = 128 * x + 16 * (warp & 7);
#pragma unroll 1
        for (int i = row0; i < row0 + 16; ++i) {
          const int qr = cur.tile * kRows + i, t = qr / sc.G;
          if (qr >= rows_seq) break;
          float* dst = pair_ends && u_first == 0
                           ? out + ((static_cast<size_t>(cur.b) * sc.n + t) * H + cur.kvh * sc.G +
                                    (qr - t * sc.G)) * D
                           : q8_part_o(ws, kRows, slot) + static_cast<size_t>(i) * D;
          *reinterpret_cast<float4*>(dst + 4 * lane) = make_float4(nan, nan, nan, nan);
        }
        u_first = 0;
      }
      cur = nxt;
    }
  } else if (warp < 20) {
    // ---- codes to f16 ------------------------------------------------------------------------
    const int ct = tid - 512, cw = ct >> 5;
    auto request = [&](const Q8Cursor& c, const CUtensorMap* map, uint8_t* dst, uint64_t* bar) {
      const int k0 = c.unit * kUnitKeys;
      mbar_arrive_expect_tx(bar, kUnitKeys * D);
      tma_load_4d(smem_u32(dst), map, 0, c.kvh, k0, c.b, bar);
    };
    int k_asked = 0, v_asked = 0, k_got = 0, v_got = 0;
    if (ct == 0) {
      request(cur, &tmap_k, sm->k_in, &sm->kin_full);
      request(cur, &tmap_v, sm->v_in, &sm->vin_full);
      k_asked = v_asked = 1;
    }
    const int k_row = key_at(ct);
    const int a = lane & 15, chunk = 2 * cw + (lane >> 4);  // V: key group, 16 dims
    for (int u = 0; cur.left > 0; ++u) {
      Q8Cursor nxt = cur;
      q8_next(sc, nxt);
      // K: row ct of the operand is key k_row
      if (!q8_wait(&sm->abort_flag, &sm->kin_full, u & 1)) break;
      ++k_got;
      uint4 in[8];
#pragma unroll
      for (int c = 0; c < 8; ++c)
        in[c] = *reinterpret_cast<const uint4*>(sm->k_in + k_row * D + ((c ^ (k_row & 7)) << 4));
      // the next copy writes through the async proxy: without the fence it overtook these loads
      fence_proxy_async_smem();
      mbar_arrive(&sm->kin_read);
      if (ct == 0 && nxt.left > 0) {
        if (!q8_wait(&sm->abort_flag, &sm->kin_read, u & 1)) break;
        request(nxt, &tmap_k, sm->k_in, &sm->kin_full);
        ++k_asked;
      }
      if (u > 0 && !q8_wait(&sm->abort_flag, &sm->k_free, (u - 1) & 1)) break;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint4 h0, h1;
        bytes_to_half(in[c].x, &h0.x, &h0.y);
        bytes_to_half(in[c].y, &h0.z, &h0.w);
        bytes_to_half(in[c].z, &h1.x, &h1.y);
        bytes_to_half(in[c].w, &h1.z, &h1.w);
        uint8_t* dst = sm->k + (c >> 2) * kHalf + ct * 128;
        *reinterpret_cast<uint4*>(dst + (((2 * (c & 3)) ^ (ct & 7)) << 4)) = h0;
        *reinterpret_cast<uint4*>(dst + (((2 * (c & 3) + 1) ^ (ct & 7)) << 4)) = h1;
      }
      fence_proxy_async_smem();
      mbar_arrive(&sm->k_full);
      // V: 8 keys x 16 dims, transposed
      if (!q8_wait(&sm->abort_flag, &sm->vin_full, u & 1)) break;
      ++v_got;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int vr = 8 * a + ((i + a) & 7);
        in[i] = *reinterpret_cast<const uint4*>(sm->v_in + vr * D + ((chunk ^ (vr & 7)) << 4));
      }
      fence_proxy_async_smem();
      mbar_arrive(&sm->vin_read);
      if (ct == 0 && nxt.left > 0) {
        if (!q8_wait(&sm->abort_flag, &sm->vin_read, u & 1)) break;
        request(nxt, &tmap_v, sm->v_in, &sm->vin_full);
        ++v_asked;
      }
      if (u > 0 && !q8_wait(&sm->abort_flag, &sm->v_free, (u - 1) & 1)) break;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        auto word = [&](const uint4& y) { return w == 0 ? y.x : w == 1 ? y.y : w == 2 ? y.z : y.w; };
        uint32_t t0[4], t1[4];
        transpose4(word(in[0]), word(in[1]), word(in[2]), word(in[3]), t0);
        transpose4(word(in[4]), word(in[5]), word(in[6]), word(in[7]), t1);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int dim = 16 * chunk + 4 * w + e;
          uint4 h;
          bytes_to_half(t0[e], &h.x, &h.y);
          bytes_to_half(t1[e], &h.z, &h.w);
          *reinterpret_cast<uint4*>(sm->v + (a >> 3) * kHalf + dim * 128 +
                                    (((a & 7) ^ (dim & 7)) << 4)) = h;
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&sm->v_full);
      cur = nxt;
    }
    if (ct == 0) {  // after an abort: copies that nobody waited for
      if (k_asked > k_got) mbar_wait(&sm->kin_full, (k_asked - 1) & 1);
      if (v_asked > v_got) mbar_wait(&sm->vin_full, (v_asked - 1) & 1);
    }
  } else if (__shfl_sync(0xffffffffu, warp, 0) == 20) {  // uniform to the compiler too
    // ---- MMAs ----------------------------------------------------------------------------------
    const uint32_t one = elect_one(), t_mem = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t d_q = sw128_desc(smem_u32(sm->q[0][0])), d_k = sw128_desc(smem_u32(sm->k)),
                   d_v = sw128_desc(smem_u32(sm->v));
    bool ok = true;
    int pairs = 0;
    // S of tile x = Q K^T for unit u; `start`: the first of a pair
    auto qk = [&](int x, int u, bool start) {
      if (x == 0) ok = mma_wait(&sm->abort_flag, &sm->k_full, u & 1);
      if (ok && start) ok = mma_wait(&sm->abort_flag, &sm->q_full[x], pairs & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      tc_fence_after();
      const uint64_t q0 = d_q + x * (4 * kHalf >> 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t off = ((j >> 2) * kHalf + (j & 3) * 32) >> 4;
        mma_ss(t_mem + 128 * x, q0 + off, d_k + off, j > 0 ? 1u : 0u, one);
        mma_ss(t_mem + 128 * x, q0 + off + (2 * kHalf >> 4), d_k + off, 1u, one);
      }
      if (one) {
        mma_commit(&sm->s_full[x]);
        if (x == 1) mma_commit(&sm->k_free);
      }
      __syncwarp();
    };
    // O of tile x += P V
    auto pv = [&](int x, int u, bool start) {
      if (x == 0) ok = mma_wait(&sm->abort_flag, &sm->v_full, u & 1);
      if (ok) ok = mma_wait(&sm->abort_flag, &sm->p_full[x], u & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      tc_fence_after();
      const uint32_t t_o = t_mem + 256 + 128 * x, t_p = t_mem + 128 * x;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t off = ((j >> 2) * kHalf + (j & 3) * 32) >> 4;
        mma_ts(t_o, t_p + 16 * j, d_v + off, !start || j > 0 ? 1u : 0u, one);
        mma_ts(t_o, t_p + 16 * j + 8, d_v + off, 1u, one);
      }
      if (one) {
        mma_commit(&sm->o_full[x]);
        if (x == 1) mma_commit(&sm->v_free);
      }
      __syncwarp();
    };
    // u = -1: the first unit's scores. Inside a pair PV_A QK_A PV_B QK_B, at its end both PV
    // before the next pair's scores, which wait for its query rows.
    bool pair_ends = true, more = true;
    int part_u = 0;  // units of the part so far: O starts anew every kDrain of them
    for (int u = -1; more && ok; ++u) {
      if (u >= 0) {
        pair_ends = cur.unit + 1 == cur.units;
        q8_next(sc, cur);
        more = cur.left > 0;
        if (more && pair_ends) ++pairs;
      }
#pragma unroll 1
      for (int i = 0; i < 4 && ok; ++i) {
        const bool is_qk = pair_ends ? i >= 2 : i & 1;
        const int x = pair_ends ? i & 1 : i >> 1;
        if (is_qk) {
          if (more) qk(x, u + 1, pair_ends);
        } else if (u >= 0) {
          pv(x, u, part_u % kDrain == 0);
        }
      }
      if (u >= 0) part_u = pair_ends ? 0 : part_u + 1;
    }
    if (one) mma_commit(&sm->drain);
    __syncwarp();
    mbar_wait(&sm->drain, 0);
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 20) tmem_dealloc(tmem, 512);
}

// k_q8_join for tiles of many rows: a warp per row, few parts each.
constexpr int kJoinWarps = 8, kJoinRows = 32;

__global__ __launch_bounds__(32 * kJoinWarps) void k_q8_join_rows(Q8Sched sc,
                                                                  const float* __restrict__ ws_,
                                                                  float* __restrict__ out) {
  float* ws = const_cast<float*>(ws_);
  const int lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  if ((sc.lens || sc.seq_len < sc.n) && blockIdx.y == 0)
    q8_zero_empty<32 * kJoinWarps>(sc, blockIdx.x, gridDim.x, out);
  const int4 note = *reinterpret_cast<const int4*>(ws + 4 * blockIdx.x);  // item, KV head, last
  if (note.x < 0) return;
  const int b = note.x / sc.tiles, tile = note.x - b * sc.tiles;
  const int c0 = blockIdx.x - 1, c1 = note.z;
#pragma unroll 2
  for (int i = threadIdx.x >> 5; i < kJoinRows; i += kJoinWarps) {
    const int row = blockIdx.y * kJoinRows + i, r = tile * sc.tile_rows + row;
    if (r >= sc.n * sc.G) return;
    const int t = r / sc.G, g = r - t * sc.G;
    float* dst = out + ((static_cast<size_t>(b) * sc.n + t) * (sc.G * sc.Hkv) + note.y * sc.G + g) * D + 4 * lane;
    float m = -INFINITY, l = 0.0f;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c = c0; c <= c1; c += 4) {  // four parts at a time
      float pm[4], pl[4];
      float4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pm[i] = -INFINITY;
        pl[i] = 0.0f;
        x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (c + i <= c1) {
          const int slot = 2 * (c + i) + (c + i == c0 ? 1 : 0);
          const float* ml = q8_part_ml(ws, sc.tile_rows, slot);
          pm[i] = ml[row];
          pl[i] = ml[sc.tile_rows + row];
          x[i] = *reinterpret_cast<const float4*>(
              q8_part_o(ws, sc.tile_rows, slot) + static_cast<size_t>(row) * D + 4 * lane);
        }
      }
      float mn = m;
#pragma unroll
      for (int i = 0; i < 4; ++i) mn = fmaxf(mn, pm[i]);
      // a part without keys, or of NaN scores only, has -inf for its maximum
      const float e = m == mn ? 1.0f : ex2(m - mn);
      l *= e;
      y = make_float4(y.x * e, y.y * e, y.z * e, y.w * e);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = pm[i] == mn ? 1.0f : ex2(pm[i] - mn);
        l = fmaf(pl[i], f, l);
        y = make_float4(fmaf(x[i].x, f, y.x), fmaf(x[i].y, f, y.y), fmaf(x[i].z, f, y.z),
                        fmaf(x[i].w, f, y.w));
      }
      m = mn;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    *reinterpret_cast<float4*>(dst) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
  }
}

}  // namespace

size_t attention_q8_many_workspace_bytes() {
  return q8_workspace(kRows, kManyMaxCtas) +
         static_cast<size_t>(kManyMaxCtas) * kRows * D * sizeof(float);  // copies of O
}

cudaError_t launch_attention_q8_many(const float* q, const Q8Cache& c, int n, int H, int seq_len,
                                     const int* lens_dev, float scale_log2, float* out, void* ws,
                                     cudaStream_t s) {
  Q8Sched sc = {c.B, n, H / c.Hkv, c.Hkv, kRows, 0, kStart, seq_len, lens_dev, 0};
  const long long rows = static_cast<long long>(n) * sc.G;
  sc.tiles = static_cast<int>((rows + kRows - 1) / kRows);
  cudaError_t e = allow_smem<&k_attn_q8_many>(sizeof(ManySmem));
  if (e != cudaSuccess) return e;
  CUtensorMap mk, mv;
  if (!q8_map(&mk, c.k, c, kUnitKeys) || !q8_map(&mv, c.v, c, kUnitKeys))
    return cudaErrorNotSupported;
  const long long bound = static_cast<long long>(sc.B) * sc.tiles * sc.Hkv *
                          ((sc.seq_len + kUnitKeys - 1) / kUnitKeys + kStart);
  sc.ctas = static_cast<int>(
      std::max<long long>(std::min<long long>(bound, std::min(num_sms_cached(), kManyMaxCtas)), 1));
  e = launch_pdl(&k_attn_q8_many, dim3(sc.ctas), kThreads, sizeof(ManySmem), s, mk, mv, q, c.k_scale,
                 c.v_scale, q8_blocks(c.S_max), sc, scale_log2, out, static_cast<float*>(ws));
  if (e != cudaSuccess) return e;
  return launch_pdl(&k_q8_join_rows, dim3(sc.ctas, kRows / kJoinRows), 32 * kJoinWarps, 0, s, sc, static_cast<float*>(ws), out);
}

}  // namespace obn
