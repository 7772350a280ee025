// kvq8_attn.cu — attention over the 8-bit KV cache for few query rows (decode, drafted tokens).
//
// softmax(q . k s_k * scale) v s_v with int8 codes k, v and a power-of-two scale per 16 keys.
// The pass has to read 2 * 128 bytes a key and KV head; everything else is arranged so that
// the HBM is what it waits for:
//
//  * Both products run on the int8 tensor cores (mma.sync m16n8k32, exact s32 sums) with the
//    codes as they lie in memory as the A operand: 16 keys x 32 dims for the scores, 16 dims
//    x 32 keys for the weighted sum. The f32 side is cut into four 8-bit digits, which are
//    columns of the same MMAs: two column tiles hold 4 query rows x 4 digits. q is a 31-bit
//    fixed point number against its row's largest element (balanced digits, s8); a weight
//    p = 2^(s - M) is one of 31 bits against M above the running maximum (u8 digits). So
//    nothing is rounded between q and the output to fewer than 24 bits, and an int8 MMA does
//    the work that two f16 MMAs (hi and lo halves) and a conversion of every code would.
//  * The columns are ordered so that an accumulator quad of a lane is the four digits of one
//    query row: joining them is lane-local, in the scores and in the sums. Weights go from
//    there to the B operand of the second product by two shuffles a 16-key block. K needs no
//    rearrangement (dims may be contracted in any order), V comes transposed from shared memory
//    (ldmatrix on 16 x 16 bytes; a byte transpose in registers took 36 against 34 us for 8 x 4 tokens).
//  * The s32 sums are carried along the keys and only turned into f32 (and rescaled) when the
//    reference M has to grow (Vr is then set anew), when a weight times its value scale comes above
//    its reference Vr, or after 2^15 keys (255 * 128 * 2^15 < 2^31). M is set 3 to 4 above the
//    maximum and Vr to 32 times the largest product: the largest keeps 26 bits or more, and few
//    later keys exceed them. A value scale alone does not set Vr: a block of large values with small
//    weights would take bits from the others.
//  * Exponentials are ex2.approx (2 ulp, flushed below 2^-126), one for each score: expf's
//    reduction and its handling of subnormals would be as many instructions again, and the error
//    stays below that of f32 products (2.2e-7 against 5.6e-7 to 2.2e-6 of the plain form).
//  * A producer warp streams 128-key units through a ring of TMA stages, past the ends of
//    pairs; each consumer warp takes slices of 32 keys of a unit with a softmax state of
//    its own, and meets the others only at a pair's end, where the states are merged in shared
//    memory. MT consumer warps share a slice when there are more than 4 query rows.
//
// 64 sequences of up to 4095 keys, 20/5 heads (176 MB): 43 us with the join, 4.0 TB/s, of which
// about 8 us are starts and the join; the stream itself runs at 5 TB/s. One sequence of 131072 (168
// MB): 40 us, 4.2 TB/s. 8 sequences of up to 5000 with 32 rows (24 MB): 33 us, where the products
// bound the warps: 16 rows cost 1.6 times what 8 do, and half of V's products cost 8 us. 12 warps
// an SM (3 CTAs whose first warp requests the units between its own) took 51, 42 and 37 us.
#include "kvq8.h"

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "kvq8_sched.cuh"

namespace obn {

int num_sms_cached();  // kernels.cu

namespace {

constexpr int D = kQ8HeadDim;
constexpr int kSlice = 32;                   // keys of a slice: the K of the PV MMA
constexpr int kTile = kUnitKeys * D;         // bytes of a unit's keys (or values)
// Units of a CTA up to which a cluster takes a pair. Cluster against dealt-out shares with a join
// (one token of 20/5 heads, us between events around the launch with a dirty L2; the kernel itself
// takes 8.9 of the first 12): 1 sequence of 2048, 4096, 8192 keys 12, 14, 16 against 13, 15, 20,
// of 16384 (8 units) 20 against 21; 3 sequences of 2048: 14 against 15; 6 of 4096: 18 against 21.
// 4 tokens of 16/2 heads, 2 sequences of 8192: 22 and 22, of 16384: 31 against 28.
constexpr int kClusterUnits = 4;
constexpr int kFlushSlices = 1024;           // 2^15 keys: 255 * 128 * 2^15 < 2^31

// MT tiles of 4 query rows times KW key slices at once: MT * KW consumer warps.
template <int MT, int KW, int ST>
struct FewSmem {
  uint8_t ring[ST][2 * kTile];  // K, V; 1024-byte aligned for the TMA swizzle
  float scale[ST][2][kUnitKeys / kQ8Block];
  // the pair's query rows as digits: [row][digit][dim]
  alignas(16) uint8_t q[4 * MT][4][D];
  alignas(16) float o[KW][4 * MT][D];
  float q_scale[4 * MT];
  float m[KW][4 * MT], l[KW][4 * MT];
  uint64_t full[ST], empty[ST];
  long long sh[MT * KW + 1 + 8];
};

OBN_DEVINL void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
OBN_DEVINL void mma_su8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two 16 x 16 tiles of bytes, transposed: lane i < 16 gives the address of row i of the first, lane
// 16 + i of the second. a[0], a[1]: columns grp and grp + 8 of rows 4 qd .. 4 qd + 3 of the first,
// a[2], a[3] of the second, an s8 MMA's A operand.
OBN_DEVINL void ld_transposed(uint32_t (&a)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];"
               : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
               : "r"(addr)
               : "memory");
}
// An overflowed score stays the largest or smallest number, a NaN stays one.
OBN_DEVINL float clamp_score(float x) {
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(FLT_MAX));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-FLT_MAX));
  return x;
}

OBN_DEVINL void cp_async4(uint32_t dst, const float* src, bool in) {  // zeros when !in
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
               "r"(in ? 4 : 0)
               : "memory");
}

// Row (of a block of 16) behind row `grp` (0 .. 7) of an MMA's A operand; row grp + 8 is 8
// further on. The order is free as long as K, the weights and V agree; with this one the
// 16-byte fragment loads of K run over the 128-byte swizzle without bank conflicts (the rows that
// one load phase reads differ in bit 2); V's rows are those of the weights' order.
OBN_DEVINL int key_row(int grp) { return 2 * ((grp >> 1) ^ (2 * (grp & 1))) + (grp & 1); }

OBN_DEVINL void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
OBN_DEVINL void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// A float (or four) at this CTA's shared address, in the CTA of rank `rank` of the cluster.
OBN_DEVINL uint32_t in_rank(const void* p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
OBN_DEVINL float ld_cluster(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
OBN_DEVINL float4 ld_cluster4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

// With CL a cluster of CTAs takes a pair, an even share of its units each, and joins the parts
// through its shared memory: one launch, and no shares to work out first.
template <int MT, int KW, int ST, int CTAS, bool CL>
__global__ __launch_bounds__(32 * (MT * KW + 1), CTAS) void k_attn_q8_few(
    const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
    const float* __restrict__ q, const float* __restrict__ k_scale,
    const float* __restrict__ v_scale, int nblk, Q8Sched sc, float scale_log2,
    float* __restrict__ out, float* __restrict__ ws) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  FewSmem<MT, KW, ST>& sm = *reinterpret_cast<FewSmem<MT, KW, ST>*>(smem_raw);
  constexpr int kWarps = MT * KW, kRows = 4 * MT, kSlices = kUnitKeys / kSlice / KW;
  constexpr int kRowsPerWarp = kRows / kWarps;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&sm.full[i], 1 + 32);
      mbar_init(&sm.empty[i], kWarps);
    }
    fence_mbar_init();
  }
  // the lengths may come from the kernel before; the join may read them once all are here
  pdl_wait();
  pdl_launch_dependents();
  Q8Cursor cur;
  if constexpr (CL) {
    cur.item = blockIdx.z;
    cur.kvh = blockIdx.y;
    q8_enter(sc, cur);
    cur.units = q8_units(sc, cur.item);
    const int rank = blockIdx.x, ranks = gridDim.x;
    cur.unit = cur.units / ranks * rank + min(rank, cur.units % ranks);
    cur.left = cur.units / ranks + (rank < cur.units % ranks ? 1 : 0);
  } else {
    int place;
    long long total;
    cur = q8_share<32 * (kWarps + 1)>(sc, blockIdx.x, &place, &total, sm.sh);
    if (tid == 0) q8_note_split(sc, cur, place, total, ws);
    if (cur.left == 0) return;
  }
  __syncthreads();
  const int H = sc.G * sc.Hkv, rows_seq = sc.n * sc.G;

  if (warp == kWarps) {  // producer
    for (int it = 0; cur.left > 0; ++it) {
      const int st = it % ST;
      if (it >= ST && !__all_sync(0xffffffffu, mbar_wait(&sm.empty[st], (it / ST - 1) & 1))) break;
      const int k0 = cur.unit * kUnitKeys, left = cur.len - k0;
      const int boxes = min((left + kSlice - 1) / kSlice, kUnitKeys / kSlice);
      if (lane == 0) mbar_arrive_expect_tx(&sm.full[st], boxes * 2 * kSlice * D);
      __syncwarp();
      if (lane < 8 && (lane & 3) < boxes)  // boxes of 32 keys: none behind the sequence
        tma_load_4d(smem_u32(sm.ring[st]) + (lane >> 2) * kTile + (lane & 3) * kSlice * D,
                    lane < 4 ? &tmap_k : &tmap_v, 0, cur.kvh, k0 + (lane & 3) * kSlice, cur.b,
                    &sm.full[st]);
      if (lane < 16) {
        const int blk = lane & 7;
        const bool in = blk * kQ8Block < left;
        cp_async4(smem_u32(&sm.scale[st][lane >> 3][blk]),
                  (lane < 8 ? k_scale : v_scale) +
                      (static_cast<size_t>(cur.b) * nblk + k0 / kQ8Block + (in ? blk : 0)) * sc.Hkv +
                      cur.kvh,
                  in);
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(
                       smem_u32(&sm.full[st]))
                   : "memory");
      q8_next(sc, cur);
    }
    if constexpr (CL) {
      cluster_arrive();
      cluster_wait();
      cluster_arrive();
      cluster_wait();
    }
    return;
  }

  const int qd = lane & 3, grp = lane >> 2;
  const int kw = warp / MT, mt = warp % MT;
  // this lane's fragments: K row and the two chunks of it, V rows of its key quad
  const int kr = key_row(grp);
  const uint32_t k_off = kr * D + ((qd ^ (kr & 7)) << 4);  // chunk qd + 4: ^ 64
  const int vr = 16 * (lane >> 4) + 8 * (lane & 1) + key_row((lane & 15) >> 1);
  const uint32_t v_off = kTile + vr * D;
  // selectors of the weights' way to the B operand
  const bool odd = grp & 1;
  const uint32_t sel_lo = odd ? 0x1054u : 0x5410u, sel_hi = odd ? 0x3276u : 0x7632u;
  const int src_a = (2 * qd + (odd ? 1 : 0)) * 4 + (grp >> 1);  // source lanes
  const int src_b = (2 * qd + (odd ? 0 : 1)) * 4 + (grp >> 1);

  bool dead = false;  // a copy did not come in time: no more waits
  int acc[8][2][4];   // [16 dims][digits 0 1 / 2 3][dim grp: 2 digits, dim grp + 8: 2 digits]
  float o[16];        // dims grp, grp + 8, .. of query row qd of the tile
  float M = -INFINITY, l = 0.0f, Vr = 0.0f, inv_vr = 0.0f, sq = 0.0f;
  int lim = 0, since = 0, most = 0, u_first = 0;
  uint32_t bq[4][2][2];  // q: [k step][digits 0 1 / 2 3][dims 16 qd + 4 k / 64 + 16 qd + 4 k]
  auto load_q = [&]() {
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint4 w = *reinterpret_cast<const uint4*>(
            &sm.q[mt * 4 + (grp >> 1)][2 * nt + (grp & 1)][64 * s + 16 * qd]);
        bq[0][nt][s] = w.x;
        bq[1][nt][s] = w.y;
        bq[2][nt][s] = w.z;
        bq[3][nt][s] = w.w;
      }
  };

  // The s32 sums into f32, and everything to the new references.
  auto flush = [&](float mn, float vn) {
    const float corr = M == mn ? 1.0f : ex2(M - mn);
    if (since > 0) {
      const float unit = Vr;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // digit 3 counts 2^24 / 2^31 of the reference
          float v = fmaf(static_cast<float>(acc[j][0][2 * i]), 0.00390625f,
                         static_cast<float>(acc[j][0][2 * i + 1]));
          v = fmaf(v, 0.00390625f, static_cast<float>(acc[j][1][2 * i]));
          v = fmaf(v, 0.00390625f, static_cast<float>(acc[j][1][2 * i + 1]));
          o[2 * j + i] = fmaf(v * 0.0078125f, unit, o[2 * j + i]) * corr;
        }
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[j][i >> 2][i & 3] = 0;
    }
    l *= corr;
    M = mn;
    Vr = vn;
    inv_vr = vn > 0.0f ? 1.0f / vn : 0.0f;
    since = 0;
  };

  float4 qx[kRowsPerWarp];  // the pair's query rows that this warp turns into digits
  auto fetch_q = [&]() {
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
      const int r = cur.tile * kRows + warp * kRowsPerWarp + i;
      const int t = r / sc.G, g = r - t * sc.G;
      qx[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (r < rows_seq)
        qx[i] = __ldg(reinterpret_cast<const float4*>(
            q + ((static_cast<size_t>(cur.b) * sc.n + t) * H + cur.kvh * sc.G + g) * D + 4 * lane));
    }
  };
  auto consumers = [&]() {
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");
  };

  // The CTA's part of a cluster's pair, in the ring when its units are done: sums [rows][128],
  // maxima and totals [rows].
  float* part = reinterpret_cast<float*>(sm.ring[0]);
  const int item = cur.item, kvh = cur.kvh;
  if (CL && cur.left == 0) {
    for (int i = tid; i < kRows * (D + 2); i += 32 * kWarps)
      part[i] = i >= kRows * D && i < kRows * (D + 1) ? -INFINITY : 0.0f;
  } else {
    fetch_q();
  }
  bool fresh = true;
  int it = 0;
  for (; cur.left > 0; ++it) {
    const int stage = it % ST;
    if (fresh) {  // a new pair
      fresh = false;
      u_first = cur.unit;
#pragma unroll
      for (int i = 0; i < kRowsPerWarp; ++i) {
        const float4 x = qx[i];
        const int row = warp * kRowsPerWarp + i;
        // the largest magnitude's bits: an infinity or NaN shows as exponent 255
        const uint32_t big = __reduce_max_sync(
            0xffffffffu, max(max(__float_as_uint(x.x) & 0x7FFFFFFFu, __float_as_uint(x.y) & 0x7FFFFFFFu),
                             max(__float_as_uint(x.z) & 0x7FFFFFFFu, __float_as_uint(x.w) & 0x7FFFFFFFu)));
        const bool bad = big >= 0x7F800000u;
        const int ex = max(static_cast<int>(big >> 23) - 126, -90);  // |x| < 2^ex
        const float up = __int_as_float((127 + 30 - ex) << 23);
        // balanced digits: adding 128 to each of the lower three and taking it off again
        auto digits = [&](float v) {
          return (static_cast<uint32_t>(bad ? 0 : __float2int_rn(v * up)) + 0x00808080u) ^ 0x00808080u;
        };
        uint32_t d[4];
        transpose4(digits(x.x), digits(x.y), digits(x.z), digits(x.w), d);
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t*>(&sm.q[row][j][4 * lane]) = d[j];
        if (lane == 0)
          sm.q_scale[row] =
              (bad ? __int_as_float(0x7FC00000) : __int_as_float((127 + ex - 30) << 23)) * scale_log2;
      }
      consumers();
      const int row = mt * 4 + qd, r = cur.tile * kRows + row;
      sq = sm.q_scale[row];
      lim = r < rows_seq ? min(cur.len, q8_limit(sc, cur.len, r)) : 0;
      most = __reduce_max_sync(0xffffffffu, lim);
      load_q();
      M = -INFINITY;
      l = Vr = inv_vr = 0.0f;
      since = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[j][i >> 2][i & 3] = 0;
    }

    if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait(&sm.full[stage], (it / ST) & 1));
    for (int sub = 0; sub < kSlices; ++sub) {
      const int slice = kw * kSlices + sub;
      const int k0 = cur.unit * kUnitKeys + slice * kSlice;
      if (k0 >= most) break;
      const uint8_t* st = sm.ring[stage] + slice * kSlice * D;
      float s[2][2];  // [16-key block][key row grp / grp + 8]
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        uint4 w[2][2];  // [key row][chunk]
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          w[hh][0] = *reinterpret_cast<const uint4*>(st + (kb * 16 + hh * 8) * D + k_off);
          w[hh][1] = *reinterpret_cast<const uint4*>(st + (kb * 16 + hh * 8) * D + (k_off ^ 64));
        }
        int cc[2][4] = {};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          auto word = [&](const uint4& v) { return ks == 0 ? v.x : ks == 1 ? v.y : ks == 2 ? v.z : v.w; };
          const uint32_t a[4] = {word(w[0][0]), word(w[1][0]), word(w[0][1]), word(w[1][1])};
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) mma_s8(cc[nt], a, bq[ks][nt][0], bq[ks][nt][1]);
        }
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)  // |sums| < 2^21: pairs of digits in integers
          s[kb][hh] = fmaf(static_cast<float>(cc[1][2 * hh + 1] * 256 + cc[1][2 * hh]), 65536.0f,
                           static_cast<float>(cc[0][2 * hh + 1] * 256 + cc[0][2 * hh]));
      }
      const float2 sk = *reinterpret_cast<const float2*>(&sm.scale[stage][0][slice * 2]);
      const float2 sv = *reinterpret_cast<const float2*>(&sm.scale[stage][1][slice * 2]);
      bool seen[2][2], grow = since >= kFlushSlices;
      const bool second = k0 + 16 < most;  // does any row see block 1
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const float f = sq * (kb ? sk.y : sk.x);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          seen[kb][hh] = k0 + kb * 16 + hh * 8 + kr < lim;
          const float x = clamp_score(s[kb][hh] * f);
          s[kb][hh] = seen[kb][hh] ? x : -INFINITY;
          grow |= s[kb][hh] > M;
        }
      }
      grow |= sv.x > Vr || (second && sv.y > Vr);
      if (__any_sync(0xffffffffu, grow)) {
        float m = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) m = fmaxf(m, shx(m, d));
        const float mn = m > M ? ceilf(m) + 3.0f : M;
        float top = 0.0f;  // largest weight times value scale
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          if (seen[0][hh]) top = fmaxf(top, ex2(s[0][hh] - mn) * sv.x);
          if (seen[1][hh]) top = fmaxf(top, ex2(s[1][hh] - mn) * sv.y);
        }
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) top = fmaxf(top, shx(top, d));
        // only of the rows that need it: no row's bits depend on another's
        // Vr goes by this slice also when M has grown, as the products before it have shrunk: a large
        // value of small score at the front must not take the later keys' bits. 1 / Vr stays finite.
        if (mn != M || top > Vr || since >= kFlushSlices)
          flush(mn, mn != M || top > Vr ? fmaxf(32.0f * top, FLT_MIN) : Vr);
      }
      uint32_t b[2][2];  // weights: [digits 0 1 / 2 3][block]
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const float svk = kb ? sv.y : sv.x;
        // a finite scale adds 0, a NaN one poisons the total
        // p f <= 1, and where f is beyond f32's range p is 0 and the weight too (0 * inf: NaN, as
        // a whole number 0)
        const float poison = svk - svk, f = svk * inv_vr;
        uint32_t w[2];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const float p = seen[kb][hh] ? ex2(s[kb][hh] - M) : 0.0f;
          l += seen[kb][hh] ? p + poison : 0.0f;
          w[hh] = __float2uint_rn(p * f * 2147483648.0f);
        }
        // this lane: two keys of query row qd; wanted: four keys of row grp / 2, and of their
        // digits grp % 2 and 2 + grp % 2. Even columns fetch digits 0 and 2 (y0), odd 1 and 3.
        const uint32_t y0 = __byte_perm(w[0], w[1], 0x6240), y1 = __byte_perm(w[0], w[1], 0x7351);
        const uint32_t za = __shfl_sync(0xffffffffu, odd ? y1 : y0, src_a);
        const uint32_t zb = __shfl_sync(0xffffffffu, odd ? y0 : y1, src_b);
        b[0][kb] = __byte_perm(za, zb, sel_lo);
        b[1][kb] = __byte_perm(za, zb, sel_hi);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // 16 dims x 32 keys
        uint32_t a[4];
        ld_transposed(a, smem_u32(st) + v_off + ((j ^ (vr & 7)) << 4));
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) mma_su8(acc[j][nt], a, b[nt][0], b[nt][1]);
      }
      ++since;
    }
    fence_proxy_async_smem();  // read, before a copy writes there again
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.empty[stage]);

    const Q8Cursor done = cur;
    q8_next(sc, cur);
    const bool pair_ends = done.unit + 1 == done.units;
    if (!pair_ends && cur.left > 0) continue;
    // merge the slices, write the pair or its part
    const bool whole = !CL && pair_ends && u_first == 0;
    if (cur.left > 0) fetch_q();
    flush(M, Vr);
    if (dead) l = __int_as_float(0x7FC00000);  // no such result passes for one
#pragma unroll
    for (int d = 4; d <= 16; d <<= 1) l += shx(l, d);
    {
      const int row = mt * 4 + qd;
      if (grp == 0) {
        sm.m[kw][row] = M;
        sm.l[kw][row] = l;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) sm.o[kw][row][8 * i + grp] = o[i];
    }
    consumers();
    const int slot = 2 * blockIdx.x + (u_first == 0 ? 1 : 0);
    float* po = CL ? part : q8_part_o(ws, kRows, slot);
    float* pml = CL ? part + kRows * D : q8_part_ml(ws, kRows, slot);
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
      const int row = warp * kRowsPerWarp + i, d4 = 4 * lane;
      float m = -INFINITY;
#pragma unroll
      for (int k = 0; k < KW; ++k) m = fmaxf(m, sm.m[k][row]);
      float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float lt = 0.0f;
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        // a slice that saw nothing has l = 0, o = 0 and -inf here; so has one of NaN scores
        // (but for l), and it must not lose them
        const float e = sm.m[k][row] == m ? 1.0f : ex2(sm.m[k][row] - m);
        const float4 x = *reinterpret_cast<const float4*>(&sm.o[k][row][d4]);
        lt = fmaf(sm.l[k][row], e, lt);
        y.x = fmaf(x.x, e, y.x);
        y.y = fmaf(x.y, e, y.y);
        y.z = fmaf(x.z, e, y.z);
        y.w = fmaf(x.w, e, y.w);
      }
      const int r = done.tile * kRows + row;
      if (whole) {
        if (r < rows_seq) {
          const int t = r / sc.G, g = r - t * sc.G;
          const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;  // no key: zeros
          *reinterpret_cast<float4*>(
              out + ((static_cast<size_t>(done.b) * sc.n + t) * H + done.kvh * sc.G + g) * D + d4) =
              make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
        }
      } else {
        *reinterpret_cast<float4*>(po + row * D + d4) = y;
        if (lane == 0) {
          pml[row] = m;
          pml[kRows + row] = lt;
        }
      }
    }
    consumers();
    fresh = true;
  }
  if (dead)  // a copy may still be on its way into this CTA's shared memory
    for (int i = 0; i < min(ST, it); ++i) mbar_wait(&sm.full[i], ((it - 1 - i) / ST) & 1);
  if constexpr (CL) {
    cluster_arrive();
    cluster_wait();
    const int ranks = gridDim.x, b = item / sc.tiles, tile = item - b * sc.tiles;
    for (int row = blockIdx.x + ranks * warp; row < kRows; row += ranks * kWarps) {  // a warp a row
      const int r = tile * kRows + row;
      if (r >= rows_seq) break;
      const bool in = lane < ranks;
      const float pm = in ? ld_cluster(in_rank(part + kRows * D + row, lane)) : -INFINITY;
      float l_all = in ? ld_cluster(in_rank(part + kRows * (D + 1) + row, lane)) : 0.0f, m = pm;
#pragma unroll
      for (int d = 8; d; d >>= 1) m = fmaxf(m, shx(m, d));
      // a part without keys, or of NaN scores only, has -inf for its maximum
      const float e = pm == m ? 1.0f : ex2(pm - m);
      l_all *= e;
#pragma unroll
      for (int d = 8; d; d >>= 1) l_all += shx(l_all, d);
      float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
      for (int i = 0; i < ranks; ++i) {
        const float ei = __shfl_sync(0xffffffffu, e, i);
        const float4 z = ld_cluster4(in_rank(part + row * D + 4 * lane, i));
        y = make_float4(fmaf(z.x, ei, y.x), fmaf(z.y, ei, y.y), fmaf(z.z, ei, y.z), fmaf(z.w, ei, y.w));
      }
      l_all = __shfl_sync(0xffffffffu, l_all, 0);
      const float inv = l_all == 0.0f ? 0.0f : 1.0f / l_all;  // no key: zeros
      const int t = r / sc.G, g = r - t * sc.G;
      *reinterpret_cast<float4*>(
          out + ((static_cast<size_t>(b) * sc.n + t) * H + kvh * sc.G + g) * D + 4 * lane) =
          make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
    }
    cluster_arrive();
    cluster_wait();  // the others have read this CTA's part
  }
}

// Joins the parts of the pairs that span CTAs (q8_note_split), and zeroes the items without keys.
// One CTA per split pair and row (4 rows: all 8 warps to a row; 8 and 16 rows, whose pairs have
// fewer parts: 2 and 4 rows to a CTA): first the parts' maxima and totals, a lane a part, then
// their sums, four loads on their way at a time.
constexpr int kJoinWarps = 8;

template <int ROWS>
__global__ __launch_bounds__(32 * kJoinWarps) void k_q8_join(Q8Sched sc, const float* __restrict__ ws_,
                                                             float* __restrict__ out) {
  constexpr int kRowsPer = ROWS / 4, W = kJoinWarps / kRowsPer;  // warps to a row
  __shared__ float s_m[kJoinWarps], s_l[kJoinWarps];
  __shared__ float4 s_o[kJoinWarps][32];
  float* ws = const_cast<float*>(ws_);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  pdl_launch_dependents();
  if ((sc.lens || sc.seq_len < sc.n) && blockIdx.y == 0)
    q8_zero_empty<32 * kJoinWarps>(sc, blockIdx.x, gridDim.x, out);
  const int4 note = *reinterpret_cast<const int4*>(ws + 4 * blockIdx.x);  // item, KV head, last
  if (note.x < 0) return;
  const int b = note.x / sc.tiles, tile = note.x - b * sc.tiles;
  const int c0 = blockIdx.x - 1, parts = note.z - c0 + 1;
  auto slot = [&](int i) { return 2 * (c0 + i) + (i == 0 ? 1 : 0); };
  const int sub = warp % W;  // of the W warps of a row: parts sub, sub + W, ...
  const int row = blockIdx.y * kRowsPer + warp / W, r = tile * ROWS + row;
  float m = -INFINITY, l = 0.0f;
  for (int i = lane * W + sub; i < parts; i += 32 * W)
    m = fmaxf(m, q8_part_ml(ws, ROWS, slot(i))[row]);
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, shx(m, d));
  float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i0 = sub; i0 < parts; i0 += 32 * W) {
    const int i = i0 + lane * W;
    float e = 0.0f;
    if (i < parts) {
      const float* ml = q8_part_ml(ws, ROWS, slot(i));
      // a part of NaN scores only has -inf here and its NaN in the total
      e = ml[row] == m ? 1.0f : ex2(ml[row] - m);
      l = fmaf(ml[ROWS + row], e, l);
    }
    const int n = min(32, (parts - i0 + W - 1) / W);
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const float ek = __shfl_sync(0xffffffffu, e, k);
      const float4 x = *reinterpret_cast<const float4*>(
          q8_part_o(ws, ROWS, slot(i0 + k * W)) + row * D + 4 * lane);
      y = make_float4(fmaf(x.x, ek, y.x), fmaf(x.y, ek, y.y), fmaf(x.z, ek, y.z), fmaf(x.w, ek, y.w));
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) l += shx(l, d);
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  s_o[warp][lane] = y;
  __syncthreads();
  if (sub || r >= sc.n * sc.G) return;
#pragma unroll
  for (int w = 0; w < W; ++w) m = fmaxf(m, s_m[warp + w]);
  l = 0.0f;
  y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int w = 0; w < W; ++w) {
    // a warp without a part has -inf, no total and no sums
    const float e = s_m[warp + w] == m ? 1.0f : ex2(s_m[warp + w] - m);
    const float4 x = s_o[warp + w][lane];
    l = fmaf(s_l[warp + w], e, l);
    y = make_float4(fmaf(x.x, e, y.x), fmaf(x.y, e, y.y), fmaf(x.z, e, y.z), fmaf(x.w, e, y.w));
  }
  const int t = r / sc.G, g = r - t * sc.G;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<float4*>(
      out + ((static_cast<size_t>(b) * sc.n + t) * (sc.G * sc.Hkv) + note.y * sc.G + g) * D + 4 * lane) =
      make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
}

template <int MT, int KW, int ST, int CTAS>
cudaError_t launch_few(const float* q, const Q8Cache& c, Q8Sched sc, float scale_log2, float* out,
                       float* ws, cudaStream_t s) {
  constexpr size_t smem = sizeof(FewSmem<MT, KW, ST>);
  constexpr int threads = 32 * (MT * KW + 1);
  static_assert(CTAS * (smem + 1024) <= 228 * 1024, "shared memory");
  CUtensorMap mk, mv;
  if (!q8_map(&mk, c.k, c, kSlice) || !q8_map(&mv, c.v, c, kSlice)) return cudaErrorNotSupported;
  const long long pairs = static_cast<long long>(sc.B) * sc.tiles * sc.Hkv;
  const long long units = (sc.seq_len + kUnitKeys - 1) / kUnitKeys;
  const long long fit = std::min(num_sms_cached() * CTAS, kQ8MaxCtas);
  const long long dealt = std::max<long long>(std::min(pairs * (units + 1), fit), 1);
  if (pairs * ((units + kClusterUnits - 1) / kClusterUnits) <= fit && units <= 16 * kClusterUnits) {
    constexpr auto* kernel = &k_attn_q8_few<MT, KW, ST, CTAS, true>;
    cudaError_t e = allow_smem<kernel>(smem);
    if (e != cudaSuccess) return e;
    // as many CTAs to a pair as let all pairs run at once
    for (int size = 16; size * kClusterUnits >= units; size /= 2) {
      const int ranks = static_cast<int>(std::max<long long>(std::min<long long>(size, units), 1));
      if (pairs <= active_clusters<kernel>(ranks, threads, smem))
        return launch_cluster(kernel, dim3(ranks, sc.Hkv, sc.B * sc.tiles), ranks, threads, smem, s,
                              mk, mv, q, c.k_scale, c.v_scale, q8_blocks(c.S_max), sc, scale_log2,
                              out, ws);
      if (size == 1) break;
    }
  }
  constexpr auto* kernel = &k_attn_q8_few<MT, KW, ST, CTAS, false>;
  cudaError_t e = allow_smem<kernel>(smem);
  if (e != cudaSuccess) return e;
  // Where the sequences are alike, a multiple of Hkv CTAs keeps the heads in step, on the same rows
  // of memory, unless that leaves out more than 1/32 of them. With against without (dirty L2, us):
  // one sequence of 131072, 5 heads: 51 against 53; of 60000, 32 heads (288 of 296 CTAs): 121, 129;
  // 8 of 3000, 40 heads (280 of 296): 78, 76; 4 of 2000 with 4 tokens, 40 heads (120 of 148): 70, 61;
  // one of 6000 with 4 tokens, 75 heads (75 of 148): 119, 75. Lengths of any mix, 16 sequences with
  // 4 tokens, 8 heads (144 of 148): 84, 82.
  const long long spare = sc.B == 1 || !sc.lens ? dealt % sc.Hkv : 0;
  sc.ctas = static_cast<int>(dealt - (32 * spare <= dealt ? spare : 0));
  e = launch_pdl(kernel, dim3(sc.ctas), threads, smem, s, mk, mv, q, c.k_scale, c.v_scale,
                 q8_blocks(c.S_max), sc, scale_log2, out, ws);
  if (e != cudaSuccess) return e;
  return launch_pdl(&k_q8_join<4 * MT>, dim3(sc.ctas, 4), 32 * kJoinWarps, 0, s, sc, ws, out);
}

}  // namespace

// Query rows of a sequence and KV head up to which the few-rows pass runs. Few against many rows'
// pass, 4 KV heads, at 32, 48 and 64 rows: 8 sequences of 5000: 54, 73, 87 against 95 us;
// one of 2048: 19, 21, 21 against 36; 32 of 1500: 66, 89, 112 against 110; one of 40000: 52, 69,
// 83 against 105. Every further 16 rows stream the keys once more, the other pass takes up to
// 256 rows for the same price.
constexpr int kFewRows = 64;

size_t attention_q8_workspace_bytes(int B, int n, int H, int Hkv, int S_max) {
  (void)B, (void)S_max;
  const long long rows = static_cast<long long>(n) * (H / Hkv);
  return rows > kFewRows ? attention_q8_many_workspace_bytes() : q8_workspace(16, kQ8MaxCtas);
}

cudaError_t launch_attention_q8(const float* q, const Q8Cache& c, int n, int H, int seq_len,
                                const int* lens_dev, float scale, float* out, void* workspace,
                                cudaStream_t s) {
  Q8Sched sc = {c.B, n, H / c.Hkv, c.Hkv, 0, 0, 1, seq_len, lens_dev, 0};
  const long long rows = static_cast<long long>(n) * sc.G;
  const float scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  if (rows > kFewRows)
    return launch_attention_q8_many(q, c, n, H, seq_len, lens_dev, scale_log2, out, workspace, s);
  sc.tile_rows = rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
  sc.tiles = static_cast<int>((rows + sc.tile_rows - 1) / sc.tile_rows);
  float* ws = static_cast<float*>(workspace);
  if (sc.tile_rows == 4) return launch_few<1, 4, 3, 2>(q, c, sc, scale_log2, out, ws, s);
  if (sc.tile_rows == 8) return launch_few<2, 4, 5, 1>(q, c, sc, scale_log2, out, ws, s);
  return launch_few<4, 2, 5, 1>(q, c, sc, scale_log2, out, ws, s);
}

}  // namespace obn
