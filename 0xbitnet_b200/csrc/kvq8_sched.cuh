// kvq8_sched.cuh — how attention over the 8-bit cache is spread over the GPU.
//
// The query rows of a sequence and KV head (t * G + g for token t and group head g) are cut
// into tiles of `tile_rows`; an item is a (sequence, tile), a pair an item with a KV head,
// and a unit kUnitKeys keys of a pair. Every pair with keys is a start, which costs about as
// much as one unit or two (decode of 64 sequences of up to 4095: without it the CTAs with 8
// short pairs took 41 us, those with one 29), and then its units. All places of all pairs in
// a row, T of them, are dealt out evenly: CTA c of C <= T takes places [c T / C, (c + 1) T / C).
// So sequences of any mix of lengths and causal tiles of any depth keep every CTA equally busy,
// and one long sequence is split as finely as many short ones. A pair that lies inside one CTA
// is written out by it; the parts of a pair that spans CTAs go to the workspace and are joined by
// k_q8_join (or k_q8_join_rows). A CTA holds at most two parts: one that continues a pair (slot
// 2c) and one that begins a pair and does not end it (slot 2c + 1).
#pragma once

#include "gemm.h"
#include "kvq8.h"
#include "obn_common.cuh"
#include "tc05.cuh"

namespace obn {

constexpr int kUnitKeys = 128;
constexpr int kQ8MaxCtas = 640;  // bounds C, and with it the workspace

struct Q8Sched {
  int B, n, G, Hkv;
  int tile_rows, tiles;  // rows per tile, tiles per sequence
  int start;             // places of a pair's start
  int seq_len;
  const int* lens;
  int ctas;
};

// Positions of sequence b.
OBN_DEVINL int q8_len(const Q8Sched& s, int b) {
  return s.lens ? min(max(s.lens[b], 0), s.seq_len) : s.seq_len;
}
// Keys that row `row` of a sequence of `len` positions sees (may be <= 0).
OBN_DEVINL int q8_limit(const Q8Sched& s, int len, int row) {
  return len - s.n + row / s.G + 1;
}
OBN_DEVINL int q8_units(const Q8Sched& s, int item) {
  const int b = item / s.tiles, tile = item - b * s.tiles;
  const int last = min((tile + 1) * s.tile_rows, s.n * s.G) - 1;
  return (max(q8_limit(s, q8_len(s, b), last), 0) + kUnitKeys - 1) / kUnitKeys;
}
// Places of a pair of `units` units.
OBN_DEVINL int q8_places(const Q8Sched& s, int units) { return units + (units > 0 ? s.start : 0); }
// CTAs that take part: every one of them has a place.
OBN_DEVINL int q8_ctas(const Q8Sched& s, long long total) {
  return static_cast<int>(min(static_cast<long long>(s.ctas), total));
}
// The first place of CTA c, and the CTA that holds place x.
OBN_DEVINL long long q8_begin(long long total, int ctas, int c) {
  if (total * ctas <= 0x7FFFFFFFll) return static_cast<int>(c * static_cast<int>(total)) / ctas;
  return c * total / ctas;
}
OBN_DEVINL int q8_owner(long long total, int ctas, long long x) {
  if (total * ctas <= 0x7FFFFFFFll)
    return (static_cast<int>(x + 1) * ctas - 1) / static_cast<int>(total);
  return static_cast<int>(((x + 1) * ctas - 1) / total);
}

// A unit on the way through a CTA's share.
struct Q8Cursor {
  int item, kvh, unit, units;  // units: those of the item
  int b, tile, len;            // the item's sequence, its tile and the sequence's positions
  int left;                    // places of the share from this unit on, 0: the share is done
};
OBN_DEVINL void q8_enter(const Q8Sched& s, Q8Cursor& c) {
  c.b = c.item / s.tiles;
  c.tile = c.item - c.b * s.tiles;
  c.len = q8_len(s, c.b);
}

// Adds up every item's places over the THREADS threads of the CTA, a run of items for each:
// *front the places of the items before this thread's run, i0 .. i1 - 1 (times Hkv). Returns
// the total. sh: THREADS / 32 shared words.
template <int THREADS>
OBN_DEVINL long long q8_scan(const Q8Sched& s, int* i0, int* i1, long long* front, long long* sh) {
  const int items = s.B * s.tiles, tid = threadIdx.x;
  const int per = (items + THREADS - 1) / THREADS;
  *i0 = min(tid * per, items);
  *i1 = min(*i0 + per, items);
  long long sum = 0;
  for (int i = *i0; i < *i1; ++i) sum += q8_places(s, q8_units(s, i));
  sum *= s.Hkv;
  long long incl = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, d);
    if (tid % 32 >= d) incl += o;
  }
  if (tid % 32 == 31) sh[tid / 32] = incl;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w == tid / 32) incl += total;
    total += sh[w];
  }
  *front = incl - sum;
  return total;
}

// The share of CTA `cta` from its first unit on (left 0: it has none). *place: where in its pair
// the share begins (the start's places, then the units); *total: all places. For all threads;
// sh: THREADS / 32 + 8 shared words.
template <int THREADS>
OBN_DEVINL Q8Cursor q8_share(const Q8Sched& s, int cta, int* place, long long* total, long long* sh) {
  Q8Cursor c = {};
  if (!s.lens && s.tiles == 1) {  // all items alike
    c.units = q8_units(s, 0);
    const int each = q8_places(s, c.units);
    *total = static_cast<long long>(each) * s.B * s.Hkv;
    const int ctas = q8_ctas(s, *total);
    if (cta >= ctas) return c;
    const long long x = q8_begin(*total, ctas, cta);
    c.left = static_cast<int>(q8_begin(*total, ctas, cta + 1) - x);
    long long pair;
    if (*total <= 0x7FFFFFFFll)
      pair = static_cast<int>(x) / each;
    else
      pair = x / each;
    c.item = static_cast<int>(pair / s.Hkv);
    c.kvh = static_cast<int>(pair - static_cast<long long>(c.item) * s.Hkv);
    *place = static_cast<int>(x - pair * each);
    q8_enter(s, c);
  } else {
    int i0, i1;
    long long at;
    *total = q8_scan<THREADS>(s, &i0, &i1, &at, sh);
    const int ctas = q8_ctas(s, *total);
    if (cta >= ctas) return c;
    const long long x = q8_begin(*total, ctas, cta);
    c.left = static_cast<int>(q8_begin(*total, ctas, cta + 1) - x);
    long long* o = sh + THREADS / 32;
    if (x >= at) {  // the thread whose run holds place x walks it
      for (int i = i0; i < i1; ++i) {
        const int u = q8_units(s, i), each = q8_places(s, u);
        const long long end = at + static_cast<long long>(each) * s.Hkv;
        if (x < end) {
          const long long in = x - at;
          const int kvh = in <= 0x7FFFFFFFll ? static_cast<int>(in) / each
                                             : static_cast<int>(in / each);
          o[0] = i;
          o[1] = kvh;
          o[2] = in - static_cast<long long>(kvh) * each;
          o[3] = u;
          o[4] = q8_len(s, i / s.tiles);
          break;
        }
        at = end;
      }
    }
    __syncthreads();
    c.item = static_cast<int>(o[0]);
    c.kvh = static_cast<int>(o[1]);
    *place = static_cast<int>(o[2]);
    c.units = static_cast<int>(o[3]);
    c.len = static_cast<int>(o[4]);
    c.b = c.item / s.tiles;
    c.tile = c.item - c.b * s.tiles;
  }
  const int skip = max(s.start - *place, 0);  // of a start
  c.left = max(c.left - skip, 0);
  c.unit = max(*place - s.start, 0);
  return c;
}

// The join's work, noted by the CTAs of the pass at the head of the workspace. If the share of
// CTA j begins inside a pair's units and CTA j - 1 holds the pair's first unit, join CTA j joins
// that pair: parts of CTAs j - 1 .. last. So each split pair has one join CTA (per row or rows),
// and there are as many as CTAs, however many pairs there are.
OBN_DEVINL void q8_note_split(const Q8Sched& s, const Q8Cursor& c, int place, long long total, float* ws) {
  const int ctas = q8_ctas(s, total), j = blockIdx.x;
  int4 note = make_int4(-1, 0, 0, 0);  // item (-1: nothing to join), KV head, last CTA
  if (j > 0 && j < ctas && place > s.start) {
    const long long x0 = q8_begin(total, ctas, j) - place + s.start;  // unit 0
    if (q8_owner(total, ctas, x0) == j - 1)
      note = make_int4(c.item, c.kvh, q8_owner(total, ctas, x0 + c.units - 1), 0);
  }
  *reinterpret_cast<int4*>(ws + 4 * j) = note;
}

// Zeros for the rows of the items without keys, spread over `ctas` CTAs of THREADS threads.
template <int THREADS>
OBN_DEVINL void q8_zero_empty(const Q8Sched& s, int cta, int ctas, float* out) {
  const int items = s.B * s.tiles, row4 = s.Hkv * s.G * kQ8HeadDim / 4;
  for (int i = cta; i < items; i += ctas) {
    if (q8_units(s, i) > 0) continue;
    const int b = i / s.tiles, tile = i - b * s.tiles;
    const int r0 = tile * s.tile_rows, r1 = min(r0 + s.tile_rows, s.n * s.G);
    // rows r0 .. r1 - 1 of every KV head; a row is 32 pieces of 16 bytes
    for (long long e = threadIdx.x; e < static_cast<long long>(r1 - r0) * s.Hkv * 32; e += THREADS) {
      const int piece = static_cast<int>(e % 32), kvh = static_cast<int>(e / 32 % s.Hkv);
      const int r = r0 + static_cast<int>(e / 32 / s.Hkv), t = r / s.G, g = r - t * s.G;
      *reinterpret_cast<float4*>(out + (static_cast<size_t>(b) * s.n + t) * row4 * 4 +
                                 (static_cast<size_t>(kvh) * s.G + g) * kQ8HeadDim + 4 * piece) =
          make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
  }
}

// Steps to the share's next unit; left becomes 0 at its end.
OBN_DEVINL void q8_next(const Q8Sched& s, Q8Cursor& c) {
  if (--c.left <= 0) return;
  if (++c.unit < c.units) return;
  c.left -= s.start;  // the next pair's
  if (c.left <= 0) {
    c.left = 0;
    return;
  }
  c.unit = 0;
  if (++c.kvh < s.Hkv) return;
  c.kvh = 0;
  do {
    ++c.item;  // an item with units follows: the share has places left
    c.units = q8_units(s, c.item);
  } while (c.units == 0);
  q8_enter(s, c);
}

OBN_DEVINL float shx(float v, int m) { return __shfl_xor_sync(0xffffffffu, v, m); }
OBN_DEVINL float ex2(float x) {  // 2^x; results below 2^-126 become 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Codes of 4 keys (rows r) x 4 dims -> 4 dims x 4 keys.
OBN_DEVINL void transpose4(uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3, uint32_t (&o)[4]) {
  const uint32_t a = __byte_perm(r0, r1, 0x5140), b = __byte_perm(r0, r1, 0x7362);
  const uint32_t c = __byte_perm(r2, r3, 0x5140), d = __byte_perm(r2, r3, 0x7362);
  o[0] = __byte_perm(a, c, 0x5410);
  o[1] = __byte_perm(a, c, 0x7632);
  o[2] = __byte_perm(b, d, 0x5410);
  o[3] = __byte_perm(b, d, 0x7632);
}

OBN_DEVINL void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

// The codes as a 4-D tensor (128 dims, KV heads, positions, sequences), boxes of `rows`
// positions of one head, 128-byte swizzle; rows past S_max read as zeros.
inline bool q8_map(CUtensorMap* map, const int8_t* codes, const Q8Cache& c, int rows) {
  const cuuint64_t row = static_cast<cuuint64_t>(c.Hkv) * kQ8HeadDim;
  const cuuint64_t dims[4] = {kQ8HeadDim, static_cast<cuuint64_t>(c.Hkv), static_cast<cuuint64_t>(c.S_max),
                              static_cast<cuuint64_t>(c.B)};
  const cuuint64_t strides[3] = {kQ8HeadDim, row, row * c.S_max};
  const cuuint32_t box[4] = {kQ8HeadDim, 1, static_cast<cuuint32_t>(rows), 1};
  const cuuint32_t one[4] = {1, 1, 1, 1};
  auto fn = tensor_map_encoder();
  return fn && fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<int8_t*>(codes), dims, strides,
                  box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Bounded wait on an mbarrier phase that leaves the issue slots to the warps that work: each
// try sleeps up to 20 us, the whole wait up to half a second. Gives up (and raises the abort flag
// and the device error word) at the bound, or once another role has.
OBN_DEVINL bool q8_wait(volatile int* abort_flag, uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < (1u << 15); ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
        : "memory");
    if (ok) return true;
    if (*abort_flag) return false;
  }
  record_error(DEVERR_MBAR_TIMEOUT);
  *abort_flag = 1;
  return false;
}

// Workspace of a pass of `rows` rows per tile: the notes of the splits; then for each of 2 C
// slots the sums [rows][128], the maxima and the totals [rows] (all f32).
OBN_DEVINL float* q8_part_o(float* ws, int rows, int slot) {
  return ws + 4 * kQ8MaxCtas + static_cast<size_t>(slot) * rows * (kQ8HeadDim + 2);
}
OBN_DEVINL float* q8_part_ml(float* ws, int rows, int slot) {
  return q8_part_o(ws, rows, slot) + static_cast<size_t>(rows) * kQ8HeadDim;
}
constexpr size_t q8_workspace(int rows, int ctas) {
  return (4 * kQ8MaxCtas + static_cast<size_t>(2) * ctas * rows * (kQ8HeadDim + 2)) * sizeof(float);
}

}  // namespace obn
