// kvq8_sched.cuh — how attention over the 8-bit cache is spread over the GPU.
//
// The query rows of a sequence and KV head (t * G + g for token t and group head g) are cut
// into tiles of `tile_rows`; an item is a (sequence, tile), a pair an item with a KV head,
// and a unit kUnitKeys keys of a pair. All units of all pairs in a row, T of them, are dealt
// out evenly: CTA c of C <= T takes units [c T / C, (c + 1) T / C). So sequences of any mix of
// lengths and causal tiles of any depth keep every CTA equally busy, and one long sequence
// is split as finely as many short ones. A pair that lies inside one CTA is written
// out by it; the parts of a pair that spans CTAs go to the workspace and are joined by
// k_q8_join. A CTA holds at most two parts: one that continues a pair (slot 2c) and one that
// begins a pair and does not end it (slot 2c + 1).
#pragma once

#include "kvq8.h"
#include "obn_common.cuh"

namespace obn {

constexpr int kUnitKeys = 128;
constexpr int kQ8MaxCtas = 640;  // bounds C, and with it the workspace

struct Q8Sched {
  int B, n, G, Hkv;
  int tile_rows, tiles;  // rows per tile, tiles per sequence
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
// CTAs that take part: every one of them has a unit, and so a part where a pair spans it.
OBN_DEVINL int q8_ctas(const Q8Sched& s, long long total) {
  return static_cast<int>(min(static_cast<long long>(s.ctas), total));
}
OBN_DEVINL long long q8_begin(long long total, int ctas, int c) { return c * total / ctas; }
// The CTA that holds unit x.
OBN_DEVINL int q8_owner(long long total, int ctas, long long x) {
  return static_cast<int>(((x + 1) * ctas - 1) / total);
}

// For all THREADS threads of the CTA: the total of units, and with `before` items given the
// units in front of item `before` (sh: THREADS + 1 shared words).
template <int THREADS>
OBN_DEVINL long long q8_total(const Q8Sched& s, int before, long long* in_front, long long* sh) {
  const int items = s.B * s.tiles, tid = threadIdx.x;
  if (!s.lens && s.tiles == 1) {
    const long long u = q8_units(s, 0);
    *in_front = u * before * s.Hkv;
    return u * items * s.Hkv;
  }
  long long all = 0, front = 0;
  for (int i = tid; i < items; i += THREADS) {
    const int u = q8_units(s, i);
    all += u;
    if (i < before) front += u;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, d);
    front += __shfl_xor_sync(0xffffffffu, front, d);
  }
  constexpr int W = THREADS / 32;
  if (tid % 32 == 0) {
    sh[tid / 32] = all;
    sh[W + tid / 32] = front;
  }
  __syncthreads();
  all = front = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    all += sh[w];
    front += sh[W + w];
  }
  __syncthreads();
  *in_front = front * s.Hkv;
  return all * s.Hkv;
}

// A place in the row of units.
struct Q8Cursor {
  int item, kvh, unit, units;  // units: those of the item
};

// The item, KV head and unit of unit `x` < total: each thread adds up a run of items, a scan
// finds the run, its thread walks it. sh: THREADS + 4 shared words.
template <int THREADS>
OBN_DEVINL Q8Cursor q8_find(const Q8Sched& s, long long x, long long* sh) {
  const int items = s.B * s.tiles, tid = threadIdx.x;
  Q8Cursor c;
  if (!s.lens && s.tiles == 1) {
    c.units = q8_units(s, 0);
    const long long pair = x / c.units;
    c.item = static_cast<int>(pair / s.Hkv);
    c.kvh = static_cast<int>(pair % s.Hkv);
    c.unit = static_cast<int>(x % c.units);
    return c;
  }
  const int per = (items + THREADS - 1) / THREADS;
  const int i0 = min(tid * per, items), i1 = min(i0 + per, items);
  long long sum = 0;
  for (int i = i0; i < i1; ++i) sum += q8_units(s, i);
  sum *= s.Hkv;
  long long incl = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, d);
    if (tid % 32 >= d) incl += o;
  }
  if (tid % 32 == 31) sh[tid / 32] = incl;
  __syncthreads();
  for (int w = 0; w < tid / 32; ++w) incl += sh[w];
  long long at = incl - sum;
  if (x >= at && x < incl) {
    int i = i0;
    for (;; ++i) {
      const long long u = static_cast<long long>(q8_units(s, i)) * s.Hkv;
      if (x < at + u) break;
      at += u;
    }
    const int u = q8_units(s, i);
    sh[THREADS] = i;
    sh[THREADS + 1] = (x - at) / u;
    sh[THREADS + 2] = (x - at) % u;
    sh[THREADS + 3] = u;
  }
  __syncthreads();
  c.item = static_cast<int>(sh[THREADS]);
  c.kvh = static_cast<int>(sh[THREADS + 1]);
  c.unit = static_cast<int>(sh[THREADS + 2]);
  c.units = static_cast<int>(sh[THREADS + 3]);
  __syncthreads();
  return c;
}

// The next unit (the caller stops at the end of its share, so there is one).
OBN_DEVINL void q8_next(const Q8Sched& s, Q8Cursor& c) {
  if (++c.unit < c.units) return;
  c.unit = 0;
  if (++c.kvh < s.Hkv) return;
  c.kvh = 0;
  const int items = s.B * s.tiles;
  do {
    if (++c.item >= items) return;
    c.units = q8_units(s, c.item);
  } while (c.units == 0);
}

// Workspace of a pass of `rows` rows per tile: for each of 2 C slots the sums [rows][128],
// then the maxima and totals [rows] (all f32).
OBN_DEVINL float* q8_part_o(float* ws, int rows, int slot) {
  return ws + static_cast<size_t>(slot) * rows * (kQ8HeadDim + 2);
}
OBN_DEVINL float* q8_part_ml(float* ws, int rows, int slot) {
  return q8_part_o(ws, rows, slot) + static_cast<size_t>(rows) * kQ8HeadDim;
}
inline size_t q8_workspace(int rows) {
  return static_cast<size_t>(2) * kQ8MaxCtas * rows * (kQ8HeadDim + 2) * sizeof(float);
}

}  // namespace obn
