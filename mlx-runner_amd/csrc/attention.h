// Pieces shared by the paged-attention kernels: what a tile of query rows sees, how the work is
// shared among workgroups, where partial results go.
//
// The g = Hq / Hkv query heads of a key head and the n new tokens of a request make n g rows
// (row = token * g + head) that read the same keys; a tile is TR of them, for one key head.  Its
// keys run from the first that any of its rows sees to the last; their cost is counted in units
// of KT keys.  All (head, tile, unit) in a line are cut into equal shares, one per workgroup, so
// requests of any lengths fill the chip evenly; a tile cut between workgroups leaves its partial
// sums (unnormalised, with the rows' maxima and sums) in the workspace, and a second kernel joins
// them.  Which workgroup runs what follows from the lengths alone: every workgroup scans them
// itself, nothing is planned on the host.
#pragma once

#include "qmm_device.h"
#include "qmm_launch.h"

namespace qmm {

constexpr int ATTN_THREADS = 256;

__device__ __forceinline__ uint32_t attn_div(uint32_t n, FastDiv d) { return __umulhi(n << 1, d.mul) >> d.shift; }

// A launch over the requests of min_rows < n g <= max_rows rows.
struct AttnShare {
  int min_rows, max_rows;
  int first;        // this launch writes the rows of no request (zeros)
  // The tiles cut between workgroups, for the joining kernel: [.][8], first and last workgroup (first -1: none),
  // q0, row0, rows, key head; one for each workgroup (it starts at most one such tile), or, where that is
  // fewer, one for each tile (by head * count + tile).
  int by_tile;
  int tiles;        // per head at most (what is over, by requests that overlap, is left out)
  int *count;       // tiles per head, workgroups with work
  int *desc;
  float *ml;        // [2 workgroups][TR][2]: maximum and sum of a partial's rows
  float *acc;       // [2 workgroups][TR][DP]
};

// The same value in all lanes, into scalar registers.
template <class T>
__device__ __forceinline__ T attn_uniform(const T &x) {
  struct Words {
    int w[sizeof(T) / 4];
  } v = __builtin_bit_cast(Words, x);
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / 4; ++i) v.w[i] = __builtin_amdgcn_readfirstlane(v.w[i]);
  return __builtin_bit_cast(T, v);
}

struct AttnReq {
  int q0, n, base;  // first row of q, tokens, position of the first
  int rows;
};

__device__ __forceinline__ AttnReq attn_req(const AttnArgs &a, int r) {
  AttnReq q;
  const int s0 = a.q_starts[r], s1 = a.q_starts[r + 1], kv = a.kv_lens[r];
  q.q0 = s0 < 0 ? 0 : s0 < a.T ? s0 : a.T;
  const int q1 = s1 < q.q0 ? q.q0 : s1 < a.T ? s1 : a.T;
  q.n = q1 - q.q0;
  q.base = (kv < 0 ? 0 : kv) - q.n;
  q.rows = q.n * a.g;
  return q;
}

// The keys of a tile: [b, e) are seen by some row, [full_b, full_e) by all.
struct AttnTile {
  int row0, rows;  // of the request; rows of the tile
  int b, e, full_b, full_e;
};

__device__ __forceinline__ AttnTile attn_tile(const AttnArgs &a, const AttnReq &q, int j, int tr) {
  AttnTile t;
  t.row0 = j * tr;
  t.rows = q.rows - t.row0 < tr ? q.rows - t.row0 : tr;
  // positions of the ends
  const int p0 = q.base + (int)attn_div(t.row0, a.by_g), p1 = q.base + (int)attn_div(t.row0 + t.rows - 1, a.by_g);
  const int64_t cap64 = (int64_t)a.W * a.block;
  const int cap = cap64 < 0x7FFF0000 ? (int)cap64 : 0x7FFF0000;  // (ends rounded up stay in range)
  t.e = p1 < cap ? p1 + 1 : cap;
  t.full_e = p0 < cap ? p0 + 1 : cap;
  t.b = 0, t.full_b = 0;
  if (a.window) {  // (p0 may be below 0 and the window 2^31 - 1: no difference of them before the comparison)
    t.b = p0 >= a.window ? p0 - a.window + 1 : 0;
    t.full_b = p1 >= a.window ? p1 - a.window + 1 : 0;
  }
  if (t.e < t.b) t.e = t.b;  // (also no key at all: e <= 0)
  return t;
}

template <int KT>
__device__ __forceinline__ int attn_units(const AttnTile &t) {
  return t.e > t.b ? (int)(((uint32_t)t.e + KT - 1) / KT - (uint32_t)t.b / KT) : 0;
}

// Inclusive sum over the wave's lanes: over each row of 16, then the rows before.
__device__ __forceinline__ uint32_t attn_wave_scan(uint32_t v) {
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);  // row_shr:1, 2, 4, 8
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1, 3
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2, 3
  return v;
}
// Over the workgroup; the total too.
__device__ __forceinline__ uint32_t attn_scan(uint32_t v, uint32_t *waves, uint32_t *total) {
  const int wave = threadIdx.x >> 6;
  v = attn_wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) waves[wave] = v;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < ATTN_THREADS / 64; ++w) {
    if (w == wave) before = all;
    all += waves[w];
  }
  *total = all;
  return before + v;
}

// A workgroup's share: `left` units from unit `u` of (head, tile) on, request r's.  Of `groups` workgroups the first
// `longer` have one unit more than the others.
struct AttnWork {
  int g, groups, share, longer;
  int tiles;         // per head
  uint32_t at;       // the place of unit `u` in the line of all units
  int head, tile, r;
  int u, left;
};

// A workgroup's LDS for this, [R] ends of the requests' tiles behind it: with the requests themselves up to ATTN_KEPT.
constexpr int ATTN_KEPT = 256;
struct __attribute__((aligned(16))) AttnPlan {
  AttnWork work[2];     // this segment's, the next one's: out of the registers
  uint32_t waves[4], found[3];
  uint16_t owner[64];   // a tile's request, and its number there
  int poison[2], redo;
};
inline __host__ __device__ size_t attn_plan_lds(int R) { return sizeof(AttnPlan) + (size_t)R * (R <= ATTN_KEPT ? 16 : 4); }

__device__ __forceinline__ int attn_end(const AttnPlan *plan, int R, int r) {
  return ((const int *)(plan + 1))[R <= ATTN_KEPT ? 4 * r : r];
}
__device__ __forceinline__ void attn_keep(AttnPlan *plan, int R, int r, uint32_t end, const AttnReq &q) {
  if (R <= ATTN_KEPT)
    ((int4 *)(plan + 1))[r] = make_int4((int)end, q.q0, q.n, q.base);
  else
    ((int *)(plan + 1))[r] = (int)end;
}
__device__ __forceinline__ AttnReq attn_req(const AttnPlan *plan, const AttnArgs &a, int r) {
  if (a.R > ATTN_KEPT) return attn_req(a, r);
  const int4 x = ((const int4 *)(plan + 1))[r];
  return AttnReq{x.y, x.z, x.w, x.z * a.g};
}
// The request of tile i: the first r with end(r) > i.
__device__ __forceinline__ int attn_find(const AttnPlan *plan, int R, int i) {
  int lo = 0, hi = R - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (attn_end(plan, R, mid) > i)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// EXTRA units a tile costs beside its keys'.
template <int TR, int KT, int EXTRA>
__device__ __forceinline__ AttnWork attn_share(const AttnArgs &a, const AttnShare &s, AttnPlan *plan) {
  const int tid = threadIdx.x, lane = tid & 63;
  const uint32_t most = (uint32_t)s.tiles;
  AttnWork w;
  w.left = 0, w.g = 0, w.groups = 0, w.r = 0;
  // this workgroup's part of the line, of `per_head` units for each head; the place of its first unit
  auto cut = [&](uint32_t per_head) __attribute__((always_inline)) -> uint32_t {
    const uint32_t total = per_head * (uint32_t)a.Hkv;
    w.groups = (int)(total < gridDim.x ? total : gridDim.x);
    w.share = (int)(total / (uint32_t)w.groups);
    w.longer = (int)(total - (uint32_t)w.share * (uint32_t)w.groups);
    // consecutive shares, which read the same keys, on one XCD (workgroups go to the 8 in turn)
    const int per = (w.groups + 7) >> 3, y = blockIdx.x >> 3;
    w.g = (blockIdx.x & 7) * per + y;
    if (y >= per || w.g >= w.groups) return 0;
    w.at = (uint32_t)w.g * (uint32_t)w.share + (uint32_t)(w.g < w.longer ? w.g : w.longer);
    w.left = w.share + (w.g < w.longer);
    w.head = (int)(w.at / per_head);
    return w.at - (uint32_t)w.head * per_head;
  };
  auto tiles_of = [&](const AttnReq &q) __attribute__((always_inline)) -> uint32_t {
    const uint32_t n = q.rows > s.min_rows && q.rows <= s.max_rows ? (uint32_t)(q.rows + TR - 1) / TR : 0u;
    return n < most ? n : most;
  };
  uint32_t run = 0, all = 0;
  if (a.R <= 64) {  // every wave for itself, a request per lane, no barrier (all write the same)
    AttnReq q{0, 0, 0, 0};
    if (lane < a.R) q = attn_req(a, lane);
    const uint32_t nt = tiles_of(q), end = attn_wave_scan(nt);
    if (lane < a.R) attn_keep(plan, a.R, lane, end < most ? end : most, q);
    run = (uint32_t)__builtin_amdgcn_readlane((int)end, 63);
    run = run < most ? run : most;
    w.tiles = (int)run;
    if (run == 0) return w;
    if (run <= 64) {  // and a tile per lane
      for (uint32_t j = 0; __any(j < nt); ++j)
        if (j < nt && end - nt + j < 64) plan->owner[end - nt + j] = (uint16_t)(lane | j << 8);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      uint32_t mine = 0, r = 0;
      if (lane < (int)run) {
        const uint32_t o = plan->owner[lane];
        r = o & 255;
        mine = (uint32_t)(attn_units<KT>(attn_tile(a, attn_req(plan, a, (int)r), (int)(o >> 8), TR)) + EXTRA);
      }
      const uint32_t to = attn_wave_scan(mine);
      const uint32_t x = cut((uint32_t)__builtin_amdgcn_readlane((int)to, 63));
      if (!w.left) return w;
      w.tile = __builtin_ctzll(__ballot(x < to && x >= to - mine) | 1ull << 63);
      w.u = (int)(x - (uint32_t)__builtin_amdgcn_readlane((int)(to - mine), w.tile));
      w.r = __builtin_amdgcn_readlane((int)r, w.tile);
      return w;
    }
  } else {
#pragma unroll 1
    for (int r0 = 0; r0 < a.R; r0 += ATTN_THREADS) {
      const int r = r0 + tid;
      AttnReq q{0, 0, 0, 0};
      if (r < a.R) q = attn_req(a, r);
      const uint32_t end = run + attn_scan(tiles_of(q), plan->waves, &all);
      if (r < a.R) attn_keep(plan, a.R, r, end < most ? end : most, q);
      run = run + all < most ? run + all : most;
    }
    w.tiles = (int)run;
  }
  __syncthreads();
  // Units of the tiles, ATTN_THREADS at a time: first all of them, for the shares; then until the tile with the
  // share's first unit (where there are no more than that, the first turn's values still serve).
  uint32_t mine = 0, end = 0, x = 0;
  int r = 0;
  run = 0;
  bool sought = false;
#pragma unroll 1
  for (int i0 = 0; i0 < w.tiles;) {
    if (!sought || w.tiles > ATTN_THREADS) {
      const int i = i0 + tid;
      mine = 0;
      if (i < w.tiles) {
        r = attn_find(plan, a.R, i);
        mine = (uint32_t)(attn_units<KT>(attn_tile(a, attn_req(plan, a, r), i - (r ? attn_end(plan, a.R, r - 1) : 0), TR)) + EXTRA);
      }
      end = run + attn_scan(mine, plan->waves, &all);
      run += all;
    }
    if (sought && x < end && x >= end - mine)
      plan->found[0] = (uint32_t)(i0 + tid), plan->found[1] = x - (end - mine), plan->found[2] = (uint32_t)r;
    i0 += ATTN_THREADS;
    if (!sought && i0 >= w.tiles) {
      x = cut(run);
      if (!w.left) return w;
      sought = true;
      i0 = 0, run = 0;
    }
  }
  __syncthreads();
  w.tile = (int)plan->found[0];
  w.u = (int)plan->found[1];
  w.r = (int)plan->found[2];
  return w;
}
// The request of the share's tile: that of the last one, the one after, or sought.
__device__ __forceinline__ int attn_request(const AttnPlan *plan, int R, const AttnWork &w) {
  if (w.tile == 0) return attn_find(plan, R, 0);
  if (attn_end(plan, R, w.r) > w.tile) return w.r;
  if (w.r + 1 < R && attn_end(plan, R, w.r + 1) > w.tile) return w.r + 1;
  return attn_find(plan, R, w.tile);
}
// The workgroup whose share unit `at` of the line is in.
__device__ __forceinline__ int attn_group_of(const AttnWork &w, uint32_t at) {
  const uint32_t head = (uint32_t)w.longer * (uint32_t)(w.share + 1);
  return (int)(at < head ? at / (uint32_t)(w.share + 1) : (uint32_t)w.longer + (at - head) / (uint32_t)w.share);
}

// What a workgroup does of the tile that its share has come to: the key units [u0, u1) of `units`.  A tile's first
// EXTRA units stand for its own overhead; who has the first key unit starts it.
struct AttnPiece {
  int take, u0, u1;
  bool whole, start, none;
};
template <int EXTRA>
__device__ __forceinline__ AttnPiece attn_piece(const AttnWork &w, int units) {
  AttnPiece p;
  const int cost = units + EXTRA;
  p.take = cost - w.u < w.left ? cost - w.u : w.left;
  p.u0 = w.u > EXTRA ? w.u - EXTRA : 0;
  p.u1 = w.u + p.take > EXTRA ? w.u + p.take - EXTRA : 0;
  p.start = p.u0 == 0;
  p.whole = p.start && p.u1 == units;
  p.none = units ? p.u1 <= p.u0 : w.u + p.take < cost;  // (a tile without keys: its zeros with its last unit)
  return p;
}
__device__ __forceinline__ void attn_move_on(AttnWork &w, int take, int cost) {
  w.left -= take;
  w.at += (uint32_t)take;
  w.u += take;
  if (w.u == cost) {
    w.u = 0;
    const bool last = ++w.tile == w.tiles;
    w.tile = last ? 0 : w.tile;
    w.head += last;
  }
}

// Notes the tile that this workgroup starts (by one thread).
__device__ __forceinline__ void attn_note(const AttnShare &s, const AttnWork &w, const AttnReq &q, const AttnTile &t,
                                          int cost, bool whole) {
  int *d = s.desc + (s.by_tile ? (int64_t)w.head * w.tiles + w.tile : (int64_t)w.g) * 8;
  if (whole) {
    if (s.by_tile) d[0] = -1;
    return;
  }
  d[0] = w.g, d[1] = attn_group_of(w, w.at - (uint32_t)w.u + (uint32_t)cost - 1u);
  d[2] = q.q0, d[3] = t.row0, d[4] = t.rows, d[5] = w.head;
}
// First of all: how many tiles and workgroups with work; no tile noted yet.
__device__ __forceinline__ void attn_note_none(const AttnShare &s, const AttnWork &w) {
  if (threadIdx.x != 0) return;
  if (blockIdx.x == 0) s.count[0] = w.tiles, s.count[1] = w.groups;
  if (!s.by_tile && w.left > 0) s.desc[w.g * 8] = -1;
}

// Zeros for the rows of no request, by all workgroups of a launch.
__device__ __forceinline__ void attn_zero_rest(const AttnArgs &a) {
  const int lo = a.R ? a.q_starts[0] : a.T, hi = a.R ? a.q_starts[a.R] : a.T;
  const int cpr = a.D / 8;
  const int64_t per_row = (int64_t)a.Hq * cpr;
  auto fill = [&](int t0, int t1) {
    for (int64_t i = t0 * per_row + (int64_t)blockIdx.x * ATTN_THREADS + threadIdx.x; i < t1 * per_row;
         i += (int64_t)gridDim.x * ATTN_THREADS)
      ((uint4 *)a.o)[i] = make_uint4(0, 0, 0, 0);
  };
  fill(0, a.R ? (lo < 0 ? 0 : lo < a.T ? lo : a.T) : a.T);
  if (a.R) fill(hi < 0 ? 0 : hi < a.T ? hi : a.T, a.T);
}

// Row `row` of a request: its (token, query head) in q, gate and o.
__device__ __forceinline__ int64_t attn_row(const AttnArgs &a, int q0, int row, int head) {
  const int tok = (int)attn_div(row, a.by_g);
  return (int64_t)(q0 + tok) * a.Hq + head * a.g + (row - tok * a.g);
}
// Eight values of a finished row (divided by its sum), d0 a multiple of 8 below D: the gate of them, times
// its sigmoid, their rounding.
__device__ __forceinline__ uint4 attn_gate8(const AttnArgs &a, int64_t row, int d0) {
  return *(const uint4 *)(a.gate + row * a.Dg + (a.Dg - a.D) + d0);
}
__device__ __forceinline__ float attn_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ void attn_times_gate(uint4 d, float (&v)[8]) {
  const uint32_t w[4] = {d.x, d.y, d.z, d.w};
  constexpr float LOG2E = 1.44269504088896341f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] *= __builtin_amdgcn_rcpf(1.f + attn_exp2(-LOG2E * __uint_as_float(w[i] << 16)));
    v[2 * i + 1] *= __builtin_amdgcn_rcpf(1.f + attn_exp2(-LOG2E * __uint_as_float(w[i] & 0xFFFF0000u)));
  }
}
__device__ __forceinline__ void attn_put8(const AttnArgs &a, int64_t row, int d0, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bf16x2_t x;
    x[0] = (__bf16)v[2 * i], x[1] = (__bf16)v[2 * i + 1];
    w[i] = __builtin_bit_cast(uint32_t, x);
  }
  *(uint4 *)(a.o + row * a.D + d0) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void attn_store8(const AttnArgs &a, int64_t row, int d0, float (&v)[8]) {
  if (a.gate) attn_times_gate(attn_gate8(a, row, d0), v);
  attn_put8(a, row, d0, v);
}

// bf16 values in pairs, those that are not finite replaced by zero.
__device__ __forceinline__ uint32_t attn_finite(uint32_t x) {
  x = (x & 0x7F80u) == 0x7F80u ? x & 0xFFFF0000u : x;
  return (x & 0x7F800000u) == 0x7F800000u ? x & 0xFFFFu : x;
}
__device__ __forceinline__ uint4 attn_finite(uint4 x) {
  return make_uint4(attn_finite(x.x), attn_finite(x.y), attn_finite(x.z), attn_finite(x.w));
}

// Adds to 8 sums of a row the values that are not finite of the keys in [ks, ke) that it sees: what was
// left out where the rows of a tile see different keys.  Slow, and only where there are any.
__device__ __forceinline__ void attn_poison(const AttnArgs &a, const AttnReq &q, const int *tabrow, int head,
                                                      int row, int ks, int ke, int d0, float (&o)[8]) {
  const int pos = q.base + (int)attn_div(row, a.by_g);
  const int hi = pos < ke - 1 ? pos : ke - 1;
  int lo = a.window && pos >= a.window && pos - a.window + 1 > ks ? pos - a.window + 1 : ks;
#pragma unroll 1
  for (int key = lo; key <= hi; ++key) {
    const uint32_t page = attn_div(key, a.by_block);
    const int blk = tabrow[page];
    if ((uint32_t)blk >= (uint32_t)a.NB) continue;
    const uint64_t r = ((uint64_t)blk * a.Hkv + head) * a.block + ((uint32_t)key - page * (uint32_t)a.block);
    const uint4 v = *(const uint4 *)(a.v + r * a.D + d0);
    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if ((x[e] & 0x7F80u) == 0x7F80u) o[2 * e] += __uint_as_float(x[e] << 16);
      if ((x[e] & 0x7F800000u) == 0x7F800000u) o[2 * e + 1] += __uint_as_float(x[e] & 0xFFFF0000u);
    }
  }
}

// LDS rows of keys or values are DP bf16 in 16-byte chunks; chunk c of row r lies at c ^ attn_swz(r), so that
// the reads of one chunk (or pair) of 16 rows touch every bank once.
template <int DP>
__device__ __forceinline__ int attn_swz(int row) {
  return DP >= 128 ? row & 15 : (row >> 1) & 7;
}


// A value that the compiler takes as new here: what follows from it (swizzled addresses) is formed
// again where it is used, a few xors, instead of being kept in registers through the loop.
__device__ __forceinline__ int attn_opaque(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// The lane's number, formed here: not kept in a register through a loop that needs all of them.
__device__ __forceinline__ uint32_t attn_lane() {
  uint32_t x;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
  return x;
}

__device__ __forceinline__ uint4 attn_zeros() {
  const uint32_t z = (uint32_t)attn_opaque(0);
  return make_uint4(z, z, z, z);
}

// x of lane ^ `other`.
__device__ __forceinline__ float attn_across(float x, int other) {
  return __int_as_float(__builtin_amdgcn_ds_bpermute(((int)attn_lane() ^ other) * 4, __float_as_int(x)));
}

// A kernel's arguments (at `offset` of its argument block) read again where they are needed, instead of
// holding scalar registers through the loop before.
template <class T>
__device__ __forceinline__ T attn_again(int offset) {
  typedef const __attribute__((address_space(4))) uint32_t *block_t;
  block_t p = (block_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  struct Words {
    uint32_t w[sizeof(T) / 4];
  } x;
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / 4; ++i) x.w[i] = p[offset / 4 + i];
  return __builtin_bit_cast(T, x);
}

typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef short i16x8_t __attribute__((ext_vector_type(8)));

// 4 x 16 values read across: the 16 lanes of a group give the addresses of four rows of 32 bytes,
// lane i that of bytes 8 (i % 4) of row i / 4; lane i gets column i of the four rows.
__device__ __forceinline__ i16x4_t attn_read_tr(uint32_t at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t *)(uintptr_t)at);
}

// Launches of the kernels (the workspace's parts in s).
size_t attn_rows_lds(int DP, int R);
size_t attn_chunk_lds(int DP, int R);
hipError_t launch_attn_chunk(const AttnArgs &a, const AttnShare &s, int DP, int grid, hipStream_t st);
hipError_t launch_attn_rows(const AttnArgs &a, const AttnShare &s, int DP, int tr, int grid, hipStream_t st);

}  // namespace qmm
