// Paged attention of many rows per key head (a prompt's chunk): bound by the matrix cores, and
// beside them by what the LDS can deliver and what the softmax costs.
//
// A tile is 256 rows, 64 for each of four waves, which share the keys and values: 64 keys at a
// time in LDS, two buffers of each, moved by DMA (each wave 16 keys) and waited for one tile
// later.  A wave's operand from LDS (32 keys x 16 values for S^T = K Q^T, 32 columns x 16 keys for
// O^T = V^T P^T, on the 32x32x16 MFMA) serves both of its 32-row halves: with 32 rows a wave the
// four waves' operands alone would take all of the LDS bandwidth.  Q^T stays in registers, and so
// do S^T and the weights: a lane holds one row and keys 8 (i / 4) + 4 (lane / 32) + i % 4, which
// is the order in which P^T and V^T (through the transposing LDS read) take a product's keys.
//
// The products of one half tile's weights with the values are issued together with the
// exponentials of the next one's scores, so that the vector unit works while the matrix unit does.
// Weights are rounded to bf16 for the product, 2^-9 of each: a second part (as for few rows) would be
// half as many products again, of a kernel that they bound.  The sum that they are divided by is that of the
// rounded ones, so that a row of one heavy key is exact.  They are relative to the row's first
// maximum, not to the running one: bf16 and f32 hold weights of 2^60 as exactly as those below 1, and
// nothing is left to multiply the sums with in the loop.  A tile with a score past 2^60 times its
// reference is run again from the maxima that the first time has found.
//
// 2048 tokens over 32768 keys (24 query heads on 4 of 256; 1.6 TFLOP): 1477-1564 us with the join, 1.02-1.08
// PFLOP/s, the matrix cores 52% busy at the clock that the power limit leaves.
#include "attention.h"
#include "gemm_pipe.h"

namespace qmm {

namespace {

constexpr int CH_TR = 256, CH_KT = 64;
constexpr int CH_EXTRA = 3;  // what a tile's own overhead (queries in, rows out) costs, in units of 64 keys
constexpr int CH_TAB = 4 * 2 * 256 + 2 * 4 * 4;  // page ids of the tiles to come, two sets per wave; valid keys

constexpr int ch_tile(int DP) { return CH_KT * DP * 2; }  // bytes of a tile of keys (or of values)

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void ch_dma4(const void *g, uint32_t l) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(l), "v"(g) : "memory", "m0");
}
// LDS DMA of 16 bytes per lane to l + `at` (see gp_dma16).
__device__ __forceinline__ void ch_dma16(const void *g, uint32_t l, int at) {
  asm volatile("s_add_i32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(l), "v"(g), "i"(at) : "memory", "m0", "scc");
}
#pragma clang diagnostic pop

// S^T's products, written out so that S^T lies in vector registers: the sums of O^T (of 256
// columns x 64 rows) take all of the accumulation registers, where the compiler puts the results of
// a kernel's MFMA builtins.  The matrix unit runs products that add to one result in order; others
// that read a result wait (an 8-pass product's can be read after 11 wait states).
__device__ __forceinline__ void ch_mfma_first(f32x16_t &c, bf16x8_t x, bf16x8_t y) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(x), "v"(y));
}
__device__ __forceinline__ void ch_mfma(f32x16_t &c, bf16x8_t x, bf16x8_t y) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(x), "v"(y));
}
__device__ __forceinline__ void ch_mfma_done(f32x16_t &c0, f32x16_t &c1) {
  asm volatile("s_nop 15\n\ts_nop 3" : "+v"(c0), "+v"(c1));
}

template <int DP, bool FULL>
__global__ __launch_bounds__(ATTN_THREADS, DP == 64 ? 2 : 1) void attn_chunk_kernel(const AttnArgs args, const AttnShare share) {
  constexpr int CPR = DP / 8;
  constexpr int KS = DP / 16;     // k steps of S^T
  constexpr int DT = DP / 32;     // 32-column tiles of O^T
  constexpr int OPS = DP / 32;    // DMA operations of a wave's 16 rows
  constexpr int TILE = ch_tile(DP), PITCH = 2 * DP;
  constexpr int PLAN = 4 * TILE + CH_TAB + 16 * ATTN_THREADS;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  uint8_t *tab = lds + 4 * TILE;
  uint32_t *vm = (uint32_t *)(tab + 4 * 2 * 256);  // [2][4]
  int *seen_at = (int *)(tab + CH_TAB);  // [thread][2][2]: what its rows see
  AttnPlan *plan = (AttnPlan *)(seen_at + 4 * ATTN_THREADS);
  int *poison = plan->poison, *redo = &plan->redo;

  const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  auto here = [&]() __attribute__((always_inline)) { return wv * 64 + (int)attn_lane(); };  // the thread's number
  int left;
  {
    const AttnWork w = attn_uniform(attn_share<CH_TR, CH_KT, CH_EXTRA>(args, share, plan));
    if (share.first) attn_zero_rest(args);
    attn_note_none(share, w);
    if (tid == 0) plan->work[0] = w;
    left = attn_uniform(w.left);
  }
  const uint32_t la = lds_addr(lds), ta = lds_addr(tab) + wv * 512;
  if constexpr (!FULL) {  // head values past D: never written by the DMA
    for (int i = tid; i < 4 * TILE / 16; i += ATTN_THREADS) ((uint4 *)lds)[i] = attn_zeros();
  }

  int turn = 0;
  while (left > 0) {
    __syncthreads();
    const AttnArgs a = attn_again<AttnArgs>(0);
    AttnPlan *plan = (AttnPlan *)((int *)lds + attn_uniform(attn_opaque(PLAN / 4)));
    const AttnWork w = attn_uniform(plan->work[turn]);
    const int r = attn_uniform(attn_request(plan, a.R, w));
    const AttnReq rq = attn_uniform(attn_req(plan, a, r));
    const AttnTile t = attn_uniform(attn_tile(a, rq, w.tile - (r ? attn_end(plan, a.R, r - 1) : 0), CH_TR));
    const int units = attn_units<CH_KT>(t);
    const AttnPiece pc = attn_piece<CH_EXTRA>(w, units);
    const int ks = (int)((uint32_t)t.b / CH_KT + pc.u0) * CH_KT, nt = pc.u1 - pc.u0;
    const bool whole = pc.whole;
    const int part = w.g * 2 + pc.start, head = w.head;
    if (pc.start && !pc.none && here() == 0) attn_note(attn_again<AttnShare>(sizeof(AttnArgs)), w, rq, t, units + CH_EXTRA, whole);
    {
      AttnWork on = w;
      on.r = r;
      attn_move_on(on, pc.take, units + CH_EXTRA);
      left = on.left;
      turn ^= 1;
      if (here() == 0) plan->work[turn] = on;
    }
    if (pc.none) continue;
    if (units == 0) {  // no keys
      const uint32_t per = (uint32_t)a.D / 8;
      for (uint32_t j = here(); j < t.rows * per; j += ATTN_THREADS) {
        const uint32_t row = j / per;
        const float z = __int_as_float(attn_opaque(0));
        float o[8] = {z, z, z, z, z, z, z, z};
        attn_store8(a, attn_row(a, rq.q0, t.row0 + row, head), (j - row * per) * 8, o);
      }
      continue;
    }

    if (here() == 0) *poison = attn_opaque(0), *redo = attn_opaque(0);
    const int *tabrow = a.table + (int64_t)r * a.W;
    const int block = a.block, NB = a.NB, Hkv = a.Hkv, D = a.D;
    const uint32_t pitch = 2 * (uint32_t)D;  // (of a cache row; a multiply-add beats a shift and two adds)
    const uint16_t *kc = a.k, *vc = a.v;
    // the lane's rows
    float m[2], l[2];
    bf16x8_t q[2][KS];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t ln = attn_lane();
      const int in = wv * 64 + u * 32 + (int)(ln & 31), lh = (int)(ln >> 5);
      const bool on = in < t.rows;
      const int row = t.row0 + (on ? in : 0);  // (a row past the end: the first one's queries)
      const int tok = (int)attn_div(row, a.by_g), pos = rq.base + tok;
      seen_at[(wv * 64 + (int)ln) * 4 + 2 * u] = a.window && pos >= a.window ? pos - a.window + 1 : 0;
      seen_at[(wv * 64 + (int)ln) * 4 + 2 * u + 1] = on ? pos : -1;
      // (a row that sees nothing needs no reference; one past the end has no weights and passes none)
      m[u] = !on ? __builtin_inff() : pos >= 0 ? -__builtin_inff() : 0.f;
      const uint16_t *qp = a.q + attn_row(a, rq.q0, row, head) * a.D + lh * 8;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if (FULL || k * 16 + lh * 8 < a.D)
          q[u][k] = *(const bf16x8_t *)(qp + k * 16);
        else
          q[u][k] = __builtin_bit_cast(bf16x8_t, u32x4_t{0u, 0u, 0u, 0u});
      }
    }
    if (!(a.scale > 0.f)) {  // a negative scale: -q, so that maxima stay maxima; none: no scores
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          u32x4_t x = __builtin_bit_cast(u32x4_t, q[u][k]);
          x = a.scale < 0.f ? x ^ 0x80008000u : u32x4_t{0u, 0u, 0u, 0u};
          q[u][k] = __builtin_bit_cast(bf16x8_t, x);
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the compiler's own waits would come between the DMA's
    const float sc = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.44269504088896341f;

    f32x16_t acc[DT][2];
    bool again = false;
    do {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][u][i] = 0.f;
    l[0] = l[1] = 0.f;
    bool passed = false;
      f32x16_t sv[2];
      bf16x8_t p[2][2];     // weights [16 keys][half]
      u32x4_t np[2][2];     // the next ones
      float ls[2], ref[2], top[2];

      // Keys on their way: this lane looks up key wv * 16 + lane % 16 of each tile.  `off` is its place in
      // its page, for the tile whose rows come next; `page` and `poff` are two tiles on.
      const uint32_t per = attn_div(CH_KT, a.by_block), rest = CH_KT - per * (uint32_t)block;
      const uint32_t first = ks + wv * 16 + ((int)attn_lane() & 15);
      const uint32_t first_page = attn_div(first, a.by_block), first_off = first - first_page * block;
      const uint32_t last_page = attn_div(t.e - 1, a.by_block);
      const int page0 = tabrow[first_page < last_page ? first_page : last_page];
      uint32_t page = first_page, poff = first_off, off = first_off;
      auto onward = [&](uint32_t &pg, uint32_t &of) __attribute__((always_inline)) {
        pg += per, of += rest;
        if (of >= (uint32_t)block) of -= block, ++pg;
      };
      auto ask = [&](int set) __attribute__((always_inline)) {  // page ids of tile `page`
        ch_dma4(tabrow + (page < last_page ? page : last_page), ta + set * 256);
      };
      uint32_t mine = 0;  // the row (of the whole cache) of this lane's key, 0 where there is none
      auto rows_of = [&](int k0, uint32_t of, int blk, int set) __attribute__((always_inline)) {
        const bool ok = k0 + wv * 16 + ((int)attn_lane() & 15) < t.e && (uint32_t)blk < (uint32_t)NB;
        mine = (((uint32_t)blk * Hkv + head) * block + of) & (ok ? ~0u : 0u);
        const uint32_t mask = (uint32_t)__ballot(ok) & 0xFFFFu;
        vm[set * 4 + wv] = mask;  // (by all lanes: no branch)
      };
      // DMA operation n: rows RPI n .. of the wave's 16, chunk (lane % CPR) ^ swizzle of each
      constexpr int RPI = 64 / CPR;
      struct From {
        uint32_t lane, c;  // whose row operation 0 moves, and where in it
        uint32_t row;      // of the next operation, asked for an operation before
      };
      auto from_of = [&](auto swz) __attribute__((always_inline)) {
        const uint32_t ln = attn_lane();
        const uint32_t lane = ln / CPR * 4;
        return From{lane, (ln % CPR ^ (uint32_t)swz((int)(ln / CPR))) * 16, (uint32_t)__builtin_amdgcn_ds_bpermute((int)lane, (int)mine)};
      };
      auto move = [&](const uint16_t *cache, From &f, int n, int to, auto swz) __attribute__((always_inline)) {
        const uint32_t row = f.row, c = f.c ^ (uint32_t)swz(RPI * n) * 16;
        if (n + 1 < OPS) f.row = __builtin_amdgcn_ds_bpermute((int)f.lane + RPI * (n + 1) * 4, (int)mine);
        if (FULL || c < 2 * (uint32_t)D)
          ch_dma16((const char *)cache + c + (uint64_t)row * pitch, la + to + wv * 16 * PITCH, n * 1024);
      };
      const auto swz_k = [](int r) { return attn_swz<DP>(r); };
      const auto swz_v = [](int r) { return attn_swz_v<DP>(r); };
      auto move_k = [&](From &f, int set, int n) __attribute__((always_inline)) { move(kc, f, n, set * TILE, swz_k); };
      auto move_v = [&](From &f, int set, int n) __attribute__((always_inline)) { move(vc, f, n, (2 + set) * TILE, swz_v); };

      // S^T of 32 keys; beside it, the DMA of a tile's values
      auto scores = [&](int set, int half, bool values) __attribute__((always_inline)) {
        // (k steps 8 apart differ by 256 bytes, which the swizzle leaves alone)
        const uint32_t ln = attn_lane();
        const int lq = ln & 31;
        const int from = set * TILE + half * 32 * PITCH + lq * PITCH + ((int)(ln >> 5) ^ attn_swz<DP>(lq)) * 16;
        auto load = [&](int k) __attribute__((always_inline)) {
          return *(const bf16x8_t *)(lds + (from ^ (k & 7) * 32) + (k >> 3) * 256);
        };
        constexpr int AHEAD = 2;
        bf16x8_t kf[KS];
        From f{};
        if (values) f = from_of(swz_v);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) kf[k] = load(k);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          if (k + AHEAD < KS) kf[k + AHEAD] = load(k + AHEAD);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (k == 0)
              ch_mfma_first(sv[u], kf[k], q[u][k]);
            else
              ch_mfma(sv[u], kf[k], q[u][k]);
          }
          if (values && k % 2 == 0) move_v(f, set, k / 2);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      // where rows see different keys, or have no reference yet
      auto special = [&](int k0, uint32_t valid, bool edge) __attribute__((always_inline)) {
        const bool fresh = __any(m[0] == -__builtin_inff() || m[1] == -__builtin_inff());
        if (!edge && !fresh) return;
        ch_mfma_done(sv[0], sv[1]);
        if (edge) {
          const int h4 = (int)attn_lane() >> 5 << 2;
          const int4 rows = *(const int4 *)(seen_at + (wv * 64 + (int)attn_lane()) * 4);
          const int seen_b[2] = {rows.x, rows.z}, seen_e[2] = {rows.y, rows.w};
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            // bit o: key k0 + o is seen
            const int lo = seen_b[u] - k0, hi = seen_e[u] - k0;
            uint32_t seen = hi < 0 ? 0u : hi > 30 ? ~0u : (2u << hi) - 1u;
            seen &= lo > 31 ? 0u : lo > 0 ? ~0u << lo : ~0u;
            seen &= valid;
            if (__all(seen == ~0u)) continue;  // (a wave's 64 rows differ on fewer keys than the tile's)
            seen >>= h4;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int on = __builtin_amdgcn_sbfe((int)seen, 8 * (i / 4) + i % 4, 1);  // 0 or -1
              sv[u][i] = __uint_as_float((__float_as_uint(sv[u][i]) & (uint32_t)on) | (0xFF800000u & ~(uint32_t)on));
            }
          }
        }
        if (fresh) {  // (before its first key a row has no sums: any reference will do from here)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float x = sv[u][0];
#pragma unroll
            for (int i = 1; i < 16; ++i) x = fmaxf(x, sv[u][i]);
            x = fmaxf(x, attn_across(x, 32)) * sc;
            m[u] = m[u] == -__builtin_inff() ? x : m[u];
          }
        }
      };
      // Step n of N: its part of the weights of sv into np, their sums into ls, the scores' maxima into top
      auto weights = [&](int n, int N) __attribute__((always_inline)) {
        if (n == 0) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
            ls[u] = 0.f, top[u] = -__builtin_inff(), ref[u] = m[u] == -__builtin_inff() ? 0.f : m[u];
        }
#pragma unroll
        for (int j = n * (16 / N); j < (n + 1) * (16 / N); ++j) {
          const int c = j >> 3, u = j >> 2 & 1, e = (j & 3) * 2;
          const float s0 = sv[u][c * 8 + e], s1 = sv[u][c * 8 + e + 1];
          asm("v_max3_f32 %0, %0, %1, %2" : "+v"(top[u]) : "v"(s0), "v"(s1));  // (fmaxf would first quiet each)
          bf16x2_t x;
          x[0] = (__bf16)attn_exp2(__builtin_fmaf(s0, sc, -ref[u]));
          x[1] = (__bf16)attn_exp2(__builtin_fmaf(s1, sc, -ref[u]));
          ls[u] = dot2_bf16(x, 0x3F803F80u, ls[u]);
          uint32_t pair = __builtin_bit_cast(uint32_t, x);
          asm volatile("" : "+v"(pair));  // (here, not later: beside the product)
          np[c][u][e / 2] = pair;
        }
      };
      // the weights become the next product's; a reference passed by 2^60: noted, and followed for the second run
      auto settle = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          l[u] += ls[u];
#pragma unroll
          for (int c = 0; c < 2; ++c) p[c][u] = __builtin_bit_cast(bf16x8_t, np[c][u]);
        }
        const bool far = top[0] * sc > m[0] + 60.f || top[1] * sc > m[1] + 60.f;
        if (__any(far)) {
          passed = true;
#pragma unroll
          for (int u = 0; u < 2; ++u) m[u] = fmaxf(m[u], top[u] * sc);
        }
      };
      // O^T += V^T P^T over 32 keys; beside it the next weights and the DMA of a tile's keys
      auto product = [&](int set, int half, bool with, int keys) __attribute__((always_inline)) {
        const uint32_t ln = attn_lane();
        const int row = 4 * (ln >> 5) + (ln >> 2 & 3);
        const int from = la + (2 + set) * TILE + (half * 32 + row) * PITCH +
                         ((int)((ln >> 4 & 1) * 2 + (ln >> 1 & 1)) ^ attn_swz_v<DP>(row)) * 16 + (ln & 1) * 8;
        constexpr int N = 2 * DT, AHEAD = 2;
        auto load = [&](int n) __attribute__((always_inline)) {
          const int d = n % DT, c = n / DT;  // (the first 16 keys' weights are done with half way)
          const uint32_t at = (from ^ (d & 3) * 64) + (d >> 2) * 256 + c * 16 * PITCH;
          const i16x4_t v0 = attn_read_tr(at), v1 = attn_read_tr(at + 8 * PITCH);
          return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        bf16x8_t vf[N];
        From f{};
        if (keys >= 0) f = from_of(swz_k);
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) vf[n] = load(n);
#pragma unroll
        for (int n = 0; n < N; ++n) {
          if (n + AHEAD < N) vf[n + AHEAD] = load(n + AHEAD);
#pragma unroll
          for (int u = 0; u < 2; ++u)
            acc[n % DT][u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[n], p[n / DT][u], acc[n % DT][u], 0, 0, 0);
          if (n == 0 && with)  // (since the last score's product: two products, six reads and their addresses)
            asm volatile("s_nop 3" : "+v"(sv[0]), "+v"(sv[1]));
          if (with) weights(n, N);
          if (keys >= 0 && n % 2 == 0) move_k(f, keys, n / 2);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      auto edge_at = [&](int k0, uint64_t valid) -> bool {
        return k0 < t.full_b || k0 + CH_KT > t.full_e || valid != ~0ull;
      };
      auto valid_of = [&](uint4 v) -> uint64_t {
        const uint32_t lo = __builtin_amdgcn_readfirstlane(v.x | v.y << 16);
        const uint32_t hi = __builtin_amdgcn_readfirstlane(v.z | v.w << 16);
        return (uint64_t)hi << 32 | lo;
      };

      rows_of(ks, off, page0, 0);
      onward(page, poff);
      ask(1);
      off = poff;
      onward(page, poff);
      {
        From f = from_of(swz_k);
#pragma unroll
        for (int n = 0; n < OPS; ++n) move_k(f, 0, n);
      }
      // Tile i: scores of its first half | values of tile i; weights of those with the product of tile i - 1's
      // second half | keys of tile i + 1; the same for its second half.
      // (what is asked for past the last tile is not used; the waits count on it)
      uint64_t valid;
      bool edge;
      auto begin = [&](int i) __attribute__((always_inline)) {
        const int set = i & 1, k0 = ks + i * CH_KT;
        gp_wait_barrier<0>();  // keys of tile i, page ids of tile i + 1, everyone's valid bits
        const uint4 bits = *(const uint4 *)(vm + set * 4);
        const int blk = *(const int *)(tab + wv * 512 + (set ^ 1) * 256 + (int)attn_lane() * 4);
        scores(set, 0, true);
        valid = valid_of(bits);
        edge = edge_at(k0, valid);
        special(k0, (uint32_t)valid, edge);
        rows_of(k0 + CH_KT, off, blk, set ^ 1);
        ask(set);
        off = poff;
        onward(page, poff);
      };
      auto middle = [&](int i) __attribute__((always_inline)) {
        const int set = i & 1;
        scores(set, 1, false);
        special(ks + i * CH_KT + 32, (uint32_t)(valid >> 32), edge);
        // values of tile i (the page ids and keys asked for after them may be on their way)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(OPS + 1) : "memory");
        const int own = ks + i * CH_KT + wv * 16;  // (the values that this wave has moved)
        if (edge && (((valid >> wv * 16) & 0xFFFFu) != 0xFFFFu || (again && (own < t.full_b || own + 16 > t.full_e)))) {
          const uint32_t ln = attn_lane();
          bool odd = false;
#pragma unroll
          for (int j = 0; j < OPS; ++j) {
            uint4 *at = (uint4 *)(lds + (2 + set) * TILE + wv * 16 * PITCH + j * 1024 + ln * 16);
            const uint4 x = *at, y = attn_finite(x);
            const bool in = valid >> (wv * 16 + (j * 64 + ln) / CPR) & 1;
            odd |= in && (x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w);
            *at = in ? y : attn_zeros();
            __builtin_amdgcn_sched_barrier(0);
          }
          if (__any(odd)) *poison = attn_opaque(1);
        }
        gp_lds_barrier();
      };
      // (before the first: no weights, and no values that they could meet)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < 2; ++c) p[c][u] = __builtin_bit_cast(bf16x8_t, u32x4_t{0u, 0u, 0u, 0u});
      for (int j = here(); j < TILE / 32; j += ATTN_THREADS) ((uint4 *)(lds + 3 * TILE + TILE / 2))[j] = attn_zeros();
#pragma unroll 1
      for (int i = 0; i < nt; ++i) {
        begin(i);
        product((i + 1) & 1, 1, true, (i + 1) & 1);
        settle();
        middle(i);
        product(i & 1, 0, true, -1);
        settle();
      }
      product((nt - 1) & 1, 1, false, -1);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (!again && (ks < t.full_b || ks + nt * CH_KT > t.full_e)) {
      // Keys that some rows do not see had weights of zero there, and 0 inf is NaN: sums that are not finite are
      // formed again with such values held back.
      float z = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          f32x16_t x = acc[d][u];
          asm volatile("" : "+a"(x));
#pragma unroll
          for (int i = 0; i < 16; ++i) z = __builtin_fmaf(x[i], 0.f, z);
          __builtin_amdgcn_sched_barrier(0);
        }
      passed |= z != 0.f;
    }
    if (__any(passed)) *redo = attn_opaque(1);
    __syncthreads();
    again = !again && *redo;
    if (again) {
#pragma unroll
      for (int u = 0; u < 2; ++u) m[u] = fmaxf(m[u], attn_across(m[u], 32));
    }
    __syncthreads();
    } while (again);

    {
    const AttnArgs a = attn_again<AttnArgs>(0);
    const AttnShare s = attn_again<AttnShare>(sizeof(AttnArgs));
    // Rows out, 32 of a wave and half of their columns at a time, through the wave's quarter of the LDS: sums in its
    // first half (pairs of 16-byte chunks, swizzled by row), the 32 rows' gates in the second.
    constexpr int HC = DP / 2, PAIRS = HC / 8, IT = 32 * PAIRS / 64;
    float *out = (float *)(lds + wv * TILE);
    const int end = ks + nt * CH_KT < t.e ? ks + nt * CH_KT : t.e;
    const bool gated = whole && a.gate;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int in0 = wv * 64 + u * 32;
      if (in0 >= t.rows) break;
      if (gated) {
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
          const uint32_t j = i * 64 + (int)attn_lane();
          int in = in0 + (int)(j / CPR);
          in = in < t.rows ? in : in0;
          const int c = (int)(j % CPR) * 8;
          if (FULL || c < a.D)
            gp_dma16(a.gate + attn_row(a, rq.q0, t.row0 + in, head) * a.Dg + (a.Dg - a.D) + c,
                     la + wv * TILE + TILE / 2 + i * 1024);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      const float lu = l[u] + attn_across(l[u], 32);
      const float scale = !whole ? 1.f : lu != 0.f ? 1.f / lu : 0.f;
      const int l32 = (int)attn_lane();
      if (!whole && l32 < 32 && in0 + l32 < t.rows) {
        const int64_t pr = (int64_t)part * CH_TR + in0 + l32;
        s.ml[pr * 2] = m[u], s.ml[pr * 2 + 1] = lu;
      }
#pragma unroll
      for (int hc = 0; hc < 2; ++hc) {
        const int ln = (int)attn_lane();  // (nothing of this is kept through the loop before)
        float *mine = out + (ln & 31) * HC + (ln >> 5) * 4;
        const int turn = ln & (PAIRS - 1);
#pragma unroll
        for (int d = 0; d < DT / 2; ++d) {
          f32x16_t x = acc[hc * (DT / 2) + d][u];
          asm volatile("" : "+a"(x));  // (from the accumulation registers here, not all of them at once)
#pragma unroll
          for (int v = 0; v < 4; ++v)
            *(float4 *)(mine + ((d * 4 + v) ^ turn) * 8) =
                make_float4(x[4 * v] * scale, x[4 * v + 1] * scale, x[4 * v + 2] * scale, x[4 * v + 3] * scale);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (hc == 0 && gated) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int it = 0; it < IT; ++it) {
          const uint32_t j = it * 64 + ln;
          const int rr = (int)(j / PAIRS), k = (int)(j % PAIRS), in = in0 + rr, d0 = hc * HC + k * 8;
          if (in >= t.rows || (!FULL && d0 >= a.D)) continue;
          const float *x = out + rr * HC + (k ^ (rr & (PAIRS - 1))) * 8;
          float o[8];
          *(float4 *)&o[0] = *(const float4 *)x, *(float4 *)&o[4] = *(const float4 *)(x + 4);
          if (*poison) attn_poison(a, rq, tabrow, head, t.row0 + in, ks, end, d0, o);
          if (whole) {
            if (gated) attn_times_gate(*(const uint4 *)(lds + wv * TILE + TILE / 2 + (rr * DP + d0) * 2), o);
            attn_put8(a, attn_row(a, rq.q0, t.row0 + in, head), d0, o);
          } else {
            float4 *to = (float4 *)(s.acc + ((int64_t)part * CH_TR + in) * DP + d0);
            to[0] = make_float4(o[0], o[1], o[2], o[3]), to[1] = make_float4(o[4], o[5], o[6], o[7]);
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the gates are read before the next ones come)
    }
    }
    if constexpr (!FULL) {
      __syncthreads();
      for (int j = here(); j < 4 * TILE / 16; j += ATTN_THREADS) ((uint4 *)lds)[j] = attn_zeros();
    }
  }
}

template <int DP, bool FULL>
hipError_t launch_t(const AttnArgs &a, const AttnShare &s, int grid, hipStream_t st) {
  static std::atomic<uint64_t> done{0};
  const void *k = (const void *)attn_chunk_kernel<DP, FULL>;
  const hipError_t e = ensure_dynamic_lds(done, k, (int)attn_chunk_lds(DP, ATTN_MAX_R));
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((attn_chunk_kernel<DP, FULL>), dim3(grid), dim3(ATTN_THREADS), attn_chunk_lds(DP, a.R), st, a, s);
  return hipGetLastError();
}

template <int DP>
hipError_t launch_dp(const AttnArgs &a, const AttnShare &s, int grid, hipStream_t st) {
  return a.D == DP ? launch_t<DP, true>(a, s, grid, st) : launch_t<DP, false>(a, s, grid, st);
}

}  // namespace

size_t attn_chunk_lds(int DP, int R) {
  return 4 * ch_tile(DP) + CH_TAB + 16 * ATTN_THREADS + attn_plan_lds(R);
}

hipError_t launch_attn_chunk(const AttnArgs &a, const AttnShare &s, int DP, int grid, hipStream_t st) {
  return DP == 64 ? launch_dp<64>(a, s, grid, st) : DP == 128 ? launch_dp<128>(a, s, grid, st) : launch_dp<256>(a, s, grid, st);
}

}  // namespace qmm
