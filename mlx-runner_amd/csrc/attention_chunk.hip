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
// Weights are rounded to bf16 for the product (see attention_rows.hip).  They are relative to the
// row's first maximum, not to the running one: bf16 and f32 hold weights of 2^60 as exactly as
// those below 1, and nothing is left to multiply the sums with in the loop.  A tile with a score
// past 2^60 times its reference is run again from the maxima that the first time has found.
#include "attention.h"
#include "gemm_pipe.h"

namespace qmm {

namespace {

constexpr int CH_TR = 256, CH_KT = 64;
constexpr int CH_TAB = 4 * 2 * 256 + 2 * 4 * 4;  // page ids of the tiles to come, two sets per wave; valid keys

constexpr int ch_tile(int DP) { return CH_KT * DP * 2; }  // bytes of a tile of keys (or of values)

// Chunk c of row r of the values: 4 rows of 64 bytes (a transposing read of 32 lanes) in distinct banks.
template <int DP>
__device__ __forceinline__ int ch_swz_v(int row) {
  return DP >= 128 ? (row & 3) << 2 : (row & 2) << 1;
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void ch_dma4(const void *g, uint32_t l) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(l), "v"(g) : "memory", "m0");
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
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  uint8_t *tab = lds + 4 * TILE;
  uint32_t *vm = (uint32_t *)(tab + 4 * 2 * 256);  // [2][4]
  uint32_t *scratch = (uint32_t *)(tab + CH_TAB);
  int *ends = (int *)((uint8_t *)scratch + ATTN_SCAN_LDS + sizeof(AttnWork)), *poison = (int *)scratch + 15, *redo = (int *)scratch + 14;

  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lq = lane & 31, lh = lane >> 5;
  const int g = args.Hq / args.Hkv;
  AttnWork *work = (AttnWork *)(scratch + ATTN_SCAN_LDS / 4);  // (this workgroup's share, out of the registers)
  int left;
  {
    if (share.first) attn_zero_rest(args);
    const AttnWork w = attn_share<CH_TR, CH_KT, 1>(args, share, ends, scratch);
    attn_note_none(share, w);
    if (tid == 0) *work = w;
    left = attn_uniform(w.left);
  }
  const uint32_t la = lds_addr(lds), ta = lds_addr(tab) + wv * 512;
  if constexpr (!FULL) {  // head values past D: never written by the DMA
    for (int i = tid; i < 4 * TILE / 16; i += ATTN_THREADS) ((uint4 *)lds)[i] = make_uint4(0, 0, 0, 0);
  }

  while (left > 0) {
    __syncthreads();
    const AttnArgs a = attn_again<AttnArgs>(0);
    const AttnWork w = attn_uniform(*work);
    const int r = attn_uniform(attn_find(ends, a.R, w.tile));
    const AttnReq rq = attn_uniform(attn_req(a, r, g));
    const AttnTile t = attn_tile(a, rq, w.tile - (r ? attn_uniform(ends[r - 1]) : 0), CH_TR, g);
    const int cost = attn_units<CH_KT>(t) + 1;
    const int take = cost - w.u < w.left ? cost - w.u : w.left;
    const int u0 = w.u > 0 ? w.u - 1 : 0, u1 = w.u + take - 1;  // (the first unit: the tile's own overhead)
    const int ks = (t.b / CH_KT + u0) * CH_KT, nt = u1 - u0;
    const bool whole = take == cost;
    const int part = w.g * 2 + (w.u == 0 ? 1 : 0), head = w.head;
    {
      const AttnShare s = attn_again<AttnShare>(sizeof(AttnArgs));
      if (w.u == 0 && tid == 0) attn_note(s, w, rq, t, cost, whole);
      left = w.left - take;
      __syncthreads();
      if (tid == 0) {
        work->left = left;
        work->at = w.at + take;
        work->u = w.u + take;
        if (w.u + take == cost) {
          const bool last = w.tile + 1 == w.tiles;
          work->u = 0;
          work->tile = last ? 0 : w.tile + 1;
          work->head = w.head + last;
        }
      }
      if (nt == 0) {  // no keys: zeros, or a part of nothing
        if (whole) {
          for (int j = tid; j < t.rows * (a.D / 8); j += ATTN_THREADS) {
            float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            attn_store8(a, attn_row(a, rq.q0, t.row0 + j / (a.D / 8), head, g), j % (a.D / 8) * 8, o);
          }
        } else if (tid < t.rows) {
          const int64_t pr = (int64_t)part * CH_TR + tid;
          s.ml[pr * 2] = -__builtin_inff(), s.ml[pr * 2 + 1] = 0.f;
        }
        continue;
      }
    }

    if (tid == 0) *poison = 0, *redo = 0;
    const int *tabrow = a.table + (int64_t)r * a.W;
    const int block = a.block, NB = a.NB, Hkv = a.Hkv, D = FULL ? DP : a.D;
    const uint16_t *kc = a.k, *vc = a.v;
    const uint32_t first = ks + wv * 16 + (lane & 15);
    const uint32_t first_page = first / (uint32_t)block, first_off = first - first_page * block;
    const uint32_t last_page = (uint32_t)(t.e - 1) / (uint32_t)block;
    const int page0 = tabrow[first_page < last_page ? first_page : last_page];
    // the lane's rows
    int seen_b[2], seen_e[2];
    bf16x8_t q[2][KS];
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int in = wv * 64 + u * 32 + lq, row = t.row0 + in;
      const bool on = in < t.rows;
      const int tok = on ? row / g : 0, hh = on ? row - tok * g : 0;
      const int pos = rq.base + tok;
      seen_e[u] = on ? pos : -1;
      seen_b[u] = a.window && pos >= a.window ? pos - a.window + 1 : 0;
      const uint16_t *qp = a.q + (((int64_t)(rq.q0 + tok) * a.Hq) + head * g + hh) * a.D;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int d0 = k * 16 + lh * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (on && (FULL || d0 < a.D) && a.scale != 0.f) v = *(const uint4 *)(qp + d0);
        v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
        q[u][k] = __builtin_bit_cast(bf16x8_t, v);
      }
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the compiler's own waits would come between the DMA's
    const float sc = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.44269504088896341f;

    f32x16_t acc[DT][2];
    float m[2], l[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) m[u] = seen_e[u] < 0 ? 0.f : -__builtin_inff();  // (a row that sees nothing)
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
      const uint32_t per = CH_KT / (uint32_t)block, rest = CH_KT % (uint32_t)block;
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
        const bool ok = k0 + wv * 16 + (attn_opaque(lane) & 15) < t.e && (uint32_t)blk < (uint32_t)NB;
        mine = ok ? ((uint32_t)blk * Hkv + head) * block + of : 0u;
        const uint32_t mask = (uint32_t)__ballot(ok) & 0xFFFFu;
        if (lane == 0) vm[set * 4 + wv] = mask;
      };
      // DMA operation n: rows RPI n .. of the wave's 16, chunk (lane % CPR) ^ swizzle of each
      constexpr int RPI = 64 / CPR;
      auto move = [&](const uint16_t *cache, int n, int to, auto swz) __attribute__((always_inline)) {
        const uint32_t ln = attn_opaque(lane);
        const uint32_t row = __builtin_amdgcn_ds_bpermute((int)(ln / CPR * 4) + RPI * n * 4, (int)mine);
        const uint32_t c = (ln % CPR ^ (uint32_t)swz((int)(ln / CPR)) ^ (uint32_t)swz(RPI * n)) * 16;
        if (FULL || c < 2 * (uint32_t)D)
          gp_dma16((const char *)cache + ((uint64_t)row * (2 * (uint32_t)D) + c), la + to + wv * 16 * PITCH + n * 1024);
      };
      auto move_k = [&](int set, int n) __attribute__((always_inline)) {
        move(kc, n, set * TILE, [](int r) { return attn_swz<DP>(r); });
      };
      auto move_v = [&](int set, int n) __attribute__((always_inline)) {
        move(vc, n, (2 + set) * TILE, [](int r) { return ch_swz_v<DP>(r); });
      };

      // S^T of 32 keys; beside it, the DMA of a tile's values
      auto scores = [&](int set, int half, bool values) __attribute__((always_inline)) {
        // (k steps 8 apart differ by 256 bytes, which the swizzle leaves alone)
        const uint32_t ln = attn_opaque(lane);
        const int lq = ln & 31;
        const int from = set * TILE + half * 32 * PITCH + lq * PITCH + ((int)(ln >> 5) ^ attn_swz<DP>(lq)) * 16;
        auto load = [&](int k) __attribute__((always_inline)) {
          return *(const bf16x8_t *)(lds + (from ^ (k & 7) * 32) + (k >> 3) * 256);
        };
        constexpr int AHEAD = 2;
        bf16x8_t kf[KS];
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
          if (values && k % 2 == 0) move_v(set, k / 2);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      // where rows see different keys, or have no reference yet
      auto special = [&](int k0, uint32_t valid, bool edge) __attribute__((always_inline)) {
        const bool fresh = __any(m[0] == -__builtin_inff() || m[1] == -__builtin_inff());
        if (!edge && !fresh) return;
        ch_mfma_done(sv[0], sv[1]);
        if (edge) {
          const int h4 = attn_opaque(4 * lh);
          const uint32_t bits = valid >> h4;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int lo = seen_b[u] - k0 - h4, hi = seen_e[u] - k0 - h4;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int o = 8 * (i / 4) + i % 4;
              if (!(o <= hi && o >= lo && (bits >> o & 1))) sv[u][i] = -__builtin_inff();
              __builtin_amdgcn_sched_barrier(0);  // (one mask at a time)
            }
          }
        }
        if (fresh) {  // (before its first key a row has no sums: any reference will do from here)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float x = sv[u][0];
#pragma unroll
            for (int i = 1; i < 16; ++i) x = fmaxf(x, sv[u][i]);
            x = fmaxf(x, __shfl_xor(x, 32, 64)) * sc;
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
          const int u = j >> 3, c = j >> 2 & 1, e = (j & 3) * 2;
          const float s0 = sv[u][c * 8 + e], s1 = sv[u][c * 8 + e + 1];
          top[u] = fmaxf(top[u], fmaxf(s0, s1));
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
        const uint32_t ln = attn_opaque(lane);
        const int row = 4 * (ln >> 5) + (ln >> 2 & 3);
        const int from = la + (2 + set) * TILE + (half * 32 + row) * PITCH +
                         ((int)((ln >> 4 & 1) * 2 + (ln >> 1 & 1)) ^ ch_swz_v<DP>(row)) * 16 + (ln & 1) * 8;
        constexpr int N = 2 * DT, AHEAD = 2;
        auto load = [&](int n) __attribute__((always_inline)) {
          const int d = n >> 1, c = n & 1;
          const uint32_t at = (from ^ (d & 3) * 64) + (d >> 2) * 256 + c * 16 * PITCH;
          const i16x4_t v0 = attn_read_tr(at), v1 = attn_read_tr(at + 8 * PITCH);
          return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        bf16x8_t vf[N];
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) vf[n] = load(n);
#pragma unroll
        for (int n = 0; n < N; ++n) {
          if (n + AHEAD < N) vf[n + AHEAD] = load(n + AHEAD);
#pragma unroll
          for (int u = 0; u < 2; ++u)
            acc[n >> 1][u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[n], p[n & 1][u], acc[n >> 1][u], 0, 0, 0);
          if (n == 0 && with) ch_mfma_done(sv[0], sv[1]);
          if (with) weights(n, N);
          if (keys >= 0 && n % 2 == 0) move_k(keys, n / 2);
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
#pragma unroll
      for (int n = 0; n < OPS; ++n) move_k(0, n);
      // Tile i: scores of its first half | values of tile i; weights of those with the product of tile i - 1's
      // second half | keys of tile i + 1; the same for its second half.
      // (what is asked for past the last tile is not used; the waits count on it)
      uint64_t valid;
      bool edge;
      auto begin = [&](int i) __attribute__((always_inline)) {
        const int set = i & 1, k0 = ks + i * CH_KT;
        gp_wait_barrier<0>();  // keys of tile i, page ids of tile i + 1, everyone's valid bits
        const uint4 bits = *(const uint4 *)(vm + set * 4);
        const int blk = *(const int *)(tab + wv * 512 + (set ^ 1) * 256 + attn_opaque(lane) * 4);
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
        if (edge) {  // (see attention_rows.hip)
          bool odd = false;
#pragma unroll 1
          for (int j = 0; j < OPS; ++j) {
            uint4 *at = (uint4 *)(lds + (2 + set) * TILE + wv * 16 * PITCH + j * 1024 + lane * 16);
            const uint4 x = *at, y = attn_finite(x);
            const bool in = valid >> (wv * 16 + (j * 64 + lane) / CPR) & 1;
            odd |= in && (x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w);
            *at = in ? y : make_uint4(0, 0, 0, 0);
          }
          if (__any(odd)) *poison = 1;
        }
        gp_lds_barrier();
      };
      begin(0);
      ch_mfma_done(sv[0], sv[1]);
      weights(0, 1);
#pragma unroll
      for (int n = 0; n < OPS; ++n) move_k(1, n);
      settle();
      middle(0);
      product(0, 0, true, -1);
      settle();
      for (int i = 1; i < nt; ++i) {
        begin(i);
        product((i + 1) & 1, 1, true, (i + 1) & 1);
        settle();
        middle(i);
        product(i & 1, 0, true, -1);
        settle();
      }
      product((nt - 1) & 1, 1, false, -1);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (__any(passed)) *redo = 1;
    __syncthreads();
    again = !again && *redo;
    if (again) {
#pragma unroll
      for (int u = 0; u < 2; ++u) m[u] = fmaxf(m[u], __shfl_xor(m[u], 32, 64));
    }
    __syncthreads();
    } while (again);

    {
    const AttnArgs a = attn_again<AttnArgs>(0);
    const AttnShare s = attn_again<AttnShare>(sizeof(AttnArgs));
    // rows out, 32 of a wave and half of their columns at a time, through the wave's quarter of the LDS
    constexpr int HC = DP / 2, OP = HC + 4, IT = 32 * (HC / 8) / 64, AT_ONCE = IT < 4 ? IT : 4;
    float *out = (float *)(lds + wv * TILE);
    const int end = ks + nt * CH_KT < t.e ? ks + nt * CH_KT : t.e;
#pragma unroll
    for (int u = 0; u < 2; ++u) l[u] += __shfl_xor(l[u], 32, 64);
#pragma unroll 1
    for (int stage = 0; stage < 4; ++stage) {
      const int u = stage >> 1, hc = stage & 1, in0 = wv * 64 + u * 32;
      if (in0 >= t.rows) break;
      const float lu = u ? l[1] : l[0], scale = !whole ? 1.f : lu != 0.f ? 1.f / lu : 0.f;
      if (!whole && hc == 0 && lane < 32 && in0 + lq < t.rows) {
        const int64_t pr = (int64_t)part * CH_TR + in0 + lq;
        s.ml[pr * 2] = u ? m[1] : m[0], s.ml[pr * 2 + 1] = lu;
      }
      auto to_lds = [&](int us, int hs) __attribute__((always_inline)) {
#pragma unroll
        for (int d = 0; d < DT / 2; ++d)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const f32x16_t &x = acc[hs * (DT / 2) + d][us];
            *(float4 *)(out + lq * OP + d * 32 + v * 8 + lh * 4) =
                make_float4(x[4 * v] * scale, x[4 * v + 1] * scale, x[4 * v + 2] * scale, x[4 * v + 3] * scale);
          }
      };
      switch (stage) {
        case 0: to_lds(0, 0); break;
        case 1: to_lds(0, 1); break;
        case 2: to_lds(1, 0); break;
        default: to_lds(1, 1); break;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      auto at = [&](int it, int *in, int *d0) -> float * {
        const int j = it * 64 + lane, rr = j / (HC / 8), c0 = j % (HC / 8) * 8;
        *in = in0 + rr, *d0 = hc * HC + c0;
        return out + rr * OP + c0;
      };
      if (*poison) {
#pragma unroll 1
        for (int it = 0; it < IT; ++it) {
          int in, d0;
          float *x = at(it, &in, &d0), o[8];
          if (in >= t.rows || d0 >= a.D) continue;
          *(float4 *)&o[0] = *(const float4 *)x, *(float4 *)&o[4] = *(const float4 *)(x + 4);
          attn_poison(a, rq, tabrow, head, t.row0 + in, g, ks, end, d0, o);
          *(float4 *)x = *(const float4 *)&o[0], *(float4 *)(x + 4) = *(const float4 *)&o[4];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
#pragma unroll 1
      for (int it0 = 0; it0 < IT; it0 += AT_ONCE) {
        uint4 gates[AT_ONCE];  // (asked for before the first is used)
        int64_t rows[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          int in, d0;
          at(it0 + i, &in, &d0);
          rows[i] = attn_row(a, rq.q0, t.row0 + in, head, g);
          if (whole && a.gate && in < t.rows && d0 < a.D) gates[i] = attn_gate8(a, rows[i], d0);
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          int in, d0;
          const float *x = at(it0 + i, &in, &d0);
          if (in >= t.rows || d0 >= a.D) continue;
          float o[8];
          *(float4 *)&o[0] = *(const float4 *)x, *(float4 *)&o[4] = *(const float4 *)(x + 4);
          if (whole) {
            if (a.gate) attn_times_gate(gates[i], o);
            attn_put8(a, rows[i], d0, o);
          } else {
            float4 *to = (float4 *)(s.acc + ((int64_t)part * CH_TR + in) * DP + d0);
            to[0] = make_float4(o[0], o[1], o[2], o[3]), to[1] = make_float4(o[4], o[5], o[6], o[7]);
          }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    }
    if constexpr (!FULL) {
      __syncthreads();
      for (int j = tid; j < 4 * TILE / 16; j += ATTN_THREADS) ((uint4 *)lds)[j] = make_uint4(0, 0, 0, 0);
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
  return 4 * ch_tile(DP) + CH_TAB + ATTN_SCAN_LDS + sizeof(AttnWork) + (size_t)R * 4;
}

hipError_t launch_attn_chunk(const AttnArgs &a, const AttnShare &s, int DP, int grid, hipStream_t st) {
  return DP == 64 ? launch_dp<64>(a, s, grid, st) : DP == 128 ? launch_dp<128>(a, s, grid, st) : launch_dp<256>(a, s, grid, st);
}

}  // namespace qmm
