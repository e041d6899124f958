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
__global__ __launch_bounds__(ATTN_THREADS, DP == 64 ? 2 : 1) void attn_chunk_kernel(const AttnArgs a, const AttnShare s) {
  constexpr int CPR = DP / 8;
  constexpr int KS = DP / 16;     // k steps of S^T
  constexpr int DT = DP / 32;     // 32-column tiles of O^T
  constexpr int OPS = DP / 32;    // DMA operations of a wave's 16 rows
  constexpr int TILE = ch_tile(DP), PITCH = 2 * DP;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  uint8_t *tab = lds + 4 * TILE;
  uint32_t *vm = (uint32_t *)(tab + 4 * 2 * 256);  // [2][4]
  uint32_t *scratch = (uint32_t *)(tab + CH_TAB);
  int *ends = (int *)((uint8_t *)scratch + ATTN_SCAN_LDS), *poison = (int *)scratch + 15, *redo = (int *)scratch + 14;

  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lq = lane & 31, lh = lane >> 5;
  if (s.first) attn_zero_rest(a);
  AttnWork w = attn_share<CH_TR, CH_KT, 1>(a, s, ends, scratch);
  if (blockIdx.x == 0 && tid == 0) s.count[0] = w.tiles;
  const int g = a.Hq / a.Hkv;
  const uint32_t la = lds_addr(lds), ta = lds_addr(tab) + wv * 512;
  if constexpr (!FULL) {  // head values past D: never written by the DMA
    for (int i = tid; i < 4 * TILE / 16; i += ATTN_THREADS) ((uint4 *)lds)[i] = make_uint4(0, 0, 0, 0);
  }

  while (w.left > 0) {
    const int r = attn_find(ends, a.R, w.tile);
    const AttnReq rq = attn_req(a, r, g);
    const AttnTile t = attn_tile(a, rq, w.tile - (r ? ends[r - 1] : 0), CH_TR, g);
    const int cost = attn_units<CH_KT>(t) + 1;
    const int take = cost - w.u < w.left ? cost - w.u : w.left;
    const int u0 = w.u > 0 ? w.u - 1 : 0, u1 = w.u + take - 1;  // (the first unit: the tile's own overhead)
    const int ks = (t.b / CH_KT + u0) * CH_KT, nt = u1 - u0;

    __syncthreads();
    if (tid == 0) *poison = 0, *redo = 0;
    const int *tabrow = a.table + (int64_t)r * a.W;
    auto page_at = [&](int k0) -> const int * {
      int key = k0 + wv * 16 + (lane & 15);
      key = key < t.e ? key : t.e - 1;
      return tabrow + (uint32_t)key / (uint32_t)a.block;
    };
    const int page0 = nt > 0 ? *page_at(ks) : 0;

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
      const uint16_t *qp = a.q + (((int64_t)(rq.q0 + tok) * a.Hq) + w.head * g + hh) * a.D;
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
    float m[2] = {-__builtin_inff(), -__builtin_inff()}, l[2];
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
    if (nt > 0) {
      f32x16_t sv[2];
      bf16x8_t p[2][2];  // [16 keys][half]
      uint32_t mine = 0;  // the row (of the whole cache) of this lane's key
      auto rows_of = [&](int k0, int blk, int set) __attribute__((always_inline)) {
        const int key = k0 + wv * 16 + (lane & 15);
        const bool ok = key < t.e && (uint32_t)blk < (uint32_t)a.NB;
        mine = ok ? ((uint32_t)blk * a.Hkv + w.head) * a.block + (uint32_t)key % (uint32_t)a.block : 0u;
        const uint32_t mask = (uint32_t)__ballot(ok) & 0xFFFFu;
        if (lane == 0) vm[set * 4 + wv] = mask;
      };
      auto move_k = [&](int set) __attribute__((always_inline)) {
        const int here = attn_opaque(lane);
#pragma unroll
        for (int i = 0; i < OPS; ++i) {
          const int row = (i * 64 + here) / CPR, c = (i * 64 + here) % CPR ^ attn_swz<DP>(row);
          const uint32_t from = __shfl(mine, row, 64);  // (by all lanes)
          if (FULL || c * 8 < a.D)
            gp_dma16(a.k + (uint64_t)from * (uint32_t)a.D + c * 8, la + set * TILE + wv * 16 * PITCH + i * 1024);
          __builtin_amdgcn_sched_barrier(0);  // (few registers at a time)
        }
      };
      auto move_v = [&](int set) __attribute__((always_inline)) {
        const int here = attn_opaque(lane);
#pragma unroll
        for (int i = 0; i < OPS; ++i) {
          const int row = (i * 64 + here) / CPR, c = (i * 64 + here) % CPR ^ ch_swz_v<DP>(row);
          const uint32_t from = __shfl(mine, row, 64);
          if (FULL || c * 8 < a.D)
            gp_dma16(a.v + (uint64_t)from * (uint32_t)a.D + c * 8, la + (2 + set) * TILE + wv * 16 * PITCH + i * 1024);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      // S^T of 32 keys
      auto scores = [&](int set, int half) __attribute__((always_inline)) {
        // (k steps 8 apart differ by 256 bytes, which the swizzle leaves alone)
        const int from = attn_opaque(set * TILE + half * 32 * PITCH + lq * PITCH + (lh ^ attn_swz<DP>(lq)) * 16);
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
          __builtin_amdgcn_sched_barrier(0);
        }
        ch_mfma_done(sv[0], sv[1]);
      };
      // masks, the references
      auto maxima = [&](int k0, uint64_t valid, bool edge) __attribute__((always_inline)) {
        if (edge) {
          const int h4 = attn_opaque(4 * lh);
          const uint32_t bits = (uint32_t)valid >> h4;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int lo = seen_b[u] - k0 - h4, hi = seen_e[u] - k0 - h4;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int o = 8 * (i / 4) + i % 4;
              if (!(o <= hi && o >= lo && (bits >> o & 1))) sv[u][i] = -__builtin_inff();
            }
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float top = sv[u][0];
#pragma unroll
          for (int i = 1; i < 16; ++i) top = fmaxf(top, sv[u][i]);
          top = fmaxf(top, __shfl_xor(top, 32, 64)) * sc;
          passed |= top > m[u] + 60.f && m[u] != -__builtin_inff();
          // (before its first key a row has no sums)
          m[u] = m[u] == -__builtin_inff() || top > m[u] + 60.f ? top : m[u];
        }
      };
      // Step n of N: its part of the weights of sv into np, their sums into ls
      bf16x8_t np[2][2];
      float ls[2], ref[2];
      auto weights = [&](int n, int N) __attribute__((always_inline)) {
        if (n == 0) {
#pragma unroll
          for (int u = 0; u < 2; ++u) ls[u] = 0.f, ref[u] = m[u] == -__builtin_inff() ? 0.f : m[u];
        }
#pragma unroll
        for (int j = n * (16 / N); j < (n + 1) * (16 / N); ++j) {
          const int u = j >> 3, c = j >> 2 & 1, e = (j & 3) * 2;
          bf16x2_t x;
          x[0] = (__bf16)attn_exp2(__builtin_fmaf(sv[u][c * 8 + e], sc, -ref[u]));
          x[1] = (__bf16)attn_exp2(__builtin_fmaf(sv[u][c * 8 + e + 1], sc, -ref[u]));
          ls[u] = dot2_bf16(x, 0x3F803F80u, ls[u]);
          np[c][u][e] = x[0], np[c][u][e + 1] = x[1];
        }
      };
      // O^T += V^T P^T over 32 keys, and with it the next weights
      auto product = [&](int set, int half, bool with) __attribute__((always_inline)) {
        const int row = 4 * lh + (lane >> 2 & 3);
        const int from = attn_opaque(la + (2 + set) * TILE + (half * 32 + row) * PITCH +
                                     (((lane >> 4 & 1) * 2 + (lane >> 1 & 1)) ^ ch_swz_v<DP>(row)) * 16 + (lane & 1) * 8);
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
          if (with) weights(n, N);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      auto edge_at = [&](int k0, uint64_t valid) -> bool {
        return k0 < t.full_b || k0 + CH_KT > t.full_e || valid != ~0ull;
      };
      auto valid_of = [&](int set) -> uint64_t {
        const uint32_t *v = vm + set * 4;
        const uint32_t lo = __builtin_amdgcn_readfirstlane(v[0] | v[1] << 16);
        const uint32_t hi = __builtin_amdgcn_readfirstlane(v[2] | v[3] << 16);
        return (uint64_t)hi << 32 | lo;
      };

      rows_of(ks, page0, 0);
      ch_dma4(page_at(ks + CH_KT), ta + 256);
      move_k(0);
      move_v(0);
      gp_wait_barrier<OPS>();  // keys of tile 0; everyone's valid bits
      uint64_t valid = valid_of(0);
      bool edge = edge_at(ks, valid);
      // the page ids of tile i + 1 are there: its keys, and the ids of tile i + 2
      auto next_keys = [&](int i) __attribute__((always_inline)) {
        const int set = (i + 1) & 1, blk = *(const int *)(tab + wv * 512 + set * 256 + lane * 4);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        rows_of(ks + (i + 1) * CH_KT, blk, set);
        ch_dma4(page_at(ks + (i + 2) * CH_KT), ta + (i & 1) * 256);
        move_k(set);
      };
      if (nt > 1) next_keys(0);
      // Step h: half h % 2 of tile h / 2.  Its scores; then its weights together with the product
      // of step h - 1.
      scores(0, 0);
      maxima(ks, valid, edge);
      weights(0, 1);
      const int steps = 2 * nt;
      for (int h = 1;; ++h) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          l[u] += ls[u];
#pragma unroll
          for (int c = 0; c < 2; ++c) p[c][u] = np[c][u];
        }
        if (h == steps) break;
        const int i = h >> 1, set = i & 1, half = h & 1;
        const bool more = i + 1 < nt;
        if (half == 0) {
          gp_wait_barrier<OPS>();  // keys of tile i (its values are still on their way)
          valid = valid_of(set);
          edge = edge_at(ks + i * CH_KT, valid);
          if (more) next_keys(i);
        }
        scores(set, half);
        maxima(ks + i * CH_KT + half * 32, valid >> half * 32, edge);
        if (half == 1) {
          // values of tile i
          if (more)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(OPS + 1) : "memory");
          else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
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
          if (more) move_v(set ^ 1);
        }
        product(((h - 1) >> 1) & 1, (h - 1) & 1, true);
      }
      product((nt - 1) & 1, 1, false);
    }
    if (__any(passed)) *redo = 1;
    __syncthreads();
    again = !again && *redo;
    __syncthreads();
    } while (again);

    const bool whole = take == cost;
    const int part = w.g * 2 + (w.u == 0 ? 1 : 0);
    if (w.u == 0 && tid == 0) {
      const int64_t last = w.at + cost - 1;
      const int g1 = (int)(((last + 1) * w.groups + w.total - 1) / w.total) - 1;
      int *d = s.desc + ((int64_t)w.head * w.tiles + w.tile) * 8;
      d[0] = whole ? -1 : w.g, d[1] = g1, d[2] = rq.q0, d[3] = t.row0, d[4] = t.rows;
    }
    // rows out, 32 of a wave and half of their columns at a time, through the wave's quarter of the LDS
    constexpr int HC = DP / 2, OP = HC + 4;
    float *out = (float *)(lds + wv * TILE);
    const bool bad = *poison != 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (wv * 64 + u * 32 >= t.rows) break;
      l[u] += __shfl_xor(l[u], 32, 64);
      const float scale = !whole ? 1.f : l[u] != 0.f ? 1.f / l[u] : 0.f;
      if (!whole && lane < 32 && wv * 64 + u * 32 + lq < t.rows) {
        const int64_t pr = (int64_t)part * CH_TR + wv * 64 + u * 32 + lq;
        s.ml[pr * 2] = m[u], s.ml[pr * 2 + 1] = l[u];
      }
#pragma unroll
      for (int hc = 0; hc < 2; ++hc) {
#pragma unroll
        for (int d = 0; d < DT / 2; ++d)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const f32x16_t &x = acc[hc * (DT / 2) + d][u];
            *(float4 *)(out + lq * OP + d * 32 + v * 8 + lh * 4) =
                make_float4(x[4 * v] * scale, x[4 * v + 1] * scale, x[4 * v + 2] * scale, x[4 * v + 3] * scale);
          }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int j = lane; j < 32 * (HC / 8); j += 64) {
          const int rr = j / (HC / 8), c0 = j % (HC / 8) * 8, d0 = hc * HC + c0, in = wv * 64 + u * 32 + rr;
          if (in >= t.rows || d0 >= a.D) continue;
          float o[8];
          *(float4 *)&o[0] = *(const float4 *)(out + rr * OP + c0);
          *(float4 *)&o[4] = *(const float4 *)(out + rr * OP + c0 + 4);
          if (bad) attn_poison(a, rq, tabrow, w.head, t.row0 + in, g, ks, ks + nt * CH_KT < t.e ? ks + nt * CH_KT : t.e, d0, o);
          if (whole) {
            attn_store8(a, rq.q0, t.row0 + in, w.head, g, d0, o);
          } else {
            float4 *to = (float4 *)(s.acc + ((int64_t)part * CH_TR + in) * DP + d0);
            to[0] = make_float4(o[0], o[1], o[2], o[3]), to[1] = make_float4(o[4], o[5], o[6], o[7]);
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

    w.left -= take;
    w.at += take;
    w.u += take;
    if (w.u == cost) {
      w.u = 0;
      if (++w.tile == w.tiles) w.tile = 0, ++w.head;
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

size_t attn_chunk_lds(int DP, int R) { return 4 * ch_tile(DP) + CH_TAB + ATTN_SCAN_LDS + (size_t)R * 4; }

hipError_t launch_attn_chunk(const AttnArgs &a, const AttnShare &s, int DP, int grid, hipStream_t st) {
  return DP == 64 ? launch_dp<64>(a, s, grid, st) : DP == 128 ? launch_dp<128>(a, s, grid, st) : launch_dp<256>(a, s, grid, st);
}

}  // namespace qmm
