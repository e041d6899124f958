// Paged attention of few rows per key head (decode, drafts being verified): the keys and values
// of a context are read once and every other thing is small beside that, so the kernel is built
// to keep HBM busy.
//
// A tile is 16 or 32 rows (NQ = 1, 2).  Each of a workgroup's four waves runs its own keys, with
// its own running maximum and sum, and never waits for another until the tile's end: it moves
// tiles of KW keys (8 KB of keys, 8 KB of values) from HBM to its own part of the LDS by DMA, the
// next keys in flight while the values are used and the other way round, two workgroups a CU:
// 128 KB in flight per CU.
//
// S^T = K Q^T and O^T = V^T P^T on the 16x16 MFMA.  In S^T a lane holds one row (lane % 16) and
// keys 4 (lane / 16) .. + 3: the shape that P^T needs as the second operand when the keys of a
// product are taken in that order, so the weights never leave their registers; V^T comes through
// the transposing LDS read in the same order of keys.  The weights are rounded to bf16 for that
// product (2^-9 of each, which averages out over keys; the sum they are divided by is that of the
// rounded ones, so that a row of one heavy key is exact).
#include "attention.h"
#include "gemm_pipe.h"

namespace qmm {

namespace {

constexpr int AR_WAVES = 4;
constexpr int AR_TILE = 8192;  // bytes of a wave's tile of keys (and of values)
constexpr int AR_STAGE = AR_WAVES * 2 * AR_TILE;
constexpr int AR_TAB = AR_WAVES * 2 * 256;  // the next tile's page ids, two sets per wave

constexpr int ar_merge(int DP) { return AR_WAVES * 16 * (DP + 4) * 4 + AR_WAVES * 16 * 8; }
constexpr int ar_fixed(int DP) { return AR_STAGE > ar_merge(DP) ? AR_STAGE : ar_merge(DP); }

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// LDS DMA of 4 bytes per lane (see gp_dma16).
__device__ __forceinline__ void ar_dma4(const void *g, uint32_t l) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(l), "v"(g) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void ar_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// FULL: D = DP (else the lanes of chunks past D stay out of the DMA).
template <int DP, int NQ, bool FULL>
__global__ __launch_bounds__(ATTN_THREADS, 2) void attn_rows_kernel(const AttnArgs a, const AttnShare s) {
  constexpr int TR = 16 * NQ;
  constexpr int KW = AR_TILE / (2 * DP);  // keys of a wave's tile: 16, 32, 64
  constexpr int KT = AR_WAVES * KW;
  constexpr int CPR = DP / 8;             // 16-byte chunks of a row
  constexpr int KB = KW / 16;             // 16-key blocks of a tile
  constexpr int ST = DP / 32, DT = DP / 16;
  constexpr int OPS = AR_TILE / 1024;     // DMA operations of a tile
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  uint8_t *tab = lds + ar_fixed(DP);
  uint32_t *scratch = (uint32_t *)(tab + AR_TAB);
  int *ends = (int *)((uint8_t *)scratch + ATTN_SCAN_LDS), *poison = (int *)scratch + 15;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lg = lane >> 4;
  if (s.first) attn_zero_rest(a);
  AttnWork w = attn_uniform(attn_share<TR, KT, 1>(a, s, ends, scratch));
  attn_note_none(s, w);
  const int g = a.Hq / a.Hkv;
  const int wv = __builtin_amdgcn_readfirstlane(wave);
  uint8_t *kl = lds + wv * 2 * AR_TILE, *vl = kl + AR_TILE;
  const uint32_t ka = lds_addr(kl), va = lds_addr(vl), ta = lds_addr(tab) + wv * 512;
  // head values past D: never written by the DMA, zero for good
  if constexpr (!FULL) {
    for (int i = tid; i < AR_STAGE / 16; i += ATTN_THREADS) ((uint4 *)lds)[i] = make_uint4(0, 0, 0, 0);
  }

  while (w.left > 0) {
    const int r = attn_uniform(attn_find(ends, a.R, w.tile));
    const AttnReq rq = attn_uniform(attn_req(a, r, g));
    const AttnTile t = attn_tile(a, rq, w.tile - (r ? attn_uniform(ends[r - 1]) : 0), TR, g);
    const int cost = attn_units<KT>(t) + 1;
    const int take = cost - w.u < w.left ? cost - w.u : w.left;
    // (a tile's first unit stands for its own overhead)
    const int u0 = w.u > 0 ? w.u - 1 : 0, u1 = w.u + take - 1;
    const int ks = (t.b / KT + u0) * KT;
    int ke = (t.b / KT + u1) * KT;
    ke = ke < t.e ? ke : t.e;

    __syncthreads();  // (the last tile's merge is read; the zeros above are written)
    if (tid == 0) *poison = 0;
    __syncthreads();
    // this wave's tiles: keys k0 = ks + KW (wave + 4 i)
    const int *tabrow = a.table + (int64_t)r * a.W;
    auto page_at = [&](int k0) -> const int * {  // of this lane's key (held below e: a page of the row)
      int key = k0 + (lane & (KW - 1));
      key = key < t.e ? key : t.e - 1;
      return tabrow + (uint32_t)key / (uint32_t)a.block;
    };
    // the rows of this lane: what they see, their queries
    int seen_b[NQ], seen_e[NQ];
    bf16x8_t q[NQ][ST];
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;  // (a negative scale: -q, so that maxima stay maxima)
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int row = t.row0 + n * 16 + lr;
      const bool on = n * 16 + lr < t.rows;
      const int tok = on ? row / g : 0, hh = on ? row - tok * g : 0;
      const int pos = rq.base + tok;
      seen_e[n] = on ? pos : -1;
      seen_b[n] = a.window ? pos - a.window + 1 : 0;
      const uint16_t *qp = a.q + (((int64_t)(rq.q0 + tok) * a.Hq) + w.head * g + hh) * a.D;
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int d0 = st * 32 + lg * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (on && d0 < a.D && a.scale != 0.f) v = *(const uint4 *)(qp + d0);
        v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
        q[n][st] = __builtin_bit_cast(bf16x8_t, v);
      }
    }
    int k0 = ks + KW * wv;
    const int page0 = k0 < ke ? *page_at(k0) : 0;
    // all of the loads above, now: the compiler's own waits for them would come between the DMA's
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    const float sc = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.44269504088896341f;

    f32x4_t acc[NQ][DT];
    float m[NQ], l[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      m[n] = -__builtin_inff(), l[n] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[n][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    // the row number (of the whole cache) of this lane's key, or row 0 where there is none
    auto row_of = [&](int k0, int blk, bool *ok) -> uint32_t {
      const int key = k0 + (lane & (KW - 1));
      *ok = key < t.e && (uint32_t)blk < (uint32_t)a.NB;
      const uint32_t off = (uint32_t)key % (uint32_t)a.block;
      return *ok ? ((uint32_t)blk * a.Hkv + w.head) * a.block + off : 0u;
    };
    uint32_t rows[OPS];  // of the tile in the keys' buffer, per DMA operation
    auto spread = [&](uint32_t mine) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < OPS; ++i) rows[i] = __shfl(mine, (i * 64 + lane) / CPR, 64);
    };
    auto move = [&](const uint16_t *cache, uint32_t to) __attribute__((always_inline)) {
      const int here = attn_opaque(lane);
#pragma unroll
      for (int i = 0; i < OPS; ++i) {
        const int row = (i * 64 + here) / CPR, c = (i * 64 + here) % CPR ^ attn_swz<DP>(row);
        if (FULL || c * 8 < a.D) gp_dma16(cache + (uint64_t)rows[i] * (uint32_t)a.D + c * 8, to + i * 1024);
      }
    };

    if (k0 < ke) {
      bool ok;
      uint32_t mine = row_of(k0, page0, &ok);
      uint64_t valid = __ballot(ok);
      spread(mine);
      if (k0 + KT < ke) ar_dma4(page_at(k0 + KT), ta + 256);
      move(a.k, ka);
      move(a.v, va);
      int buf = 1;
      while (true) {
        const bool more = k0 + KT < ke;
        ar_wait<OPS>();  // the keys are here (and the next page ids, which were asked for before them)
        const bool edge = k0 < t.full_b || k0 + KW > t.full_e || valid != ~0ull;
        const uint64_t now = valid;
        // S^T
        f32x4_t sv[NQ][KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
#pragma unroll
          for (int n = 0; n < NQ; ++n) sv[n][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
          const int row = b * 16 + lr, from = attn_opaque(row * (2 * DP) + (lg ^ attn_swz<DP>(row)) * 16);
#pragma unroll
          for (int st = 0; st < ST; ++st) {
            const bf16x8_t kf = *(const bf16x8_t *)(kl + (from ^ st * 64));
#pragma unroll
            for (int n = 0; n < NQ; ++n) sv[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[n][st], sv[n][b], 0, 0, 0);
          }
        }
        if (more) {  // the next keys into the buffer just read
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          int blk = *(const int *)(tab + wv * 512 + buf * 256 + lane * 4);
          mine = row_of(k0 + KT, blk, &ok);
          valid = __ballot(ok);
        }
        if (more) {
          buf ^= 1;
          if (k0 + 2 * KT < ke)
            ar_dma4(page_at(k0 + 2 * KT), ta + buf * 256);
          else
            ar_dma4(page_at(k0), ta + buf * 256);  // (not read; the waits count on it)
          spread(mine);
          move(a.k, ka);
        }
        // the softmax's weights
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          if (edge) {
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int o = b * 16 + lg * 4 + i, key = k0 + o;
                if (!(key <= seen_e[n] && key >= seen_b[n] && (now >> o & 1))) sv[n][b][i] = -__builtin_inff();
              }
          }
          float top = sv[n][0][0];
#pragma unroll
          for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, sv[n][b][i]);
          top = fmaxf(top, __shfl_xor(top, 16, 64));
          top = fmaxf(top, __shfl_xor(top, 32, 64)) * sc;
          // the reference maximum follows only when it is passed by 2^8: the weights stay in range
          if (__any(top > m[n] + 8.f)) {
            const float mn = fmaxf(m[n], top);
            const float f = mn == -__builtin_inff() ? 1.f : attn_exp2(m[n] - mn);
            m[n] = mn;
            l[n] *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[n][d] *= f;
          }
        }
        i16x4_t p[NQ][KB];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const float ref = m[n] == -__builtin_inff() ? 0.f : m[n];
#pragma unroll
          for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const __bf16 e = (__bf16)attn_exp2(__builtin_fmaf(sv[n][b][i], sc, -ref));
              l[n] += (float)e;
              p[n][b][i] = __builtin_bit_cast(short, e);
            }
        }
        // the values
        if (more)
          ar_wait<OPS + 1>();
        else
          ar_wait<0>();
        if (edge) {
          // keys that are none: zeros, whatever was loaded; values that are not finite, which must not reach
          // the rows that do not see their keys (0 inf is NaN): zeros for now
          bool odd = false;
#pragma unroll
          for (int i = 0; i < OPS; ++i) {
            uint4 *at = (uint4 *)(vl + i * 1024 + lane * 16);
            uint4 x = *at;
            const bool in = now >> ((i * 64 + lane) / CPR) & 1;
            const uint4 y = attn_finite(x);
            odd |= in && (x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w);
            *at = in ? y : make_uint4(0, 0, 0, 0);
          }
          if (__any(odd)) *poison = 1;
        }
        // (this lane's place in the 16 x 16 block (b, 0) of the values)
        int from[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          const int row = b * 16 + lg * 4 + (lr >> 2);
          from[b] = attn_opaque(row * (2 * DP) + ((lane >> 1 & 1) ^ attn_swz<DP>(row)) * 16 + (lane & 1) * 8);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          auto col = [&](int b) __attribute__((always_inline)) { return attn_read_tr(va + (from[b] ^ d * 32)); };
          if constexpr (KB == 1) {
            const i16x4_t vf = col(0);
#pragma unroll
            for (int n = 0; n < NQ; ++n)
              acc[n][d] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(vf, p[n][0], acc[n][d], 0, 0, 0);
          } else {
#pragma unroll
            for (int b = 0; b < KB; b += 2) {
              const i16x8_t vf = __builtin_shufflevector(col(b), col(b + 1), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
              for (int n = 0; n < NQ; ++n) {
                const i16x8_t pf = __builtin_shufflevector(p[n][b], p[n][b + 1], 0, 1, 2, 3, 4, 5, 6, 7);
                acc[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vf),
                                                                    __builtin_bit_cast(bf16x8_t, pf), acc[n][d], 0, 0, 0);
              }
            }
          }
        }
        if (!more) break;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        move(a.v, va);
        k0 += KT;
      }
    }

    // the four waves' parts, 16 rows at a time through the stage's LDS
    const bool whole = take == cost;
    const int part = w.g * 2 + (w.u == 0 ? 1 : 0);
    if (w.u == 0 && tid == 0) attn_note(s, w, rq, t, cost, whole);
    float *macc = (float *)lds;                                  // [wave][16][DP + 4]
    float *mml = (float *)(lds + AR_WAVES * 16 * (DP + 4) * 4);  // [wave][16][2]
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      if (n * 16 >= t.rows) break;
      __syncthreads();
      l[n] += __shfl_xor(l[n], 16, 64);
      l[n] += __shfl_xor(l[n], 32, 64);
      if (lg == 0) mml[(wave * 16 + lr) * 2] = m[n], mml[(wave * 16 + lr) * 2 + 1] = l[n];
#pragma unroll
      for (int d = 0; d < DT; ++d) *(f32x4_t *)(macc + (wave * 16 + lr) * (DP + 4) + d * 16 + lg * 4) = acc[n][d];
      __syncthreads();
      for (int i = tid; i < 16 * CPR; i += ATTN_THREADS) {
        const int row = i / CPR, d0 = i % CPR * 8;
        if (n * 16 + row >= t.rows || d0 >= a.D) continue;
        float top = -__builtin_inff(), f[AR_WAVES], sum = 0.f, o[8];
#pragma unroll
        for (int v = 0; v < AR_WAVES; ++v) top = fmaxf(top, mml[(v * 16 + row) * 2]);
#pragma unroll
        for (int v = 0; v < AR_WAVES; ++v) {
          const float mv = mml[(v * 16 + row) * 2];
          f[v] = mv == -__builtin_inff() ? 0.f : attn_exp2(mv - top);
          sum += f[v] * mml[(v * 16 + row) * 2 + 1];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = 0.f;
#pragma unroll
        for (int v = 0; v < AR_WAVES; ++v) {
          const float4 x = *(const float4 *)(macc + (v * 16 + row) * (DP + 4) + d0);
          const float4 y = *(const float4 *)(macc + (v * 16 + row) * (DP + 4) + d0 + 4);
          o[0] += f[v] * x.x, o[1] += f[v] * x.y, o[2] += f[v] * x.z, o[3] += f[v] * x.w;
          o[4] += f[v] * y.x, o[5] += f[v] * y.y, o[6] += f[v] * y.z, o[7] += f[v] * y.w;
        }
        if (*poison) attn_poison(a, rq, tabrow, w.head, t.row0 + n * 16 + row, g, ks, ke, d0, o);
        if (whole) {
          const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] *= inv;
          attn_store8(a, attn_row(a, rq.q0, t.row0 + n * 16 + row, w.head, g), d0, o);
        } else {
          const int64_t pr = (int64_t)part * TR + n * 16 + row;
          float4 *to = (float4 *)(s.acc + pr * DP + d0);
          to[0] = make_float4(o[0], o[1], o[2], o[3]), to[1] = make_float4(o[4], o[5], o[6], o[7]);
          if (d0 == 0) s.ml[pr * 2] = top, s.ml[pr * 2 + 1] = sum;
        }
      }
    }
    if constexpr (!FULL) {  // the merge has overwritten the zeros past D
      __syncthreads();
      for (int i = tid; i < AR_STAGE / 16; i += ATTN_THREADS) ((uint4 *)lds)[i] = make_uint4(0, 0, 0, 0);
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

template <int DP, int NQ, bool FULL>
hipError_t launch_t(const AttnArgs &a, const AttnShare &s, int grid, hipStream_t st) {
  static std::atomic<uint64_t> done{0};
  const void *k = (const void *)attn_rows_kernel<DP, NQ, FULL>;
  const hipError_t e = ensure_dynamic_lds(done, k, (int)attn_rows_lds(DP, ATTN_MAX_R));
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((attn_rows_kernel<DP, NQ, FULL>), dim3(grid), dim3(ATTN_THREADS), attn_rows_lds(DP, a.R), st, a, s);
  return hipGetLastError();
}

template <int DP>
hipError_t launch_dp(const AttnArgs &a, const AttnShare &s, int tr, int grid, hipStream_t st) {
  if (a.D == DP) return tr == 16 ? launch_t<DP, 1, true>(a, s, grid, st) : launch_t<DP, 2, true>(a, s, grid, st);
  return tr == 16 ? launch_t<DP, 1, false>(a, s, grid, st) : launch_t<DP, 2, false>(a, s, grid, st);
}

}  // namespace

size_t attn_rows_lds(int DP, int R) { return ar_fixed(DP) + AR_TAB + ATTN_SCAN_LDS + (size_t)R * 4; }

hipError_t launch_attn_rows(const AttnArgs &a, const AttnShare &s, int DP, int tr, int grid, hipStream_t st) {
  return DP == 64 ? launch_dp<64>(a, s, tr, grid, st)
                  : DP == 128 ? launch_dp<128>(a, s, tr, grid, st) : launch_dp<256>(a, s, tr, grid, st);
}

}  // namespace qmm
