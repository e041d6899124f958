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
// the transposing LDS read in the same order of keys.  A weight goes into that product as two bf16
// parts, its rounding and what that has taken (2^-17 of it is lost): HBM leaves the matrix cores the time.
//
// One token over 262144 keys (24 query heads on 4 of 256; 1.07 GB, each byte fetched once): 189-191 us, 5.65
// TB/s, the matrix cores 6% busy.  64 requests of 1 to 8192 keys (32 on 8 of 128; 370 MB): 77-79 us.
#include "attention.h"
#include "gemm_pipe.h"

namespace qmm {

namespace {

constexpr int AR_WAVES = 4;
constexpr int AR_EXTRA = 1;  // a tile's own overhead, in units of its keys
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
__global__ __launch_bounds__(ATTN_THREADS, 2) void attn_rows_kernel(const AttnArgs args, const AttnShare share) {
  constexpr int TR = 16 * NQ;
  constexpr int KW = AR_TILE / (2 * DP);  // keys of a wave's tile: 16, 32, 64
  constexpr int KT = AR_WAVES * KW;
  constexpr int CPR = DP / 8;             // 16-byte chunks of a row
  constexpr int RPI = 64 / CPR;           // rows of a DMA operation
  constexpr int KB = KW / 16;             // 16-key blocks of a tile
  constexpr int ST = DP / 32, DT = DP / 16, PITCH = 2 * DP;
  constexpr int OPS = AR_TILE / 1024;     // DMA operations of a tile
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  uint8_t *tab = lds + ar_fixed(DP);
  int *seen_at = (int *)(tab + AR_TAB);  // [thread][2][2]: what its rows see
  AttnPlan *plan = (AttnPlan *)(seen_at + 4 * ATTN_THREADS);

  const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  auto here = [&]() __attribute__((always_inline)) { return wv * 64 + (int)attn_lane(); };  // the thread's number
  int left;
  {
    const AttnWork w = attn_uniform(attn_share<TR, KT, AR_EXTRA>(args, share, plan));
    if (share.first) attn_zero_rest(args);
    attn_note_none(share, w);
    if (tid == 0) plan->work[0] = w, plan->poison[0] = 0;
    left = w.left;
  }
  uint8_t *kl = lds + wv * 2 * AR_TILE, *vl = kl + AR_TILE;
  const uint32_t ka = lds_addr(kl), va = lds_addr(vl), ta = lds_addr(tab) + wv * 512;
  // head values past D: never written by the DMA, zero for good
  if constexpr (!FULL) {
    for (int i = tid; i < AR_STAGE / 16; i += ATTN_THREADS) ((uint4 *)lds)[i] = attn_zeros();
  }

  int turn = 0;
#pragma unroll 1
  while (left > 0) {
    __syncthreads();  // (the last tile's merge is read; the zeros above are written)
    const AttnArgs a = attn_again<AttnArgs>(0);
    const AttnWork w = attn_uniform(plan->work[turn]);
    int *poison = &plan->poison[turn];
    const int r = attn_uniform(attn_request(plan, a.R, w));
    const AttnReq rq = attn_uniform(attn_req(plan, a, r));
    const AttnTile t = attn_uniform(attn_tile(a, rq, w.tile - (r ? attn_end(plan, a.R, r - 1) : 0), TR));
    const int units = attn_units<KT>(t);
    const AttnPiece pc = attn_piece<AR_EXTRA>(w, units);
    const bool whole = pc.whole;
    const int ks = (int)(((uint32_t)t.b / KT + pc.u0) * KT), part = w.g * 2 + pc.start, head = w.head;
    int ke = (int)(((uint32_t)t.b / KT + pc.u1) * KT);
    ke = ke < t.e ? ke : t.e;
    if (pc.start && !pc.none && here() == 0)
      attn_note(attn_again<AttnShare>(sizeof(AttnArgs)), w, rq, t, units + AR_EXTRA, whole);
    {
      AttnWork on = w;
      on.r = r;
      attn_move_on(on, pc.take, units + AR_EXTRA);
      left = on.left;
      turn ^= 1;
      if (here() == 0) plan->work[turn] = on, plan->poison[turn] = 0;
    }
    if (pc.none) continue;

    // This wave's tiles are the keys k0 = ks + KW (wave + 4 i), this lane's key of them the (lane % KW)th: `page`
    // and `off` of the tile whose page ids are asked for next (held to the last page), `at` its place in its page.
    const int block = a.block, NB = a.NB, Hkv = a.Hkv, D = FULL ? DP : a.D;
    const uint16_t *kc = a.k, *vc = a.v;
    const int *tabrow = a.table + (int64_t)r * a.W;
    int k0 = ks + KW * wv;
    const uint32_t last_page = t.e > 0 ? attn_div(t.e - 1, a.by_block) : 0u;
    const uint32_t first = k0 + (attn_lane() & (KW - 1));
    uint32_t page = attn_div(first, a.by_block), off = first - page * block;
    const int page0 = k0 < ke ? tabrow[page < last_page ? page : last_page] : 0;

    // the rows of this lane: what they see, their queries
    float m[NQ], l[NQ];
    const int ln0 = (int)attn_lane(), lr = ln0 & 15, lg = ln0 >> 4;
    bf16x8_t q[NQ][ST];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const bool on = n * 16 + lr < t.rows;
      const int row = t.row0 + (on ? n * 16 + lr : 0);  // (a row past the end: the first one's queries)
      const int pos = rq.base + (int)attn_div(row, a.by_g);
      seen_at[here() * 4 + 2 * n] = a.window && pos >= a.window ? pos - a.window + 1 : 0;
      seen_at[here() * 4 + 2 * n + 1] = on ? pos : -1;
      // (a row that sees nothing needs no reference; one past the end has no weights and passes none)
      m[n] = !on ? __builtin_inff() : pos >= 0 ? -__builtin_inff() : 0.f;
      const uint16_t *qp = a.q + attn_row(a, rq.q0, row, head) * a.D + lg * 8;
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        if (FULL || st * 32 + lg * 8 < a.D)
          q[n][st] = *(const bf16x8_t *)(qp + st * 32);
        else
          q[n][st] = __builtin_bit_cast(bf16x8_t, u32x4_t{0u, 0u, 0u, 0u});
      }
    }
    if (!(a.scale > 0.f)) {  // a negative scale: -q, so that maxima stay maxima; none: no scores
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          u32x4_t x = __builtin_bit_cast(u32x4_t, q[n][st]);
          x = a.scale < 0.f ? x ^ 0x80008000u : u32x4_t{0u, 0u, 0u, 0u};
          q[n][st] = __builtin_bit_cast(bf16x8_t, x);
        }
    }
    // all of the loads above, now: the compiler's own waits for them would come between the DMA's
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    const float sc = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.44269504088896341f;

    f32x4_t acc[NQ][DT];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      l[n] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[n][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    if (k0 < ke) {
      const uint32_t per = attn_div(KT, a.by_block), rest = KT - per * block;
      uint32_t at = off;
      auto onward = [&]() __attribute__((always_inline)) {
        page += per, off += rest;
        const uint32_t over = off >= (uint32_t)block;
        off -= over ? block : 0, page += over;
      };
      auto ask = [&](int buf) __attribute__((always_inline)) {
        ar_dma4(tabrow + (page < last_page ? page : last_page), ta + buf * 256);
      };
      // the row (of the whole cache) of this lane's key, 0 where there is none; a bit for each key that there is
      uint32_t mine;
      uint64_t valid;
      auto rows_of = [&](int k, int blk) __attribute__((always_inline)) {
        const bool ok = k + ((int)attn_lane() & (KW - 1)) < t.e && (uint32_t)blk < (uint32_t)NB;
        mine = (((uint32_t)blk * Hkv + head) * block + at) & (ok ? ~0u : 0u);
        valid = __ballot(ok);
      };
      // DMA operations: RPI rows each, chunk (lane % CPR) ^ swizzle
      auto move = [&](const uint16_t *cache, uint32_t to) __attribute__((always_inline)) {
        const uint32_t ln = attn_lane(), c0 = ln % CPR ^ (uint32_t)attn_swz<DP>((int)(ln / CPR));
#pragma unroll
        for (int i = 0; i < OPS; ++i) {
          const uint32_t row = __builtin_amdgcn_ds_bpermute((int)(ln / CPR * 4) + RPI * i * 4, (int)mine);
          const uint32_t c = (c0 ^ (uint32_t)attn_swz<DP>(RPI * i)) * 16;
          if (FULL || c < 2 * (uint32_t)D)
            gp_dma16((const char *)cache + ((uint64_t)row * (2 * (uint32_t)D) + c), to + i * 1024);
          if (i % 2) __builtin_amdgcn_sched_barrier(0);  // (few registers at a time)
        }
      };

      rows_of(k0, page0);
      onward();
      at = off;
      ask(1);
      onward();
      move(kc, ka);
      move(vc, va);
      int buf = 1;
#pragma unroll 1
      while (true) {
        const bool more = k0 + KT < ke;
        ar_wait<OPS>();  // the keys are here (and the next page ids, which were asked for before them)
        const uint64_t now = valid;
        const bool edge = k0 < t.full_b || k0 + KW > t.full_e || now != ~0ull;
        // S^T
        f32x4_t sv[NQ][KB];
        {
          const uint32_t ln = attn_lane();
          const int row = ln & 15, from = row * PITCH + ((int)(ln >> 4) ^ attn_swz<DP>(row)) * 16;
          auto load = [&](int j) __attribute__((always_inline)) {  // k step j % ST of block j / ST
            return *(const bf16x8_t *)(kl + (from ^ (j % ST & 3) * 64) + (j % ST >> 2) * 256 + j / ST * 16 * PITCH);
          };
          bf16x8_t kf[KB * ST];
          constexpr int AHEAD = NQ == 1 ? 4 : 2;
#pragma unroll
          for (int j = 0; j < AHEAD && j < KB * ST; ++j) kf[j] = load(j);
#pragma unroll
          for (int j = 0; j < KB * ST; ++j) {
            if (j + AHEAD < KB * ST) kf[j + AHEAD] = load(j + AHEAD);
#pragma unroll
            for (int n = 0; n < NQ; ++n)
              sv[n][j / ST] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  kf[j], q[n][j % ST], j % ST ? sv[n][j / ST] : f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        if (more) {  // the next keys into the buffer just read
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          const int blk = *(const int *)(tab + wv * 512 + buf * 256 + (int)attn_lane() * 4);
          rows_of(k0 + KT, blk);
          at = off;
          buf ^= 1;
          ask(buf);  // (past the end: not read; the waits count on it)
          onward();
          move(kc, ka);
        }
        if (edge) {
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            // bit o: key k0 + o is seen
            const int *rows = seen_at + (wv * 64 + (int)attn_lane()) * 4 + 2 * n;
            const int lo = rows[0] - k0, hi = rows[1] - k0;
            uint64_t seen = hi < 0 ? 0ull : hi > 62 ? ~0ull : (2ull << hi) - 1ull;
            seen &= lo > 63 ? 0ull : lo > 0 ? ~0ull << lo : ~0ull;
            seen = (seen & now) >> (attn_lane() >> 4 << 2);
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int on = __builtin_amdgcn_sbfe((int)(seen >> (b & ~1) * 16), (b & 1) * 16 + i, 1);  // 0 or -1
                sv[n][b][i] = __uint_as_float((__float_as_uint(sv[n][b][i]) & (uint32_t)on) | (0xFF800000u & ~(uint32_t)on));
              }
          }
        }
        // The weights' reference is the row's first maximum; it follows (and the sums with it) when a score passes
        // it by 2^60: bf16 and f32 hold such weights as exactly as those below 1.
        float top[NQ];
        bool far = false;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          top[n] = sv[n][0][0];
#pragma unroll
          for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) top[n] = fmaxf(top[n], sv[n][b][i]);
          top[n] *= sc;
          far |= top[n] > m[n] + 60.f;
        }
        if (__any(far)) {
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            top[n] = fmaxf(top[n], attn_across(top[n], 16));
            top[n] = fmaxf(top[n], attn_across(top[n], 32));
            const bool up = top[n] > m[n] + 60.f;
            const float f = up ? attn_exp2(m[n] - top[n]) : 1.f;
            m[n] = up ? top[n] : m[n];
            l[n] *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[n][d] *= f;
          }
        }
        i16x4_t p[NQ][KB], pl[NQ][KB];  // weights rounded, and what the rounding has taken
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const float ref = m[n] == -__builtin_inff() ? 0.f : m[n];
#pragma unroll
          for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const float e0 = attn_exp2(__builtin_fmaf(sv[n][b][i], sc, -ref));
              const float e1 = attn_exp2(__builtin_fmaf(sv[n][b][i + 1], sc, -ref));
              l[n] += e0 + e1;
              bf16x2_t x, y;
              x[0] = (__bf16)e0, x[1] = (__bf16)e1;
              const uint32_t w = __builtin_bit_cast(uint32_t, x);
              y[0] = (__bf16)(e0 - __uint_as_float(w << 16)), y[1] = (__bf16)(e1 - __uint_as_float(w & 0xFFFF0000u));
              p[n][b][i] = __builtin_bit_cast(short, (__bf16)x[0]), p[n][b][i + 1] = __builtin_bit_cast(short, (__bf16)x[1]);
              pl[n][b][i] = __builtin_bit_cast(short, (__bf16)y[0]), pl[n][b][i + 1] = __builtin_bit_cast(short, (__bf16)y[1]);
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
#pragma unroll 1
          for (int i = 0; i < OPS; ++i) {
            const uint32_t lane = attn_lane();
            uint4 *x4 = (uint4 *)(vl + i * 1024 + lane * 16);
            const uint4 x = *x4, y = attn_finite(x);
            const bool in = now >> ((uint32_t)(i * 64 + lane) / CPR) & 1;
            odd |= in && (x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w);
            const uint32_t keep = in ? ~0u : 0u;
            *x4 = make_uint4(y.x & keep, y.y & keep, y.z & keep, y.w & keep);
          }
          if (__any(odd)) *poison = 1;
        }
        {
          const uint32_t ln = attn_lane();
          const int row = (int)((ln >> 4) * 4 + (ln >> 2 & 3));
          // this lane's place in the 16 x 16 block (b, d) of the values
          const uint32_t from = va + row * PITCH + ((int)(ln >> 1 & 1) ^ attn_swz<DP>(row)) * 16 + (ln & 1) * 8;
          // (16 rows on, the swizzle is the same)
          constexpr int CB = KB == 1 ? 1 : KB / 2, N = DT * CB, AHEAD = NQ == 1 ? 2 : 1;
          auto load = [&](int j) __attribute__((always_inline)) {  // key blocks 2 (j % CB) and the next, columns j / CB
            const int d = j / CB, b = j % CB * 2;
            const uint32_t x = (from ^ (d & 7) * 32) + (d >> 3) * 256 + b * 16 * PITCH;
            i16x8_t v{};
            const i16x4_t v0 = attn_read_tr(x);
            if constexpr (KB > 1) {
              const i16x4_t v1 = attn_read_tr(x + 16 * PITCH);
              v = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
            } else {
              v = __builtin_shufflevector(v0, v0, 0, 1, 2, 3, 0, 1, 2, 3);
            }
            return v;
          };
          i16x8_t vf[N];
#pragma unroll
          for (int j = 0; j < AHEAD; ++j) vf[j] = load(j);
#pragma unroll
          for (int j = 0; j < N; ++j) {
            if (j + AHEAD < N) vf[j + AHEAD] = load(j + AHEAD);
            const int d = j / CB, b = j % CB * 2;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
              if constexpr (KB == 1) {  // (one product: 16 keys with the weights, the same 16 with their rests)
                const i16x8_t pf = __builtin_shufflevector(p[n][0], pl[n][0], 0, 1, 2, 3, 4, 5, 6, 7);
                acc[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vf[j]),
                                                                    __builtin_bit_cast(bf16x8_t, pf), acc[n][d], 0, 0, 0);
              } else {
                const i16x8_t pf = __builtin_shufflevector(p[n][b], p[n][b + 1], 0, 1, 2, 3, 4, 5, 6, 7);
                const i16x8_t pr = __builtin_shufflevector(pl[n][b], pl[n][b + 1], 0, 1, 2, 3, 4, 5, 6, 7);
                acc[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vf[j]),
                                                                    __builtin_bit_cast(bf16x8_t, pf), acc[n][d], 0, 0, 0);
                acc[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vf[j]),
                                                                    __builtin_bit_cast(bf16x8_t, pr), acc[n][d], 0, 0, 0);
              }
            }
            if (j % 2) __builtin_amdgcn_sched_barrier(0);
          }
        }
        if (!more) break;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        move(vc, va);
        k0 += KT;
      }
    }

    // the four waves' parts, 16 rows at a time through the stage's LDS
    {
      const AttnArgs a = attn_again<AttnArgs>(0);
      const AttnShare s = attn_again<AttnShare>(sizeof(AttnArgs));
      float *macc = (float *)lds;                                  // [wave][16][DP + 4]
      float *mml = (float *)(lds + AR_WAVES * 16 * (DP + 4) * 4);  // [wave][16][2]
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        if (n * 16 >= t.rows) break;
        __syncthreads();
        l[n] += attn_across(l[n], 16);
        l[n] += attn_across(l[n], 32);
        const int ln = (int)attn_lane(), lr = ln & 15, lg = ln >> 4;
        if (lg == 0) mml[(wv * 16 + lr) * 2] = m[n], mml[(wv * 16 + lr) * 2 + 1] = l[n];
#pragma unroll
        for (int d = 0; d < DT; ++d) *(f32x4_t *)(macc + (wv * 16 + lr) * (DP + 4) + d * 16 + lg * 4) = acc[n][d];
        __syncthreads();
#pragma unroll 1
        for (uint32_t i = here(); i < 16 * CPR; i += ATTN_THREADS) {
          const int row = (int)(i / CPR), d0 = (int)(i % CPR * 8);
          if (n * 16 + row >= t.rows || d0 >= D) continue;
          const int64_t orow = attn_row(a, rq.q0, t.row0 + n * 16 + row, head);
          uint4 gate = attn_zeros();
          const bool gated = whole && a.gate;
          if (gated) gate = attn_gate8(a, orow, d0);
          float top = -__builtin_inff(), f[AR_WAVES], sum = 0.f, o[8];
#pragma unroll
          for (int v = 0; v < AR_WAVES; ++v) {
            // (a wave without keys for this row has no sums)
            const float mv = mml[(v * 16 + row) * 2];
            f[v] = mml[(v * 16 + row) * 2 + 1] != 0.f ? mv : -__builtin_inff();
            top = fmaxf(top, f[v]);
          }
#pragma unroll
          for (int v = 0; v < AR_WAVES; ++v) {
            f[v] = f[v] == -__builtin_inff() ? 0.f : attn_exp2(f[v] - top);
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
          float z = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) z = __builtin_fmaf(o[e], 0.f, z);
          if (*poison || (z != 0.f && sum == sum)) {
            // values that are not finite: those held back; and those that met both parts of a weight (inf - inf), whose
            // own sum says what the result is (where weights are NaN, as of NaN queries, it is that anyway)
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            attn_poison(a, rq, tabrow, head, t.row0 + n * 16 + row, ks, ke, d0, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = o[e] * 0.f == 0.f ? o[e] + x[e] : x[e] * 0.f == 0.f ? o[e] : x[e];
          }
          if (whole) {
            const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] *= inv;
            if (gated) attn_times_gate(gate, o);
            attn_put8(a, orow, d0, o);
          } else {
            const int64_t pr = (int64_t)part * TR + n * 16 + row;
            float4 *to = (float4 *)(s.acc + pr * DP + d0);
            to[0] = make_float4(o[0], o[1], o[2], o[3]), to[1] = make_float4(o[4], o[5], o[6], o[7]);
            if (d0 == 0) s.ml[pr * 2] = top, s.ml[pr * 2 + 1] = sum;
          }
        }
      }
    }
    if constexpr (!FULL) {  // the merge has overwritten the zeros past D
      __syncthreads();
      for (int i = here(); i < AR_STAGE / 16; i += ATTN_THREADS) ((uint4 *)lds)[i] = attn_zeros();
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

size_t attn_rows_lds(int DP, int R) {
  return ar_fixed(DP) + AR_TAB + 16 * ATTN_THREADS + attn_plan_lds(R);
}

hipError_t launch_attn_rows(const AttnArgs &a, const AttnShare &s, int DP, int tr, int grid, hipStream_t st) {
  return DP == 64 ? launch_dp<64>(a, s, tr, grid, st)
                  : DP == 128 ? launch_dp<128>(a, s, tr, grid, st) : launch_dp<256>(a, s, tr, grid, st);
}

}  // namespace qmm
