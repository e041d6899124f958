// Paged attention of many rows per key head over a cache of E4M3 codes.
//
// S^T = K Q^T in bf16: every wave widens the keys that it has moved, with their scales (exact), into LDS.  (The scaled
// 32x32x64 MFMA takes codes as they are, and bf16 queries as two E4M3 parts at the same cost.  But it aligns the products of
// eight values to the largest and drops what lies below 2^-13 of that one's power of two: beside keys' large channels a score of
// 1057 came out 0.04 off, and weights by percents.  2048 tokens over 32768 keys, 24 heads on 4 of 256: 1.50-1.55 ms so, 1.65-1.68
// with bf16, where eight waves' keys take LDS's bandwidth and widening a second barrier; widened by each wave for itself, in
// registers, 1.68-1.71.  4000 tokens of 32 heads on 8 of 128: 198 and 201 us.)
//
// O^T = V^T P^T, where a head has at most 128 values (WIDE): values are widened like keys, and the weights, rounded to bf16
// once, take the values' scales as exponents of two.  With 256 values LDS has no room for that (half of the queries 64 KB, one
// tile's keys 32 KB, two tiles' codes of values 32 KB): the codes go into the scaled MFMA as they are, and the weights in two
// E4M3 parts (2^-8 of a weight lost), scaled for each row and 32 keys by a power of two of those keys' own maximum, which the
// matrix unit takes off again; what E4M3's 18 binades cannot hold is 2^-22 of the largest weight of 32 keys, what the unit drops
// of eight products less than 2^-10 of the largest.  A page's scale of values is the other operand's where the tile's keys
// share it; else it goes into the weights, relative to the tile's largest.  The products cost the same; two parts cost 2.5
// instructions a weight, one rounding half of one: 4000 tokens of 32 heads on 8 of 128 228 us with two parts, 201 with bf16;
// chunks of 7 prompts, 16 heads of 64, window 1000, 124 and 107.
//
// A tile is 256 rows, 32 for each of eight waves, two a SIMD (D 64: four): one's softmax beside the other's products, with
// nothing interleaved by hand.  64 keys at a time, eight keys by each wave, moved a tile ahead: by DMA into two buffers, keys of
// 256 values into registers; one barrier a tile, with 256 values two (one buffer for the widened keys).
//
// Bound by matrix unit, vector unit and LDS in turn: 2048 tokens over 32768 keys, 24 heads on 4 of 256, 1.65-1.68 ms, 0.96
// PFLOP/s (bf16 pages 1.43-1.48), the matrix unit busy for 41% of it.
#include <type_traits>

#include "attention.h"
#include "gemm_pipe.h"

namespace qmm {

namespace {

constexpr int C8_THREADS = 512, C8_WAVES = C8_THREADS / 64;
constexpr int C8_TR = 256, C8_KT = 64;
constexpr int C8_EXTRA = 3;   // what a tile's own overhead costs, in units of 64 keys
constexpr int C8_SCALES = 2 * 2 * 256;                  // scale bytes of the keys, of the values; a dword each, two sets
constexpr int C8_TAB = C8_WAVES * 2 * 32;               // page ids of the tiles to come
constexpr int C8_VALID = 2 * C8_WAVES;                  // bits of the keys that there are, two sets
constexpr int C8_SMALL = C8_SCALES + C8_TAB + C8_VALID + 8 * C8_THREADS;
constexpr int C8_RANGE = 40;  // weights up to 2^60 times scales up to 2^40 times codes stay far below f32's end
constexpr int C8_NEAR = 8;  // scales of 32 keys' values that differ by up to 2^8 go in relative to the largest

// Whether keys, values and weights lie in LDS, or go in, as bf16
constexpr bool c8_wide(int DP) { return DP < 256; }
constexpr int c8_tile(int DP) { return C8_KT * DP; }
constexpr int c8_tiles(int DP) { return (c8_wide(DP) ? 12 : 4) * c8_tile(DP); }
// The queries' upper halves, where registers do not hold them
constexpr int c8_queries(int DP) { return DP == 128 ? 0 : C8_TR * DP; }
constexpr int c8_fixed(int DP) {
  const int out = C8_WAVES * 32 * 64 * 4, in = c8_tiles(DP) + c8_queries(DP);  // (rows out: 64 columns of a wave's rows at a time)
  return in > out ? in : out;
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void c8_dma4(const void *g, uint32_t l) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(l), "v"(g) : "memory", "m0");
}
__device__ __forceinline__ void c8_dma1(const void *g, uint32_t l) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off" ::"s"(l), "v"(g) : "memory", "m0");
}
#pragma clang diagnostic pop

// A register as it is: for conversions that write half of one.
__device__ __forceinline__ int c8_any() {
  int x;
  asm volatile("" : "=v"(x));
  return x;
}
// (fmaxf would first quiet each)
__device__ __forceinline__ float c8_max3(float x, float y, float z) {
  asm("v_max3_f32 %0, %0, %1, %2" : "+v"(x) : "v"(y), "v"(z));
  return x;
}
// The larger of x here and 32 lanes away.
__device__ __forceinline__ float c8_pair_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <int DP, bool FULL>
__global__ __launch_bounds__(C8_THREADS, DP == 64 ? 4 : 2) void attn_chunk8_kernel(const AttnArgs args, const AttnShare share) {
  constexpr int CPR = DP / 16;     // 16-byte chunks of a row
  constexpr int KS = DP / 16;      // k steps of S^T
  constexpr int DT = DP / 32;      // 32-column tiles of O^T
  constexpr int RPI = 64 / CPR;    // rows of a DMA operation
  constexpr int OPS = 8 > RPI ? 8 / RPI : 1;  // operations of a wave's 8 rows
  constexpr int TILE = c8_tile(DP), PITCH = DP;
  constexpr bool WIDE = c8_wide(DP);
  constexpr int KR = c8_queries(DP) ? KS / 2 : KS;  // of them with queries in registers
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  uint8_t *qup = lds + c8_tiles(DP);
  uint8_t *scl = lds + c8_fixed(DP);                 // [2][keys, values][64]
  uint8_t *tab = scl + C8_SCALES;                    // [wave][2][8]
  uint8_t *vm = tab + C8_TAB;                        // [2][8 waves], a byte each
  int *seen_at = (int *)(vm + C8_VALID);             // [thread][2]: what its row sees
  AttnPlan *plan = (AttnPlan *)(seen_at + 2 * C8_THREADS);

  const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  auto here = [&]() __attribute__((always_inline)) { return wv * 64 + (int)attn_lane(); };  // the thread's number
  int left;
  {
    const AttnWork w = attn_uniform(attn_share<C8_TR, C8_KT, C8_EXTRA, C8_THREADS>(args, share, plan));
    if (share.first) attn_zero_rest<C8_THREADS>(args);
    attn_note_none(share, w);
    if (tid == 0) plan->work[0] = w, plan->poison[0] = 0;
    left = w.left;
  }
  const uint32_t la = lds_addr(lds), ta = lds_addr(tab) + wv * 64, sa = lds_addr(scl);
  if constexpr (!FULL) {  // head values past D: never written by the DMA, zero for good
    for (int i = tid; i < 4 * TILE / 16; i += C8_THREADS) ((uint4 *)lds)[i] = attn_zeros();
  }

  int turn = 0;
#pragma unroll 1
  while (left > 0) {
    __syncthreads();
    const AttnArgs a = attn_again<AttnArgs>(0);
    const AttnWork w = attn_uniform(plan->work[turn]);
    int *poison = &plan->poison[turn];
    const int r = attn_uniform(attn_request(plan, a.R, w));
    const AttnReq rq = attn_uniform(attn_req(plan, a, r));
    const AttnTile t = attn_uniform(attn_tile(a, rq, w.tile - (r ? attn_end(plan, a.R, r - 1) : 0), C8_TR));
    const int units = attn_units<C8_KT>(t);
    const AttnPiece pc = attn_piece<C8_EXTRA>(w, units);
    const int ks = (int)((uint32_t)t.b / C8_KT + pc.u0) * C8_KT, nt = pc.u1 - pc.u0;
    const bool whole = pc.whole;
    const int part = w.g * 2 + pc.start, head = w.head;
    if (pc.start && !pc.none && here() == 0)
      attn_note(attn_again<AttnShare>(sizeof(AttnArgs)), w, rq, t, units + C8_EXTRA, whole);
    {
      AttnWork on = w;
      on.r = r;
      attn_move_on(on, pc.take, units + C8_EXTRA);
      left = on.left;
      turn ^= 1;
      if (here() == 0) plan->work[turn] = on, plan->poison[turn] = 0;
    }
    if (pc.none) continue;

    const int *tabrow = a.table + (int64_t)r * a.W;
    const int block = a.block, NB = a.NB, Hkv = a.Hkv, D = FULL ? DP : a.D;
    const uint8_t *kc = (const uint8_t *)a.k, *vc = (const uint8_t *)a.v, *ksc = a.k_scales, *vsc = a.v_scales;
    const float sc = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.44269504088896341f;

    // the lane's row: what it sees, its queries
    float m, l = 0.f;
    bf16x8_t q[KR];
    {
      const int ln = (int)attn_lane(), in = wv * 32 + (ln & 31), lh = ln >> 5;
      const bool on = in < t.rows;
      const int row = t.row0 + (on ? in : 0);  // (a row past the end: the first one's queries)
      const int pos = rq.base + (int)attn_div(row, a.by_g);
      seen_at[here() * 2] = a.window && pos >= a.window ? pos - a.window + 1 : 0;
      seen_at[here() * 2 + 1] = on ? pos : -1;
      // (a row that sees nothing needs no reference; one past the end has no weights and passes none)
      m = !on ? __builtin_inff() : pos >= 0 ? -__builtin_inff() : 0.f;
      const uint16_t *qp = a.q + attn_row(a, rq.q0, row, head) * a.D;
      u16x2_t top = {0, 0};  // of the magnitudes, by their bits
      bf16x8_t *const up = (bf16x8_t *)(qup + wv * 32 * DP) + ln;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int at = s * 16 + lh * 8;
        u32x4_t x = {0u, 0u, 0u, 0u};
        if (at < D) x = *(const u32x4_t *)(qp + at);
        // a negative scale: -q, so that maxima stay maxima; none: no scores
        x = a.scale > 0.f ? x : a.scale < 0.f ? x ^ 0x80008000u : u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, x[i] & 0x7FFF7FFFu));
        if (s < KR)
          q[s < KR ? s : 0] = __builtin_bit_cast(bf16x8_t, x);
        else
          up[(s - KR) * 64] = __builtin_bit_cast(bf16x8_t, x);
      }
      // a query that is not finite: NaN
      const uint32_t nan = top[0] >= 0x7F80u || top[1] >= 0x7F80u ? 0x7FC07FC0u : 0u;
      q[0] = __builtin_bit_cast(bf16x8_t, __builtin_bit_cast(u32x4_t, q[0]) | nan);
    }
    f32x16_t acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;

    if (nt > 0) {
      // Keys on their way: this lane looks up key wv * 8 + lane % 8 of each tile; `page` and `off` (its place in its page)
      // are those of the tile whose page ids are asked for next.
      const uint32_t per = attn_div(C8_KT, a.by_block), rest = C8_KT - per * (uint32_t)block;
      const uint32_t first = ks + wv * 8 + ((int)attn_lane() & 7);
      uint32_t page = attn_div(first, a.by_block), off = first - page * block;
      const uint32_t last_page = attn_div(t.e - 1, a.by_block);
      auto onward = [&]() __attribute__((always_inline)) {
        page += per, off += rest;
        if (off >= (uint32_t)block) off -= block, ++page;
      };
      auto ask = [&](int set) __attribute__((always_inline)) {
        if (attn_lane() < 8) c8_dma4(tabrow + (page < last_page ? page : last_page), attn_uniform(ta + set * 32));
      };
      // tile j's rows of the whole cache, for this lane's key (0 where there is none), and their pages' scales' places
      uint32_t mine = 0, of = 0, there = 0;
      auto look_up = [&](int j, int blk, uint32_t at) __attribute__((always_inline)) {
        const bool page_there = (uint32_t)blk < (uint32_t)NB;
        const bool ok = page_there && ks + j * C8_KT + wv * 8 + ((int)attn_lane() & 7) < t.e;
        of = ((uint32_t)blk * Hkv + head) & (page_there ? ~0u : 0u);
        mine = (of * block + at) & (ok ? ~0u : 0u);
        there = (uint32_t)__ballot(ok) & 0xFFu;
        vm[(j & 1) * C8_WAVES + wv] = (uint8_t)there;
      };
      auto move = [&](const uint8_t *cache, int to) __attribute__((always_inline)) {
        const uint32_t ln = attn_lane();
        const uint32_t c0 = ln % CPR;
#pragma unroll
        for (int n = 0; n < OPS; ++n) {
          const uint32_t in = n * RPI + ln / CPR;  // of the wave's 8 rows
          const uint32_t row = __builtin_amdgcn_ds_bpermute((int)in * 4, (int)mine);
          const uint32_t c = (c0 ^ (uint32_t)attn_swz8<DP>((int)(wv * 8 + in))) * 16;
          if ((RPI <= 8 || ln < 8 * CPR) && (FULL || c < (uint32_t)D))
            gp_dma16(cache + ((uint64_t)row * (uint32_t)D + c), attn_uniform(la + to + wv * 8 * PITCH + n * 1024));
        }
      };
      u32x4_t keys[WIDE ? 1 : OPS];  // (not WIDE: on their way in registers; zeros past D)
      auto move_all = [&](int j) __attribute__((always_inline)) {
        const int set = j & 1;
        if (attn_lane() < 8) {
          c8_dma1(ksc + of, attn_uniform(sa + set * 512 + wv * 32));
          c8_dma1(vsc + of, attn_uniform(sa + set * 512 + 256 + wv * 32));
        }
        if constexpr (WIDE) {
          move(kc, set * TILE);
        } else {
          const uint32_t ln = attn_lane();
#pragma unroll
          for (int n = 0; n < OPS; ++n) {
            const uint32_t row = __builtin_amdgcn_ds_bpermute((int)(n * RPI + ln / CPR) * 4, (int)mine), c = ln % CPR * 16;
            keys[n] = u32x4_t{0u, 0u, 0u, 0u};
            if (FULL || c < (uint32_t)D) keys[n] = *(const u32x4_t *)(kc + ((uint64_t)row * (uint32_t)D + c));
          }
        }
        move(vc, (2 + set) * TILE);
      };
      auto valid_of = [&](int j) __attribute__((always_inline)) -> uint64_t {
        const uint2 bits = *(const uint2 *)(vm + (j & 1) * C8_WAVES);
        return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)bits.y) << 32 |
               (uint32_t)__builtin_amdgcn_readfirstlane((int)bits.x);
      };
      // whether rows of the tile see different keys of tile j
      auto differ = [&](int j) __attribute__((always_inline)) -> bool {
        const int k0 = ks + j * C8_KT;
        return k0 < t.full_b || k0 + C8_KT > t.full_e;
      };

      f32x16_t sv[2];
      int sb = 0, tvv = 0;  // the second product's scales
      i32x8_t ph{}, pl{};
      bf16x8_t pb[4]{};  // (WIDE: the weights of 16 keys each)
      const f32x16_t z = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      // S^T of tile j: 2 x 32 keys
      auto scores = [&](int j) __attribute__((always_inline)) {
        const uint32_t ln = attn_lane();
        const int row = ln & 31;
        const int from = (WIDE ? (8 + 2 * (j & 1)) * TILE : 0) + row * 2 * PITCH + ((int)(ln >> 5) ^ attn_swz<DP>(row)) * 16;
        const bf16x8_t *const up = (const bf16x8_t *)(qup + wv * 32 * DP) + ln;
        constexpr int N = 2 * KS, AHEAD = 3;
        auto load = [&](int n) __attribute__((always_inline)) {  // step n / 2 of half n % 2
          return *(const bf16x8_t *)(lds + (from ^ n / 2 % 8 * 32) + n / 16 * 256 + n % 2 * 32 * 2 * PITCH);
        };
        bf16x8_t kf[N], qs = q[0];
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) kf[n] = load(n);
#pragma unroll
        for (int n = 0; n < N; ++n) {
          if (n + AHEAD < N) kf[n + AHEAD] = load(n + AHEAD);
          if (n % 2 == 0) qs = n / 2 < KR ? q[n / 2 < KR ? n / 2 : 0] : up[(n / 2 < KR ? 0 : n / 2 - KR) * 64];
          sv[n % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[n], qs, n < 2 ? z : sv[n % 2], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("" : "+v"(sv[0]), "+v"(sv[1]));  // (as after a product)
      };
      // What the scales of tile j's values do to its weights: of eight keys each (they have one, where pages are multiples of
      // eight), how far it is below the largest of their half, 4 bits each; `far`: the halves where that does not do.
      // (Pages whose scale is NaN add that to the rows that see them at the end.)
      // WIDE: 2^up of each eight keys' scale and 2^-up, `far` where eight differ or pass 2^(+-C8_RANGE).
      int tv[2], less = 0, far = 0;
      float up[8], down[8];
      auto prepare = [&](int j) __attribute__((always_inline)) {
        const uint32_t ln = attn_lane();
        const int vs = *((const int *)(scl + (j & 1) * 512 + 256) + ln);
        const uint64_t valid = valid_of(j);
        const uint64_t nan = __ballot(vs == 255) & valid, fine = valid & ~nan;
        if (nan) *poison = 1;
        if constexpr (WIDE) {
          const uint64_t other = __ballot(vs != __builtin_amdgcn_update_dpp(vs, vs, 0x111, 0xF, 0xF, false)) & 0xFEFEFEFEFEFEFEFEull;
          far = (other | (__ballot(vs - (127 - C8_RANGE) > 2u * C8_RANGE) & valid)) != 0;
          // (2^-up is finite for keys that there are not too, at any byte: their weights are zeros, and so is what they add)
          const int x = __float_as_int((float)(vs - 127)), y = (254 - (vs < 254 ? vs : 254)) << 23;
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            up[v] = __int_as_float(__builtin_amdgcn_readlane(x, v * 8));
            down[v] = __int_as_float(__builtin_amdgcn_readlane(y, v * 8));
          }
          return;
        }
        // (a lane beside the one before it, but for the first of eight; one that is not there has its page's, or the first page's)
        const uint64_t other = __ballot(vs != __builtin_amdgcn_update_dpp(vs, vs, 0x111, 0xF, 0xF, false)) & 0xFEFEFEFEFEFEFEFEull;
        far = ((uint32_t)other != 0) | ((uint32_t)(other >> 32) != 0) << 1;
        less = 0;
        int of = vs;  // that of the eight's first key that there is, -1: none
        if (fine != ~0ull) {
          const uint32_t in = (uint32_t)(fine >> (ln & 56)) & 0xFFu;
          of = __builtin_amdgcn_ds_bpermute((int)((ln & 56) + (in ? __builtin_ctz(in) : 0)) * 4, vs);
          of = in ? of : -1;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          int x[4], most = 0;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            x[v] = __builtin_amdgcn_readlane(of, half * 32 + v * 8);
            most = x[v] > most ? x[v] : most;
          }
          tv[half] = most;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int d = x[v] < 0 ? 0 : most - x[v];
            far |= (d > C8_NEAR) << half;
            less |= (d & 15) << (half * 16 + v * 4);
          }
          if (far >> half & 1) {  // the largest of all
            uint64_t keys = 0xFFFFFFFFull << 32 * half & fine;
            while (keys) {  // (once for each scale there is)
              const int y = __builtin_amdgcn_readlane(vs, __builtin_ctzll(keys));
              tv[half] = y > tv[half] ? y : tv[half];
              keys &= ~__ballot(vs == y);
            }
          }
        }
      };
      // the weights of tile j's scores
      auto soften = [&](int j) __attribute__((always_inline)) {
        const int k0 = ks + j * C8_KT;
        const uint64_t valid = valid_of(j);
        const bool edge = differ(j) || valid != ~0ull;
        // (inline assembly reads S^T below: even a 16-pass product's results can be read after 19 wait states)
        asm volatile("s_nop 15\n\ts_nop 3" : "+v"(sv[0]), "+v"(sv[1]));
        if (edge) {
          const int h4 = (int)attn_lane() >> 5 << 2;
          const int2 sees = *(const int2 *)(seen_at + here() * 2);
          const int lo = sees.x - k0, hi = sees.y - k0;
          // bit o: key k0 + o is seen
          uint64_t seen = hi < 0 ? 0ull : hi > 62 ? ~0ull : (2ull << hi) - 1ull;
          seen &= lo > 63 ? 0ull : lo > 0 ? ~0ull << lo : ~0ull;
          seen &= valid;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t s32 = (uint32_t)(seen >> 32 * half) >> h4;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const int on = __builtin_amdgcn_sbfe((int)s32, 8 * (j / 4) + j % 4, 1);  // 0 or -1
              sv[half][j] = __uint_as_float((__float_as_uint(sv[half][j]) & (uint32_t)on) | (0xFF800000u & ~(uint32_t)on));
            }
          }
        }

        const int *vsl = (const int *)(scl + (j & 1) * 512 + 256);
        if constexpr (WIDE) {
          float top = -__builtin_inff();
#pragma unroll
          for (int j = 0; j < 32; j += 2) top = c8_max3(top, sv[j >> 4][j & 15], sv[j >> 4][(j & 15) + 1]);
          // The reference is the row's first maximum; it follows, and the sums with it, when a score passes it by 2^60.
          if (__any(m == -__builtin_inff() || top * sc > m + 60.f)) {
            const float all = __builtin_ceilf(c8_pair_max(top) * sc);
            m = m == -__builtin_inff() ? all : m;
            const bool rise = all > m + 60.f;
            const float f = rise ? attn_exp2(m - all) : 1.f;
            m = rise ? all : m;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= f;
          }
          const float ref = m == -__builtin_inff() ? 0.f : m;
          auto pack = [&](int v, const float (&x)[4]) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 4; ++j) pb[v >> 1][(v & 1) * 4 + j] = (__bf16)x[j];
          };
          // the weights with their values' scales, f32's exponents over
          if (far) {
#pragma unroll
            for (int v = 0; v < 8; ++v) {
              const i32x4_t vs = *(const i32x4_t *)(vsl + v * 8 + ((int)attn_lane() >> 5) * 4);
              float x[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) x[j] = attn_exp2(__builtin_fmaf(sv[v >> 2][(v & 3) * 4 + j], sc, -ref));
              l += (x[0] + x[1]) + (x[2] + x[3]);
#pragma unroll
              for (int j = 0; j < 4; ++j) x[j] = __builtin_amdgcn_ldexpf(x[j], vs[j] - 127);
              pack(v, x);
              __builtin_amdgcn_sched_barrier(0);  // (few registers at a time)
            }
          } else {
#pragma unroll
            for (int v = 0; v < 8; ++v) {
              const float from = up[v] - ref;
              float x[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) x[j] = attn_exp2(__builtin_fmaf(sv[v >> 2][(v & 3) * 4 + j], sc, from));
              l = __builtin_fmaf((x[0] + x[1]) + (x[2] + x[3]), down[v], l);
              pack(v, x);
            }
          }
          return;
        }

        // Maxima of the scores, in powers of two, rounded up
        float top[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          top[half] = -__builtin_inff();
#pragma unroll
          for (int j = 0; j < 16; j += 2) top[half] = c8_max3(top[half], sv[half][j], sv[half][j + 1]);
          top[half] = __builtin_ceilf(c8_pair_max(top[half]) * sc);
        }
        // (the matrix unit reads its scale operands after the instruction has issued, and the compiler does not know: they
        // stay in their registers until the products are read)
        asm volatile("" ::"v"(sb), "v"(tvv), "v"(top[0]), "v"(top[1]));
        {
          // The reference is the row's first maximum; it follows, and the sums with it, when a score passes it by 2^60.
          const float all = fmaxf(top[0], top[1]);
          m = m == -__builtin_inff() ? all : m;
          if (__any(all > m + 60.f)) {
            const bool up = all > m + 60.f;
            const float f = up ? attn_exp2(m - all) : 1.f;
            m = up ? all : m;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= f;
          }
        }
        const float ref = m == -__builtin_inff() ? 0.f : m;
        int by[2];
        // x = 2^(scale s - d - e), d how far eight keys' scale is below the largest.  FAR: relative to the largest of what the
        // weights with their scales come to, which e does not follow otherwise.
        auto weights = [&](auto half_c, auto far_c) __attribute__((always_inline)) {
          constexpr int half = decltype(half_c)::value;
          constexpr bool FAR = decltype(far_c)::value;
          float most = top[half];
          if constexpr (FAR) {
            most = -__builtin_inff();
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const i32x4_t vs = *(const i32x4_t *)(vsl + half * 32 + v * 8 + ((int)attn_lane() >> 5) * 4);
              float y[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) y[j] = __builtin_fmaf(sv[half][v * 4 + j], sc, (float)(uint8_t)vs[j]);
              most = c8_max3(c8_max3(most, y[0], y[1]), y[2], y[3]);
              __builtin_amdgcn_sched_barrier(0);
            }
            most = __builtin_ceilf(c8_pair_max(most) - (float)tv[half]);
          }
          // weights up to 2^8 relative to 2^e, which the product takes back
          const float e = fmaxf(most - 8.f, ref - 120.f);
          const float from = FAR ? fmaxf(top[half], ref - 120.f) : e;
          const int rest = FAR ? (int)(from - e) - tv[half] : 0;
          float sum = 0.f;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float x[4];
            i32x4_t vs;
            if constexpr (FAR) vs = *(const i32x4_t *)(vsl + half * 32 + v * 8 + ((int)attn_lane() >> 5) * 4);
            const int d = FAR ? 0 : less >> (half * 16 + v * 4) & 15;
            const float down = -from - (float)d;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = attn_exp2(__builtin_fmaf(sv[half][v * 4 + j], sc, down));
            sum = __builtin_fmaf((x[0] + x[1]) + (x[2] + x[3]), (float)(1 << d), sum);
            if constexpr (FAR) {
#pragma unroll
              for (int j = 0; j < 4; ++j) x[j] = __builtin_amdgcn_ldexpf(x[j], vs[j] + rest);
            }
            int hi = c8_any();
            hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], hi, false);
            hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], hi, true);
            ph[half * 4 + v] = hi;
            const f32x2_t b0 = __builtin_amdgcn_cvt_pk_f32_fp8(hi, false), b1 = __builtin_amdgcn_cvt_pk_f32_fp8(hi, true);
            const float under = __uint_as_float((127u - 5u) << 23);  // the rest is at most 2^3: times 2^5
            i16x2_t lo = __builtin_bit_cast(i16x2_t, c8_any());
            lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, x[0] - b0.x, x[1] - b0.y, under, false);
            lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, x[2] - b1.x, x[3] - b1.y, under, true);
            pl[half * 4 + v] = __builtin_bit_cast(int, lo);
            if constexpr (FAR) __builtin_amdgcn_sched_barrier(0);  // (few registers at a time)
          }
          l += __builtin_amdgcn_ldexpf(sum, (int)(from - ref));
          by[half] = (int)(e - ref) + 127;
        };
        auto weights_of = [&](auto half_c) __attribute__((always_inline)) {
          constexpr int half = decltype(half_c)::value;
          if (far >> half & 1)
            weights(half_c, std::true_type{});
          else
            weights(half_c, std::false_type{});
        };
        weights_of(std::integral_constant<int, 0>{});
        weights_of(std::integral_constant<int, 1>{});
        // (the lanes' scales are those of the two halves' keys)
        const bool upper = (int)attn_lane() >> 5;
        sb = upper ? by[1] : by[0];
        sb = sb < 254 ? sb : 254;
        sb = sb * 257 - (5 << 8);

        tvv = upper ? tv[1] : tv[0];
        asm volatile("" : "+v"(tvv));  // (in a register of its own)
      };
      // Keys that are none, and codes that are NaN (which must not reach the rows that do not see their keys): zeros for now,
      // in the rows of the values that this wave has moved
      auto clean = [&](int j) __attribute__((always_inline)) {
        if (!differ(j) && there == 0xFFu) return;
        bool odd = false;
        const uint32_t ln = attn_lane();
#pragma unroll
        for (int n = 0; n < OPS; ++n) {
          if (RPI <= 8 || ln < 8 * CPR) {
            uint4 *to = (uint4 *)(lds + (2 + (j & 1)) * TILE + wv * 8 * PITCH + n * 1024 + ln * 16);
            const uint4 x = *to, y = attn_finite_codes(x);
            const bool in = there >> (n * RPI + ln / CPR) & 1;
            odd |= in && (x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w);
            *to = in ? y : attn_zeros();
          }
        }
        if (__any(odd)) *poison = 1;
      };
      // The rows that this wave has moved as bf16: keys with their scales, values (WIDE) without (codes are exact there), those
      // cleaned as above
      auto wide16 = [&](u32x4_t w, float f, u32x4_t (&o)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const bf16x2_t y = k & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[k >> 1], f, true)
                                   : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[k >> 1], f, false);
          o[k >> 2][k & 3] = __builtin_bit_cast(uint32_t, y);
        }
      };
      auto widen_key = [&](int j, u32x4_t codes, int row, int chunk) __attribute__((always_inline)) {
        u32x4_t o[2];
        wide16(codes, __int_as_float(((const int *)(scl + (j & 1) * 512))[row] << 23), o);
        uint8_t *to = lds + (WIDE ? (8 + 2 * (j & 1)) * TILE : 0) + row * 2 * PITCH;
        *(u32x4_t *)(to + (chunk ^ attn_swz<DP>(row)) * 16) = o[0];
        *(u32x4_t *)(to + ((chunk + 1) ^ attn_swz<DP>(row)) * 16) = o[1];
      };
      auto widen_keys = [&](int j) __attribute__((always_inline)) {
        const uint32_t ln = attn_lane();
#pragma unroll
        for (int n = 0; n < OPS; ++n) widen_key(j, keys[WIDE ? 0 : n], wv * 8 + n * RPI + (int)(ln / CPR), 2 * (int)(ln % CPR));
      };
      auto widen = [&](int j) __attribute__((always_inline)) {
        const bool strict = differ(j) || there != 0xFFu;
        bool odd = false;
        const uint32_t ln = attn_lane();
#pragma unroll
        for (int n = 0; n < OPS; ++n) {
          if (RPI <= 8 || ln < 8 * CPR) {
            const int at = wv * 8 * PITCH + n * 1024 + ln * 16;
            uint4 x = *(const uint4 *)(lds + (2 + (j & 1)) * TILE + at);
            const int own = n * RPI + ln / CPR, row = wv * 8 + own;  // (of the wave's 8, of the tile's)
            const int chunk = 2 * ((int)(ln % CPR) ^ attn_swz8<DP>(row));
            u32x4_t o[2];
            widen_key(j, *(const u32x4_t *)(lds + (j & 1) * TILE + at), row, chunk);
            if (strict) {
              const uint4 y = attn_finite_codes(x);
              const bool in = there >> own & 1;
              odd |= in && (x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w);
              x = in ? y : attn_zeros();
            }
            wide16(u32x4_t{x.x, x.y, x.z, x.w}, 1.f, o);
            const int c = chunk ^ attn_swz_v<DP>(row);  // (its two chunks stay side by side)
            u32x4_t *to = (u32x4_t *)(lds + (4 + 2 * (j & 1)) * TILE + row * 2 * PITCH + c * 16);
            to[0] = o[0], to[1] = o[1];
          }
        }
        if (strict && __any(odd)) *poison = 1;
      };
      auto product_wide = [&](int j) __attribute__((always_inline)) {
        const uint32_t ln = attn_lane();
        const int row = 4 * (ln >> 5) + (ln >> 2 & 3);
        const uint32_t from = la + (4 + 2 * (j & 1)) * TILE + row * 2 * PITCH +
                              ((int)((ln >> 4 & 1) * 2 + (ln >> 1 & 1)) ^ attn_swz_v<DP>(row)) * 16 + (ln & 1) * 8;
        constexpr int N = 4 * DT, AHEAD = 3;
        auto load = [&](int n) __attribute__((always_inline)) {
          const int d = n % DT, c = n / DT;
          const uint32_t at = (from ^ d * 64) + c * 16 * 2 * PITCH;
          const i16x4_t v0 = attn_read_tr(at), v1 = attn_read_tr(at + 8 * 2 * PITCH);
          return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        bf16x8_t vf[N];
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) vf[n] = load(n);
#pragma unroll
        for (int n = 0; n < N; ++n) {
          if (n + AHEAD < N) vf[n + AHEAD] = load(n + AHEAD);
          acc[n % DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[n], pb[n / DT], acc[n % DT], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) asm volatile("" : "+v"(acc[d]));  // (as below)
      };
      // O^T += V^T P^T
      auto product = [&](int j) __attribute__((always_inline)) {
        const int set = j & 1;
        const uint32_t ln = attn_lane();
        const int row = (int)((ln >> 3 & 1) * 8 + (ln >> 5) * 4 + (ln >> 1 & 3));
        const uint32_t from = la + (2 + set) * TILE + row * PITCH + ((int)(ln >> 4 & 1) ^ attn_swz8<DP>(row)) * 16 + (ln & 1) * 8;
        auto load = [&](int d) __attribute__((always_inline)) {
          i32x8_t v;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const i32x2_t x = attn_read_tr8((from ^ d * 32) + n * 16 * PITCH);
            v[2 * n] = x.x, v[2 * n + 1] = x.y;
          }
          return v;
        };
        i32x8_t vf[DT];
        constexpr int AHEAD = 3;
#pragma unroll
        for (int d = 0; d < AHEAD && d < DT; ++d) vf[d] = load(d);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          if (d + AHEAD < DT) vf[d + AHEAD] = load(d + AHEAD);
          acc[d] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(vf[d], ph, acc[d], 0, 0, 0, tvv, 0, sb);
          acc[d] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(vf[d], pl, acc[d], 0, 0, 0, tvv, 1, sb);
          __builtin_amdgcn_sched_barrier(0);
        }
        // (the compiler would put products off behind the branches that follow, and keep their operands till then)
#pragma unroll
        for (int d = 0; d < DT; ++d) asm volatile("" : "+v"(acc[d]));
      };

      look_up(0, tabrow[page < last_page ? page : last_page], off);
      move_all(0);
      onward();
      ask(1);
#pragma unroll 1
      for (int i = 0; i < nt; ++i) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if constexpr (WIDE) {
          widen(i);
        } else {
          gp_lds_barrier();  // everyone has done with the last tile's keys (LDS has room for one tile of them)
          widen_keys(i);
          clean(i);
        }
        gp_lds_barrier();  // tile i, its valid bits, page ids of tile i + 1; everyone has done with tile i - 1
        if (i + 1 < nt) {
          const int blk = *(const int *)(tab + wv * 64 + ((i + 1) & 1) * 32 + (attn_lane() & 7) * 4);
          look_up(i + 1, blk, off);
          move_all(i + 1);
          onward();
          ask(i & 1);
        }
        scores(i);
        prepare(i);
        soften(i);
        if constexpr (WIDE)
          product_wide(i);
        else
          product(i);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      asm volatile("" ::"v"(sb), "v"(tvv));
    }

    // Rows out, 64 columns of a wave's 32 rows at a time, through its part of the LDS (16-byte chunks, swizzled by row)
    {
      const AttnArgs a = attn_again<AttnArgs>(0);
      const AttnShare s = attn_again<AttnShare>(sizeof(AttnArgs));
      __syncthreads();
      const int in0 = wv * 32;
      if (in0 < t.rows) {
        const float lu = l + attn_across(l, 32);
        const float scale = !whole ? 1.f : lu != 0.f ? 1.f / lu : 0.f;
        const int ln = (int)attn_lane();
        if (!whole && ln < 32 && in0 + ln < t.rows) {
          const int64_t pr = (int64_t)part * C8_TR + in0 + ln;
          s.ml[pr * 2] = m, s.ml[pr * 2 + 1] = lu;
        }
        float *out = (float *)(lds + wv * 32 * 64 * 4);
        const int end = ks + nt * C8_KT < t.e ? ks + nt * C8_KT : t.e;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
#pragma unroll
          for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const f32x16_t &x = acc[c * 2 + d];
              *(float4 *)(out + (ln & 31) * 64 + ((d * 8 + v * 2 + (ln >> 5)) ^ (ln & 15)) * 4) =
                  make_float4(x[4 * v] * scale, x[4 * v + 1] * scale, x[4 * v + 2] * scale, x[4 * v + 3] * scale);
            }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
#pragma unroll 1
          for (int it = 0; it < 4; ++it) {
            const int rr = it * 8 + (ln >> 3), k = ln & 7, in = in0 + rr, d0 = c * 64 + k * 8;
            if (in >= t.rows || (!FULL && d0 >= a.D)) continue;
            const float *x = out + rr * 64;
            float o[8];
            *(float4 *)&o[0] = *(const float4 *)(x + ((2 * k) ^ (rr & 15)) * 4);
            *(float4 *)&o[4] = *(const float4 *)(x + ((2 * k + 1) ^ (rr & 15)) * 4);
            if (*poison) attn_poison<true>(a, rq, tabrow, head, t.row0 + in, ks, end, d0, o);
            if (whole) {
              attn_store8(a, attn_row(a, rq.q0, t.row0 + in, head), d0, o);
            } else {
              float4 *to = (float4 *)(s.acc + ((int64_t)part * C8_TR + in) * DP + d0);
              to[0] = make_float4(o[0], o[1], o[2], o[3]), to[1] = make_float4(o[4], o[5], o[6], o[7]);
            }
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
        }
      }
    }
    if constexpr (!FULL) {
      __syncthreads();
      for (int j = here(); j < 4 * TILE / 16; j += C8_THREADS) ((uint4 *)lds)[j] = attn_zeros();
    }
  }
}

template <int DP, bool FULL>
hipError_t launch_t(const AttnArgs &a, const AttnShare &s, int grid, hipStream_t st) {
  static std::atomic<uint64_t> done{0};
  const void *k = (const void *)attn_chunk8_kernel<DP, FULL>;
  const hipError_t e = ensure_dynamic_lds(done, k, (int)attn_chunk8_lds(DP, ATTN_MAX_R));
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((attn_chunk8_kernel<DP, FULL>), dim3(grid), dim3(C8_THREADS), attn_chunk8_lds(DP, a.R), st, a, s);
  return hipGetLastError();
}

template <int DP>
hipError_t launch_dp(const AttnArgs &a, const AttnShare &s, int grid, hipStream_t st) {
  return a.D == DP ? launch_t<DP, true>(a, s, grid, st) : launch_t<DP, false>(a, s, grid, st);
}

}  // namespace

size_t attn_chunk8_lds(int DP, int R) { return c8_fixed(DP) + C8_SMALL + attn_plan_lds(R); }

hipError_t launch_attn_chunk8(const AttnArgs &a, const AttnShare &s, int DP, int grid, hipStream_t st) {
  return DP == 64 ? launch_dp<64>(a, s, grid, st) : DP == 128 ? launch_dp<128>(a, s, grid, st) : launch_dp<256>(a, s, grid, st);
}

}  // namespace qmm
