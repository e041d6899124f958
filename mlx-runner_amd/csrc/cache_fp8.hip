// A paged cache held in 8 bits: E4M3 codes [pages, heads, block, D], a scale 2^(X - 127) for each page and head.
//
// cache_write_kernel: y = the head's values after norm and rotation (rope.h), in f32.  The call's rows of one page (a run:
// they follow one another) and one head share
//
//   t = min { t >= -127 : 448 * 2^t >= max |y| }  (finite y),   t' = t if the run holds the page's first row, else max(t, old t)
//   code = rne_e4m3(y * 2^-t');   a page whose scale grows: its codes c -> rne_e4m3(c * 2^(old t - t'))
//
// An E4M3 value keeps 4 significant bits at any scale that leaves it normal (2^-6 .. 448), so one power of two for a whole
// page loses next to nothing, and when it grows only codes that become subnormal are rounded again.
//
// A workgroup takes one head of k or v and the runs that start in a window of as many tokens as its lanes hold rows
// (16 values a lane), or of fewer where there are few, so a run is seen whole by one workgroup and no atomics leave it.  Rows
// past the window (of its last run) take further turns.  The workgroups that turn q's heads lie between them.
//
// One token 5.4 us (latency: slots, the page's old scale, the head's sums, the maximum through LDS), 2048 tokens of 24 heads on
// 4 of 256 (63 MB) 17.1-17.6 us, 3.6 TB/s, bound by the copy rate and the ramp as rope_kernel.
#include <atomic>

#include "rope.h"

namespace qmm {

namespace {

constexpr int CW_RUNS = 64;  // of a window at most
constexpr int CW_WIDE = 1024, CW_MANY = 512;

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }

// Codes of eight values over 2^t; what is not finite: NaN.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], int t) {
  const float scale = e8m0_scale_operand(t < 127 ? t : 127);
  uint32_t w[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = finite(x[4 * k + j]) ? x[4 * k + j] : __uint_as_float(0x7FC00000u);
    i16x2_t c = {0, 0};
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, y[0], y[1], scale, false);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, y[2], y[3], scale, true);
    w[k] = __builtin_bit_cast(uint32_t, c);
  }
  return make_uint2(w[0], w[1]);
}
// Four codes times 2^-by.
__device__ __forceinline__ uint32_t shrink4(uint32_t w, int by) {
  const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  int c = __builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(a.x, -by), ldexpf(a.y, -by), 0, false);
  c = __builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(b.x, -by), ldexpf(b.y, -by), c, true);
  return (uint32_t)c;
}

struct CacheWrite {
  uint8_t *scales[2];  // of k, of v
  int windows, span;  // tokens of a window
  bool early;         // few workgroups: loads ahead of what says whether they are needed
  // The grid: `writers` workgroups for k and v, `pairs` (a head of k or v each) times `columns` (a window each), one before every `period` - 1 of
  // those that turn q's heads, `parts` to a token.
  int writers, pairs, columns, period, parts;
  int angles;  // (cw_angles)
  FastDiv by_block, by_half, by_pairs, by_period;
};

__device__ __forceinline__ int fast_quot(int n, FastDiv d) { return (int)(__umulhi((uint32_t)n << 1, d.mul) >> d.shift); }

// Dynamic LDS: cos and sin of a turn's angles (as of one token's, by the workgroups of q), and 16 values a thread (ACROSS).
constexpr int cw_angles(int threads, int lph, int half) {
  const int n = (threads >> lph) * half;
  return n < 128 ? 128 : (n + 3) & ~3;
}
constexpr size_t cw_lds(int pairs, int threads, int lph, int half) {
  return (size_t)cw_angles(threads, lph, half) * 8 + (pairs == ACROSS ? threads * 64 : 0);
}

// THREADS: ROPE_THREADS, workgroups of q among them, or CW_WIDE, without.
template <int PAIRS, bool IN_F32, int THREADS>
__global__ __launch_bounds__(THREADS, THREADS > ROPE_THREADS ? 4 : PAIRS == ACROSS ? 3 : IN_F32 ? 4 : 5)
void cache_write_kernel(const RopeArgs a, const CacheWrite w, int lph) {
  extern __shared__ __attribute__((aligned(16))) float cw_dynamic[];
  __shared__ __attribute__((aligned(16))) float norm[ROPE_MAX_SETS][256];
  __shared__ float freq[128];
  __shared__ int pos[THREADS / 4];
  __shared__ uint32_t top[CW_RUNS];
  __shared__ int begun[CW_RUNS], exponent[CW_RUNS], grown[CW_RUNS], grown_page[CW_RUNS], n_grown;
  float *cs = cw_dynamic, *sn = cs + w.angles, *swap = sn + w.angles;
  const int writer = fast_quot(blockIdx.x, w.by_period);
  if constexpr (THREADS == ROPE_THREADS) {
    if (writer >= w.writers || (int)blockIdx.x != writer * w.period) {
      const int before = writer < w.writers ? writer + 1 : w.writers;
      rope_heads<PAIRS, IN_F32, false>(a, 1, lph, w.parts, blockIdx.x - before, cs, sn, norm, swap);
      return;
    }
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int rows = THREADS >> lph;  // of a turn
  const int l = tid & ((1 << lph) - 1), g = tid >> lph;
  const bool turned = PAIRS != ACROSS && l < a.half / 8;
  const int d0 = (PAIRS == HALVES && turned ? l : 2 * l) * 8, d1 = PAIRS == HALVES && turned ? d0 + a.half : d0 + 8;
  const bool in0 = d0 < a.D, in1 = d1 < a.D;
  const int heads = a.set[1].heads;

  auto page_of = [&](int slot) -> int {  // -1: none
    const int page = fast_quot(slot, w.by_block);
    return slot >= 0 && page < a.NB ? page : -1;
  };
  const int window0 = fast_quot(writer, w.by_pairs), pair0 = writer - window0 * w.pairs;
#pragma unroll 1
  for (int window = window0, pair = pair0; window < w.windows; pair += w.pairs) {
    if (pair >= 2 * heads) {
      pair = pair0 - w.pairs, window += w.columns;
      continue;
    }
    const int side = pair >= heads, head = side ? pair - heads : pair, w0 = window * w.span;
    const RopeHeads &s = a.set[1 + side];
    // What the first steps need, on its way at once: slots from the window's first row on (64 at least), weights and
    // frequencies, and the rows and positions of a turn from there on (of use where the first run starts there and it is the
    // only turn).
    const int w1 = a.T - w0 < w.span ? a.T : w0 + w.span;
    const int t = w0 + lane;
    const int slot_t = t < a.T ? a.slots[t] : -1, slot_b = w0 > 0 ? a.slots[w0 - 1] : -1;
    const float freq_l = s.rotate && tid < a.half ? a.freqs[tid] : 0.f;
    const int pos_l = w.early && s.rotate && tid < rows && w0 + tid < a.T ? a.positions[w0 + tid] : 0;
    auto load = [&](int row, Eight<IN_F32> (&raw)[2]) __attribute__((always_inline)) {
      const int64_t at = ((int64_t)row * heads + head) * s.in_stride;
      if (in0) raw[0] = load8<IN_F32>(s.in, at + d0);
      if (in1) raw[1] = load8<IN_F32>(s.in, at + d1);
    };
    Eight<IN_F32> early[2] = {};
    if (w.early && w0 + g < a.T) load(w0 + g, early);
    float norm_l = 0.f;
    if (s.norm && tid < a.D)
      norm_l = s.norm_f32 ? ((const float *)s.norm)[tid] : __uint_as_float((uint32_t)((const uint16_t *)s.norm)[tid] << 16);

    // the runs that start in the window, by every wave for itself: a bit for the first row of each
    const int mine = page_of(slot_t);
    const int up = __shfl_up(mine, 1, 64), before = lane ? up : page_of(slot_b);
    const uint64_t starts = __ballot(t < w1 && mine >= 0 && mine != before);
    if (starts == 0) continue;
    const int lead = __builtin_ctzll(starts), first = w0 + lead;
    const int last_page = __builtin_amdgcn_readlane(mine, w1 - w0 - 1);
    int end = w1;
    if (last_page >= 0 && end < a.T) {  // its last run's end
      uint64_t other = __ballot(t >= a.T || mine != last_page);
      other &= w.span < 64 ? ~0ull << w.span : 0;
      end = w0 + 64;
      while (!other) {
        other = __ballot(end + lane >= a.T || page_of(a.slots[end + lane]) != last_page);
        end += 64;
      }
      end += __builtin_ctzll(other) - 64;
    }
    const bool starter = tid < 64 && (starts >> lane & 1);  // has a run of its own
    uint8_t *const scale = w.scales[side] + (int64_t)mine * heads + head;
    const int old = starter ? (int)*scale - 127 : 0;
    __syncthreads();  // (the last item's are read)
    if (tid < CW_RUNS) top[tid] = 0, begun[tid] = 0;
    if (tid < 128) freq[tid] = freq_l;
    if (THREADS == 256 || tid < 256) norm[0][tid & 255] = norm_l;

    auto run_of = [&](int row) -> int {
      const int i = row - w0;
      return __popcll(starts & (i < 63 ? (2ull << i) - 1 : ~0ull)) - 1;
    };
    // The turns, last to first, for the maxima: then the first two's values are still there, and only the others' are formed
    // again for their codes (16 rows of 256, 32 of 128 or 64 of 64 values are one turn).
    const int turns = (end - first + rows - 1) >> ((THREADS == ROPE_THREADS ? 8 : 10) - lph);
    const bool there = w.early && lead == 0 && turns == 1;
    float before_x[2][8] = {};
    int slot_before = -1;
#pragma unroll 1
    for (int step = 0; step < 2 * turns - 1; step += step == turns - 1 ? 2 : 1) {
      const int row0 = first + (step < turns ? turns - 1 - step : step - turns + 1) * rows, row = row0 + g;
      if (step) __syncthreads();  // (the angles of the turn before are read)
      Eight<IN_F32> raw[2] = {early[0], early[1]};
      if (!there) load(row < end ? row : first, raw);
      const int slot = row < end ? a.slots[row] : -1;
      if (s.rotate) {
        if (tid < rows) pos[tid] = there ? pos_l : row0 + tid < end ? a.positions[row0 + tid] : 0;
        __syncthreads();
        const int half = a.half, n = (end - row0 < rows ? end - row0 : rows) * half;
        for (int i = tid; i < n; i += THREADS) {
          const int r = fast_quot(i, w.by_half), j = i - r * half;
          float sv, c;
          rope_angle(pos[r], freq[j], sv, c);
          cs[i] = c * a.amplitude, sn[i] = sv * a.amplitude * a.sign;
        }
      }
      __syncthreads();
      float x[2][8];
#pragma unroll
      for (int k = 0; k < 2; ++k) widen<IN_F32>(raw[k], x[k]);
      if (s.norm) rope_norm(x, &norm[0][d0 & 255], &norm[0][d1 & 255], in0, in1, lph, a.D, a.eps);
      if constexpr (PAIRS == ACROSS) {
        if (s.rotate)
          rope_turn_across(x, swap + (tid >> lph << lph) * 16, l, a.half, a.interleaved, cs + g * a.half, sn + g * a.half);
      } else if (s.rotate && turned) {
        float c[8], sv[8];
#pragma unroll
        for (int j = 0; j < 8; j += 4)
          *(float4 *)&c[j] = *(const float4 *)&cs[g * a.half + l * 8 + j],
          *(float4 *)&sv[j] = *(const float4 *)&sn[g * a.half + l * 8 + j];
        rope_turn<PAIRS>(x, c, sv);
      }
      const int page = page_of(slot);
      if (step < turns) {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (in0 && finite(x[0][j])) m = fmaxf(m, fabsf(x[0][j]));
          if (in1 && finite(x[1][j])) m = fmaxf(m, fabsf(x[1][j]));
        }
        m = over_head(m, lph, [](float a, float b) { return fmaxf(a, b); });
        if (l == 0 && page >= 0) {
          const int run = run_of(row);
          atomicMax(&top[run], __float_as_uint(m));
          if (slot == page * a.block) begun[run] = 1;
        }
      }
      if (step == turns - 1) {  // the scales, and older codes where they grow
        __syncthreads();
        if (tid < 64) {
          const int run = __popcll(starts & ((1ull << lane) - 1));
          int by = 0;
          if (starter) {
            const float m = __uint_as_float(top[run]);
            int e = m > 0.f ? ceil_scale_exp(m) : -127;
            if (!begun[run]) {
              by = e > old ? e - old : 0;
              e = e > old ? e : old;
            }
            *scale = (uint8_t)(e + 127);
            exponent[run] = e;
          }
          const uint64_t all = __ballot(by > 0);
          const int i = __popcll(all & ((1ull << lane) - 1));
          if (by > 0) grown[i] = by, grown_page[i] = mine;
          if (lane == 0) n_grown = __popcll(all);
        }
        __syncthreads();
        if (n_grown) {
          const int64_t words = (int64_t)a.block * a.D / 16;  // of a page, 16 codes each
          int64_t i = tid;
          int r = 0;
#pragma unroll 1
          while (true) {
            while (r < n_grown && i >= words) i -= words, ++r;
            if (r >= n_grown) break;
            uint4 *codes = (uint4 *)((uint8_t *)s.out + ((int64_t)grown_page[r] * heads + head) * a.block * a.D) + i;
            const int by = grown[r];
            const uint4 c = *codes;
            *codes = make_uint4(shrink4(c.x, by), shrink4(c.y, by), shrink4(c.z, by), shrink4(c.w, by));
            i += THREADS;
          }
          __syncthreads();  // (their rows of this call come after)
        }
      }
      auto store = [&](int row, int slot, const float (&x)[2][8]) __attribute__((always_inline)) {
        const int page = page_of(slot);
        if (page < 0) return;
        const int e = exponent[run_of(row)];
        uint8_t *to = (uint8_t *)s.out + (((int64_t)page * heads + head) * a.block + (slot - page * a.block)) * a.D;
        if (in0) *(uint2 *)(to + d0) = codes8(x[0], e);
        if (in1) *(uint2 *)(to + d1) = codes8(x[1], e);
      };
      if (step >= turns - 1) store(row, slot, x);
      if (step == turns - 1) {
        if (turns > 1) store(row + rows, slot_before, before_x);
      } else {
        slot_before = slot;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) before_x[k][j] = x[k][j];
      }
    }
  }
}

// Codes to values, E to a lane: 16 bytes out of each at a time.  Bound by the copy rate; results are stored past the caches,
// which they would only fill: 9 prefixes of 100 to 32768 rows as bfloat16 (658 MB) 133 us through them, 123 past them, 32000
// rows of 4 heads of 256 as float32 (328 MB) 84 and 50, 6.6 TB/s.
template <bool F32>
__global__ __launch_bounds__(256) void cache_read_kernel(const CacheReadArgs a, int chunks) {
  constexpr int E = F32 ? 4 : 8, U = 4;
  const int set = blockIdx.y;
  const uint8_t *codes = a.codes[set], *scales = a.scales[set];
  const int cpr = a.D / E;
  const int64_t t0 = (int64_t)blockIdx.x * (256 * U) / chunks;
  const int i0 = (int)((int64_t)blockIdx.x * (256 * U) - t0 * chunks) + (int)threadIdx.x;
  uint32_t w[U][E / 4];
  int e[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = i0 + u * 256, t = i / chunks, j = i - t * chunks, h = j / cpr, c = j - h * cpr;
    e[u] = -1;
    if (t0 + t >= a.T) continue;
    const int slot = a.slots[t0 + t], page = slot / a.block;
    if (slot < 0 || page >= a.NB) continue;
    const int64_t at = (int64_t)page * a.H + h;
    e[u] = scales[at];
    const uint32_t *p = (const uint32_t *)(codes + (at * a.block + (slot - page * a.block)) * a.D + c * E);
#pragma unroll
    for (int k = 0; k < E / 4; ++k) w[u][k] = p[k];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t at = (t0 * chunks + i0 + u * 256) * E;
    if (at >= (int64_t)a.T * chunks * E) continue;
    float v[E];
    const float f = e[u] < 0 ? 0.f : e8m0_to_f32((uint32_t)e[u]);
#pragma unroll
    for (int k = 0; k < E / 4; ++k) {
      const f32x2_t x = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[u][k], false), y = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[u][k], true);
      v[4 * k] = x.x * f, v[4 * k + 1] = x.y * f, v[4 * k + 2] = y.x * f, v[4 * k + 3] = y.y * f;
    }
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] = e[u] < 0 ? 0.f : v[k];
    if constexpr (F32) {
      __builtin_nontemporal_store(f32x4_t{v[0], v[1], v[2], v[3]}, (f32x4_t *)((float *)a.out[set] + at));
    } else {
      u32x4_t y;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        bf16x2_t x;
        x[0] = (__bf16)v[2 * k], x[1] = (__bf16)v[2 * k + 1];
        y[k] = __builtin_bit_cast(uint32_t, x);
      }
      __builtin_nontemporal_store(y, (u32x4_t *)((uint16_t *)a.out[set] + at));
    }
  }
}

template <int PAIRS, bool IN_F32, int THREADS>
hipError_t launch_write(const RopeArgs &a, const CacheWrite &w, unsigned grid, int lph, hipStream_t st) {
  if (cw_lds(PAIRS, THREADS, lph, a.half) > 32 << 10) {
    static std::atomic<uint64_t> done{0};
    const void *k = (const void *)cache_write_kernel<PAIRS, IN_F32, THREADS>;
    const hipError_t e = ensure_dynamic_lds(done, k, (int)cw_lds(PAIRS, THREADS, 2, 32));
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((cache_write_kernel<PAIRS, IN_F32, THREADS>), dim3(grid), dim3(THREADS), cw_lds(PAIRS, THREADS, lph, a.half), st,
                     a, w, lph);
  return hipGetLastError();
}
template <int PAIRS>
hipError_t launch_pairs(const RopeArgs &a, const CacheWrite &w, unsigned grid, int lph, int threads, hipStream_t st) {
  if (PAIRS != ACROSS && threads == CW_WIDE)
    return a.in_f32 ? launch_write<PAIRS == ACROSS ? HALVES : PAIRS, true, CW_WIDE>(a, w, grid, lph, st)
                    : launch_write<PAIRS == ACROSS ? HALVES : PAIRS, false, CW_WIDE>(a, w, grid, lph, st);
  return a.in_f32 ? launch_write<PAIRS, true, ROPE_THREADS>(a, w, grid, lph, st)
                  : launch_write<PAIRS, false, ROPE_THREADS>(a, w, grid, lph, st);
}

}  // namespace

hipError_t launch_rope_fp8(const RopeArgs &a, uint8_t *const (&scales)[ROPE_MAX_SETS], hipStream_t st) {
  if (a.T <= 0 || a.D < 16 || a.D > 256 || a.D % 16 || a.half < 0 || 2 * a.half > a.D || a.sets != 3 || a.block < 1 ||
      a.T > 1 << 30 || a.set[0].heads > INT32_MAX / 4 || a.set[1].heads < 1 || a.set[1].heads > 1 << 29 || a.set[1].heads != a.set[2].heads)
    return hipErrorInvalidValue;
  // Pages of more rows than two turns have, and more tokens than decoding requests mostly have together: 1024 threads, q in a
  // launch of its own.  What decides is how many rows of a page there are, which only the GPU knows.  (24 heads on 4 of 256, pages
  // of 64 rows: 2048 tokens of one prompt with 256 threads 35-40 us, with 1024 26; 1024 tokens 24 and 17; 512 17.6 and 13.9; 64 to
  // 256 16 and 12.  300 decoding requests 8.5 and 16; 600 8.4 and 18; 1000 11.5 and 15.9; 171 of 3 tokens 9.7 and 14.3.  Pages of
  // 128 and 256: 2048 tokens 51-59 and 26-34, 107 and 48; 512 tokens 32 and 17.6.)
  const int lph = a.D <= 64 ? 2 : a.D <= 128 ? 3 : 4;
  const int threads = a.block > 2 * ROPE_THREADS >> lph && a.T > CW_MANY && a.half % 8 == 0 ? CW_WIDE : ROPE_THREADS, rows = threads >> lph;
  CacheWrite w{};
  w.scales[0] = scales[1], w.scales[1] = scales[2];
  w.pairs = a.set[1].heads < 1 << 15 ? 2 * a.set[1].heads : 1 << 16;
  // few tokens: windows of fewer, down to one each, until there is a workgroup a CU (64 sequences' steps of 128 tokens in all,
  // 4 heads of 96: 10.2 us with windows of 32, 6.2 us with those of 4, where fewer angles are formed one after the other)
  w.span = rows < CW_RUNS ? rows : CW_RUNS;
  while (w.span > 1 && ((int64_t)a.T + w.span - 1) / w.span * w.pairs < 256) w.span /= 2;
  w.windows = (int)(((int64_t)a.T + w.span - 1) / w.span);
  w.early = (int64_t)w.windows * w.pairs <= 512;
  w.columns = w.windows < (1 << 20) / w.pairs ? w.windows : (1 << 20) / w.pairs;
  w.writers = w.pairs * w.columns;
  w.by_block = fast_div(a.block), w.by_half = fast_div(a.half ? a.half : 1), w.by_pairs = fast_div(w.pairs);
  int64_t grid = w.writers;
  w.period = 1;
  w.angles = cw_angles(threads, lph, a.half);
  if (threads != ROPE_THREADS || a.T > ROPE_TOKENS) {  // (a grid's lanes are counted in 32 bits: q in launches of its own)
    RopeArgs q = a;
    q.sets = 1;
    if (q.set[0].heads > 0) {
      const hipError_t e = launch_rope(q, st);
      if (e != hipSuccess) return e;
    }
  } else {
    w.parts = (int)rope_parts(a, 1, lph);
    const int64_t turners = (int64_t)a.T * w.parts;
    grid += turners;
    w.period = 1 + (int)(turners / w.writers);
  }
  w.by_period = fast_div(w.period);
  return a.half % 8      ? launch_pairs<ACROSS>(a, w, (unsigned)grid, lph, threads, st)
         : a.interleaved ? launch_pairs<NEXT>(a, w, (unsigned)grid, lph, threads, st)
                         : launch_pairs<HALVES>(a, w, (unsigned)grid, lph, threads, st);
}

hipError_t launch_cache_read(const CacheReadArgs &a, hipStream_t st) {
  if (a.T <= 0 || a.sets < 1 || a.sets > 2 || a.H < 1 || a.D < 16 || a.D > 256 || a.D % 16 || a.block < 1)
    return hipErrorInvalidValue;
  const int E = a.out_f32 ? 4 : 8;
  const int64_t chunks = (int64_t)a.H * (a.D / E);
  if (chunks > INT32_MAX / 2) return hipErrorInvalidValue;
  // (a grid's lanes are counted in 32 bits: what is over in further launches)
  CacheReadArgs part = a;
  const int64_t most = ((int64_t)1 << 33) / chunks / 8 * 8 > 0 ? ((int64_t)1 << 33) / chunks / 8 * 8 : 1;
  for (int64_t t0 = 0; t0 < a.T; t0 += part.T) {
    part.T = (int)(a.T - t0 < most ? a.T - t0 : most);
    part.slots = a.slots + t0;
    for (int i = 0; i < a.sets; ++i) part.out[i] = (char *)a.out[i] + t0 * a.H * a.D * (a.out_f32 ? 4 : 2);
    const dim3 grid((unsigned)((part.T * chunks + 1023) / 1024), a.sets);
    if (a.out_f32)
      hipLaunchKernelGGL((cache_read_kernel<true>), grid, dim3(256), 0, st, part, (int)chunks);
    else
      hipLaunchKernelGGL((cache_read_kernel<false>), grid, dim3(256), 0, st, part, (int)chunks);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace qmm
