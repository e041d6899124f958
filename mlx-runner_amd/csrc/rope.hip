// Rotary positions, alone or together with the head norms before them and the write of k and
// v to their cache rows after them.  Per token t and pair i of a head's 2 `half` rotated values:
//
//   th = positions[t] * freqs[i];  c = amplitude cos th, s = amplitude sin th
//   (a, b) -> (a c - b s, a s + b c),  a, b = x[i], x[i + half] or x[2 i], x[2 i + 1]
//
// and x = x * rsqrt(mean(x^2) + eps) * w first where a norm is given.  All in f32, rounded once.
//
// A token's angles are the same for all of its heads: a workgroup takes one token (or a part
// of its heads, where there are few tokens), forms the `half` angles once and goes through the
// heads, 4, 8 or 16 lanes to a head (D up to 64, 128, 256), 16 values to a lane.  Where `half` is a
// multiple of 8 a lane's two chunks of 8 hold both sides of its pairs (HALVES: i and i + half;
// NEXT: neighbours) and nothing leaves it; else (ACROSS) the sides meet through LDS, within a wave.
// Bound by the copy rate: 4096 tokens of 24 heads of 256 (101 MB) 22.7-23.0 us, 4.4 TB/s; where a
// pair's halves met through LDS 28.2 us, bound by the vector unit.
#include "qmm_device.h"
#include "qmm_launch.h"

namespace qmm {

namespace {

constexpr int ROPE_THREADS = 256;

// Eight values as they lie in memory.
template <bool F32>
struct Eight {
  uint4 w[F32 ? 2 : 1];
};
template <bool F32>
__device__ __forceinline__ Eight<F32> load8(const void *p, int64_t i) {
  Eight<F32> x;
  if constexpr (F32) {
    x.w[0] = ((const uint4 *)((const float *)p + i))[0];
    x.w[1] = ((const uint4 *)((const float *)p + i))[1];
  } else {
    x.w[0] = *(const uint4 *)((const uint16_t *)p + i);
  }
  return x;
}
template <bool F32>
__device__ __forceinline__ void widen(const Eight<F32> &x, float (&o)[8]) {
  if constexpr (F32) {
    const uint32_t w[8] = {x.w[0].x, x.w[0].y, x.w[0].z, x.w[0].w, x.w[1].x, x.w[1].y, x.w[1].z, x.w[1].w};
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = __uint_as_float(w[j]);
  } else {
    const uint32_t w[4] = {x.w[0].x, x.w[0].y, x.w[0].z, x.w[0].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[2 * j] = __uint_as_float(w[j] << 16);
      o[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
  }
}

template <bool F32>
__device__ __forceinline__ void store8(void *p, int64_t i, const float (&v)[8]) {
  if constexpr (F32) {
    float4 *o = (float4 *)((float *)p + i);
    o[0] = make_float4(v[0], v[1], v[2], v[3]);
    o[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bf16x2_t x;
      x[0] = (__bf16)v[2 * j], x[1] = (__bf16)v[2 * j + 1];
      w[j] = __builtin_bit_cast(uint32_t, x);
    }
    *(uint4 *)((uint16_t *)p + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Where the pairs of a head lie: both sides (HALVES) or all (NEXT) in a lane's 16 values, or anywhere.
enum { HALVES, NEXT, ACROSS };

// lph: log2 of a head's lanes (16 values each); a wave takes heads of one set only.
template <int PAIRS, bool IN_F32, bool OUT_F32>
__global__ __launch_bounds__(ROPE_THREADS) void rope_kernel(const RopeArgs a, int lph, int parts) {
  constexpr int WAVES = ROPE_THREADS / 64;
  constexpr int TURNS = IN_F32 ? 1 : 2;  // loads of so many heads in flight per lane
  __shared__ __attribute__((aligned(16))) float cs[128], sn[128], norm[ROPE_MAX_SETS][256];
  __shared__ __attribute__((aligned(16))) float swap[PAIRS == ACROSS ? ROPE_THREADS * 16 : 4];
  const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l = tid & ((1 << lph) - 1), g = (tid & 63) >> lph, hpw = 64 >> lph;
  const int t = blockIdx.x / parts, part = blockIdx.x - t * parts;
  // the lane's two chunks of eight values: both sides of eight pairs, or neighbours
  const bool turned = PAIRS != ACROSS && l < a.half / 8;
  const int d0 = (PAIRS == HALVES && turned ? l : 2 * l) * 8, d1 = PAIRS == HALVES && turned ? d0 + a.half : d0 + 8;
  const bool in0 = d0 < a.D, in1 = d1 < a.D;

  // wave item i -> its set, its first head there
  auto which = [&](int &i) __attribute__((always_inline)) -> int {
    int set = 0, n;
    while (set < a.sets && i >= (n = (a.set[set].heads + hpw - 1) >> (6 - lph))) i -= n, ++set;
    i *= hpw;
    return set;
  };
  Eight<IN_F32> raw[TURNS][2];
  auto fetch = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
      int h = i0 + u * parts * WAVES;
      const int set = which(h);
      if (set == a.sets) break;
      const RopeHeads &s = a.set[set];
      if (h + g >= s.heads) continue;
      const int64_t at = ((int64_t)t * s.heads + h + g) * s.in_stride;
      if (in0) raw[u][0] = load8<IN_F32>(s.in, at + d0);
      if (in1) raw[u][1] = load8<IN_F32>(s.in, at + d1);
    }
  };
  // everything that is read on its way before the first is waited for
  int i0 = part * WAVES + wv;
  const int pos = a.positions[t];
  const int slot = a.slots ? a.slots[t] : -1;
  const float freq = tid < a.half ? a.freqs[tid] : 0.f;
  float nw[ROPE_MAX_SETS];
#pragma unroll
  for (int i = 0; i < ROPE_MAX_SETS; ++i) {
    nw[i] = 0.f;
    if (i < a.sets && a.set[i].norm && tid < a.D)
      nw[i] = a.set[i].norm_f32 ? ((const float *)a.set[i].norm)[tid]
                                : __uint_as_float((uint32_t)((const uint16_t *)a.set[i].norm)[tid] << 16);
  }
  fetch(i0);

  if (tid < a.half) {
    // in turns and in 64 bits: at position 2^18 an f32 product is off by up to 2^-7 rad
    double turns = (double)pos * (double)freq * 0.15915494309189533577;
    turns -= __builtin_rint(turns);
    float s, c;
    sincospif(2.f * (float)turns, &s, &c);
    cs[tid] = c * a.amplitude;
    sn[tid] = s * a.amplitude * a.sign;
  }
#pragma unroll
  for (int i = 0; i < ROPE_MAX_SETS; ++i) norm[i][tid] = nw[i];
  __syncthreads();
  float c[8], sv[8];  // of the lane's pairs
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = sv[j] = 0.f;
  if (turned) {
#pragma unroll
    for (int j = 0; j < 8; j += 4)
      *(float4 *)&c[j] = *(const float4 *)&cs[l * 8 + j], *(float4 *)&sv[j] = *(const float4 *)&sn[l * 8 + j];
  }

  const int page = slot / a.block;
  const bool kept = slot >= 0 && page < a.NB;
  while (true) {
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
      int h = i0 + u * parts * WAVES;
      const int set = which(h);
      if (set == a.sets) return;
      const RopeHeads &s = a.set[set];
      const bool on = h + g < s.heads;
      float x[2][8];
#pragma unroll
      for (int k = 0; k < 2; ++k) widen<IN_F32>(raw[u][k], x[k]);
      if (s.norm) {
        float sq[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) sq[k] = __builtin_fmaf(x[k][j], x[k][j], sq[k]);
        float sum = (in0 ? sq[0] : 0.f) + (in1 ? sq[1] : 0.f);
        for (int off = 1 << lph >> 1; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
        const float r = 1.f / sqrtf(sum / (float)a.D + a.eps);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < 8; j += 4) {
            const float4 w = *(const float4 *)&norm[set][((k ? d1 : d0) & 255) + j];
            x[k][j] *= r * w.x, x[k][j + 1] *= r * w.y, x[k][j + 2] *= r * w.z, x[k][j + 3] *= r * w.w;
          }
      }
      if (PAIRS != ACROSS && s.rotate && turned) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float &p = PAIRS == NEXT ? x[j >> 2][(j & 3) * 2] : x[0][j], &q = PAIRS == NEXT ? x[j >> 2][(j & 3) * 2 + 1] : x[1][j];
          const float v = p;
          p = v * c[j] - q * sv[j], q = v * sv[j] + q * c[j];
        }
      }
      if (PAIRS == ACROSS && s.rotate) {  // (a head's lanes are lanes of one wave: no barrier)
        float *mine = swap + (tid >> lph << lph) * 16;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < 8; j += 4) *(float4 *)&mine[(2 * l + k) * 8 + j] = *(float4 *)&x[k][j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const bool next = a.interleaved;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int d = (2 * l + k) * 8 + j;
            if (d >= 2 * a.half) continue;
            const bool first = next ? j % 2 == 0 : d < a.half;
            const int i = next ? d / 2 : first ? d : d - a.half;
            const float other = mine[next ? d ^ 1 : first ? d + a.half : i];
            x[k][j] = first ? x[k][j] * cs[i] - other * sn[i] : other * sn[i] + x[k][j] * cs[i];
          }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
      if (!on || (s.cache && !kept)) continue;
      const int64_t at = s.cache ? (((int64_t)page * s.heads + h + g) * a.block + (slot - page * a.block)) * a.D
                                 : ((int64_t)t * s.heads + h + g) * a.D;
      if (in0) store8<OUT_F32>(s.out, at + d0, x[0]);
      if (in1) store8<OUT_F32>(s.out, at + d1, x[1]);
    }
    i0 += TURNS * parts * WAVES;
    fetch(i0);
  }
}

template <int PAIRS>
void launch_pairs(const RopeArgs &a, unsigned grid, int lph, int parts, hipStream_t st) {
  const dim3 g(grid), b(ROPE_THREADS);
  if (a.in_f32 && a.out_f32)
    hipLaunchKernelGGL((rope_kernel<PAIRS, true, true>), g, b, 0, st, a, lph, parts);
  else if (a.in_f32)
    hipLaunchKernelGGL((rope_kernel<PAIRS, true, false>), g, b, 0, st, a, lph, parts);
  else
    hipLaunchKernelGGL((rope_kernel<PAIRS, false, false>), g, b, 0, st, a, lph, parts);
}

}  // namespace

// Tokens of a launch at most: a grid's lanes are counted in 32 bits (past that the count wraps, with no error).
constexpr int ROPE_TOKENS = 1 << 23;
static_assert((int64_t)ROPE_TOKENS * ROPE_THREADS < (int64_t)1 << 32, "lanes of a grid");

hipError_t launch_rope(const RopeArgs &a, hipStream_t st) {
  if (a.T > ROPE_TOKENS) {
    RopeArgs part = a;
    for (int t0 = 0; t0 < a.T; t0 += part.T) {
      part.T = a.T - t0 < ROPE_TOKENS ? a.T - t0 : ROPE_TOKENS;
      part.positions = a.positions + t0, part.slots = a.slots ? a.slots + t0 : nullptr;
      for (int i = 0; i < a.sets; ++i) {
        const int64_t row = (int64_t)t0 * a.set[i].heads;
        part.set[i].in = (const char *)a.set[i].in + row * a.set[i].in_stride * (a.in_f32 ? 4 : 2);
        if (!a.set[i].cache) part.set[i].out = (char *)a.set[i].out + row * a.D * (a.out_f32 ? 4 : 2);
      }
      const hipError_t e = launch_rope(part, st);
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  }
  if (a.T <= 0 || a.D < 8 || a.D > 256 || a.D % 8 || a.half < 0 || 2 * a.half > a.D || a.sets < 1 ||
      a.sets > ROPE_MAX_SETS || (!a.in_f32 && a.out_f32) || a.block < 1)
    return hipErrorInvalidValue;
  const int lph = a.D <= 64 ? 2 : a.D <= 128 ? 3 : 4;
  int64_t items = 0;  // of a wave
  for (int i = 0; i < a.sets; ++i) {
    if (a.set[i].heads > INT32_MAX / 4) return hipErrorInvalidValue;
    items += (a.set[i].heads + (64 >> lph) - 1) >> (6 - lph);
  }
  if (items == 0) return hipSuccess;
  // few tokens: a token's heads over several workgroups
  const int64_t turns = (items + ROPE_THREADS / 64 - 1) / (ROPE_THREADS / 64);
  int64_t parts = 1024 / a.T;
  parts = parts < 1 ? 1 : parts > turns ? turns : parts;
  const unsigned grid = (unsigned)(a.T * parts);
  a.half % 8    ? launch_pairs<ACROSS>(a, grid, lph, (int)parts, st)
  : a.interleaved ? launch_pairs<NEXT>(a, grid, lph, (int)parts, st)
                  : launch_pairs<HALVES>(a, grid, lph, (int)parts, st);
  return hipGetLastError();
}

}  // namespace qmm
