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
#include "rope.h"

namespace qmm {

namespace {

// lph: log2 of a head's lanes (16 values each).
template <int PAIRS, bool IN_F32, bool OUT_F32>
__global__ __launch_bounds__(ROPE_THREADS) void rope_kernel(const RopeArgs a, int lph, int parts) {
  __shared__ __attribute__((aligned(16))) float cs[128], sn[128], norm[ROPE_MAX_SETS][256];
  __shared__ __attribute__((aligned(16))) float swap[PAIRS == ACROSS ? ROPE_THREADS * 16 : 4];
  rope_heads<PAIRS, IN_F32, OUT_F32>(a, a.sets, lph, parts, blockIdx.x, cs, sn, norm, swap);
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
  for (int i = 0; i < a.sets; ++i)
    if (a.set[i].heads > INT32_MAX / 4) return hipErrorInvalidValue;
  const int64_t parts = rope_parts(a, a.sets, lph);
  if (parts == 0) return hipSuccess;
  const unsigned grid = (unsigned)(a.T * parts);
  a.half % 8    ? launch_pairs<ACROSS>(a, grid, lph, (int)parts, st)
  : a.interleaved ? launch_pairs<NEXT>(a, grid, lph, (int)parts, st)
                  : launch_pairs<HALVES>(a, grid, lph, (int)parts, st);
  return hipGetLastError();
}

}  // namespace qmm
