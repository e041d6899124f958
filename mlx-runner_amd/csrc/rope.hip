// Rotary positions, alone or together with the head norms before them and the write of k and
// v to their cache rows after them.  Per token t and pair i of a head's 2 `half` rotated values:
//
//   th = positions[t] * freqs[i];  c = amplitude cos th, s = amplitude sin th
//   (a, b) -> (a c - b s, a s + b c),  a, b = x[i], x[i + half] or x[2 i], x[2 i + 1]
//
// and x = x * rsqrt(mean(x^2) + eps) * w first where a norm is given.  All in f32, rounded once.
//
// A token's angles are the same for all of its heads: a workgroup takes one token (or a part
// of its heads, where there are few tokens), forms the half angles once and goes through the
// heads, LPH lanes to a head, 8 values to a lane.  The two halves of a pair meet through LDS.
#include "qmm_device.h"
#include "qmm_launch.h"

namespace qmm {

namespace {

constexpr int ROPE_THREADS = 256;

template <bool F32>
__device__ __forceinline__ void load8(const void *p, int64_t i, float (&o)[8]) {
  if constexpr (F32) {
    const float4 a = ((const float4 *)((const float *)p + i))[0], b = ((const float4 *)((const float *)p + i))[1];
    o[0] = a.x, o[1] = a.y, o[2] = a.z, o[3] = a.w, o[4] = b.x, o[5] = b.y, o[6] = b.z, o[7] = b.w;
  } else {
    const uint4 a = *(const uint4 *)((const uint16_t *)p + i);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
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
    for (int j = 0; j < 4; ++j) w[j] = f32_to_bf16_rne(v[2 * j]) | (uint32_t)f32_to_bf16_rne(v[2 * j + 1]) << 16;
    *(uint4 *)((uint16_t *)p + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// LPH: lanes of a head, the power of two from D / 8 up (8, 16 or 32).
template <int LPH, bool IN_F32, bool OUT_F32>
__global__ __launch_bounds__(ROPE_THREADS) void rope_kernel(const RopeArgs a, int parts) {
  constexpr int G = ROPE_THREADS / LPH;  // heads in flight
  __shared__ float cs[128], sn[128];
  __shared__ float swap[G][8][LPH];  // [value of the lane][lane]
  const int tid = threadIdx.x, l = tid % LPH, g = tid / LPH;
  const int t = blockIdx.x / parts, part = blockIdx.x - t * parts;
  int heads = 0;
  for (int i = 0; i < a.sets; ++i) heads += a.set[i].heads;
  const int d0 = l * 8;
  const bool live = d0 < a.D;
  const int pos = a.positions ? a.positions[t] : 0;
  const int slot = a.slots ? a.slots[t] : -1;

  if (tid < a.half) {
    // in turns and in 64 bits: at position 2^18 an f32 product is off by up to 2^-7 rad
    double turns = (double)pos * (double)a.freqs[tid] * 0.15915494309189533577;
    turns -= __builtin_rint(turns);
    float s, c;
    sincospif(2.f * (float)turns, &s, &c);
    cs[tid] = c * a.amplitude;
    sn[tid] = s * a.amplitude * a.sign;
  }
  __syncthreads();

  for (int h0 = part * G; h0 < heads; h0 += parts * G) {
    const int head = h0 + g;
    const bool on = head < heads;
    RopeHeads s = a.set[0];
    int h = head;
    for (int i = 1; i < a.sets; ++i)
      if (h >= s.heads) h -= s.heads, s = a.set[i];
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (on && live) load8<IN_F32>(s.in, ((int64_t)t * s.heads + h) * s.in_stride + d0, x);
    if (s.norm) {
      float sq = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = __builtin_fmaf(x[j], x[j], sq);
#pragma unroll
      for (int off = LPH / 2; off >= 1; off >>= 1) sq += __shfl_xor(sq, off, LPH);
      const float r = 1.f / sqrtf(sq / (float)a.D + a.eps);
      float w[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (live) {
        if (s.norm_f32)
          load8<true>(s.norm, d0, w);
        else
          load8<false>(s.norm, d0, w);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] * r * w[j];
    }
    if (a.interleaved) {
      if (s.rotate) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = l * 4 + j;
          if (i < a.half) {
            const float c = cs[i], sv = sn[i], u = x[2 * j], v = x[2 * j + 1];
            x[2 * j] = u * c - v * sv;
            x[2 * j + 1] = u * sv + v * c;
          }
        }
      }
    } else {
      // (the lanes of a head are lanes of one wave: no barrier, the LDS unit keeps their order)
#pragma unroll
      for (int j = 0; j < 8; ++j) swap[g][j][l] = x[j];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (s.rotate) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int d = d0 + j;
          if (d < 2 * a.half) {
            const bool lo = d < a.half;
            const int i = lo ? d : d - a.half, e = lo ? d + a.half : i;
            const float other = swap[g][e & 7][e >> 3];
            x[j] = lo ? x[j] * cs[i] - other * sn[i] : other * sn[i] + x[j] * cs[i];
          }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    if (!(on && live)) continue;
    if (s.cache) {
      const int page = slot / a.block;
      if (slot >= 0 && page < a.NB)
        store8<OUT_F32>(s.out, (((int64_t)page * s.heads + h) * a.block + (slot - page * a.block)) * a.D + d0, x);
    } else {
      store8<OUT_F32>(s.out, ((int64_t)t * s.heads + h) * a.D + d0, x);
    }
  }
}

template <int LPH>
void launch_lph(const RopeArgs &a, unsigned grid, int parts, hipStream_t st) {
  const dim3 g(grid), b(ROPE_THREADS);
  if (a.in_f32 && a.out_f32)
    hipLaunchKernelGGL((rope_kernel<LPH, true, true>), g, b, 0, st, a, parts);
  else if (a.in_f32)
    hipLaunchKernelGGL((rope_kernel<LPH, true, false>), g, b, 0, st, a, parts);
  else
    hipLaunchKernelGGL((rope_kernel<LPH, false, false>), g, b, 0, st, a, parts);
}

}  // namespace

hipError_t launch_rope(const RopeArgs &a, hipStream_t st) {
  if (a.T <= 0 || a.D < 8 || a.D > 256 || a.D % 8 || a.half < 0 || 2 * a.half > a.D || a.sets < 1 ||
      a.sets > ROPE_MAX_SETS || (!a.in_f32 && a.out_f32) || a.block < 1)
    return hipErrorInvalidValue;
  int64_t heads = 0;
  for (int i = 0; i < a.sets; ++i) heads += a.set[i].heads;
  if (heads <= 0) return hipSuccess;
  if (heads > INT32_MAX / 2) return hipErrorInvalidValue;
  const int lph = a.D <= 64 ? 8 : a.D <= 128 ? 16 : 32;
  // few tokens: a token's heads over several workgroups
  const int64_t turns = (heads * lph + ROPE_THREADS - 1) / ROPE_THREADS;
  int64_t parts = 1024 / a.T;
  parts = parts < 1 ? 1 : parts > turns ? turns : parts;
  if (a.T * parts > INT32_MAX) return hipErrorInvalidValue;
  const unsigned grid = (unsigned)(a.T * parts);
  lph == 8 ? launch_lph<8>(a, grid, (int)parts, st)
           : lph == 16 ? launch_lph<16>(a, grid, (int)parts, st) : launch_lph<32>(a, grid, (int)parts, st);
  return hipGetLastError();
}

}  // namespace qmm
