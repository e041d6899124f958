// Pieces shared by the rotations: values to and from f32, a pair's turn, a head's norm.  A head's values lie 16 to a
// lane, in two chunks of eight, in 4, 8 or 16 lanes (D up to 64, 128, 256).
#pragma once

#include "qmm_device.h"
#include "qmm_launch.h"

namespace qmm {

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

// cos and sin of a position's angle, in turns and in 64 bits (at position 2^18 an f32 product is off by up to 2^-7 rad).
__device__ __forceinline__ void rope_angle(int pos, float freq, float &s, float &c) {
  double turns = (double)pos * (double)freq * 0.15915494309189533577;
  turns -= __builtin_rint(turns);
  sincospif(2.f * (float)turns, &s, &c);
}

// The value of lane ^ OFF, within the vector unit; lane ^ 8 only where a row of 16 lanes is one head's.
template <int OFF>
__device__ __forceinline__ float lane_xor(float v) {
  const int x = __float_as_int(v);
  if constexpr (OFF == 1) return __int_as_float(__builtin_amdgcn_mov_dpp(x, 0xB1, 0xF, 0xF, true));   // quad_perm 1,0,3,2
  if constexpr (OFF == 2) return __int_as_float(__builtin_amdgcn_mov_dpp(x, 0x4E, 0xF, 0xF, true));   // quad_perm 2,3,0,1
  if constexpr (OFF == 8) return __int_as_float(__builtin_amdgcn_mov_dpp(x, 0x128, 0xF, 0xF, true));  // row_ror:8
  const int up = __builtin_amdgcn_update_dpp(x, x, 0x104, 0xF, 0x5, true);  // row_shl:4 into quads 0, 2
  return __int_as_float(__builtin_amdgcn_update_dpp(up, x, 0x114, 0xF, 0xA, true));  // row_shr:4 into quads 1, 3
}
// f over a head's lanes (4, 8 or 16), halves first.
template <class F>
__device__ __forceinline__ float over_head(float v, int lph, F f) {
  if (lph > 3) v = f(v, lane_xor<8>(v));
  if (lph > 2) v = f(v, lane_xor<4>(v));
  v = f(v, lane_xor<2>(v));
  return f(v, lane_xor<1>(v));
}

// x * rsqrt(mean(x^2) + eps) * w over the head's D values; in0, in1: whether the lane's chunks are of them.
__device__ __forceinline__ void rope_norm(float (&x)[2][8], const float *w0, const float *w1, bool in0, bool in1, int lph,
                                          int D, float eps) {
  float sq[2] = {0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) sq[k] = __builtin_fmaf(x[k][j], x[k][j], sq[k]);
  float sum = (in0 ? sq[0] : 0.f) + (in1 ? sq[1] : 0.f);
  sum = over_head(sum, lph, [](float a, float b) { return a + b; });
  const float r = 1.f / sqrtf(sum / (float)D + eps);
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      const float4 w = *(const float4 *)((k ? w1 : w0) + j);
      x[k][j] *= r * w.x, x[k][j + 1] *= r * w.y, x[k][j + 2] *= r * w.z, x[k][j + 3] *= r * w.w;
    }
}

// The lane's eight pairs (HALVES, NEXT).
template <int PAIRS>
__device__ __forceinline__ void rope_turn(float (&x)[2][8], const float (&c)[8], const float (&sv)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float &p = PAIRS == NEXT ? x[j >> 2][(j & 3) * 2] : x[0][j], &q = PAIRS == NEXT ? x[j >> 2][(j & 3) * 2 + 1] : x[1][j];
    const float v = p;
    p = v * c[j] - q * sv[j], q = v * sv[j] + q * c[j];
  }
}

// Pairs that meet through LDS (ACROSS): `mine` the head's 16 << lph values there; a head's lanes are lanes of one wave: no
// barrier.
__device__ __forceinline__ void rope_turn_across(float (&x)[2][8], float *mine, int l, int half, bool next, const float *cs,
                                                 const float *sn) {
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int j = 0; j < 8; j += 4) *(float4 *)&mine[(2 * l + k) * 8 + j] = *(float4 *)&x[k][j];
  asm volatile("" : "+s"(half));  // (else the sixteen conditions below are held as masks through the caller's loop)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = (2 * l + k) * 8 + j;
      if (d >= 2 * half) continue;
      const bool first = next ? j % 2 == 0 : d < half;
      const int i = next ? d / 2 : first ? d : d - half;
      const float other = mine[next ? d ^ 1 : first ? d + half : i];
      x[k][j] = first ? x[k][j] * cs[i] - other * sn[i] : other * sn[i] + x[k][j] * cs[i];
    }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Part `block % parts` of the heads (of the first `sets` sets) of token `block / parts`.  lph: log2 of a head's lanes; a wave takes heads of one set
// only.  LDS, 16-byte aligned: cs and sn 128 values each, norm ROPE_MAX_SETS rows, swap (ACROSS) 16 a thread.
template <int PAIRS, bool IN_F32, bool OUT_F32>
__device__ __forceinline__ void rope_heads(const RopeArgs &a, int sets, int lph, int parts, unsigned block, float *cs,
                                           float *sn, float (*norm)[256], float *swap) {
  constexpr int WAVES = ROPE_THREADS / 64;
  constexpr int TURNS = IN_F32 || PAIRS == ACROSS ? 1 : 2;  // loads of so many heads in flight per lane
  const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l = tid & ((1 << lph) - 1), g = (tid & 63) >> lph, hpw = 64 >> lph;
  const int t = (int)(block / parts), part = (int)block - t * parts;
  // the lane's two chunks of eight values: both sides of eight pairs, or neighbours
  const bool turned = PAIRS != ACROSS && l < a.half / 8;
  const int d0 = (PAIRS == HALVES && turned ? l : 2 * l) * 8, d1 = PAIRS == HALVES && turned ? d0 + a.half : d0 + 8;
  const bool in0 = d0 < a.D, in1 = d1 < a.D;

  // wave item i -> its set, its first head there
  auto which = [&](int &i) __attribute__((always_inline)) -> int {
    int set = 0, n;
    while (set < sets && i >= (n = (a.set[set].heads + hpw - 1) >> (6 - lph))) i -= n, ++set;
    i *= hpw;
    return set;
  };
  Eight<IN_F32> raw[TURNS][2];
  auto fetch = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
      int h = i0 + u * parts * WAVES;
      const int set = which(h);
      if (set == sets) break;
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
    if (i < sets && a.set[i].norm && tid < a.D)
      nw[i] = a.set[i].norm_f32 ? ((const float *)a.set[i].norm)[tid]
                                : __uint_as_float((uint32_t)((const uint16_t *)a.set[i].norm)[tid] << 16);
  }
  fetch(i0);

  if (tid < a.half) {
    float s, c;
    rope_angle(pos, freq, s, c);
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
      if (set == sets) return;
      const RopeHeads &s = a.set[set];
      const bool on = h + g < s.heads;
      float x[2][8];
#pragma unroll
      for (int k = 0; k < 2; ++k) widen<IN_F32>(raw[u][k], x[k]);
      if (s.norm) rope_norm(x, &norm[set][d0 & 255], &norm[set][d1 & 255], in0, in1, lph, a.D, a.eps);
      if (PAIRS != ACROSS && s.rotate && turned) rope_turn<PAIRS>(x, c, sv);
      if (PAIRS == ACROSS && s.rotate) rope_turn_across(x, swap + (tid >> lph << lph) * 16, l, a.half, a.interleaved, cs, sn);
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

// Workgroups of a token: several where there are few tokens.  0: no heads.
inline int64_t rope_parts(const RopeArgs &a, int sets, int lph) {
  int64_t items = 0;  // of a wave
  for (int i = 0; i < sets; ++i) items += (a.set[i].heads + (64 >> lph) - 1) >> (6 - lph);
  const int64_t turns = (items + ROPE_THREADS / 64 - 1) / (ROPE_THREADS / 64);
  int64_t parts = 1024 / a.T;
  return parts < 1 && turns ? 1 : parts > turns ? turns : parts;
}

// Tokens of a launch at most: a grid's lanes are counted in 32 bits (past that the count wraps, with no error).
constexpr int ROPE_TOKENS = 1 << 23;
static_assert((int64_t)ROPE_TOKENS * ROPE_THREADS < (int64_t)1 << 32, "lanes of a grid");

}  // namespace qmm
