// Attention of the requests' new tokens over their pages: request r's tokens are rows
// [q_starts[r], q_starts[r + 1]) of q, its keys positions 0 .. kv_lens[r] - 1, the new tokens
// the last of them.  Token i of n is at position p = kv_len - n + i and sees the keys j with
// j <= p, and j > p - window where there is one:
//
//   o = sum_j softmax_j(scale q . k_j) v_j  (zero where nothing is seen), times sigmoid(gate)
#include "qmm_device.h"
#include "qmm_launch.h"

namespace qmm {

namespace {

// One wave per token and query head: a running maximum and sum over the keys, four values of
// the head per lane.
__global__ __launch_bounds__(64) void attention_simple_kernel(const AttnArgs a) {
  const int t = blockIdx.x / a.Hq, hq = blockIdx.x - t * a.Hq, h = hq / (a.Hq / a.Hkv), lane = threadIdx.x;
  int r = -1, q0 = 0, q1 = 0;
  for (int i = 0; i < a.R; ++i)
    if (a.q_starts[i] <= t && t < a.q_starts[i + 1]) r = i, q0 = a.q_starts[i], q1 = a.q_starts[i + 1];
  const int64_t row = (int64_t)t * a.Hq + hq;
  const int d0 = lane * 4;
  float q[4] = {0.f, 0.f, 0.f, 0.f}, o[4] = {0.f, 0.f, 0.f, 0.f};
  if (d0 < a.D)
    for (int j = 0; j < 4; ++j) q[j] = bf16_to_f32(a.q[row * a.D + d0 + j]) * a.scale;
  float m = -__builtin_inff(), l = 0.f;
  if (r >= 0) {
    const int pos = a.kv_lens[r] - (q1 - q0) + (t - q0);
    int64_t end = (int64_t)pos + 1;
    if (end > (int64_t)a.W * a.block) end = (int64_t)a.W * a.block;
    int j0 = a.window > 0 ? pos - a.window + 1 : 0;
    for (int64_t j = j0 < 0 ? 0 : j0; j < end; ++j) {
      const int b = a.table[(int64_t)r * a.W + j / a.block];
      if (b < 0 || b >= a.NB) continue;
      const int64_t at = (((int64_t)b * a.Hkv + h) * a.block + j % a.block) * a.D + d0;
      float s = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
      if (d0 < a.D)
        for (int e = 0; e < 4; ++e) s += q[e] * bf16_to_f32(a.k[at + e]), v[e] = bf16_to_f32(a.v[at + e]);
      s = wave_sum(s);
      if (s == -__builtin_inff()) continue;
      const float mn = fmaxf(m, s), f = expf(m - mn), p = expf(s - mn);
      m = mn;
      l = l * f + p;
      for (int e = 0; e < 4; ++e) o[e] = o[e] * f + p * v[e];
    }
  }
  if (d0 < a.D)
    for (int e = 0; e < 4; ++e) {
      float y = l > 0.f ? o[e] / l : 0.f;
      if (a.gate) y /= 1.f + expf(-bf16_to_f32(a.gate[row * a.Dg + a.Dg - a.D + d0 + e]));
      a.o[row * a.D + d0 + e] = f32_to_bf16_rne(y);
    }
}

}  // namespace

size_t attention_workspace(const AttnArgs &) { return 0; }

hipError_t launch_attention(const AttnArgs &a, void *, hipStream_t st) {
  const int64_t grid = (int64_t)a.T * a.Hq;
  if (grid > INT32_MAX) return hipErrorInvalidValue;
  hipLaunchKernelGGL(attention_simple_kernel, dim3((unsigned)grid), dim3(64), 0, st, a);
  return hipGetLastError();
}

}  // namespace qmm
