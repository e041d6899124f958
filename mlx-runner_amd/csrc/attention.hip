// Attention of the requests' new tokens over their pages: request r's tokens are rows
// [q_starts[r], q_starts[r + 1]) of q, its keys positions 0 .. kv_lens[r] - 1, the new tokens
// the last of them.  Token i of n is at position p = kv_len - n + i and sees the keys j with
// j <= p, and j > p - window where there is one:
//
//   o = sum_j softmax_j(scale q . k_j) v_j  (zero where nothing is seen), times sigmoid(gate)
//
// Here: which kernels run, their workspace, and the joining of the partial sums of tiles that
// several workgroups shared:  M = max_p m_p,  o = sum_p 2^(m_p - M) acc_p / sum_p 2^(m_p - M) l_p.
#include "attention.h"

namespace qmm {

namespace {

constexpr int AC_MOST = 1024;  // workgroups of a launch, so partials of a tile

// One workgroup per tile and row: the waves take the partials in turn.
template <int DP>
__global__ __launch_bounds__(ATTN_THREADS) void attn_join_kernel(const AttnArgs a, const AttnShare s, int tr) {
  constexpr int LPR = DP / 4;                // lanes of a row, four values each
  constexpr int SETS = ATTN_THREADS / LPR;   // partials in flight
  __shared__ float wt[AC_MOST], red[8];
  __shared__ __attribute__((aligned(16))) float part[SETS][DP];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tiles = s.count[0];
  if ((int64_t)blockIdx.x >= (int64_t)tiles * a.Hkv) return;
  const int *d = s.desc + (int64_t)blockIdx.x * 8;
  const int g0 = d[0], row = blockIdx.y;
  if (g0 < 0 || row >= d[4]) return;
  const int np = d[1] - g0 + 1;
  auto place = [&](int p) -> int64_t { return (int64_t)((g0 + p) * 2 + (p == 0)) * tr + row; };
  float top = -__builtin_inff();
  for (int p = tid; p < np; p += ATTN_THREADS) top = fmaxf(top, s.ml[place(p) * 2]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  if (lane == 0) red[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  float sum = 0.f;
  for (int p = tid; p < np; p += ATTN_THREADS) {
    const float2 ml = *(const float2 *)(s.ml + place(p) * 2);
    const float f = ml.x == -__builtin_inff() ? 0.f : attn_exp2(ml.x - top);
    wt[p] = f;
    sum += f * ml.y;
  }
  sum = wave_sum(sum);
  if (lane == 0) red[4 + wave] = sum;
  __syncthreads();
  sum = red[4] + red[5] + red[6] + red[7];
  const int set = tid / LPR, d0 = tid % LPR * 4;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (d0 < a.D) {
#pragma unroll 8
    for (int p = set; p < np; p += SETS) {
      const float4 x = *(const float4 *)(s.acc + place(p) * DP + d0);
      const float f = wt[p];
      o.x += f * x.x, o.y += f * x.y, o.z += f * x.z, o.w += f * x.w;
    }
  }
  *(float4 *)&part[set][d0] = o;
  __syncthreads();
  if (tid * 8 < a.D) {
    float v[8];
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = 0.f;
#pragma unroll
      for (int i = 0; i < SETS; ++i) v[e] += part[i][tid * 8 + e];
      v[e] *= inv;
    }
    attn_store8(a, d[2], d[3] + row, (int)(blockIdx.x / tiles), a.Hq / a.Hkv, tid * 8, v);
  }
}

struct Route {
  int DP, g, tr, grid;
  int64_t tiles;  // at most, per head
  size_t desc, ml, acc, bytes;
};

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

Route route_of(const AttnArgs &a) {
  Route r;
  r.DP = a.D <= 64 ? 64 : a.D <= 128 ? 128 : 256;
  r.g = a.Hq / a.Hkv;
  r.tr = a.T <= a.R && r.g <= 16 ? 16 : 32;
  const int cus = device_cu_count();
  r.grid = 2 * (cus > 0 ? cus : 256) / 8 * 8;
  if (r.grid > AC_MOST) r.grid = AC_MOST;
  r.tiles = (int64_t)a.T * r.g / r.tr + a.R;
  r.desc = 256;
  r.ml = r.desc + up256((size_t)r.tiles * a.Hkv * 32);
  r.acc = r.ml + up256((size_t)r.grid * 2 * r.tr * 8);
  r.bytes = r.acc + (size_t)r.grid * 2 * r.tr * r.DP * 4;
  return r;
}

}  // namespace

size_t attention_workspace(const AttnArgs &a) { return route_of(a).bytes; }

hipError_t launch_attention(const AttnArgs &a, void *workspace, hipStream_t st) {
  if (a.R == 0 || a.W == 0 || a.NB == 0)  // no keys at all
    return launch_fill_zero(a.o, (size_t)a.T * a.Hq * a.D * 2, st);
  const Route r = route_of(a);
  if (r.tiles * a.Hkv > INT32_MAX) return hipErrorInvalidValue;
  AttnShare s;
  s.min_rows = 0, s.max_rows = INT32_MAX, s.first = 1;
  s.count = (int *)workspace;
  s.desc = (int *)((char *)workspace + r.desc);
  s.ml = (float *)((char *)workspace + r.ml);
  s.acc = (float *)((char *)workspace + r.acc);
  hipError_t e = launch_attn_rows(a, s, r.DP, r.tr, r.grid, st);
  if (e != hipSuccess) return e;
  const dim3 grid((unsigned)(r.tiles * a.Hkv), (unsigned)r.tr), block(ATTN_THREADS);
  if (r.DP == 64)
    hipLaunchKernelGGL((attn_join_kernel<64>), grid, block, 0, st, a, s, r.tr);
  else if (r.DP == 128)
    hipLaunchKernelGGL((attn_join_kernel<128>), grid, block, 0, st, a, s, r.tr);
  else
    hipLaunchKernelGGL((attn_join_kernel<256>), grid, block, 0, st, a, s, r.tr);
  return hipGetLastError();
}

}  // namespace qmm
