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

// Over the wave's lanes, in all of them.
__device__ __forceinline__ float wave_top(float x) {
#define QMM_STEP(ctrl, rows)                                                                                    \
  x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), ctrl, rows, 0xF, false)))
  QMM_STEP(0x111, 0xF);  // row_shr:1, 2, 4, 8; row_bcast:15, 31 (as attn_wave_scan)
  QMM_STEP(0x112, 0xF);
  QMM_STEP(0x114, 0xF);
  QMM_STEP(0x118, 0xF);
  QMM_STEP(0x142, 0xA);
  QMM_STEP(0x143, 0xC);
#undef QMM_STEP
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
__device__ __forceinline__ float wave_total(float x) {
#define QMM_STEP(ctrl, rows) \
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, rows, 0xF, false))
  QMM_STEP(0x111, 0xF);
  QMM_STEP(0x112, 0xF);
  QMM_STEP(0x114, 0xF);
  QMM_STEP(0x118, 0xF);
  QMM_STEP(0x142, 0xA);
  QMM_STEP(0x143, 0xC);
#undef QMM_STEP
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// The tile that a workgroup joins; none: first < 0.  (Its entry is read beside the count that says whether there is one.)
struct Cut {
  int first, last, q0, row0, rows, head;
};
__device__ __forceinline__ Cut cut_of(const AttnArgs &a, const AttnShare &s) {
  const int4 x = *(const int4 *)(s.desc + (int64_t)blockIdx.x * 8);
  const int2 y = *(const int2 *)(s.desc + (int64_t)blockIdx.x * 8 + 4);
  const int2 n = *(const int2 *)s.count;
  Cut c{x.x, x.y, x.z, x.w, y.x, y.y};
  if ((int64_t)blockIdx.x >= (s.by_tile ? (int64_t)n.x * a.Hkv : (int64_t)n.y)) c.first = -1;
  return c;
}

// A part's weight beside the largest of its row: 0 where it has no keys of the row (and no sums), -1 where f32 has no weight
// for it.
__device__ __forceinline__ float part_weight(float m, float top) {
  const float f = attn_exp2(m - top);
  return m == -__builtin_inff() ? 0.f : f == 0.f ? -1.f : f;
}
__device__ __forceinline__ void part_add(float4 &o, float f, float4 v) {
  if (f > 0.f) o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
}
// Of a part without weight, only what is not finite: it reaches the row, whatever the scores, as it does within a part.
__device__ __forceinline__ void part_add_odd(float4 &o, float f, float4 v) {
  auto odd = [f](float x) { return f < 0.f && x * 0.f != 0.f ? x : 0.f; };
  o.x += odd(v.x), o.y += odd(v.y), o.z += odd(v.z), o.w += odd(v.w);
}

// One workgroup per tile, row and COLS columns.  All that it reads is asked for at once, up to 8 partials a lane; every
// wave works out the partials' weights for itself.  MORE: tiles may have more rows than the grid, so a workgroup goes on to
// every gridDim.y-th (what the compiler forms ahead of such a loop costs 0.2 us where there is one row for each).
// Latency: 2.4-5 us, of which 2 are a launch's.
template <int DP, int COLS, bool MORE>
__global__ __launch_bounds__(ATTN_THREADS) void attn_join_kernel(const AttnArgs a, const AttnShare s, int tr) {
  constexpr int LPR = COLS / 4;              // lanes of a row, four values each
  constexpr int SETS = ATTN_THREADS / LPR;   // partials side by side
  constexpr int HELD = 4, AHEAD = 8;
  __shared__ float wt[ATTN_THREADS / 64][AC_MOST];
  __shared__ __attribute__((aligned(16))) float part[SETS][COLS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Cut c = cut_of(a, s);
  int row = blockIdx.y;
  if (c.first < 0 || row >= c.rows) return;
  const int np = c.last - c.first + 1;
  auto place = [&](int p) -> int64_t { return (int64_t)((c.first + p) * 2 + (p == 0)) * tr + row; };
  const int set = tid / LPR, d0 = blockIdx.z * COLS + tid % LPR * 4, col = blockIdx.z * COLS + tid;
  const bool in = d0 < a.D, out = tid < COLS && col < a.D;
#pragma unroll 1
  do {
    float2 ml[HELD];
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      ml[k] = make_float2(-__builtin_inff(), 0.f);
      if (k * 64 + lane < np) ml[k] = *(const float2 *)(s.ml + place(k * 64 + lane) * 2);
    }
    float4 x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (set + i * SETS < np && in) x[i] = *(const float4 *)(s.acc + place(set + i * SETS) * DP + d0);
    const int64_t orow = attn_row(a, c.q0, c.row0 + row, c.head);
    uint32_t gate = 0;
    if (a.gate && out) gate = a.gate[orow * a.Dg + (a.Dg - a.D) + col];

    float top = ml[0].x, sum = 0.f;
#pragma unroll
    for (int k = 1; k < HELD; ++k) top = fmaxf(top, ml[k].x);
    for (int p = HELD * 64 + lane; p < np; p += 64) top = fmaxf(top, s.ml[place(p) * 2]);
    top = wave_top(top);
    bool weightless = false;
    auto weigh = [&](int p, float2 v) __attribute__((always_inline)) {
      const float f = part_weight(v.x, top);
      wt[wave][p] = f;
      weightless |= f < 0.f;
      sum += fmaxf(f, 0.f) * v.y;
    };
#pragma unroll
    for (int k = 0; k < HELD; ++k)
      if (k * 64 + lane < np) weigh(k * 64 + lane, ml[k]);
    for (int p = HELD * 64 + lane; p < np; p += 64) weigh(p, *(const float2 *)(s.ml + place(p) * 2));
    sum = wave_total(sum);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (set + i * SETS < np && in) part_add(o, wt[wave][set + i * SETS], x[i]);
#pragma unroll 8
    for (int p = set + AHEAD * SETS; p < np; p += SETS)
      if (in) part_add(o, wt[wave][p], *(const float4 *)(s.acc + place(p) * DP + d0));
    if (__any(weightless)) {
#pragma unroll 1
      for (int p = set; p < np; p += SETS)
        if (in) part_add_odd(o, wt[wave][p], *(const float4 *)(s.acc + place(p) * DP + d0));
    }
    *(float4 *)&part[set][tid % LPR * 4] = o;
    __syncthreads();
    if (out) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < SETS; ++i) v += part[i][tid];
      v *= sum != 0.f ? 1.f / sum : 0.f;
      if (a.gate) v *= __builtin_amdgcn_rcpf(1.f + attn_exp2(-1.44269504088896341f * __uint_as_float(gate << 16)));
      a.o[orow * a.D + col] = __builtin_bit_cast(uint16_t, (__bf16)v);
    }
    if (MORE) __syncthreads();  // (part is read)
    row += gridDim.y;
  } while (MORE && row < c.rows);
}

// Tiles of many rows, mostly cut in few parts: 16 rows per workgroup, their weights while the first parts are on their way.
// Bound by the reads: 134 MB of partials (2048 tokens of 24 heads of 256, all tiles cut) in 30-37 us, 3.6-4.5 TB/s.
constexpr int AJ_ROWS = 16;
template <int DP>
__global__ __launch_bounds__(ATTN_THREADS) void attn_join_rows_kernel(const AttnArgs a, const AttnShare s, int tr) {
  constexpr int LPR = DP / 4, RP = ATTN_THREADS / LPR, TURNS = AJ_ROWS / RP, AHEAD = 2;
  __shared__ float wt[AJ_ROWS][AC_MOST / 2], total[AJ_ROWS];
  __shared__ int odd[ATTN_THREADS / 64];  // whether a wave's rows have parts without weight
  __shared__ __attribute__((aligned(16))) float part[AJ_ROWS][DP];
  const int tid = threadIdx.x;
  const Cut c = cut_of(a, s);
  const int row0 = blockIdx.y * AJ_ROWS, rows = c.rows;
  if (c.first < 0 || row0 >= rows) return;
  const int np = c.last - c.first + 1;
  auto place = [&](int p, int row) -> int64_t { return (int64_t)((c.first + p) * 2 + (p == 0)) * tr + row0 + row; };
  const int r0 = tid / LPR, d0 = tid % LPR * 4;
  const int row = tid >> 4, l = tid & 15;
  const bool on = row0 + row < rows;
  float2 ml = make_float2(-__builtin_inff(), 0.f);
  if (l < np && on) ml = *(const float2 *)(s.ml + place(l, row) * 2);
  float4 x[AHEAD][TURNS];
#pragma unroll
  for (int p = 0; p < AHEAD; ++p)
#pragma unroll
    for (int t = 0; t < TURNS; ++t)
      if (p < np && row0 + t * RP + r0 < rows && d0 < a.D) x[p][t] = *(const float4 *)(s.acc + place(p, t * RP + r0) * DP + d0);
  {
    float top = ml.x, sum = 0.f;
    bool weightless = false;
    for (int p = l + 16; p < np && on; p += 16) top = fmaxf(top, s.ml[place(p, row) * 2]);
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 16));
    for (int p = l; p < np && on; p += 16) {
      if (p >= 16) ml = *(const float2 *)(s.ml + place(p, row) * 2);
      const float f = part_weight(ml.x, top);
      wt[row][p] = f;
      weightless |= f < 0.f;
      sum += fmaxf(f, 0.f) * ml.y;
    }
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 16);
    if (l == 0) total[row] = sum;
    weightless = __any(weightless);
    if ((tid & 63) == 0) odd[tid >> 6] = weightless;
  }
  __syncthreads();
  float4 o[TURNS];
#pragma unroll
  for (int t = 0; t < TURNS; ++t) o[t] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int p = 0; p < AHEAD; ++p)
#pragma unroll
    for (int t = 0; t < TURNS; ++t)
      if (p < np && row0 + t * RP + r0 < rows && d0 < a.D) part_add(o[t], wt[t * RP + r0][p], x[p][t]);
#pragma unroll 1
  for (int p = AHEAD; p < np; ++p) {
#pragma unroll
    for (int t = 0; t < TURNS; ++t)
      if (row0 + t * RP + r0 < rows && d0 < a.D) x[0][t] = *(const float4 *)(s.acc + place(p, t * RP + r0) * DP + d0);
#pragma unroll
    for (int t = 0; t < TURNS; ++t)
      if (row0 + t * RP + r0 < rows && d0 < a.D) part_add(o[t], wt[t * RP + r0][p], x[0][t]);
  }
  int any = 0;
#pragma unroll
  for (int w = 0; w < ATTN_THREADS / 64; ++w) any |= odd[w];
  if (any) {
#pragma unroll 1
    for (int p = 0; p < np; ++p)
#pragma unroll
      for (int t = 0; t < TURNS; ++t)
        if (row0 + t * RP + r0 < rows && d0 < a.D)
          part_add_odd(o[t], wt[t * RP + r0][p], *(const float4 *)(s.acc + place(p, t * RP + r0) * DP + d0));
  }
#pragma unroll
  for (int t = 0; t < TURNS; ++t) *(float4 *)&part[t * RP + r0][d0] = o[t];
  __syncthreads();
  for (int i = tid; i < AJ_ROWS * (a.D / 8); i += ATTN_THREADS) {
    const int row = i / (a.D / 8), c0 = i % (a.D / 8) * 8;
    if (row0 + row >= rows) break;
    const float inv = total[row] != 0.f ? 1.f / total[row] : 0.f;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = part[row][c0 + e] * inv;
    attn_store8(a, attn_row(a, c.q0, c.row0 + row0 + row, c.head), c0, v);
  }
}

// The kernels of a call: requests of up to 32 rows per key head (tokens x query heads that share
// it) on the kernel that streams, the others on the one for many rows.  Lengths are known on the
// GPU only, so both are launched where both kinds can be expected (a launch without work: 3-5 us); where
// shapes say that no request has over 256 rows, if each has a token, the streaming kernel takes
// them all, 16 or 32 at a time.  That is a guess for speed only (a request may have none of the tokens and
// another all of them): every kernel takes requests of any lengths.  Without the guess every decode step of many
// requests would launch the second kernel and its join (7 us beside 77); with it, 512 tokens in one of 512
// slots take 58 us, 55 on the kernel for chunks (24 heads on 4 of 256).
constexpr int ROWS_MOST = 32;

struct Part {
  int tr = 0, grid = 0, min_rows = 0, max_rows = 0;
  int rows = 0;       // of a tile, for the joining launch's grid
  bool more = false;  // a tile may have more, up to tr
  int by_tile = 0;
  int64_t tiles = 0;  // at most, per head
  size_t at = 0, desc = 0, ml = 0, acc = 0;
};
struct Route {
  int DP, g;
  Part rows, chunk;  // (tr 0: not launched)
  size_t bytes;
};

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

size_t lay_out(Part &p, const AttnArgs &a, int DP, int g, size_t at) {
  p.tiles = p.max_rows <= p.tr ? a.R : (int64_t)a.T * g / p.tr + a.R;
  p.by_tile = p.tiles * a.Hkv <= p.grid;
  p.at = at;
  p.desc = at + 256;
  p.ml = p.desc + up256((size_t)(p.by_tile ? p.tiles * a.Hkv : p.grid) * 32);
  p.acc = p.ml + up256((size_t)p.grid * 2 * p.tr * 8);
  return p.acc + (size_t)p.grid * 2 * p.tr * DP * 4;
}

Route route_of(const AttnArgs &a) {
  Route r;
  r.DP = a.D <= 64 ? 64 : a.D <= 128 ? 128 : 256;
  r.g = a.Hq / a.Hkv;
  int cus = device_cu_count();
  cus = (cus > 0 ? cus : 256) / 8 * 8;
  cus = cus < 8 ? 8 : cus < AC_MOST / 2 ? cus : AC_MOST / 2;
  // (most: the rows of the longest request, if each has a token)
  const int64_t most = (int64_t)(a.T > a.R ? a.T - a.R + 1 : 1) * r.g;
  const bool few = most <= 8 * ROWS_MOST;
  const bool one = a.R == 1 && (int64_t)a.T * r.g > ROWS_MOST;
  if (!one) {
    r.rows.tr = most <= 16 ? 16 : 32;
    // (E4M3 pages of up to 128 values: a CU holds three workgroups, with tiles of 4 KB a wave.  Two with 8 KB, and three, when
    // scores still came from the scaled MFMA (64 requests of 1 to 8192 keys 38.0 us then, 37.0 now): 16 heads of 64, 64 requests of 300 keys 23.4 and 20.1 us, 3000 keys 48.9 and 51.2; 32 heads on 8 of 128, one request of 300
    // keys 12.8 and 11.5, 128 of them 32.7 and 26.5, 64 of 3000 53.3 and 53.8; 12 heads of 96 16 of 3000 28.2 and 24.7)
    r.rows.grid = a.k_scales && r.DP <= 128 ? 3 * cus < AC_MOST ? 3 * cus : AC_MOST : 2 * cus;
    r.rows.min_rows = 0, r.rows.max_rows = few ? INT32_MAX : ROWS_MOST;
    // (one token each, as when decoding, is the common case of T <= R; 16 rows for 6 would be 10 empty workgroups a tile)
    const bool each = a.R > 1 && a.T <= a.R;
    const int64_t rows = each ? r.g : (int64_t)a.T * r.g;
    r.rows.rows = (int)(rows < r.rows.tr ? rows : r.rows.tr);
    r.rows.more = each && r.rows.rows < r.rows.tr;
  }
  if (one || !few) {
    r.chunk.tr = r.chunk.rows = 256;
    r.chunk.grid = r.DP == 64 ? 2 * cus : cus;
    r.chunk.min_rows = one ? 0 : ROWS_MOST, r.chunk.max_rows = INT32_MAX;
  }
  r.bytes = 0;
  if (r.rows.tr) r.bytes = up256(lay_out(r.rows, a, r.DP, r.g, r.bytes));
  if (r.chunk.tr) r.bytes = lay_out(r.chunk, a, r.DP, r.g, r.bytes);
  return r;
}

AttnShare share_of(const Part &p, void *workspace) {
  char *w = (char *)workspace;
  AttnShare s;
  s.min_rows = p.min_rows, s.max_rows = p.max_rows, s.first = 0;
  s.by_tile = p.by_tile, s.tiles = (int)p.tiles;
  s.count = (int *)(w + p.at), s.desc = (int *)(w + p.desc);
  s.ml = (float *)(w + p.ml), s.acc = (float *)(w + p.acc);
  return s;
}

template <int DP, int COLS>
void join_few(const AttnArgs &a, const Part &p, const AttnShare &s, unsigned n, hipStream_t st) {
  const dim3 grid(n, p.rows, DP / COLS), block(ATTN_THREADS);
  if (p.more)
    hipLaunchKernelGGL((attn_join_kernel<DP, COLS, true>), grid, block, 0, st, a, s, p.tr);
  else
    hipLaunchKernelGGL((attn_join_kernel<DP, COLS, false>), grid, block, 0, st, a, s, p.tr);
}

template <int DP>
void join(const AttnArgs &a, const Part &p, const AttnShare &s, hipStream_t st) {
  const unsigned n = (unsigned)(p.by_tile ? p.tiles * a.Hkv : p.grid);
  if (p.tr > 32)
    hipLaunchKernelGGL((attn_join_rows_kernel<DP>), dim3(n, p.rows / AJ_ROWS), dim3(ATTN_THREADS), 0, st, a, s, p.tr);
  // A row's columns over several workgroups where that leaves few.  (Over E4M3 pages a tile is cut in more parts for its time,
  // and of 256 columns only four are side by side: 8 requests of 18 rows, up to 32768 keys, 9.0 us on one workgroup a row,
  // 6.9 on four; 64 of 4 rows of 128 columns 4.2 on one, 5.6 on two.)
  else if (DP > 64 && n * (unsigned)p.rows <= (a.k_scales && DP == 256 ? 2048u : 1024u))
    join_few<DP, 64>(a, p, s, n, st);
  else
    join_few<DP, DP>(a, p, s, n, st);
}

}  // namespace

// What of a call passes the kernels' 32-bit counts (NULL: nothing).
const char *attention_limits(const AttnArgs &a) {
  if ((double)a.T * (a.Hq / a.Hkv) > 1 << 27) return "rows per key head";
  const Route r = route_of(a);
  for (const Part *p : {&r.rows, &r.chunk})
    if (p->tr && (double)p->tiles * a.Hkv * ((double)a.W * a.block / 64 + 4) > INT32_MAX) return "keys of all tiles together";
  return nullptr;
}

size_t attention_workspace(const AttnArgs &a) { return route_of(a).bytes; }

hipError_t launch_attention(const AttnArgs &args, void *workspace, hipStream_t st) {
  AttnArgs a = args;
  a.g = a.Hq / a.Hkv;
  a.by_g = fast_div((uint32_t)a.g);
  a.by_block = fast_div((uint32_t)a.block);
  if (a.R == 0 || a.W == 0 || a.NB == 0)  // no keys at all
    return launch_fill_zero(a.o, (size_t)a.T * a.Hq * a.D * 2, st);
  const Route r = route_of(a);
  bool first = true;
  for (const Part *p : {&r.rows, &r.chunk}) {
    if (!p->tr) continue;
    AttnShare s = share_of(*p, workspace);
    s.first = first;
    first = false;
    const hipError_t e = p == &r.rows   ? launch_attn_rows(a, s, r.DP, p->tr, p->grid, st)
                         : a.k_scales ? launch_attn_chunk8(a, s, r.DP, p->grid, st)
                                      : launch_attn_chunk(a, s, r.DP, p->grid, st);
    if (e != hipSuccess) return e;
    r.DP == 64 ? join<64>(a, *p, s, st) : r.DP == 128 ? join<128>(a, *p, s, st) : join<256>(a, *p, s, st);
  }
  return hipGetLastError();
}

}  // namespace qmm
