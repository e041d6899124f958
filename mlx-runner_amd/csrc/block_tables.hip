// Block tables, slots and positions of a step's tokens, built on the GPU from the requests'
// lengths.  With c_r tokens cached and n_r new ones of request r, pages of `block` tokens, a
// table [R, W] and free pages free[head], free[head + 1], ...:
//
//   q_0 = 0, q_(r+1) = min(q_r + n_r, T);  kv_r = c_r + q_(r+1) - q_r
//   o_r = min(ceil(c_r / block), W),  w_r = min(ceil(kv_r / block), W)
//   f_r = head + sum_{s < r} (w_s - o_s)
//   table[r, p] = free[f_r + p - o_r] for o_r <= p < w_r (-1 past the list's end)
//   positions[t] = c_r + t - q_r;  slots[t] = table[r, pos / block] * block + pos % block
//
// Every workgroup scans the lengths itself (one request per thread and turn) and then takes
// its share of tokens and of requests' pages.  Latency (two scans and three dependent reads): 5.0 us for 64
// decoding requests, 6.8 for 512 with 12 prompts' chunks.  In place, where the lengths are overwritten, one
// workgroup does it all.
#include "qmm_device.h"
#include "qmm_launch.h"

namespace qmm {

namespace {

constexpr int BT_THREADS = 1024;
constexpr int BT_WAVES = BT_THREADS / 64;

__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b, uint32_t most) {
  const uint32_t s = a + b;  // (each at most 2^31 - 1)
  return s < most ? s : most;
}

// Inclusive scan over the workgroup of sums held at `most` (such sums associate); the total too.
__device__ __forceinline__ uint32_t scan_sat(uint32_t v, uint32_t most, uint32_t *waves, uint32_t *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t u = __shfl_up(v, off, 64);
    if (lane >= off) v = sat_add(v, u, most);
  }
  __syncthreads();  // (waves' previous readers)
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < BT_WAVES; ++w) {
    if (w == wave) before = all;
    all = sat_add(all, waves[w], most);
  }
  *total = all;
  return sat_add(before, v, most);
}

// (tokens: two int32 added, below 2^32)
__device__ __forceinline__ int pages_of(int64_t tokens, int block, int W) {
  const uint32_t p = tokens ? ((uint32_t)tokens - 1u) / (uint32_t)block + 1u : 0u;
  return p < (uint32_t)W ? (int)p : W;
}

__global__ __launch_bounds__(BT_THREADS) void block_tables_kernel(const BlockTableArgs a) {
  __shared__ int qs[BLOCK_TABLES_MAX_R + 1], cs[BLOCK_TABLES_MAX_R], fs[BLOCK_TABLES_MAX_R];
  __shared__ uint32_t waves[BT_WAVES];
  const int tid = threadIdx.x;
  const bool first = blockIdx.x == 0;
  const int head0 = a.head[0];
  uint32_t tokens = 0, pages = head0 < 0 ? 0u : (uint32_t)head0;
  for (int r0 = 0; r0 < a.R; r0 += BT_THREADS) {
    const int r = r0 + tid;
    int c = 0, n = 0;
    if (r < a.R) {
      c = a.cached[r], n = a.fresh[r];
      c = c < 0 ? 0 : c, n = n < 0 ? 0 : n < a.T ? n : a.T;
    }
    uint32_t all;
    const uint32_t q1 = sat_add(tokens, scan_sat((uint32_t)n, (uint32_t)a.T, waves, &all), (uint32_t)a.T);
    // (a scan held at T and then offset is the offset scan held at T)
    uint32_t q0 = __shfl_up(q1, 1, 64);
    __syncthreads();
    if ((tid & 63) == 63) waves[tid >> 6] = q1;
    __syncthreads();
    if ((tid & 63) == 0) q0 = tid ? waves[(tid >> 6) - 1] : tokens;
    const int got = (int)(q1 - q0);
    const int64_t kv = (int64_t)c + got;
    const int held = pages_of(c, a.block, a.W), need = pages_of(kv, a.block, a.W);
    uint32_t more;
    const uint32_t mine = r < a.R ? (uint32_t)(need - held) : 0u;
    const uint32_t f1 = sat_add(pages, scan_sat(mine, 0x7FFFFFFFu, waves, &more), 0x7FFFFFFFu);
    if (r < a.R) {
      qs[r] = (int)q0, cs[r] = c, fs[r] = (int)(f1 - mine);
      if (first) {
        a.q_starts[r] = (int)q0;
        a.kv_lens[r] = kv < 0x7FFFFFFF ? (int)kv : 0x7FFFFFFF;
      }
    }
    tokens = sat_add(tokens, all, (uint32_t)a.T);
    pages = sat_add(pages, more, 0x7FFFFFFFu);
  }
  if (tid == 0) {
    qs[a.R] = (int)tokens;
    if (first) a.q_starts[a.R] = (int)tokens, a.head_out[0] = (int)pages;
  }
  __syncthreads();

  // tokens: the request by bisection of the starts
  for (int64_t t = (int64_t)blockIdx.x * BT_THREADS + tid; t < a.T; t += (int64_t)gridDim.x * BT_THREADS) {
    int pos = 0, slot = -1;
    if (t < (int64_t)tokens) {
      int lo = 0, hi = a.R;  // the last r with qs[r] <= t and a token of its own
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (qs[mid] <= t)
          lo = mid;
        else
          hi = mid;
      }
      const int64_t at = (int64_t)cs[lo] + (t - qs[lo]);
      pos = at < 0x7FFFFFFF ? (int)at : 0x7FFFFFFF;
      const int64_t p = (uint32_t)at / (uint32_t)a.block;
      if (p < a.W) {
        const int held = pages_of(cs[lo], a.block, a.W);
        int b;
        if (p < held) {
          b = a.table[(int64_t)lo * a.W + p];
        } else {
          const int64_t f = (int64_t)fs[lo] + (p - held);
          b = f < a.F ? a.free_blocks[f] : -1;
        }
        const int64_t s = (int64_t)b * a.block + (at - p * a.block);
        slot = b >= 0 && s <= 0x7FFFFFFF ? (int)s : -1;
      }
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
  }

  // pages: a wave per request; the rest of the row too where the table is another array
  const int lane = tid & 63, nw = gridDim.x * BT_WAVES;
  for (int r = blockIdx.x * BT_WAVES + (tid >> 6); r < a.R; r += nw) {
    const int c = cs[r], held = pages_of(c, a.block, a.W);
    const int need = pages_of((int64_t)c + (qs[r + 1] - qs[r]), a.block, a.W);
    const int64_t row = (int64_t)r * a.W;
    const bool copy = a.table_out != a.table;
    for (int64_t p = (copy ? 0 : held) + lane; p < (copy ? a.W : need); p += 64) {
      int b;
      if (p >= held && p < need) {
        const int64_t f = (int64_t)fs[r] + (p - held);
        b = f < a.F ? a.free_blocks[f] : -1;
      } else {
        b = a.table[row + p];
      }
      a.table_out[row + p] = b;
    }
  }
}

}  // namespace

hipError_t launch_block_tables(const BlockTableArgs &a, hipStream_t st) {
  if (a.R < 0 || a.R > BLOCK_TABLES_MAX_R || a.T < 0 || a.W < 0 || a.F < 0 || a.block < 1) return hipErrorInvalidValue;
  // One workgroup where results overwrite the lengths or the head that others would still read.
  const bool alone = a.head_out == a.head || a.kv_lens == a.cached || a.kv_lens == a.fresh;
  int64_t grid = 1;
  if (!alone) {
    grid = (a.T + BT_THREADS - 1) / BT_THREADS;
    const int64_t by_pages = (a.R + 4 * BT_WAVES - 1) / (4 * BT_WAVES);
    grid = grid > by_pages ? grid : by_pages;
    grid = grid < 1 ? 1 : grid > 256 ? 256 : grid;
  }
  hipLaunchKernelGGL(block_tables_kernel, dim3((unsigned)grid), dim3(BT_THREADS), 0, st, a);
  return hipGetLastError();
}

}  // namespace qmm
