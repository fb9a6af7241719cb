// Selection of the pages that a decoded token attends to.  Every page carries the channel minima and maxima of its keys;
// with u the sum of the KV group's query heads, sum_d max(u_d min_d, u_d max_d) bounds from above what any key of the page
// scores on the group's average.  The pages with the highest bounds are taken, ties to the lowest page; sums are in fp64,
// so that the choice is the definition's.
#pragma once
#include "paged_cache.cuh"

namespace sq {

struct PagedSelectParams {
  PagedPool pool;
  BlockTable table;
  const uint8_t* q;
  long long q_sb, q_sh;
  const int* kv_lens;
  int batch, groups;
  int budget, sink_pages, recent_pages;
  unsigned long long* keys;  // [B, Hkv, max_pages] ordered scores
  int* out;                  // [B, Hkv, budget]
};

// order-preserving map of a double to an unsigned integer; NaN becomes the lowest value, one above "no page" (0)
__device__ __forceinline__ unsigned long long ordered_key(double x) {
  if (!(x == x)) return 1ull;
  const long long b = __double_as_longlong(x == 0.0 ? 0.0 : x);
  return static_cast<unsigned long long>(b < 0 ? ~b : (b | static_cast<long long>(0x8000000000000000ull)));
}

__device__ __forceinline__ int held_pages(const PagedSelectParams& p, int b) {
  const long long len = max(p.kv_lens[b], 0);
  const long long n = (len + (1 << p.pool.ps_shift) - 1) >> p.pool.ps_shift;
  return static_cast<int>(min(n, static_cast<long long>(p.table.max_pages)));
}

template <int D, bool BF16>
__global__ void __launch_bounds__(256) paged_score_kernel(const __grid_constant__ PagedSelectParams p) {
  __shared__ double u[D];
  const int h = blockIdx.y, b = blockIdx.z;
  if (threadIdx.x < D) {
    double s = 0.0;
    for (int g = 0; g < p.groups; ++g)
      s += static_cast<double>(to_f32<BF16>(*reinterpret_cast<const uint16_t*>(p.q + 2 * (b * p.q_sb + (h * p.groups + g) * p.q_sh + threadIdx.x))));
    u[threadIdx.x] = s;
  }
  __syncthreads();
  const int held = held_pages(p, b);
  for (int i = blockIdx.x * 256 + threadIdx.x; i < p.table.max_pages; i += 256 * gridDim.x) {
    unsigned long long key = 0ull;
    if (i < held) {
      if (i < p.sink_pages || i >= held - p.recent_pages) {
        key = ~0ull;
      } else {
        const int page = page_of(p.table, b, i, p.pool.num_pages);
        if (page >= 0) {
          const uint16_t* lo = reinterpret_cast<const uint16_t*>(p.pool.k_bounds) + (static_cast<long long>(page) * p.pool.hkv + h) * 2 * D;
          double s = 0.0;
          for (int d = 0; d < D; ++d) {
            const double a = u[d] * static_cast<double>(to_f32<BF16>(lo[d])), c = u[d] * static_cast<double>(to_f32<BF16>(lo[D + d]));
            s += (a != a || a > c) ? a : c;
          }
          key = ordered_key(s);
        }
      }
    }
    p.keys[(static_cast<long long>(b) * p.pool.hkv + h) * p.table.max_pages + i] = key;
  }
}

// One CTA per (KV head, sequence): a page is taken if fewer than `budget` come before it; the list is ascending.
__global__ void __launch_bounds__(1024) paged_pick_kernel(const __grid_constant__ PagedSelectParams p) {
  __shared__ int base, warp_sum[32];
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned long long* keys = p.keys + (static_cast<long long>(b) * p.pool.hkv + h) * p.table.max_pages;
  int* out = p.out + (static_cast<long long>(b) * p.pool.hkv + h) * p.budget;
  const int held = held_pages(p, b);
  if (threadIdx.x == 0) base = 0;
  __syncthreads();
  for (int i0 = 0; i0 < held; i0 += 1024) {
    const int i = i0 + threadIdx.x;
    bool take = false;
    if (i < held) {
      const unsigned long long mine = keys[i];
      int before = 0;
      for (int j = 0; j < held; ++j) before += keys[j] > mine || (keys[j] == mine && j < i);
      take = before < p.budget;
    }
    const unsigned votes = __ballot_sync(0xffffffffu, take);
    if (lane == 0) warp_sum[warp] = __popc(votes);
    __syncthreads();
    int at = base + __popc(votes & ((1u << lane) - 1u));
    for (int w = 0; w < warp; ++w) at += warp_sum[w];
    if (take) out[at] = i;
    __syncthreads();
    if (threadIdx.x == 1023) base = at + take;
    __syncthreads();
  }
  for (int i = base + threadIdx.x; i < p.budget; i += 1024) out[i] = -1;
}

}  // namespace sq
