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

constexpr int kScorePages = 4;                                   // pages per lane group, loaded ahead of their use
__host__ __device__ constexpr int score_pages_per_cta(int d) { return 256 / (d / 8) * kScorePages; }

// Sum of x[j] over the LANES lanes of a group for each of the four j; lane c of the group gets the sum of j = c & 3.  Lanes give
// away half of their values at a time, so that four sums take 10 shuffles and not 32.
template <int LANES>
__device__ __forceinline__ double group_sums4(const double (&x)[4], int c) {
  const bool odd = c & 1, high = c & 2;
  double a = odd ? x[1] : x[0], z = odd ? x[3] : x[2];
  a += __shfl_xor_sync(0xffffffffu, odd ? x[0] : x[1], 1);
  z += __shfl_xor_sync(0xffffffffu, odd ? x[2] : x[3], 1);
  double s = high ? z : a;
  s += __shfl_xor_sync(0xffffffffu, high ? a : z, 2);
#pragma unroll
  for (int o = 4; o < LANES; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// D / 8 lanes take a page: 8 channels each, of which a 16-byte load brings the minima and another the maxima.  The larger of
// u min and u max is the product with the bound of u's sign, so a channel costs one DFMA.  Bound by the bounds' bytes (512 a
// page and KV head at D = 128) and the latency of three dependent loads, so a CTA goes over several groups of pages and has
// the next ones in flight.
template <int D, bool BF16>
__global__ void __launch_bounds__(256, 3) paged_score_kernel(const __grid_constant__ PagedSelectParams p) {
  constexpr int kLanes = D / 8, kGroups = 256 / kLanes, kPer = score_pages_per_cta(D);
  __shared__ double u_s[D];
  griddep_launch();
  griddep_wait();
  const int h = blockIdx.y, b = blockIdx.z;
  const int grp = threadIdx.x / kLanes, c = threadIdx.x % kLanes;
  int first = blockIdx.x * kPer + grp;
  int page[kScorePages];
  auto look_up = [&](int at) {
#pragma unroll
    for (int j = 0; j < kScorePages; ++j) page[j] = page_of(p.table, b, at + j * kGroups, p.pool.num_pages);
  };
  look_up(first);   // beside the length
  const int held = held_pages(p, b);
  if (held <= p.budget || static_cast<int>(blockIdx.x) * kPer >= held) return;   // all of them are taken: nothing to score
  uint4 lo[kScorePages], hi[kScorePages];
  unsigned on = 0;   // which of the pages there are
  auto load = [&](int at) {
    on = 0;
#pragma unroll
    for (int j = 0; j < kScorePages; ++j) {
      lo[j] = hi[j] = make_uint4(0, 0, 0, 0);
      if (page[j] >= 0 && at + j * kGroups < held) {
        const uint4* row = reinterpret_cast<const uint4*>(p.pool.k_bounds) + (static_cast<long long>(page[j]) * p.pool.hkv + h) * 2 * kLanes;
        lo[j] = row[c];
        hi[j] = row[kLanes + c];
        on |= 1u << j;
      }
    }
  };
  load(first);
  if (threadIdx.x < D) {
    double s = 0.0;
#pragma unroll 8
    for (int g = 0; g < p.groups; ++g)
      s += static_cast<double>(to_f32<BF16>(*reinterpret_cast<const uint16_t*>(p.q + 2 * (b * p.q_sb + (h * p.groups + g) * p.q_sh + threadIdx.x))));
    u_s[threadIdx.x] = s;
  }
  __syncthreads();
  double u[8];
  uint32_t sign[4];  // which half of a pair takes its maximum
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = u_s[c * 8 + i];
#pragma unroll
  for (int i = 0; i < 4; ++i) sign[i] = (u[2 * i] >= 0.0 ? 0x0000ffffu : 0u) | (u[2 * i + 1] >= 0.0 ? 0xffff0000u : 0u);
  unsigned long long* out = p.keys + (static_cast<long long>(b) * p.pool.hkv + h) * p.table.max_pages;
  const int stride = gridDim.x * kPer;
  for (int base = blockIdx.x * kPer; base < held; base += stride, first += stride) {
    const unsigned here = on;
    uint32_t w[kScorePages][4];   // the bounds that count
#pragma unroll
    for (int j = 0; j < kScorePages; ++j) {
      const uint32_t a[4] = {lo[j].x, lo[j].y, lo[j].z, lo[j].w}, z[4] = {hi[j].x, hi[j].y, hi[j].z, hi[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) w[j][i] = (max16x2_nan<BF16>(a[i], z[i]) & sign[i]) | (min16x2_nan<BF16>(a[i], z[i]) & ~sign[i]);
    }
    if (base + stride < held) {   // the next group's loads fly while this one is summed
      look_up(first + stride);
      load(first + stride);
    }
    double s[kScorePages];
#pragma unroll
    for (int j = 0; j < kScorePages; ++j) {
      s[j] = 0.0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[j] = fma(u[2 * i], static_cast<double>(to_f32<BF16>(static_cast<uint16_t>(w[j][i] & 0xffffu))), s[j]);
        s[j] = fma(u[2 * i + 1], static_cast<double>(to_f32<BF16>(static_cast<uint16_t>(w[j][i] >> 16))), s[j]);
      }
    }
    const double mine = group_sums4<kLanes>(s, c);
    const int i = first + (c & 3) * kGroups;
    if (c < kScorePages && i < held) {
      unsigned long long key = (here >> c) & 1u ? ordered_key(mine) : 0ull;
      if (i < p.sink_pages || i >= held - p.recent_pages) key = ~0ull;
      out[i] = key;
    }
  }
}

constexpr int kPickBins = 2048;
constexpr int kPickKeys = 16;                    // keys of a thread
constexpr int kPickChunk = 1024 * kPickKeys;     // keys of a CTA at a time

// exclusive sum over the CTA's 1024 threads in thread order; `total` is everyone's sum.  Ends with a barrier.
__device__ __forceinline__ int cta_exclusive_sum(int x, int* scratch, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) scratch[warp] = inc;
  __syncthreads();
  int w = scratch[lane], wi = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, wi, o);
    if (lane >= o) wi += y;
  }
  total = __shfl_sync(0xffffffffu, wi, 31);
  const int before = __shfl_sync(0xffffffffu, wi - w, warp);
  __syncthreads();
  return before + inc - x;
}

// Places, in ascending order of the keys' indexes, of the marked keys of a chunk: key j of thread t has index 1024 j + t, so
// counts go by j and warp.  Afterwards counts[32 j + warp] marked keys come before those of this warp with that j; returns the
// number marked.
__device__ __forceinline__ int chunk_counts(unsigned marked, int* counts, int* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int j = 0; j < kPickKeys; ++j) {
    const unsigned votes = __ballot_sync(0xffffffffu, (marked >> j) & 1u);
    if (lane == 0) counts[j * 32 + warp] = __popc(votes);
  }
  __syncthreads();
  int total;
  const int mine = threadIdx.x < kPickKeys * 32 ? counts[threadIdx.x] : 0;
  const int before = cta_exclusive_sum(mine, scratch, total);
  if (threadIdx.x < kPickKeys * 32) counts[threadIdx.x] = before;
  __syncthreads();
  return total;
}
__device__ __forceinline__ int chunk_place(unsigned marked, int j, const int* counts) {
  const unsigned votes = __ballot_sync(0xffffffffu, (marked >> j) & 1u);
  return counts[j * 32 + (threadIdx.x >> 5)] + __popc(votes & ((1u << (threadIdx.x & 31)) - 1u));
}

// One CTA per (KV head, sequence).  The budget-th highest key is found by histograms: 2048 equal bins over the range of the
// keys still in question, then over the bin that the budget ends in, until that bin holds no more keys than are wanted or one
// value only (two rounds for scores as they occur, six at most).  Up to 16384 pages the keys stay in registers; more are read
// again in every round.
__global__ void __launch_bounds__(1024) paged_pick_kernel(const __grid_constant__ PagedSelectParams p) {
  __shared__ int hist[kPickBins], scratch[32], found[3];
  __shared__ uint32_t red[2][32];
  griddep_launch();
  griddep_wait();  // the keys come from the kernel launched just before, the lengths from anywhere
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned long long* keys = p.keys + (static_cast<long long>(b) * p.pool.hkv + h) * p.table.max_pages;
  int* out = p.out + (static_cast<long long>(b) * p.pool.hkv + h) * p.budget;
  const int held = held_pages(p, b);
  if (held <= p.budget) {
    for (int i = tid; i < p.budget; i += 1024) out[i] = i < held ? i : -1;
    return;
  }
  // pages that are taken without a score (sink + recent <= budget < held, so the two do not meet)
  const int lo_i = p.sink_pages, hi_i = held - p.recent_pages;
  const bool many = held > kPickChunk;
  unsigned long long k[kPickKeys];
  unsigned in = 0;  // which of them are in the running
  auto load = [&](int i0) {
    in = 0;
#pragma unroll
    for (int j = 0; j < kPickKeys; ++j) {
      const int i = i0 + j * 1024 + tid;
      const bool on = i >= lo_i && i < hi_i;
      k[j] = on ? keys[i] : 0ull;
      in |= static_cast<unsigned>(on) << j;
    }
  };
  load(0);
  int want = p.budget - p.sink_pages - p.recent_pages;
  // bounds of the keys by their high words
  uint32_t low_word = ~0u, high_word = 0u;
  for (int i0 = 0; i0 < held; i0 += kPickChunk) {
    if (i0 > 0) load(i0);
#pragma unroll
    for (int j = 0; j < kPickKeys; ++j)
      if ((in >> j) & 1u) { low_word = min(low_word, static_cast<uint32_t>(k[j] >> 32)); high_word = max(high_word, static_cast<uint32_t>(k[j] >> 32)); }
  }
  low_word = __reduce_min_sync(0xffffffffu, low_word);
  high_word = __reduce_max_sync(0xffffffffu, high_word);
  if (lane == 0) { red[0][warp] = low_word; red[1][warp] = high_word; }
  __syncthreads();
  low_word = __reduce_min_sync(0xffffffffu, red[0][lane]);
  high_word = __reduce_max_sync(0xffffffffu, red[1][lane]);
  // (hi < ~0: no score has that key)
  unsigned long long lo = static_cast<unsigned long long>(low_word) << 32, hi = min((static_cast<unsigned long long>(high_word) << 32) | 0xffffffffull, ~1ull);
  // keys above `hi` are taken, keys below `lo` are not, `want` of those between are
  unsigned long long from = hi + 1ull;  // what is taken without a look at its place
  // one round: the histogram has been counted; narrows lo .. hi to a bin, true when there is nothing left to decide
  auto narrow = [&](int shift) {
    __syncthreads();
    // from the highest bin down: thread t has bins 2047 - 2 t and 2046 - 2 t
    const int b0 = kPickBins - 1 - 2 * tid, n0 = hist[b0], n1 = hist[b0 - 1];
    int total;
    const int above = cta_exclusive_sum(n0 + n1, scratch, total);
    if (above < want && above + n0 + n1 >= want) {
      const bool second = above + n0 < want;
      found[0] = second ? b0 - 1 : b0;
      found[1] = second ? above + n0 : above;  // keys in higher bins
      found[2] = second ? n1 : n0;
    }
    __syncthreads();
    const int bin = found[0], higher = found[1], inside = found[2];
    want -= higher;
    const unsigned long long bin_lo = lo + (static_cast<unsigned long long>(bin) << shift);
    const unsigned long long width = (1ull << shift) - 1ull;
    const unsigned long long bin_hi = hi - bin_lo < width ? hi : bin_lo + width;
    lo = bin_lo;
    hi = bin_hi;
    from = hi + 1ull;
    if (inside == want) { from = lo; want = 0; return true; }  // all of the bin
    return lo == hi;                                           // one value: the lowest pages of it
  };
  bool done = want == 0;
  if (!done && !many) {
    // the first rounds on the upper 32 bits of key - lo, which cost a third of the instructions
    const int shift = max(0, 32 - __clzll(hi - lo));
    uint32_t top[kPickKeys];
#pragma unroll
    for (int j = 0; j < kPickKeys; ++j) top[j] = static_cast<uint32_t>((k[j] - lo) >> shift);
    uint32_t above = 0;   // the bits that the rounds have settled
#pragma unroll
    for (int round = 0; round < 2; ++round) {
      if (done) break;
      const int place = round == 0 ? 21 : 10;
      hist[tid] = hist[1024 + tid] = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kPickKeys; ++j)
        if (((in >> j) & 1u) && (round == 0 || (top[j] >> 21) == above)) atomicAdd(&hist[(top[j] >> place) & 2047], 1);
      done = narrow(shift + place);
      above = found[0];
      __syncthreads();
    }
  }
  while (!done) {
    const int shift = max(0, 53 - __clzll(hi - lo));  // (hi - lo) >> shift < 2048
    hist[tid] = hist[1024 + tid] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < held; i0 += kPickChunk) {
      if (many) load(i0);
#pragma unroll
      for (int j = 0; j < kPickKeys; ++j)
        if (((in >> j) & 1u) && k[j] >= lo && k[j] <= hi) atomicAdd(&hist[static_cast<int>((k[j] - lo) >> shift)], 1);
    }
    done = narrow(shift);
    __syncthreads();
  }
  __syncthreads();
  int taken = 0, ties = 0;  // before this chunk
  for (int i0 = 0; i0 < held; i0 += kPickChunk) {
    if (many) load(i0);
    unsigned take = 0, tie = 0;
#pragma unroll
    for (int j = 0; j < kPickKeys; ++j) {
      const int i = i0 + j * 1024 + tid;
      const bool on = (in >> j) & 1u;
      if (i < held && (!on || k[j] >= from)) take |= 1u << j;
      else if (on && k[j] == lo) tie |= 1u << j;
    }
    if (want > 0) {   // of the keys equal to lo the first `want`
      const int n = chunk_counts(tie, hist, scratch);
      unsigned more = 0;
#pragma unroll
      for (int j = 0; j < kPickKeys; ++j) {
        const int place = chunk_place(tie, j, hist);
        if (((tie >> j) & 1u) && ties + place < want) more |= 1u << j;
      }
      take |= more;
      ties += n;
      __syncthreads();
    }
    const int n = chunk_counts(take, hist, scratch);
#pragma unroll
    for (int j = 0; j < kPickKeys; ++j) {
      const int place = chunk_place(take, j, hist);
      if ((take >> j) & 1u) out[taken + place] = i0 + j * 1024 + tid;
    }
    taken += n;
    __syncthreads();
  }
}

}  // namespace sq
