// Attention of one new token per sequence over a paged key/value cache, over all pages or over listed ones.
//
// Memory bound: per key and KV head 2 * row bytes (+ 8 for codes) are read once for all query heads of the group.
//
// Work.  A tile is 32 or 64 keys of one (sequence, KV head) segment.  All tiles of all segments stand in one row, and every
// warp of the grid takes an equal stretch of it, whatever the lengths, which the kernel reads itself; so a captured launch
// stays balanced while the cache grows, and a ragged batch needs no plan.  A segment that lies in one warp's stretch is
// finished by that warp alone; pieces of a segment that several warps share are joined at the end of the CTA, and what CTAs
// share by paged_merge_kernel.
//
// Copies.  A warp is its own producer: it keeps kStages of its tiles in flight in a ring of its own (TMA boxes of 16 to 64
// rows, 128-byte swizzle, scales by bulk copies), so that warps never wait for one another before the end of the CTA, and the
// ring runs on across segments.  Where a tile's pages lie is looked up by one lane per tile, 32 tiles at a time, and that lane
// issues the tile's copies.
//
// Arithmetic.  S^T = K Q^T and O^T = V^T P^T on mma.sync m16n8k16 with the keys (channels) as rows and the query heads as
// the 8 columns: with at most 8 heads to a group no product is padding but the unused heads' columns.  The products do not
// bound the kernel (at 128 channels a key takes 0.5 KFLOP a head for 128-512 bytes), so the tcgen05 path, which would need 64 or 128
// rows of queries, has nothing to give here.
//   codes, scores: integer products m16n8k32 of the keys' bytes as they lie (4-bit codes as the high halves of bytes: a mask) with
//     q as 24-bit integers, a power of two per head high, in a signed high and two unsigned lower bytes: sums are exact, and q is
//     off by at most 2^-23 of the head's largest, half a step of fp32.  Two bytes (2^-15) are not enough beside a head's large
//     channels: with one of 64 times the others scores were off by 1e-3.  The third product costs 512K int4 tokens 66.6 -> 70.8 us,
//     64 ragged int4 sequences 78.0 -> 80.4, 16 ragged int8 ones 152 -> 157; leaving it out for heads without large channels gains
//     0.5 us of that, adding `low` up in integers nothing.
//   codes, output: codes become f16 exactly by exponent tricks; a value's scale multiplies its weight p in fp32, and the product
//     is rounded to f16 relative to the largest value scale so far (as a power of two), 2^14 high.  For bf16 outputs that
//     rounding (2^-11) vanishes beside theirs (2^-8); for f16 outputs, which have the same, the weight is split as below.  The
//     output's type decides, whatever the queries' is.
//   The conversions are what costs: on this part an ALU or f16x2 instruction takes an SM quarter 2 clocks, a f16 product
//     m16n8k16 8.3, an integer product m16n8k32 8.1, and they hardly overlap.
//   native: p is split into two 16-bit parts, so that its rounding (2^-16 or 2^-22) vanishes beside the output's.  A low part
//     may be zero or negative, so infinite values enter by a product of their own, with 1 for every weight that is not zero.
//     Looking for them costs 64 multiplications by zero a lane and tile; with the code for them a call of 1000 keys takes 8.6 us
//     for 8.4, of 8000 15.4 for 14.8, of 1M the same.
// Scores of -inf (a key with an infinity) count as keys: where all of a sequence's are, the output is NaN as the softmax is, and
// the LSE -inf.  Until the last join such a part has the LSE kAllMinusInf, one without keys -inf.
// Channels and keys may enter a product in any order as long as both operands agree, so codes are taken from shared memory
// in the order in which they lie (16 bytes a lane); `row_perm` below orders the keys so that those loads do not collide.
#pragma once
#include <cuda.h>

#include "decode.cuh"
#include "paged_cache.cuh"

namespace sq {

constexpr int kPagedMaxBatch = 1024;
constexpr float kAllMinusInf = -3.402823466e38f;   // below every LSE that a sequence can have
constexpr int kPagedCluster = 8;
constexpr int kPagedMaxClusters = 16;  // two to a GPC, and as many as the device has places for

struct PagedDecodeParams {
  PagedPool pool;
  BlockTable table;
  const uint8_t* q;  // [B, Hq, D] through element strides
  long long q_sb, q_sh;
  uint8_t* o;
  long long o_sb, o_sh;
  float* lse;  // [B, Hq] or null
  const int* kv_lens;
  const int* list;  // [B, Hkv, list_len] pages of the sequence to attend to, or null: all of them
  int list_len;
  int max_len;  // what the table, or the caller's bound, holds
  int batch, hq, groups, o_bf16;
  int q_bf16;        // codes: type of the queries (native: BF16)
  int clusters;      // a cluster of kPagedCluster CTAs for each segment: they join its parts themselves
  int q_align;       // bytes that every head's row is aligned to: 16, 4 or 2
  float scale_log2;  // softmax scale * log2(e)
  float* part_o;     // [grid + B * Hkv, groups, D] fp32, each divided by its own sum
  float* part_lse;   // [grid + B * Hkv, groups]
  float* piece_o;    // [grid * warps, 8 or 16 columns, D] fp32: what a warp's first segment has of it, if that ends inside the stretch
  int* plan;         // [B + 2]: tiles per KV head before each sequence, then tiles per CTA
  int* cut;          // [grid]: segment that begins in the CTA before and goes on in this one, or -1
};

template <int FMT, int D, int NT>
struct PagedDecodeCfg {
  static constexpr int kRow = kv_row_bytes<FMT>(D);
  // Measured (us; 1M native | 16 ragged int8 | 512K int4, 28/4 and 32/8 heads): native 8 warps of one tile in flight 319, 4 of two
  // 321, of three 338-351; int8 8 of two 131, 10 137, 12 147, 6 149; int4 12 warps of two 64-key tiles 68, of two 32-key tiles 75,
  // 16 of two 32-key tiles 84, 8 86.  More than about 130 KB in flight an SM is slower, whatever holds it.  (Codes: with queries of
  // two bytes.  With three, 512K int4 tokens take 12 warps 70.8, 11 75.5, 10 79.2.)
  static constexpr int kTile = FMT == kKvInt4 ? 64 : 32;                 // keys of a tile
  static constexpr int kWarps = FMT == kKvInt4 && NT == 1 ? 12 : 8;
  static constexpr int kStages = FMT == kKvNative && D == 128 ? 1 : 2;   // tiles a warp has in flight
  static constexpr int kTensor = kTile * kRow;                           // a tile's keys or values
  static constexpr int kRingWarp = kStages * 2 * kTensor;
  static constexpr int kScaleOff = kWarps * kRingWarp;                   // [warp][stage][K, V][kTile] fp32
  static constexpr int kScaleStage = FMT == kKvNative ? 0 : 2 * kTile * 4;
  static constexpr int kMlOff = kScaleOff + kWarps * kStages * kScaleStage;  // [2 warps][8 NT] maxima, then sums
  static constexpr int kBarOff = kMlOff + 2 * kWarps * 8 * NT * 8;       // [warp][stage]
  static constexpr int kInfoOff = kBarOff + kWarps * kStages * 8;        // [warp][stage] valid keys
  static constexpr int kRecOff = (kInfoOff + kWarps * kStages * 4 + 15) / 16 * 16;  // [warp][32 tiles] where their pages lie
  static constexpr int kSegOff = kRecOff + kWarps * 32 * 32;             // [2 warps] segments of the pieces
  static constexpr int kMiscOff = kSegOff + 2 * kWarps * 4;              // abort flag, exponents of codes
  static constexpr int kPlanOff = (kMiscOff + 16 + 15) / 16 * 16;        // [B + 1]
  __host__ __device__ static constexpr int share_off(int batch) { return (kPlanOff + (batch + 1) * 4 + 15) / 16 * 16; }  // clusters: a CTA's part [8 NT][D], LSE [8 NT]
  __host__ __device__ static constexpr int total(int batch, bool clusters) { return share_off(batch) + (clusters ? 8 * NT * (D + 1) * 4 : 0) + 1024; }
  static_assert(total(kPagedMaxBatch, false) <= 227 * 1024 && total(kPagedMaxClusters, true) <= 227 * 1024, "shared memory of a CTA");
  static_assert(8 * NT * D * 4 <= kRingWarp, "a warp's last piece takes the place of its ring");
};

// C[16][8] += A[16][32] B[32][8] in integers: signed bytes by the signed high bytes (kHigh) or the unsigned lower bytes of 24-bit numbers
template <bool kHigh>
__device__ __forceinline__ void mma_16832_int(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (kHigh)
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// every thread of the cluster, with its shared memory's writes; a thread that has ended counts as arrived
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_address(uint32_t local, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 cluster_load2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
// what kAllMinusInf stands for in the end
__device__ __forceinline__ void settle_minus_inf(float& val, float& lse) {
  if (lse == kAllMinusInf) { val = __int_as_float(0x7fc00000); lse = -INFINITY; }
}
// t + 0 * x for two 16-bit numbers: NaN once x is infinite or NaN
template <bool BF16>
__device__ __forceinline__ uint32_t add_zero_times(uint32_t x, uint32_t t) {
  uint32_t r;
  if (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(t));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(t));
  return r;
}
__device__ __forceinline__ uint32_t h2_add(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Codes to f16 pairs, exactly.  The bits of a biased code (sign bit flipped) under the exponent of 1024 are 1024 + code + bias;
// four bits further up they are 64 + code + bias under the exponent of 64.
//   bytes 0, 2 of x / bytes 1, 3 of x;   nibbles 0, 4 / 1, 5 of x
// One of the two constants of (x & mask) ^ exponent has to be in a register for one instruction to do it: the exponents come
// from memory, so that the compiler cannot make them immediates (which then take two instructions).
struct CodeExponents { uint32_t byte, low, high; };  // of 1024 for bytes and low nibbles, of 64 for nibbles 4 bits up; bias in it
constexpr uint32_t kByteExponent = 0x64806480u, kLowExponent = 0x64086408u, kHighExponent = 0x54805480u;
__device__ __forceinline__ void bytes_to_h2(uint32_t x, const CodeExponents& ce, uint32_t& even, uint32_t& odd) {
  constexpr uint32_t kMinus1152 = 0xe480e480u;
  even = h2_add((x & 0x00ff00ffu) ^ ce.byte, kMinus1152);
  odd = h2_add(((x >> 8) & 0x00ff00ffu) ^ ce.byte, kMinus1152);
}
__device__ __forceinline__ void nibbles_to_h2(uint32_t x, const CodeExponents& ce, uint32_t& n0, uint32_t& n1) {
  constexpr uint32_t kMinus1032 = 0xe408e408u, kMinus72 = 0xd480d480u;
  n0 = h2_add((x & 0x000f000fu) ^ ce.low, kMinus1032);
  n1 = h2_add((x & 0x00f000f0u) ^ ce.high, kMinus72);
}

// Key that row r (0..7; +8 likewise) of a product's 16 keys stands for.  A quarter or half warp reads the rows of four lanes t
// (values: rows 2t, then 2t + 1) or of two to four lanes g (keys) at once; with these orders their 16-, 8- or 4-byte pieces
// fall on different banks under the 128-byte swizzle.
template <int ROW>
__device__ __forceinline__ int row_perm(int r) {
  constexpr uint32_t kOrder = ROW == 128 ? 0x76543210u : (ROW == 64 ? 0x65742130u : 0x53427160u);
  return (kOrder >> (4 * r)) & 7;
}
__device__ __forceinline__ uint32_t swizzle128(uint32_t o) { return o ^ ((o >> 3) & 0x70u); }

// tiles of one (sequence, KV head) segment
__device__ __forceinline__ int paged_len(const PagedDecodeParams& p, int b) { return min(max(p.kv_lens[b], 0), p.max_len); }
template <int TILE>
__device__ __forceinline__ int paged_tiles(const PagedDecodeParams& p, int len) {
  if (len == 0) return 0;
  const int keys = p.list ? p.list_len << p.pool.ps_shift : len;
  return static_cast<int>((static_cast<unsigned>(keys) + TILE - 1) / TILE);
}

// BF16: type of pages and queries where pages are native, of the outputs where they are codes
template <int FMT, int D, bool BF16, int NT>
__global__ void __launch_bounds__(PagedDecodeCfg<FMT, D, NT>::kWarps * 32, 1)
paged_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ PagedDecodeParams p) {
  using C = PagedDecodeCfg<FMT, D, NT>;
  constexpr int W = C::kWarps, S = C::kStages, ROW = C::kRow, TILE = C::kTile, MT = TILE / 16, NTHR = W * 32, H = 8 * NT;
  constexpr bool kNative = FMT == kKvNative;
  constexpr bool kTwoParts = kNative || !BF16;   // weights in two 16-bit parts
  // f16 weights are kept 2^14 high, away from that type's subnormal numbers; bf16 has none to fear, and its values could overflow
  constexpr float kLift = kNative && BF16 ? 0.0f : 14.0f, kUnlift = kNative && BF16 ? 1.0f : 1.0f / 16384.0f;
  constexpr uint32_t kAllValid = MT == 2 ? 0x1010u : 0x10101010u;
  griddep_launch();
  griddep_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int hkv = p.pool.hkv;
  auto store_o = [&](int b, int hq, int d, float x) {
    reinterpret_cast<uint16_t*>(p.o)[b * p.o_sb + hq * p.o_sh + d] = p.o_bf16 ? from_f32<true>(x) : from_f32<false>(x);
  };
  const bool gave_up = device_failed();   // asked for here, answered at the first barrier
  // aligned by an offset: a pointer that went through an integer would be loaded from with generic instructions
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((0u - smem_u32(smem_raw)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  volatile int* cta_abort = reinterpret_cast<volatile int*>(smem + C::kMiscOff);
  int* pre = reinterpret_cast<int*>(smem + C::kPlanOff);
  int* seg_of = reinterpret_cast<int*>(smem + C::kSegOff);   // [warp][piece of the first segment, piece of the last]
  float* ml = reinterpret_cast<float*>(smem + C::kMlOff);    // their maxima [2 W][H], then sums [2 W][H]
  const uint32_t bars = sbase + C::kBarOff + warp * S * 8;
  volatile uint32_t* info = reinterpret_cast<volatile uint32_t*>(smem + C::kInfoOff) + warp * S;

  // ---- plan: tiles (of one KV head) before each sequence.  Many lengths are fetched by all warps, or the scan would wait for
  // each 32 of them in turn
  const bool many = p.batch > 64;
  if (many) {
    for (int b = tid; b < p.batch; b += NTHR) pre[b] = paged_tiles<TILE>(p, paged_len(p, b));
    __syncthreads();
  }
  if (warp == 0) {
    int run = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      const int b = b0 + lane;
      const int mine = b >= p.batch ? 0 : many ? pre[b] : paged_tiles<TILE>(p, paged_len(p, b));
      int x = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (b < p.batch) pre[b] = run + x - mine;
      run += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) pre[p.batch] = run;
  } else if (warp == 1) {
    if (lane < 2 * W) seg_of[lane] = -1;
    if (lane == 0) {
      cta_abort[0] = 0;
      cta_abort[1] = kByteExponent;
      cta_abort[2] = kLowExponent;
      cta_abort[3] = kHighExponent;
      for (int i = 0; i < W * S; ++i) mbar_init(sbase + C::kBarOff + 8 * i, kNative ? 1 : 33);  // codes: every lane's scales, too
      fence_barrier_init();
      fence_proxy_async();
    }
  }
  // after a wait has given up on this device, here or in an earlier launch, the caller gets NaN and no stale memory
  if (__syncthreads_or(gave_up)) {
    const float nan = __int_as_float(0x7fc00000);
    const long long rows = static_cast<long long>(p.batch) * p.hq;
    for (long long i = blockIdx.x * static_cast<long long>(NTHR) + tid; i < rows * D; i += static_cast<long long>(gridDim.x) * NTHR) {
      const long long row = i / D;
      store_o(static_cast<int>(row / p.hq), static_cast<int>(row % p.hq), static_cast<int>(i % D), nan);
      if (p.lse && i % D == 0) p.lse[row] = nan;
    }
    if (p.clusters) {   // the others of the cluster may not have noticed: they find the failure in this CTA's part
      float* part_lse = reinterpret_cast<float*>(smem + C::share_off(p.batch)) + H * D;
      if (tid < H) part_lse[tid] = nan;
      cluster_barrier();
      cluster_barrier();
    }
    return;
  }
  // the host has checked that all tiles of a call fit 31 bits
  const int total = pre[p.batch] * hkv;
  const int per = max((total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x), W);
  int x0, x1;
  if (p.clusters) {
    const int seg = blockIdx.x / kPagedCluster, b = seg / hkv, n = pre[b + 1] - pre[b], mine = (n + kPagedCluster - 1) / kPagedCluster;
    const int first = pre[b] * hkv + seg % hkv * n;
    x0 = min(first + n, first + static_cast<int>(blockIdx.x % kPagedCluster) * mine);
    x1 = min(first + n, x0 + mine);
  } else {
    const long long first = static_cast<long long>(blockIdx.x) * per;
    x0 = static_cast<int>(min(first, static_cast<long long>(total)));
    x1 = static_cast<int>(min(first + per, static_cast<long long>(total)));
  }

  // sequence of tile x
  auto seq_of = [&](int x) {
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] * hkv <= x) lo = mid; else hi = mid;
    }
    return lo;
  };
  if (blockIdx.x == 0 && !p.clusters) {
    for (int b = tid; b <= p.batch; b += NTHR) p.plan[b] = pre[b];
    if (tid == 0) p.plan[p.batch + 1] = per;
  }
  if (tid == 0 && !p.clusters) {
    int cut = -1;
    if (x0 > 0 && x0 < x1) {
      const int b = seq_of(x0), n = pre[b + 1] - pre[b], h = (x0 - pre[b] * hkv) / n, first = pre[b] * hkv + h * n;
      if (first < x0 && first / per == static_cast<int>(blockIdx.x) - 1) cut = b * hkv + h;
    }
    p.cut[blockIdx.x] = cut;
  }
  // sequences without keys: zeros
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
    if (pre[b + 1] == pre[b])
      for (int i = tid; i < p.hq * D; i += NTHR) {
        store_o(b, i / D, i % D, 0.0f);
        if (p.lse && i % D == 0) p.lse[static_cast<long long>(b) * p.hq + i / D] = -INFINITY;
      }
  float* share = reinterpret_cast<float*>(smem + C::share_off(p.batch));   // clusters: this CTA's part
  if (p.clusters && tid < H) share[H * D + tid] = -INFINITY;
  if (x0 < x1) {
  // this warp's tiles: xw0, xw0 + step, .. below xw1.  In a CTA whose tiles are all of one segment the warps take turns, so that
  // together they read neighbouring rows (1M tokens native, three tiles in flight: 348 us in stretches, 338 in turns)
  int xw0, xw1, step;
  {
    const int b = seq_of(x0), n = pre[b + 1] - pre[b], first = pre[b] * hkv + (x0 - pre[b] * hkv) / n * n;
    if (x1 <= first + n) {
      xw0 = min(x1, x0 + warp); xw1 = x1; step = W;
    } else {
      const int share = (x1 - x0 + W - 1) / W;
      xw0 = min(x1, x0 + warp * share); xw1 = min(x1, xw0 + share); step = 1;
    }
  }

  // ---- copies.  Lane i looks up the i-th of the warp's next 32 tiles: for each 16 keys of it page * Hkv + head and the number of
  // valid ones (8 bits each), and the first row inside the page (pages of fewer rows than a tile begin at their row 0).  Scales
  // come by 16-byte copies of the lanes: as bulk copies, of 64 to 256 bytes each, they took as many instructions again as the rows
  const int ps = 1 << p.pool.ps_shift;
  const uint32_t ring = sbase + warp * C::kRingWarp;
  const uint32_t scales = sbase + C::kScaleOff + warp * S * C::kScaleStage;
  const int box = kNative ? 16 : min(ps, TILE);   // rows of a copy, as the tensor maps have it
  uint32_t* rec = reinterpret_cast<uint32_t*>(smem + C::kRecOff) + warp * 256;   // [tile][4 pages, first row, valid keys]
  auto look_up = [&](int x) {
    uint32_t* mine = rec + lane * 8;
    uint32_t nv = 0;
    if (x < xw1) {
      const int b = seq_of(x);
      const int n = pre[b + 1] - pre[b], rem = x - pre[b] * hkv;
      const int h = rem / n, key = (rem - h * n) * TILE;
      const int len = paged_len(p, b);
      const int held = static_cast<int>((static_cast<unsigned>(len) + ps - 1) >> p.pool.ps_shift);
      int at_last = -1, ph = 0, first = 0;
#pragma unroll
      for (int s = 0; s < MT; ++s) {
        const int at = static_cast<int>(static_cast<unsigned>(key + 16 * s) >> p.pool.ps_shift);
        if (at != at_last) {
          at_last = at;
          int index = at;
          if (p.list) index = at < p.list_len ? p.list[(static_cast<long long>(b) * hkv + h) * p.list_len + at] : -1;
          const int page = index >= 0 && index < held ? page_of(p.table, b, index, p.pool.num_pages) : -1;
          ph = page * hkv + h;
          first = page >= 0 ? index << p.pool.ps_shift : len;   // position of the page's row 0
        }
        mine[s] = ph;
        const int left = len - first - ((key + 16 * s) & (ps - 1));
        nv |= static_cast<uint32_t>(min(max(left, 0), 16)) << (8 * s);
      }
      mine[4] = key & (ps - 1);
    }
    mine[5] = nv;
  };
  int xi = xw0, ahead = 32;  // next tile to copy, its place among the looked-up ones
  auto issue = [&](int st) {
    if (xi >= xw1) return;
    if (ahead == 32) {
      look_up(xi + lane * step);
      ahead = 0;
      __syncwarp();
    }
    const uint32_t* r = rec + ahead * 8;
    const uint32_t nv = r[5];
    const int row0 = r[4];
    const uint32_t bar = bars + 8 * st;
    if (lane == 0) {
      info[st] = nv;
      const uint32_t dst = ring + st * (2 * C::kTensor);
      const int every = box >> 4;   // in units of 16 rows
      // valid rows come first in a page, so a box has some if its first 16 have
      int boxes = 0;
#pragma unroll
      for (int s = 0; s < MT; ++s) boxes += (s & (every - 1)) == 0 && ((nv >> (8 * s)) & 0xffu) != 0u;
      mbar_expect_tx(bar, boxes * box * (2 * ROW));
#pragma unroll
      for (int s = 0; s < MT; ++s)
        if ((s & (every - 1)) == 0 && ((nv >> (8 * s)) & 0xffu) != 0u) {
          const int row = (row0 + 16 * s) & (ps - 1), line = kNative ? row : row * ROW / 128;
          tma_load_4d(dst + s * (16 * ROW), &tm_k, bar, 0, line, 0, r[s]);
          tma_load_4d(dst + C::kTensor + s * (16 * ROW), &tm_v, bar, 0, line, 0, r[s]);
        }
    }
    if (!kNative) {
      // scales of four keys a lane: the keys' by the first TILE / 4 lanes, the values' by the next
      const int c = lane & (TILE / 4 - 1), s = c >> 2, which = lane / (TILE / 4);
      if (which < 2 && ((nv >> (8 * s)) & 0xffu) != 0u) {
        const float* src = which ? p.pool.v_scale : p.pool.k_scale;
        src += (static_cast<long long>(r[s]) << p.pool.ps_shift) + ((row0 + 16 * s) & (ps - 1)) + 4 * (c & 3);
        cp_async_16(scales + st * C::kScaleStage + which * (TILE * 4) + c * 16, src);
      }
      cp_async_arrive(bar);
    }
    ++ahead;
    xi += step;
    __syncwarp();
  };
#pragma unroll 1
  for (int st = 0; st < S; ++st) issue(st);

  // ---- where this lane's pieces of a tile lie.  The swizzle repeats every 1024 bytes, so these are the places that differ
  // by less; codes: keys [rows 0-7 or 8-15][piece], values [rows 2t, 2t+1, 2t+8, 2t+9]; native: 16-byte chunks by ldmatrix
  // lane of channels 16 i .. 16 i + 15 within 64
  uint32_t kx[4], vx[8];
  if (kNative) {
    const int kr = (lane & 7) + ((lane >> 3) & 1) * 8, kc = lane >> 4;
    const int vr = (lane & 7) + (lane >> 4) * 8, vc = (lane >> 3) & 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kx[i] = kr * 128 + (((2 * i + kc) ^ (kr & 7)) << 4);
      vx[i] = C::kTensor + vr * 128 + (((2 * i + vc) ^ (vr & 7)) << 4);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // ROW 128: i = piece;  64: i = rows 0-7 / 8-15;  32: i = rows 0-7, 8-15, 16-23, 24-31
      const int row = ROW == 128 ? 0 : 8 * i, piece = ROW == 128 ? 2 * t + (i & 1) : t;
      kx[i] = swizzle128((row + row_perm<ROW>(g)) * ROW + piece * (ROW == 32 ? 8 : 16));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      vx[i] = C::kTensor + swizzle128(((i >> 1) * 8 + row_perm<ROW>(2 * t + (i & 1))) * ROW + g * (ROW / 8));
  }
  // offsets of 16 keys' pieces from those
  auto k_off = [&](int mt, int hi, int j) -> uint32_t {
    if (ROW == 128) return kx[j] + (mt * 2 + hi) * 1024;
    if (ROW == 64) return kx[hi] + mt * 1024;
    return kx[(mt & 1) * 2 + hi] + (mt >> 1) * 1024;
  };
  auto v_off = [&](int mt, int i) -> uint32_t {
    if (ROW == 128) return vx[i & 1] + (mt * 2 + (i >> 1)) * 1024;
    if (ROW == 64) return vx[i] + mt * 1024;
    return vx[(mt & 1) * 4 + i] + (mt >> 1) * 1024;
  };
  const int key_row = kNative ? g : row_perm<ROW>(g);  // this lane's first key of 16: that row and the one 8 further

  CodeExponents ce;
  ce.byte = cta_abort[1];
  ce.low = cta_abort[2];
  ce.high = cta_abort[3];

  int st = 0;
  uint32_t parity = 0;
  bool ok = true;
  int xc = xw0;
  int b = seq_of(min(xw0, total - 1));
  while (xc < xw1) {
    // ---- segment (b, h): tiles [xc, seg_end) of it are this warp's
    while (pre[b + 1] * hkv <= xc) ++b;
    const int n = pre[b + 1] - pre[b], b_start = pre[b] * hkv;
    const int h = (xc - b_start) / n;
    const int seg_first = b_start + h * n, seg_last = seg_first + n, seg_end = min(seg_last, xw1);
    const bool whole = step == 1 && seg_first >= xw0 && seg_last <= xw1;

    // ---- query heads as the products' 8 columns
    uint32_t qb[NT][kNative ? D / 16 : D * 3 / 32][2];  // native: [channels 16 i ..][r]; codes: [32 of the channels i / 3, byte from the top i % 3][r]
    float cs[NT][2];             // score factor of this lane's two columns
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int head = nt * 8 + g;
      const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) + b * p.q_sb + static_cast<long long>(h * p.groups + head) * p.q_sh;
      if (kNative) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int d = kk * 16 + 2 * t + 8 * r;
            qb[nt][kk][r] = head >= p.groups ? 0u
                            : p.q_align >= 4 ? *reinterpret_cast<const uint32_t*>(src + d)
                                             : static_cast<uint32_t>(src[d]) | (static_cast<uint32_t>(src[d + 1]) << 16);
          }
        cs[nt][0] = cs[nt][1] = p.scale_log2;
      } else {
        float f[D / 4], top = 0.0f;
        // the lane's channels in the order in which their codes are taken from shared memory: D / 4 in a row
        uint32_t v[D / 8];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint16_t* at = src + t * (D / 4) + 8 * i;
          uint4 x = make_uint4(0, 0, 0, 0);
          if (head < p.groups) {
            if (p.q_align >= 16) {
              x = *reinterpret_cast<const uint4*>(at);
            } else {
              x.x = at[0] | (static_cast<uint32_t>(at[1]) << 16); x.y = at[2] | (static_cast<uint32_t>(at[3]) << 16);
              x.z = at[4] | (static_cast<uint32_t>(at[5]) << 16); x.w = at[6] | (static_cast<uint32_t>(at[7]) << 16);
            }
          }
          v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
        }
#pragma unroll
        for (int i = 0; i < D / 4; ++i) {
          const uint16_t w = static_cast<uint16_t>(i & 1 ? v[i / 2] >> 16 : v[i / 2] & 0xffffu);
          f[i] = p.q_bf16 ? to_f32<true>(w) : to_f32<false>(w);
          top = fmaxf(top, fabsf(f[i]));
          if (f[i] != f[i]) top = INFINITY;
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // a power of two brings the largest to [2^22, 2^23), sums come back in units of 2^8; 4-bit codes arrive 16 times as large
        const uint32_t e = max(__float_as_uint(top) >> 23, 27u);
        const float up = __uint_as_float((276u - e) << 23);
        const float down = e == 255u ? __int_as_float(0x7fc00000) : p.scale_log2 * __uint_as_float((e - (FMT == kKvInt4 ? 6u : 2u)) << 23);   // 2^12 of the key scales' too
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            uint32_t hi = 0, mid = 0, lo = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {   // bytes of word 2 j + r, or even and odd nibbles of word j
              const uint32_t v = static_cast<uint32_t>(__float2int_rn(f[FMT == kKvInt8 ? 8 * j + 4 * r + i : 8 * j + 2 * i + r] * up));
              hi |= ((v >> 16) & 0xffu) << (8 * i);
              mid |= ((v >> 8) & 0xffu) << (8 * i);
              lo |= (v & 0xffu) << (8 * i);
            }
            qb[nt][3 * j][r] = hi;
            qb[nt][3 * j + 1][r] = mid;
            qb[nt][3 * j + 2][r] = lo;
          }
        cs[nt][0] = __shfl_sync(0xffffffffu, down, 8 * t);
        cs[nt][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
      }
    }
    float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
    }
    uint32_t vexp = 27u << 23;  // exponent of the largest value scale so far
    bool keys = false;          // whether there has been any key
    bool odd = false;           // native: whether a value was infinite or NaN

    for (; xc < seg_end; xc += step) {
      ok = ok && mbar_wait_warp(bars + 8 * st, parity, cta_abort, 401);
      if (!ok) break;
      const uint32_t nv = info[st];
      const uint32_t tile = ring + st * (2 * C::kTensor);
      if (nv != 0) {
        keys = true;
        if (kNative && nv != kAllValid) {
          // rows behind the sequence (or of a page that is not there) may hold anything: zeros, so that 0 * x is 0
          for (int i = lane; i < TILE * (ROW / 16); i += 32) {
            const int r = i / (ROW / 16), c = i % (ROW / 16);
            if ((r & 15) >= static_cast<int>((nv >> (8 * (r >> 4))) & 0xffu))
              *reinterpret_cast<uint4*>(smem + (tile - sbase) + C::kTensor + (r >> 4) * (16 * ROW) + (c >> 3) * 2048 + (r & 15) * 128 + (c & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
          __syncwarp();
        }
        // ---- scores
        float s[NT][MT][4];
        float vs[MT][2];  // value scales of this lane's keys
        if (kNative) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) s[nt][mt][0] = s[nt][mt][1] = s[nt][mt][2] = s[nt][mt][3] = 0.0f;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              uint32_t a[4];
              ldmatrix_x4(tile + kx[kk & 3] + mt * (16 * ROW) + (kk >> 2) * 2048, a[0], a[1], a[2], a[3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_16816<BF16>(s[nt][mt], a, qb[nt][kk][0], qb[nt][kk][1]);
            }
        } else {
          const uint8_t* tp = smem + (tile - sbase);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            constexpr int kWords = ROW / 16;  // 4-byte words of a key per lane
            uint32_t w[2][kWords];
#pragma unroll
            for (int hi = 0; hi < 2; ++hi)
#pragma unroll
              for (int j = 0; j < (kWords + 3) / 4; ++j) {
                if (kWords == 2) {
                  const uint2 v = *reinterpret_cast<const uint2*>(tp + k_off(mt, hi, 0));
                  w[hi][0] = v.x; w[hi][1] = v.y;
                } else {
                  const uint4 v = *reinterpret_cast<const uint4*>(tp + k_off(mt, hi, j));
                  w[hi][4 * j] = v.x; w[hi][4 * j + 1] = v.y; w[hi][4 * j + 2] = v.z; w[hi][4 * j + 3] = v.w;
                }
              }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              int high[4] = {0, 0, 0, 0}, middle[4] = {0, 0, 0, 0}, low[4] = {0, 0, 0, 0};
#pragma unroll
              for (int j = 0; j < D / 32; ++j) {
                uint32_t a[4];
#pragma unroll
                for (int hi = 0; hi < 2; ++hi) {
                  if (FMT == kKvInt8) {
                    a[hi] = w[hi][2 * j];
                    a[2 + hi] = w[hi][2 * j + 1];
                  } else {   // nibbles as the high halves of signed bytes: 16 times the code
                    a[hi] = (w[hi][j] << 4) & 0xf0f0f0f0u;
                    a[2 + hi] = w[hi][j] & 0xf0f0f0f0u;
                  }
                }
                mma_16832_int<true>(high, a[0], a[1], a[2], a[3], qb[nt][3 * j][0], qb[nt][3 * j][1]);
                mma_16832_int<false>(middle, a[0], a[1], a[2], a[3], qb[nt][3 * j + 1][0], qb[nt][3 * j + 1][1]);
                mma_16832_int<false>(low, a[0], a[1], a[2], a[3], qb[nt][3 * j + 2][0], qb[nt][3 * j + 2][1]);
              }
#pragma unroll
              for (int e = 0; e < 4; ++e)   // the upper two below 2^30, then rounded as fp32 sums are
                s[nt][mt][e] = fmaf(static_cast<float>(low[e]), 1.0f / 256.0f, static_cast<float>(high[e] * 256 + middle[e]));
            }
          }
          // scales
          const float* sc = reinterpret_cast<const float*>(smem + (scales - sbase) + st * C::kScaleStage);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
              const float ks = sc[mt * 16 + hi * 8 + key_row] * (1.0f / 4096.0f);   // sums of up to 2^30: keys near the type's largest stay in range
              vs[mt][hi] = sc[TILE + mt * 16 + hi * 8 + key_row];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) { s[nt][mt][2 * hi] *= ks; s[nt][mt][2 * hi + 1] *= ks; }
            }
        }
        if (nv != kAllValid) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi)
              if (hi * 8 + key_row >= static_cast<int>((nv >> (8 * mt)) & 0xffu)) {
                vs[mt][hi] = 0.0f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][mt][2 * hi] = s[nt][mt][2 * hi + 1] = -INFINITY;
              }
        }
        // ---- running maxima
        bool moved = false;
        float m_new[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = fmaxf(s[nt][0][c], s[nt][0][c + 2]);
#pragma unroll
            for (int mt = 1; mt < MT; ++mt) x = max3(x, s[nt][mt][c], s[nt][mt][c + 2]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            m_new[nt][c] = fmaxf(m[nt][c], x);
            moved |= m_new[nt][c] > m[nt][c];
          }
        uint32_t vexp_new = vexp;
        if (!kNative) {
          float top = fmaxf(vs[0][0], vs[0][1]);
#pragma unroll
          for (int mt = 1; mt < MT; ++mt) top = max3(top, vs[mt][0], vs[mt][1]);
          vexp_new = max(vexp, __reduce_max_sync(0xffffffffu, __float_as_uint(top)) & 0x7f800000u);
        }
        if (__any_sync(0xffffffffu, moved) || vexp_new != vexp) {
          // 2^(old - new) of the value scales' exponents
          const float shrink = kNative ? 1.0f : __uint_as_float(max(static_cast<int>(0x3f800000u - (vexp_new - vexp)), 0));
          vexp = vexp_new;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float a[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float base = m_new[nt][c] == -INFINITY ? 0.0f : m_new[nt][c];
              a[c] = ex2_approx((m[nt][c] - base) * cs[nt][c]);
              l[nt][c] *= a[c];
              a[c] *= shrink;
              m[nt][c] = m_new[nt][c];
            }
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              o[nt][i][0] *= a[0]; o[nt][i][1] *= a[1]; o[nt][i][2] *= a[0]; o[nt][i][3] *= a[1];
            }
          }
        }
        // ---- weights and their two 16-bit parts, for codes of their products with the value scales
        uint32_t pb[NT][MT][2], pl[NT][MT][2];
        const float inv = __uint_as_float((254u << 23) - vexp);
        if (!kNative) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) { vs[mt][0] *= inv; vs[mt][1] *= inv; }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float off[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) off[c] = kLift - (m[nt][c] == -INFINITY ? 0.0f : m[nt][c] * cs[nt][c]);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
              const float w0 = ex2_approx(fmaf(s[nt][mt][2 * hi], cs[nt][0], off[0]));
              const float w1 = ex2_approx(fmaf(s[nt][mt][2 * hi + 1], cs[nt][1], off[1]));
              l[nt][0] += w0;
              l[nt][1] += w1;
              if (kNative) {
                const uint32_t head = BF16 ? pack_bf16x2(w0, w1) : pack_f16x2(w0, w1);
                const float h0 = to_f32<BF16>(static_cast<uint16_t>(head & 0xffffu)), h1 = to_f32<BF16>(static_cast<uint16_t>(head >> 16));
                pb[nt][mt][hi] = movmatrix_trans(head);
                pl[nt][mt][hi] = movmatrix_trans(BF16 ? pack_bf16x2(w0 - h0, w1 - h1) : pack_f16x2(w0 - h0, w1 - h1));
              } else {
                const float a = w0 * vs[mt][hi], z = w1 * vs[mt][hi];
                const uint32_t head = pack_f16x2(a, z);
                pb[nt][mt][hi] = movmatrix_trans(head);
                if (kTwoParts) {
                  const float h0 = to_f32<false>(static_cast<uint16_t>(head & 0xffffu)), h1 = to_f32<false>(static_cast<uint16_t>(head >> 16));
                  pl[nt][mt][hi] = movmatrix_trans(pack_f16x2(a - h0, z - h1));
                }
              }
            }
        }
        // ---- values
        bool infinite = odd;
        if (kNative && !odd) {
          uint32_t t0 = 0u, t1 = 0u;   // 0 * every value
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              uint32_t a[4];
              ldmatrix_x4_trans(tile + vx[i & 3] + mt * (16 * ROW) + (i >> 2) * 2048, a[0], a[1], a[2], a[3]);
              t0 = add_zero_times<BF16>(a[1], add_zero_times<BF16>(a[0], t0));
              t1 = add_zero_times<BF16>(a[3], add_zero_times<BF16>(a[2], t1));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_16816<BF16>(o[nt][i], a, pb[nt][mt][0], pb[nt][mt][1]);
                mma_16816<BF16>(o[nt][i], a, pl[nt][mt][0], pl[nt][mt][1]);
              }
            }
          infinite = __any_sync(0xffffffffu, ((t0 | t1) & 0x7fff7fffu) != 0u);
        }
        if (kNative && infinite) {
          constexpr uint32_t kExp = BF16 ? 0x7f807f80u : 0x7c007c00u;
          constexpr uint16_t kOne = BF16 ? 0x3f80 : 0x3c00;
          uint32_t any[NT][MT][2];   // 1 where a weight is not zero
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int hi = 0; hi < 2; ++hi) {
                uint32_t two = 0u;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  const float off = kLift - (m[nt][c] == -INFINITY ? 0.0f : m[nt][c] * cs[nt][c]);
                  if (ex2_approx(fmaf(s[nt][mt][2 * hi + c], cs[nt][c], off)) > 0.0f) two |= static_cast<uint32_t>(kOne) << (16 * c);
                }
                any[nt][mt][hi] = movmatrix_trans(two);
              }
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            float c[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.0f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              uint32_t a[4], z[4];   // the finite values, the others
              ldmatrix_x4_trans(tile + vx[i & 3] + mt * (16 * ROW) + (i >> 2) * 2048, a[0], a[1], a[2], a[3]);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t those = __vcmpeq2(a[j] & kExp, kExp);
                z[j] = a[j] & those;
                a[j] &= ~those;
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_16816<BF16>(c[nt], z, any[nt][mt][0], any[nt][mt][1]);
                if (odd) {
                  mma_16816<BF16>(o[nt][i], a, pb[nt][mt][0], pb[nt][mt][1]);
                  mma_16816<BF16>(o[nt][i], a, pl[nt][mt][0], pl[nt][mt][1]);
                }
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                // the first such tile is in the sums already: channels that have an infinity in it hold that and nothing else
                const bool finite = fabsf(c[nt][e]) < INFINITY;
                o[nt][i][e] = odd ? o[nt][i][e] + c[nt][e] : finite ? o[nt][i][e] : c[nt][e];
              }
          }
          odd = true;
        }
        if (!kNative) {
          const uint8_t* tp = smem + (tile - sbase);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            constexpr int kWords = ROW / 32;
            uint32_t w[4][kWords];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (kWords == 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(tp + v_off(mt, i));
                w[i][0] = v.x; w[i][1 % kWords] = v.y; w[i][2 % kWords] = v.z; w[i][3 % kWords] = v.w;
              } else if (kWords == 2) {
                const uint2 v = *reinterpret_cast<const uint2*>(tp + v_off(mt, i));
                w[i][0] = v.x; w[i][1 % kWords] = v.y;
              } else {
                w[i][0] = *reinterpret_cast<const uint32_t*>(tp + v_off(mt, i));
              }
            }
#pragma unroll
            for (int u = 0; u < kWords; ++u)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                // channels of two keys side by side: 2 bytes or 4 nibbles of each
                const uint32_t lo = __byte_perm(w[0][u], w[1][u], half ? 0x7632 : 0x5410);
                const uint32_t hi = __byte_perm(w[2][u], w[3][u], half ? 0x7632 : 0x5410);
                if (FMT == kKvInt8) {
                  uint32_t a[4];
                  bytes_to_h2(lo, ce, a[0], a[1]);
                  bytes_to_h2(hi, ce, a[2], a[3]);
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt) {
                    mma_16816<false>(o[nt][2 * u + half], a, pb[nt][mt][0], pb[nt][mt][1]);
                    if (kTwoParts) mma_16816<false>(o[nt][2 * u + half], a, pl[nt][mt][0], pl[nt][mt][1]);
                  }
                } else {
#pragma unroll
                  for (int q = 0; q < 2; ++q) {
                    uint32_t a[4];
                    nibbles_to_h2(lo >> (8 * q), ce, a[0], a[1]);
                    nibbles_to_h2(hi >> (8 * q), ce, a[2], a[3]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                      mma_16816<false>(o[nt][4 * u + 2 * half + q], a, pb[nt][mt][0], pb[nt][mt][1]);
                      if (kTwoParts) mma_16816<false>(o[nt][4 * u + 2 * half + q], a, pl[nt][mt][0], pl[nt][mt][1]);
                    }
                  }
                }
              }
          }
        }
      }
      __syncwarp();
      issue(st);
      if (++st == S) { st = 0; parity ^= 1; }
    }

    // ---- this warp's result of the segment
    const float nan = __int_as_float(0x7fc00000);
    const float unit = (kNative ? 1.0f : __uint_as_float(vexp)) * kUnlift;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], sh);
        l[nt][c] = ok ? l[nt][c] * kUnlift : nan;
        m[nt][c] = m[nt][c] != -INFINITY ? m[nt][c] * cs[nt][c] : keys && l[nt][c] == 0.0f ? kAllMinusInf : -INFINITY;  // a NaN sum has no maximum of its own
      }
    // channel of o[nt][i][e]; e & 1 is the column
    auto channel = [&](int i, int e) { return kNative ? 16 * i + g + 8 * (e >> 1) : (D / 8) * g + 2 * i + (e >> 1); };
    if (whole) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col = nt * 8 + 2 * t + c;
          if (col < p.groups) {
            const float f = l[nt][c] != 0.0f ? unit / l[nt][c] : keys ? nan : 0.0f;
            uint16_t* row = reinterpret_cast<uint16_t*>(p.o) + b * p.o_sb + static_cast<long long>(h * p.groups + col) * p.o_sh;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              const float a = o[nt][i][c] * f, z = o[nt][i][c + 2] * f;
              const uint32_t two = p.o_bf16 ? pack_bf16x2(a, z) : pack_f16x2(a, z);
              if (kNative) {
                row[channel(i, 0)] = static_cast<uint16_t>(two & 0xffffu);
                row[channel(i, 2)] = static_cast<uint16_t>(two >> 16);
              } else {
                *reinterpret_cast<uint32_t*>(row + channel(i, 0)) = two;
              }
            }
            if (p.lse && g == 0)
              p.lse[static_cast<long long>(b) * p.hq + h * p.groups + col] =
                  l[nt][c] != 0.0f ? log2f(l[nt][c]) + (m[nt][c] == -INFINITY ? 0.0f : m[nt][c]) : -INFINITY;
          }
        }
    } else {
      // a piece: the last one of the stretch into the ring, which is empty by then, one before it to global scratch
      const bool last = seg_end == xw1 || !ok;
      const int slot = warp * 2 + (last ? 1 : 0);
      // in the order of the products' results, 16 bytes a lane: by rows of the output the stores would fall on two banks
      float4* to = reinterpret_cast<float4*>(last ? reinterpret_cast<float*>(smem + warp * C::kRingWarp)
                                                  : p.piece_o + (static_cast<long long>(blockIdx.x) * W + warp) * (H * D)) + lane;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (ok) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            to[(nt * (D / 16) + i) * 32] = make_float4(o[nt][i][0] * unit, o[nt][i][1] * unit, o[nt][i][2] * unit, o[nt][i][3] * unit);
        }
        if (g == 0) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int col = nt * 8 + 2 * t + c;
            ml[slot * H + col] = m[nt][c];
            ml[(2 * W + slot) * H + col] = l[nt][c];
          }
        }
      }
      if (lane == 0) seg_of[slot] = b * hkv + h;
    }
    if (!ok) break;
  }
  // after a wait that gave up: the copies in flight land before the shared memory is given back (or this wait gives up too),
  // and what this warp would still have finished is NaN
  if (!ok) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    for (int x = xc; x < xi; x += step) {
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(bars + 8 * st, parity) && globaltimer_ns() - t0 < kWaitLimitNs) {}
      if (++st == S) { st = 0; parity ^= 1; }
    }
    for (int x = xw0; x < xw1;) {
      const int bb = seq_of(x), n = pre[bb + 1] - pre[bb], h = (x - pre[bb] * hkv) / n, first = pre[bb] * hkv + h * n;
      for (int i = lane; i < p.groups * D; i += 32) {
        store_o(bb, h * p.groups + i / D, i % D, __int_as_float(0x7fc00000));
        if (p.lse && i % D == 0) p.lse[static_cast<long long>(bb) * p.hq + h * p.groups + i / D] = __int_as_float(0x7fc00000);
      }
      x = first + n;
    }
  }

  // ---- pieces of one segment are joined, warps in order.  First the factors, a warp for each head and a lane for each piece;
  // pieces of one segment are neighbours among those there are: the last pieces of some warps, then perhaps a first piece
  __syncthreads();
  const bool failed = *cta_abort != 0;
  const int piece_seg = lane < 2 * W ? seg_of[lane] : -1;
  const uint32_t mates = __match_any_sync(0xffffffffu, piece_seg);
  const bool leads = piece_seg >= 0 && (mates & ((1u << lane) - 1u)) == 0u;
  const uint32_t leaders = __ballot_sync(0xffffffffu, leads);
  for (int head = warp; head < H; head += W) {   // unused columns, too: they are read in pairs
    const bool on = piece_seg >= 0;
    const float mine = on ? ml[lane * H + head] : -INFINITY, sum = on ? ml[(2 * W + lane) * H + head] : 0.0f;
    float top = -INFINITY, den = 0.0f;
#pragma unroll
    for (int e = 0; e < 2 * W; ++e) {
      const float x = __shfl_sync(0xffffffffu, mine, e);
      if ((mates >> e) & 1u) top = fmaxf(top, x);
    }
    // (a NaN sum has no maximum of its own)
    const float f = sum != 0.0f ? ex2_approx(mine == -INFINITY ? 0.0f : mine - top) : 0.0f;
    const float share_of = f * sum;
#pragma unroll
    for (int e = 0; e < 2 * W; ++e) {
      const float x = __shfl_sync(0xffffffffu, share_of, e);
      if ((mates >> e) & 1u) den += x;
    }
    if (on) {
      ml[lane * H + head] = den != 0.0f ? f / den : 0.0f;
      ml[(2 * W + lane) * H + head] = den != 0.0f ? log2f(den) + (top == -INFINITY ? 0.0f : top) : top;
    }
  }
  __syncthreads();
  // then the sums, in the order in which the pieces lie: four of a lane's results at a time
  const int chains = __popc(leaders);
  for (int i = tid; i < chains * (H * D / 4); i += NTHR) {
    const int chain = i / (H * D / 4), at = i % (H * D / 4), nt = at / (D / 16 * 32), fi = at / 32 % (D / 16), fl = at % 32;
    const int col = nt * 8 + 2 * (fl & 3);
    if (col >= p.groups) continue;
    uint32_t from = leaders;
    for (int c = 0; c < chain; ++c) from &= from - 1u;
    const int e0 = __ffs(from) - 1, seg = seg_of[e0];
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int e = e0; e < 2 * W; ++e) {
      const int es = seg_of[e];
      if (es < 0) continue;
      if (es != seg) break;
      const float2 f = *reinterpret_cast<const float2*>(ml + e * H + col);
      const float4 x = reinterpret_cast<const float4*>((e & 1) ? reinterpret_cast<const float*>(smem + (e >> 1) * C::kRingWarp)
                                                               : p.piece_o + (static_cast<long long>(blockIdx.x) * W + (e >> 1)) * (H * D))[at];
      acc.x += f.x * x.x; acc.y += f.y * x.y; acc.z += f.x * x.z; acc.w += f.y * x.w;
    }
    float2 lse = *reinterpret_cast<const float2*>(ml + (2 * W + e0) * H + col);
    if (failed) acc.x = acc.y = acc.z = acc.w = lse.x = lse.y = __int_as_float(0x7fc00000);
    const int sb = seg / hkv, h = seg % hkv, n = pre[sb + 1] - pre[sb], first = pre[sb] * hkv + h * n;
    const bool inside = first >= x0 && first + n <= x1;
    if (p.clusters) {
      reinterpret_cast<float4*>(share)[at] = acc;
      if (at % (D / 16 * 32) < 4) { share[H * D + col] = lse.x; share[H * D + col + 1] = lse.y; }
      continue;
    }
    const int fg = fl >> 2, d0 = kNative ? 16 * fi + fg : (D / 8) * fg + 2 * fi, d1 = kNative ? d0 + 8 : d0 + 1;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (col + c >= p.groups) break;
      float a0 = c ? acc.y : acc.x, a1 = c ? acc.w : acc.z, l1 = c ? lse.y : lse.x;
      const int hq = h * p.groups + col + c;
      if (inside) {
        if (l1 == kAllMinusInf) a1 = __int_as_float(0x7fc00000);
        settle_minus_inf(a0, l1);
        store_o(sb, hq, d0, a0);
        store_o(sb, hq, d1, a1);
        if (at % (D / 16 * 32) < 4 && p.lse) p.lse[static_cast<long long>(sb) * p.hq + hq] = l1;
      } else {
        const long long part = (static_cast<long long>(blockIdx.x) + seg) * p.groups + col + c;
        p.part_o[part * D + d0] = a0;
        p.part_o[part * D + d1] = a1;
        if (at % (D / 16 * 32) < 4) p.part_lse[part] = l1;
      }
    }
  }
  }
  if (!p.clusters) return;

  // ---- a cluster's parts of one segment: every CTA joins an eighth of the columns' channels
  cluster_barrier();
  {
    const int rank = blockIdx.x % kPagedCluster, seg = blockIdx.x / kPagedCluster, sb = seg / hkv, h = seg % hkv;
    constexpr int kMine = H * D / 4 / kPagedCluster;
    const uint32_t at_o = sbase + C::share_off(p.batch), at_lse = at_o + H * D * 4;
    if (pre[sb + 1] > pre[sb])
      for (int i = tid; i < kMine; i += NTHR) {
        const int at = rank * kMine + i, nt = at / (D / 16 * 32), fi = at / 32 % (D / 16), fl = at % 32, col = nt * 8 + 2 * (fl & 3);
        if (col >= p.groups) continue;
        float2 lse[kPagedCluster], top = make_float2(-INFINITY, -INFINITY), den = make_float2(0.0f, 0.0f);
        float4 x[kPagedCluster], acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int r = 0; r < kPagedCluster; ++r) {
          lse[r] = cluster_load2(cluster_address(at_lse + col * 4, r));
          x[r] = cluster_load4(cluster_address(at_o + at * 16, r));
        }
#pragma unroll
        for (int r = 0; r < kPagedCluster; ++r) { top.x = fmaxf(top.x, lse[r].x); top.y = fmaxf(top.y, lse[r].y); }
#pragma unroll
        for (int r = 0; r < kPagedCluster; ++r) {
          // a part without keys has an LSE of -inf and whatever the memory held
          const float f0 = lse[r].x == -INFINITY ? 0.0f : ex2_approx(lse[r].x - top.x), f1 = lse[r].y == -INFINITY ? 0.0f : ex2_approx(lse[r].y - top.y);
          if (lse[r].x != -INFINITY) { acc.x += f0 * x[r].x; acc.z += f0 * x[r].z; }
          if (lse[r].y != -INFINITY) { acc.y += f1 * x[r].y; acc.w += f1 * x[r].w; }
          den.x += f0;
          den.y += f1;
        }
        const int fg = fl >> 2, d0 = kNative ? 16 * fi + fg : (D / 8) * fg + 2 * fi, d1 = kNative ? d0 + 8 : d0 + 1;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (col + c >= p.groups) break;
          const float sum = c ? den.y : den.x;
          float inv = sum != 0.0f ? 1.0f / sum : 0.0f, l1 = sum != 0.0f ? log2f(sum) + (c ? top.y : top.x) : -INFINITY;
          settle_minus_inf(inv, l1);
          const int hq = h * p.groups + col + c;
          store_o(sb, hq, d0, (c ? acc.y : acc.x) * inv);
          store_o(sb, hq, d1, (c ? acc.w : acc.z) * inv);
          if (at % (D / 16 * 32) < 4 && p.lse) p.lse[static_cast<long long>(sb) * p.hq + hq] = l1;
        }
      }
  }
  cluster_barrier();   // nobody leaves while its shared memory is being read
}

// Joins the partial results of segments that lie in several CTAs.  Segment s = b * Hkv + h of tiles [first, last) has a part
// from each of the CTAs first / per .. (last - 1) / per, at index CTA + s.  A CTA here takes one query head: of every segment
// (grid Hq x B), or where there are more segments than cuts of the segment that is cut first at CTA y + 1 (grid group x cuts).
template <int D>
__global__ void __launch_bounds__(128 * kMergeGroups) paged_merge_kernel(const __grid_constant__ PagedDecodeParams p, const int by_cut) {
  __shared__ MergeScratch sm;
  griddep_launch();
  griddep_wait();
  const bool failed = cta_device_failed();
  int b = blockIdx.y, h = blockIdx.x / p.groups;
  const int head = blockIdx.x % p.groups;
  if (by_cut) {
    const int seg = p.cut[blockIdx.y + 1];
    if (failed) {   // then there may be no cuts: some CTA or other writes every row
      for (long long row = blockIdx.y; row < static_cast<long long>(p.batch) * p.pool.hkv; row += gridDim.y)
        if (threadIdx.x < D) {
          const int rb = static_cast<int>(row / p.pool.hkv), hq = static_cast<int>(row % p.pool.hkv) * p.groups + head;
          const float nan = __int_as_float(0x7fc00000);
          reinterpret_cast<uint16_t*>(p.o)[rb * p.o_sb + hq * p.o_sh + threadIdx.x] = p.o_bf16 ? from_f32<true>(nan) : from_f32<false>(nan);
          if (threadIdx.x == 0 && p.lse) p.lse[static_cast<long long>(rb) * p.hq + hq] = nan;
        }
      return;
    }
    if (seg < 0) return;
    b = seg / p.pool.hkv;
    h = seg % p.pool.hkv;
  }
  const int hq = h * p.groups + head;
  float val = __int_as_float(0x7fc00000), lse = val;
  if (!failed) {
    const int n = p.plan[b + 1] - p.plan[b], per = p.plan[p.batch + 1];
    if (n == 0) return;
    const int first = p.plan[b] * p.pool.hkv + h * n;
    const int c0 = first / per, c1 = (first + n - 1) / per;
    if (c0 == c1) return;
    const long long base = (static_cast<long long>(c0) + b * p.pool.hkv + h) * p.groups + head;
    merge_row_partials(p.part_o, p.part_lse, base, p.groups, c1 - c0 + 1, D, sm, val, lse);
    settle_minus_inf(val, lse);
  }
  if (threadIdx.x < D) {
    reinterpret_cast<uint16_t*>(p.o)[b * p.o_sb + hq * p.o_sh + threadIdx.x] = p.o_bf16 ? from_f32<true>(val) : from_f32<false>(val);
    if (threadIdx.x == 0 && p.lse) p.lse[static_cast<long long>(b) * p.hq + hq] = lse;
  }
}

}  // namespace sq
