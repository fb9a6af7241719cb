// Attention of one new token per sequence over a paged key/value cache, over all pages or over listed ones.
//
// Memory bound: per key and KV head 2 * row bytes (+ 8 for codes) are read once for all query heads of the group.
//
// Work.  A tile is 32 keys of one (sequence, KV head) segment.  All tiles of all segments stand in one row, and every CTA
// takes an equal stretch of it, whatever the lengths, which the kernel reads itself; so a captured launch stays balanced
// while the cache grows, and a ragged batch needs no plan.  A segment that lies in one CTA is finished there, one that is
// cut leaves partial results for paged_merge_kernel.
//
// Copies.  A warp is its own producer: it keeps kStages of its tiles in flight in a ring of its own (TMA boxes of 16 or 32
// rows, 128-byte swizzle, scales by bulk copies), so that warps never wait for one another between segments, and the ring
// runs on across segments.  Where a tile's pages lie is looked up by one lane per tile, 32 tiles at a time.
//
// Arithmetic.  S^T = K Q^T and O^T = V^T P^T on mma.sync m16n8k16 with the keys (channels) as rows and the query heads as
// the 8 columns: with at most 8 heads to a group no product is padding but the unused heads' columns.  The products do not
// bound the kernel (a key takes 0.25 KFLOP a head for 128-512 bytes), so the tcgen05 path, which would need 64 or 128
// rows of queries, has nothing to give here.
//   codes: int8 and 4-bit codes become f16 exactly by exponent tricks; q is brought to f16 by a power of two per head
//     (bf16's 8 bits are kept), a key's scale multiplies its scores and a value's scale its weight p, in fp32.  The weight
//     p * scale is rounded to f16 relative to the largest value scale so far (as a power of two), 2^14 high.
//   native: p is split into two 16-bit parts, so that its rounding (2^-16 or 2^-22) vanishes beside the output's.
// Channels and keys may enter a product in any order as long as both operands agree, so codes are taken from shared memory
// in the order in which they lie (16 bytes a lane); `row_perm` below orders the keys so that those loads do not collide.
#pragma once
#include <cuda.h>

#include "decode.cuh"
#include "paged_cache.cuh"

namespace sq {

constexpr int kPagedTile = 32;
constexpr int kPagedMaxBatch = 1024;

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
  int batch, hq, groups, q_bf16, o_bf16;
  int min_tiles;     // a CTA takes at least so many
  float scale_log2;  // softmax scale * log2(e)
  float* part_o;     // [grid + B * Hkv, groups, D] fp32, each divided by its own sum
  float* part_lse;   // [grid + B * Hkv, groups]
  int* plan;         // [B + 2]: tiles per KV head before each sequence, then tiles per CTA
};

template <int FMT, int D, int NT>
struct PagedDecodeCfg {
  static constexpr int kRow = kv_row_bytes<FMT>(D);
  static constexpr int kWarps = (FMT == kKvNative && D == 128) ? 4 : 8;
  static constexpr int kStages = FMT == kKvNative ? (D == 128 && NT == 1 ? 3 : 2) : (FMT == kKvInt8 && D == 128 ? 2 : 4);
  static constexpr int kTensor = kPagedTile * kRow;                      // a tile's keys or values
  static constexpr int kRing = kWarps * kStages * 2 * kTensor;
  static constexpr int kScaleOff = kRing;                                // [warp][stage][K, V][32] fp32
  static constexpr int kScales = FMT == kKvNative ? 0 : kWarps * kStages * 256;
  static constexpr int kRedOff = kScaleOff + kScales;                    // [warp][8 NT][D] fp32
  static constexpr int kMlOff = kRedOff + kWarps * 8 * NT * D * 4;       // [warp][8 NT] maxima, then sums
  static constexpr int kBarOff = kMlOff + kWarps * 8 * NT * 8;           // [warp][stage]
  static constexpr int kInfoOff = kBarOff + kWarps * kStages * 8;        // [warp][stage] valid keys
  static constexpr int kMiscOff = kInfoOff + kWarps * kStages * 4;       // abort flag
  static constexpr int kPlanOff = (kMiscOff + 16 + 15) / 16 * 16;        // [B + 1]
  static constexpr int total(int batch) { return kPlanOff + (batch + 1) * 4 + 1024; }
  static_assert(total(kPagedMaxBatch) <= 227 * 1024, "shared memory of a CTA");
};

// untiled copy global -> shared, completion counted in bytes on `bar`
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t h2_add(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// Codes to f16 pairs, exactly.  The bits of a biased code (sign bit flipped) under the exponent of 1024 are 1024 + code + bias.
//   bytes 0, 2 of x / bytes 1, 3 of x;   nibbles 0, 4 / 1, 5 / 2, 6 / 3, 7 of x (the odd ones arrive 16 times as large)
__device__ __forceinline__ void bytes_to_h2(uint32_t x, uint32_t& even, uint32_t& odd) {
  constexpr uint32_t kMinus1152 = 0xe480e480u;
  even = h2_add((x & 0x00ff00ffu) ^ 0x64806480u, kMinus1152);
  odd = h2_add(((x >> 8) & 0x00ff00ffu) ^ 0x64806480u, kMinus1152);
}
__device__ __forceinline__ void nibbles_to_h2(uint32_t x, uint32_t& n0, uint32_t& n1) {
  constexpr uint32_t kMinus1032 = 0xe408e408u, kSixteenth = 0x2c002c00u, kMinus72 = 0xd480d480u;
  n0 = h2_add((x & 0x000f000fu) ^ 0x64086408u, kMinus1032);
  n1 = h2_fma((x & 0x00f000f0u) ^ 0x64806480u, kSixteenth, kMinus72);
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
__device__ __forceinline__ int paged_tiles(const PagedDecodeParams& p, int len) {
  if (len == 0) return 0;
  const long long keys = p.list ? static_cast<long long>(p.list_len) << p.pool.ps_shift : len;
  return static_cast<int>((keys + kPagedTile - 1) / kPagedTile);
}

template <int FMT, int D, bool BF16, int NT>
__global__ void __launch_bounds__(PagedDecodeCfg<FMT, D, NT>::kWarps * 32, 1)
paged_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ PagedDecodeParams p) {
  using C = PagedDecodeCfg<FMT, D, NT>;
  constexpr int W = C::kWarps, S = C::kStages, ROW = C::kRow, NTHR = W * 32, H = 8 * NT;
  constexpr bool kNative = FMT == kKvNative;
  griddep_launch();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int hkv = p.pool.hkv;
  auto store_o = [&](int b, int hq, int d, float x) {
    reinterpret_cast<uint16_t*>(p.o)[b * p.o_sb + hq * p.o_sh + d] = p.o_bf16 ? from_f32<true>(x) : from_f32<false>(x);
  };
  // after a wait has given up on this device, here or in an earlier launch, the caller gets NaN and no stale memory
  if (cta_device_failed()) {
    const float nan = __int_as_float(0x7fc00000);
    const long long rows = static_cast<long long>(p.batch) * p.hq;
    for (long long i = blockIdx.x * static_cast<long long>(NTHR) + tid; i < rows * D; i += static_cast<long long>(gridDim.x) * NTHR) {
      const long long row = i / D;
      store_o(static_cast<int>(row / p.hq), static_cast<int>(row % p.hq), static_cast<int>(i % D), nan);
      if (p.lse && i % D == 0) p.lse[row] = nan;
    }
    return;
  }
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  volatile int* cta_abort = reinterpret_cast<volatile int*>(smem + C::kMiscOff);
  int* pre = reinterpret_cast<int*>(smem + C::kPlanOff);
  float* red = reinterpret_cast<float*>(smem + C::kRedOff);
  float* ml = reinterpret_cast<float*>(smem + C::kMlOff);
  const uint32_t bars = sbase + C::kBarOff + warp * S * 8;
  volatile int* info = reinterpret_cast<volatile int*>(smem + C::kInfoOff) + warp * S;

  // ---- plan: tiles (of one KV head) before each sequence
  if (warp == 0) {
    int run = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      const int b = b0 + lane;
      const int mine = b < p.batch ? paged_tiles(p, paged_len(p, b)) : 0;
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
  } else if (warp == 1 && lane == 0) {
    *cta_abort = 0;
    for (int i = 0; i < W * S; ++i) mbar_init(sbase + C::kBarOff + 8 * i, 1);
    fence_barrier_init();
    fence_proxy_async();
  }
  __syncthreads();
  const long long total = static_cast<long long>(pre[p.batch]) * hkv;
  const long long share = (total + gridDim.x - 1) / gridDim.x;
  const int per = static_cast<int>(share > p.min_tiles ? share : p.min_tiles);
  if (blockIdx.x == 0) {
    for (int b = tid; b <= p.batch; b += NTHR) p.plan[b] = pre[b];
    if (tid == 0) p.plan[p.batch + 1] = per;
  }
  // sequences without keys: zeros
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
    if (pre[b + 1] == pre[b])
      for (int i = tid; i < p.hq * D; i += NTHR) {
        store_o(b, i / D, i % D, 0.0f);
        if (p.lse && i % D == 0) p.lse[static_cast<long long>(b) * p.hq + i / D] = -INFINITY;
      }
  const long long x0 = static_cast<long long>(blockIdx.x) * per;
  const long long x1 = min(total, x0 + per);
  if (x0 >= x1) return;

  // sequence of tile x
  auto seq_of = [&](long long x) {
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (static_cast<long long>(pre[mid]) * hkv <= x) lo = mid; else hi = mid;
    }
    return lo;
  };

  // ---- copies.  Lane i looks up the i-th of the warp's next 32 tiles: rec_ph page * Hkv + head of its (one or two) pages,
  // rec_row the first row inside the page, rec_nv the valid keys of its first and second half
  const int ps = 1 << p.pool.ps_shift;
  const uint32_t ring = sbase + warp * (S * 2 * C::kTensor);
  const uint32_t scales = sbase + C::kScaleOff + warp * S * 256;
  int rec_ph[2], rec_row = 0, rec_nv = 0;
  auto look_up = [&](long long x) {
    rec_ph[0] = rec_ph[1] = 0;
    rec_row = rec_nv = 0;
    if (x >= x1) return;
    const int b = seq_of(x);
    const int n = pre[b + 1] - pre[b];
    const long long rem = x - static_cast<long long>(pre[b]) * hkv;
    const int h = static_cast<int>(rem / n);
    const int key = static_cast<int>(rem % n) * kPagedTile;
    const int len = paged_len(p, b);
    const int held = static_cast<int>((static_cast<long long>(len) + ps - 1) >> p.pool.ps_shift);
    rec_row = key & (ps - 1);
#pragma unroll
    for (int s = 0; s < 2; ++s) {   // the tile's halves lie in one page unless pages have 16 rows
      const int at = (key + 16 * s) >> p.pool.ps_shift;
      int index = at;
      if (p.list) index = at < p.list_len ? p.list[(static_cast<long long>(b) * hkv + h) * p.list_len + at] : -1;
      if (index < 0 || index >= held) continue;
      const int page = page_of(p.table, b, index, p.pool.num_pages);
      if (page < 0) continue;
      rec_ph[s] = page * hkv + h;
      const long long left = len - ((static_cast<long long>(index) << p.pool.ps_shift) + ((key + 16 * s) & (ps - 1)));
      rec_nv |= static_cast<int>(min(max(left, 0ll), 16ll)) << (8 * s);
    }
  };
  long long xi = x0 + warp;  // next tile to copy
  int ahead = 32;            // place of that tile among the looked-up ones
  auto issue = [&](int st) {
    if (xi >= x1) return;
    if (ahead == 32) {
      look_up(xi + static_cast<long long>(lane) * W);
      ahead = 0;
    }
    const int ph0 = __shfl_sync(0xffffffffu, rec_ph[0], ahead), ph1 = __shfl_sync(0xffffffffu, rec_ph[1], ahead);
    const int row = __shfl_sync(0xffffffffu, rec_row, ahead), nv = __shfl_sync(0xffffffffu, rec_nv, ahead);
    ++ahead;
    xi += W;
    if (lane == 0) {
      info[st] = nv;
      const uint32_t bar = bars + 8 * st, dst = ring + st * (2 * C::kTensor), sdst = scales + st * 256;
      const bool a = (nv & 0xff) != 0, b = (nv >> 8) != 0;
      if (kNative || p.pool.ps_shift == 4) {
        // boxes of 16 rows
        constexpr int kBox = 16 * ROW, kBlk = kNative ? 16 : 16 * ROW / 128;
        constexpr uint32_t kBytes = 2 * kBox + (kNative ? 0 : 128);
        mbar_expect_tx(bar, (a ? kBytes : 0u) + (b ? kBytes : 0u));
        const int row1 = p.pool.ps_shift == 4 ? 0 : row + 16;
#pragma unroll
        for (int s = 0; s < 2; ++s)
          if (s ? b : a) {
            const int ph = s ? ph1 : ph0, r = s ? row1 : row;
            tma_load_4d(dst + s * kBox, &tm_k, bar, 0, r / 16 * kBlk, 0, ph);
            tma_load_4d(dst + C::kTensor + s * kBox, &tm_v, bar, 0, r / 16 * kBlk, 0, ph);
            if (!kNative) {
              const long long off = (static_cast<long long>(ph) << p.pool.ps_shift) + r;
              bulk_load(sdst + s * 64, p.pool.k_scale + off, 64, bar);
              bulk_load(sdst + 128 + s * 64, p.pool.v_scale + off, 64, bar);
            }
          }
      } else {
        // one box of 32 rows
        mbar_expect_tx(bar, a ? 2u * C::kTensor + 256u : 0u);
        if (a) {
          tma_load_4d(dst, &tm_k, bar, 0, row / 32 * (32 * ROW / 128), 0, ph0);
          tma_load_4d(dst + C::kTensor, &tm_v, bar, 0, row / 32 * (32 * ROW / 128), 0, ph0);
          const long long off = (static_cast<long long>(ph0) << p.pool.ps_shift) + row;
          bulk_load(sdst, p.pool.k_scale + off, 128, bar);
          bulk_load(sdst + 128, p.pool.v_scale + off, 128, bar);
        }
      }
    }
    __syncwarp();
  };
#pragma unroll 1
  for (int st = 0; st < S; ++st) issue(st);

  // ---- where this lane's pieces of a tile lie
  uint32_t koff[2][2][2], voff[2][4];  // codes: [half of the tile][rows 0-7, 8-15][piece], [half][rows 2t, 2t+1, 2t+8, 2t+9]
  uint32_t kx[4], vx[4];               // native: 16-byte chunks (by ldmatrix lane) of channels 16 i .. 16 i + 15 within 64
  if (kNative) {
    const int kr = (lane & 7) + ((lane >> 3) & 1) * 8, kc = lane >> 4;
    const int vr = (lane & 7) + (lane >> 4) * 8, vc = (lane >> 3) & 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kx[i] = kr * 128 + (((2 * i + kc) ^ (kr & 7)) << 4);
      vx[i] = C::kTensor + vr * 128 + (((2 * i + vc) ^ (vr & 7)) << 4);
    }
  } else {
    constexpr int kPiece = ROW == 32 ? 8 : 16, kPieces = ROW == 128 ? 2 : 1;  // keys: ROW / 4 bytes a lane; values: ROW / 8
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int hi = 0; hi < 2; ++hi)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          koff[mt][hi][j] = swizzle128((mt * 16 + hi * 8 + row_perm<ROW>(g)) * ROW + (t * kPieces + (j < kPieces ? j : 0)) * kPiece);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        voff[mt][i] = C::kTensor + swizzle128((mt * 16 + (i >> 1) * 8 + row_perm<ROW>(2 * t + (i & 1))) * ROW + g * (ROW / 8));
    }
  }
  const int key_row = kNative ? g : row_perm<ROW>(g);  // this lane's first key in a half: that row and the one 8 further

  int st = 0;
  uint32_t parity = 0;
  bool ok = true;
  long long xc = x0 + warp;
  int b = seq_of(x0);
  for (long long seg_x = x0; seg_x < x1;) {
    // ---- segment (b, h): tiles [seg_x, seg_end) of it are this CTA's
    while (static_cast<long long>(pre[b + 1]) * hkv <= seg_x) ++b;
    const int n = pre[b + 1] - pre[b];
    const long long b_start = static_cast<long long>(pre[b]) * hkv;
    const int h = static_cast<int>((seg_x - b_start) / n);
    const long long seg_first = b_start + static_cast<long long>(h) * n, seg_last = seg_first + n;
    const long long seg_end = min(seg_last, x1);

    // ---- query heads as the products' 8 columns
    uint32_t qb[NT][D / 16][2];
    float cs[NT][2];  // score factor of this lane's two columns
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
            qb[nt][kk][r] = head < p.groups ? static_cast<uint32_t>(src[d]) | (static_cast<uint32_t>(src[d + 1]) << 16) : 0u;
          }
        cs[nt][0] = cs[nt][1] = p.scale_log2;
      } else {
        float f[D / 4], top = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 4; ++i) {
          // the lane's i-th channel in the order in which its codes are taken from shared memory
          const int d = FMT == kKvInt4 ? t * (D / 4) + i : (D == 128 ? (2 * t + i / 16) * 16 + i % 16 : t * 16 + i);
          const uint16_t v = head < p.groups ? src[d] : static_cast<uint16_t>(0);
          f[i] = p.q_bf16 ? to_f32<true>(v) : to_f32<false>(v);
          top = fmaxf(top, fabsf(f[i]));
          if (f[i] != f[i]) top = INFINITY;
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // a power of two brings the largest to [2^13, 2^14)
        const uint32_t e = max(__float_as_uint(top) >> 23, 27u);
        const float up = __uint_as_float((267u - e) << 23);
        const float down = p.scale_log2 * __uint_as_float((e - 13u) << 23);
#pragma unroll
        for (int w = 0; w < D / 16; ++w) {
          if (FMT == kKvInt8) {   // bytes 0, 2 and 1, 3 of word w
            qb[nt][w][0] = pack_f16x2(f[4 * w] * up, f[4 * w + 2] * up);
            qb[nt][w][1] = pack_f16x2(f[4 * w + 1] * up, f[4 * w + 3] * up);
          } else {                // nibbles 0, 4 and 1, 5, then 2, 6 and 3, 7 of word w / 2
            const int o = 8 * (w / 2) + 2 * (w & 1);
            qb[nt][w][0] = pack_f16x2(f[o] * up, f[o + 4] * up);
            qb[nt][w][1] = pack_f16x2(f[o + 1] * up, f[o + 5] * up);
          }
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
    const bool any_tile = xc < seg_end;

    for (; ok && xc < seg_end; xc += W) {
      ok = mbar_wait_warp(bars + 8 * st, parity, cta_abort, 401);
      if (!ok) break;
      const int nv = info[st];
      const uint32_t tile = ring + st * (2 * C::kTensor);
      if (nv != 0) {
        if (kNative && nv != 0x1010) {
          // rows behind the sequence (or of a page that is not there) may hold anything: zeros, so that 0 * x is 0
          for (int i = lane; i < 32 * (ROW / 16); i += 32) {
            const int r = i / (ROW / 16), c = i % (ROW / 16);
            if ((r & 15) >= ((nv >> (8 * (r >> 4))) & 0xff))
              *reinterpret_cast<uint4*>(smem + (tile - sbase) + C::kTensor + (r >> 4) * (16 * ROW) + (c >> 3) * 2048 + (r & 15) * 128 + (c & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
          __syncwarp();
        }
        // ---- scores
        float s[NT][2][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) s[nt][mt][0] = s[nt][mt][1] = s[nt][mt][2] = s[nt][mt][3] = 0.0f;
        float vs[2][2];  // value scales of this lane's keys
        if (kNative) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              uint32_t a[4];
              ldmatrix_x4(tile + kx[kk & 3] + mt * (16 * ROW) + (kk >> 2) * 2048, a[0], a[1], a[2], a[3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_16816<BF16>(s[nt][mt], a, qb[nt][kk][0], qb[nt][kk][1]);
            }
        } else {
          const uint8_t* tp = smem + (tile - sbase);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            constexpr int kWords = ROW / 16;  // 4-byte words of a key per lane
            uint32_t w[2][kWords];
#pragma unroll
            for (int hi = 0; hi < 2; ++hi)
#pragma unroll
              for (int j = 0; j < (kWords + 3) / 4; ++j) {
                if (kWords == 2) {
                  const uint2 v = *reinterpret_cast<const uint2*>(tp + koff[mt][hi][0]);
                  w[hi][0] = v.x; w[hi][1] = v.y;
                } else {
                  const uint4 v = *reinterpret_cast<const uint4*>(tp + koff[mt][hi][j]);
                  w[hi][4 * j] = v.x; w[hi][4 * j + 1] = v.y; w[hi][4 * j + 2] = v.z; w[hi][4 * j + 3] = v.w;
                }
              }
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
              if (FMT == kKvInt8) {
                uint32_t a[4];
                bytes_to_h2(w[0][i], a[0], a[2]);
                bytes_to_h2(w[1][i], a[1], a[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_16816<false>(s[nt][mt], a, qb[nt][i][0], qb[nt][i][1]);
              } else {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  uint32_t a[4];
                  nibbles_to_h2(w[0][i] >> (8 * u), a[0], a[2]);
                  nibbles_to_h2(w[1][i] >> (8 * u), a[1], a[3]);
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt) mma_16816<false>(s[nt][mt], a, qb[nt][2 * i + u][0], qb[nt][2 * i + u][1]);
                }
              }
            }
          }
          // scales
          const float* sc = reinterpret_cast<const float*>(smem + C::kScaleOff + (warp * S + st) * 256);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
              const float ks = sc[mt * 16 + hi * 8 + key_row];
              vs[mt][hi] = sc[32 + mt * 16 + hi * 8 + key_row];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) { s[nt][mt][2 * hi] *= ks; s[nt][mt][2 * hi + 1] *= ks; }
            }
        }
        if (nv != 0x1010) {
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi)
              if (hi * 8 + key_row >= ((nv >> (8 * mt)) & 0xff)) {
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
            float x = fmaxf(fmaxf(s[nt][0][c], s[nt][0][c + 2]), fmaxf(s[nt][1][c], s[nt][1][c + 2]));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            m_new[nt][c] = fmaxf(m[nt][c], x);
            moved |= m_new[nt][c] > m[nt][c];
          }
        uint32_t vexp_new = vexp;
        if (!kNative) {
          const uint32_t top = __float_as_uint(fmaxf(fmaxf(vs[0][0], vs[0][1]), fmaxf(vs[1][0], vs[1][1])));
          vexp_new = max(vexp, __reduce_max_sync(0xffffffffu, top) & 0x7f800000u);
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
        // ---- weights, 2^14 high, and their two 16-bit parts (native) or products with the value scales (codes)
        uint32_t pb[NT][2][2], pl[NT][2][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float off[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) off[c] = 14.0f - (m[nt][c] == -INFINITY ? 0.0f : m[nt][c] * cs[nt][c]);
          const float inv = __uint_as_float((254u << 23) - vexp);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
              float w0 = ex2_approx(fmaf(s[nt][mt][2 * hi], cs[nt][0], off[0]));
              float w1 = ex2_approx(fmaf(s[nt][mt][2 * hi + 1], cs[nt][1], off[1]));
              l[nt][0] += w0;
              l[nt][1] += w1;
              if (kNative) {
                const uint32_t head = BF16 ? pack_bf16x2(w0, w1) : pack_f16x2(w0, w1);
                const float h0 = to_f32<BF16>(static_cast<uint16_t>(head & 0xffffu)), h1 = to_f32<BF16>(static_cast<uint16_t>(head >> 16));
                pb[nt][mt][hi] = movmatrix_trans(head);
                pl[nt][mt][hi] = movmatrix_trans(BF16 ? pack_bf16x2(w0 - h0, w1 - h1) : pack_f16x2(w0 - h0, w1 - h1));
              } else {
                const float f = vs[mt][hi] * inv;
                pb[nt][mt][hi] = movmatrix_trans(pack_f16x2(w0 * f, w1 * f));
              }
            }
        }
        // ---- values
        if (kNative) {
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              uint32_t a[4];
              ldmatrix_x4_trans(tile + vx[i & 3] + mt * (16 * ROW) + (i >> 2) * 2048, a[0], a[1], a[2], a[3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_16816<BF16>(o[nt][i], a, pb[nt][mt][0], pb[nt][mt][1]);
                mma_16816<BF16>(o[nt][i], a, pl[nt][mt][0], pl[nt][mt][1]);
              }
            }
        } else {
          const uint8_t* tp = smem + (tile - sbase);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            constexpr int kWords = ROW / 32;
            uint32_t w[4][kWords];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (kWords == 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(tp + voff[mt][i]);
                w[i][0] = v.x; w[i][1 % kWords] = v.y; w[i][2 % kWords] = v.z; w[i][3 % kWords] = v.w;
              } else if (kWords == 2) {
                const uint2 v = *reinterpret_cast<const uint2*>(tp + voff[mt][i]);
                w[i][0] = v.x; w[i][1 % kWords] = v.y;
              } else {
                w[i][0] = *reinterpret_cast<const uint32_t*>(tp + voff[mt][i]);
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
                  bytes_to_h2(lo, a[0], a[1]);
                  bytes_to_h2(hi, a[2], a[3]);
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt) mma_16816<false>(o[nt][2 * u + half], a, pb[nt][mt][0], pb[nt][mt][1]);
                } else {
#pragma unroll
                  for (int q = 0; q < 2; ++q) {
                    uint32_t a[4];
                    nibbles_to_h2(lo >> (8 * q), a[0], a[1]);
                    nibbles_to_h2(hi >> (8 * q), a[2], a[3]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_16816<false>(o[nt][4 * u + 2 * half + q], a, pb[nt][mt][0], pb[nt][mt][1]);
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

    // ---- the warps' results of this segment: sums over the lanes of a column, then through shared memory
    __syncthreads();  // everyone is done reading the previous segment's
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], sh);
        if (g == 0) {
          const int col = nt * 8 + 2 * t + c;
          ml[warp * H + col] = m[nt][c] == -INFINITY ? -INFINITY : m[nt][c] * cs[nt][c];
          ml[(W + warp) * H + col] = l[nt][c];
        }
      }
    if (any_tile) {
      const float unit = kNative ? 1.0f : __uint_as_float(vexp);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = kNative ? 16 * i + g + 8 * (e >> 1) : (D / 8) * g + 2 * i + (e >> 1);
            red[(warp * H + nt * 8 + 2 * t + (e & 1)) * D + d] = o[nt][i][e] * unit;
          }
    }
    __syncthreads();
    const bool whole = seg_first >= x0 && seg_last <= x1;
    const long long part = (blockIdx.x + static_cast<long long>(b) * hkv + h) * p.groups;
    const bool failed = *cta_abort != 0;
    for (int i = tid; i < p.groups * D; i += NTHR) {
      const int head = i / D, d = i % D;
      float top = -INFINITY, den = 0.0f, acc = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, ml[w * H + head]);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float lw = ml[(W + w) * H + head], mw = ml[w * H + head];
        if (lw != 0.0f) {  // a warp without keys here has written nothing else
          const float f = ex2_approx(mw == -INFINITY ? 0.0f : mw - top);
          den += f * lw;
          acc += f * red[(w * H + head) * D + d];
        }
      }
      const float nan = __int_as_float(0x7fc00000);
      float val = den != 0.0f ? acc / den : 0.0f;
      // 2^14 of the weights; a NaN sum has no maximum of its own
      float lse = den != 0.0f ? log2f(den) - 14.0f + (top == -INFINITY ? 0.0f : top) : -INFINITY;
      if (failed) val = lse = nan;
      if (whole) {
        store_o(b, h * p.groups + head, d, val);
        if (d == 0 && p.lse) p.lse[static_cast<long long>(b) * p.hq + h * p.groups + head] = lse;
      } else {
        p.part_o[(part + head) * D + d] = val;
        if (d == 0) p.part_lse[part + head] = lse;
      }
    }
    seg_x = seg_end;
  }
  // after a wait that gave up: the copies in flight land before the shared memory is given back (or this wait gives up too)
  if (!ok)
    for (; xc < xi; xc += W) {
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(bars + 8 * st, parity) && globaltimer_ns() - t0 < kWaitLimitNs) {}
      if (++st == S) { st = 0; parity ^= 1; }
    }
}

// Joins the partial results of segments that were cut: one CTA per query head.  Segment s = b * Hkv + h of tiles
// [first, last) has a part from each of the CTAs first / per .. (last - 1) / per, at index CTA + s.
template <int D>
__global__ void __launch_bounds__(128 * kMergeGroups) paged_merge_kernel(const __grid_constant__ PagedDecodeParams p) {
  __shared__ MergeScratch sm;
  griddep_launch();
  griddep_wait();
  const int hq = blockIdx.x, b = blockIdx.y, h = hq / p.groups;
  const bool failed = cta_device_failed();
  float val = __int_as_float(0x7fc00000), lse = val;
  if (!failed) {
    const int n = p.plan[b + 1] - p.plan[b], per = p.plan[p.batch + 1];
    if (n == 0) return;
    const long long first = static_cast<long long>(p.plan[b]) * p.pool.hkv + static_cast<long long>(h) * n;
    const long long c0 = first / per, c1 = (first + n - 1) / per;
    if (c0 == c1) return;
    const long long base = (c0 + static_cast<long long>(b) * p.pool.hkv + h) * p.groups + hq % p.groups;
    merge_row_partials(p.part_o, p.part_lse, base, p.groups, static_cast<int>(c1 - c0 + 1), D, sm, val, lse);
  }
  if (threadIdx.x < D) {
    reinterpret_cast<uint16_t*>(p.o)[b * p.o_sb + hq * p.o_sh + threadIdx.x] = p.o_bf16 ? from_f32<true>(val) : from_f32<false>(val);
    if (threadIdx.x == 0 && p.lse) p.lse[static_cast<long long>(b) * p.hq + hq] = lse;
  }
}

}  // namespace sq
