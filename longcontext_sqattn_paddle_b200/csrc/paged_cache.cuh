// The paged key/value cache: geometry of a layer's pool, the kernel that quantises new rows into pages and the one that
// reads rows back.
//
// A pool holds P pages of `page_size` tokens: [P, Hkv, page_size, D] for keys and for values, so that the rows of one page
// and head are one contiguous block (what the attention kernel loads).  Formats: the 16-bit values themselves, int8 codes,
// or 4-bit codes two to a byte (even channel in the low half); codes have one fp32 scale per row, [P, Hkv, page_size]:
//   s = max(fl32(max|x| * fl32(1/Q)), 2^-100), Q = 127 or 7,   code = nearest integer to x / s (ties to even),   value = code * s.
// A row with an infinity or a NaN gets the scale NaN and zero codes, so that it reads back as NaN.  The floor of the scale
// keeps 1/s finite for rows of (nearly) zeros.
// The paged kernels are launched with programmatic stream serialisation: they become resident while the kernel before them
// drains and wait for it before they read or write anything.  A decode step is a row of short kernels (append, score, pick,
// attend, each 3 to 15 us), and launch latency lies between them otherwise.
//
// k_bounds [P, Hkv, 2, D] (optional) holds the channel minima and maxima of the page's keys as they were given.
#pragma once
#include "prep.cuh"

namespace sq {

enum { kKvNative = 0, kKvInt8 = 1, kKvInt4 = 2 };

template <int FMT>
__host__ __device__ constexpr int kv_row_bytes(int d) { return FMT == kKvNative ? 2 * d : (FMT == kKvInt8 ? d : d / 2); }
template <int FMT>
__host__ __device__ constexpr float kv_code_step() { return FMT == kKvInt8 ? 1.0f / 127.0f : 1.0f / 7.0f; }
constexpr float kKvSmallestScale = 7.888609052210118e-31f;  // 2^-100

struct PagedPool {
  uint8_t *k_pages, *v_pages;
  float *k_scale, *v_scale;
  uint8_t* k_bounds;
  int num_pages, hkv, ps_shift;  // page_size = 1 << ps_shift
};

struct BlockTable {
  const int* ids;  // [batch, max_pages]
  long long stride;
  int max_pages;
};
// the page that holds a sequence's page `index`, -1 where the table or the id does not reach the pool
__device__ __forceinline__ int page_of(const BlockTable& t, int b, long long index, int num_pages) {
  if (index < 0 || index >= t.max_pages) return -1;
  const int id = t.ids[b * t.stride + index];
  return (id >= 0 && id < num_pages) ? id : -1;
}

// the smaller and the larger of two pairs, NaN where either is NaN
template <bool BF16>
__device__ __forceinline__ uint32_t min16x2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if (BF16) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t max16x2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if (BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Quantise one row spread over D / 8 consecutive lanes, 8 channels each; every lane gets the scale.  The codes come out as
// the integers' low bytes (int8) or nibbles (int4), packed in channel order.
//
// The code is the nearest integer to the exact quotient x / s.  The product with an approximate 1/s is off by at most
// 127 (2^-22 + 2^-24) < 4e-5 (the reciprocal's error, the product's rounding), so its nearest integer is the answer unless it
// lies within 1e-4 of a half-integer; there the remainder x - code * s decides, which one fused multiply-add gives exactly (x is
// a multiple of s's last place whenever code != 0, and the difference is below s in magnitude).  x = max/2 is the common case
// there.  The kernel is bound by issuing these instructions about as much as by memory, so fp32 goes in pairs.
template <int FMT, int D, bool BF16>
__device__ __forceinline__ void quantise_row8(const uint4& x, float& scale, uint32_t (&packed)[2]) {
  constexpr int kLanes = D / 8;
  constexpr uint32_t kNonFinite = BF16 ? 0x7f80u : 0x7c00u;
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: added, it leaves the nearest integer in the low bits
  uint32_t a = max16x2_nan<BF16>(max16x2_nan<BF16>(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), max16x2_nan<BF16>(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) a = max16x2_nan<BF16>(a, __shfl_xor_sync(0xffffffffu, a, o));
  const uint32_t top = max(a & 0x7fffu, (a >> 16) & 0x7fffu);
  const bool finite = top < kNonFinite;
  const float s = fmaxf(to_f32<BF16>(static_cast<uint16_t>(top)) * kv_code_step<FMT>(), kKvSmallestScale);
  scale = finite ? s : __int_as_float(0x7fc00000);
  const float inv = finite ? __fdividef(1.0f, s) : 0.0f;
  float f[8];
  unpack8<BF16>(x, f);
  uint32_t c[8];
  float off = 0.0f;  // how far from its integer the furthest of the products is
  const uint64_t inv2 = f32x2_pack(inv, inv), round2 = f32x2_pack(kRound, kRound);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t t = f32x2_mul(f32x2_pack(f[2 * i], f[2 * i + 1]), inv2), r = f32x2_add(t, round2), d = f32x2_sub(t, f32x2_sub(r, round2));
    float r0, r1, d0, d1;
    f32x2_unpack(r, r0, r1);
    f32x2_unpack(d, d0, d1);
    off = max3(off, fabsf(d0), fabsf(d1));
    c[2 * i] = __float_as_uint(r0);
    c[2 * i + 1] = __float_as_uint(r1);
  }
  if (off > 0.4999f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float r = __uint_as_float(c[i]) - kRound, e = __fmaf_rn(-r, s, f[i]), half = 0.5f * s;
      const bool odd = (c[i] & 1u) != 0u;
      if (e > half || (e == half && odd)) ++c[i];
      if (e < -half || (e == -half && odd)) --c[i];
    }
  }
  if (__any_sync(0xffffffffu, !finite)) {   // a branch that is hardly ever taken
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = finite ? c[i] : 0u;
  }
  if (FMT == kKvInt8) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      packed[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040), __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040), 0x5410);
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= (c[i] & 15u) << (4 * i);
    packed[0] = w;
  }
}

struct PagedWriteParams {
  PagedPool pool;
  BlockTable table;
  const uint8_t *k, *v;  // [B, rows, Hkv, D] through element strides
  long long k_sb, k_sh, k_sn, v_sb, v_sh, v_sn;
  int rows;
  const int* positions;  // [B] position of the first new row
  const int* counts;     // [B] or null: number of new rows
};

// One CTA per (KV head, page that new rows fall into, sequence): it alone writes that page's rows and bounds, so the bounds
// need no atomics.  D / 8 lanes hold a row, 8 channels each; the rows of the page are dealt to the CTA's lane groups, whose
// loads of kWriteRows rows are in flight together.  Heads are the fastest index, so that CTAs that run together read the pieces
// of the same rows.
constexpr int kWriteRows = 4;
template <int FMT, int D, bool BF16>
__global__ void __launch_bounds__(128, 6) paged_write_kernel(const __grid_constant__ PagedWriteParams p) {
  constexpr int kLanes = D / 8, kGroups = 128 / kLanes;
  griddep_launch();
  griddep_wait();
  const int b = blockIdx.z, h = blockIdx.x;
  const int ps = 1 << p.pool.ps_shift;
  const int pos = p.positions[b];
  const int count = p.counts ? min(max(p.counts[b], 0), p.rows) : p.rows;
  if (pos < 0) return;
  const long long index = (pos >> p.pool.ps_shift) + static_cast<long long>(blockIdx.y);
  const long long first = index * ps - pos;  // new row that falls on the page's row 0 (negative: the page was begun before)
  if (first >= count) return;
  const int page = page_of(p.table, b, index, p.pool.num_pages);   // looked at after the first rows have been asked for
  const int r0 = first < 0 ? static_cast<int>(-first) : 0;
  const int r1 = static_cast<int>(min(static_cast<long long>(ps), count - first));
  const int c = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const uint8_t* kb = p.k + 2 * (b * p.k_sb + h * p.k_sh + c * 8);
  const uint8_t* vb = p.v + 2 * (b * p.v_sb + h * p.v_sh + c * 8);
  constexpr uint32_t kInf = BF16 ? 0x7f807f80u : 0x7c007c00u, kMinusInf = BF16 ? 0xff80ff80u : 0xfc00fc00u;
  uint32_t lo[4] = {kInf, kInf, kInf, kInf}, hi[4] = {kMinusInf, kMinusInf, kMinusInf, kMinusInf};
  const uint8_t* kat = kb + 2 * (first + r0 + grp) * p.k_sn;
  const uint8_t* vat = vb + 2 * (first + r0 + grp) * p.v_sn;
  const long long k_step = 2 * kGroups * p.k_sn, v_step = 2 * kGroups * p.v_sn;
  uint4 kx[kWriteRows], vx[kWriteRows];
  auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < kWriteRows; ++u) {
      kx[u] = vx[u] = make_uint4(0, 0, 0, 0);
      if (base + u * kGroups + grp < r1) {
        kx[u] = *reinterpret_cast<const uint4*>(kat);
        vx[u] = *reinterpret_cast<const uint4*>(vat);
      }
      kat += k_step;
      vat += v_step;
    }
  };
  load(r0);
  if (page < 0) return;
  long long row = (static_cast<long long>(page) * p.pool.hkv + h) * ps + r0 + grp;
  for (int base = r0; base < r1; base += kGroups * kWriteRows) {
    if (base > r0) load(base);
#pragma unroll
    for (int u = 0; u < kWriteRows; ++u, row += kGroups) {
      if (base + u * kGroups >= r1) break;   // of the whole CTA: the shuffles of a row's scale need whole warps
      const bool on = base + u * kGroups + grp < r1;
      if (on) {
        const uint32_t w[4] = {kx[u].x, kx[u].y, kx[u].z, kx[u].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { lo[i] = min16x2_nan<BF16>(lo[i], w[i]); hi[i] = max16x2_nan<BF16>(hi[i], w[i]); }
      }
      if (FMT == kKvNative) {
        if (on) {
          reinterpret_cast<uint4*>(p.pool.k_pages)[row * kLanes + c] = kx[u];
          reinterpret_cast<uint4*>(p.pool.v_pages)[row * kLanes + c] = vx[u];
        }
      } else {
        float ks, vs;
        uint32_t kc[2], vc[2];
        quantise_row8<FMT, D, BF16>(kx[u], ks, kc);
        quantise_row8<FMT, D, BF16>(vx[u], vs, vc);
        if (on) {
          if (FMT == kKvInt8) {
            reinterpret_cast<uint2*>(p.pool.k_pages)[row * kLanes + c] = make_uint2(kc[0], kc[1]);
            reinterpret_cast<uint2*>(p.pool.v_pages)[row * kLanes + c] = make_uint2(vc[0], vc[1]);
          } else {
            reinterpret_cast<uint32_t*>(p.pool.k_pages)[row * kLanes + c] = kc[0];
            reinterpret_cast<uint32_t*>(p.pool.v_pages)[row * kLanes + c] = vc[0];
          }
          if (c == 0) { p.pool.k_scale[row] = ks; p.pool.v_scale[row] = vs; }
        }
      }
    }
  }
  if (!p.pool.k_bounds) return;
  __shared__ uint32_t red[kGroups][2][D / 2];
#pragma unroll
  for (int i = 0; i < 4; ++i) { red[grp][0][c * 4 + i] = lo[i]; red[grp][1][c * 4 + i] = hi[i]; }
  __syncthreads();
  if (threadIdx.x < D) {  // one channel pair of the minima or the maxima each
    const int which = threadIdx.x / (D / 2), ch = threadIdx.x % (D / 2);
    uint32_t x = red[0][which][ch];
#pragma unroll
    for (int g = 1; g < kGroups; ++g) x = which ? max16x2_nan<BF16>(x, red[g][which][ch]) : min16x2_nan<BF16>(x, red[g][which][ch]);
    uint32_t* out = reinterpret_cast<uint32_t*>(p.pool.k_bounds) +
                    ((static_cast<long long>(page) * p.pool.hkv + h) * 2 + which) * (D / 2) + ch;
    if (r0 > 0) x = which ? max16x2_nan<BF16>(x, *out) : min16x2_nan<BF16>(x, *out);
    *out = x;
  }
}

// 8 channels of a row as they lie (16, 8 or 4 bytes) and as 16-bit values
template <int FMT> struct Piece8 { uint4 a; };
template <> struct Piece8<kKvInt8> { uint2 a; };
template <> struct Piece8<kKvInt4> { uint32_t a; };
template <int FMT, bool BF16>
__device__ __forceinline__ uint4 piece8_values(const Piece8<FMT>& x, float scale) {
  if constexpr (FMT == kKvNative) {
    return x.a;
  } else {
    // a biased code under the exponent of 2^23 is 2^23 + code + bias: two instructions, a conversion of its own runs at a quarter
    // of the rate
    float f[8];
    if constexpr (FMT == kKvInt8) {
      const uint32_t w[2] = {x.a.x ^ 0x80808080u, x.a.y ^ 0x80808080u};
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = (__uint_as_float(__byte_perm(w[i >> 2], 0x4b000000u, 0x7650 + (i & 3))) - 8388736.0f) * scale;
    } else {
      const uint32_t w = x.a ^ 0x88888888u;
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = (__uint_as_float(((w >> (4 * i)) & 15u) | 0x4b000000u) - 8388616.0f) * scale;
    }
    return pack8<BF16>(f);
  }
}

struct PagedReadParams {
  PagedPool pool;
  BlockTable table;
  uint8_t *k, *v;  // [B, rows, Hkv, D] through element strides
  long long k_sb, k_sh, k_sn, v_sb, v_sh, v_sn;
  int rows, rows_per_cta;
  const int* starts;  // [B] position of the first row read
  const int* ends;    // [B] or null: rows at or past this position are zeros
};

// Row i of sequence b is position starts[b] + i; rows outside the sequence or the table are written as zeros.  A CTA takes up
// to kReadRows rows of a sequence, a thread 8 channels of a row's keys and values at a time (so that a warp's stores are
// contiguous), kReadPieces of them in flight.  Where the rows lie is looked up once, by one thread a row.
constexpr int kReadRows = 32;
constexpr int kReadPieces = 4;
template <int FMT, int D, bool BF16>
__global__ void __launch_bounds__(256, 4) paged_read_kernel(const __grid_constant__ PagedReadParams p) {
  __shared__ long long at[kReadRows];   // row of the pool for head 0, -1: none
  griddep_launch();
  griddep_wait();
  const int b = blockIdx.y, i0 = blockIdx.x * p.rows_per_cta, rows = min(p.rows_per_cta, p.rows - i0);
  if (static_cast<int>(threadIdx.x) < rows) {
    const int end = p.ends ? p.ends[b] : 2147483647;   // beside the start: the page does not wait for it
    const long long pos = static_cast<long long>(p.starts[b]) + i0 + threadIdx.x;
    const int page = page_of(p.table, b, pos >> p.pool.ps_shift, p.pool.num_pages);
    at[threadIdx.x] = page < 0 || (p.ends && pos >= end) ? -1ll : ((static_cast<long long>(page) * p.pool.hkv) << p.pool.ps_shift) + (pos & ((1 << p.pool.ps_shift) - 1));
  }
  __syncthreads();
  constexpr int kParts = D / 8;
  const int per_row = p.pool.hkv * kParts;
  uint8_t* ko = p.k + 2 * (b * p.k_sb + i0 * p.k_sn);
  uint8_t* vo = p.v + 2 * (b * p.v_sb + i0 * p.v_sn);
  const Piece8<FMT>* kp = reinterpret_cast<const Piece8<FMT>*>(p.pool.k_pages);
  const Piece8<FMT>* vp = reinterpret_cast<const Piece8<FMT>*>(p.pool.v_pages);
  // a thread keeps to one piece of a row (or to every 256th) and goes down the rows
  const int rows_at_once = per_row < 256 ? 256 / per_row : 1, my_row = threadIdx.x / per_row < rows_at_once ? threadIdx.x / per_row : rows;
  for (int col = per_row < 256 ? threadIdx.x % per_row : threadIdx.x; col < per_row; col += 256) {
    const int h = col / kParts, c = col % kParts;
    const long long piece = (static_cast<long long>(h) << p.pool.ps_shift) * kParts + c, scale = static_cast<long long>(h) << p.pool.ps_shift;
    uint8_t* kd = ko + 2 * (h * p.k_sh + c * 8);
    uint8_t* vd = vo + 2 * (h * p.v_sh + c * 8);
    for (int i1 = per_row < 256 ? my_row : 0; i1 < rows; i1 += rows_at_once * kReadPieces) {
      Piece8<FMT> k[kReadPieces], v[kReadPieces];
      float ks[kReadPieces], vs[kReadPieces];
      bool there[kReadPieces];
#pragma unroll
      for (int u = 0; u < kReadPieces; ++u) {
        const int i = i1 + u * rows_at_once;
        const long long r = i < rows ? at[i] : -1ll;
        there[u] = r >= 0;
        ks[u] = vs[u] = 1.0f;
        if (there[u]) {
          k[u] = kp[r * kParts + piece];
          v[u] = vp[r * kParts + piece];
          if (FMT != kKvNative) { ks[u] = p.pool.k_scale[r + scale]; vs[u] = p.pool.v_scale[r + scale]; }
        }
      }
#pragma unroll
      for (int u = 0; u < kReadPieces; ++u) {
        const int i = i1 + u * rows_at_once;
        if (i >= rows) break;
        uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
        if (there[u]) {
          kx = piece8_values<FMT, BF16>(k[u], ks[u]);
          vx = piece8_values<FMT, BF16>(v[u], vs[u]);
        }
        *reinterpret_cast<uint4*>(kd + 2 * i * p.k_sn) = kx;
        *reinterpret_cast<uint4*>(vd + 2 * i * p.v_sn) = vx;
      }
    }
  }
}

}  // namespace sq
