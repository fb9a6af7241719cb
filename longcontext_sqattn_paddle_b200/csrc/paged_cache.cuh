// The paged key/value cache: geometry of a layer's pool, the kernel that quantises new rows into pages and the one that
// reads rows back.
//
// A pool holds P pages of `page_size` tokens: [P, Hkv, page_size, D] for keys and for values, so that the rows of one page
// and head are one contiguous block (what the attention kernel loads).  Formats: the 16-bit values themselves, int8 codes,
// or 4-bit codes two to a byte (even channel in the low half); codes have one fp32 scale per row, [P, Hkv, page_size]:
//   s = max(fl32(max|x| * fl32(1/Q)), 2^-100), Q = 127 or 7,   code = nearest integer to x / s (ties to even),   value = code * s.
// A row with an infinity or a NaN gets the scale NaN and zero codes, so that it reads back as NaN.  The floor of the scale
// keeps 1/s finite for rows of (nearly) zeros.
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

template <bool BF16>
__device__ __forceinline__ uint32_t min16x2(uint32_t a, uint32_t b) {
  if (BF16) {
    const __nv_bfloat162 r = __hmin2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  const __half2 r = __hmin2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <bool BF16>
__device__ __forceinline__ uint32_t max16x2(uint32_t a, uint32_t b) {
  if (BF16) {
    const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Quantise one row spread over D / 8 consecutive lanes, 8 channels each; every lane gets the scale.  The codes come out as
// the integers' low bytes (int8) or nibbles (int4), packed in channel order.
//
// The code is the nearest integer to the exact quotient x / s.  The product with an approximate 1/s is off by at most
// 127 * 2^-20, so its nearest integer is the answer unless it lies that close to a half-integer; there the remainder
// x - code * s decides, which one fused multiply-add gives exactly (x is a multiple of s's last place whenever code != 0,
// and the difference is below s in magnitude).  That branch is taken by 0.1 % of the values (x = max/2 is the common one).
template <int FMT, int D, bool BF16>
__device__ __forceinline__ void quantise_row8(const uint4& x, float& scale, uint32_t (&packed)[2]) {
  constexpr int kLanes = D / 8;
  constexpr uint32_t kNonFinite = BF16 ? 0x7f80u : 0x7c00u;
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: added, it leaves the nearest integer in the low bits
  uint32_t a = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) a = __vmaxu2(a, __shfl_xor_sync(0xffffffffu, a, o));
  const uint32_t top = max(a & 0xffffu, a >> 16);
  const bool finite = top < kNonFinite;
  const float s = fmaxf(to_f32<BF16>(static_cast<uint16_t>(top)) * kv_code_step<FMT>(), kKvSmallestScale);
  scale = finite ? s : __int_as_float(0x7fc00000);
  const float inv = finite ? __fdividef(1.0f, s) : 0.0f;
  float f[8];
  unpack8<BF16>(x, f);
  uint32_t c[8];
  bool near_half = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = f[i] * inv, r = t + kRound;
    near_half |= fabsf(t - (r - kRound)) > 0.499f;
    c[i] = __float_as_uint(r);
  }
  if (near_half) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float r = __uint_as_float(c[i]) - kRound, e = __fmaf_rn(-r, s, f[i]), half = 0.5f * s;
      const bool odd = (c[i] & 1u) != 0u;
      if (e > half || (e == half && odd)) ++c[i];
      if (e < -half || (e == -half && odd)) --c[i];
    }
  }
  if (!finite) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = 0u;
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

// One CTA per (page that new rows fall into, KV head, sequence): it alone writes that page's rows and bounds, so the bounds
// need no atomics.  D / 8 lanes hold a row, 8 channels each; the rows of the page are dealt to the CTA's lane groups.
template <int FMT, int D, bool BF16>
__global__ void __launch_bounds__(128) paged_write_kernel(const __grid_constant__ PagedWriteParams p) {
  constexpr int kLanes = D / 8, kGroups = 128 / kLanes;
  const int b = blockIdx.z, h = blockIdx.y;
  const int ps = 1 << p.pool.ps_shift;
  const int pos = p.positions[b];
  const int count = p.counts ? min(max(p.counts[b], 0), p.rows) : p.rows;
  if (pos < 0) return;
  const long long index = (pos >> p.pool.ps_shift) + static_cast<long long>(blockIdx.x);
  const long long first = index * ps - pos;  // new row that falls on the page's row 0 (negative: the page was begun before)
  if (first >= count) return;
  const int page = page_of(p.table, b, index, p.pool.num_pages);
  if (page < 0) return;
  const int r0 = first < 0 ? static_cast<int>(-first) : 0;
  const int r1 = static_cast<int>(min(static_cast<long long>(ps), count - first));
  const int c = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const long long block = (static_cast<long long>(page) * p.pool.hkv + h) * ps;  // first row of the page's block
  const uint8_t* kb = p.k + 2 * (b * p.k_sb + h * p.k_sh + c * 8);
  const uint8_t* vb = p.v + 2 * (b * p.v_sb + h * p.v_sh + c * 8);
  constexpr uint32_t kInf = BF16 ? 0x7f807f80u : 0x7c007c00u, kMinusInf = BF16 ? 0xff80ff80u : 0xfc00fc00u;
  uint32_t lo[4] = {kInf, kInf, kInf, kInf}, hi[4] = {kMinusInf, kMinusInf, kMinusInf, kMinusInf};
  // every lane group runs the same number of steps: the shuffles of a row's scale need whole warps
  for (int base = r0; base < r1; base += kGroups) {
    const int r = base + grp;
    const bool on = r < r1;
    uint4 kx = make_uint4(0, 0, 0, 0), vx = make_uint4(0, 0, 0, 0);
    if (on) {
      kx = *reinterpret_cast<const uint4*>(kb + 2 * (first + r) * p.k_sn);
      vx = *reinterpret_cast<const uint4*>(vb + 2 * (first + r) * p.v_sn);
      const uint32_t w[4] = {kx.x, kx.y, kx.z, kx.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) { lo[i] = min16x2<BF16>(lo[i], w[i]); hi[i] = max16x2<BF16>(hi[i], w[i]); }
    }
    const long long row = block + r;
    if (FMT == kKvNative) {
      if (on) {
        reinterpret_cast<uint4*>(p.pool.k_pages)[row * kLanes + c] = kx;
        reinterpret_cast<uint4*>(p.pool.v_pages)[row * kLanes + c] = vx;
      }
    } else {
      float ks, vs;
      uint32_t kc[2], vc[2];
      quantise_row8<FMT, D, BF16>(kx, ks, kc);
      quantise_row8<FMT, D, BF16>(vx, vs, vc);
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
  if (!p.pool.k_bounds) return;
  __shared__ uint32_t red[kGroups][2][D / 2];
#pragma unroll
  for (int i = 0; i < 4; ++i) { red[grp][0][c * 4 + i] = lo[i]; red[grp][1][c * 4 + i] = hi[i]; }
  __syncthreads();
  if (threadIdx.x < D) {  // one channel pair of the minima or the maxima each
    const int which = threadIdx.x / (D / 2), ch = threadIdx.x % (D / 2);
    uint32_t x = red[0][which][ch];
#pragma unroll
    for (int g = 1; g < kGroups; ++g) x = which ? max16x2<BF16>(x, red[g][which][ch]) : min16x2<BF16>(x, red[g][which][ch]);
    uint32_t* out = reinterpret_cast<uint32_t*>(p.pool.k_bounds) +
                    ((static_cast<long long>(page) * p.pool.hkv + h) * 2 + which) * (D / 2) + ch;
    if (r0 > 0) x = which ? max16x2<BF16>(x, *out) : min16x2<BF16>(x, *out);
    *out = x;
  }
}

// 8 channels of a row, in fp32: x is what the row's lane loads (16, 8 or 4 bytes)
template <int FMT, bool BF16>
__device__ __forceinline__ void load_row8(const uint8_t* pages, const float* scales, long long row, int lanes, int c, float (&f)[8]) {
  if (FMT == kKvNative) {
    unpack8<BF16>(reinterpret_cast<const uint4*>(pages)[row * lanes + c], f);
  } else {
    const float s = scales[row];
    if (FMT == kKvInt8) {
      const uint2 w = reinterpret_cast<const uint2*>(pages)[row * lanes + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)))) * s;
    } else {
      const uint32_t w = reinterpret_cast<const uint32_t*>(pages)[row * lanes + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(static_cast<int>(w << (28 - 4 * i)) >> 28) * s;
    }
  }
}

struct PagedReadParams {
  PagedPool pool;
  BlockTable table;
  uint8_t *k, *v;  // [B, rows, Hkv, D] through element strides
  long long k_sb, k_sh, k_sn, v_sb, v_sh, v_sn;
  int batch, rows;
  const int* starts;  // [B] position of the first row read
  const int* ends;    // [B] or null: rows at or past this position are zeros
};

// Row i of sequence b is position starts[b] + i; rows outside the sequence or the table are written as zeros.  One thread
// takes 8 channels of a row of keys and of values.
template <int FMT, int D, bool BF16>
__global__ void __launch_bounds__(256) paged_read_kernel(const __grid_constant__ PagedReadParams p) {
  constexpr int kLanes = D / 8;
  const long long total = static_cast<long long>(p.batch) * p.rows * p.pool.hkv * kLanes;
  for (long long idx = blockIdx.x * 256ll + threadIdx.x; idx < total; idx += 256ll * gridDim.x) {
    const int c = static_cast<int>(idx % kLanes);
    long long rest = idx / kLanes;
    const int h = static_cast<int>(rest % p.pool.hkv);
    rest /= p.pool.hkv;
    const int i = static_cast<int>(rest % p.rows), b = static_cast<int>(rest / p.rows);
    const long long pos = static_cast<long long>(p.starts[b]) + i;
    const bool inside = pos >= 0 && (!p.ends || pos < p.ends[b]);
    const int page = inside ? page_of(p.table, b, pos >> p.pool.ps_shift, p.pool.num_pages) : -1;
    float k[8] = {0, 0, 0, 0, 0, 0, 0, 0}, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (page >= 0) {
      const long long row = (((static_cast<long long>(page) * p.pool.hkv + h)) << p.pool.ps_shift) + (pos & ((1 << p.pool.ps_shift) - 1));
      load_row8<FMT, BF16>(p.pool.k_pages, p.pool.k_scale, row, kLanes, c, k);
      load_row8<FMT, BF16>(p.pool.v_pages, p.pool.v_scale, row, kLanes, c, v);
    }
    *reinterpret_cast<uint4*>(p.k + 2 * (b * p.k_sb + h * p.k_sh + i * p.k_sn + c * 8)) = pack8<BF16>(k);
    *reinterpret_cast<uint4*>(p.v + 2 * (b * p.v_sb + h * p.v_sh + i * p.v_sn + c * 8)) = pack8<BF16>(v);
  }
}

}  // namespace sq
