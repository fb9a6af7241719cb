// Attention of one new token per sequence over a paged key/value cache.
#pragma once
#include "paged_cache.cuh"

namespace sq {

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
  float scale_log2;  // softmax scale * log2(e)
};

// One CTA per (query head, sequence): its warps take every eighth key, a lane holds D / 32 channels.
template <int FMT, int D, bool BF16>
__global__ void __launch_bounds__(256) paged_decode_kernel(const __grid_constant__ PagedDecodeParams p) {
  constexpr int C = D / 32;
  const int hq = blockIdx.x, b = blockIdx.y, h = hq / p.groups, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ps = 1 << p.pool.ps_shift;
  const int len = min(max(p.kv_lens[b], 0), p.max_len);
  float q[C], o[C], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    q[i] = to_f32<BF16>(*reinterpret_cast<const uint16_t*>(p.q + 2 * (b * p.q_sb + hq * p.q_sh + lane * C + i)));
    o[i] = 0.f;
  }
  const int pages = p.list ? p.list_len : (len + ps - 1) >> p.pool.ps_shift;
  for (int e = 0; e < pages; ++e) {
    const int index = p.list ? p.list[(static_cast<long long>(b) * p.pool.hkv + h) * p.list_len + e] : e;
    const int page = page_of(p.table, b, index, p.pool.num_pages);
    if (page < 0) continue;
    const int rows = static_cast<int>(min(static_cast<long long>(ps), len - static_cast<long long>(index) * ps));
    const long long block = (static_cast<long long>(page) * p.pool.hkv + h) << p.pool.ps_shift;
    for (int r = warp; r < rows; r += 8) {
      float k8[8], v8[8], k[C], v[C];
      // 8 channels are loaded and this lane's C taken out of them
      load_row8<FMT, BF16>(p.pool.k_pages, p.pool.k_scale, block + r, D / 8, lane * C / 8, k8);
      load_row8<FMT, BF16>(p.pool.v_pages, p.pool.v_scale, block + r, D / 8, lane * C / 8, v8);
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        k[i] = v[i] = 0.f;
#pragma unroll
        for (int u = 0; u < 8 / C; ++u)
          if (lane % (8 / C) == u) { k[i] = k8[u * C + i]; v[i] = v8[u * C + i]; }
        s += q[i] * k[i];
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      s *= p.scale_log2;
      const float m_new = fmaxf(m, s);
      const float a = m_new == -INFINITY ? 1.f : exp2f(m - m_new), w = m_new == -INFINITY && s == s ? 0.f : exp2f(s - m_new);
      l = l * a + w;
#pragma unroll
      for (int i = 0; i < C; ++i) o[i] = o[i] * a + w * v[i];
      m = m_new;
    }
  }
  __shared__ float so[8][D], sm[8], sl[8];
#pragma unroll
  for (int i = 0; i < C; ++i) so[warp][lane * C + i] = o[i];
  if (lane == 0) { sm[warp] = m; sl[warp] = l; }
  __syncthreads();
  if (threadIdx.x < D) {
    float top = -INFINITY, den = 0.f, acc = 0.f;
    for (int w = 0; w < 8; ++w) top = fmaxf(top, sm[w]);
    for (int w = 0; w < 8; ++w) {
      const float f = sm[w] == -INFINITY && !(sl[w] != sl[w]) ? 0.f : exp2f(sm[w] - top);
      den += sl[w] * f;
      acc += so[w][threadIdx.x] * f;
    }
    const float val = den > 0.f ? acc / den : (den == den ? 0.f : den);
    uint16_t* out = reinterpret_cast<uint16_t*>(p.o + 2 * (b * p.o_sb + hq * p.o_sh + threadIdx.x));
    *out = p.o_bf16 ? from_f32<true>(val) : from_f32<false>(val);
    if (threadIdx.x == 0 && p.lse)
      p.lse[static_cast<long long>(b) * p.hq + hq] = den > 0.f ? log2f(den) + top : (den == den ? -INFINITY : den);
  }
}

}  // namespace sq
