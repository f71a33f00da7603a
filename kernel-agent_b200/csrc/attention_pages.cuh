// Attention of a few query tokens over the paged FP8 cache (kv_pages.cuh):
// softmax(q K^T * scale) V per query row, K = code * page scale, and the weight that every cached
// token receives added to its mass.
#pragma once

#include "kv_pages.cuh"

namespace kab {

struct PagesAttnArgs {
  PagePool pool;
  const void* q;
  int64_t qb, qh, qt;
  void* out;
  float scale_log2;  // sm_scale * log2(e)
  int heads_q, q_len, causal;
  float* ml;  // [batch, heads_q, q_len, 2]: each row's maximum (log2 units) and sum
};

template <int T>
__device__ __forceinline__ void store_elem(void* base, int64_t i, float v) {
  if constexpr (T == kF32) static_cast<float*>(base)[i] = v;
  else if constexpr (T == kBF16) static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(base)[i] = __float2half_rn(v);
}

// One block per (query head, query token, sequence): each warp takes every fourth token, its
// lanes share the head dimension, and carries the running maximum, sum and output of its tokens.
template <int T, int D>
__global__ void __launch_bounds__(128) pages_attention_kernel(PagesAttnArgs a, unsigned* status) {
  constexpr int E = D / 32;
  const PagePool& p = a.pool;
  const int hq = blockIdx.x / a.q_len, qi = blockIdx.x % a.q_len, b = blockIdx.y;
  const int h = hq / (a.heads_q / p.heads), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int P = 1 << p.page_shift;
  const int n = page_length(p, b, status);
  const int seen = a.causal ? max(0, n - a.q_len + 1 + qi) : n;
  float q[E], o[E] = {};
#pragma unroll
  for (int e = 0; e < E; ++e) q[e] = load_elem<T>(a.q, b * a.qb + hq * a.qh + qi * a.qt + lane * E + e) * a.scale_log2;
  float m = -INFINITY, l = 0.0f;
  for (int t = warp; t < seen; t += 4) {
    const int page = page_of(p, b, t >> p.page_shift, status);
    if (page < 0) continue;
    const uint8_t* k = p.codes[0] + page * p.sp[0] + h * p.sh[0] + (t & (P - 1)) * p.st[0] + lane * E;
    const uint8_t* v = p.codes[1] + page * p.sp[1] + h * p.sh[1] + (t & (P - 1)) * p.st[1] + lane * E;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], e4m3_value_hw(k[e]), s);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= p.scale[0][page * p.ssp[0] + h * p.ssh[0]];
    const float top = fmaxf(m, s), old = m == -INFINITY ? 0.0f : exp2f(m - top), w = exp2f(s - top);
    const float vs = w * p.scale[1][page * p.ssp[1] + h * p.ssh[1]];
    l = l * old + w;
    m = top;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * old + vs * e4m3_value_hw(v[e]);
  }
  __shared__ float sm[4], sl[4], so[4][D];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
  __syncthreads();
  const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float total = 0.0f, w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = sm[i] == -INFINITY ? 0.0f : exp2f(sm[i] - top);
    total += w[i] * sl[i];
  }
  const int64_t row = (static_cast<int64_t>(b) * a.heads_q + hq) * a.q_len + qi;
  if (threadIdx.x < D) {
    float acc = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc += w[i] * so[i][threadIdx.x];
    store_elem<T>(a.out, row * D + threadIdx.x, seen > 0 ? acc / total : 0.0f);
  }
  if (a.ml != nullptr && threadIdx.x == 0) {
    a.ml[2 * row] = top;
    a.ml[2 * row + 1] = total;
  }
}

// One warp per (token, KV head): the weights of its query rows, recomputed and summed in order.
template <int T, int D>
__global__ void __launch_bounds__(128) pages_mass_kernel(PagesAttnArgs a, unsigned* status) {
  constexpr int E = D / 32;
  const PagePool& p = a.pool;
  const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31;
  const int P = 1 << p.page_shift, group = a.heads_q / p.heads;
  const int n = page_length(p, b, status);
  for (int t = blockIdx.x * 4 + (threadIdx.x >> 5); t < n; t += gridDim.x * 4) {
    const int page = page_of(p, b, t >> p.page_shift, status);
    if (page < 0) continue;
    const uint8_t* k = p.codes[0] + page * p.sp[0] + h * p.sh[0] + (t & (P - 1)) * p.st[0] + lane * E;
    const float ks = p.scale[0][page * p.ssp[0] + h * p.ssh[0]];
    float received = 0.0f;
    for (int r = 0; r < group * a.q_len; ++r) {
      const int hq = h * group + r / a.q_len, qi = r % a.q_len;
      if (a.causal && t >= n - a.q_len + 1 + qi) continue;
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e)
        s = fmaf(load_elem<T>(a.q, b * a.qb + hq * a.qh + qi * a.qt + lane * E + e) * a.scale_log2,
                 e4m3_value_hw(k[e]), s);
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      const float* ml = a.ml + 2 * ((static_cast<int64_t>(b) * a.heads_q + hq) * a.q_len + qi);
      received += exp2f(s * ks - ml[0]) / ml[1];
    }
    if (lane == 0) p.mass[page * p.msp + h * p.msh + (t & (P - 1))] += received;
  }
}

}  // namespace kab
