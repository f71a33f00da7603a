// The paged FP8 KV cache: appending tokens to pages that hold one scale per (page, KV head),
// and moving the tokens that an eviction keeps into other pages. The attention over the pages is
// in attention_pages.cuh.
//
// A page's scale is a power of two, the smallest s with |value| <= 448 s. e4m3 codes carry their
// own exponent, so against amax / 448 this costs no precision but at the subnormal end (below
// s * 2^-6), and codes that move to another power-of-two scale, when a page grows or tokens of
// several pages meet in one, stay exactly what they were unless they become subnormal.
#pragma once

#include "codes.cuh"

namespace kab {

// The pool as the kernels see it (KabKvPages with ints where 32 bits suffice).
struct PagePool {
  uint8_t* codes[2];  // K, V
  float* scale[2];
  float* mass;
  int64_t sp[2], sh[2], st[2];  // code strides: page, head, token (bytes)
  int64_t ssp[2], ssh[2];       // scale strides: page, head
  int64_t msp, msh;             // mass strides: page, head
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lengths;
  int num_pages, heads, page_shift, max_pages, batch;
};

// Tokens of sequence b, cut to what the page table can hold.
__device__ __forceinline__ int page_length(const PagePool& p, int b, unsigned* status) {
  const int n = p.lengths[b], cap = p.max_pages << p.page_shift;
  if (n < 0 || n > cap) {
    atomicOr(status, kDevBounds);
    return n < 0 ? 0 : cap;
  }
  return n;
}
// The page of logical page i of sequence b, or -1 for a number outside the pool.
__device__ __forceinline__ int page_of(const PagePool& p, int b, int i, unsigned* status) {
  const int page = __ldg(p.table + b * p.table_stride + i);
  if (page < 0 || page >= p.num_pages) {
    atomicOr(status, kDevBounds);
    return -1;
  }
  return page;
}

// The smallest power of two s >= 2^-126 with amax <= 448 s, from the bits of a finite amax >= 0:
// 448 = 1.75 * 2^8, so s = 2^(e - 8) for a significand up to 1.75, else 2^(e - 7).
__device__ __forceinline__ float page_scale_of(uint32_t amax_bits) {
  const int e = static_cast<int>(amax_bits >> 23) + ((amax_bits & 0x7FFFFFu) > 0x600000u) - 8;
  return __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23);
}
// Division by a page scale: a multiplication where the scale is a power of two with a normal
// reciprocal (every scale that this library writes), the IEEE division otherwise.
struct PageDivisor {
  float s, inv;
  __device__ __forceinline__ explicit PageDivisor(float s_) : s(s_), inv(0.0f) {
    const uint32_t b = __float_as_uint(s_), e = b >> 23;
    if ((b & 0x7FFFFFu) == 0 && e >= 1 && e <= 253) inv = __uint_as_float((254u - e) << 23);
  }
  __device__ __forceinline__ float operator()(float v) const {
    return inv != 0.0f ? __fmul_rn(v, inv) : __fdiv_rn(v, s);
  }
};

__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}
// Block-wide maximum; `red` holds 32 words.
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, lane < warps ? red[lane] : 0u);
}
// 16 e4m3 codes as fp32 values, and back.
__device__ __forceinline__ void e4m3_unpack16(const uint4& raw, float (&v)[16]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
        static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 e4m3_pack16(const float (&v)[16]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = e4m3_pair(v[4 * i], v[4 * i + 1]) |
           (static_cast<uint32_t>(e4m3_pair(v[4 * i + 2], v[4 * i + 3])) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// ------------------------------------------------------------------ append

struct AppendArgs {
  PagePool pool;
  const void* x[2];        // K, V
  int64_t xb[2], xh[2], xt[2];
  const int32_t* counts;
  int32_t* lengths_out;    // NULL: another launch advances the lengths
  int new_tokens, touched, d_shift;  // d_shift: log2(head_dim / 8)
};

// One block per (sequence and touched page, head, K or V): the new tokens' values stay in
// registers (CH chunks of 8 per thread) between the maximum and the codes, so they are read once.
template <int T, int CH>
__global__ void __launch_bounds__(256) append_pages_kernel(AppendArgs a, unsigned* status) {
  __shared__ uint32_t red[32];
  const PagePool& p = a.pool;
  const int b = blockIdx.x / a.touched, j = blockIdx.x % a.touched, h = blockIdx.y, kv = blockIdx.z;
  const int P = 1 << p.page_shift, cap = p.max_pages << p.page_shift;
  const int start = page_length(p, b, status);
  int count = a.counts != nullptr ? a.counts[b] : a.new_tokens;
  if (count < 0 || count > a.new_tokens || count > cap - start) {
    if (threadIdx.x == 0) atomicOr(status, kDevBounds);
    count = max(0, min(min(count, a.new_tokens), cap - start));
  }
  const int end = start + count;
  if (a.lengths_out != nullptr && j == 0 && h == 0 && kv == 0 && threadIdx.x == 0) a.lengths_out[b] = end;
  const int pi = (start >> p.page_shift) + j;
  const int lo = max(start, pi << p.page_shift), hi = min(end, (pi + 1) << p.page_shift);
  if (lo >= hi) return;
  const int page = page_of(p, b, pi, status);
  if (page < 0) return;
  const int held = lo & (P - 1), rows = hi - lo;
  float* scale = p.scale[kv] + page * p.ssp[kv] + h * p.ssh[kv];
  const float s_old = held > 0 ? *scale : 0.0f;

  using E = typename InTraits<T>::type;
  constexpr int kWords = T == kF32 ? 2 : 1;
  const int chunks = rows << a.d_shift, mask = (1 << a.d_shift) - 1;
  const E* x = static_cast<const E*>(a.x[kv]) + b * a.xb[kv] + h * a.xh[kv] + (lo - start) * a.xt[kv];
  uint4 raw[CH][kWords];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = threadIdx.x + i * 256;
    if (c < chunks) {
      const uint4* src = reinterpret_cast<const uint4*>(x + (c >> a.d_shift) * a.xt[kv] + (c & mask) * 8);
#pragma unroll
      for (int w = 0; w < kWords; ++w) raw[i][w] = __ldg(src + w);
    }
  }
  auto values = [&](int i, float(&v)[8]) {
    if constexpr (T == kF32) {
      const uint32_t w[8] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w,
                             raw[i][1].x, raw[i][1].y, raw[i][1].z, raw[i][1].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(w[e]);
    } else {
      unpack8<T>(raw[i][0], v);
    }
  };
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    if (static_cast<int>(threadIdx.x) + i * 256 < chunks) {
      float v[8];
      values(i, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, finite_bits(v[e]));
    }
  }
  const float s = fmaxf(page_scale_of(block_max(top, red)), s_old);
  const PageDivisor by(s);
  uint8_t* codes = p.codes[kv] + page * p.sp[kv] + h * p.sh[kv];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = threadIdx.x + i * 256;
    if (c < chunks) {
      float v[8];
      values(i, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = by(v[e]);
      *reinterpret_cast<uint2*>(codes + (held + (c >> a.d_shift)) * p.st[kv] + (c & mask) * 8) = e4m3x8(v);
    }
  }
  if (held > 0 && s != s_old) {  // the page grew past its scale: its tokens move to the larger one
    const int half = a.d_shift - 1, hmask = (1 << half) - 1;
    for (int c = threadIdx.x; c < held << half; c += 256) {
      uint4* at = reinterpret_cast<uint4*>(codes + (c >> half) * p.st[kv] + (c & hmask) * 16);
      float v[16];
      e4m3_unpack16(*at, v);
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = by(__fmul_rn(v[e], s_old));
      *at = e4m3_pack16(v);
    }
  }
  if (threadIdx.x == 0) *scale = s;
  if (kv == 0 && p.mass != nullptr && static_cast<int>(threadIdx.x) < rows)
    p.mass[page * p.msp + h * p.msh + held + threadIdx.x] = 0.0f;
}

// lengths_out = lengths + counts after the append, for lengths that are advanced in place.
__global__ void advance_lengths_kernel(const int32_t* lengths, const int32_t* counts, int new_tokens, int cap,
                                       int batch, int32_t* out) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= batch) return;
  const int start = min(max(lengths[b], 0), cap);
  const int count = counts != nullptr ? min(max(counts[b], 0), new_tokens) : new_tokens;
  out[b] = start + min(count, cap - start);
}

// ------------------------------------------------------------------ evict

// Masses in an unsigned order: larger mass, larger key; +0 and -0 alike; NaN above everything.
__device__ __forceinline__ uint32_t mass_key(float m) {
  const uint32_t b = __float_as_uint(m);
  if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
  if ((b & 0x7FFFFFFFu) == 0) return 0x80000000u;
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

struct EvictArgs {
  PagePool pool;
  const int32_t* out_table;
  int64_t out_stride;
  int32_t* kept;
  int32_t* lengths_out;
  int budget, recent, sinks;
};

// One block per (sequence, KV head): the key of the last token that stays is found eight bits at
// a time, from the top, by histograms of the keys that share the bits found so far; a pass over
// the tokens in order then writes those above it and, of those equal to it, the first ones.
__global__ void __launch_bounds__(1024) evict_select_kernel(EvictArgs a, unsigned* status) {
  const PagePool& p = a.pool;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int P = 1 << p.page_shift;
  const int n = page_length(p, b, status);
  int32_t* kept = a.kept + (static_cast<int64_t>(b) * p.heads + h) * a.budget;
  if (n <= a.budget) {
    for (int i = tid; i < a.budget; i += 1024) kept[i] = i < n ? i : -1;
    return;
  }
  __shared__ uint32_t hist[256];
  __shared__ uint32_t found[2];
  __shared__ int above[32], equal[32];
  const int lo = a.sinks, hi = n - a.recent;  // the tokens that compete
  auto key_at = [&](int t) -> uint32_t {
    const int page = page_of(p, b, t >> p.page_shift, status);
    return page < 0 ? 0u : mass_key(p.mass[page * p.msp + h * p.msh + (t & (P - 1))]);
  };
  uint32_t want = static_cast<uint32_t>(a.budget - a.sinks - a.recent), prefix = 0;
  for (int i = tid; i < a.sinks; i += 1024) kept[i] = i;
  for (int i = tid; i < a.recent; i += 1024) kept[a.budget - a.recent + i] = hi + i;
  if (want == 0) return;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += 1024) hist[i] = 0;
    __syncthreads();
    for (int t = lo + tid; t < hi; t += 1024) {
      const uint32_t k = key_at(t);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (warp == 0) {  // the largest digit with at least `want` keys at or above it
      uint32_t c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += c[i] = hist[255 - (lane * 8 + i)];
      uint32_t upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      uint32_t before = upto - sum;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (before < want && before + c[i] >= want) {
          found[0] = prefix | (static_cast<uint32_t>(255 - (lane * 8 + i)) << shift);
          found[1] = want - before;
        }
        before += c[i];
      }
    }
    __syncthreads();
    prefix = found[0];
    want = found[1];  // how many of the keys with these bits stay
  }
  int out = a.sinks, ties = 0;
  for (int t0 = lo; t0 < hi; t0 += 1024) {
    const int t = t0 + tid;
    const uint32_t k = t < hi ? key_at(t) : 0u;
    const bool is_above = t < hi && k > prefix, is_equal = t < hi && k == prefix;
    const uint32_t ma = __ballot_sync(0xffffffffu, is_above), me = __ballot_sync(0xffffffffu, is_equal);
    if (lane == 0) {
      above[warp] = __popc(ma);
      equal[warp] = __popc(me);
    }
    __syncthreads();
    int pa = 0, pe = 0, ta = 0, te = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) {
        pa += above[w];
        pe += equal[w];
      }
      ta += above[w];
      te += equal[w];
    }
    const uint32_t before = (1u << lane) - 1u;
    const int rank_e = ties + pe + __popc(me & before);  // equal keys before this token
    const int rank_a = pa + __popc(ma & before);         // larger keys before it in this tile
    const int limit = static_cast<int>(want);
    if (is_above || (is_equal && rank_e < limit))
      kept[out + rank_a + min(rank_e, limit) - min(ties, limit)] = t;
    out += ta + min(ties + te, limit) - min(ties, limit);
    ties += te;
    __syncthreads();
  }
}

// One block per (output page, KV head, sequence): gathers the page's tokens (K and V rows in
// registers), finds the scale that holds them and writes codes, scales and masses.
template <int CH>
__global__ void __launch_bounds__(128) evict_move_kernel(EvictArgs a, int half, unsigned* status) {
  __shared__ uint32_t red[32];
  __shared__ int src_page[128], src_slot[128];
  const PagePool& p = a.pool;
  const int j = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, P = 1 << p.page_shift;
  const int stay = min(page_length(p, b, status), a.budget);
  if (a.lengths_out != nullptr && j == 0 && h == 0 && tid == 0) a.lengths_out[b] = stay;
  const int first = j << p.page_shift, rows = min(stay - first, P);
  if (rows <= 0) return;
  const int to = __ldg(a.out_table + b * a.out_stride + j);
  if (to < 0 || to >= p.num_pages) {
    if (tid == 0) atomicOr(status, kDevBounds);
    return;
  }
  const int32_t* kept = a.kept + (static_cast<int64_t>(b) * p.heads + h) * a.budget + first;
  if (tid < rows) {
    const int t = kept[tid];
    const int page = page_of(p, b, t >> p.page_shift, status);
    src_page[tid] = page;
    src_slot[tid] = t & (P - 1);
    if (p.mass != nullptr && page >= 0)
      p.mass[to * p.msp + h * p.msh + tid] = p.mass[page * p.msp + h * p.msh + (t & (P - 1))];
  }
  __syncthreads();
  const int chunks = rows << half, mask = (1 << half) - 1;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    uint4 raw[CH];
    float from[CH];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = tid + i * 128;
      raw[i] = make_uint4(0, 0, 0, 0);
      from[i] = 0.0f;
      if (c < chunks) {
        const int r = c >> half, page = src_page[r];
        if (page >= 0) {
          raw[i] = __ldg(reinterpret_cast<const uint4*>(p.codes[kv] + page * p.sp[kv] + h * p.sh[kv] +
                                                        src_slot[r] * p.st[kv] + (c & mask) * 16));
          from[i] = __ldg(p.scale[kv] + page * p.ssp[kv] + h * p.ssh[kv]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float v[16];
      e4m3_unpack16(raw[i], v);
#pragma unroll
      for (int e = 0; e < 16; ++e) top = max(top, finite_bits(__fmul_rn(v[e], from[i])));
    }
    const float s = page_scale_of(block_max(top, red));
    const PageDivisor by(s);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = tid + i * 128;
      if (c < chunks) {
        float v[16];
        e4m3_unpack16(raw[i], v);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = by(__fmul_rn(v[e], from[i]));
        *reinterpret_cast<uint4*>(p.codes[kv] + to * p.sp[kv] + h * p.sh[kv] + (c >> half) * p.st[kv] +
                                  (c & mask) * 16) = e4m3_pack16(v);
      }
    }
    if (tid == 0) p.scale[kv][to * p.ssp[kv] + h * p.ssh[kv]] = s;
  }
}

}  // namespace kab
