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

// The largest finite magnitude of 16 codes. Codes order like their magnitudes, so the maximum is
// taken on the codes, two at a time; only a NaN (0x7F) needs the values.
__device__ __forceinline__ float e4m3_amax16(const uint4& raw) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = __vmaxu2(top, __vmaxu2(w[i] & 0x007F007Fu, (w[i] >> 8) & 0x007F007Fu));
  const uint32_t code = max(top & 0xFFFFu, top >> 16);
  if (code != 0x7Fu) return e4m3_value_hw(static_cast<uint8_t>(code));
  float v[16], most = 0.0f;
  e4m3_unpack16(raw, v);
#pragma unroll
  for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(v[e]));  // fmaxf leaves NaN out
  return most;
}
// e4m3(code * from / s) of 16 codes. Where from / s is a power of two 2^k with -15 <= k <= 15 the
// products are exact in f16 (a code's last bit is at least 2^-9, and no result is above 448), two at a
// time; otherwise in fp32.
__device__ __forceinline__ uint4 e4m3_rescale16(const uint4& raw, float from, const PageDivisor& by) {
  const float ratio = by(from);
  const uint32_t bits = __float_as_uint(ratio);
  if ((bits & 0x7FFFFFu) == 0 && bits >= (112u << 23) && bits <= (142u << 23) && by.inv != 0.0f) {
    const __half2 f = __float2half2_rn(ratio);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i]), __NV_E4M3);
      const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i] >> 16), __NV_E4M3);
      const __half2 l = __hmul2(*reinterpret_cast<const __half2*>(&lo), f);
      const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&hi), f);
      const uint32_t a = __nv_cvt_halfraw2_to_fp8x2(*reinterpret_cast<const __half2_raw*>(&l), __NV_SATFINITE, __NV_E4M3);
      const uint32_t b = __nv_cvt_halfraw2_to_fp8x2(*reinterpret_cast<const __half2_raw*>(&h), __NV_SATFINITE, __NV_E4M3);
      o[i] = a | b << 16;
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
  }
  float v[16];
  e4m3_unpack16(raw, v);
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = by(__fmul_rn(v[e], from));
  return e4m3_pack16(v);
}

struct EvictArgs {
  PagePool pool;
  const int32_t* out_table;
  int64_t out_stride;
  int32_t* kept;
  int32_t* lengths_out;
  int budget, recent, sinks;
};

// One cluster of blocks per (sequence, KV head), each block with an equal run of the tokens that
// compete, KEYS keys per thread in registers (tokens past that are read again in each pass).
// The key of the last token that stays is found 11, 11 and 10 bits at a time, from the top: a histogram
// per block of the keys that share the bits found so far, the cluster's histograms summed through
// distributed shared memory by every block. A pass over the tokens in order then writes those above
// the key and, of those equal to it, the first ones. (One block per head, eight bits at a time and
// the masses read again in each of five passes, took 113 us at 32768 tokens and 8 heads with its move.)
constexpr int kSelectThreads = 512;

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive;\n barrier.cluster.wait;" ::: "memory");
}
// The four words at the same shared-memory address (16-byte aligned) of block `rank` of the cluster.
__device__ __forceinline__ uint4 load_cluster(const uint32_t* p, int rank) {
  uint32_t at;
  uint4 v;
  const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(p));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(mine), "r"(rank));
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(at)
               : "memory");
  return v;
}

template <int KEYS>
__global__ void __launch_bounds__(kSelectThreads, KEYS == 8 ? 2 : 1) evict_select_kernel(EvictArgs a, int blocks, unsigned* status) {
  // the move may be set up while this kernel runs: it waits for its end by itself
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const PagePool& p = a.pool;
  const int rank = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int P = 1 << p.page_shift;
  const int n = page_length(p, b, status);
  int32_t* kept = a.kept + (static_cast<int64_t>(b) * p.heads + h) * a.budget;
  if (n <= a.budget) {  // the same for every block of the cluster
    for (int i = rank * kSelectThreads + tid; i < a.budget; i += blocks * kSelectThreads) kept[i] = i < n ? i : -1;
    return;
  }
  __shared__ __align__(16) uint32_t hist[3][2048];
  __shared__ __align__(16) uint32_t totals[4];      // this block's keys above the last one that stays, and equal to it
  constexpr int WARPS = kSelectThreads / 32;
  __shared__ uint32_t found[2], sums[WARPS];
  __shared__ int above[WARPS], equal[WARPS];
  const int lo = a.sinks, hi = n - a.recent;  // the tokens that compete
  for (int i = rank * kSelectThreads + tid; i < a.sinks; i += blocks * kSelectThreads) kept[i] = i;
  for (int i = rank * kSelectThreads + tid; i < a.recent; i += blocks * kSelectThreads)
    kept[a.budget - a.recent + i] = hi + i;
  uint32_t want = static_cast<uint32_t>(a.budget - a.sinks - a.recent), prefix = 0;
  if (want == 0) return;

  const int span = (hi - lo + blocks - 1) / blocks, first = lo + rank * span, last = min(first + span, hi);
  auto key_at = [&](int t) -> uint32_t {
    const int page = page_of(p, b, t >> p.page_shift, status);
    return page < 0 ? 0u : mass_key(p.mass[page * p.msp + h * p.msh + (t & (P - 1))]);
  };
  uint32_t keys[KEYS];
#pragma unroll
  for (int i = 0; i < KEYS; ++i) {
    const int t = first + i * kSelectThreads + tid;
    keys[i] = t < last ? key_at(t) : 0u;
  }
  // f(token, key) for every token of this thread, in its order
  auto each = [&](auto&& f) {
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const int t = first + i * kSelectThreads + tid;
      if (t < last) f(t, keys[i]);
    }
    for (int t = first + KEYS * kSelectThreads + tid; t < last; t += kSelectThreads) f(t, key_at(t));
  };
  for (int i = tid; i < 3 * 2048; i += kSelectThreads) (&hist[0][0])[i] = 0;
  if (tid < 2) totals[tid] = 0;
  __syncthreads();
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, done = pass == 0 ? 32 : pass == 1 ? 21 : 10;
    const uint32_t mask = pass == 2 ? 1023u : 2047u;
    each([&](int, uint32_t k) {
      if (done == 32 || (k >> done) == (prefix >> done)) atomicAdd(&hist[pass][(k >> shift) & mask], 1u);
    });
    cluster_barrier();
    // bins 2047 - 4 tid and the three below, over the cluster; the largest digit with at least `want`
    // keys at or above it
    static_assert(kSelectThreads * 4 == 2048, "four bins per thread");
    uint4 bins[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) bins[r] = r < blocks ? load_cluster(&hist[pass][2044 - 4 * tid], r) : make_uint4(0, 0, 0, 0);
    uint32_t c[4] = {0, 0, 0, 0};
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      c[0] += bins[r].w;
      c[1] += bins[r].z;
      c[2] += bins[r].y;
      c[3] += bins[r].x;
    }
    const uint32_t here = c[0] + c[1] + c[2] + c[3];
    uint32_t upto = here;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    uint32_t before = __reduce_add_sync(0xffffffffu, lane < warp ? sums[lane] : 0u) + upto - here;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (before < want && before + c[i] >= want) {
        found[0] = prefix | (static_cast<uint32_t>(2047 - 4 * tid - i) << shift);
        found[1] = want - before;
      }
      before += c[i];
    }
    __syncthreads();
    prefix = found[0];
    want = found[1];  // how many of the keys with these bits stay
  }
  uint32_t mine[2] = {0, 0};
  each([&](int, uint32_t k) {
    mine[0] += k > prefix;
    mine[1] += k == prefix;
  });
  const uint32_t m0 = __reduce_add_sync(0xffffffffu, mine[0]), m1 = __reduce_add_sync(0xffffffffu, mine[1]);
  if (lane == 0) {
    atomicAdd(&totals[0], m0);
    atomicAdd(&totals[1], m1);
  }
  cluster_barrier();
  const int limit = static_cast<int>(want);
  int out = a.sinks, ties = 0;  // places and equal keys taken by the blocks before this one
  for (int r = 0; r < rank; ++r) {
    const uint4 there = load_cluster(totals, r);
    out += static_cast<int>(there.x);
    ties += static_cast<int>(there.y);
  }
  out += min(ties, limit);
  cluster_barrier();  // no block leaves while another may still read its shared memory
  auto tile = [&](int t, uint32_t k) {
    const bool is_above = t < last && k > prefix, is_equal = t < last && k == prefix;
    const uint32_t ma = __ballot_sync(0xffffffffu, is_above), me = __ballot_sync(0xffffffffu, is_equal);
    if (lane == 0) {
      above[warp] = __popc(ma);
      equal[warp] = __popc(me);
    }
    __syncthreads();
    const int va = lane < WARPS ? above[lane] : 0, ve = lane < WARPS ? equal[lane] : 0;
    const int pa = __reduce_add_sync(0xffffffffu, lane < warp ? va : 0), pe = __reduce_add_sync(0xffffffffu, lane < warp ? ve : 0);
    const int ta = __reduce_add_sync(0xffffffffu, va), te = __reduce_add_sync(0xffffffffu, ve);
    const uint32_t below = (1u << lane) - 1u;
    const int rank_e = ties + pe + __popc(me & below);  // equal keys before this token
    const int rank_a = pa + __popc(ma & below);         // larger keys before it in this tile
    if (is_above || (is_equal && rank_e < limit))
      kept[out + rank_a + min(rank_e, limit) - min(ties, limit)] = t;
    out += ta + min(ties + te, limit) - min(ties, limit);
    ties += te;
    __syncthreads();
  };
#pragma unroll
  for (int i = 0; i < KEYS; ++i) {
    const int t0 = first + i * kSelectThreads;
    if (t0 < last) tile(t0 + tid, keys[i]);
  }
  for (int t0 = first + KEYS * kSelectThreads; t0 < last; t0 += kSelectThreads) {
    const int t = t0 + tid;
    tile(t, t < last ? key_at(t) : 0u);
  }
}

// One block per (output page, KV head, sequence): gathers the page's tokens (K and V rows in
// registers), finds the scale that holds them and writes codes, scales and masses.
template <int CH>
__global__ void __launch_bounds__(128) evict_move_kernel(EvictArgs a, int half, unsigned* status) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
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
  uint4 raw[2][CH];  // K and V: all loads before the first maximum
  float from[2][CH];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = tid + i * 128;
      raw[kv][i] = make_uint4(0, 0, 0, 0);
      from[kv][i] = 0.0f;
      if (c < chunks) {
        const int r = c >> half, page = src_page[r];
        if (page >= 0) {
          raw[kv][i] = __ldg(reinterpret_cast<const uint4*>(p.codes[kv] + page * p.sp[kv] + h * p.sh[kv] +
                                                            src_slot[r] * p.st[kv] + (c & mask) * 16));
          from[kv][i] = __ldg(p.scale[kv] + page * p.ssp[kv] + h * p.ssh[kv]);
        }
      }
    }
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) top = max(top, finite_bits(__fmul_rn(e4m3_amax16(raw[kv][i]), from[kv][i])));
    const float s = page_scale_of(block_max(top, red));
    const PageDivisor by(s);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = tid + i * 128;
      if (c < chunks) {
        uint4 out = raw[kv][i];
        if (from[kv][i] != s) out = e4m3_rescale16(out, from[kv][i], by);
        *reinterpret_cast<uint4*>(p.codes[kv] + to * p.sp[kv] + h * p.sh[kv] + (c >> half) * p.st[kv] +
                                  (c & mask) * 16) = out;
      }
    }
    if (tid == 0) p.scale[kv][to * p.ssp[kv] + h * p.ssh[kv]] = s;
  }
}

}  // namespace kab
