// Weight-only FP4 linear for a few tokens: out[m, n] = ts * sum_k x[m, k] * e2m1(c[n, k]) *
// s[n, k / block] (+ bias), the activations as they are.
//
// The weight's bytes bound it (N K / 2 codes and N K / block scales against 2 M N K operations), so
// everything serves the stream of codes:
//
//  * The weight is the 16-row operand of mma.sync.m16n8k16 and the tokens its 8 columns (one to four
//    groups of 8): one conversion of the codes serves all tokens. A lane loads 16 bytes (32 codes) of
//    rows g and g + 8, and the products' order along K is chosen so that those 32 codes are the
//    lane's share of eight consecutive MMAs; nothing is exchanged between lanes. (tcgen05 would want
//    the scales in its own layout and M padded to its tile; at these M the tensor pipe is idle either
//    way.)
//  * e2m1 -> f16 is one exact conversion per two codes. An NVFP4 code times its e4m3 scale has at
//    most 6 significant bits and lies in [2^-10, 2688]: exact in f16, one packed multiplication per
//    two codes. An MXFP4 scale does not fit f16: the four 32-code blocks of a row's 128 codes are
//    taken in units of the first one's scale where they lie within 2^-20 .. 2^13 of it (exact), and
//    the 16 x 8 products of the 128 codes are added in fp32 with that scale; otherwise each block is
//    taken by itself.
//  * x enters as f16, each token (and K slice) in units of a power of two that puts its largest
//    finite value in [2^14, 2^15): bf16 and f16 keep all their bits down to 2^-29 of it; fp32 is
//    split into two f16 terms (22 bits) and multiplied twice. It is converted once per block and
//    stays in shared memory while the block streams its rows.
//  * Each warp keeps four 128-code chunks of its rows in flight in registers, across the block's row
//    tiles; the warps of a block share a tile's K and add their sums in shared memory. Blocks take
//    equal numbers of rows (not of tiles). Where x does not fit, or the rows are too few to occupy
//    the GPU, K is cut into slices whose sums meet in a second launch.
#pragma once

#include "codes.cuh"

namespace kab {

struct GemvArgs {
  const void* x;
  int64_t ldx;
  const uint8_t* codes;
  const uint8_t* scales;
  int swizzle;
  const float* ts;
  int ts_per_row;
  int m, n, k;
  const void* bias;
  int bias_dtype;
  void* out;
  int64_t ldo;
  int chunks, slice_chunks, slices;  // 128-code chunks of K, of a slice of it, and slices
  int k_warps;                       // warps of a block that share a tile's K
  int blocks;                        // blocks per slice
  float* partial;                    // [slices, m, n] where there is more than one slice
};

// ------------------------------------------------------------------ instructions

// The two e2m1 codes of byte B of `w` (low nibble first) as exact f16.
template <int B>
__device__ __forceinline__ uint32_t e2m1_f16(uint32_t w) {
  uint32_t r;
  if constexpr (B == 0)
    asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %1;\n cvt.rn.f16x2.e2m1x2 %0, a;\n}" : "=r"(r) : "r"(w));
  else if constexpr (B == 1)
    asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %1;\n cvt.rn.f16x2.e2m1x2 %0, b;\n}" : "=r"(r) : "r"(w));
  else if constexpr (B == 2)
    asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %1;\n cvt.rn.f16x2.e2m1x2 %0, c;\n}" : "=r"(r) : "r"(w));
  else
    asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %1;\n cvt.rn.f16x2.e2m1x2 %0, d;\n}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void mma_m16n8k16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load_stream16(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 load_stream8(const uint8_t* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == KAB_F32) return static_cast<const float*>(p)[i];
  if (dtype == KAB_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
template <int T>
__device__ __forceinline__ void store_any(void* p, int64_t i, float v) {
  if constexpr (T == kF32) static_cast<float*>(p)[i] = v;
  else if constexpr (T == kBF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// ------------------------------------------------------------------ layout

constexpr int kGemvThreads = 256, kGemvWarps = 8, kGemvDepth = 4;

// Bytes of one token's slice of x (hi terms, and lo terms for fp32): a multiple of 256 and 64 more,
// so that the tokens of a group lie in different banks.
__host__ __device__ constexpr int gemv_pitch(int slice_chunks) { return slice_chunks * 256 + 64; }
__host__ __device__ constexpr int gemv_smem(int m, int slice_chunks, int nt, bool split) {
  return m * gemv_pitch(slice_chunks) * (split ? 2 : 1) + 2 * kGemvWarps * 16 * 8 * nt * 4 + 8 * nt * 4;
}

// ------------------------------------------------------------------ the kernel

// MX: MXFP4 (e8m0 per 32), else NVFP4 (e4m3 per 16). NT: groups of 8 tokens. WIDE: rows of codes
// start on 16 bytes (K a multiple of 32 and an aligned weight), else on 8.
template <int T, int MX, int NT, int WIDE>
__global__ void __launch_bounds__(kGemvThreads, 2) gemv_fp4_kernel(GemvArgs a) {
  constexpr bool SPLIT = T == kF32;
  constexpr int COLS = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int slice = blockIdx.y, m0 = blockIdx.z * COLS, tokens = min(COLS, a.m - m0);
  const int c_first = slice * a.slice_chunks, c_count = min(a.slice_chunks, a.chunks - c_first);
  const int pitch = gemv_pitch(a.slice_chunks);
  float* sums = reinterpret_cast<float*>(smem + tokens * pitch * (SPLIT ? 2 : 1));  // [2][8 warps][16][COLS]
  float* unit = sums + 2 * kGemvWarps * 16 * COLS;                                  // [COLS]

  // ---- this warp's stream: rows of the block's tiles, chunks kw, kw + KW, ... of the slice
  const int KW = a.k_warps, RW = kGemvWarps / KW, kw = warp & (KW - 1), rw = warp / KW;
  const int64_t row_lo = static_cast<int64_t>(a.n) * blockIdx.x / a.blocks;
  const int64_t row_hi = static_cast<int64_t>(a.n) * (blockIdx.x + 1) / a.blocks;
  const int tiles = static_cast<int>((row_hi - row_lo + 16 * RW - 1) / (16 * RW));
  const int mine = kw < c_count ? (c_count - kw + KW - 1) / KW : 0;  // chunks per tile
  const int cols = a.k >> (MX ? 5 : 4), half = a.k >> 1;

  struct Slot {
    uint4 w0, w1;      // 32 codes of rows g and g + 8
    uint32_t s0, s1;   // their scales: two e4m3 bytes, or one e8m0
  };
  const int k_last = max(0, (a.k - 1) / 32 * 32);  // the last 32 codes (or 16) of a row
  Slot slots[kGemvDepth] = {};
  int is_tile = 0, is_chunk = 0;  // what the next issue loads
  // the first scale of 32 codes; NVFP4 has two
  auto scale_at = [&](int64_t row, int col) -> uint32_t {
    if constexpr (MX) {
      return __ldg(a.scales + (a.swizzle ? scale_offset_swizzled(row, col, cols) : row * cols + col));
    } else if constexpr (WIDE) {  // col is even: both lie in one 4-column block
      return __ldg(reinterpret_cast<const uint16_t*>(
          a.scales + (a.swizzle ? scale_offset_swizzled(row, col, cols) : row * cols + col)));
    } else {
      const int next = min(col + 1, cols - 1);
      const uint32_t s0 = __ldg(a.scales + (a.swizzle ? scale_offset_swizzled(row, col, cols) : row * cols + col));
      const uint32_t s1 = __ldg(a.scales + (a.swizzle ? scale_offset_swizzled(row, next, cols) : row * cols + next));
      return s0 | s1 << 8;
    }
  };
  // Every load is made, at the nearest place that exists: rows past the block's are not written, and
  // x is zero past K. (Loads under conditions were waited for at once: 98 us where these take 40 at
  // 1 x 28672 x 8192.)
  auto issue = [&](Slot& s) {
    const int64_t row = row_lo + (static_cast<int64_t>(is_tile) * RW + rw) * 16 + g;
    const int k0 = min((c_first + kw + is_chunk * KW) * 128 + t * 32, k_last), col = k0 >> (MX ? 5 : 4);
    const int64_t r0 = min(row, row_hi - 1), r1 = min(row + 8, row_hi - 1);
    const uint8_t* p0 = a.codes + r0 * half + (k0 >> 1);
    const uint8_t* p1 = a.codes + r1 * half + (k0 >> 1);
    if constexpr (WIDE) {
      s.w0 = load_stream16(p0);
      s.w1 = load_stream16(p1);
    } else {
      const int next = k0 + 16 < a.k ? 8 : 0;
      const uint2 x0 = load_stream8(p0), y0 = load_stream8(p0 + next), x1 = load_stream8(p1), y1 = load_stream8(p1 + next);
      s.w0 = make_uint4(x0.x, x0.y, y0.x, y0.y);
      s.w1 = make_uint4(x1.x, x1.y, y1.x, y1.y);
    }
    s.s0 = scale_at(r0, col);
    s.s1 = scale_at(r1, col);
    if (++is_chunk >= mine) {
      is_chunk = 0;
      ++is_tile;
    }
  };
  if (a.k > 0)
#pragma unroll
  for (int i = 0; i < kGemvDepth; ++i) issue(slots[i]);

  // ---- x: the slice's largest finite value per token, then f16 terms in units of it. A lane reads
  // its 8 codes' worth of two MMAs (16 bytes) at unit (k % 32 / 8) * 4 + k % 128 / 32 of a chunk.
  {
    const int k_lo = c_first * 128, count = c_count * 16;  // groups of 8 values
    for (int mt = warp; mt < tokens; mt += kGemvWarps) {
      uint32_t top = 0;
      for (int i = lane; i < count; i += 32) {
        const int k = k_lo + i * 8;
        if (k < a.k) {
          float v[8];
          load8<T>(a.x, (m0 + mt) * a.ldx + k, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t b = __float_as_uint(v[e]) & 0x7FFFFFFFu;
            top = max(top, b < 0x7F800000u ? b : 0u);
          }
        }
      }
      top = __reduce_max_sync(0xffffffffu, top);
      const int e = max(static_cast<int>(top >> 23) - 127, -100);
      const float up = top == 0 ? 1.0f : __uint_as_float((127u + 14u - e) << 23);
      if (lane == 0) unit[mt] = 1.0f / up;
      uint8_t* row = smem + mt * pitch;
      for (int i = lane; i < count; i += 32) {
        const int k = k_lo + i * 8;
        float v[8] = {};
        if (k < a.k) load8<T>(a.x, (m0 + mt) * a.ldx + k, v);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) {
          const __half2 h = __floats2half2_rn(v[2 * e2] * up, v[2 * e2 + 1] * up);
          hi[e2] = *reinterpret_cast<const uint32_t*>(&h);
          if constexpr (SPLIT) {
            const float2 f = __half22float2(h);
            // an infinity has no second term
            const __half2 l = __floats2half2_rn(isinf(f.x) ? 0.0f : v[2 * e2] * up - f.x,
                                                isinf(f.y) ? 0.0f : v[2 * e2 + 1] * up - f.y);
            lo[e2] = *reinterpret_cast<const uint32_t*>(&l);
          }
        }
        const int at = (i >> 4) * 256 + ((i & 3) * 4 + ((i >> 2) & 3)) * 16;
        *reinterpret_cast<uint4*>(row + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if constexpr (SPLIT) *reinterpret_cast<uint4*>(row + tokens * pitch + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
  }
  __syncthreads();

  // columns past the tokens repeat the last one; nobody reads them
  const uint8_t* x_at[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) x_at[j] = smem + min(j * 8 + g, tokens - 1) * pitch + t * 16;
  const int lo_at = tokens * pitch;

  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;

  // products of 128 codes, scaled by f16 pairs m0 / m1 (rows g, g + 8; first and second 16 codes)
  auto products = [&](const Slot& s, int chunk, const uint32_t (&f0)[2], const uint32_t (&f1)[2], float (&c)[NT][4]) {
    const uint32_t w0[4] = {s.w0.x, s.w0.y, s.w0.z, s.w0.w}, w1[4] = {s.w1.x, s.w1.y, s.w1.z, s.w1.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // 8 codes of each row: two MMAs
      const uint32_t a00 = mul_f16x2(e2m1_f16<0>(w0[i]), f0[i >> 1]), a01 = mul_f16x2(e2m1_f16<1>(w0[i]), f0[i >> 1]);
      const uint32_t a02 = mul_f16x2(e2m1_f16<2>(w0[i]), f0[i >> 1]), a03 = mul_f16x2(e2m1_f16<3>(w0[i]), f0[i >> 1]);
      const uint32_t a10 = mul_f16x2(e2m1_f16<0>(w1[i]), f1[i >> 1]), a11 = mul_f16x2(e2m1_f16<1>(w1[i]), f1[i >> 1]);
      const uint32_t a12 = mul_f16x2(e2m1_f16<2>(w1[i]), f1[i >> 1]), a13 = mul_f16x2(e2m1_f16<3>(w1[i]), f1[i >> 1]);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint4 b = *reinterpret_cast<const uint4*>(x_at[j] + chunk * 256 + i * 64);
        mma_m16n8k16(c[j], a00, a10, a01, a11, b.x, b.y);
        mma_m16n8k16(c[j], a02, a12, a03, a13, b.z, b.w);
        if constexpr (SPLIT) {
          const uint4 l = *reinterpret_cast<const uint4*>(x_at[j] + lo_at + chunk * 256 + i * 64);
          mma_m16n8k16(c[j], a00, a10, a01, a11, l.x, l.y);
          mma_m16n8k16(c[j], a02, a12, a03, a13, l.z, l.w);
        }
      }
    }
  };
  auto consume = [&](const Slot& s, int chunk) {
    if constexpr (!MX) {
      const __half2_raw h0 = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(s.s0), __NV_E4M3);
      const __half2_raw h1 = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(s.s1), __NV_E4M3);
      const uint32_t p0 = *reinterpret_cast<const uint32_t*>(&h0), p1 = *reinterpret_cast<const uint32_t*>(&h1);
      const uint32_t f0[2] = {__byte_perm(p0, p0, 0x1010), __byte_perm(p0, p0, 0x3232)};
      const uint32_t f1[2] = {__byte_perm(p1, p1, 0x1010), __byte_perm(p1, p1, 0x3232)};
      products(s, chunk, f0, f1, acc);
    } else {
      const int e0 = s.s0, e1 = s.s1;
      const int r0 = __shfl_sync(0xffffffffu, e0, lane & 28), r1 = __shfl_sync(0xffffffffu, e1, lane & 28);
      auto pow2 = [](int d) -> uint32_t {  // 2^d as an f16 pair, d in -24 .. 15
        const uint32_t h = d >= -14 ? static_cast<uint32_t>(d + 15) << 10 : 1u << (d + 24);
        return h | (h << 16);
      };
      // the scale of 32 zeros does not count
      const bool near0 = e0 - r0 >= -20 && e0 - r0 <= 13, near1 = e1 - r1 >= -20 && e1 - r1 <= 13;
      const bool ok0 = near0 || (s.w0.x | s.w0.y | s.w0.z | s.w0.w) == 0, ok1 = near1 || (s.w1.x | s.w1.y | s.w1.z | s.w1.w) == 0;
      if (__all_sync(0xffffffffu, ok0 && ok1 && e0 != 255 && e1 != 255)) {
        const uint32_t m_0 = near0 ? pow2(e0 - r0) : 0u, m_1 = near1 ? pow2(e1 - r1) : 0u;
        const uint32_t f0[2] = {m_0, m_0}, f1[2] = {m_1, m_1};
        float c[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.0f;
        products(s, chunk, f0, f1, c);
        const float u0 = e8m0_value(static_cast<uint8_t>(r0)), u1 = e8m0_value(static_cast<uint8_t>(r1));
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          acc[j][0] = fmaf(c[j][0], u0, acc[j][0]);
          acc[j][1] = fmaf(c[j][1], u0, acc[j][1]);
          acc[j][2] = fmaf(c[j][2], u1, acc[j][2]);
          acc[j][3] = fmaf(c[j][3], u1, acc[j][3]);
        }
      } else {
        for (int q = 0; q < 4; ++q) {  // lane q's blocks of every row
          const uint32_t one = t == q ? 0x3C003C00u : 0u;
          const uint32_t f[2] = {one, one};
          float c[NT][4];
#pragma unroll
          for (int j = 0; j < NT; ++j) c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.0f;
          products(s, chunk, f, f, c);
          const float u0 = e8m0_value(static_cast<uint8_t>(__shfl_sync(0xffffffffu, e0, (lane & 28) | q)));
          const float u1 = e8m0_value(static_cast<uint8_t>(__shfl_sync(0xffffffffu, e1, (lane & 28) | q)));
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            acc[j][0] = fmaf(c[j][0], u0, acc[j][0]);
            acc[j][1] = fmaf(c[j][1], u0, acc[j][1]);
            acc[j][2] = fmaf(c[j][2], u1, acc[j][2]);
            acc[j][3] = fmaf(c[j][3], u1, acc[j][3]);
          }
        }
      }
    }
  };

  // the sums of a tile: every warp's fragments to shared memory, then one thread per output
  int done_chunks = 0, tile = 0;
  auto finish_tile = [&]() {
    float* buf = sums + (tile & 1) * kGemvWarps * 16 * COLS;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float* at = buf + (warp * 16 + g) * COLS + j * 8 + 2 * t;
      *reinterpret_cast<float2*>(at) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2*>(at + 8 * COLS) = make_float2(acc[j][2], acc[j][3]);
      acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
    }
    __syncthreads();  // the other buffer is free once every warp is here again
    for (int i = tid; i < RW * 16 * tokens; i += kGemvThreads) {
      const int r = i % (RW * 16), mt = i / (RW * 16);
      const int64_t row = row_lo + static_cast<int64_t>(tile) * RW * 16 + r;
      if (row < row_hi) {
        const float* from = buf + (r >> 4) * KW * 16 * COLS + (r & 15) * COLS + mt;
        float y = from[0];
        for (int w = 1; w < KW; ++w) y += from[w * 16 * COLS];
        y *= unit[mt] * a.ts[a.ts_per_row ? row : 0];
        if (a.slices > 1) {
          a.partial[(static_cast<int64_t>(slice) * a.m + m0 + mt) * a.n + row] = y;
        } else {
          if (a.bias != nullptr) y += load_any(a.bias, a.bias_dtype, row);
          store_any<T>(a.out, (m0 + mt) * a.ldo + row, y);
        }
      }
    }
    ++tile;
  };
  if (mine == 0) {  // no chunk of the slice is left for this warp: its sums are zeros
    while (tile < tiles) finish_tile();
    return;
  }
  const int total = tiles * mine;
  for (int i0 = 0; i0 < total; i0 += kGemvDepth) {
#pragma unroll
    for (int i = 0; i < kGemvDepth; ++i) {
      if (i0 + i < total) {
        consume(slots[i], kw + done_chunks * KW);
        if (a.k > 0) issue(slots[i]);
        if (++done_chunks == mine) {
          done_chunks = 0;
          finish_tile();
        }
      }
    }
  }
}

// The slices' sums (each in units already undone and times the tensor scale), added in order.
template <int T>
__global__ void __launch_bounds__(256) gemv_join_kernel(GemvArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int row = blockIdx.x * 256 + threadIdx.x, mt = blockIdx.y;
  if (row >= a.n) return;
  float y = 0.0f;
#pragma unroll 4
  for (int s = 0; s < a.slices; ++s) y += __ldg(a.partial + (static_cast<int64_t>(s) * a.m + mt) * a.n + row);
  if (a.bias != nullptr) y += load_any(a.bias, a.bias_dtype, row);
  store_any<T>(a.out, mt * a.ldo + row, y);
}

}  // namespace kab
