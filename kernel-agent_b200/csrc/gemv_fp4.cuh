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
//  * e2m1 -> f16 is one exact conversion per two codes. For few tokens (GROUPED) the scales never
//    touch the codes: the MMA's 8 columns hold one token's blocks apart. A lane's 32 codes are the two
//    NVFP4 blocks 2 t and 2 t + 1 of the 128 of the quad (or MXFP4's block t), and column n carries x
//    only in the lane that owns block n, zeros elsewhere, so column n sums block n alone; one
//    multiply-add per row and block then applies the scale in fp32, exactly for every scale. NVFP4
//    fills the columns with one token, MXFP4 with two; more tokens take more MMAs on the same
//    converted codes. (Scaling the codes costs 32 packed multiplications per chunk instead: 37 us
//    against GROUPED's 29 for one token at 28672 x 8192.)
//  * For more tokens the codes are scaled. An NVFP4 code times its e4m3 scale has at most 6
//    significant bits and lies in [2^-10, 2688]: exact in f16, one packed multiplication per two
//    codes. An MXFP4 scale does not fit f16: the four 32-code blocks of a row's 128 codes are taken in
//    units of the first one's scale where they lie within 2^-20 .. 2^13 of it (exact), and the 16 x 8
//    products of the 128 codes are added in fp32 with that scale; otherwise each block is taken by
//    itself.
//  * x enters as f16, each token (and K slice) in units of a power of two that puts its largest
//    finite value in [2^14, 2^15): bf16 and f16 keep all their bits down to 2^-29 of it; fp32 is
//    split into two f16 terms (22 bits) and multiplied twice. It is converted once per block and
//    stays in shared memory while the block streams its rows.
//  * The (16-row tile, 128-code chunk) pairs of a K slice stand in one line, cut into equal parts for
//    the blocks and again for their warps: every warp streams its part with kGemvDepth chunks in
//    flight in registers and waits for nobody. Tiles that lie within a warp are written by it; those
//    that several warps of a block share are added in shared memory at the end, those that two
//    blocks share (and the slices of K, where x does not fit in shared memory) in a second launch.
//    Always in the order of the line.
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
  int tiles, blocks;                 // 16-row tiles; blocks per slice
  float* partial;                    // [2, slices, m, n]: a tile's sum or its first part, and its second part
};

// The line of `total` units cut into `parts`: the first total % parts take one more.
struct GemvCut {
  int share, longer;
  __host__ __device__ GemvCut(int total, int parts) : share(total / parts), longer(total % parts) {}
  __host__ __device__ int begin(int part) const { return share * part + (part < longer ? part : longer); }
  __host__ __device__ int part_of(int unit) const {
    const int split = longer * (share + 1);
    return unit < split ? unit / (share + 1) : longer + (unit - split) / share;
  }
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
__host__ __device__ constexpr int gemv_smem(int m, int slice_chunks, int columns, bool split) {
  return m * gemv_pitch(slice_chunks) * (split ? 2 : 1) + 256 + 2 * kGemvWarps * 16 * columns * 4 + columns * 4 +
         2 * kGemvWarps * 4;
}

// ------------------------------------------------------------------ the kernel

// Tokens that NT groups of the MMA's columns take.
constexpr int gemv_columns(bool mx, int nt, bool grouped) { return grouped ? (mx ? 2 * nt : nt) : 8 * nt; }

// MX: MXFP4 (e8m0 per 32), else NVFP4 (e4m3 per 16). NT: groups of 8 MMA columns. WIDE: rows of codes
// start on 16 bytes (K a multiple of 32 and an aligned weight), else on 8.
template <int T, int MX, int NT, int WIDE, int GROUPED>
__global__ void __launch_bounds__(kGemvThreads, 2) gemv_fp4_kernel(GemvArgs a) {
  constexpr bool SPLIT = T == kF32;
  constexpr int COLS = gemv_columns(MX, NT, GROUPED);
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int slice = blockIdx.y, m0 = blockIdx.z * COLS, tokens = min(COLS, a.m - m0);
  const int c_first = slice * a.slice_chunks, c_count = min(a.slice_chunks, a.chunks - c_first);
  const int pitch = gemv_pitch(a.slice_chunks);
  uint8_t* zeros = smem + tokens * pitch * (SPLIT ? 2 : 1);  // 256 bytes: what a column's other lanes read
  float* sums = reinterpret_cast<float*>(zeros + 256);  // [8 warps][2][16][COLS]
  float* unit = sums + 2 * kGemvWarps * 16 * COLS;                                  // [COLS]

  int* seg_tile = reinterpret_cast<int*>(unit + COLS);  // [8 warps][2]: 2 * tile + (its end is here), or -1

  // ---- this warp's part of the line
  const GemvCut cut(a.tiles * c_count, a.blocks);
  const int b_lo = cut.begin(blockIdx.x), b_hi = cut.begin(blockIdx.x + 1);
  const GemvCut warps(b_hi - b_lo, kGemvWarps);
  const int u_lo = b_lo + warps.begin(warp), u_hi = b_lo + warps.begin(warp + 1);
  const int cols = a.k >> (MX ? 5 : 4), half = a.k >> 1;
  if (tid < 2 * kGemvWarps) seg_tile[tid] = -1;
  if (tid < 16) reinterpret_cast<uint4*>(zeros)[tid] = make_uint4(0, 0, 0, 0);

  struct Slot {
    uint4 w0, w1;      // 32 codes of rows g and g + 8
    uint32_t s0, s1;   // their scales: two e4m3 bytes, or one e8m0
  };
  Slot slots[kGemvDepth] = {};
  int is_unit = u_lo, is_tile = u_lo / c_count, is_chunk = u_lo % c_count;  // what the next issue loads
  const uint8_t *code0, *code1, *scale0, *scale1;  // the tile's rows g and g + 8
  auto point = [&]() {
    const int r0 = min(is_tile * 16 + g, a.n - 1), r1 = min(is_tile * 16 + g + 8, a.n - 1);
    code0 = a.codes + static_cast<int64_t>(r0) * half;
    code1 = a.codes + static_cast<int64_t>(r1) * half;
    scale0 = a.scales + (a.swizzle ? scale_offset_swizzled(r0, 0, cols) : static_cast<int64_t>(r0) * cols);
    scale1 = a.scales + (a.swizzle ? scale_offset_swizzled(r1, 0, cols) : static_cast<int64_t>(r1) * cols);
  };
  point();
  // Every load is made, at the nearest place that exists: rows past n are not written, and x is zero
  // past K. (Loads under conditions were waited for at once: 98 us against 53 at 1 x 28672 x 8192.)
  const int last = max(0, (a.k - 1) / 32);  // the last 32 codes (or 16) of a row
  auto issue = [&](Slot& s) {
    if (is_unit >= u_hi) return;
    const int at = min((c_first + is_chunk) * 4 + t, last);  // in 32 codes
    if constexpr (WIDE) {
      s.w0 = load_stream16(code0 + at * 16);
      s.w1 = load_stream16(code1 + at * 16);
    } else {
      const int next = at * 32 + 16 < a.k ? 8 : 0;
      const uint2 x0 = load_stream8(code0 + at * 16), y0 = load_stream8(code0 + at * 16 + next);
      const uint2 x1 = load_stream8(code1 + at * 16), y1 = load_stream8(code1 + at * 16 + next);
      s.w0 = make_uint4(x0.x, x0.y, y0.x, y0.y);
      s.w1 = make_uint4(x1.x, x1.y, y1.x, y1.y);
    }
    const int col = MX ? at : 2 * at, off = a.swizzle ? (col >> 2) * 512 + (col & 3) : col;
    if constexpr (MX) {
      s.s0 = __ldg(scale0 + off);
      s.s1 = __ldg(scale1 + off);
    } else if constexpr (WIDE) {  // col is even: both scales lie in one 4-column block
      s.s0 = __ldg(reinterpret_cast<const uint16_t*>(scale0 + off));
      s.s1 = __ldg(reinterpret_cast<const uint16_t*>(scale1 + off));
    } else {
      const int next = col + 1 < cols ? 1 : 0;
      s.s0 = __ldg(scale0 + off) | static_cast<uint32_t>(__ldg(scale0 + off + next)) << 8;
      s.s1 = __ldg(scale1 + off) | static_cast<uint32_t>(__ldg(scale1 + off + next)) << 8;
    }
    ++is_unit;
    if (++is_chunk == c_count) {
      is_chunk = 0;
      ++is_tile;
      point();
    }
  };
  if (a.k > 0) {
#pragma unroll
    for (int i = 0; i < kGemvDepth; ++i) issue(slots[i]);
  }

  // ---- x: the slice's largest finite value per token, then f16 terms in units of it. A lane reads
  // its 8 codes' worth of two MMAs (16 bytes) at unit (k % 32 / 8) * 4 + k % 128 / 32 of a chunk.
  {
    const int k_lo = c_first * 128, count = c_count * 16;  // groups of 8 values
    uint32_t* tops = reinterpret_cast<uint32_t*>(unit);
    if (tid < COLS) tops[tid] = 0;
    __syncthreads();
    // eight warps share the tokens, or a token where there are fewer
    const int per = tokens > 4 ? 1 : tokens > 2 ? 2 : tokens > 1 ? 4 : 8, step = per * 32;
    const int first = warp % per * 32 + lane;
    for (int mt = warp / per; mt < tokens; mt += kGemvWarps / per) {
      uint32_t top = 0;
#pragma unroll 4
      for (int i = first; i < count; i += step) {
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
      if (lane == 0 && top != 0) atomicMax(tops + mt, top);
    }
    __syncthreads();
    for (int mt = warp / per; mt < tokens; mt += kGemvWarps / per) {
      const uint32_t top = tops[mt];
      const int e = max(static_cast<int>(top >> 23) - 127, -100);
      const float up = top == 0 ? 1.0f : __uint_as_float((127u + 14u - e) << 23);
      uint8_t* row = smem + mt * pitch;
#pragma unroll 4
      for (int i = first; i < count; i += step) {
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
    __syncthreads();
    if (tid < tokens) {
      const uint32_t top = tops[tid];
      unit[tid] = top == 0 ? 1.0f : 1.0f / __uint_as_float((127u + 14u - max(static_cast<int>(top >> 23) - 127, -100)) << 23);
    }
  }
  __syncthreads();

  const int lo_at = tokens * pitch;
  // where a lane reads column g of group j; `step`: 256 bytes per chunk, or none in the zeros. With
  // NVFP4 blocks apart the lane's first block and its second have a column each.
  constexpr int SIDES = GROUPED && !MX ? 2 : 1;
  const uint8_t* x_at[NT][SIDES];
  int x_step[NT][SIDES];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int side = 0; side < SIDES; ++side) {
      // columns past the tokens repeat the last one; nobody reads them
      const int token = !GROUPED ? j * 8 + g : MX ? 2 * j + (g & 1) : j;
      const bool here = !GROUPED || (MX ? t == g >> 1 : g == 2 * t + side);
      x_at[j][side] = here ? smem + min(token, tokens - 1) * pitch + t * 16 : zeros;
      x_step[j][side] = here ? 256 : 0;
    }
  }

  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;

  // products of 128 codes, in GROUPED as they are, else scaled by f16 pairs f0 / f1 (rows g, g + 8;
  // first and second 16 codes)
  auto products = [&](const Slot& s, int chunk, const uint32_t (&f0)[2], const uint32_t (&f1)[2], float (&c)[NT][4]) {
    const uint32_t w0[4] = {s.w0.x, s.w0.y, s.w0.z, s.w0.w}, w1[4] = {s.w1.x, s.w1.y, s.w1.z, s.w1.w};
    float c2[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // with one group: halves the chain of dependent products
    auto scaled = [&](uint32_t v, uint32_t f) { return GROUPED ? v : mul_f16x2(v, f); };
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // 8 codes of each row: two MMAs
      const uint32_t a00 = scaled(e2m1_f16<0>(w0[i]), f0[i >> 1]), a01 = scaled(e2m1_f16<1>(w0[i]), f0[i >> 1]);
      const uint32_t a02 = scaled(e2m1_f16<2>(w0[i]), f0[i >> 1]), a03 = scaled(e2m1_f16<3>(w0[i]), f0[i >> 1]);
      const uint32_t a10 = scaled(e2m1_f16<0>(w1[i]), f1[i >> 1]), a11 = scaled(e2m1_f16<1>(w1[i]), f1[i >> 1]);
      const uint32_t a12 = scaled(e2m1_f16<2>(w1[i]), f1[i >> 1]), a13 = scaled(e2m1_f16<3>(w1[i]), f1[i >> 1]);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int side = SIDES == 2 ? i >> 1 : 0;
        const uint8_t* at = x_at[j][side] + chunk * x_step[j][side] + i * 64;
        const uint4 b = *reinterpret_cast<const uint4*>(at);
        mma_m16n8k16(c[j], a00, a10, a01, a11, b.x, b.y);
        mma_m16n8k16(NT == 1 ? c2 : c[j], a02, a12, a03, a13, b.z, b.w);
        if constexpr (SPLIT) {
          const uint4 l = *reinterpret_cast<const uint4*>(x_step[j][side] ? at + lo_at : at);
          mma_m16n8k16(c[j], a00, a10, a01, a11, l.x, l.y);
          mma_m16n8k16(NT == 1 ? c2 : c[j], a02, a12, a03, a13, l.z, l.w);
        }
      }
    }
    if constexpr (NT == 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) c[0][e] += c2[e];
    }
  };
  auto consume = [&](const Slot& s, int chunk) {
    if constexpr (GROUPED) {
      const uint32_t none[2] = {0, 0};
      float c[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.0f;
      products(s, chunk, none, none, c);
      if constexpr (MX) {  // columns 2 t and 2 t + 1: block t, two tokens
        const float u0 = e8m0_value(static_cast<uint8_t>(s.s0)), u1 = e8m0_value(static_cast<uint8_t>(s.s1));
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          acc[j][0] = fmaf(c[j][0], u0, acc[j][0]);
          acc[j][1] = fmaf(c[j][1], u0, acc[j][1]);
          acc[j][2] = fmaf(c[j][2], u1, acc[j][2]);
          acc[j][3] = fmaf(c[j][3], u1, acc[j][3]);
        }
      } else {  // columns 2 t and 2 t + 1: the lane's two blocks
        const __half2_raw h0 = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(s.s0), __NV_E4M3);
        const __half2_raw h1 = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(s.s1), __NV_E4M3);
        const float2 u0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
        const float2 u1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          acc[j][0] = fmaf(c[j][0], u0.x, acc[j][0]);
          acc[j][1] = fmaf(c[j][1], u0.y, acc[j][1]);
          acc[j][2] = fmaf(c[j][2], u1.x, acc[j][2]);
          acc[j][3] = fmaf(c[j][3], u1.y, acc[j][3]);
        }
      }
    } else if constexpr (!MX) {
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

  // one output of a tile: the final value, or one of its two partial sums
  auto put = [&](int tile, int r, int mt, float y, int part) {
    const int64_t row = static_cast<int64_t>(tile) * 16 + r;
    if (row >= a.n || mt >= tokens) return;
    y *= unit[mt] * a.ts[a.ts_per_row ? row : 0];
    if (part < 0 && a.slices == 1) {
      if (a.bias != nullptr) y += load_any(a.bias, a.bias_dtype, row);
      store_any<T>(a.out, (m0 + mt) * a.ldo + row, y);
    } else {
      a.partial[((static_cast<int64_t>(max(part, 0)) * a.slices + slice) * a.m + m0 + mt) * a.n + row] = y;
    }
  };
  int tile = u_lo / c_count, chunk = u_lo % c_count, begun = chunk;
  auto end_segment = [&]() {
    const bool ends = chunk == c_count - 1, whole = begun == 0 && ends;
    const int seg = warp * 2 + (begun == 0);  // 0: the tile began before this warp, 1: it begins here
    auto one = [&](int r, int mt, float y) {
      if (whole) put(tile, r, mt, y, -1);
      else sums[(seg * 16 + r) * COLS + mt] = y;
    };
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if constexpr (GROUPED) {
        // the blocks' sums meet: over the quad, and with NVFP4 over a lane's two blocks
        float v[4] = {acc[j][0], acc[j][1], acc[j][2], acc[j][3]};
        if constexpr (!MX) {
          v[0] += v[1];
          v[2] += v[3];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] += __shfl_xor_sync(0xffffffffu, v[e], 1);
          v[e] += __shfl_xor_sync(0xffffffffu, v[e], 2);
        }
        if (t == 0) {
          if constexpr (MX) {
            one(g, 2 * j, v[0]);
            one(g, 2 * j + 1, v[1]);
            one(g + 8, 2 * j, v[2]);
            one(g + 8, 2 * j + 1, v[3]);
          } else {
            one(g, j, v[0]);
            one(g + 8, j, v[2]);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) one(g + 8 * (e >> 1), j * 8 + 2 * t + (e & 1), acc[j][e]);
      }
      acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
    }
    if (!whole && lane == 0) seg_tile[seg] = 2 * tile + ends;
    begun = 0;
  };
  for (int u = u_lo; u < u_hi; u += kGemvDepth) {
#pragma unroll
    for (int i = 0; i < kGemvDepth; ++i) {
      if (u + i < u_hi) {
        consume(slots[i], chunk);
        if (a.k > 0) issue(slots[i]);
        if (chunk == c_count - 1 || u + i == u_hi - 1) end_segment();
        if (++chunk == c_count) {
          chunk = 0;
          ++tile;
        }
      }
    }
  }
  __syncthreads();
  // the tiles that warps share: from where they begin in this block (a warp's second segment, or the
  // first warp's first), through the following warps' first segments
  for (int i = tid; i < (kGemvWarps + 1) * 16 * COLS; i += kGemvThreads) {
    const int head = i / (16 * COLS), cell = i % (16 * COLS);
    const int seg = head == 0 ? 0 : (head - 1) * 2 + 1, first = seg_tile[seg];
    if (first < 0) continue;
    float y = sums[seg * 16 * COLS + cell];
    int end = first & 1;
    for (int w = (seg >> 1) + 1; w < kGemvWarps && seg_tile[2 * w] >= 0 && seg_tile[2 * w] >> 1 == first >> 1; ++w) {
      y += sums[2 * w * 16 * COLS + cell];
      end = seg_tile[2 * w] & 1;
    }
    put(first >> 1, cell / COLS, cell % COLS, y, head == 0 ? 1 : end ? -1 : 0);
  }
}

// The tiles that two blocks share and the slices of K, added in order (units and the tensor scale
// are in the sums already).
template <int T>
__global__ void __launch_bounds__(256) gemv_join_kernel(GemvArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int row = blockIdx.x * 256 + threadIdx.x, mt = blockIdx.y, tile = row / 16;
  if (row >= a.n) return;
  float y = 0.0f;
  for (int s = 0; s < a.slices; ++s) {
    const int count = min(a.slice_chunks, a.chunks - s * a.slice_chunks);
    const GemvCut cut(a.tiles * count, a.blocks);
    const bool shared = cut.part_of(tile * count) != cut.part_of(tile * count + count - 1);
    if (a.slices == 1 && !shared) return;
    const float* at = a.partial + (static_cast<int64_t>(s) * a.m + mt) * a.n + row;
    y += __ldg(at);
    if (shared) y += __ldg(at + static_cast<int64_t>(a.slices) * a.m * a.n);
  }
  if (a.bias != nullptr) y += load_any(a.bias, a.bias_dtype, row);
  store_any<T>(a.out, mt * a.ldo + row, y);
}

}  // namespace kab
