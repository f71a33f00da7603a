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
//    converted codes. (With scaled codes, 32 packed multiplications per 128 x 16 codes, one token took
//    37.0 us at 28672 x 8192, with blocks apart 34.1 in the same form of the kernel.)
//  * For more tokens the codes are scaled. An NVFP4 code times its e4m3 scale has at most 6
//    significant bits and lies in [2^-10, 2688]: exact in f16, one packed multiplication per two
//    codes. An MXFP4 scale does not fit f16: the four 32-code blocks of a row's 128 codes are taken in
//    units of the first one's scale where they lie within 2^-20 .. 2^13 of it (exact), and the 16 x 8
//    products of the 128 codes are added in fp32 with that scale; otherwise each block is taken by
//    itself.
//  * x enters as f16, each token (and K slice) in units of a power of two that puts its largest
//    finite value in [2^14, 2^15): bf16 and f16 keep all their bits down to 2^-29 of it; fp32 is
//    split into two f16 terms (22 bits) and multiplied twice, the products of 128 codes added to the rest in
//    fp32 (sums carried by the MMAs alone, which cut them, were off by 3e-6 at 8 x 8192 x 8192 and 7e-6 at K =
//    28672; 3e-7 now, at the same time). It stays in shared memory while a block
//    streams its rows, converted there for one token, by a launch before for more (5 x 1001 x 4080: 8.1 us,
//    with every block converting for itself 13.3).
//  * The (32-row tile, 256-code chunk) pairs of a K slice stand in one line, cut into equal parts for
//    the blocks. A block's warps take its units in turn, each through a ring of its own in shared
//    memory (cp.async, whole 128-byte lines of a row), and wait for nobody: every warp leaves its sums
//    of every tile in shared memory and they are added at the end, in the order of the warps. Where
//    those sums would leave room for one block per SM only (three tokens and more, many tiles per
//    block) each warp takes a contiguous part of the block's instead, and leaves only the sums of a tile
//    that began before its part, beside its ring, and of the one that it does not finish, in it. (In
//    turns against contiguous parts: 33 us against 39 at 1 x 8192 x 28672, 22.6 against 24.8 at 8 x 4096
//    x 14336 MXFP4; 51 against 49 at 8 x 28672 x 8192, where turns leave one block per SM.)
//  * 32 rows share one read of x, and whole lines in place of 64-byte pieces keep L1's data pipe, which
//    bounded an earlier form (66 % busy at 3.9 TB/s), below the stream.
//  * Tiles that two blocks share, and the slices of K where x does not fit in shared memory, are added
//    by another launch, in the order of the line.
//
// One token at 28672 x 8192 NVFP4: 31 us = 4.27 TB/s = 0.65 of the measured copy. About 5 us of it
// are fixed (x's conversion, the join's launch); the rest streams at 5.2 TB/s, and no faster from L2:
// 16 warps per SM, each a chain of conversions and MMAs (issue slots 45 % used, ALU 43 %), bound it.
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
  int chunks, slice_chunks, slices;  // 256-code chunks of K, of a slice of it, and slices
  int tiles, blocks;                 // 32-row tiles; blocks per slice
  float* partial;                    // [2, slices, m, n]: a tile's sum or its first part, and its second part
  uint8_t* x_terms;                  // [slices, m, 1 or 2 terms, slice_chunks * 512]: x as f16, or NULL
  float* x_units;                    // [slices, m]
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
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int BYTES>
__device__ __forceinline__ void gemv_copy(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
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

constexpr int kGemvThreads = 256, kGemvWarps = 8, kGemvRows = 32, kGemvCodes = 256;
// A warp's ring: 32 rows x 128 bytes of codes, and for each row the 4-byte words that hold its scales
// of these codes (one word more than needed where they do not start on 4 bytes).
constexpr int kGemvStages = 2;
__host__ __device__ constexpr int gemv_scale_pitch(bool mx) { return mx ? 12 : 20; }
__host__ __device__ constexpr int gemv_stage_bytes(bool mx) { return kGemvRows * (128 + gemv_scale_pitch(mx)); }

// Bytes of one token's slice of x (hi terms, and lo terms for fp32): a multiple of 512 and 64 more,
// so that the tokens of a group lie in different banks.
__host__ __device__ constexpr int gemv_pitch(int slice_chunks) { return slice_chunks * 512 + 64; }
// `spans`: tiles that a block's part of the line can touch, where its warps take turns, else 1.
__host__ __device__ constexpr int gemv_smem(bool mx, int m, int slice_chunks, int columns, bool split, int spans) {
  return kGemvWarps * kGemvStages * gemv_stage_bytes(mx) + m * gemv_pitch(slice_chunks) * (split ? 2 : 1) + 256 +
         spans * kGemvWarps * kGemvRows * columns * 4 + columns * 4 + 2 * kGemvWarps * 4;
}
// Tokens that NT groups of the MMA's columns take.
constexpr int gemv_columns(bool mx, int nt, bool grouped) { return grouped ? (mx ? 2 * nt : nt) : 8 * nt; }

// ------------------------------------------------------------------ x as f16

// The largest finite value's bits -> the power of two that puts it in [2^14, 2^15).
__device__ __forceinline__ float gemv_up(uint32_t top) {
  return top == 0 ? 1.0f : __uint_as_float((127u + 14u - max(static_cast<int>(top >> 23) - 127, -100)) << 23);
}
template <int T>
__device__ __forceinline__ uint32_t gemv_top8(const GemvArgs& a, int64_t row, int k, uint32_t top) {
  if (k >= a.k) return top;
  float v[8];
  load8<T>(a.x, row * a.ldx + k, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = __float_as_uint(v[e]) & 0x7FFFFFFFu;
    top = max(top, b < 0x7F800000u ? b : 0u);
  }
  return top;
}
// Eight values (the i-th eight of a slice) as f16 terms, at their place: a lane reads its 8 codes'
// worth of two MMAs (16 bytes) at unit (k % 32 / 8) * 4 + k % 128 / 32 of each 128 values.
template <int T>
__device__ __forceinline__ void gemv_convert8(const GemvArgs& a, int64_t row, int k, float up, int i, uint8_t* hi_to,
                                              uint8_t* lo_to) {
  float v[8] = {};
  if (k < a.k) load8<T>(a.x, row * a.ldx + k, v);
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float x0 = v[2 * e] * up, x1 = v[2 * e + 1] * up;
    const __half2 h = __floats2half2_rn(x0, x1);
    hi[e] = *reinterpret_cast<const uint32_t*>(&h);
    if constexpr (T == kF32) {
      const float2 f = __half22float2(h);
      // an infinity has no second term
      const __half2 l = __floats2half2_rn(isinf(f.x) ? 0.0f : x0 - f.x, isinf(f.y) ? 0.0f : x1 - f.y);
      lo[e] = *reinterpret_cast<const uint32_t*>(&l);
    }
  }
  const int at = (i >> 4) * 256 + ((i & 3) * 4 + ((i >> 2) & 3)) * 16;
  *reinterpret_cast<uint4*>(hi_to + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  if constexpr (T == kF32) *reinterpret_cast<uint4*>(lo_to + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

// One block per slice and token: x's terms and unit for every block of the product.
template <int T>
__global__ void __launch_bounds__(256) gemv_x_kernel(GemvArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ uint32_t red[8];
  const int slice = blockIdx.x, mt = blockIdx.y, tid = threadIdx.x;
  const int k_lo = slice * a.slice_chunks * kGemvCodes, count = a.slice_chunks * (kGemvCodes / 8);
  uint32_t top = 0;
#pragma unroll 8
  for (int i = tid; i < count; i += 256) top = gemv_top8<T>(a, mt, k_lo + i * 8, top);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = max(top, red[w]);
  const float up = gemv_up(top);
  const int64_t at = static_cast<int64_t>(slice) * a.m + mt, bytes = a.slice_chunks * 512;
  uint8_t* hi = a.x_terms + at * bytes * (T == kF32 ? 2 : 1);
#pragma unroll 4
  for (int i = tid; i < count; i += 256) gemv_convert8<T>(a, mt, k_lo + i * 8, up, i, hi, hi + bytes);
  if (tid == 0) a.x_units[at] = 1.0f / up;
}

// ------------------------------------------------------------------ the kernel

// MX: MXFP4 (e8m0 per 32), else NVFP4 (e4m3 per 16). NT: groups of 8 MMA columns. WIDE: rows of codes
// start on 16 bytes and rows of scales on 4 (K a multiple of 64 for NVFP4, 128 for MXFP4, and an aligned
// weight), else on 8 and 1.
// TURNS: a block's warps take its units in turn, else a contiguous part each.
template <int T, int MX, int NT, int WIDE, int GROUPED, int TURNS>
__global__ void __launch_bounds__(kGemvThreads, gemv_columns(MX, NT, GROUPED) > 8 ? 1 : 2) gemv_fp4_kernel(GemvArgs a) {
  constexpr bool SPLIT = T == kF32;
  constexpr int COLS = gemv_columns(MX, NT, GROUPED), STAGE = gemv_stage_bytes(MX), SPITCH = gemv_scale_pitch(MX);
  extern __shared__ __align__(128) uint8_t smem_all[];
  uint8_t* smem = smem_all + kGemvWarps * kGemvStages * STAGE;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int slice = blockIdx.y, m0 = blockIdx.z * COLS, tokens = min(COLS, a.m - m0);
  const int c_first = slice * a.slice_chunks, c_count = min(a.slice_chunks, a.chunks - c_first);
  const int pitch = gemv_pitch(a.slice_chunks);
  uint8_t* zeros = smem + tokens * pitch * (SPLIT ? 2 : 1);  // 256 bytes: what a column's other lanes read
  float* unit = reinterpret_cast<float*>(zeros + 256);        // [COLS]
  int* seg_tile = reinterpret_cast<int*>(unit + COLS);        // [8 warps][2]: 2 * tile + (its end is here), or -1
  float* sums = reinterpret_cast<float*>(seg_tile + 2 * kGemvWarps);  // [tiles of the block or 1][8 warps][32][COLS]

  // ---- this block's part of the line
  const GemvCut cut(a.tiles * c_count, a.blocks);
  const int b_lo = cut.begin(blockIdx.x), b_hi = cut.begin(blockIdx.x + 1);
  constexpr int STEP = TURNS ? kGemvWarps : 1;
  const GemvCut warps(b_hi - b_lo, kGemvWarps);
  const int u_lo = TURNS ? b_lo + warp : b_lo + warps.begin(warp), u_hi = TURNS ? b_hi : b_lo + warps.begin(warp + 1);
  const int tile_lo = b_lo / c_count, spans = (b_hi - 1) / c_count - tile_lo + 1;
  const int step_tiles = STEP / c_count, step_chunks = STEP % c_count;
  if constexpr (TURNS) {
    for (int i = tid; i < spans * kGemvWarps * kGemvRows * COLS; i += kGemvThreads) sums[i] = 0.0f;
  } else {
    if (tid < 2 * kGemvWarps) seg_tile[tid] = -1;
  }
  // without turns: the sums of a tile that began before warp w, or of the one that it leaves unfinished:
  // its last, so they fit in its ring
  auto sums_of = [&](int w, bool before) -> float* {
    return before ? sums + w * kGemvRows * COLS : reinterpret_cast<float*>(smem_all + w * kGemvStages * STAGE);
  };
  static_assert(kGemvStages * STAGE >= kGemvRows * COLS * 4, "a tile's sums fit in a ring");
  const int cols = a.k >> (MX ? 5 : 4), half = a.k >> 1;
  if (tid < 16) reinterpret_cast<uint4*>(zeros)[tid] = make_uint4(0, 0, 0, 0);

  // what the next issue loads
  int is_unit = u_lo, is_tile = is_unit / c_count, is_chunk = is_unit % c_count;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem_all)) + warp * kGemvStages * STAGE;
  const int64_t scale_bytes = static_cast<int64_t>(a.n) * cols;
  // A quarter of a row's 16-byte pieces change places on odd rows, so that the fragments' reads (two
  // neighbouring rows x four pieces) touch all banks. Every copy is made at the nearest place that
  // exists: rows past n are not written, and x is zero past K.
  auto issue = [&](int stage) {
    if (is_unit < u_hi) {
      const uint32_t to = ring + stage * STAGE;
      const int chunk = c_first + is_chunk, row0 = is_tile * kGemvRows;
      {
        const int piece = lane & 7, byte = min(chunk * 128 + piece * 16, (half - 1) & ~15);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = i * 4 + (lane >> 3);
          const uint8_t* from = a.codes + static_cast<int64_t>(min(row0 + r, a.n - 1)) * half + byte;
          const uint32_t at = to + r * 128 + ((piece ^ ((r & 1) << 2)) << 4);
          if constexpr (WIDE) {
            gemv_copy<16>(at, from);
          } else {
            gemv_copy<8>(at, from);
            gemv_copy<8>(at + 8, byte + 8 < half ? from + 8 : from);
          }
        }
      }
      constexpr int WORDS = (MX ? 2 : 4) + (WIDE ? 0 : 1);  // per row
      const int col0 = chunk * (MX ? 8 : 16);
#pragma unroll
      for (int i = 0; i < (kGemvRows * WORDS + 31) / 32; ++i) {
        const int item = i * 32 + lane, r = item / WORDS, w = item % WORDS;
        const int row = min(row0 + r, a.n - 1);
        const uint32_t at = to + kGemvRows * 128 + r * SPITCH + w * 4;
        if (a.swizzle) {
          const int col = min(col0 + w * 4, (cols - 1) & ~3);
          gemv_copy<4>(at, a.scales + scale_offset_swizzled(row, col, cols));
        } else if constexpr (WIDE) {
          gemv_copy<4>(at, a.scales + static_cast<int64_t>(row) * cols + min(col0 + w * 4, cols - 4));
        } else {
          // the aligned words around the row's scales; the weight's last word may be short
          const int64_t word = (static_cast<int64_t>(row) * cols + col0) / 4 * 4 + w * 4;
          const int64_t there = min(word, (scale_bytes - 1) / 4 * 4);
          const int bytes = static_cast<int>(min(static_cast<int64_t>(4), scale_bytes - there));
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(at), "l"(a.scales + there), "r"(bytes) : "memory");
        }
      }
      is_unit += STEP;
      is_tile += step_tiles;
      is_chunk += step_chunks;
      if (is_chunk >= c_count) {
        is_chunk -= c_count;
        ++is_tile;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (a.k > 0) {
#pragma unroll
    for (int i = 0; i < kGemvStages - 1; ++i) issue(i);
  }

  // ---- x: from the launch before, or converted here
  if (a.x_terms != nullptr) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int bytes = a.slice_chunks * 512, pieces = bytes / 16, terms = SPLIT ? 2 : 1;
    for (int i = tid; i < tokens * terms * pieces; i += kGemvThreads) {
      const int row = i / pieces, piece = i % pieces, mt = row / terms, term = row % terms;
      const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(smem + (term * tokens + mt) * pitch + piece * 16));
      gemv_copy<16>(at, a.x_terms + ((static_cast<int64_t>(slice) * a.m + m0 + mt) * terms + term) * bytes + piece * 16);
    }
    asm volatile("cp.async.commit_group;\n cp.async.wait_group 0;" ::: "memory");
    if (tid < tokens) unit[tid] = __ldg(a.x_units + static_cast<int64_t>(slice) * a.m + m0 + tid);
  } else {
    const int k_lo = c_first * kGemvCodes, count = c_count * (kGemvCodes / 8);
    uint32_t* tops = reinterpret_cast<uint32_t*>(unit);
    if (tid < COLS) tops[tid] = 0;
    __syncthreads();
    for (int mt = 0; mt < tokens; ++mt) {
      uint32_t top = 0;
#pragma unroll 4
      for (int i = tid; i < count; i += kGemvThreads) top = gemv_top8<T>(a, m0 + mt, k_lo + i * 8, top);
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0 && top != 0) atomicMax(tops + mt, top);
    }
    __syncthreads();
    for (int mt = 0; mt < tokens; ++mt) {
      const float up = gemv_up(tops[mt]);
#pragma unroll 4
      for (int i = tid; i < count; i += kGemvThreads)
        gemv_convert8<T>(a, m0 + mt, k_lo + i * 8, up, i, smem + mt * pitch, smem + (tokens + mt) * pitch);
    }
    __syncthreads();
    if (tid < tokens) unit[tid] = 1.0f / gemv_up(tops[tid]);
  }
  __syncthreads();

  const int lo_at = tokens * pitch;
  // where a lane reads column g of group j; `step`: 256 bytes per 128 codes, or none in the zeros. With
  // NVFP4 blocks apart the lane's first block and its second have a column each.
  constexpr int SIDES = GROUPED && !MX ? 2 : 1;
  int x_at[NT][SIDES], x_step[NT][SIDES];  // bytes from smem
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int side = 0; side < SIDES; ++side) {
      // columns past the tokens repeat the last one; nobody reads them
      const int token = !GROUPED ? j * 8 + g : MX ? 2 * j + (g & 1) : j;
      const bool here = !GROUPED || (MX ? t == g >> 1 : g == 2 * t + side);
      x_at[j][side] = here ? min(token, tokens - 1) * pitch + t * 16 : tokens * pitch * (SPLIT ? 2 : 1);
      x_step[j][side] = here ? 256 : 0;
    }
  }

  // two 16-row tiles: [tile][group][rows g, g + 8 x columns 2 t, 2 t + 1]
  using Sums = float[2][NT][4];
  Sums acc;
  auto clear = [&](Sums& c) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int j = 0; j < NT; ++j) c[q][j][0] = c[q][j][1] = c[q][j][2] = c[q][j][3] = 0.0f;
    }
  };
  clear(acc);

  // 128 codes of both tiles: w[tile][row half], in GROUPED as they are, else scaled by the f16 pairs
  // f[tile][row half][first, second 16 codes]
  auto products = [&](const uint4 (&w)[2][2], int half_chunk, const uint32_t (&f)[2][2][2], Sums& c) {
    auto scaled = [&](uint32_t v, uint32_t m) { return GROUPED ? v : mul_f16x2(v, m); };
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // 8 codes of each row: two MMAs
      uint4 b[NT], l[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int side = SIDES == 2 ? i >> 1 : 0;
        const int at = x_at[j][side] + half_chunk * x_step[j][side] + i * 64;
        b[j] = *reinterpret_cast<const uint4*>(smem + at);
        if constexpr (SPLIT) l[j] = *reinterpret_cast<const uint4*>(smem + (x_step[j][side] ? at + lo_at : at));
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t w0 = i == 0 ? w[q][0].x : i == 1 ? w[q][0].y : i == 2 ? w[q][0].z : w[q][0].w;
        const uint32_t w1 = i == 0 ? w[q][1].x : i == 1 ? w[q][1].y : i == 2 ? w[q][1].z : w[q][1].w;
        const uint32_t f0 = f[q][0][i >> 1], f1 = f[q][1][i >> 1];
        const uint32_t a00 = scaled(e2m1_f16<0>(w0), f0), a01 = scaled(e2m1_f16<1>(w0), f0);
        const uint32_t a02 = scaled(e2m1_f16<2>(w0), f0), a03 = scaled(e2m1_f16<3>(w0), f0);
        const uint32_t a10 = scaled(e2m1_f16<0>(w1), f1), a11 = scaled(e2m1_f16<1>(w1), f1);
        const uint32_t a12 = scaled(e2m1_f16<2>(w1), f1), a13 = scaled(e2m1_f16<3>(w1), f1);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma_m16n8k16(c[q][j], a00, a10, a01, a11, b[j].x, b[j].y);
          mma_m16n8k16(c[q][j], a02, a12, a03, a13, b[j].z, b[j].w);
          if constexpr (SPLIT) {
            mma_m16n8k16(c[q][j], a00, a10, a01, a11, l[j].x, l[j].y);
            mma_m16n8k16(c[q][j], a02, a12, a03, a13, l[j].z, l[j].w);
          }
        }
      }
    }
  };
  // acc += c, rows times u[tile][row half]
  auto add_scaled = [&](const Sums& c, const float (&u)[2][2]) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[q][j][e] = fmaf(c[q][j][e], u[q][e >> 1], acc[q][j][e]);
      }
    }
  };
  // s[tile][row half]: the lane's two e4m3 bytes, or its e8m0
  auto consume = [&](const uint4 (&w)[2][2], const uint32_t (&s)[2][2], int half_chunk) {
    if constexpr (GROUPED) {
      const uint32_t none[2][2][2] = {};
      Sums c;
      clear(c);
      products(w, half_chunk, none, c);
      if constexpr (MX) {  // columns 2 t and 2 t + 1: block t, two tokens
        float u[2][2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          u[q][0] = e8m0_value(static_cast<uint8_t>(s[q][0]));
          u[q][1] = e8m0_value(static_cast<uint8_t>(s[q][1]));
        }
        add_scaled(c, u);
      } else {  // columns 2 t and 2 t + 1: the lane's two blocks
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const __half2_raw p = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(s[q][h]), __NV_E4M3);
            const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&p));
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              acc[q][j][2 * h] = fmaf(c[q][j][2 * h], u.x, acc[q][j][2 * h]);
              acc[q][j][2 * h + 1] = fmaf(c[q][j][2 * h + 1], u.y, acc[q][j][2 * h + 1]);
            }
          }
        }
      }
    } else if constexpr (!MX) {
      uint32_t f[2][2][2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const __half2_raw p = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(s[q][h]), __NV_E4M3);
          const uint32_t v = *reinterpret_cast<const uint32_t*>(&p);
          f[q][h][0] = __byte_perm(v, v, 0x1010);
          f[q][h][1] = __byte_perm(v, v, 0x3232);
        }
      }
      if constexpr (SPLIT) {  // an MMA cuts its sum to 24 bits: fp32 results get a rounded addition per 128 codes
        Sums c;
        clear(c);
        products(w, half_chunk, f, c);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[q][j][e] += c[q][j][e];
          }
        }
      } else {
        products(w, half_chunk, f, acc);
      }
    } else {
      auto pow2 = [](int d) -> uint32_t {  // 2^d as an f16 pair, d in -24 .. 15
        const uint32_t h = d >= -14 ? static_cast<uint32_t>(d + 15) << 10 : 1u << (d + 24);
        return h | (h << 16);
      };
      uint32_t f[2][2][2];
      float u[2][2];
      bool ok = true;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int e = s[q][h], r = __shfl_sync(0xffffffffu, e, lane & 28), d = e - r;
          const bool near = d >= -20 && d <= 13;
          // the scale of 32 zeros does not count
          ok = ok && e != 255 && (near || (w[q][h].x | w[q][h].y | w[q][h].z | w[q][h].w) == 0);
          f[q][h][0] = f[q][h][1] = near ? pow2(d) : 0u;
          u[q][h] = e8m0_value(static_cast<uint8_t>(r));
        }
      }
      if (__all_sync(0xffffffffu, ok)) {
        Sums c;
        clear(c);
        products(w, half_chunk, f, c);
        add_scaled(c, u);
      } else {
        for (int x = 0; x < 4; ++x) {  // lane x's blocks of every row
          Sums c;
          clear(c);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              f[q][h][0] = f[q][h][1] = t == x ? 0x3C003C00u : 0u;
              u[q][h] = e8m0_value(static_cast<uint8_t>(__shfl_sync(0xffffffffu, s[q][h], (lane & 28) | x)));
            }
          }
          products(w, half_chunk, f, c);
          add_scaled(c, u);
        }
      }
    }
  };

  // one output of a tile: the final value, or one of its two partial sums
  auto put = [&](int tile, int r, int mt, float y, int part) {
    const int64_t row = static_cast<int64_t>(tile) * kGemvRows + r;
    if (row >= a.n || mt >= tokens) return;
    // one rounding: in fp32 the product of the two factors, or of y and one of them, may leave the normal range
    // where the result does not
    y = static_cast<float>(static_cast<double>(y) * unit[mt] * __ldg(a.ts + (a.ts_per_row ? row : 0)));
    if (part < 0 && a.slices == 1) {
      if (a.bias != nullptr) y += load_any(a.bias, a.bias_dtype, row);
      store_any<T>(a.out, (m0 + mt) * a.ldo + row, y);
    } else {
      a.partial[((static_cast<int64_t>(max(part, 0)) * a.slices + slice) * a.m + m0 + mt) * a.n + row] = y;
    }
  };
  int tile = u_lo / c_count, chunk = u_lo % c_count, begun = chunk;
  // this warp's sums of a tile; `ends`: its last chunk is among them
  auto leave = [&](bool ends) {
    const bool whole = !TURNS && begun == 0 && ends;
    float* at = TURNS ? sums + ((tile - tile_lo) * kGemvWarps + warp) * kGemvRows * COLS : sums_of(warp, begun != 0);
    if constexpr (!TURNS) __syncwarp();  // the ring's last reads
    auto one = [&](int r, int mt, float y) {
      if (whole) put(tile, r, mt, y, -1);
      else at[r * COLS + mt] = y;
    };
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int r = q * 16 + g;
        if constexpr (GROUPED) {
          // the blocks' sums meet: over the quad, and with NVFP4 over a lane's two blocks
          float v[4] = {acc[q][j][0], acc[q][j][1], acc[q][j][2], acc[q][j][3]};
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
              one(r, 2 * j, v[0]);
              one(r, 2 * j + 1, v[1]);
              one(r + 8, 2 * j, v[2]);
              one(r + 8, 2 * j + 1, v[3]);
            } else {
              one(r, j, v[0]);
              one(r + 8, j, v[2]);
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) one(r + 8 * (e >> 1), j * 8 + 2 * t + (e & 1), acc[q][j][e]);
        }
      }
    }
    if (!TURNS && !whole && lane == 0) seg_tile[2 * warp + (begun == 0)] = 2 * tile + ends;
    begun = 0;
    clear(acc);
  };

  int stage = 0;
  for (int u = u_lo; u < u_hi; u += STEP) {
    if (a.k > 0) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kGemvStages - 2) : "memory");
      __syncwarp();
      issue(stage == 0 ? kGemvStages - 1 : stage - 1);  // the stage that was consumed before this one
      const uint8_t* from = smem_all + (warp * kGemvStages + stage) * STAGE;
      const uint8_t* sc = from + kGemvRows * 128;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {  // 128 codes; once in the code, which short streams fetch cold
        uint4 w[2][2];
        uint32_t s[2][2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = q * 16 + i * 8 + g;
            w[q][i] = *reinterpret_cast<const uint4*>(from + r * 128 + (((h * 4 + t) ^ ((g & 1) << 2)) << 4));
            int off = r * SPITCH + h * (MX ? 4 : 8) + t * (MX ? 1 : 2);
            if constexpr (WIDE) {
              s[q][i] = MX ? sc[off] : *reinterpret_cast<const uint16_t*>(sc + off);
            } else {
              if (!a.swizzle) {  // the row's scales begin within the first word
                const int row = min(tile * kGemvRows + r, a.n - 1);
                off += static_cast<int>((static_cast<int64_t>(row) * cols + (c_first + chunk) * (MX ? 8 : 16)) & 3);
              }
              s[q][i] = sc[off] | (MX ? 0u : static_cast<uint32_t>(sc[off + 1]) << 8);
            }
          }
        }
        if constexpr (!WIDE) {
          // past K there may be any byte: no scale
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = (c_first + chunk) * kGemvCodes + h * 128 + t * 32;
            if (k >= a.k) s[i >> 1][i & 1] = 0;
            else if (!MX && k + 16 >= a.k) s[i >> 1][i & 1] &= 0xFFu;
          }
        }
        consume(w, s, chunk * 2 + h);
      }
    }
    const int next_chunk = chunk + step_chunks, next_tile = tile + step_tiles + (next_chunk >= c_count);
    if (next_tile != tile || u + STEP >= u_hi) leave(chunk == c_count - 1);
    tile = next_tile;
    chunk = next_chunk >= c_count ? next_chunk - c_count : next_chunk;
    stage = stage == kGemvStages - 1 ? 0 : stage + 1;
  }
  __syncthreads();
  if constexpr (TURNS) {
    for (int i = tid; i < spans * kGemvRows * COLS; i += kGemvThreads) {
      const int s = i / (kGemvRows * COLS), cell = i % (kGemvRows * COLS), first = (tile_lo + s) * c_count;
      const float* at = sums + s * kGemvWarps * kGemvRows * COLS + cell;
      float y = at[0];
#pragma unroll
      for (int w = 1; w < kGemvWarps; ++w) y += at[w * kGemvRows * COLS];
      // begun in the block before: its second part; ended in the next one: its first
      put(tile_lo + s, cell / COLS, cell % COLS, y, first < b_lo ? 1 : first + c_count > b_hi ? 0 : -1);
    }
  } else {
    // the tiles that warps share: from where they begin in this block (a warp's unfinished one, or the
    // one that began before the block), through the following warps' first sums
    for (int i = tid; i < (kGemvWarps + 1) * kGemvRows * COLS; i += kGemvThreads) {
      const int head = i / (kGemvRows * COLS), cell = i % (kGemvRows * COLS);
      const int seg = head == 0 ? 0 : (head - 1) * 2 + 1, first = seg_tile[seg];
      if (first < 0) continue;
      float y = sums_of(seg >> 1, head == 0)[cell];
      int end = first & 1;
      for (int w = (seg >> 1) + 1; w < kGemvWarps && seg_tile[2 * w] >= 0 && seg_tile[2 * w] >> 1 == first >> 1; ++w) {
        y += sums_of(w, true)[cell];
        end = seg_tile[2 * w] & 1;
      }
      put(first >> 1, cell / COLS, cell % COLS, y, head == 0 ? 1 : end ? -1 : 0);
    }
  }
}

// The tiles that two blocks share and the slices of K, added in order (units and the tensor scale
// are in the sums already). A warp has one tile and its lane i says whether two blocks share it in the i-th
// of 32 slices, before the sums are there: at 8 x 28672 x 8192 that took 3 us less of 48.6
// than a division by every lane for every slice.
template <int T>
__global__ void __launch_bounds__(256) gemv_join_kernel(GemvArgs a) {
  static_assert(kGemvRows == 32, "a row per lane");
  const int lane = threadIdx.x & 31, row = blockIdx.x * 256 + threadIdx.x, mt = blockIdx.y, tile = row / kGemvRows;
  auto shared_in = [&](int s) -> uint32_t {  // slices s .. s + 31
    bool shared = false;
    if (s + lane < a.slices && tile < a.tiles) {
      const int count = min(a.slice_chunks, a.chunks - (s + lane) * a.slice_chunks);
      const GemvCut cut(a.tiles * count, a.blocks);
      shared = cut.part_of(tile * count) != cut.part_of(tile * count + count - 1);
    }
    return __ballot_sync(0xffffffffu, shared);
  };
  uint32_t shared = shared_in(0);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (tile >= a.tiles || (a.slices == 1 && shared == 0)) return;  // the whole warp
  const int64_t step = static_cast<int64_t>(a.m) * a.n, second = a.slices * step;
  const float* at = a.partial + static_cast<int64_t>(mt) * a.n + min(row, a.n - 1);
  float y = 0.0f;
  for (int s = 0;;) {
#pragma unroll 4
    for (int i = 0; i < min(32, a.slices - s); ++i, at += step) {
      const bool both = shared >> i & 1;
      const float first = __ldg(at), rest = both ? __ldg(at + second) : 0.0f;
      y += first;
      if (both) y += rest;
    }
    if ((s += 32) >= a.slices) break;
    shared = shared_in(s);
  }
  if (row >= a.n) return;
  if (a.bias != nullptr) y += load_any(a.bias, a.bias_dtype, row);
  store_any<T>(a.out, mt * a.ldo + row, y);
}

}  // namespace kab
