// extern "C" entry points of the weight-only FP4 linear (gemv_fp4.cuh).
#include <algorithm>

#include "kab_host.h"

#include "gemv_fp4.cuh"

namespace kab {
namespace {

int gemv_check(int64_t m, int64_t n, int64_t k, int fmt, int dtype) {
  KAB_REQUIRE(fmt == KAB_NVFP4 || fmt == KAB_MXFP4, "unknown FP4 format %d", fmt);
  KAB_REQUIRE(valid_dtype(dtype), "unknown dtype %d", dtype);
  KAB_REQUIRE(m >= 0 && n >= 0 && k >= 0, "negative shape");
  KAB_REQUIRE(k % (fmt == KAB_NVFP4 ? 16 : 32) == 0, "K = %lld is not a multiple of the block", (long long)k);
  KAB_REQUIRE((n + 31) / 32 * ((k + 255) / 256 + 1) < (int64_t(1) << 31), "problem too large");
  KAB_REQUIRE(m < 65536 && n < (int64_t(1) << 30) && k < (int64_t(1) << 30), "problem too large");
  return KAB_OK;
}

// How a shape is cut: slices of K so that a slice of x fits in shared memory, and blocks per slice,
// two per SM where their shared memory allows.
constexpr int kSmemOne = 226 * 1024, kSmemTwo = 113 * 1024;
struct GemvPlan {
  bool grouped, turns, join, terms;
  int nt, columns, tokens, chunks, slice_chunks, slices, tiles, blocks, smem;
  size_t partial, x_terms, x_units;  // workspace bytes
  size_t bytes() const { return partial + x_terms + x_units; }
};
size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Blocks apart (GROUPED) while its MMAs (8 per 128 codes and group) stay below the stream's time: one
// or two tokens of NVFP4, up to four of MXFP4 (half of that in fp32, whose x has two terms). Blocks apart
// against scaled codes at 28672 x 8192 (4096 x 4096): two tokens of NVFP4 36.7 and 39.4 us (7.3 and 8.3),
// three 62.9 and 39.9 (10.9 and 9.0); four of MXFP4 40.0 and 49.0 (8.4 and 9.7), five 70.1 and 52.3 (12.1 and
// 9.8).
GemvPlan gemv_plan(int64_t m, int64_t n, int64_t k, int fmt, int dtype) {
  GemvPlan p{};
  const bool mx = fmt == KAB_MXFP4, split = dtype == KAB_F32;
  const int most = (mx ? 4 : 2) / (split ? 2 : 1);
  p.grouped = m <= most;
  p.nt = p.grouped ? static_cast<int>(mx ? (m + 1) / 2 : m) : m <= 8 ? 1 : m <= 16 ? 2 : 4;
  p.columns = gemv_columns(mx, p.nt, p.grouped);
  p.tokens = static_cast<int>(std::min<int64_t>(m, p.columns));
  p.chunks = static_cast<int>(std::max<int64_t>(1, (k + kGemvCodes - 1) / kGemvCodes));
  p.tiles = static_cast<int>((n + kGemvRows - 1) / kGemvRows);
  const int64_t per_chunk = static_cast<int64_t>(p.tokens) * 512 * (split ? 2 : 1);
  // A block's warps in turns where the tiles of its part, whose sums stay in shared memory, are few
  // enough in one wave of blocks; else a contiguous part per warp. Two blocks per SM with at least 4
  // chunks of x each (or all of it) where that fits, one for 16 columns and more (by registers).
  const int need = std::min(p.chunks, 4);
  for (p.turns = p.columns <= 8; ; p.turns = false) {
    const int spans = !p.turns ? 1 : p.columns <= 2 ? 8 : 4;
    const int fixed = gemv_smem(mx, 0, 0, p.columns, split, spans) + p.tokens * 64 * (split ? 2 : 1);
    const int room = p.columns <= 8 && fixed + need * per_chunk <= kSmemTwo ? kSmemTwo : kSmemOne;
    const int fit = static_cast<int>(std::max<int64_t>(1, (room - fixed) / per_chunk));
    const int want = (p.chunks + fit - 1) / fit;
    p.slice_chunks = (p.chunks + want - 1) / want;
    p.slices = (p.chunks + p.slice_chunks - 1) / p.slice_chunks;
    p.smem = gemv_smem(mx, p.tokens, p.slice_chunks, p.columns, split, spans);
    const int wave = std::max(1, (room == kSmemTwo ? 2 : 1) * sm_count() / p.slices);
    p.blocks = std::min(p.tiles, wave);
    if (!p.turns || p.tiles <= wave * (spans - 1)) break;
    if (p.columns <= 2) {  // more waves, as few as keep a block's part within its tiles
      p.blocks = std::min(p.tiles, (p.tiles + wave * (spans - 1) - 1) / (wave * (spans - 1)) * wave);
      break;
    }
  }
  p.join = p.slices > 1 || p.tiles % p.blocks != 0;  // else every block has whole tiles
  p.partial = p.join ? round256(static_cast<size_t>(2) * p.slices * m * n * 4) : 0;
  // x converted by a launch of its own where every block would have to convert more than one token
  p.terms = m > 1;
  p.x_terms = p.terms ? round256(static_cast<size_t>(p.slices) * m * p.slice_chunks * 512 * (split ? 2 : 1)) : 0;
  p.x_units = p.terms ? round256(static_cast<size_t>(p.slices) * m * 4) : 0;
  return p;
}

// Rows of x that share the launches of a call: all where their partial sums and terms fit in 256 MB, else as
// many groups of 32 as do (2048 x 28672 x 8192 would take 2.3 GB; the weight is read again for every 32 rows
// either way).
constexpr size_t kGemvMost = size_t(256) << 20;
int64_t gemv_rows(int64_t m, int64_t n, int64_t k, int fmt, int dtype) {
  if (m <= 32 || gemv_plan(m, n, k, fmt, dtype).bytes() <= kGemvMost) return m;
  return std::max<int64_t>(1, kGemvMost / gemv_plan(32, n, k, fmt, dtype).bytes()) * 32;
}
size_t gemv_bytes(int64_t m, int64_t n, int64_t k, int fmt, int dtype) {
  const int64_t rows = gemv_rows(m, n, k, fmt, dtype), rest = m % rows;
  const size_t most = gemv_plan(rows, n, k, fmt, dtype).bytes();
  return rest == 0 ? most : std::max(most, gemv_plan(rest, n, k, fmt, dtype).bytes());
}

// A launch that may be set up while the one before it runs (it waits by itself).
cudaError_t launch_after(void (*kern)(GemvArgs), dim3 grid, int threads, int smem, cudaStream_t s, const GemvArgs& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

template <int T, int MX, int NT, int WIDE, int GROUPED, int TURNS>
int launch_gemv(const GemvArgs& a, const GemvPlan& p, cudaStream_t s) {
  auto kern = gemv_fp4_kernel<T, MX, NT, WIDE, GROUPED, TURNS>;
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(KAB_ECUDA, "no current device");
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemOne) != cudaSuccess)
      return fail(KAB_ECUDA, "cannot configure the FP4 linear");
    configured[dev] = true;
  }
  const dim3 grid(p.blocks, p.slices, (a.m + p.columns - 1) / p.columns);
  if (p.terms) {
    gemv_x_kernel<T><<<dim3(p.slices, a.m), 256, 0, s>>>(a);
    if (int e = check_launch("kab_gemv_fp4 x")) return e;
    launch_after(kern, grid, kGemvThreads, p.smem, s, a);
  } else {
    kern<<<grid, kGemvThreads, p.smem, s>>>(a);
  }
  if (int e = check_launch("kab_gemv_fp4")) return e;
  if (!p.join) return KAB_OK;
  launch_after(gemv_join_kernel<T>, dim3((a.n + 255) / 256, a.m), 256, 0, s, a);
  return check_launch("kab_gemv_fp4 join");
}
template <int T, int MX, int NT, int GROUPED>
int launch_gemv(const GemvArgs& a, const GemvPlan& p, cudaStream_t s) {
  const bool wide = a.k % (MX ? 128 : 64) == 0 && aligned(a.codes, 16) && aligned(a.scales, 4);
  constexpr int columns = gemv_columns(MX, NT, GROUPED);
  if constexpr (columns <= 8) {
    if (p.turns) return wide ? launch_gemv<T, MX, NT, 1, GROUPED, 1>(a, p, s) : launch_gemv<T, MX, NT, 0, GROUPED, 1>(a, p, s);
  }
  if constexpr (columns > 2)
    return wide ? launch_gemv<T, MX, NT, 1, GROUPED, 0>(a, p, s) : launch_gemv<T, MX, NT, 0, GROUPED, 0>(a, p, s);
  return fail(KAB_EUNSUPPORTED, "no kernel for this plan");
}
template <int T, int MX>
int launch_gemv(const GemvArgs& a, const GemvPlan& p, cudaStream_t s) {
  if (p.grouped) {
    if (p.nt == 1) return launch_gemv<T, MX, 1, 1>(a, p, s);
    if constexpr (T != kF32) return launch_gemv<T, MX, 2, 1>(a, p, s);
    return fail(KAB_EUNSUPPORTED, "no kernel for this plan");
  }
  return p.nt == 1 ? launch_gemv<T, MX, 1, 0>(a, p, s) : p.nt == 2 ? launch_gemv<T, MX, 2, 0>(a, p, s)
                                                                   : launch_gemv<T, MX, 4, 0>(a, p, s);
}
template <int T>
int launch_gemv(const GemvArgs& a, const GemvPlan& p, int fmt, cudaStream_t s) {
  return fmt == KAB_MXFP4 ? launch_gemv<T, 1>(a, p, s) : launch_gemv<T, 0>(a, p, s);
}

}  // namespace
}  // namespace kab

using namespace kab;

extern "C" {

int kab_gemv_fp4_workspace(int64_t m, int64_t n, int64_t k, int fmt, int dtype, size_t* bytes) {
  if (int e = gemv_check(m, n, k, fmt, dtype)) return e;
  KAB_REQUIRE(bytes != nullptr, "null pointer");
  *bytes = m == 0 || n == 0 ? 0 : gemv_bytes(m, n, k, fmt, dtype);
  return KAB_OK;
}

int kab_gemv_fp4(const void* x, int dtype, int64_t ldx, const uint8_t* codes, const uint8_t* scales, int swizzle,
                 int fmt, const float* tensor_scale, int scale_per_row, int64_t m, int64_t n, int64_t k,
                 const void* bias, int bias_dtype, void* out, int64_t ldo, void* workspace, size_t workspace_bytes,
                 void* stream) {
  if (int e = gemv_check(m, n, k, fmt, dtype)) return e;
  if (m == 0 || n == 0) return KAB_OK;
  KAB_REQUIRE(out != nullptr && tensor_scale != nullptr && (k == 0 || (x && codes && scales)), "null pointer");
  KAB_REQUIRE(bias == nullptr || valid_dtype(bias_dtype), "unknown bias dtype %d", bias_dtype);
  KAB_REQUIRE(aligned(x, 16) && ldx % 8 == 0, "x must be 16-byte aligned, its row stride a multiple of 8");
  KAB_REQUIRE(aligned(codes, 8), "codes must be 8-byte aligned");
  KAB_REQUIRE(aligned(scales, 4), "scales must be 4-byte aligned");
  KAB_REQUIRE(ldo >= n && ldx >= k, "ldx %lld or ldo %lld is too short", (long long)ldx, (long long)ldo);
  const size_t need = gemv_bytes(m, n, k, fmt, dtype);
  KAB_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && aligned(workspace, 256)),
              "the workspace needs %zu bytes, 256-byte aligned (kab_gemv_fp4_workspace)", need);
  GemvArgs a{};
  a.ldx = ldx, a.codes = codes, a.scales = scales, a.swizzle = swizzle;
  a.ts = tensor_scale, a.ts_per_row = scale_per_row;
  a.n = static_cast<int>(n), a.k = static_cast<int>(k);
  a.bias = bias, a.bias_dtype = bias_dtype, a.ldo = ldo;
  const cudaStream_t s = as_stream(stream);
  const int64_t step = gemv_rows(m, n, k, fmt, dtype), size = dtype == KAB_F32 ? 4 : 2;
  for (int64_t m0 = 0; m0 < m; m0 += step) {
    const int64_t rows = std::min(step, m - m0);
    const GemvPlan p = gemv_plan(rows, n, k, fmt, dtype);
    a.x = static_cast<const uint8_t*>(x) + m0 * ldx * size;
    a.out = static_cast<uint8_t*>(out) + m0 * ldo * size;
    a.m = static_cast<int>(rows);
    a.chunks = p.chunks, a.slice_chunks = p.slice_chunks, a.slices = p.slices;
    a.tiles = p.tiles, a.blocks = p.blocks, a.partial = static_cast<float*>(workspace);
    a.x_terms = p.terms ? static_cast<uint8_t*>(workspace) + p.partial : nullptr;
    a.x_units = p.terms ? reinterpret_cast<float*>(a.x_terms + p.x_terms) : nullptr;
    const int e = dtype == KAB_BF16 ? launch_gemv<kBF16>(a, p, fmt, s)
                  : dtype == KAB_F16 ? launch_gemv<kF16>(a, p, fmt, s)
                                     : launch_gemv<kF32>(a, p, fmt, s);
    if (e != KAB_OK) return e;
  }
  return KAB_OK;
}

}  // extern "C"
