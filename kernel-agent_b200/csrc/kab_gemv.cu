// extern "C" entry points of the weight-only FP4 linear (gemv_fp4.cuh).
#include "kab_host.h"

#include "gemv_fp4.cuh"

namespace kab {
namespace {

int gemv_check(int64_t m, int64_t n, int64_t k, int fmt, int dtype) {
  KAB_REQUIRE(fmt == KAB_NVFP4 || fmt == KAB_MXFP4, "unknown FP4 format %d", fmt);
  KAB_REQUIRE(valid_dtype(dtype), "unknown dtype %d", dtype);
  KAB_REQUIRE(m >= 0 && n >= 0 && k >= 0, "negative shape");
  KAB_REQUIRE(k % (fmt == KAB_NVFP4 ? 16 : 32) == 0, "K = %lld is not a multiple of the block", (long long)k);
  KAB_REQUIRE(m < (int64_t(1) << 18) && n < (int64_t(1) << 31) && k < (int64_t(1) << 31), "problem too large");
  return KAB_OK;
}

template <int T>
void launch_gemv(const GemvArgs& a, int fmt, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((a.n + 7) / 8), static_cast<unsigned>((a.m + 7) / 8));
  if (fmt == KAB_MXFP4) gemv_fp4_kernel<T, 1><<<grid, 256, 0, s>>>(a);
  else gemv_fp4_kernel<T, 0><<<grid, 256, 0, s>>>(a);
}

}  // namespace
}  // namespace kab

using namespace kab;

extern "C" {

int kab_gemv_fp4_workspace(int64_t m, int64_t n, int64_t k, int fmt, int dtype, size_t* bytes,
                           size_t* zero_bytes) {
  if (int e = gemv_check(m, n, k, fmt, dtype)) return e;
  KAB_REQUIRE(bytes != nullptr && zero_bytes != nullptr, "null pointer");
  *bytes = 0;
  *zero_bytes = 0;
  return KAB_OK;
}

int kab_gemv_fp4(const void* x, int dtype, int64_t ldx, const uint8_t* codes, const uint8_t* scales, int swizzle,
                 int fmt, const float* tensor_scale, int scale_per_row, int64_t m, int64_t n, int64_t k,
                 const void* bias, int bias_dtype, void* out, int64_t ldo, void* workspace, size_t workspace_bytes,
                 void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  if (int e = gemv_check(m, n, k, fmt, dtype)) return e;
  if (m == 0 || n == 0) return KAB_OK;
  KAB_REQUIRE(out != nullptr && tensor_scale != nullptr && (k == 0 || (x && codes && scales)), "null pointer");
  KAB_REQUIRE(bias == nullptr || valid_dtype(bias_dtype), "unknown bias dtype %d", bias_dtype);
  KAB_REQUIRE(aligned(x, 16) && ldx % 8 == 0, "x must be 16-byte aligned, its row stride a multiple of 8");
  KAB_REQUIRE(aligned(codes, 8), "codes must be 8-byte aligned");
  KAB_REQUIRE(ldo >= n && ldx >= k, "ldx %lld or ldo %lld is too short", (long long)ldx, (long long)ldo);
  GemvArgs a{x, ldx, codes, scales, swizzle, tensor_scale, scale_per_row, m, n, k, bias, bias_dtype, out, ldo};
  const cudaStream_t s = as_stream(stream);
  if (dtype == KAB_BF16) launch_gemv<kBF16>(a, fmt, s);
  else if (dtype == KAB_F16) launch_gemv<kF16>(a, fmt, s);
  else launch_gemv<kF32>(a, fmt, s);
  return check_launch("kab_gemv_fp4");
}

}  // extern "C"
