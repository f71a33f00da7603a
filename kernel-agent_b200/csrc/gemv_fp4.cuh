// Weight-only FP4 linear for a few tokens: out[m, n] = ts * sum_k x[m, k] * e2m1(c[n, k]) *
// s[n, k / block] (+ bias), the activations as they are.
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
  int64_t m, n, k;
  const void* bias;
  int bias_dtype;
  void* out;
  int64_t ldo;
};

// The two e2m1 values of a byte (low nibble first) as exact f16.
__device__ __forceinline__ uint32_t e2m1_pair(uint32_t byte) {
  uint32_t r;
  asm("{\n .reg .b8 b0, b1, b2, b3;\n mov.b32 {b0, b1, b2, b3}, %1;\n cvt.rn.f16x2.e2m1x2 %0, b0;\n}"
      : "=r"(r)
      : "r"(byte));
  return r;
}

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == KAB_F32) return static_cast<const float*>(p)[i];
  if (dtype == KAB_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// One warp per weight row and eight tokens, its lanes over the row's 8-code words.
template <int T, int MX>
__global__ void __launch_bounds__(256) gemv_fp4_kernel(GemvArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5), m0 = blockIdx.y * 8;
  if (n >= a.n) return;
  // each token in units of a power of two near its largest value, so that no product of a large
  // activation and a large block scale overflows before the tensor scale is applied
  float unit[8], per[8];
#pragma unroll
  for (int m = 0; m < 8; ++m) {
    uint32_t top = 0;
    if (m0 + m < a.m)
      for (int64_t w = lane; w < a.k / 8; w += 32) {
        float x[8];
        load8<T>(a.x, (m0 + m) * a.ldx + w * 8, x);
        top = abs_bits_max8(x, top);
      }
    const uint32_t e = min(max(__reduce_max_sync(0xffffffffu, top) >> 23, 1u), 253u);
    unit[m] = __uint_as_float(e << 23);
    per[m] = __uint_as_float((254u - e) << 23);
  }
  float acc[8] = {};
  const int64_t cols = a.k >> (MX ? 5 : 4);
  for (int64_t w = lane; w < a.k / 8; w += 32) {
    const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(a.codes + n * (a.k / 2)) + w);
    const int64_t col = w >> (MX ? 2 : 1);
    const uint8_t sb = __ldg(a.scales + (a.swizzle ? scale_offset_swizzled(n, col, cols) : n * cols + col));
    const float s = MX ? e8m0_value(sb) : e4m3_value_hw(sb);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t h = e2m1_pair((c >> (8 * i)) & 255u);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      v[2 * i] = f.x * s;
      v[2 * i + 1] = f.y * s;
    }
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      if (m0 + m < a.m) {
        float x[8];
        load8<T>(a.x, (m0 + m) * a.ldx + w * 8, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[m] = fmaf(x[i] * per[m], v[i], acc[m]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < 8; ++m) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], o);
    if (lane == 0 && m0 + m < a.m) {
      float y = acc[m] * (unit[m] * a.ts[a.ts_per_row ? n : 0]);
      if (a.bias != nullptr) y += load_any(a.bias, a.bias_dtype, n);
      if constexpr (T == kF32) static_cast<float*>(a.out)[(m0 + m) * a.ldo + n] = y;
      else if constexpr (T == kBF16) static_cast<__nv_bfloat16*>(a.out)[(m0 + m) * a.ldo + n] = __float2bfloat16_rn(y);
      else static_cast<__half*>(a.out)[(m0 + m) * a.ldo + n] = __float2half_rn(y);
    }
  }
}

}  // namespace kab
