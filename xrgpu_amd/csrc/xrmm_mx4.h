// Device helpers of the MX4 products (xrmm_mx4.hip, xrmm_mx4_gemm.hip).
#pragma once
#include "xrmm_lowbit.h"

namespace xrmm {

constexpr uint32_t MX_OOB = 0x80000000u;  // past every buffer bound here: loads return zero
constexpr int64_t MX_COUNTERS = 4096;     // bytes of arrival counters at the head of the workspace

template <int AT>
struct MxFrag { typedef bf16x8 t; };
template <>
struct MxFrag<LT_F16> { typedef f16x8 t; };

// Eight codes of a dword times the scale s, exact in bfloat16, and in binary16 where mx_f16_fits.
template <int AT>
__device__ __forceinline__ typename MxFrag<AT>::t mx_dq8(uint32_t w, float s) {
  if constexpr (AT == LT_F16) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  } else {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
}

// x = hi + lo with both terms bfloat16: the upper eight significant bits and the rest (a binary16 has
// eleven). An infinity or NaN stays in hi alone.
__device__ __forceinline__ void split_f16(f16x8 x, bf16x8& hi, bf16x8& lo) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = static_cast<float>(x[i]);
    const uint32_t b = __builtin_bit_cast(uint32_t, f);
    const float h = __builtin_bit_cast(float, b & 0xFFFF0000u);
    const bool fin = (b & 0x7F800000u) != 0x7F800000u;
    hi[i] = __builtin_bit_cast(bf16, static_cast<uint16_t>(b >> 16));
    lo[i] = static_cast<bf16>(fin ? f - h : 0.f);
  }
}

// Whether a block's values are exact in binary16: a scale in 2^-23 .. 2^13, or no value but zero.
__device__ __forceinline__ bool mx_f16_fits(uint32_t byte, u32x4 w) {
  return byte - 104u <= 36u || (byte != 255u && ((w[0] | w[1] | w[2] | w[3]) & 0x77777777u) == 0u);
}

__device__ __forceinline__ i32x8 mx_fp4(u32x4 x) {
  return i32x8{static_cast<int>(x[0]), static_cast<int>(x[1]), static_cast<int>(x[2]), static_cast<int>(x[3]), 0, 0, 0, 0};
}

// The tiled product (xrmm_mx4_gemm.hip): its plan for a geometry, and the launch.
struct MxPlan {
  int t;               // a tile has 64 t rows and columns (1, 2 or 4); 0: the geometry is left to k_mx4_rows
  uint32_t mt;         // row tiles
  uint32_t nb, ns;     // column tiles of 64 t columns, and of 192 behind them (t 4 only)
  uint32_t splits;     // of K
  uint32_t per;        // K steps of a split
  int64_t ws_bytes;
};
MxPlan mx4_gemm_plan(int64_t M, int64_t K, int64_t N, int a_type, bool have_ws);
hipError_t launch_mx4_gemm(const MxArgs& a, const MxPlan& p, hipStream_t st);

}  // namespace xrmm
