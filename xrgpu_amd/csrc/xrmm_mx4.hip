// Microscaled 4-bit values (MX4): blocks of 32 along K, E2M1 codes, one E8M0 scale a block.
//
//   quantise: E = floor(log2 max|x|), scale byte max(E + 127 - 2, 0), code = the E2M1 value
//             nearest x / 2^(byte - 127), ties to even, saturated at 6, sign kept
//   product:  Y[m, n] = sum_k A[m, k] e2m1(code[n, k]) 2^(byte[n, k / 32] - 127) (+ bias[n])
#include "xrmm_mx4.h"

namespace xrmm {
namespace {

// ---------------------------------------------------------------------------
// Quantisation. A lane holds eight consecutive values, so four lanes hold a block: the
// largest magnitude goes round the quad in two exchanges of the bit pattern (ordered like
// the magnitudes, with infinity and NaN above every finite value), and each lane writes
// its four bytes. VB: bytes per load (rows that are no multiple of 16 bytes start
// unaligned). The conversion instruction divides by the scale and rounds as above.

template <typename T, int VB>
__global__ __launch_bounds__(256) void k_mx4_quant(MxQuantArgs a) {
  constexpr int PER = VB / static_cast<int>(sizeof(T));  // values per load
  typedef T vec __attribute__((ext_vector_type(PER)));
  const int64_t lane = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t blk = lane >> 2;  // block of the whole tensor
  const int q = static_cast<int>(lane & 3);
  const bool have = blk < a.rows * a.kb;
  const int64_t row = have ? blk / a.kb : 0, b = have ? blk - row * a.kb : 0;
  const int64_t k0 = b * MX_BLOCK + q * 8;
  const T* src = static_cast<const T*>(a.x) + row * a.K + k0;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; i += PER) {
    if (have && k0 + i < a.K) {  // K is a multiple of PER: a load is whole or absent
      const vec x = *reinterpret_cast<const vec*>(src + i);
#pragma unroll
      for (int j = 0; j < PER; ++j) v[i + j] = static_cast<float>(x[j]);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) v[i + j] = 0.f;
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t m = __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu;
    top = top > m ? top : m;
  }
#pragma unroll
  for (int x = 1; x <= 2; x <<= 1) {
    const uint32_t o = static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), x, 64));
    top = top > o ? top : o;
  }
  if (!have) return;
  const uint32_t e = top >> 23;  // floor(log2) + 127; 255: an infinity or NaN is among them
  const uint32_t byte = e == 255u ? 255u : e > 2u ? e - 2u : 0u;
  uint32_t code = 0;
  if (e != 255u) {
    const float s = e8m0(byte);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[0], v[1], s, 0);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[2], v[3], s, 1);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[4], v[5], s, 2);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[6], v[7], s, 3);
  }
  *reinterpret_cast<uint32_t*>(a.codes + blk * MX_BLOB + q * 4) = code;
  if (q == 0) a.scales[blk] = static_cast<uint8_t>(byte);
}

template <typename T>
hipError_t quantize_for(const MxQuantArgs& a, hipStream_t st) {
  const int64_t lanes = a.rows * a.kb * 4;
  const dim3 grid(static_cast<uint32_t>((lanes + 255) / 256));
  const uintptr_t step = reinterpret_cast<uintptr_t>(a.x) | static_cast<uintptr_t>(a.K * sizeof(T));
  constexpr int S = static_cast<int>(sizeof(T));
  if (step % 16 == 0) k_mx4_quant<T, 16><<<grid, 256, 0, st>>>(a);
  else if (step % 8 == 0) k_mx4_quant<T, 8><<<grid, 256, 0, st>>>(a);
  else k_mx4_quant<T, S><<<grid, 256, 0, st>>>(a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Product, few rows. The weights are the MFMA's first operand: lane (c, g) = (lane % 16,
// lane / 16) loads blocks 8 it + 2 g + {0, 1} of column c, 32 consecutive bytes, straight
// into the fragment (the order of k inside an MFMA is free as long as both operands agree),
// and the second operand's lane (c, g) holds the same blocks of row c. float16 / bfloat16
// activations: each byte pair of codes becomes two 16-bit values with its block's scale in one
// conversion instruction, v_mfma_f32_16x16x32 four times a block. MX4 activations: one
// v_mfma_scale_f32_16x16x128 for four blocks, scales applied by the instruction.
//
// A bfloat16 holds every E2M1 value times 2^(byte - 127) exactly. A binary16 does for scales in
// [2^-23, 2^13]; a wave that meets another scale takes that block's weights in bfloat16 and the
// activations as the sum of two bfloat16 terms (8 and 3 bits: exact), so every scale is right.

constexpr int MXR_WAVES = 8;

template <int AT, int NT, int CT, bool AL>
__global__ __launch_bounds__(64 * MXR_WAVES) void k_mx4_rows(MxArgs a, uint32_t col_tiles) {
  constexpr bool MX = AT < 0;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n0 = static_cast<int64_t>(blockIdx.x % col_tiles) * (16 * CT);
  const int64_t m0 = static_cast<int64_t>(blockIdx.x / col_tiles) * (16 * NT);
  const uint32_t kb = static_cast<uint32_t>(a.kb), K = static_cast<uint32_t>(a.K);
  const uint32_t rowsB = static_cast<uint32_t>(a.N - n0 < 16 * CT ? a.N - n0 : 16 * CT);
  const uint32_t rowsA = static_cast<uint32_t>(a.M - m0 < 16 * NT ? a.M - m0 : 16 * NT);
  const rsrc_t rB = mk_rsrc(a.B + n0 * a.kb * MX_BLOB, rowsB * kb * MX_BLOB);
  const rsrc_t rS = mk_rsrc(a.S + n0 * a.kb, rowsB * kb);
  const rsrc_t rA = MX ? mk_rsrc(static_cast<const uint8_t*>(a.A) + m0 * a.kb * MX_BLOB, rowsA * kb * MX_BLOB)
                       : mk_rsrc(static_cast<const uint16_t*>(a.A) + m0 * a.K, rowsA * K * 2u);
  const rsrc_t rAs = mk_rsrc(MX ? a.As + m0 * a.kb : a.S, MX ? rowsA * kb : 0u);

  f32x4 acc[CT][NT];
#pragma unroll
  for (int i = 0; i < CT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const uint32_t its = (kb + 7) / 8;
  for (uint32_t it = static_cast<uint32_t>(wave); it < its; it += MXR_WAVES) {
    u32x4 w[CT][2];
    uint32_t s[CT][2];
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t b = it * 8 + g * 2 + u, r = i * 16 + c;
        const bool ok = b < kb && r < rowsB;
        w[i][u] = bld16_nt(rB, ok ? (r * kb + b) * MX_BLOB : MX_OOB, 0);
        s[i][u] = bld_u8(rS, ok ? r * kb + b : MX_OOB, 0);
      }
    if constexpr (MX) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t b = it * 8 + g * 2 + u, r = j * 16 + c;
          const bool ok = b < kb && r < rowsA;
          const u32x4 x = bld16(rA, ok ? (r * kb + b) * MX_BLOB : MX_OOB, 0);
          const int xs = static_cast<int>(bld_u8(rAs, ok ? r * kb + b : MX_OOB, 0));
#pragma unroll
          for (int i = 0; i < CT; ++i) {
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_fp4(w[i][u]), mx_fp4(x), acc[i][j], 4, 4, 0, static_cast<int>(s[i][u]), 0, xs);
          }
        }
    } else {
      typedef typename MxFrag<AT>::t frag;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        frag x[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t k = (it * 8 + g * 2 + u) * MX_BLOCK + q * 8, r = j * 16 + c;
            if constexpr (AL) {  // K a multiple of 8: a piece is whole or absent
              x[j][q] = __builtin_bit_cast(frag, bld16(rA, (k < K && r < rowsA) ? (r * K + k) * 2u : MX_OOB, 0));
            } else {
              u32x4 v;
#pragma unroll
              for (uint32_t d = 0; d < 4; ++d) {
                const uint32_t k2 = k + 2 * d;
                const uint32_t lo = bld_u16(rA, (k2 < K && r < rowsA) ? (r * K + k2) * 2u : MX_OOB, 0);
                const uint32_t hi = bld_u16(rA, (k2 + 1 < K && r < rowsA) ? (r * K + k2 + 1) * 2u : MX_OOB, 0);
                v[d] = lo | (hi << 16);
              }
              x[j][q] = __builtin_bit_cast(frag, v);
            }
          }
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          const float sf = e8m0(s[i][u]);
          bool wide = false;
          if constexpr (AT == LT_F16) {
            wide = __any(!mx_f16_fits(s[i][u], w[i][u]));
          }
          if (wide) {
            if constexpr (AT == LT_F16) {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const bf16x8 wf = mx_dq8<LT_BF16>(w[i][u][q], sf);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                  bf16x8 hi, lo;
                  split_f16(x[j][q], hi, lo);
                  acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, hi, acc[i][j], 0, 0, 0);
                  acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, lo, acc[i][j], 0, 0, 0);
                }
              }
            }
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const frag wf = mx_dq8<AT>(w[i][u][q], sf);
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                if constexpr (AT == LT_F16) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf, x[j][q], acc[i][j], 0, 0, 0);
                else acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, x[j][q], acc[i][j], 0, 0, 0);
              }
            }
          }
        }
      }
    }
  }

  // The waves' sums meet in LDS and are added in wave order.
  __shared__ f32x4 red[MXR_WAVES][CT * NT][64];
#pragma unroll
  for (int i = 0; i < CT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) red[wave][i * NT + j][lane] = acc[i][j];
  __syncthreads();
  for (int p = tid; p < CT * NT * 64; p += 64 * MXR_WAVES) {
    const int t = p >> 6, l = p & 63;
    f32x4 v = red[0][t][l];
#pragma unroll
    for (int w = 1; w < MXR_WAVES; ++w) v += red[w][t][l];
    const int64_t m = m0 + (t % NT) * 16 + (l & 15), n = n0 + (t / NT) * 16 + (l >> 4) * 4;
    if (m >= a.M) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.N) st_lt(a.Y, m * a.N + n + e, v[e] + (a.bias ? ld_lt(a.bias, n + e, a.out) : 0.f), a.out);
  }
}

template <int AT, int NT, int CT>
hipError_t rows_for(const MxArgs& a, hipStream_t st) {
  const int64_t ct = (a.N + 16 * CT - 1) / (16 * CT), mt = (a.M + 16 * NT - 1) / (16 * NT);
  if (ct * mt > 0x7FFFFFFF) return hipErrorInvalidValue;
  const dim3 grid(static_cast<uint32_t>(ct * mt));
  const bool al = a.K % 8 == 0 && (reinterpret_cast<uintptr_t>(a.A) & 15u) == 0;
  if (AT < 0 || al) k_mx4_rows<AT, NT, CT, true><<<grid, 64 * MXR_WAVES, 0, st>>>(a, static_cast<uint32_t>(ct));
  else k_mx4_rows<AT, NT, CT, false><<<grid, 64 * MXR_WAVES, 0, st>>>(a, static_cast<uint32_t>(ct));
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mx4_quantize(const MxQuantArgs& a, hipStream_t st) {
  if (a.rows == 0) return hipSuccess;
  if (a.rows * a.kb > (int64_t(1) << 36)) return hipErrorInvalidValue;  // launch limit: 2^31 workgroups of 64 blocks
  switch (a.dtype) {
    case LT_F32: return quantize_for<float>(a, st);
    case LT_F16: return quantize_for<f16>(a, st);
    default: return quantize_for<bf16>(a, st);
  }
}

int64_t mx4_workspace_bytes(int64_t M, int64_t K, int64_t N, int a_type) { return mx4_gemm_plan(M, K, N, a_type, true).ws_bytes; }

const char* mx4_kernel_name(const MxArgs& a) {
  switch (mx4_gemm_plan(a.M, a.K, a.N, a.a_type, true).t) {
    case 4: return "mx4_gemm_256";
    case 2: return "mx4_gemm_128";
    case 1: return "mx4_gemm_64";
  }
  return "mx4_rows";
}

hipError_t launch_matmul_mx4(const MxArgs& a, hipStream_t st) {
  if (a.M == 0) return hipSuccess;
  MxPlan p = mx4_gemm_plan(a.M, a.K, a.N, a.a_type, a.ws != nullptr);
  if (p.ws_bytes > a.ws_bytes) p = mx4_gemm_plan(a.M, a.K, a.N, a.a_type, false);
  if (p.t != 0) return launch_mx4_gemm(a, p, st);
  switch (a.a_type) {
    case LT_F16: return rows_for<LT_F16, 1, 1>(a, st);
    case LT_BF16: return rows_for<LT_BF16, 1, 1>(a, st);
    default: return rows_for<-1, 1, 1>(a, st);
  }
}

}  // namespace xrmm
