// Microscaled 4-bit values (MX4): blocks of 32 along K, E2M1 codes, one E8M0 scale a block.
//
//   quantise: E = floor(log2 max|x|), scale byte max(E + 127 - 2, 0), code = the E2M1 value
//             nearest x / 2^(byte - 127), ties to even, saturated at 6, sign kept
//   product:  Y[m, n] = sum_k A[m, k] e2m1(code[n, k]) 2^(byte[n, k / 32] - 127) (+ bias[n])
#include <type_traits>

#include "xrmm_mx4.h"

namespace xrmm {

int device_cus();

namespace {

// ---------------------------------------------------------------------------
// Quantisation. A lane holds eight consecutive values, so four lanes hold a block: the
// largest magnitude goes round the quad in two exchanges of the bit pattern (ordered like
// the magnitudes, with infinity and NaN above every finite value), and each lane writes
// its four bytes. VB: bytes per load (rows that are no multiple of 16 bytes start
// unaligned). The conversion instruction divides by the scale and rounds as above. Bytes bound it: 14336 x 4090 float32 in
// 61 us (4.4 TB/s), 4096 x 4096 bfloat16 in 10.

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
// Product, up to 16 rows (and any number past the tiled product's K): a workgroup takes 16 rows and columns, its waves every WV-th group of four blocks along K. Nothing goes through
// LDS until the waves' sums meet, so no wave waits for another, and K is not split over workgroups, whose exchange costs
// three trips past the caches (8 to 10 us). The loop is short on purpose: the kernel lives for a few
// microseconds, and code that is run once or twice is fetched slower than it runs (unrolled by four with loads ahead: 21 us at
// 1 x 4096 x 14336 for 15).
//
// The weights are the MFMA's first operand. Lane (c, g) = (lane % 16, lane / 16) loads block g of column c, 16
// consecutive bytes. MX4 activations are loaded alike, and one v_mfma_scale_f32_16x16x128 takes both with
// their scales. 16-bit activations: eight values of a lane in the order of the weights' loads would lie 64 bytes from the
// next lane's (28.5 us at 16 x 4096 x 14336 for 25.4, 23.2 at 16 x 14336 x 4096 for 22.2). So the
// weights are transposed among the four lane groups (v_permlane swaps): lane (c, g) then
// holds dword g of each block, and the activations' loads are runs of 64 bytes. Each byte of codes becomes two 16-bit values
// times its block's scale in one conversion; v_mfma_f32_16x16x32 takes a block. What bounds it past four rows is that
// every 16 columns load all activations anew: 128 KB from L2 beside 34 KB of weights at 16 x 4096, of which a CU gets about 40 GB/s. A wave
// that keeps its share of the activations over several column tiles, as k_gemv_sk does, would load them once.
//
// A bfloat16 holds every E2M1 value times 2^(byte - 127) exactly. A binary16 does for scales in
// [2^-23, 2^13]; a workgroup that met another scale sums everything again, with weights in bfloat16 and the
// activations as the sum of two bfloat16 terms (8 and 3 bits: exact), so every scale is right.

// (a, b) -> a's lower half and b's lower half, a's upper half and b's upper half; and the same of odd and even rows of 16 lanes
__device__ __forceinline__ void mx_swap32(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
__device__ __forceinline__ void mx_swap16(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}

template <int AT, int WV, bool AL>
__global__ __launch_bounds__(64 * WV, 4) void k_mx4_rows(MxArgs a, uint32_t col_tiles) {
  constexpr bool MX = AT < 0;
  typedef typename MxFrag<AT>::t frag;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n0 = static_cast<int64_t>(blockIdx.x % col_tiles) * 16, m0 = static_cast<int64_t>(blockIdx.x / col_tiles) * 16;
  const uint32_t kb = static_cast<uint32_t>(a.kb), K = static_cast<uint32_t>(a.K);
  const uint32_t rowsB = static_cast<uint32_t>(a.N - n0 < 16 ? a.N - n0 : 16), rowsA = static_cast<uint32_t>(a.M - m0 < 16 ? a.M - m0 : 16);
  const uint32_t rowA = MX ? kb * MX_BLOB : K * 2u;
  const uint8_t* pA = static_cast<const uint8_t*>(a.A) + m0 * rowA;
  const uint32_t mis = AL ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(pA)) & 3u;
  const rsrc_t rA = mk_rsrc(pA - mis, (rowsA * rowA + mis + 3u) & ~3u);
  const rsrc_t rB = mk_rsrc(a.B + n0 * a.kb * MX_BLOB, rowsB * kb * MX_BLOB);
  const rsrc_t rS = mk_rsrc(a.S + n0 * a.kb, rowsB * kb);
  const rsrc_t rT = mk_rsrc(MX ? a.As + m0 * a.kb : a.S, MX ? rowsA * kb : 0u);
  const bool okb = static_cast<uint32_t>(c) < rowsB;
  const uint32_t cb = c * kb;

  // Eight values of K from k on of the lane's row
  auto piece = [&](uint32_t k) {
    const uint32_t at = c * rowA + k * 2u + mis;
    const bool ok = static_cast<uint32_t>(c) < rowsA && k < K;
    if constexpr (AL) {  // K a multiple of 8: a piece is whole or absent
      return bld16(rA, ok ? at : MX_OOB, 0);
    } else {
      u32x4 v = bld16(rA, ok ? at & ~3u : MX_OOB, 0);
      const uint32_t x = bld_u32(rA, ok ? (at & ~3u) + 16u : MX_OOB, 0);
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {
        const uint32_t ke = k + 2 * e, y = __builtin_amdgcn_alignbyte(e < 3 ? v[e + 1] : x, v[e], at & 3u);
        v[e] = ke + 1 < K ? y : ke < K ? y & 0xFFFFu : 0u;
      }
      return v;
    }
  };

  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  bool misfit = false;
  u32x4 w;
  uint32_t s;
  auto load = [&](uint32_t b) {
    const bool ok = okb && b < kb;
    w = bld16_nt(rB, ok ? (cb + b) * MX_BLOB : MX_OOB, 0);
    s = bld_u8(rS, ok ? cb + b : MX_OOB, 0);
  };
  load(wave * 4 + g);
#pragma unroll 1
  for (uint32_t b0 = wave * 4; b0 < kb; b0 += WV * 4) {
    const uint32_t nb = b0 + WV * 4 + g;
    if constexpr (MX) {
      const bool have = static_cast<uint32_t>(c) < rowsA && b0 + g < kb;
      const u32x4 x = bld16(rA, have ? (cb + b0 + g) * MX_BLOB : MX_OOB, 0), wc = w;
      const uint32_t t = bld_u8(rT, have ? cb + b0 + g : MX_OOB, 0), sc = s;
      load(nb);
      acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_fp4(wc), mx_fp4(x), acc, 4, 4, 0, static_cast<int>(sc), 0, static_cast<int>(t));
    } else {
      u32x4 x[4];
#pragma unroll
      for (uint32_t d = 0; d < 4; ++d) x[d] = piece((b0 + d) * MX_BLOCK + 8 * g);
      uint32_t y[4] = {w[0], w[1], w[2], w[3]}, s1 = s << (8 * g);
      if (AT == LT_F16) misfit |= !mx_f16_fits(s, w);
      load(nb);
      mx_swap32(y[0], y[2]);
      mx_swap32(y[1], y[3]);
      mx_swap16(y[0], y[1]);
      mx_swap16(y[2], y[3]);
      uint32_t s2 = s1;
      mx_swap32(s1, s2);
      s1 |= s2;
      s2 = s1;
      mx_swap16(s1, s2);
      s1 |= s2;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const frag wf = mx_dq8<AT>(y[d], e8m0((s1 >> (8 * d)) & 255u));
        if constexpr (AT == LT_F16) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf, __builtin_bit_cast(f16x8, x[d]), acc, 0, 0, 0);
        else acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, __builtin_bit_cast(bf16x8, x[d]), acc, 0, 0, 0);
      }
    }
  }
  if constexpr (AT == LT_F16) {
    if (__syncthreads_or(misfit)) {
      acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (uint32_t q = wave; q < kb; q += WV) {  // one block at a time
        const float sf = e8m0(bld_u8(rS, okb ? cb + q : MX_OOB, 0));
        const bf16x8 wf = mx_dq8<LT_BF16>(bld_u32(rB, okb ? (cb + q) * MX_BLOB + 4 * g : MX_OOB, 0), sf);
        bf16x8 hi, lo;
        split_f16(__builtin_bit_cast(f16x8, piece(q * MX_BLOCK + 8 * g)), hi, lo);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, hi, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, lo, acc, 0, 0, 0);
      }
    }
  }

  // The waves' sums meet in LDS and are added in wave order.
  __shared__ f32x4 red[WV][64];
  red[wave][lane] = acc;
  __syncthreads();
  const int64_t m = m0 + c, n = n0 + g * 4;
  if (wave != 0 || m >= a.M) return;
  f32x4 v = red[0][lane];
#pragma unroll
  for (int w2 = 1; w2 < WV; ++w2) v += red[w2][lane];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < a.N) st_lt(a.Y, m * a.N + n + e, v[e] + (a.bias ? ld_lt(a.bias, n + e, a.out) : 0.f), a.out);
}

// ---------------------------------------------------------------------------
// Product, one or two rows of 16-bit activations. A wave holds 64 blocks of K, one a lane, of every row in
// registers and walks over columns: a column's 64 blocks are one load of 1 KB. A lane sums its block
// from the codes as they are (exact in 16 bits whatever the scale; two products and a float32 sum in one v_dot2) and
// then applies the scale to the sum's exponent, so no scale is out of range. For bfloat16 activations the codes count 2^-8 of their
// value meanwhile: 32 products of 6 and the largest bfloat16 would pass float32. The lanes' sums meet by DPP, the chunks of K in LDS,
// in order. Nothing but the loop over columns repeats, and it is short: the kernel lives for a few microseconds, and
// unrolled code is fetched slower than it runs. 1 x 4096 x 14336: 8.9 us, 31 MB (k_gemv_dot reads 6 % more bytes at
// this size in 7 to 7.7: two or three workgroups a CU and two columns in flight a wave leave the rest).

template <int AT>
__device__ __forceinline__ float mx_dot2(uint32_t a, uint32_t b, float c) {
  if constexpr (AT == LT_F16) return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, a), __builtin_bit_cast(f16x2, b), c, false);
  else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a), __builtin_bit_cast(bf16x2, b), c, false);
}

__device__ __forceinline__ float mx_wave_total(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, false));
  };
  v += dpp(v, std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  v += dpp(v, std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  v += dpp(v, std::integral_constant<int, 0x141>{});  // row_half_mirror
  v += dpp(v, std::integral_constant<int, 0x140>{});  // row_mirror
  auto at = [&](int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l)); };
  return (at(0) + at(16)) + (at(32) + at(48));
}

constexpr int MXD_MAX_WAVES = 16, MXD_MAX_COLS = 64;

template <int AT, int R, bool AL>
__global__ __launch_bounds__(64 * MXD_MAX_WAVES) void k_mx4_dot(MxArgs a, uint32_t ncols, uint32_t chunk_waves, uint32_t col_waves) {
  constexpr int P = 2;  // columns whose loads are in flight together
  constexpr int UP = AT == LT_F16 ? 0 : 8;
  __shared__ float part[MXD_MAX_WAVES][MXD_MAX_COLS][R];
  const int tid = threadIdx.x, lane = tid & 63;
  const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(tid >> 6));
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * ncols;
  const uint32_t kb = static_cast<uint32_t>(a.kb), K = static_cast<uint32_t>(a.K), M = static_cast<uint32_t>(a.M);
  const uint32_t cols = a.N - n0 < ncols ? static_cast<uint32_t>(a.N - n0) : ncols;
  const uint32_t mis = AL ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(a.A)) & 3u;
  const rsrc_t rA = mk_rsrc(static_cast<const uint8_t*>(a.A) - mis, (M * K * 2u + mis + 3u) & ~3u);
  const rsrc_t rB = mk_rsrc(a.B + n0 * a.kb * MX_BLOB, cols * kb * MX_BLOB);
  const rsrc_t rS = mk_rsrc(a.S + n0 * a.kb, cols * kb);
  const uint32_t cw = wave % chunk_waves, gw = wave / chunk_waves;
  for (uint32_t c = gw; c < cols; c += col_waves)
    if (lane < R) part[wave][c][lane] = 0.f;
#pragma unroll 1
  for (uint32_t chunk = cw; chunk * 64 < kb; chunk += chunk_waves) {
    const uint32_t b = chunk * 64 + lane, k = b * MX_BLOCK;
    const bool in = b < kb;
    u32x4 x[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t off = (r * K + k) * 2u + mis;
#pragma unroll
      for (uint32_t d = 0; d < 4; ++d)  // pieces past K are absent; unaligned, the last value may lie in the next piece's first dword
        x[r][d] = bld16(rA, in && static_cast<uint32_t>(r) < M && k + 8 * d < (AL ? K : K + 1) ? (off & ~3u) + 16 * d : MX_OOB, 0);
      if constexpr (!AL) {
        const uint32_t last = bld_u32(rA, in && static_cast<uint32_t>(r) < M ? (off & ~3u) + 64u : MX_OOB, 0), sh = off & 3u;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t next = e < 3 ? x[r][d][e + 1] : d < 3 ? x[r][d < 3 ? d + 1 : 0][0] : last;
            const uint32_t ke = k + 8 * d + 2 * e, y = __builtin_amdgcn_alignbyte(next, x[r][d][e], sh);
            x[r][d][e] = ke + 1 < K ? y : ke < K ? y & 0xFFFFu : 0u;
          }
      }
    }
#pragma unroll 1
    for (uint32_t c = gw; c < cols; c += P * col_waves) {
      u32x4 w[P];
      uint32_t s[P];
#pragma unroll
      for (uint32_t p = 0; p < P; ++p) {
        const uint32_t cp = c + p * col_waves;
        const bool ok = in && cp < cols;
        w[p] = bld16_nt(rB, ok ? (cp * kb + b) * MX_BLOB : MX_OOB, 0);
        s[p] = bld_u8(rS, ok ? cp * kb + b : MX_OOB, 0);
      }
#pragma unroll
      for (uint32_t p = 0; p < P; ++p) {
        const uint32_t cp = c + p * col_waves;
        float sum[R];
#pragma unroll
        for (int r = 0; r < R; ++r) sum[r] = 0.f;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const u32x4 wv = __builtin_bit_cast(u32x4, mx_dq8<AT>(w[p][d], 1.f / (1 << UP)));
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int r = 0; r < R; ++r) sum[r] = mx_dot2<AT>(wv[e], x[r][d][e], sum[r]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float scaled = s[p] == 255u ? __builtin_nanf("") : __builtin_ldexpf(sum[r], static_cast<int>(s[p]) - 127 + UP);
          const float t = mx_wave_total(in ? scaled : 0.f);
          if (lane == r && cp < cols) part[wave][cp][r] += t;
        }
      }
    }
  }
  __syncthreads();
  for (uint32_t x = tid; x < cols * M; x += blockDim.x) {
    const uint32_t c = x % cols, r = x / cols, w0 = (c % col_waves) * chunk_waves;
    float v = part[w0][c][r];
    for (uint32_t w = 1; w < chunk_waves; ++w) v += part[w0 + w][c][r];
    const int64_t n = n0 + c;
    st_lt(a.Y, r * a.N + n, v + (a.bias ? ld_lt(a.bias, n, a.out) : 0.f), a.out);
  }
}

template <int AT, int R>
hipError_t dot_r(const MxArgs& a, hipStream_t st) {
  const int64_t chunks = (a.kb + 63) / 64, cus = device_cus() > 0 ? device_cus() : 256;
  // a wave for each chunk of K, and as many times that as fit eight waves
  const uint32_t cw = static_cast<uint32_t>(chunks < MXD_MAX_WAVES ? chunks : MXD_MAX_WAVES), gw = cw < 8 ? 8 / cw : 1;
  // columns of a workgroup: about 20 waves a CU (4 to 64 columns at 1 x 4096 x 14336: 9.1 us at 8, 8.9 at 16, 9.4 at 32, 11.7 at
  // 64; at 1 x 14336 x 4096: 12.3 us at 2, 10.6 at 4, 10.0 at 8, 11.8 at 16)
  int64_t cols = (a.N * cw * gw + 20 * cus - 1) / (20 * cus);
  cols = (cols + gw - 1) / gw * gw;
  cols = cols < MXD_MAX_COLS ? cols : MXD_MAX_COLS;
  const dim3 grid(static_cast<uint32_t>((a.N + cols - 1) / cols)), block(64 * cw * gw);
  const bool al = a.K % 8 == 0 && (reinterpret_cast<uintptr_t>(a.A) & 15u) == 0;
  if (al) k_mx4_dot<AT, R, true><<<grid, block, 0, st>>>(a, static_cast<uint32_t>(cols), cw, gw);
  else k_mx4_dot<AT, R, false><<<grid, block, 0, st>>>(a, static_cast<uint32_t>(cols), cw, gw);
  return hipGetLastError();
}

template <int AT>
hipError_t dot_for(const MxArgs& a, hipStream_t st) {
  switch (a.M) {
    case 1: return dot_r<AT, 1>(a, st);
    default: return dot_r<AT, 2>(a, st);
  }
}

constexpr int MXR_WAVES = 8;  // sixteen: 26.2 for 25.4 us at 16 x 4096 x 14336

template <int AT>
hipError_t rows_for(const MxArgs& a, hipStream_t st) {
  const int64_t ct = (a.N + 15) / 16, n = ct * ((a.M + 15) / 16);
  if (n > 0x7FFFFFFF) return hipErrorInvalidValue;
  const dim3 grid(static_cast<uint32_t>(n)), block(64 * MXR_WAVES);
  const bool al = a.K % 8 == 0 && (reinterpret_cast<uintptr_t>(a.A) & 15u) == 0;
  if (AT < 0 || al) k_mx4_rows<AT, MXR_WAVES, true><<<grid, block, 0, st>>>(a, static_cast<uint32_t>(ct));
  else if constexpr (AT >= 0) k_mx4_rows<AT, MXR_WAVES, false><<<grid, block, 0, st>>>(a, static_cast<uint32_t>(ct));
  return hipGetLastError();
}

// Rows that k_mx4_dot takes: at 4096 x 14336 one row takes 8.9 us there and 15 in k_mx4_rows, two 11.8, four 19 and 18
// (a wave's activations are loaded anew for every few columns, and outgrow the weights).
bool use_dot(int64_t M, int a_type) { return M <= 2 && a_type >= 0; }

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

int64_t mx4_workspace_bytes(int64_t M, int64_t K, int64_t N, int a_type) {
  return mx4_gemm_plan(M, K, N, a_type, true).ws_bytes;
}

const char* mx4_kernel_name(const MxArgs& a) {
  switch (mx4_gemm_plan(a.M, a.K, a.N, a.a_type, true).t) {
    case 4: return "mx4_gemm_256";
    case 2: return "mx4_gemm_128";
    case 1: return "mx4_gemm_64";
  }
  return use_dot(a.M, a.a_type) ? "mx4_dot" : "mx4_rows";
}

hipError_t launch_matmul_mx4(const MxArgs& a, hipStream_t st) {
  if (a.M == 0) return hipSuccess;
  MxPlan p = mx4_gemm_plan(a.M, a.K, a.N, a.a_type, a.ws != nullptr);
  if (p.ws_bytes > a.ws_bytes) p = mx4_gemm_plan(a.M, a.K, a.N, a.a_type, false);
  if (p.t != 0) return launch_mx4_gemm(a, p, st);
  if (use_dot(a.M, a.a_type)) return a.a_type == LT_F16 ? dot_for<LT_F16>(a, st) : dot_for<LT_BF16>(a, st);
  switch (a.a_type) {
    case LT_F16: return rows_for<LT_F16>(a, st);
    case LT_BF16: return rows_for<LT_BF16>(a, st);
    default: return rows_for<-1>(a, st);
  }
}

}  // namespace xrmm
