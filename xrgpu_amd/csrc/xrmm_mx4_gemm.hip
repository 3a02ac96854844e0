// MX4 product, many rows: Y = A W^T (+ bias) on tiles of 32 WM TM rows by 64 TN columns.
//
// WM x 2 waves, each with TM x TN accumulators of 32 x 32. A K step stages 128 bytes of every row: 64 values of 16-bit
// activations and of the weights, converted on the way into LDS, or 256 codes where both operands are
// MX4 (v_mfma_scale takes them and their scales as they are). Either way a row is eight pieces of 16 bytes; piece p of row r lies
// in slot p ^ (r % 8), which spreads a fragment's rows over all banks without padding.
//
// Two stages. While step s computes, the pieces of step s + 1 go from registers to the other
// stage, a quarter beside each K slice. Their loads left two or four steps before (mxg_ahead). The barrier stands before the last slice's MFMAs: the next stage's first fragments are
// read behind them.
//
// 256-tiles of two MX4 operands need no conversion, and their pieces go from memory to LDS without registers: once all
// waves have read the last fragments of a stage, step s + 2 is fetched into it. With pieces in registers the tile
// spilled (4096 x 4096 x 14336 with the activations' quantisation 182 us, 174 on the same box, 174 to 187 on others; 4096 x 14336 x 4096
// alone 153 -> 142). Four waves of 128 x 128 read a third less LDS, but one wave a SIMD
// covers less: 190 us. What bounds it is the pieces' way from L2: a step's 64 KB take 2.2 us of a CU (7.6 TB/s of all), the step 1.8 without
// them; half steps fetched three ahead arrive no sooner (182 us: twice the requests).
//
// The weights are the MFMAs' first operand: a lane then holds four consecutive columns of one row.
#include <atomic>

#include "xrmm_mx4.h"

namespace xrmm {

int device_cus();

namespace {

// K steps that loads run ahead. Tiles of 64 and 128 with 16-bit activations take four: one of the few workgroups that K's
// split leaves a CU waits on its loads (512 x 4096 x 4096 on 128-tiles 57 -> 48 us, split in two 43 -> 39; 128 rows on 64-tiles
// 34 -> 30). An MX4 step computes four times as long for the same bytes, and the registers of 256-tiles hold no more: two
// (MX4 512 x 4096 x 4096 on 128-tiles 22.9 us, with four 25.7).
constexpr int mxg_ahead(bool mx, int t) { return mx || t > 2 ? 2 : 4; }

template <int AT, int WM, int TM, int TN>
struct MxTile {
  static constexpr bool MX = AT < 0;
  static constexpr int T = 128 * WM, RA = 32 * WM * TM, RB = 64 * TN;
  static constexpr int CODES = (RA + RB) * 128;                    // bytes of a stage's rows
  static constexpr int STAGE = CODES + (MX ? (RA + RB + T - 1) / T * T * 8 : 0);  // and of its scales, one row a thread
  static constexpr int STRIP = 32 * (32 * TN * 4 + 16);            // of a wave's rows on their way out
  static constexpr int LDS = 2 * STAGE > 2 * WM * STRIP ? 2 * STAGE : 2 * WM * STRIP;
  static constexpr int BLOCKS = MX ? 8 : 2;                        // blocks of 32 along K in a step
};

struct MxGrid {
  uint32_t mt, nb, ns, nbig, splits, per;
};

// 16 bytes a lane from memory to LDS, at `to` (the same for the wave) + 16 times the lane.
__device__ __forceinline__ void lds16(rsrc_t r, unsigned char* to, uint32_t voff, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)to, 16, static_cast<int>(voff), static_cast<int>(soff), 0, 0);
}

template <int AT, int WM, int TM, int TN, bool AL>
__device__ __forceinline__ void mx_tile(const MxArgs& a, uint32_t row, int64_t n0, const MxGrid& g, uint32_t tile, uint32_t split) {
  typedef MxTile<AT, WM, TM, TN> Ti;
  constexpr bool MX = Ti::MX;
  constexpr int T = Ti::T, RA = Ti::RA, RB = Ti::RB, NA = RA * 8 / T, NB = MX ? RB * 8 / T : (2 * RB + T - 1) / T;
  constexpr int D = mxg_ahead(MX, TN);
  constexpr bool DMA = MX && TN > 2;   // pieces go from memory to LDS by themselves
  constexpr bool ONE = !MX && TN > 2;  // one set of pieces: see part
  constexpr int NS = MX ? (RA + RB + T - 1) / T : NB, TR = T / 8;  // TR: rows that the threads cover with one piece each
  typedef typename MxFrag<AT>::t half8;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int64_t m0 = static_cast<int64_t>(row) * RA;
  const uint32_t kb = static_cast<uint32_t>(a.kb), K = static_cast<uint32_t>(a.K);
  const uint32_t rowsA = static_cast<uint32_t>(a.M - m0 < RA ? a.M - m0 : RA);
  const uint32_t rowsB = static_cast<uint32_t>(a.N - n0 < RB ? a.N - n0 : RB);
  const uint32_t s0 = split * g.per, s1 = s0 + g.per;  // a multiple of D steps
  // the split's end along K, in blocks and values: what lies past it loads as zeros
  const uint32_t kbe = s1 * Ti::BLOCKS < kb ? s1 * Ti::BLOCKS : kb, Ke = kbe * MX_BLOCK < K ? kbe * MX_BLOCK : K;

  const uint32_t rowA = MX ? kb * MX_BLOB : K * 2u, rowB = kb * MX_BLOB;
  // an unaligned A: its resource starts at the dword that holds its first byte
  const uint8_t* pA = static_cast<const uint8_t*>(a.A) + m0 * rowA;
  const uint32_t misA = AL ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(pA)) & 3u;
  const rsrc_t rA = mk_rsrc(pA - misA, (rowsA * rowA + misA + 3u) & ~3u);
  const rsrc_t rB = mk_rsrc(a.B + n0 * rowB, rowsB * rowB);
  // scales: a wave's threads hold rows of one operand each; MX4 scales at any alignment start at a dword
  rsrc_t rS[NS];
  uint32_t sbase[NS];  // byte offset of the thread's row (MX) or block (16-bit activations)
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    if constexpr (MX) {
      const bool isA = wave * 64 + T * i < RA;
      const uint8_t* ps = isA ? a.As + m0 * a.kb : a.S + n0 * a.kb;
      const uint32_t mis = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ps)) & 3u, rows = isA ? rowsA : rowsB;
      rS[i] = mk_rsrc(ps - mis, (rows * kb + mis + 3u) & ~3u);
      const uint32_t r = static_cast<uint32_t>(tid + T * i) - (isA ? 0u : RA);
      sbase[i] = r < rows ? r * kb + mis : MX_OOB;
    } else {
      const uint32_t c = static_cast<uint32_t>(tid + T * i), r = c >> 1;
      rS[i] = mk_rsrc(a.S + n0 * a.kb, rowsB * kb);
      sbase[i] = r < rowsB && r < RB ? r * kb + (c & 1u) : MX_OOB;
    }
  }

  // ---- staging registers
  struct Set {
    u32x4 b[DMA ? 1 : NB];  // 16-bit activations: blocks of weights; MX4: pieces
    uint32_t s[NS][MX ? 3 : 1];
    u32x4 a[ONE || DMA ? 1 : NA];
    uint32_t x[ONE || AL ? 1 : NA];
  };
  u32x4 oa[NA];
  uint32_t ox[AL ? 1 : NA];
  bool misfit = false;

  // A thread's place in each row it loads, past every bound where there is none; a step adds a scalar offset, and one
  // comparison a step says whether the thread's piece lies before the split's end.
  const uint32_t srow = static_cast<uint32_t>(tid >> 3), spiece = static_cast<uint32_t>((tid & 7) ^ (srow & 7u));
  uint32_t va[NA], vb[NB];
#pragma unroll
  for (int i = 0; i < NA; ++i) {
    const uint32_t r = srow + TR * i;
    va[i] = r < rowsA ? ((r * rowA + misA) & ~3u) + spiece * 16u : MX_OOB;
  }
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    if constexpr (MX) {
      const uint32_t r = srow + TR * i;
      vb[i] = r < rowsB ? r * rowB + spiece * MX_BLOB : MX_OOB;
    } else {
      const uint32_t c = static_cast<uint32_t>(tid + T * i), r = c >> 1;
      vb[i] = r < rowsB && r < RB ? r * rowB + (c & 1u) * MX_BLOB : MX_OOB;
    }
  }
  auto inside = [&](uint32_t s) { return MX ? s * 8u + spiece < kbe : s * 64u + spiece * 8u < Ke; };
  auto load_a = [&](int i, uint32_t s, bool in, u32x4* ra, uint32_t* rx) {
    const uint32_t v = in ? va[i] : MX_OOB;
    ra[i] = bld16(rA, v, s * 128u);
    if constexpr (!MX && !AL) rx[i] = bld_u32(rA, v + 16u, s * 128u);
  };
  auto load_b = [&](int i, uint32_t s, bool in, u32x4* rb) { rb[i] = bld16(rB, in ? vb[i] : MX_OOB, s * 128u); };  // MX4 operands
  auto load_set = [&](Set& w, uint32_t s) {
    if constexpr (!ONE && !DMA) {
      const bool in = inside(s);
#pragma unroll
      for (int i = 0; i < NA; ++i) load_a(i, s, in, w.a, w.x);
      if constexpr (MX)
#pragma unroll
        for (int i = 0; i < NB; ++i) load_b(i, s, in, w.b);
    }
    if constexpr (MX) {
      // eight scale bytes a row: three dwords
      const uint32_t b = s * 8u < kbe ? s * 8u : (kbe - 1u) & ~7u;  // past the end the last step's, which part() drops
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int d = 0; d < 3; ++d) w.s[i][MX ? d : 0] = bld_u32(rS[i], (sbase[i] & ~3u) + 4u * d, b);
    } else {
      const bool in = s * 2u + static_cast<uint32_t>(tid & 1) < kbe;
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        w.b[DMA ? 0 : i] = bld16(rB, in ? vb[i] : MX_OOB, s * 32u);
        w.s[i][0] = bld_u8(rS[i], in ? sbase[i] : MX_OOB, s * 2u);
      }
    }
  };
  // DMA: step s to LDS stage `st`. What lies past a row's or the split's end may stay as it was there: codes are finite whatever their
  // bits, rows past the end leave no output, and blocks past it have the scale 2^-127 on both sides.
  auto fetch = [&](uint32_t s, int st) {
    const bool in = inside(s);
    unsigned char* base = smem + st * Ti::STAGE + wave * 1024;  // lane l writes 16 bytes at 16 l
#pragma unroll
    for (int i = 0; i < NA; ++i) lds16(rA, base + TR * i * 128, in ? va[i] : MX_OOB, s * 128u);
    if constexpr (MX)
#pragma unroll
      for (int i = 0; i < NB; ++i) lds16(rB, base + (RA + TR * i) * 128, in ? vb[i] : MX_OOB, s * 128u);
  };
  // Quarter d of the pieces of step s to LDS stage `st`; with one set of pieces, each piece's load for step s + 1
  auto part = [&](int d, uint32_t s, int st, const Set& w) {
    unsigned char* base = smem + st * Ti::STAGE;
    const bool in = inside(s + 1);
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      if (DMA || i * 4 / NA != d) continue;
      u32x4 v = ONE ? oa[i] : w.a[ONE || DMA ? 0 : i];
      if constexpr (!MX && !AL) {
        const uint32_t k = s * 64u + spiece * 8u, r = srow + TR * i;
        const uint32_t sh = (r * rowA + misA) & 3u;  // a step's pieces start at multiples of 16 bytes of a row
        const u32x4 x = v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_alignbyte(e < 3 ? x[e + 1] : ONE ? ox[AL ? 0 : i] : w.x[ONE || AL ? 0 : i], x[e], sh);
        if (k + 8u > K) {  // the row's last piece: what lies past it is the next row's
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t ke = k + 2u * e;
            v[e] = ke + 1u < K ? v[e] : ke < K ? v[e] & 0xFFFFu : 0u;
          }
        }
      }
      *reinterpret_cast<u32x4*>(base + (srow + TR * i) * 128 + (tid & 7) * 16) = v;
      if (ONE) load_a(i, s + 1, in, oa, ox);
    }
    if constexpr (MX) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        if (DMA || i * 4 / NB != d) continue;
        *reinterpret_cast<u32x4*>(base + (RA + srow + TR * i) * 128 + (tid & 7) * 16) = w.b[DMA ? 0 : i];
      }
      if (d == (DMA ? 3 : 0)) {
        const uint32_t b0 = s * 8u, n = b0 < kbe ? kbe - b0 : 0u;  // scales of blocks past K are 2^-127 on both sides: products of 0
        const uint32_t k0 = n >= 4u ? ~0u : (1u << (8u * n)) - 1u, k1 = n >= 8u ? ~0u : n <= 4u ? 0u : (1u << (8u * (n - 4u))) - 1u;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          const int r = tid + T * i;
          const uint32_t sh = sbase[i] & 3u;
          u32x2 v;
          v[0] = __builtin_amdgcn_alignbyte(w.s[i][MX ? 1 : 0], w.s[i][0], sh) & k0;
          v[1] = __builtin_amdgcn_alignbyte(w.s[i][MX ? 2 : 0], w.s[i][MX ? 1 : 0], sh) & k1;
          *reinterpret_cast<u32x2*>(base + Ti::CODES + r * 8) = v;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int c = tid + T * i, r = c >> 1;
        const u32x4 wb = w.b[DMA ? 0 : i];
        if (AT == LT_F16 && d == 0) misfit |= !mx_f16_fits(w.s[i][0], wb);
        if (NB * T == 2 * RB || c < 2 * RB)
          *reinterpret_cast<half8*>(base + (RA + r) * 128 + ((((c & 1) * 4 + d) ^ (r & 7)) * 16)) = mx_dq8<AT>(wb[d], e8m0(w.s[i][0]));
      }
    }
  };

  f32x16 acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.f;

  // ---- fragments: lane (r, h) = (lane % 32, lane / 32) reads piece 2 kk + h of row r

  u32x4 fa[2][TM], fb[2][TN];
  u32x2 ta[MX ? TM : 1], tb[MX ? TN : 1];  // scales of the step, moved so that byte 2 kk is this half's
  const int fr = lane & 31, fh = lane >> 5;
  auto read = [&](int st, int kk) {
    const int buf = kk & 1;
    const unsigned char* base = smem + st * Ti::STAGE + (((2 * kk + fh) ^ (fr & 7)) * 16) + fr * 128;
#pragma unroll
    for (int i = 0; i < TM; ++i) fa[buf][i] = *reinterpret_cast<const u32x4*>(base + (wm * TM + i) * 4096);
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[buf][j] = *reinterpret_cast<const u32x4*>(base + RA * 128 + (wn * TN + j) * 4096);
  };
  auto read_scales = [&](int st) {
    if constexpr (MX) {
      const unsigned char* base = smem + st * Ti::STAGE + Ti::CODES + fr * 8;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        ta[i] = *reinterpret_cast<const u32x2*>(base + (wm * TM + i) * 256);
        ta[i] >>= fh * 8;
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        tb[j] = *reinterpret_cast<const u32x2*>(base + RA * 8 + (wn * TN + j) * 256);
        tb[j] >>= fh * 8;
      }
    }
  };
  auto mfmas = [&](auto kkc) {
    constexpr int kk = decltype(kkc)::value, buf = kk & 1;
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if constexpr (MX)
          acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_fp4(fb[buf][j]), mx_fp4(fa[buf][i]), acc[j][i], 4, 4, (kk & 1) * 2,
                                                                       static_cast<int>(tb[j][kk >> 1]), (kk & 1) * 2, static_cast<int>(ta[i][kk >> 1]));
        else if constexpr (AT == LT_F16)
          acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, fb[buf][j]), __builtin_bit_cast(f16x8, fa[buf][i]), acc[j][i], 0, 0, 0);
        else
          acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fb[buf][j]), __builtin_bit_cast(bf16x8, fa[buf][i]), acc[j][i], 0, 0, 0);
      }
  };
  auto step = [&](uint32_t s, int st, Set& nxt, Set& fill) {
    load_set(fill, s + D);
    read(st, 1);
    part(0, s + 1, st ^ 1, nxt);
    mfmas(std::integral_constant<int, 0>{});
    read(st, 2);
    part(1, s + 1, st ^ 1, nxt);
    mfmas(std::integral_constant<int, 1>{});
    read(st, 3);
    part(2, s + 1, st ^ 1, nxt);
    part(3, s + 1, st ^ 1, nxt);
    mfmas(std::integral_constant<int, 2>{});
    __syncthreads();
    read(st ^ 1, 0);
    mfmas(std::integral_constant<int, 3>{});
    read_scales(st ^ 1);
  };

  Set w[D];
  if constexpr (ONE) {
#pragma unroll
    for (int i = 0; i < NA; ++i) load_a(i, s0, inside(s0), oa, ox);
  }
  if constexpr (DMA) {
    auto joined = [&]() {  // what this wave fetched has arrived, and then every wave's
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt 0
      __syncthreads();
    };
    fetch(s0, 0);
    load_set(w[0], s0);
    part(3, s0, 0, w[0]);
    joined();
    load_set(w[0], s0 + 1);
    fetch(s0 + 1, 1);
    read(0, 0);
    read_scales(0);
    auto round = [&](uint32_t s, int st) {
      read(st, 1);
      __builtin_amdgcn_sched_barrier(0);
      mfmas(std::integral_constant<int, 0>{});
      __builtin_amdgcn_sched_barrier(0);
      read(st, 2);
      __builtin_amdgcn_sched_barrier(0);
      mfmas(std::integral_constant<int, 1>{});
      __builtin_amdgcn_sched_barrier(0);
      read(st, 3);
      __builtin_amdgcn_sched_barrier(0);
      mfmas(std::integral_constant<int, 2>{});
      part(3, s + 1, st ^ 1, w[0]);
      __builtin_amdgcn_sched_barrier(0);
      joined();
      read(st ^ 1, 0);
      __builtin_amdgcn_sched_barrier(0);
      load_set(w[0], s + 2);
      fetch(s + 2, st);
      mfmas(std::integral_constant<int, 3>{});
      read_scales(st ^ 1);
      __builtin_amdgcn_sched_barrier(0);
    };
    for (uint32_t s = s0; s < s1; s += 2) {
      round(s, 0);
      round(s + 1, 1);
    }
    joined();
  } else {
#pragma unroll
  for (int i = 0; i < D; ++i) load_set(w[i], s0 + i);
#pragma unroll
  for (int d = 0; d < 4; ++d) part(d, s0, 0, w[0]);
  __syncthreads();
  read(0, 0);
  read_scales(0);
  for (uint32_t s = s0; s < s1; s += D) {
#pragma unroll
    for (int i = 0; i < D; ++i) step(s + i, i & 1, w[(i + 1) % D], w[i]);
  }
  }

  if constexpr (AT == LT_F16) {
    // A block of the tile has a scale that binary16 cannot hold (or NaN): the tile again, slowly, with weights in
    // bfloat16 and each activation as the sum of two bfloat16 terms, exact for every scale.
    if (__syncthreads_or(misfit)) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.f;
      for (uint32_t q = s0 * 4u; q < kbe * 2u; ++q) {  // 16 values of K
        const uint32_t b = q >> 1, k = q * 16u + fh * 8u;
        bf16x8 wf[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const uint32_t r = (wn * TN + j) * 32 + fr;
          const uint32_t w = bld_u32(rB, r < rowsB ? r * rowB + b * MX_BLOB + ((q & 1u) * 2u + fh) * 4u : MX_OOB, 0);
          wf[j] = mx_dq8<LT_BF16>(w, e8m0(bld_u8(rS[0], r < rowsB ? r * kb + b : MX_OOB, 0)));
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const uint32_t r = (wm * TM + i) * 32 + fr;
          f16x8 x;
#pragma unroll
          for (uint32_t e = 0; e < 8; ++e)
            x[e] = __builtin_bit_cast(f16, static_cast<uint16_t>(bld_u16(rA, (r < rowsA && k + e < K) ? r * rowA + (k + e) * 2u + misA : MX_OOB, 0)));
          bf16x8 hi, lo;
          split_f16(x, hi, lo);
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wf[j], hi, acc[j][i], 0, 0, 0);
            acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wf[j], lo, acc[j][i], 0, 0, 0);
          }
        }
      }
    }
  }

  // ---- output: 32 rows at a time through the wave's part of LDS as float32, then in a loop of few instructions (a
  // workgroup passes here once, and code that is fetched for one pass costs more than it does) eight columns a lane.
  // Split K: the parts meet in the workspace as float32, with coherent stores (sc0 sc1) and one relaxed
  // arrival count a workgroup; the last one adds them in split order.
  constexpr int COHERENT = 1 | 16, PITCH = 32 * TN + 4, PPR = 4 * TN;  // values of a strip's row, pieces of eight
  constexpr uint32_t BYTES = RA * RB * 4;
  const rsrc_t rW = g.splits > 1 ? mk_rsrc(static_cast<uint8_t*>(a.ws) + MX_COUNTERS + static_cast<int64_t>(tile) * g.splits * BYTES, g.splits * BYTES)
                                 : mk_rsrc(a.A, 0);
  float* strip = reinterpret_cast<float*>(smem + wave * Ti::STRIP);
  const uint32_t at = static_cast<uint32_t>(wave) * (TM * TN * 4096u);
  const int64_t nw = n0 + wn * 32 * TN, mw = m0 + wm * 32 * TM;
  const int osz = a.out == LT_F32 ? 4 : 2;
  typedef f32x4 f32x4_4 __attribute__((aligned(4)));  // wide stores start at any dword
  typedef u32x4 u32x4_4 __attribute__((aligned(4)));
  const bool vec = (a.N * osz & 3) == 0 && (reinterpret_cast<uintptr_t>(a.Y) & 3u) == 0;
  auto finish = [&](int r, int p, float (&v)[8]) {  // eight values of row r of the wave's rows, from column 8 p on
    const int64_t m = mw + r, n = nw + 8 * p;
    if (m >= a.M || n >= a.N) return;
    const int left = a.N - n < 8 ? static_cast<int>(a.N - n) : 8;
    if (a.bias != nullptr) {
      if (a.out == LT_F32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += static_cast<const float*>(a.bias)[e < left ? n + e : n];
      } else {
        uint16_t b[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = static_cast<const uint16_t*>(a.bias)[e < left ? n + e : n];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          v[e] += a.out == LT_F16 ? static_cast<float>(__builtin_bit_cast(f16, b[e])) : static_cast<float>(__builtin_bit_cast(bf16, b[e]));
      }
    }
    const int64_t o = m * a.N + n;
    if (a.out == LT_F32) {
      float* y = static_cast<float*>(a.Y) + o;
      if (vec && left == 8) {
        *reinterpret_cast<f32x4_4*>(y) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4_4*>(y + 4) = f32x4{v[4], v[5], v[6], v[7]};
        return;
      }
    } else if (vec && left == 8) {
      u32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] = a.out == LT_F16 ? __builtin_bit_cast(uint32_t, f16x2{static_cast<f16>(v[2 * e]), static_cast<f16>(v[2 * e + 1])})
                               : __builtin_bit_cast(uint32_t, bf16x2{static_cast<bf16>(v[2 * e]), static_cast<bf16>(v[2 * e + 1])});
      *reinterpret_cast<u32x4_4*>(static_cast<uint16_t*>(a.Y) + o) = x;
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) st_lt(a.Y, o + e, v[e], a.out);
  };
  __syncthreads();
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(strip + fr * PITCH + 32 * j + 8 * q + 4 * fh) =
            f32x4{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int x = lane; x < 32 * PPR; x += 64) {
      const int r = x / PPR, p = x % PPR;
      const f32x4 lo = *reinterpret_cast<const f32x4*>(strip + r * PITCH + 8 * p), hi = *reinterpret_cast<const f32x4*>(strip + r * PITCH + 8 * p + 4);
      if (g.splits > 1) {
        if (mw + 32 * i + r >= a.M) continue;
        const uint32_t o = split * BYTES + at + (static_cast<uint32_t>(i) * 32 * PPR + x) * 32u;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, lo), rW, o, 0, COHERENT);
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, hi), rW, o + 16, 0, COHERENT);
      } else {
        float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        finish(32 * i + r, p, v);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  if (g.splits == 1) return;
  __shared__ int s_last;
  uint32_t* cnt = static_cast<uint32_t*>(a.ws);
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (tid == 0) s_last = __hip_atomic_fetch_add(cnt + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == g.splits - 1;
  __syncthreads();
  if (!s_last) return;
  // 32 loads in flight: each batch costs a trip past the caches
  constexpr int XB = TM * 32 * PPR / 64 < 4 ? TM * 32 * PPR / 64 : 4, SB = 16 / XB;
#pragma unroll 1
  for (int x0 = lane; x0 < TM * 32 * PPR; x0 += 64 * XB) {
    f32x4 lo[XB], hi[XB];
#pragma unroll
    for (int k = 0; k < XB; ++k) lo[k] = hi[k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (uint32_t sp = 0; sp < g.splits; sp += SB) {  // past the last split zeros
      f32x4 pl[XB][SB], ph[XB][SB];
#pragma unroll
      for (int k = 0; k < XB; ++k)
#pragma unroll
        for (uint32_t i = 0; i < SB; ++i) {
          const int x = x0 + 64 * k;
          const uint32_t o = sp + i < g.splits && mw + x / PPR < a.M ? (sp + i) * BYTES + at + x * 32u : MX_OOB;
          pl[k][i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rW, o, 0, COHERENT));
          ph[k][i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rW, o + 16, 0, COHERENT));
        }
#pragma unroll
      for (int k = 0; k < XB; ++k)
#pragma unroll
        for (int i = 0; i < SB; ++i) {
          lo[k] += pl[k][i];
          hi[k] += ph[k][i];
        }
    }
#pragma unroll
    for (int k = 0; k < XB; ++k) {
      const int x = x0 + 64 * k;
      float v[8] = {lo[k][0], lo[k][1], lo[k][2], lo[k][3], hi[k][0], hi[k][1], hi[k][2], hi[k][3]};
      finish(x / PPR, x % PPR, v);
    }
  }
  if (tid == 0) __hip_atomic_store(cnt + tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Tile l of a raster in groups of four row tiles, row fastest inside a group: the tiles that one XCD
// runs at once share few row and column panels in its L2.
__device__ __forceinline__ void mx_raster(uint32_t l, uint32_t mt, uint32_t nc, uint32_t& row, uint32_t& col) {
  constexpr uint32_t G = 4;
  const uint32_t q = l / (G * nc), rows = mt - q * G < G ? mt - q * G : G, r = l - q * G * nc;
  row = q * G + r % rows;
  col = r / rows;
}

template <int AT, int WM, int TM, int TN, bool AL>
__global__ __launch_bounds__(128 * WM, TM == 1 ? 3 : 2) void k_mx4_gemm(MxArgs a, MxGrid g) {
  uint32_t row, col;
  const uint32_t bid = blockIdx.x;
  if (TN < 4 || bid < g.nbig) {
    const uint32_t n = g.mt * g.nb * g.splits, l = xcd_slot(bid, n), split = l % g.splits;
    mx_raster(l / g.splits, g.mt, g.nb, row, col);
    mx_tile<AT, WM, TM, TN, AL>(a, row, static_cast<int64_t>(col) * (64 * TN), g, l / g.splits, split);
  } else if constexpr (TN == 4) {
    const uint32_t n = g.mt * g.ns, l = xcd_slot(bid - g.nbig, n);
    mx_raster(l, g.mt, g.ns, row, col);
    mx_tile<AT, WM, TM, 3, AL>(a, row, static_cast<int64_t>(g.nb) * 256 + static_cast<int64_t>(col) * 192, g, 0, 0);
  }
}

template <int AT, int WM, int TM, int TN, bool AL>
hipError_t gemm_al(const MxArgs& a, const MxPlan& p, hipStream_t st) {
  auto kern = k_mx4_gemm<AT, WM, TM, TN, AL>;
  constexpr int lds = MxTile<AT, WM, TM, TN>::LDS;
  static std::atomic<int> done[kMaxDevices];
  if (lds > 65536) {
    const hipError_t e = raise_lds_cap(reinterpret_cast<const void*>(kern), lds, done);
    if (e != hipSuccess) return e;
  }
  const MxGrid g{p.mt, p.nb, p.ns, p.mt * p.nb * p.splits, p.splits, p.per};
  const int64_t n = static_cast<int64_t>(p.mt) * p.nb * p.splits + static_cast<int64_t>(p.mt) * p.ns;
  if (n > 0x7FFFFFFF) return hipErrorInvalidValue;
  kern<<<dim3(static_cast<uint32_t>(n)), 128 * WM, lds, st>>>(a, g);
  return hipGetLastError();
}

template <int AT, int WM, int TM, int TN>
hipError_t gemm_for(const MxArgs& a, const MxPlan& p, hipStream_t st) {
  if (AT < 0 || (a.K % 8 == 0 && (reinterpret_cast<uintptr_t>(a.A) & 15u) == 0)) return gemm_al<AT, WM, TM, TN, true>(a, p, st);
  if constexpr (AT >= 0) return gemm_al<AT, WM, TM, TN, false>(a, p, st);
  return hipErrorInvalidValue;
}

template <int AT>
hipError_t gemm_at(const MxArgs& a, const MxPlan& p, hipStream_t st) {
  if (p.t == 4) return gemm_for<AT, 4, 2, 4>(a, p, st);
  if (p.t == 2) return gemm_for<AT, 2, 2, 2>(a, p, st);
  return gemm_for<AT, 2, 1, 1>(a, p, st);
}

}  // namespace

// The plan with the least estimated time. A tile size costs a CU so much for a K step: what one workgroup alone takes,
// or the work of all its workgroups at the rate of a full CU (units of 64 x 64; us measured at 2.4 GHz); and a start, and
// so much more for each further round of the CUs:
//   16-bit activations, steps of 64:  64-tiles 0.43, 3.3 units a us; 128-tiles 0.66, 6; 256-tiles 1.8, 8.9; starts 3, 5, 12 (a round)
//   both MX4, steps of 256:           64-tiles 0.60, 2.35 units a us; 128-tiles 1.0, 4.3; 256-tiles 1.0, 6.67; starts 3, 5 (1.7 a round),
//                                     8.2 (a round)
// MX4 256-tiles wait on memory that all CUs share: a round that leaves CUs out is faster, 0.4 of a full one with a few
// tiles, 0.9 with half the CUs. A split exchange costs 5 us and what its parts weigh.
// It places 512 x 4096 x 4096 of 16 bits on 64- or 128-tiles (39 to 44 us; 256-tiles 55), 128 rows on 64-tiles with K split (21; 128-tiles 25),
// 2048 x 4096 x 14336 on 256-tiles (231 to 244 by the box; 128-tiles 281); MX4 700 x 4096 x 14336 on 256-tiles (44 us; 128-tiles 53), 512 rows on 128-tiles
// (38.5; 256-tiles 45, 64-tiles 53).
MxPlan mx4_gemm_plan(int64_t M, int64_t K, int64_t N, int a_type, bool have_ws) {
  MxPlan best{};
  const bool mx = a_type < 0;
  const int64_t kb = (K + MX_BLOCK - 1) / MX_BLOCK;
  if (M <= 16 || K > (int64_t(1) << 21)) return best;  // 256 rows of 16-bit values stay below 2^31 bytes
  const int64_t cus = device_cus() > 0 ? device_cus() : 256;
  const int64_t steps = (kb + (mx ? 7 : 1)) / (mx ? 8 : 2);
  struct Cost {
    int t;
    double alone, rate, start, more;
  };
  static constexpr Cost kCost[2][3] = {{{1, 0.43, 3.3, 3, 0}, {2, 0.66, 6.0, 5, 0}, {4, 1.8, 8.9, 12, 12}},
                                       {{1, 0.60, 2.35, 3, 0}, {2, 1.0, 4.3, 5, 1.7}, {4, 1.0, 6.67, 8.2, 8.2}}};
  double least = 0;
  for (const Cost& c : kCost[mx ? 1 : 0]) {
    const int64_t mt = (M + 64 * c.t - 1) / (64 * c.t), nt = (N + 64 * c.t - 1) / (64 * c.t), n = mt * nt;
    if (n > 0x3FFFFFFF) continue;
    const int64_t ahead = mxg_ahead(mx, c.t);  // a split's steps are a multiple
    for (int64_t s = 1; s <= 8; ++s) {
      if (s > 1 && (!have_ws || n > MX_COUNTERS / 4 || n * s > 2 * cus || steps < 4 * s)) break;
      MxPlan p{};
      p.t = c.t;
      p.mt = static_cast<uint32_t>(mt);
      p.nb = static_cast<uint32_t>(nt);
      p.per = static_cast<uint32_t>((steps + ahead * s - 1) / (ahead * s) * ahead);
      p.splits = static_cast<uint32_t>((steps + p.per - 1) / p.per);
      if (p.splits != s) continue;
      double rounds = static_cast<double>((n * s + cus - 1) / cus);  // tiles of the fullest CU
      if (mx && c.t == 4 && n * s % cus != 0) {
        const double part = static_cast<double>(n * s % cus) / static_cast<double>(cus);
        rounds = static_cast<double>(n * s / cus) + 0.4 + (part < 0.6 ? part : 0.6);
      }
      if (c.t == 4 && s == 1 && rounds > 1 && cus % mt == 0) {
        // columns of wide tiles and narrow ones (192) mixed, where that makes fewer rounds of the CUs: k whole rounds of wide
        // ones, and at most j of narrow ones, as many as the columns behind them need
        const int64_t per = cus / mt;
        for (int64_t j = 1; j <= 16; ++j) {
          const int64_t rest = N - 192 * j * per, k = rest > 0 ? (rest + 256 * per - 1) / (256 * per) : 0;
          const double r = static_cast<double>(k) + 0.75 * static_cast<double>(j);
          if (r < rounds - 0.05) {
            rounds = r;
            p.nb = static_cast<uint32_t>(k * per);
            p.ns = static_cast<uint32_t>((N - 256 * k * per + 191) / 192);
          }
        }
      }
      const double units = static_cast<double>(c.t * c.t), step = units * rounds / c.rate;
      double time = c.start + c.more * (rounds > 1 ? rounds - 1 : 0) + static_cast<double>(p.per) * (step > c.alone ? step : c.alone);
      if (s > 1) {
        p.ws_bytes = MX_COUNTERS + n * s * c.t * c.t * 16384;
        time += 5.0 + static_cast<double>(p.ws_bytes) * 0.5e-6;  // written and read back at about 4 TB/s
      }
      if (best.t == 0 || time < least) {
        best = p;
        least = time;
      }
    }
  }
  return best;
}

hipError_t launch_mx4_gemm(const MxArgs& a, const MxPlan& p, hipStream_t st) {
  switch (a.a_type) {
    case LT_F16: return gemm_at<LT_F16>(a, p, st);
    case LT_BF16: return gemm_at<LT_BF16>(a, p, st);
    default: return gemm_at<-1>(a, p, st);
  }
}

}  // namespace xrmm
