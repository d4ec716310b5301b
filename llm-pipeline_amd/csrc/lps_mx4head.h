// LM head over a 4-bit weight: logits[m, n] = sum over k of x[m, k] w[n, k], x in
// bf16, fp16 or 4 bits, w in microscaled 4-bit floats (lps_mx4.h), fp32
// accumulation, with the 16-bit head's epilogue (lps_lmhead.h: block statistics).
//
// x in 4 bits: v_mfma_scale_f32_32x32x64_f8f6f4 on the codes themselves.  Lane l
// holds A row and B column l % 32 and one whole block, k = 32 (l / 32) .. +31 of
// the 64, as its 16 bytes, and the block's scale byte in a register that the
// instruction picks a byte of (checked on gfx950).
//
// x in 16 bits: the codes are converted in registers (v_cvt_scalef32_pk_*_fp4,
// exact) and multiplied by v_mfma_f32_32x32x16_*.  The order of a product's
// terms is free, so a lane takes a whole block of w again (lanes l and l + 32
// neighbouring ones) and spends it over four instructions, against the chunks of
// x that belong to it: w is read from LDS in 16 bytes a lane, once, with one
// scale a lane.  bf16 holds every value of w.  fp16 holds those of scales 2^-23 ..
// 2^13; a stage in which a wave meets another scale takes x apart into two bf16
// (11 bits as 8 and 3) and runs the bf16 instruction twice, which is exact too.
#pragma once

#include <type_traits>

#include "lps_common.h"
#include "lps_lmhead.h"
#include "lps_mx4.h"

namespace lps {

struct Mx4HeadParams {
  LmHeadParams h;            // x, w (codes); x_stride in elements (bytes of codes), w_stride in bytes
  const uint8_t* ws;         // scales of w, rows on 4-byte lines
  const uint8_t* xs;         // scales of a 4-bit x, rows on 4-byte lines
  int64_t ws_stride, xs_stride;
  int wide;                  // rows of scales lie and end on 16-byte lines
};

// One workgroup of WM x WN waves computes a BM x BN tile; K is walked in stages of
// NB blocks (32 NB values) through a ring of NS LDS buffers, filled by loads that
// cost no registers (lps_lmhead.h).  A stage holds the x rows, then the w rows (16
// bytes a block, chunk c of row r at place c ^ f(r)).  XB: bytes of a block of x,
// 64 or 16.  A row has 4 bytes of scales where it has 64 of codes: loaded by the
// stage they cost as many cache lines as the codes do (2048 x 4096 -> 151936 in 4
// bits 1112 us, 732 without them), so that they come 32 blocks at a time, into two
// buffers of their own.
constexpr int M4_SB = 32;
constexpr int64_t M4_MAX_STRIDE = 1 << 23;   // bytes: 256 rows of it fit 32-bit offsets
template <int BM_, int BN_, int WM_, int WN_, int NB_, int NS_, int WPE_, int XB_>
struct M4Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NB = NB_, NS = NS_, WPE = WPE_, XB = XB_;
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int MT = BM / WM / 32, CT = BN / WN / 32;    // accumulators per wave: rows x columns
  static constexpr int WTN = 32 * CT;
  static constexpr int XC = NB * XB / 16, WC = NB;              // 16-byte chunks per row
  static constexpr int XRI = 64 / XC, WRI = 64 / WC;            // rows a wave's load instruction covers
  static constexpr int XI = BM / XRI, WI = BN / WRI;            // load instructions of a stage
  static constexpr int XPW = (XI + NW - 1) / NW, WPW = WI / NW; // ... of a wave (with more waves than XI some load the same)
  static constexpr bool XS = XB == 16;
  static constexpr int SROWS = BN + (XS ? BM : 0);              // rows with scales: w's, then x's
  static constexpr int LPW = XPW + WPW;
  static constexpr int XBYTES = BM * XC * 16, WBYTES = BN * WC * 16;
  static constexpr int STAGE = XBYTES + WBYTES;
  static constexpr int SBYTES = SROWS * M4_SB;
  static constexpr int KS = NB / 2;                             // steps of two blocks
  static constexpr int PER = M4_SB / NB;                        // stages to a buffer of scales
  static_assert(NB == 4 || NB == 8, "chunk places");
  static_assert((XI % NW == 0 || NW % XI == 0) && WI % NW == 0, "whole load instructions per wave");
  static_assert(BN % 32 == 0 && BM % 32 == 0, "whole loads of scales");
  static_assert(BM % (32 * WM) == 0 && BN % (32 * WN) == 0 && BN % LMH_BN == 0, "tile shape");
  static_assert(PER >= NS - 1, "scales are asked for before the stage that needs them");
  static_assert((NS - 1) * LPW + 4 * SROWS / 32 / NW + 1 < 64, "the load counter holds 63");
  __device__ __forceinline__ static int xperm(int row) { return XC >= 8 ? (row & 7) : ((row >> 1) & 3); }
  __device__ __forceinline__ static int wperm(int row) { return WC >= 8 ? (row & 7) : ((row >> 1) & 3); }
};
template <typename T, int ES>
constexpr int m4_lds_bytes() {
  return T::NS * T::STAGE + 2 * T::SBYTES > lmh_epi_bytes<T, ES>() ? T::NS * T::STAGE + 2 * T::SBYTES : lmh_epi_bytes<T, ES>();
}

#ifndef LPS_HOST_EMU
// Byte address in LDS of a shared array.
__device__ __forceinline__ uint32_t m4_lds(const char* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}
// 16 / 4 bytes per lane from base + off (base uniform) to LDS at (uniform) dst + 16 / 4 * lane.
template <bool NTL>
__device__ __forceinline__ void m4_dma16(const char* base, uint32_t off, uint32_t dst) {
  if constexpr (NTL)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(dst), "v"(off), "s"(base) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void m4_dma4(const char* base, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(dst), "v"(off), "s"(base) : "memory");
}
#else
inline uint64_t m4_lds(const char* p) { return (uint64_t)(uintptr_t)p; }
template <bool NTL>
inline void m4_dma16(const char* base, uint32_t off, uint64_t dst) {
  memcpy(reinterpret_cast<char*>(dst) + 16 * ((int)threadIdx.x & 63), base + off, 16);
}
inline void m4_dma4(const char* base, uint32_t off, uint64_t dst) {
  memcpy(reinterpret_cast<char*>(dst) + 4 * ((int)threadIdx.x & 63), base + off, 4);
}
#endif

// Eight codes as one fragment of the 16-bit instruction.
template <int DT>
__device__ __forceinline__ u32x4 m4_frag(uint32_t codes, float s) {
  u32x4 r;
  if constexpr (DT == LPS_DTYPE_BF16) {
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 0));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 1));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 2));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 3));
  } else {
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, 0));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, 1));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, 2));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, 3));
  }
  return r;
}

// Eight fp16 as two bf16 fragments whose sum they are: the top 8 bits of each
// (cut off), and the rest (at most 3 bits, exact; 0 for infinities and NaN).
__device__ __forceinline__ void m4_split(u32x4 x, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint32_t h[2], r[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const float f = f16_to_f32((x[i] >> (16 * e)) & 0xFFFFu);
      h[e] = __float_as_uint(f) & 0xFFFF0000u;
      const bool fine = (h[e] & 0x7F800000u) != 0x7F800000u;
      // (a NaN whose set bits are all below the cut stays one)
      if (!fine && f != f) h[e] |= 0x00400000u;
      r[e] = fine ? __float_as_uint(__fsub_rn(f, __uint_as_float(h[e]))) : 0u;
    }
    hi[i] = (h[0] >> 16) | h[1];
    lo[i] = (r[0] >> 16) | (r[1] & 0xFFFF0000u);
  }
}

// Whether any of four scale bytes is outside 104 .. 140 (2^-23 .. 2^13).
__device__ __forceinline__ bool m4_far_scale(uint32_t w) {
  bool far = false;
#pragma unroll
  for (int k = 0; k < 4; k++) far = far || ((w >> (8 * k)) & 255u) - 104u > 36u;
  return far;
}

// The position of a lane in a tile, and its reads of a stage.
template <typename T>
struct M4Lane {
  int half, xr, wr, px, pw;
  __device__ __forceinline__ M4Lane(int wm, int wn, int l)
      : half(l >> 5), xr(wm * (T::MT * 32) + (l & 31)), wr(wn * T::WTN + (l & 31)), px(T::xperm(xr)), pw(T::wperm(wr)) {}
  // (rows 32 apart share their permutation)
  __device__ __forceinline__ u32x4 x(const char* stage, int i, int c) const {
    return *reinterpret_cast<const u32x4*>(stage + ((xr + 32 * i) * T::XC + (c ^ px)) * 16);
  }
  __device__ __forceinline__ u32x4 w(const char* stage, int i, int c) const {
    return *reinterpret_cast<const u32x4*>(stage + T::XBYTES + ((wr + 32 * i) * T::WC + (c ^ pw)) * 16);
  }
  // four blocks' scales of a row (word d of the stage); this lane's are in bytes 0 and 2
  __device__ __forceinline__ uint32_t ws_all(const char* scales, int i, int d) const {
    return *reinterpret_cast<const uint32_t*>(scales + (wr + 32 * i) * M4_SB + 4 * d);
  }
  __device__ __forceinline__ uint32_t ws(const char* scales, int i, int d) const { return ws_all(scales, i, d) >> (8 * half); }
  __device__ __forceinline__ uint32_t xs(const char* scales, int i, int d) const {
    return *reinterpret_cast<const uint32_t*>(scales + (T::BN + xr + 32 * i) * M4_SB + 4 * d) >> (8 * half);
  }
};

// A byte of a word of scales as the conversions' scale: its neighbours land in the
// sign and the mantissa, which they ignore.
__device__ __forceinline__ float m4_scale(uint32_t w, int j) { return __uint_as_float((j & 1) ? w << 7 : w << 23); }

typedef int i32x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ i32x8 m4_operand(u32x4 v) { return i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0}; }
template <typename ACC>
__device__ __forceinline__ ACC m4_mma4(u32x4 a, u32x4 b, ACC c, uint32_t sa, uint32_t sb, int j) {
  if (j & 1) return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(m4_operand(a), m4_operand(b), c, 4, 4, 2, (int)sa, 2, (int)sb);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(m4_operand(a), m4_operand(b), c, 4, 4, 0, (int)sa, 0, (int)sb);
}

// The accumulators plus `steps` steps of two blocks, one after another: the last
// columns of a row, and (FAR) stages of fp16 with scales that it does not hold.
template <int XDT, typename T, bool FAR, typename ACC>
__device__ __forceinline__ void m4_plain_stage(const char* stage, const char* scales, const M4Lane<T>& L,
                                               ACC (&acc)[T::MT][T::CT], int steps) {
#pragma unroll 1
  for (int j = 0; j < steps; j++) {
    const int c = 2 * j + L.half;
#pragma unroll
    for (int b = 0; b < T::CT; b++) {
      const u32x4 cw = L.w(stage, b, c);
      const uint32_t byte = (L.ws_all(scales, b, j >> 1) >> (8 * (c & 3))) & 255u;
      if constexpr (T::XS) {
#pragma unroll
        for (int a = 0; a < T::MT; a++)
          acc[a][b] = m4_mma4(L.x(stage, a, c), cw, acc[a][b], L.xs(scales, a, j >> 1) >> (16 * (j & 1)), byte, 0);
      } else {
        const float s = __uint_as_float(byte << 23);
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const u32x4 fw = m4_frag<FAR ? LPS_DTYPE_BF16 : XDT>(cw[q], s);
#pragma unroll
          for (int a = 0; a < T::MT; a++) {
            const u32x4 fx = L.x(stage, a, 4 * c + q);
            if constexpr (FAR) {
              u32x4 hi, lo;
              m4_split(fx, hi, lo);
              acc[a][b] = MfmaOps<LPS_DTYPE_BF16>::mma(hi, fw, acc[a][b]);
              acc[a][b] = MfmaOps<LPS_DTYPE_BF16>::mma(lo, fw, acc[a][b]);
            } else {
              acc[a][b] = MfmaOps<XDT>::mma(fx, fw, acc[a][b]);
            }
          }
        }
      }
    }
  }
}

// XDT: BF16, F16 or MX4; T::XB 64 or 16 accordingly.
template <int XDT, int ODT, typename T, bool NTL>
__global__ __launch_bounds__(T::NT, T::WPE) void mx4head_kernel(Mx4HeadParams Q) {
  constexpr int ES = ODT == LPS_DTYPE_F32 ? 4 : 2;
  constexpr int ADT = XDT == LPS_DTYPE_F16 ? LPS_DTYPE_F16 : LPS_DTYPE_BF16;   // (the accumulators are alike)
  constexpr int MT = T::MT, CT = T::CT, NB = T::NB, KS = T::KS;
  __shared__ __attribute__((aligned(1024))) char lds[m4_lds_bytes<T, ES>()];
  const LmHeadParams& P = Q.h;
  // tiles over the XCDs as in lmhead_kernel: a run each, the row tiles of one column tile first
  const int per = (P.tiles + 7) >> 3;
  const int t = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
  if (((int)blockIdx.x >> 3) >= per || t >= P.tiles) return;   // uniform over the workgroup
  const int m0 = (t % P.mtiles) * T::BM, n0 = (t / P.mtiles) * T::BN;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), l = (int)threadIdx.x & 63;
  const int wm = wv / T::WN, wn = wv % T::WN;
  const int64_t xstep = T::XS ? P.x_stride : 2 * P.x_stride;   // bytes of a row of x
  const char* const X = reinterpret_cast<const char*>(P.x) + (int64_t)m0 * xstep;
  const char* const W = reinterpret_cast<const char*>(P.w) + (int64_t)n0 * P.w_stride;
  // rows of the tile, clamped into range (the others' results are dropped); their
  // offsets in it fit 32 bits (M4_MAX_STRIDE)
  auto mrow = [&](int r) { return m0 + r < P.M ? r : P.M - 1 - m0; };
  auto nrow = [&](int r) { return n0 + r < P.V ? r : P.V - 1 - n0; };

  uint32_t xoff[T::XPW], woff[T::WPW];
#pragma unroll
  for (int i = 0; i < T::XPW; i++) {
    const int row = ((i * T::NW + wv) % T::XI) * T::XRI + l / T::XC, c = (l % T::XC) ^ T::xperm(row);
    xoff[i] = (uint32_t)mrow(row) * (uint32_t)xstep + c * 16;
  }
#pragma unroll
  for (int i = 0; i < T::WPW; i++) {
    const int row = (i * T::NW + wv) * T::WRI + l / T::WC, c = (l % T::WC) ^ T::wperm(row);
    woff[i] = (uint32_t)nrow(row) * (uint32_t)P.w_stride + c * 16;
  }
  const auto lds0 = m4_lds(lds);
  auto issue = [&](int s, int buf) {   // stage s into ring buffer buf
    const char* xb = X + (int64_t)s * (NB * T::XB);
    const char* wb = W + (int64_t)s * (NB * 16);
    const auto d = lds0 + buf * T::STAGE;
#pragma unroll
    for (int i = 0; i < T::XPW; i++) m4_dma16<false>(xb, xoff[i], d + ((i * T::NW + wv) % T::XI) * 1024);
#pragma unroll
    for (int i = 0; i < T::WPW; i++) m4_dma16<NTL>(wb, woff[i], d + T::XBYTES + (i * T::NW + wv) * 1024);
  };
  const int ns = P.H / (32 * NB);   // whole stages of whole blocks; the rest of H follows them
  // scales of blocks 32 u .. +31, as far as the whole stages go: a row's 32 bytes
  // by two lanes, or by eight where it does not lie on 16-byte lines
  char* const sbuf = lds + T::NS * T::STAGE;
  const auto sdst = lds0 + T::NS * T::STAGE;
  const char* const WS = reinterpret_cast<const char*>(Q.ws) + (int64_t)n0 * Q.ws_stride;
  const char* const XSC = T::XS ? reinterpret_cast<const char*>(Q.xs) + (int64_t)m0 * Q.xs_stride : nullptr;
  auto issue_scales = [&](int u) {
    const auto d = sdst + (u & 1) * T::SBYTES;
    const int rl = Q.wide ? 32 : 8, groups = T::SROWS / rl, r0 = Q.wide ? l >> 1 : l >> 3;
    int b = M4_SB * u + (Q.wide ? 16 * (l & 1) : 4 * (l & 7));
    b = b < NB * ns ? b : 0;          // (a row without them: others of its own)
    for (int i = wv; i < groups; i += T::NW) {
      const bool ofx = T::XS && rl * i >= T::BN;
      const char* base = ofx ? XSC : WS;
      const uint32_t off = (ofx ? (uint32_t)mrow(rl * i + r0 - T::BN) * (uint32_t)Q.xs_stride
                                : (uint32_t)nrow(rl * i + r0) * (uint32_t)Q.ws_stride) + b;
      if (Q.wide) m4_dma16<false>(base, off, d + i * 1024);
      else m4_dma4(base, off, d + i * 256);
    }
  };

  typename MfmaOps<ADT>::acc acc[MT][CT] = {};
  const M4Lane<T> L(wm, wn, l);
  // Fragments are read one step ahead of their matrix instructions and, of a
  // 16-bit x, the codes converted one ahead, in the shadow of the matrix cores;
  // the last step of a stage waits for the next one and reads its first.
  constexpr int STEPS = T::XS ? KS : 4 * KS;       // matrix steps of a stage (64 or 16 values)
  u32x4 fx[2][MT], cw[2][CT], fw[2][CT];
  uint32_t sw[NB / 4][CT], sx[NB / 4][MT];
  auto read_scales = [&](const char* scales) {
#pragma unroll
    for (int d = 0; d < NB / 4; d++) {
#pragma unroll
      for (int i = 0; i < CT; i++) sw[d][i] = L.ws(scales, i, d);
      if constexpr (T::XS) {
#pragma unroll
        for (int i = 0; i < MT; i++) sx[d][i] = L.xs(scales, i, d);
      }
    }
  };
  auto read_x = [&](const char* stage, int k) {    // for matrix step k
    const int c = T::XS ? 2 * k + L.half : 4 * (2 * (k >> 2) + L.half) + (k & 3);
#pragma unroll
    for (int i = 0; i < MT; i++) fx[k & 1][i] = L.x(stage, i, c);
  };
  auto read_w = [&](const char* stage, int j) {    // for blocks 2 j and 2 j + 1
#pragma unroll
    for (int i = 0; i < CT; i++) cw[j & 1][i] = L.w(stage, i, 2 * j + L.half);
  };
  auto convert = [&](int k) {
    if constexpr (!T::XS) {
      const int j = k >> 2;
#pragma unroll
      for (int i = 0; i < CT; i++) fw[k & 1][i] = m4_frag<XDT>(cw[j & 1][i][k & 3], m4_scale(sw[j >> 1][i], j));
    }
  };
  auto far_scales = [&](const char* scales) {      // (uniform over the wave)
    bool far = false;
    if constexpr (XDT == LPS_DTYPE_F16) {
#pragma unroll
      for (int d = 0; d < NB / 4; d++)
#pragma unroll
        for (int i = 0; i < CT; i++) far = far || m4_far_scale(L.ws_all(scales, i, d));
      far = wballot(far) != 0;
    }
    return far;
  };
  auto scales_of = [&](int s) { return sbuf + ((s / T::PER) & 1) * T::SBYTES + (s % T::PER) * NB; };
  if (ns > 0) {
    issue_scales(0);
    for (int s = 0; s < T::NS && s < ns; s++) issue(s, s);
    if (ns >= T::NS) lmh_wait_barrier<(T::NS - 1) * T::LPW>();
    else lmh_wait_barrier<0>();
    read_scales(scales_of(0));
    read_w(lds, 0);
    read_x(lds, 0);
    convert(0);
    int buf = 0;
    for (int s = 0; s < ns; s++) {
      const char* cur = lds + buf * T::STAGE;
      const int nb = buf + 1 == T::NS ? 0 : buf + 1;
      const bool far = far_scales(scales_of(s));
      if (XDT == LPS_DTYPE_F16 && far) m4_plain_stage<XDT, T, true>(cur, scales_of(s), L, acc, KS);
#pragma unroll
      for (int k = 0; k < STEPS; k++) {
        if (k + 1 < STEPS) {
          if (XDT == LPS_DTYPE_F16 && far) continue;
          if constexpr (T::XS) read_w(cur, k + 1);
          else if ((k & 3) == 1 && (k >> 2) + 1 < KS) read_w(cur, (k >> 2) + 1);
          read_x(cur, k + 1);
          __builtin_amdgcn_sched_barrier(0);   // (the compiler would move the reads down to their use)
        }
        if (k + 1 == STEPS) {
          uint32_t ow[CT], ox[MT];   // (this step's scales)
          if constexpr (T::XS) {
#pragma unroll
            for (int i = 0; i < CT; i++) ow[i] = sw[NB / 4 - 1][i];
#pragma unroll
            for (int i = 0; i < MT; i++) ox[i] = sx[NB / 4 - 1][i];
          }
          if (s + 1 < ns) {
            // every wave holds its last fragments of stage s, stage s + 1 has landed
            // (and its scales, asked for before it)
            lmh_wait_stage<T>(ns - 2 - s);
            if (s % T::PER == 0 && s + T::PER < ns) issue_scales(s / T::PER + 1);
            if (s + T::NS < ns) issue(s + T::NS, buf);
            read_scales(scales_of(s + 1));
            read_w(lds + nb * T::STAGE, 0);
            read_x(lds + nb * T::STAGE, 0);
            __builtin_amdgcn_sched_barrier(0);
          }
          if (!(XDT == LPS_DTYPE_F16 && far)) {
#pragma unroll
            for (int a = 0; a < MT; a++)
#pragma unroll
              for (int b = 0; b < CT; b++) {
                if constexpr (T::XS) acc[a][b] = m4_mma4(fx[k & 1][a], cw[k & 1][b], acc[a][b], ox[a], ow[b], k);
                else acc[a][b] = MfmaOps<ADT>::mma(fx[k & 1][a], fw[k & 1][b], acc[a][b]);
              }
          }
          if (s + 1 < ns) convert(0);
        } else {
#pragma unroll
          for (int a = 0; a < MT; a++)
#pragma unroll
            for (int b = 0; b < CT; b++) {
              if constexpr (T::XS) acc[a][b] = m4_mma4(fx[k & 1][a], cw[k & 1][b], acc[a][b], sx[k >> 1][a], sw[k >> 1][b], k);
              else acc[a][b] = MfmaOps<ADT>::mma(fx[k & 1][a], fw[k & 1][b], acc[a][b]);
            }
          convert(k + 1);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      buf = nb;
    }
    __syncthreads();
  }
  const int k0 = ns * 32 * NB;
  if (k0 < P.H) {
    // the columns past the last whole stage, zeros up to one (with scales of 1)
    const int nblk = (P.H + 31) >> 5, b0 = ns * NB;
    for (int i = threadIdx.x; i < T::BM * T::XC; i += T::NT) {
      const int row = i / T::XC, c = (i % T::XC) ^ T::xperm(row);
      u32x4 v = {0u, 0u, 0u, 0u};
      const char* xr = X + (int64_t)mrow(row) * xstep;
      if constexpr (T::XS) {
        if (b0 + c < nblk) v = *reinterpret_cast<const u32x4*>(xr + (b0 + c) * 16);
      } else {
        const int e0 = k0 + 8 * c;
        if (e0 < P.H) v = load_piece<ADT>(xr, e0, P.H).q[0];
      }
      *reinterpret_cast<u32x4*>(lds + i * 16) = v;
    }
    char* wb = lds + T::XBYTES;
    for (int i = threadIdx.x; i < T::BN * T::WC; i += T::NT) {
      const int row = i / T::WC, b = b0 + ((i % T::WC) ^ T::wperm(row));
      u32x4 v = {0u, 0u, 0u, 0u};
      if (b < nblk) {
        v = *reinterpret_cast<const u32x4*>(W + (int64_t)nrow(row) * P.w_stride + b * 16);
#pragma unroll
        for (int e = 0; e < 4; e++) {               // (codes past the row's end count as zeros, whatever they hold)
          const int keep = P.H - 32 * b - 8 * e;
          v[e] = keep >= 8 ? v[e] : keep <= 0 ? 0u : v[e] & ((1u << (4 * keep)) - 1u);
        }
      }
      *reinterpret_cast<u32x4*>(wb + i * 16) = v;
    }
    for (int i = threadIdx.x; i < T::SROWS * NB; i += T::NT) {
      const int row = i / NB, b = b0 + i % NB;
      const char* sr = WS + (int64_t)nrow(row < T::BN ? row : 0) * Q.ws_stride;
      if constexpr (T::XS)
        if (row >= T::BN) sr = XSC + (int64_t)mrow(row - T::BN) * Q.xs_stride;
      sbuf[row * M4_SB + i % NB] = b < nblk ? sr[b] : (char)127;
    }
    __syncthreads();
    const int steps = (nblk - b0 + 1) / 2;
    if (XDT == LPS_DTYPE_F16 && far_scales(sbuf)) m4_plain_stage<XDT, T, true>(lds, sbuf, L, acc, steps);
    else m4_plain_stage<XDT, T, false>(lds, sbuf, L, acc, steps);
    __syncthreads();
  }
  lmh_epilogue<ADT, ODT, T>(P, lds, acc, n0, m0, wv, l);
}

}  // namespace lps
