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
};

// One workgroup of WM x WN waves computes a BM x BN tile; K is walked in stages of
// NB blocks (32 NB values) through a ring of NS LDS buffers, filled by loads that
// cost no registers (lps_lmhead.h).  A stage holds the x rows, the w rows (16
// bytes a block, chunk c of row r at place c ^ f(r)), then the scales of both, 4
// bytes a row.  XB: bytes of a block of x, 64 or 16.
template <int BM_, int BN_, int WM_, int WN_, int NS_, int WPE_, int XB_>
struct M4Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NS = NS_, WPE = WPE_, XB = XB_;
  static constexpr int NB = 4;                                  // blocks per stage
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int MT = BM / WM / 32, CT = BN / WN / 32;    // accumulators per wave: rows x columns
  static constexpr int WTN = 32 * CT;
  static constexpr int XC = NB * XB / 16, WC = NB;              // 16-byte chunks per row
  static constexpr int XRI = 64 / XC, WRI = 64 / WC;            // rows a wave's load instruction covers
  static constexpr int XI = BM / XRI, WI = BN / WRI;             // load instructions of a stage
  static constexpr int XPW = (XI + NW - 1) / NW, WPW = WI / NW; // ... of a wave (with more waves than XI some load the same)
  static constexpr bool XS = XB == 16;
  static constexpr int SMR = BM < 64 ? 64 : BM;                 // scale rows of x a stage holds
  static constexpr int LPW = XPW + WPW + 1 + (XS ? 1 : 0);      // loads per wave and stage
  static constexpr int XBYTES = BM * XC * 16, WBYTES = BN * WC * 16;
  static constexpr int STAGE = XBYTES + WBYTES + BN * 4 + (XS ? SMR * 4 : 0);
  static constexpr int KS = NB / 2;                             // steps of two blocks
  static_assert((XI % NW == 0 || NW % XI == 0) && WI % NW == 0, "whole load instructions per wave");
  static_assert(BN / 64 <= NW && SMR / 64 <= NW, "a load of scales per wave covers the tile");
  static_assert(BM % (32 * WM) == 0 && BN % (32 * WN) == 0 && BN % LMH_BN == 0, "tile shape");
  static_assert((NS - 1) * LPW < 64, "the load counter holds 63");
  __device__ __forceinline__ static int xperm(int row) { return XC >= 8 ? (row & 7) : ((row >> 1) & 3); }
  __device__ __forceinline__ static int wperm(int row) { return (row >> 1) & 3; }
};
template <typename T, int ES>
constexpr int m4_lds_bytes() {
  return T::NS * T::STAGE > lmh_epi_bytes<T, ES>() ? T::NS * T::STAGE : lmh_epi_bytes<T, ES>();
}

#ifndef LPS_HOST_EMU
// 4 bytes per lane from g to LDS at (wave-uniform) base + 4 * lane.
__device__ __forceinline__ void lmh_dma4(const char* g, char* base) {
  const uint32_t m0 = (uint32_t)__builtin_amdgcn_readfirstlane(
      (int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)base);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(m0), "v"(g) : "memory", "m0");
}
#else
inline void lmh_dma4(const char* g, char* base) { memcpy(base + 4 * ((int)threadIdx.x & 63), g, 4); }
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

// The accumulators plus one stage of NB blocks.
template <int XDT, typename T, typename ACC>
__device__ __forceinline__ void m4_stage(const char* stage, ACC (&acc)[T::MT][T::CT], int wm, int wn, int l, int steps) {
  constexpr int MT = T::MT, CT = T::CT;
  const int half = l >> 5;
  const int xr = wm * (MT * 32) + (l & 31), wr = wn * T::WTN + (l & 31);
  const int px = T::xperm(xr), pw = T::wperm(wr);   // (rows 32 apart share it)
  const char* wb = stage + T::XBYTES;
  const uint32_t* ws = reinterpret_cast<const uint32_t*>(wb + T::WBYTES);
  uint32_t sw[CT];
#pragma unroll
  for (int i = 0; i < CT; i++) sw[i] = ws[wr + 32 * i];
  if constexpr (T::XS) {
    const uint32_t* xs = ws + T::BN;
    uint32_t sx[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) sx[i] = xs[xr + 32 * i] >> (8 * half);
#pragma unroll
    for (int i = 0; i < CT; i++) sw[i] >>= 8 * half;
#pragma unroll
    for (int j = 0; j < T::KS; j++) {
      if (j >= steps) break;
      typedef int i32x8 __attribute__((ext_vector_type(8)));
      const int c = 2 * j + half;
      u32x4 fx[MT], fw[CT];
#pragma unroll
      for (int i = 0; i < MT; i++) fx[i] = *reinterpret_cast<const u32x4*>(stage + ((xr + 32 * i) * T::XC + (c ^ px)) * 16);
#pragma unroll
      for (int i = 0; i < CT; i++) fw[i] = *reinterpret_cast<const u32x4*>(wb + ((wr + 32 * i) * T::WC + (c ^ pw)) * 16);
#pragma unroll
      for (int a = 0; a < MT; a++)
#pragma unroll
        for (int b = 0; b < CT; b++) {
          const i32x8 A = {(int)fx[a].x, (int)fx[a].y, (int)fx[a].z, (int)fx[a].w, 0, 0, 0, 0};
          const i32x8 B = {(int)fw[b].x, (int)fw[b].y, (int)fw[b].z, (int)fw[b].w, 0, 0, 0, 0};
          if (j == 0)
            acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, acc[a][b], 4, 4, 0, (int)sx[a], 0, (int)sw[b]);
          else
            acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, acc[a][b], 4, 4, 2, (int)sx[a], 2, (int)sw[b]);
        }
    }
  } else {
    bool far = false;
    if constexpr (XDT == LPS_DTYPE_F16) {
#pragma unroll
      for (int i = 0; i < CT; i++) far = far || m4_far_scale(sw[i]);
      far = wballot(far) != 0;
    }
#pragma unroll
    for (int j = 0; j < T::KS; j++) {
      if (j >= steps) break;
      const int c = 2 * j + half;
      u32x4 cw[CT];
      float s[CT];
#pragma unroll
      for (int i = 0; i < CT; i++) {
        cw[i] = *reinterpret_cast<const u32x4*>(wb + ((wr + 32 * i) * T::WC + (c ^ pw)) * 16);
        s[i] = __uint_as_float(((sw[i] >> (8 * c)) & 255u) << 23);
      }
      auto step = [&](auto far_c) {
        constexpr bool FAR = decltype(far_c)::value;
#pragma unroll
        for (int q = 0; q < 4; q++) {
          u32x4 fx[MT];
#pragma unroll
          for (int i = 0; i < MT; i++)
            fx[i] = *reinterpret_cast<const u32x4*>(stage + ((xr + 32 * i) * T::XC + ((4 * c + q) ^ px)) * 16);
          if constexpr (!FAR) {
#pragma unroll
            for (int b = 0; b < CT; b++) {
              const u32x4 fw = m4_frag<XDT>(cw[b][q], s[b]);
#pragma unroll
              for (int a = 0; a < MT; a++) acc[a][b] = MfmaOps<XDT>::mma(fx[a], fw, acc[a][b]);
            }
          } else {
#pragma unroll
            for (int a = 0; a < MT; a++) {
              u32x4 hi, lo;
              m4_split(fx[a], hi, lo);
#pragma unroll
              for (int b = 0; b < CT; b++) {
                const u32x4 fw = m4_frag<LPS_DTYPE_BF16>(cw[b][q], s[b]);
                acc[a][b] = MfmaOps<LPS_DTYPE_BF16>::mma(hi, fw, acc[a][b]);
                acc[a][b] = MfmaOps<LPS_DTYPE_BF16>::mma(lo, fw, acc[a][b]);
              }
            }
          }
        }
      };
      if (XDT == LPS_DTYPE_F16 && far) step(std::true_type{});
      else step(std::false_type{});
    }
  }
}

// XDT: BF16, F16 or MX4; T::XB 64 or 16 accordingly.
template <int XDT, int ODT, typename T, bool NTL>
__global__ __launch_bounds__(T::NT, T::WPE) void mx4head_kernel(Mx4HeadParams Q) {
  constexpr int ES = ODT == LPS_DTYPE_F32 ? 4 : 2;
  constexpr int ADT = XDT == LPS_DTYPE_F16 ? LPS_DTYPE_F16 : LPS_DTYPE_BF16;   // (the accumulators are alike)
  constexpr int MT = T::MT, CT = T::CT, NB = T::NB;
  __shared__ __attribute__((aligned(1024))) char lds[m4_lds_bytes<T, ES>()];
  const LmHeadParams& P = Q.h;
  // tiles over the XCDs as in lmhead_kernel: a run each, the row tiles of one column tile first
  const int per = (P.tiles + 7) >> 3;
  const int t = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
  if (((int)blockIdx.x >> 3) >= per || t >= P.tiles) return;   // uniform over the workgroup
  const int m0 = (t % P.mtiles) * T::BM, n0 = (t / P.mtiles) * T::BN;
  const int wv = (int)threadIdx.x >> 6, l = (int)threadIdx.x & 63;
  const int wm = wv / T::WN, wn = wv % T::WN;
  auto mrow = [&](int r) { const int m = m0 + r; return (int64_t)(m < P.M ? m : P.M - 1); };
  auto nrow = [&](int r) { const int n = n0 + r; return (int64_t)(n < P.V ? n : P.V - 1); };
  const char* const X = reinterpret_cast<const char*>(P.x);
  const char* const W = reinterpret_cast<const char*>(P.w);
  const int64_t xstep = T::XS ? P.x_stride : 2 * P.x_stride;   // bytes of a row of x

  // sources of this lane's chunks (rows clamped into range; their results are dropped)
  const char* xsrc[T::XPW];
  const char* wsrc[T::WPW];
#pragma unroll
  for (int i = 0; i < T::XPW; i++) {
    const int row = ((i * T::NW + wv) % T::XI) * T::XRI + l / T::XC, c = (l % T::XC) ^ T::xperm(row);
    xsrc[i] = X + mrow(row) * xstep + c * 16;
  }
#pragma unroll
  for (int i = 0; i < T::WPW; i++) {
    const int row = (i * T::NW + wv) * T::WRI + l / T::WC, c = (l % T::WC) ^ T::wperm(row);
    wsrc[i] = W + nrow(row) * P.w_stride + c * 16;
  }
  // (with more waves than groups of 64 rows some load the same scales)
  const int sg = wv % (T::BN / 64), xg = wv % (T::SMR / 64);
  const char* ssrc = reinterpret_cast<const char*>(Q.ws) + nrow(64 * sg + l) * Q.ws_stride;
  const char* xssrc = T::XS ? reinterpret_cast<const char*>(Q.xs) + mrow(64 * xg + l) * Q.xs_stride : nullptr;
  auto issue = [&](int buf) {   // the next stage into ring buffer buf
    char* base = lds + buf * T::STAGE;
#pragma unroll
    for (int i = 0; i < T::XPW; i++) {
      lmh_dma16<false>(xsrc[i], base + ((i * T::NW + wv) % T::XI) * 1024);
      xsrc[i] += NB * T::XB;
    }
    base += T::XBYTES;
#pragma unroll
    for (int i = 0; i < T::WPW; i++) {
      lmh_dma16<NTL>(wsrc[i], base + (i * T::NW + wv) * 1024);
      wsrc[i] += NB * 16;
    }
    base += T::WBYTES;
    lmh_dma4(ssrc, base + sg * 256);
    ssrc += NB;
    if constexpr (T::XS) {
      lmh_dma4(xssrc, base + T::BN * 4 + xg * 256);
      xssrc += NB;
    }
  };

  typename MfmaOps<ADT>::acc acc[MT][CT] = {};
  const int ns = P.H / (32 * NB);   // whole stages of whole blocks; the rest of H follows them
  for (int s = 0; s < T::NS - 1 && s < ns; s++) issue(s);
  int buf = 0;
  for (int s = 0; s < ns; s++) {
    // stage s has landed, and every wave is done with stage s - 1
    lmh_wait_stage<T>(ns - 1 - s);
    if (s + T::NS - 1 < ns) issue(buf == 0 ? T::NS - 1 : buf - 1);
    m4_stage<XDT, T>(lds + buf * T::STAGE, acc, wm, wn, l, T::KS);
    buf = buf + 1 == T::NS ? 0 : buf + 1;
  }
  lmh_wait_barrier<0>();
  const int k0 = ns * 32 * NB;
  if (k0 < P.H) {
    // the columns past the last whole stage, zeros up to one (with scales of 1)
    const int nb = (P.H + 31) >> 5, b0 = ns * NB;
    for (int i = threadIdx.x; i < T::BM * T::XC; i += T::NT) {
      const int row = i / T::XC, c = (i % T::XC) ^ T::xperm(row);
      u32x4 v = {0u, 0u, 0u, 0u};
      if constexpr (T::XS) {
        if (b0 + c < nb) v = *reinterpret_cast<const u32x4*>(X + mrow(row) * xstep + (b0 + c) * 16);
      } else {
        const int e0 = k0 + 8 * c;
        if (e0 < P.H) v = load_piece<ADT>(X + mrow(row) * xstep, e0, P.H).q[0];
      }
      *reinterpret_cast<u32x4*>(lds + i * 16) = v;
    }
    char* wb = lds + T::XBYTES;
    for (int i = threadIdx.x; i < T::BN * T::WC; i += T::NT) {
      const int row = i / T::WC, b = b0 + ((i % T::WC) ^ T::wperm(row));
      u32x4 v = {0u, 0u, 0u, 0u};
      if (b < nb) {
        v = *reinterpret_cast<const u32x4*>(W + nrow(row) * P.w_stride + b * 16);
#pragma unroll
        for (int e = 0; e < 4; e++) {               // (codes past the row's end count as zeros, whatever they hold)
          const int keep = P.H - 32 * b - 8 * e;
          v[e] = keep >= 8 ? v[e] : keep <= 0 ? 0u : v[e] & ((1u << (4 * keep)) - 1u);
        }
      }
      *reinterpret_cast<u32x4*>(wb + i * 16) = v;
    }
    uint8_t* sb = reinterpret_cast<uint8_t*>(wb + T::WBYTES);
    for (int i = threadIdx.x; i < T::BN * NB; i += T::NT)
      sb[i] = b0 + i % NB < nb ? Q.ws[nrow(i / NB) * Q.ws_stride + b0 + i % NB] : 127;
    if constexpr (T::XS)
      for (int i = threadIdx.x; i < T::BM * NB; i += T::NT)
        sb[T::BN * 4 + i] = b0 + i % NB < nb ? Q.xs[mrow(i / NB) * Q.xs_stride + b0 + i % NB] : 127;
    __syncthreads();
    m4_stage<XDT, T>(lds, acc, wm, wn, l, (nb - b0 + 1) / 2);
    __syncthreads();
  }
  lmh_epilogue<ADT, ODT, T>(P, lds, acc, n0, m0, wv, l);
}

}  // namespace lps
