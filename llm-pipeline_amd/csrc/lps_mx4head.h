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
// scale a lane.  bf16 holds every value of w that fp32 does.  fp16 holds those of scales 2^-23 ..
// 2^13; a stage in which a wave meets another scale takes x apart into two bf16
// (11 bits as 8 and 3) and runs the bf16 instruction twice, which is exact too.
//
// What bounds it: up to ~32 rows w's pass over HBM (1 row of 4096 -> 151936: 58 us, 5.7
// TB/s; a read reaches 7.0), from ~128 rows of 16 bits the matrix cores (2048 rows 2.15
// ms, 1.19 PFLOP/s; the library's bf16 product takes 2.10) and from ~256 of 4 bits they
// and the writing of the logits (2048 rows 768 us, 3.3 PFLOP/s).  Between them (64 rows
// of 16 bits 101 us) stages of x and w wait for each other's latency: two workgroups of
// 72 KB LDS on a CU are worth more than a deeper ring in one (64 x 128 tiles with 5
// stages of w ahead 120 us; 64 x 256 tiles 111), and so are x held in registers with w
// streamed past it (155) and a stage read whole into registers, a stage ahead (101).
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

// One workgroup of WM x WN x KW waves computes a BM x BN tile; the KW groups of waves
// take turns at K, two blocks at a time, and add their accumulators at the end.  x
// and w stream into LDS rings of their own by loads that cost no registers
// (lps_lmhead.h): w in NSW stages of 8 blocks, x in NSX stages of XNB.  The first
// NXW waves load x, the others w and the scales: a wave's loads land in their
// order, so that one which loads both could not wait for x (soon there, from the
// caches) without waiting for the w stages ahead of it.
// - Rows of w are read in whole lines of 128 bytes (8 blocks): reads of 64 bytes
//   reach 3.5 TB/s of HBM here, of 128 bytes 7.0 (28 and 55 bytes a clock and CU
//   out of the L2), of 16 bytes 0.9.
// - Scales, a byte to 16 of codes, come 32 blocks at a time into two buffers: read
//   by the stage they cost more than a third of the time (2048 x 4096 -> 151936 in
//   4 bits 1112 us, 732 without them).
// A stage's row r keeps its 16-byte chunk c at place c ^ f(r).  Of x, XR rows are
// held (row r stands in for r + XR, ..: results that are dropped).  XB: bytes of a
// block of x, 64 or 16.
constexpr int M4_NB = 8;
constexpr int M4_SB = 32;
constexpr int M4_PER = M4_SB / M4_NB;
constexpr int64_t M4_MAX_STRIDE = 1 << 23;   // bytes: 256 rows of it fit 32-bit offsets
template <int BM_, int BN_, int WM_, int WN_, int KW_, int XNB_, int NSX_, int NSW_, int NXW_, int WPE_, int XB_, int XR_ = BM_>
struct M4Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, KW = KW_, XNB = XNB_, NSX = NSX_, NSW = NSW_;
  static constexpr int NXW = NXW_, WPE = WPE_, XB = XB_, XR = XR_;
  static constexpr int EW = WM * WN;                            // waves of one group (the epilogue's)
  static constexpr int NWK = EW * KW, NTK = 64 * NWK, NWW = NWK - NXW;
  static constexpr int MT = BM / WM / 32, CT = BN / WN / 32;    // accumulators per wave: rows x columns
  static constexpr int WTN = 32 * CT;
  static constexpr int XC = XNB * XB / 16, WC = M4_NB;          // 16-byte chunks per row
  static constexpr int XRI = 64 / XC, WRI = 64 / WC;            // rows a wave's load instruction covers
  static constexpr int XI = XR / XRI, WI = BN / WRI;            // load instructions of a stage
  static constexpr int XPW = (XI + NXW - 1) / NXW, WPW = WI / NWW;   // ... of a wave (with more waves than XI some load the same)
  static constexpr bool XS = XB == 16;
  static constexpr int SROWS = BN + (XS ? XR : 0);              // rows with scales: w's, then x's
  static constexpr int XBYTES = XR * XC * 16, WBYTES = BN * WC * 16, SBYTES = SROWS * M4_SB;
  static constexpr int WOFF = NSX * XBYTES, SOFF = WOFF + NSW * WBYTES, BYTES = SOFF + 2 * SBYTES;
  static constexpr int ITS = M4_NB / XNB;                       // x stages to one of w
  static constexpr int JS = XNB / 2 / KW;                       // pairs of blocks of a wave per x stage
  static_assert(XNB == 4 || XNB == 8, "x stages");
  static_assert((XI % NXW == 0 || NXW % XI == 0) && WI % NWW == 0 && NXW < NWK, "whole load instructions per wave");
  static_assert(SROWS % 32 == 0 && XR % 8 == 0 && BM % XR == 0, "whole loads of scales");
  static_assert(BM % (32 * WM) == 0 && BN % (32 * WN) == 0 && BN % LMH_BN == 0 && JS >= 1, "tile shape");
  static_assert(M4_PER >= NSW - 1, "scales are asked for before the stage that needs them");
  static_assert((NSW - 1) * WPW + SROWS / 8 / NWW + 1 < 64 && (NSX - 1) * XPW < 64, "the load counter holds 63");
  // (the 64 banks hold 16 chunks: those that 16 neighbouring rows read at once lie in
  // places of their own; of 128-byte rows two share the banks)
  __device__ __forceinline__ static int xperm(int row) { return XC >= 16 ? (row & 15) : ((row >> 1) & 7); }
  __device__ __forceinline__ static int wperm(int row) { return (row >> 1) & 7; }
};
// The waves that write a tile out, as lmh_epilogue sees them.
template <typename T>
struct M4Epi {
  static constexpr int BM = T::BM, BN = T::BN, WM = T::WM, WN = T::WN, MT = T::MT, CT = T::CT, WTN = T::WTN;
  static constexpr int NW = T::EW, NT = 64 * T::EW;
};
template <typename T, int ES>
constexpr int m4_lds_bytes() {
  constexpr int epi = lmh_epi_bytes<M4Epi<T>, ES>();
  return T::BYTES > epi ? T::BYTES : epi;
}

#ifndef LPS_HOST_EMU
// Byte address in LDS of a shared array.
__device__ __forceinline__ uint32_t m4_lds(const char* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}
// 16 / 4 bytes per lane from base + off (base uniform) to LDS at (uniform) dst + 16 /
// 4 * lane.  The compiler does not see a load here: five wait states stand between
// it and a vector instruction that may have written base just before (a reload of
// a spilled scalar register).
template <bool NTL>
__device__ __forceinline__ void m4_dma16(const char* base, uint32_t off, uint32_t dst) {
  dst = (uint32_t)__builtin_amdgcn_readfirstlane((int)dst);
  if constexpr (NTL)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(dst), "v"(off), "s"(base) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void m4_dma4(const char* base, uint32_t off, uint32_t dst) {
  dst = (uint32_t)__builtin_amdgcn_readfirstlane((int)dst);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2" ::"s"(dst), "v"(off), "s"(base) : "memory", "m0");
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
#ifndef LPS_HOST_EMU
template <int N>
__device__ __forceinline__ void m4_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void m4_barrier() {   // this wave's LDS reads are done, then every wave's
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
#else
template <int N>
inline void m4_wait() {}
inline void m4_barrier() { __syncthreads(); }
#endif
// Until at most `left` stages of PW loads each are in flight (left <= MAX).
template <int PW, int MAX>
__device__ __forceinline__ void m4_wait_left(int left) {
  if constexpr (MAX == 0) m4_wait<0>();
  else if (left >= MAX) m4_wait<MAX * PW>();
  else m4_wait_left<PW, MAX - 1>(left);
}

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

// Eight fp16 as two bf16 fragments whose sum they are: the top 8 bits of each (cut
// off) and the rest (at most 3 bits, exact).  Where nothing is left, infinities and
// NaN among them, two halves: a weight past fp32's range is an infinity, and a zero
// times it would be NaN.
__device__ __forceinline__ void m4_split(u32x4 x, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint32_t h[2], r[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const float f = f16_to_f32((x[i] >> (16 * e)) & 0xFFFFu);
      const uint32_t top = __float_as_uint(f) & 0xFFFF0000u, half = __float_as_uint(__fmul_rn(0.5f, f)) & 0xFFFF0000u;
      const float rest = __fsub_rn(f, __uint_as_float(top));
      const bool some = (top & 0x7F800000u) != 0x7F800000u && rest != 0.0f;
      h[e] = some ? top : half;
      r[e] = some ? __float_as_uint(rest) : half;
    }
    hi[i] = (h[0] >> 16) | h[1];
    lo[i] = (r[0] >> 16) | (r[1] & 0xFFFF0000u);
  }
}

// Nonzero when any of four scale bytes is outside 104 .. 140 (2^-23 .. 2^13): of a byte
// under 128, 24 more must reach 128, of the low 7 bits of another 115 more must not.
__device__ __forceinline__ uint32_t m4_far_scale(uint32_t w) {
  const uint32_t low = (w & 0x7F7F7F7Fu) + 0x18181818u, high = (w & 0x7F7F7F7Fu) + 0x73737373u;
  return ((~w & ~low) | (w & high)) & 0x80808080u;
}

// The position of a lane in a tile, and its reads of the stages.  A stage's chunks
// of w and its scales are those of its 8 blocks.
template <typename T>
struct M4Lane {
  int half, kg, xr, wr, px, pw;
  __device__ __forceinline__ M4Lane(int wv, int l) {
    const int e = wv % T::EW;
    half = l >> 5;
    kg = wv / T::EW;
    xr = (e / T::WN) * (T::MT * 32) + (l & 31);
    wr = (e % T::WN) * T::WTN + (l & 31);
    px = T::xperm(xr % T::XR);      // (rows 32 apart share it)
    pw = T::wperm(wr);
  }
  __device__ __forceinline__ u32x4 x(const char* xs, int i, int c) const {
    return *reinterpret_cast<const u32x4*>(xs + ((xr + 32 * i) % T::XR * T::XC + (c ^ px)) * 16);
  }
  __device__ __forceinline__ u32x4 w(const char* ws, int i, int c) const {
    return *reinterpret_cast<const u32x4*>(ws + ((wr + 32 * i) * T::WC + (c ^ pw)) * 16);
  }
  // four blocks' scales of a row
  __device__ __forceinline__ uint32_t wscales(const char* scales, int i, int d) const {
    return *reinterpret_cast<const uint32_t*>(scales + (wr + 32 * i) * M4_SB + 4 * d);
  }
  __device__ __forceinline__ uint32_t xscales(const char* scales, int i, int d) const {
    return *reinterpret_cast<const uint32_t*>(scales + (T::BN + (xr + 32 * i) % T::XR) * M4_SB + 4 * d);
  }
};

// A byte of a word of scales (0, or with odd j 2) as the conversions' scale: its
// neighbours land in the sign and the mantissa, which they ignore.
__device__ __forceinline__ float m4_scale(uint32_t w, int j) { return __uint_as_float((j & 1) ? w << 7 : w << 23); }

typedef int i32x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ i32x8 m4_operand(u32x4 v) { return i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0}; }
template <typename ACC>
__device__ __forceinline__ ACC m4_mma4(u32x4 a, u32x4 b, ACC c, uint32_t sa, uint32_t sb, int j) {
  if (j & 1) return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(m4_operand(a), m4_operand(b), c, 4, 4, 2, (int)sa, 2, (int)sb);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(m4_operand(a), m4_operand(b), c, 4, 4, 0, (int)sa, 0, (int)sb);
}

// The accumulators plus the wave's share of `pairs` pairs of blocks, one after
// another: the last columns of a row, and (FAR) stages of fp16 with scales that it
// does not hold.  w0: the first pair's first block in the w stage.
template <int XDT, typename T, bool FAR, typename ACC>
__device__ __forceinline__ void m4_plain_stage(const char* xs, const char* ws, int w0, const char* scales, const M4Lane<T>& L,
                                               ACC (&acc)[T::MT][T::CT], int pairs) {
#pragma unroll 1
  for (int p = L.kg; p < pairs; p += T::KW) {
    const int c = 2 * p + L.half;
#pragma unroll
    for (int b = 0; b < T::CT; b++) {
      const u32x4 cw = L.w(ws, b, w0 + c);
      const uint32_t byte = (L.wscales(scales, b, (w0 + c) >> 2) >> (8 * ((w0 + c) & 3))) & 255u;
      if constexpr (T::XS) {
#pragma unroll
        for (int a = 0; a < T::MT; a++)
          acc[a][b] = m4_mma4(L.x(xs, a, c), cw, acc[a][b], L.xscales(scales, a, (w0 + c) >> 2) >> (8 * ((w0 + c) & 3)), byte, 0);
      } else {
        const float s = __uint_as_float(byte << 23);
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const u32x4 fw = m4_frag<FAR ? LPS_DTYPE_BF16 : XDT>(cw[q], s);
#pragma unroll
          for (int a = 0; a < T::MT; a++) {
            const u32x4 fx = L.x(xs, a, 4 * c + q);
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
__global__ __launch_bounds__(T::NTK, T::WPE) void mx4head_kernel(Mx4HeadParams Q) {
  constexpr int ES = ODT == LPS_DTYPE_F32 ? 4 : 2;
  constexpr int ADT = XDT == LPS_DTYPE_F16 ? LPS_DTYPE_F16 : LPS_DTYPE_BF16;   // (the accumulators are alike)
  constexpr int MT = T::MT, CT = T::CT, NB = M4_NB, XNB = T::XNB, KW = T::KW, JS = T::JS;
  __shared__ __attribute__((aligned(1024))) char lds[m4_lds_bytes<T, ES>()];
  const LmHeadParams& P = Q.h;
  // tiles over the XCDs as in lmhead_kernel: a run each, the row tiles of one column tile first
  const int per = (P.tiles + 7) >> 3;
  const int t = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
  if (((int)blockIdx.x >> 3) >= per || t >= P.tiles) return;   // uniform over the workgroup
  const int m0 = (t % P.mtiles) * T::BM, n0 = (t / P.mtiles) * T::BN;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), l = (int)threadIdx.x & 63;
  const bool loads_x = wv < T::NXW;
  const int lw = loads_x ? wv : wv - T::NXW;                   // among the waves that load the same
  const int64_t xstep = T::XS ? P.x_stride : 2 * P.x_stride;   // bytes of a row of x
  const char* const X = reinterpret_cast<const char*>(P.x) + (int64_t)m0 * xstep;
  const char* const W = reinterpret_cast<const char*>(P.w) + (int64_t)n0 * P.w_stride;
  // rows of the tile, clamped into range (the others' results are dropped); their
  // offsets in it fit 32 bits (M4_MAX_STRIDE)
  auto mrow = [&](int r) { return m0 + r < P.M ? r : P.M - 1 - m0; };
  auto nrow = [&](int r) { return n0 + r < P.V ? r : P.V - 1 - n0; };

  // offsets of this lane's chunk of the k-th row that its wave loads, rl + k R, clamped
  // to the last row
  constexpr int RX = T::NXW * T::XRI, RW = T::NWW * T::WRI, LPM = T::XPW > T::WPW ? T::XPW : T::WPW;
  constexpr bool KEEP = !(T::XS && MT * CT >= 8);   // (beside 128 accumulators computed when they are needed)
  static_assert(KEEP || (RX % 16 == 0 && RW % 16 == 0), "there the rows share their chunk's place");
  const int rl = loads_x ? lw % T::XI * T::XRI + l / T::XC : lw * T::WRI + l / T::WC;
  const uint32_t rstep = loads_x ? (uint32_t)xstep : (uint32_t)P.w_stride;
  const uint32_t rlast = (uint32_t)(loads_x ? mrow(T::XR - 1) : nrow(T::BN - 1)) * rstep;
  const uint32_t roff = (uint32_t)rl * rstep;
  auto chunk = [&](int row) { return (uint32_t)(loads_x ? (l % T::XC) ^ T::xperm(row) : (l % T::WC) ^ T::wperm(row)) * 16u; };
  auto compute = [&](int k) {
    uint32_t o = roff;
    if constexpr (!KEEP) LPS_KEEP_VGPR(o);
    o += (uint32_t)k * rstep * (uint32_t)(loads_x ? RX : RW);
    return (o < rlast ? o : rlast) + chunk(KEEP ? rl + k * (loads_x ? RX : RW) : rl);
  };
  uint32_t offs[KEEP ? LPM : 1];
  if constexpr (KEEP) {
#pragma unroll
    for (int k = 0; k < LPM; k++) offs[k] = compute(k);
  }
  auto off = [&](int k) {
    if constexpr (KEEP) return offs[k];
    else return compute(k);
  };
  const auto lds0 = m4_lds(lds);
  auto issue_x = [&](int i, int slot) {
    const char* base = X + (int64_t)i * (XNB * T::XB);
#pragma unroll
    for (int k = 0; k < T::XPW; k++)
      m4_dma16<false>(base, off(k), lds0 + slot * T::XBYTES + ((k * T::NXW + lw) % T::XI) * 1024);
  };
  auto issue_w = [&](int s, int slot) {
    const char* base = W + (int64_t)s * (NB * 16);
#pragma unroll
    for (int k = 0; k < T::WPW; k++)
      m4_dma16<NTL>(base, off(k), lds0 + T::WOFF + slot * T::WBYTES + (k * T::NWW + lw) * 1024);
  };
  const int ns = P.H / (32 * NB), its = ns * T::ITS;   // whole stages of whole blocks; the rest of H follows them
  // scales of blocks 32 u .. +31, as far as the whole stages go: a row's 32 bytes
  // by two lanes, or by eight where it does not lie on 16-byte lines
  const char* const WS = reinterpret_cast<const char*>(Q.ws) + (int64_t)n0 * Q.ws_stride;
  const char* const XSC = T::XS ? reinterpret_cast<const char*>(Q.xs) + (int64_t)m0 * Q.xs_stride : nullptr;
  auto issue_scales = [&](int u) {
    const auto d = lds0 + T::SOFF + (u & 1) * T::SBYTES;
    const int rl = Q.wide ? 32 : 8, groups = T::SROWS / rl, r0 = Q.wide ? l >> 1 : l >> 3;
    int b = M4_SB * u + (Q.wide ? 16 * (l & 1) : 4 * (l & 7));
    b = b < NB * ns ? b : 0;          // (a row without them: others of its own)
    for (int i = lw; i < groups; i += T::NWW) {
      const bool ofx = T::XS && rl * i >= T::BN;
      const char* base = ofx ? XSC : WS;
      const uint32_t o = (ofx ? (uint32_t)mrow(rl * i + r0 - T::BN) * (uint32_t)Q.xs_stride
                              : (uint32_t)nrow(rl * i + r0) * (uint32_t)Q.ws_stride) + b;
      if (Q.wide) m4_dma16<false>(base, o, d + i * 1024);
      else m4_dma4(base, o, d + i * 256);
    }
  };

  typename MfmaOps<ADT>::acc acc[MT][CT] = {};
  const M4Lane<T> L(wv, l);
  constexpr int STEPS = T::XS ? JS : 4 * JS;       // matrix steps of a wave in an x stage (64 or 16 values)
  constexpr int WDS = T::XS ? 1 : XNB / 4;         // words of scales that are held
  u32x4 fx[2][MT], cw[2][CT], fw[2][CT];
  uint32_t sw[WDS][CT], sx[MT];
  // pair jj of a wave is pair jj KW + kg of the stage: word and (after the shift)
  // byte of its scales
  auto word = [](int jj) { return KW == 2 ? jj : jj >> 1; };
  auto odd = [](int jj) { return KW == 2 ? 0 : jj & 1; };
  const int shift = 8 * L.half + (KW == 2 ? 16 * L.kg : 0);
  uint32_t far_any = 0;                            // fp16: whether this lane met a scale that it does not hold
  auto read_word = [&](const char* scales, int d, int to) {
#pragma unroll
    for (int i = 0; i < CT; i++) {
      const uint32_t w = L.wscales(scales, i, d);
      if constexpr (XDT == LPS_DTYPE_F16) far_any |= m4_far_scale(w);
      sw[to][i] = w >> shift;
    }
    if constexpr (T::XS) {
#pragma unroll
      for (int i = 0; i < MT; i++) sx[i] = L.xscales(scales, i, d) >> shift;
    }
  };
  auto read_scales = [&](const char* scales, int w0) {
    far_any = 0;
#pragma unroll
    for (int d = 0; d < WDS; d++) read_word(scales, (w0 >> 2) + d, d);
  };
  // (b: the buffer of registers)
  auto read_x = [&](const char* xs, int k, int b) {   // for matrix step k
    const int blk = 2 * ((T::XS ? k : k >> 2) * KW + L.kg) + L.half, c = T::XS ? blk : 4 * blk + (k & 3);
#pragma unroll
    for (int i = 0; i < MT; i++) fx[b][i] = L.x(xs, i, c);
  };
  auto read_w = [&](const char* ws, int w0, int jj, int b) {   // for the wave's pair jj
#pragma unroll
    for (int i = 0; i < CT; i++) cw[b][i] = L.w(ws, i, w0 + 2 * (jj * KW + L.kg) + L.half);
  };
  auto convert = [&](int k, int b, int fb) {
    if constexpr (!T::XS) {
      const int jj = k >> 2;
#pragma unroll
      for (int i = 0; i < CT; i++) fw[fb][i] = m4_frag<XDT>(cw[b][i][k & 3], m4_scale(sw[word(jj)][i], odd(jj)));
    }
  };
  auto xslot = [&](int slot) { return lds + slot * T::XBYTES; };
  auto wslot = [&](int slot) { return lds + T::WOFF + slot * T::WBYTES; };
  auto scales_of = [&](int s) { return lds + T::SOFF + ((s / M4_PER) & 1) * T::SBYTES + (s % M4_PER) * NB; };
  if (ns > 0) {
    if (loads_x) {
      for (int i = 0; i < T::NSX && i < its; i++) issue_x(i, i);
    } else {
      issue_scales(0);
      for (int s = 0; s < T::NSW && s < ns; s++) issue_w(s, s);
    }
    int xb = 0, wb = 0;                            // the places of x stage i and of its w stage
    // until x stage i (and the w stage that it begins, and its scales, asked for before
    // it) has landed, with up to MORE stages after it in flight, for every wave
    auto wait_stage = [&](int i, auto more_c) {
      constexpr int MORE = decltype(more_c)::value;
      if (loads_x) m4_wait_left<T::XPW, T::NSX - MORE>(its - 1 - i);
      else if (i % T::ITS == 0) m4_wait_left<T::WPW, T::NSW - MORE>(ns - 1 - i / T::ITS);
      m4_barrier();
    };
    // every wave is done with x stage i: the next ones into its places
    auto refill = [&](int i, int xplace, int wplace) {
      if (loads_x) {
        if (i + T::NSX < its) issue_x(i + T::NSX, xplace);
      } else if ((i + 1) % T::ITS == 0) {
        const int s = i / T::ITS;
        if (s % M4_PER == 0 && s + M4_PER < ns) issue_scales(s / M4_PER + 1);
        if (s + T::NSW < ns) issue_w(s + T::NSW, wplace);
      }
    };
    constexpr std::integral_constant<int, 1> first{};   // (the ring is full)
    constexpr std::integral_constant<int, 2> later{};   // (but for the stage that has just been read)
    if constexpr (T::XS) {
      // A step reads its own fragments; the compiler moves the next ones' reads up among
      // its matrix instructions as registers allow.
      for (int i = 0; i < its; i++) {
        if (i == 0) wait_stage(0, first);
        else wait_stage(i, later);
        if (i > 0) refill(i - 1, xb == 0 ? T::NSX - 1 : xb - 1, wb == 0 ? T::NSW - 1 : wb - 1);
        const char* const xs = xslot(xb);
        const char* const ws = wslot(wb);
        static_assert(!T::XS || T::ITS == 1, "4-bit x: a w stage to an x stage");
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
          read_w(ws, 0, k, 0);
          read_x(xs, k, 0);
          if (!odd(k)) read_word(scales_of(i), word(k), 0);
#pragma unroll
          for (int a = 0; a < MT; a++)
#pragma unroll
            for (int b = 0; b < CT; b++) acc[a][b] = m4_mma4(fx[0][a], cw[0][b], acc[a][b], sx[a], sw[0][b], odd(k));
        }
        xb = xb + 1 == T::NSX ? 0 : xb + 1;
        wb = wb + 1 == T::NSW ? 0 : wb + 1;
      }
    } else {
      // Fragments are read one step ahead of their matrix instructions and the codes
      // converted one ahead, in the shadow of the matrix cores; the last step of a stage
      // waits for the next one and reads its first.  (With all of a stage read at once, a
      // stage ahead: 8 rows 74 us for 59, 64 rows 101 for 101.)
      wait_stage(0, first);
      read_scales(scales_of(0), 0);
      read_w(wslot(0), 0, 0, 0);
      read_x(xslot(0), 0, 0);
      convert(0, 0, 0);
      // (an odd number of pairs a stage: the buffers of codes swap from stage to stage)
      auto stage = [&](int i, auto par_c) {
        constexpr int PAR = decltype(par_c)::value;  // the buffer of the stage's first codes
        const int w0 = (i % T::ITS) * XNB, s = i / T::ITS;
        const char* const xs = xslot(xb);
        const char* const ws = wslot(wb);
        const bool far = XDT == LPS_DTYPE_F16 && wballot(far_any != 0) != 0;   // (uniform over the wave)
        if constexpr (XDT == LPS_DTYPE_F16)
          if (far) m4_plain_stage<XDT, T, true>(xs, ws, w0, scales_of(s), L, acc, XNB / 2);
        const int nxb = xb + 1 == T::NSX ? 0 : xb + 1;
        const int nwb = (i + 1) % T::ITS != 0 ? wb : wb + 1 == T::NSW ? 0 : wb + 1;
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
          const int jj = k >> 2;
          const int fb = k & 1, fn = fb ^ 1;         // fragments of this step, the next one's
          const int cb = (jj + PAR) & 1, cn = cb ^ 1;   // codes of this pair, the next one's
          if (k + 1 < STEPS) {
            if (far) continue;
            if ((k & 3) == 1 && jj + 1 < JS) read_w(ws, w0, jj + 1, cn);
            read_x(xs, k + 1, fn);
          } else if (i + 1 < its) {
            // (every wave holds its last fragments of the stage)
            wait_stage(i + 1, later);
            refill(i, xb, wb);
            read_scales(scales_of((i + 1) / T::ITS), (i + 1) % T::ITS * XNB);
            read_w(wslot(nwb), ((i + 1) % T::ITS) * XNB, 0, cn);
            read_x(xslot(nxb), 0, fn);
          }
          __builtin_amdgcn_sched_barrier(0);   // (the compiler would move the reads down to their use)
          if (!far) {
#pragma unroll
            for (int a = 0; a < MT; a++)
#pragma unroll
              for (int b = 0; b < CT; b++) acc[a][b] = MfmaOps<ADT>::mma(fx[fb][a], fw[fb][b], acc[a][b]);
          }
          if (k + 1 < STEPS) convert(k + 1, ((k + 1) >> 2) == jj ? cb : cn, fn);
          else if (i + 1 < its) convert(0, cn, fn);
          __builtin_amdgcn_sched_barrier(0);
        }
        xb = nxb;
        wb = nwb;
      };
      if constexpr (JS % 2 == 0) {
        for (int i = 0; i < its; i++) stage(i, std::integral_constant<int, 0>{});
      } else {
        for (int i = 0; i < its; i += 2) {
          stage(i, std::integral_constant<int, 0>{});
          if (i + 1 < its) stage(i + 1, std::integral_constant<int, 1>{});
        }
      }
    }
    m4_barrier();
  }
  const int nblk = (P.H + 31) >> 5;
  for (int b0 = ns * NB; b0 < nblk; b0 += XNB) {
    // the columns past the last whole stage, zeros up to an x stage (with scales of 1)
    for (int i = threadIdx.x; i < T::XR * T::XC; i += T::NTK) {
      const int row = i / T::XC, c = (i % T::XC) ^ T::xperm(row);
      u32x4 v = {0u, 0u, 0u, 0u};
      const char* xr = X + (int64_t)mrow(row) * xstep;
      if constexpr (T::XS) {
        if (b0 + c < nblk) v = *reinterpret_cast<const u32x4*>(xr + (b0 + c) * 16);
      } else {
        const int e0 = 32 * b0 + 8 * c;
        if (e0 < P.H) v = load_piece<ADT>(xr, e0, P.H).q[0];
      }
      *reinterpret_cast<u32x4*>(lds + i * 16) = v;
    }
    char* const wst = lds + T::WOFF;
    for (int i = threadIdx.x; i < T::BN * T::WC; i += T::NTK) {
      const int row = i / T::WC, c = (i % T::WC) ^ T::wperm(row), b = b0 + c;
      u32x4 v = {0u, 0u, 0u, 0u};
      if (c < XNB && b < nblk) {
        v = *reinterpret_cast<const u32x4*>(W + (int64_t)nrow(row) * P.w_stride + b * 16);
#pragma unroll
        for (int e = 0; e < 4; e++) {               // (codes past the row's end count as zeros, whatever they hold)
          const int keep = P.H - 32 * b - 8 * e;
          v[e] = keep >= 8 ? v[e] : keep <= 0 ? 0u : v[e] & ((1u << (4 * keep)) - 1u);
        }
      }
      *reinterpret_cast<u32x4*>(wst + i * 16) = v;
    }
    char* const sst = lds + T::SOFF;
    for (int i = threadIdx.x; i < T::SROWS * XNB; i += T::NTK) {
      const int row = i / XNB, b = b0 + i % XNB;
      const char* sr = WS + (int64_t)nrow(row < T::BN ? row : 0) * Q.ws_stride;
      if constexpr (T::XS)
        if (row >= T::BN) sr = XSC + (int64_t)mrow(row - T::BN) * Q.xs_stride;
      sst[row * M4_SB + i % XNB] = b < nblk ? sr[b] : (char)127;
    }
    __syncthreads();
    const int left = nblk - b0, pairs = ((left < XNB ? left : XNB) + 1) / 2;
    if constexpr (XDT == LPS_DTYPE_F16) read_scales(sst, 0);
    if (XDT == LPS_DTYPE_F16 && wballot(far_any != 0) != 0) m4_plain_stage<XDT, T, true>(lds, wst, 0, sst, L, acc, pairs);
    else m4_plain_stage<XDT, T, false>(lds, wst, 0, sst, L, acc, pairs);
    __syncthreads();
  }
  if constexpr (KW == 2) {
    // the second group's accumulators join the first's
    static_assert(T::EW * MT * CT * 4096 <= T::BYTES, "they fit the stages' place");
    u32x4* const d = reinterpret_cast<u32x4*>(lds) + (wv % T::EW) * (MT * CT * 256) + l;
    if (L.kg == 1) {
#pragma unroll
      for (int a = 0; a < MT; a++)
#pragma unroll
        for (int b = 0; b < CT; b++)
#pragma unroll
          for (int q = 0; q < 4; q++)
            d[((a * CT + b) * 4 + q) * 64] = u32x4{__float_as_uint(acc[a][b][4 * q]), __float_as_uint(acc[a][b][4 * q + 1]),
                                                   __float_as_uint(acc[a][b][4 * q + 2]), __float_as_uint(acc[a][b][4 * q + 3])};
    }
    __syncthreads();
    if (L.kg == 1) return;   // (later barriers count the waves that are left)
#pragma unroll
    for (int a = 0; a < MT; a++)
#pragma unroll
      for (int b = 0; b < CT; b++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const u32x4 v = d[((a * CT + b) * 4 + q) * 64];
#pragma unroll
          for (int e = 0; e < 4; e++) acc[a][b][4 * q + e] = __fadd_rn(acc[a][b][4 * q + e], __uint_as_float(v[e]));
        }
    __syncthreads();
  }
  lmh_epilogue<ADT, ODT, M4Epi<T>>(P, lds, acc, n0, m0, wv, l);
}

}  // namespace lps
