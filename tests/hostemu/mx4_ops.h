// The CDNA4 scale conversions and the scaled matrix instruction that the
// vocabulary table's kernels use, on the host (from their definition: the scale
// is the exponent field of an fp32, e2m1 codes, ties to the even code).
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>

namespace lps_emu {
typedef float f2v __attribute__((ext_vector_type(2)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));

inline double e8m0(uint32_t byte) { return byte == 255u ? std::nan("") : std::ldexp(1.0, (int)byte - 127); }
inline uint32_t exp_byte(float s) { return (__float_as_uint(s) >> 23) & 255u; }
inline double e2m1(uint32_t c) {
  static const double v[8] = {0, 0.5, 1, 1.5, 2, 3, 4, 6};
  return (c & 8u) ? -v[c & 7u] : v[c & 7u];
}
inline double fp4(uint32_t codes, int i, float s) { return e2m1((codes >> (4 * i)) & 15u) * e8m0(exp_byte(s)); }
inline uint32_t to_fp4(double x, float s) {
  static const double v[8] = {0, 0.5, 1, 1.5, 2, 3, 4, 6};
  const double a = std::fabs(x) / e8m0(exp_byte(s));
  uint32_t best = 0;
  for (uint32_t c = 1; c < 8; c++) {
    const double mid = (v[c - 1] + v[c]) / 2;
    if (a > mid || (a == mid && !(c & 1u))) best = c;
  }
  return best | (std::signbit(x) ? 8u : 0u);
}
inline uint32_t put_pair(uint32_t old, double a, double b, float s, int sel) {
  const uint32_t byte = to_fp4(a, s) | to_fp4(b, s) << 4;
  return (old & ~(0xFFu << (8 * sel))) | byte << (8 * sel);
}
// v_mfma_scale_f32_32x32x64_f8f6f4 with 4-bit operands: lane l holds A row and B
// column l % 32, the 32 values of its block at k = 32 (l / 32) .., in 16 bytes,
// and that block's scale as byte `sel` of its scale register.
template <typename A, typename C>
inline C mfma_fp4(A a, A b, C c, int sa, int isa, int sb, int isb) {
  struct Ops { uint64_t v[2][64][2]; uint32_t s[2][64]; } o;
  for (int m = 0; m < 2; m++) {
    uint64_t h[2];
    memcpy(h, m == 0 ? &a : &b, 16);
    for (int p = 0; p < 2; p++)
      xchg<uint64_t>(h[p], [&](const uint64_t* w, uint64_t) {
        for (int l = 0; l < 64; l++) o.v[m][l][p] = w[l];
        return (uint64_t)0;
      });
    xchg<uint32_t>((uint32_t)(m == 0 ? isa : isb), [&](const uint64_t* w, uint64_t) {
      for (int l = 0; l < 64; l++) o.s[m][l] = ((uint32_t)w[l] >> (8 * (m == 0 ? sa : sb))) & 255u;
      return 0u;
    });
  }
  const int l = lane();
  for (int i = 0; i < 16; i++) {
    const int row = 8 * (i >> 2) + 4 * (l >> 5) + (i & 3), col = l & 31;
    double s = c[i];
    for (int h = 0; h < 2; h++) {
      const int ra = row + 32 * h, cb = col + 32 * h;
      const double sc = e8m0(o.s[0][ra]) * e8m0(o.s[1][cb]);
      for (int k = 0; k < 32; k++)
        s += e2m1((uint32_t)(o.v[0][ra][k >> 4] >> (4 * (k & 15))) & 15u) * e2m1((uint32_t)(o.v[1][cb][k >> 4] >> (4 * (k & 15))) & 15u) * sc;
    }
    c[i] = (float)s;
  }
  return c;
}
}  // namespace lps_emu

#define __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, sel) \
  (::lps_emu::f2v{(float)::lps_emu::fp4((c), 2 * (sel), (s)), (float)::lps_emu::fp4((c), 2 * (sel) + 1, (s))})
#define __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, sel) \
  (::lps_emu::b2v{(__bf16)(float)::lps_emu::fp4((c), 2 * (sel), (s)), (__bf16)(float)::lps_emu::fp4((c), 2 * (sel) + 1, (s))})
#define __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, sel) \
  (::lps_emu::h2v{(_Float16)::lps_emu::fp4((c), 2 * (sel), (s)), (_Float16)::lps_emu::fp4((c), 2 * (sel) + 1, (s))})
#define __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, a, b, s, sel) (::lps_emu::put_pair((o), (a), (b), (s), (sel)))
#define __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, p, s, sel) \
  ([&] { uint32_t t_; const ::lps_emu::b2v p_ = (p); memcpy(&t_, &p_, 4); \
         return ::lps_emu::put_pair((o), __uint_as_float(t_ << 16), __uint_as_float(t_ & 0xFFFF0000u), (s), (sel)); }())
#define __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, p, s, sel) \
  ([&] { const ::lps_emu::h2v t_ = (p); return ::lps_emu::put_pair((o), (double)t_.x, (double)t_.y, (s), (sel)); }())
#define __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, fa, fb, sa, isa, sb, isb) \
  (::lps_emu::mfma_fp4((a), (b), (c), (sa), (isa), (sb), (isb)))
#define __builtin_amdgcn_sched_barrier(mask) ((void)0)
