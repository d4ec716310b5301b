// Microscaled 4-bit floats: the block format, its quantiser, and the row
// gather behind the table lookup and the dequantiser (gfx950).
//
// A block is 32 values of a row (the last one may hold fewer).  Its scale is
// 2^s, s = max(floor(log2 top) - 2, -126) for the largest magnitude top, held
// as the byte s + 127; 255 marks a block with a value that is not finite and
// stands for NaN.  A value's code is e2m1 with a sign: the nearest of 0, 0.5,
// 1, 1.5, 2, 3, 4, 6 to |x| / 2^s, ties to the even code, and 6 above it (top
// lies in [4, 8) scales, so that 6 is at most a quarter off).  Codes lie two to
// a byte, the even element in the low half; 16 bytes hold a block.
//
// The conversions are the CDNA4 instructions v_cvt_scalef32_pk_*: they take the
// scale as the exponent field of an fp32 operand (byte << 23; 0 is 2^-127, 255
// is NaN; sign and mantissa are ignored), round to nearest even and saturate:
// checked on gfx950 against the definition for every 16-bit value and scale.
#pragma once

#include "lps_common.h"
#include "lps_wave.h"

namespace lps {

constexpr int MX4_BLOCK = 32;
constexpr int MX4_MAX_HIDDEN = 1 << 24;   // of every operator on rows: offsets within one stay in 32 bits
constexpr int64_t MX4_STREAM = 32 << 20;   // bytes: the card's L2s

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
// 16 bytes at any element's address (global loads and stores need no wider one)
typedef uint32_t u32x4e2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4e4 __attribute__((ext_vector_type(4), aligned(4)));

template <int DT> struct ElemBytes { static constexpr int value = DT == LPS_DTYPE_F32 ? 4 : 2; };

// Eight consecutive elements as they lie in memory.
template <int DT> struct Piece { u32x4 q[DT == LPS_DTYPE_F32 ? 2 : 1]; };

template <int DT> struct Line { typedef u32x4e2 type; };   // 16 bytes at an element's alignment
template <> struct Line<LPS_DTYPE_F32> { typedef u32x4e4 type; };
template <int DT, bool NTL>
__device__ __forceinline__ u32x4 ld16(const char* p) {
  typedef typename Line<DT>::type L;
  if constexpr (NTL) return __builtin_nontemporal_load(reinterpret_cast<const L*>(p));
  else return *reinterpret_cast<const L*>(p);
}
template <int DT, bool NTS>
__device__ __forceinline__ void st16(char* p, u32x4 v) {
  typedef typename Line<DT>::type L;
  if constexpr (NTS) __builtin_nontemporal_store((L)v, reinterpret_cast<L*>(p));
  else *reinterpret_cast<L*>(p) = v;
}

// Elements e0 .. e0 + 7 of a row of n (zeros past its end; e0 < n).
template <int DT, bool NTL = false>
__device__ __forceinline__ Piece<DT> load_piece(const void* row, int e0, int n) {
  constexpr int ES = ElemBytes<DT>::value;
  Piece<DT> r;
  const char* p = static_cast<const char*>(row) + (int64_t)e0 * ES;
  if (e0 + 8 <= n) {
    r.q[0] = ld16<DT, NTL>(p);
    if constexpr (DT == LPS_DTYPE_F32) r.q[1] = ld16<DT, NTL>(p + 16);
  } else {
    uint32_t w[DT == LPS_DTYPE_F32 ? 8 : 4] = {};
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if (e0 + e < n) {
        if constexpr (DT == LPS_DTYPE_F32) w[e] = reinterpret_cast<const uint32_t*>(p)[e];
        else w[e >> 1] |= (uint32_t)reinterpret_cast<const unsigned short*>(p)[e] << (16 * (e & 1));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      r.q[0][i] = w[i];
      if constexpr (DT == LPS_DTYPE_F32) r.q[1][i] = w[4 + i];
    }
  }
  return r;
}

template <int DT>
__device__ __forceinline__ void piece_values(const Piece<DT>& r, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e++) {
    if constexpr (DT == LPS_DTYPE_F32) v[e] = __uint_as_float(r.q[e >> 2][e & 3]);
    else {
      const uint32_t h = (r.q[0][e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
      v[e] = DT == LPS_DTYPE_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
    }
  }
}

// The values rounded to the output type (to nearest even) and stored as
// elements e0 .. e0 + 7 of a row of n (e0 < n).
template <int DT, bool NTS = false>
__device__ __forceinline__ void store_piece(void* row, int e0, int n, const float (&v)[8]) {
  constexpr int ES = ElemBytes<DT>::value;
  char* p = static_cast<char*>(row) + (int64_t)e0 * ES;
  uint32_t w[DT == LPS_DTYPE_F32 ? 8 : 4];
  if constexpr (DT == LPS_DTYPE_F32) {
#pragma unroll
    for (int e = 0; e < 8; e++) w[e] = __float_as_uint(v[e]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const f32x2 t = {v[2 * i], v[2 * i + 1]};
      if constexpr (DT == LPS_DTYPE_BF16) w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(t, bf16x2));
      else w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(t, f16x2));
    }
  }
  if (e0 + 8 <= n) {
    st16<DT, NTS>(p, u32x4{w[0], w[1], w[2], w[3]});
    if constexpr (DT == LPS_DTYPE_F32) st16<DT, NTS>(p + 16, u32x4{w[4], w[5], w[6], w[7]});
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if (e0 + e < n) {
        if constexpr (DT == LPS_DTYPE_F32) reinterpret_cast<uint32_t*>(p)[e] = w[e];
        else reinterpret_cast<unsigned short*>(p)[e] = (unsigned short)(w[e >> 1] >> (16 * (e & 1)));
      }
    }
  }
}

// fp32 elements e0 .. e0 + 3, the first or the second four of v.
template <bool NTS>
__device__ __forceinline__ void store_half(void* row, int e0, int n, const float (&v)[8], bool second) {
  uint32_t* p = static_cast<uint32_t*>(row) + e0;
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; e++) w[e] = __float_as_uint(second ? v[4 + e] : v[e]);
  if (e0 + 4 <= n) {
    st16<LPS_DTYPE_F32, NTS>(reinterpret_cast<char*>(p), u32x4{w[0], w[1], w[2], w[3]});
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (e0 + e < n) p[e] = w[e];
  }
}

// Eight codes (element i in bits 4 i .. 4 i + 3) to their values.
__device__ __forceinline__ void mx4_values(uint32_t codes, uint32_t scale_byte, float (&v)[8]) {
  const float s = __uint_as_float(scale_byte << 23);
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 1),
              c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 3);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}

template <int DT>
__device__ __forceinline__ uint32_t mx4_codes(const Piece<DT>& r, float scale) {
  uint32_t c = 0;
  if constexpr (DT == LPS_DTYPE_F32) {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(r.q[0].x), __uint_as_float(r.q[0].y), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(r.q[0].z), __uint_as_float(r.q[0].w), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(r.q[1].x), __uint_as_float(r.q[1].y), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(r.q[1].z), __uint_as_float(r.q[1].w), scale, 3);
  } else if constexpr (DT == LPS_DTYPE_BF16) {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, (uint32_t)r.q[0].x), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, (uint32_t)r.q[0].y), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, (uint32_t)r.q[0].z), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, (uint32_t)r.q[0].w), scale, 3);
  } else {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, (uint32_t)r.q[0].x), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, (uint32_t)r.q[0].y), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, (uint32_t)r.q[0].z), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2, (uint32_t)r.q[0].w), scale, 3);
  }
  return c;
}

// The largest magnitude of a piece as the bits of an fp32 (ordered as the
// magnitudes are; infinities and NaN are at or above 0x7F800000).
template <int DT>
__device__ __forceinline__ uint32_t piece_top(const Piece<DT>& r) {
  if constexpr (DT == LPS_DTYPE_F32) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint32_t b = r.q[e >> 2][e & 3] & 0x7FFFFFFFu;
      m = b > m ? b : m;
    }
    return m;
  } else {
    u16x2 m = __builtin_bit_cast(u16x2, (uint32_t)r.q[0].x & 0x7FFF7FFFu);
#pragma unroll
    for (int i = 1; i < 4; i++)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, (uint32_t)r.q[0][i] & 0x7FFF7FFFu));
    const uint32_t h = m.x > m.y ? m.x : m.y;
    return DT == LPS_DTYPE_BF16 ? h << 16 : __float_as_uint(f16_to_f32(h));
  }
}

struct Mx4Params {
  const void* x;      // [rows, hidden]
  uint8_t* codes;     // [rows, 16 blocks]
  uint8_t* scales;    // [rows, blocks]
  int64_t x_stride, codes_stride, scales_stride;   // elements; bytes
  int rows, hidden, blocks;
  int lg_tpr;         // log2 of the threads on a row
  int words;          // scale rows begin on 4-byte lines
};

// ---------------------------------------------------------------------------
// Quantiser: a thread takes eight values, four neighbours a block (its largest
// magnitude over two DPP moves), 16 neighbours four blocks (their scales are one
// 4-byte store); 16 to 256 threads a row, two pieces of each in flight.
// Bound by HBM: es + 17/32 bytes a value.  NTS: stores past the caches, for outputs
// that do not fit them (MX4_STREAM).  151936 x 4096 bf16: 243 us, 5.9 TB/s read and
// written (260 through the caches); a copy reaches 5.1, a fill 6.9.
// ---------------------------------------------------------------------------
template <int DT, bool NTS>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(Mx4Params P) {
  const int tid = (int)threadIdx.x, tpr = 1 << P.lg_tpr, t = tid & (tpr - 1);
  const int64_t row = (int64_t)blockIdx.x * (256 >> P.lg_tpr) + (tid >> P.lg_tpr);
  const bool live = row < P.rows;
  const char* x = static_cast<const char*>(P.x) + (live ? row : 0) * P.x_stride * ElemBytes<DT>::value;
  uint8_t* codes = P.codes + (live ? row : 0) * P.codes_stride;
  uint8_t* scales = P.scales + (live ? row : 0) * P.scales_stride;
  const int pieces = 4 * P.blocks;
  // (every lane stays in the loop: the lane moves need their neighbours)
  for (int p0 = 0; p0 < pieces; p0 += 2 * tpr) {
    Piece<DT> v[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int e0 = 8 * (p0 + u * tpr + t);
      v[u] = Piece<DT>{};
      if (live && e0 < P.hidden) v[u] = load_piece<DT, true>(x, e0, P.hidden);
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int p = p0 + u * tpr + t;
      uint32_t top = piece_top(v[u]);
      top = OpMax{}(top, dpp_t<0xB1>(top, top));   // quad_perm [1,0,3,2]
      top = OpMax{}(top, dpp_t<0x4E>(top, top));   // quad_perm [2,3,0,1]
      const bool fine = top < 0x7F800000u;
      const uint32_t e = top >> 23, byte = !fine ? 255u : e > 3u ? e - 2u : 1u;
      const uint32_t c = fine ? mx4_codes(v[u], __uint_as_float(byte << 23)) : 0u;
      uint32_t w = byte << (8 * ((t >> 2) & 3));
      w |= dpp_t<0x141>(w, w);                     // row_half_mirror: the other block of eight lanes
      w |= dpp_t<0x140>(w, w);                     // row_mirror: the other two of sixteen
      if (live && p < pieces) {
        uint32_t* d = reinterpret_cast<uint32_t*>(codes + 4 * (int64_t)p);
        if constexpr (NTS) __builtin_nontemporal_store(c, d);
        else *d = c;
        const int b = p >> 2;
        if (P.words && (b | 3) < P.blocks) {
          if ((t & 15) == 0) *reinterpret_cast<uint32_t*>(scales + b) = w;
        } else if ((t & 3) == 0) {
          scales[b] = (uint8_t)byte;
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Row gather: out[i] = scale * table[id_i], zeros where the id is outside the
// table; without ids row i itself (the dequantiser).  fp32 arithmetic, rounded
// once.  A thread has two pieces of eight values (of fp32 outputs four) in flight; few rows are cut over
// more workgroups.  16384 bf16 rows of 4096: 32 us (35 through the caches), of a
// 4-bit table 22.5 (27.5); the dequantiser, 151936 rows: 285 us, 5.5 TB/s.
// ---------------------------------------------------------------------------
constexpr int DT_MX4 = LPS_DTYPE_MX4;

struct GatherParams {
  const void* ids;       // int32 / int64 [n], or null
  const void* table;     // [vocab, hidden], or 4-bit codes
  const uint8_t* scales; // 4-bit tables
  void* out;             // [n, hidden]
  int64_t table_stride;  // elements (bytes of a 4-bit table)
  int64_t scales_stride; // bytes
  int64_t out_stride;    // elements
  int64_t n, vocab;
  int hidden, id_bytes;
  int lg_tpr;            // log2 of the threads on a row
  float scale;
};

__device__ __forceinline__ int64_t load_id(const void* ids, int id_bytes, int64_t i) {
  return id_bytes == 8 ? static_cast<const int64_t*>(ids)[i] : (int64_t)static_cast<const int32_t*>(ids)[i];
}

template <int TDT> struct GatherPiece { Piece<TDT> v; };
template <> struct GatherPiece<DT_MX4> { uint32_t codes, scale; };

// values that a thread stores at once, 16 bytes: of fp32, half of a piece that it and
// its neighbour both read.  (A whole piece in two stores leaves every other 16 bytes
// of a line to the second: 16384 bf16 rows of 4096 to fp32 94 us against 52, of a
// 4-bit table 109 against 49.)
template <int ODT> constexpr int GATHER_VALUES = ODT == LPS_DTYPE_F32 ? 4 : 8;

template <int TDT, int ODT, bool NTS>
__global__ __launch_bounds__(256) void gather_kernel(GatherParams P) {
  const int tid = (int)threadIdx.x, tpr = 1 << P.lg_tpr, t = tid & (tpr - 1);
  const int64_t i = (int64_t)blockIdx.x * (256 >> P.lg_tpr) + (tid >> P.lg_tpr);
  if (i >= P.n) return;
  const int64_t id = P.ids ? load_id(P.ids, P.id_bytes, i) : i;
  const bool valid = id >= 0 && id < P.vocab;
  const int64_t at = valid ? id : 0;
  const char* row = static_cast<const char*>(P.table) +
                    at * P.table_stride * (TDT == DT_MX4 ? 1 : ElemBytes<TDT>::value);
  const uint8_t* srow = TDT == DT_MX4 ? P.scales + at * P.scales_stride : nullptr;
  char* out = static_cast<char*>(P.out) + i * P.out_stride * ElemBytes<ODT>::value;
  constexpr int E = GATHER_VALUES<ODT>;
  const int parts = (P.hidden + E - 1) / E, step = tpr * (int)gridDim.y;
  for (int p0 = (int)blockIdx.y * tpr + t; p0 < parts; p0 += 2 * step) {
    GatherPiece<TDT> g[2] = {};
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int p = p0 + u * step;
      if (valid && p < parts) {
        const int q = p / (8 / E);                 // the piece
        if constexpr (TDT == DT_MX4) {
          g[u].codes = *reinterpret_cast<const uint32_t*>(row + 4 * (int64_t)q);
          g[u].scale = srow[q >> 2];
        } else {
          g[u].v = load_piece<TDT>(row, 8 * q, P.hidden);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int p = p0 + u * step;
      if (p < parts) {
        float v[8];
        if constexpr (TDT == DT_MX4) mx4_values(g[u].codes, g[u].scale, v);
        else piece_values(g[u].v, v);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = valid ? __fmul_rn(v[e], P.scale) : 0.0f;
        if constexpr (E == 8) store_piece<ODT, NTS>(out, 8 * p, P.hidden, v);
        else store_half<NTS>(out, 4 * p, P.hidden, v, p & 1);
      }
    }
  }
}

}  // namespace lps
