// C ABI of the LM head over a 4-bit weight (declaration in include/lps.h).
// Launches only; no allocation, no synchronisation.
#include <hip/hip_runtime.h>

#include "lps_host.h"
#include "lps_mx4head.h"

using namespace lps;

namespace {

// (131070 row tiles of 32 times 16383 column tiles of 128 are fewer than 2^31)
constexpr int kMaxHeadVocab = 1 << 21;

template <int XDT, int ODT, typename T, bool NTL>
hipError_t launch_mx4head(Mx4HeadParams Q, hipStream_t s) {
  Q.h.mtiles = (Q.h.M + T::BM - 1) / T::BM;
  Q.h.tiles = Q.h.mtiles * ((Q.h.V + T::BN - 1) / T::BN);
  hipLaunchKernelGGL((mx4head_kernel<XDT, ODT, T, NTL>), dim3((unsigned)(Q.h.tiles + 7) / 8 * 8), dim3(T::NTK), 0, s, Q);
  return hipGetLastError();
}
// The tile shape by rows and tiles.  A grid whose tiles all run at once takes the
// smallest shape of which that is true: two workgroups of some shapes share a CU
// (the third column).  Larger grids go by their rows: while w's pass over HBM is
// the bound one row tile, so that it is read once and streamed past the caches.
// Measured at hidden 4096 (us; x in 16 bits, by shape): 128 rows of V 8192 17, 23,
// 46; 256 of 8192 25, 26, 48; 512 of 8192 47, 40, 60; 1024 of 8192 94, 78, 62; 128 of
// 32000 45, 41, 50; 256 of 32000 85, 76, 58; 64 of 151936 -, 95, 160.  x in 4 bits:
// 256 rows of V 8192 -, 13, 18, 35; 512 of 8192 -, 24, 21, 38; 1024 of 8192 -, 42, 29,
// 40; 512 of 32000 -, 80, 47, 41; 512 of 151936 -, -, 251, 204; 2048 -, -, 964, 764.
struct M4Shape { int bm, bn, per_cu, rows; };
constexpr M4Shape M4_SHAPES16[] = {{32, 128, 2, 32}, {64, 128, 2, 64}, {128, 256, 1, 0}};
constexpr M4Shape M4_SHAPES4[] = {{32, 128, 1, 32}, {64, 128, 1, 64}, {128, 128, 2, 128}, {256, 256, 1, 0}};
template <int N>
int mx4head_shape(const M4Shape (&shapes)[N], int M, int V, int cus) {
  for (int i = 0; i < N; i++) {
    const int64_t tiles = (int64_t)((M + shapes[i].bm - 1) / shapes[i].bm) * ((V + shapes[i].bn - 1) / shapes[i].bn);
    if (tiles <= (int64_t)cus * shapes[i].per_cu || i + 1 == N || M <= shapes[i].rows) return i;
  }
  return N - 1;
}

template <int XDT, int ODT>
hipError_t launch_mx4head_rows(const Mx4HeadParams& Q, hipStream_t s) {
  const int M = Q.h.M, V = Q.h.V, cus = device_cus();
  if constexpr (XDT == DT_MX4) {
    switch (mx4head_shape(M4_SHAPES4, M, V, cus)) {
      case 0: return launch_mx4head<XDT, ODT, M4Tile<32, 128, 1, 4, 2, 8, 2, 2, 4, 2, 16>, true>(Q, s);
      case 1: return launch_mx4head<XDT, ODT, M4Tile<64, 128, 2, 2, 2, 8, 2, 2, 4, 2, 16>, true>(Q, s);
      case 2: return launch_mx4head<XDT, ODT, M4Tile<128, 128, 2, 4, 1, 8, 2, 2, 4, 4, 16>, false>(Q, s);
      default: return launch_mx4head<XDT, ODT, M4Tile<256, 256, 2, 4, 1, 8, 2, 2, 4, 2, 16>, false>(Q, s);
    }
  } else {
    // two workgroups to a CU: fp16's two paths have to be held to their 128 registers
    // (bf16's fit by themselves; held to it, 16 rows take 74 us for 63)
    constexpr int WPE = XDT == LPS_DTYPE_F16 ? 4 : 2;
    switch (mx4head_shape(M4_SHAPES16, M, V, cus)) {
      case 0:
        // few rows leave LDS for stages further ahead (8 rows of V 151936: 57 us, 74 with 32 held; 16: 63, 75)
        if (M <= 8) return launch_mx4head<XDT, ODT, M4Tile<32, 128, 1, 4, 2, 8, 3, 3, 4, WPE, 64, 8>, true>(Q, s);
        if (M <= 16) return launch_mx4head<XDT, ODT, M4Tile<32, 128, 1, 4, 2, 8, 3, 3, 4, WPE, 64, 16>, true>(Q, s);
        return launch_mx4head<XDT, ODT, M4Tile<32, 128, 1, 4, 2, 4, 4, 2, 4, 4, 64>, true>(Q, s);
      case 1:
        // (fp16's second path does not fit 128 registers beside two columns of accumulators)
        if constexpr (XDT == LPS_DTYPE_F16) return launch_mx4head<XDT, ODT, M4Tile<64, 128, 2, 4, 1, 4, 2, 2, 4, 4, 64>, true>(Q, s);
        else return launch_mx4head<XDT, ODT, M4Tile<64, 128, 2, 2, 2, 4, 2, 2, 4, 4, 64>, true>(Q, s);
      default: return launch_mx4head<XDT, ODT, M4Tile<128, 256, 2, 4, 1, 4, 2, 2, 4, 2, 64>, false>(Q, s);
    }
  }
}
template <int XDT>
hipError_t dispatch_mx4head(const Mx4HeadParams& Q, int out_dtype, hipStream_t s) {
  switch (out_dtype) {
    case LPS_DTYPE_F32: return launch_mx4head_rows<XDT, LPS_DTYPE_F32>(Q, s);
    case LPS_DTYPE_BF16: return launch_mx4head_rows<XDT, LPS_DTYPE_BF16>(Q, s);
    default: return launch_mx4head_rows<XDT, LPS_DTYPE_F16>(Q, s);
  }
}

}  // namespace

extern "C" int lps_lm_head_mx4(const lps_lm_head_mx4_args* a, void* stream) {
  if (!a) return LPS_EINVAL;
  const bool x4 = a->dtype == LPS_DTYPE_MX4;
  if (!x4 && a->dtype != LPS_DTYPE_BF16 && a->dtype != LPS_DTYPE_F16) return LPS_EUNSUPPORTED_DTYPE;
  if (!dtype_ok(a->out_dtype)) return LPS_EUNSUPPORTED_DTYPE;
  if (a->rows < 0 || a->vocab < 1 || a->hidden < 1 || a->rows > LMH_MAX_ROWS || a->vocab > kMaxHeadVocab ||
      a->hidden > MX4_MAX_HIDDEN)
    return LPS_EINVAL;
  if (a->rows == 0) return LPS_OK;
  if (!a->x || !a->w || !a->w_scales || !a->out || (x4 && !a->x_scales)) return LPS_EINVAL;
  const int64_t nb = ((int64_t)a->hidden + MX4_BLOCK - 1) / MX4_BLOCK;
  Mx4HeadParams Q{};
  LmHeadParams& P = Q.h;
  // (a single row's stride does not count)
  P.x_stride = a->rows > 1 ? a->x_stride : 0;
  P.w_stride = a->vocab > 1 ? a->w_stride : 0;
  P.out_stride = a->rows > 1 ? a->out_stride : a->vocab;
  Q.ws_stride = a->vocab > 1 ? a->w_scales_stride : 0;
  Q.xs_stride = x4 && a->rows > 1 ? a->x_scales_stride : 0;
  if (a->rows > 1 && (P.x_stride < (x4 ? 16 * nb : a->hidden) || P.out_stride < a->vocab)) return LPS_EINVAL;
  if (a->vocab > 1 && (P.w_stride < 16 * nb || Q.ws_stride < nb)) return LPS_EINVAL;
  if (x4 && a->rows > 1 && Q.xs_stride < nb) return LPS_EINVAL;
  if ((x4 ? 1 : 2) * P.x_stride > M4_MAX_STRIDE || P.w_stride > M4_MAX_STRIDE || Q.ws_stride > M4_MAX_STRIDE ||
      Q.xs_stride > M4_MAX_STRIDE)
    return LPS_EINVAL;
  // 16-byte operand loads, 4-byte loads of scales
  if (reinterpret_cast<uintptr_t>(a->x) % 16 || P.x_stride % (x4 ? 16 : 8) || reinterpret_cast<uintptr_t>(a->w) % 16 ||
      P.w_stride % 16)
    return LPS_EINVAL;
  if (reinterpret_cast<uintptr_t>(a->w_scales) % 4 || Q.ws_stride % 4) return LPS_EINVAL;
  if (x4 && (reinterpret_cast<uintptr_t>(a->x_scales) % 4 || Q.xs_stride % 4)) return LPS_EINVAL;
  P.x = a->x;
  P.w = a->w;
  P.out = a->out;
  P.stats = a->stats;
  P.M = a->rows;
  P.V = a->vocab;
  P.H = a->hidden;
  P.G = (a->vocab + LMH_BN - 1) / LMH_BN;
  Q.ws = static_cast<const uint8_t*>(a->w_scales);
  Q.xs = static_cast<const uint8_t*>(a->x_scales);
  auto wide = [&](const void* p, int64_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 16 == 0; };
  Q.wide = nb % 16 == 0 && wide(Q.ws, Q.ws_stride) && (!x4 || wide(Q.xs, Q.xs_stride));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e = x4 ? dispatch_mx4head<DT_MX4>(Q, a->out_dtype, s)
                       : a->dtype == LPS_DTYPE_BF16 ? dispatch_mx4head<LPS_DTYPE_BF16>(Q, a->out_dtype, s)
                                                    : dispatch_mx4head<LPS_DTYPE_F16>(Q, a->out_dtype, s);
  return e == hipSuccess ? LPS_OK : LPS_ELAUNCH;
}
