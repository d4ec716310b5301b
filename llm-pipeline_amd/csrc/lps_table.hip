// C ABI of the vocabulary table's operators (declarations in include/lps.h):
// 4-bit quantisation, the lookup and its gradient.  Launches only; no
// allocation, no synchronisation, no state.
#include <hip/hip_runtime.h>

#include "lps_embgrad.h"
#include "lps_host.h"
#include "lps_mx4.h"

using namespace lps;

namespace {

constexpr int kMaxPositions = 1 << 30;   // of a gradient: its kernels count a little past them in 32 bits
constexpr int64_t kMaxGroups = 0xFFFFFFFFu / 256;   // workgroups of 256: a launch has fewer than 2^32 threads

bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
size_t elem_bytes(int dtype) { return dtype == LPS_DTYPE_F32 ? 4 : 2; }
int blocks_of(int hidden) { return (hidden + MX4_BLOCK - 1) / MX4_BLOCK; }

// Threads on a row of `pieces` (two pieces a thread where the row has that
// many): a power of two from 16 to 256, as its logarithm.
int lg_threads_per_row(int pieces) {
  int lg = 4;
  while (lg < 8 && (2 << lg) < pieces) lg++;
  return lg;
}

template <int TDT, int ODT>
hipError_t launch_gather(GatherParams P, hipStream_t s) {
  const int pieces = (P.hidden + GATHER_VALUES<ODT> - 1) / GATHER_VALUES<ODT>;
  P.lg_tpr = lg_threads_per_row(pieces);
  const int64_t wgs = (P.n + (256 >> P.lg_tpr) - 1) >> (8 - P.lg_tpr);
  // few rows: a long row over several workgroups
  const int chunks = (pieces + (1 << P.lg_tpr) - 1) >> P.lg_tpr;
  const unsigned y = wgs < 1024 ? (unsigned)(chunks < 65535 ? chunks : 65535) : 1u;
  const bool past = P.n * P.hidden * ElemBytes<ODT>::value > MX4_STREAM;
  // (rows that outgrow a launch: the next ones in another)
  const int64_t most = kMaxGroups << (8 - P.lg_tpr);
  for (int64_t left = P.n; left > 0; left -= most) {
    P.n = left < most ? left : most;
    const dim3 grid((unsigned)((P.n + (256 >> P.lg_tpr) - 1) >> (8 - P.lg_tpr)), y);
    if (past) hipLaunchKernelGGL((gather_kernel<TDT, ODT, true>), grid, dim3(256), 0, s, P);
    else hipLaunchKernelGGL((gather_kernel<TDT, ODT, false>), grid, dim3(256), 0, s, P);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    P.out = static_cast<char*>(P.out) + P.n * P.out_stride * ElemBytes<ODT>::value;
    if (P.ids) {
      P.ids = static_cast<const char*>(P.ids) + P.n * P.id_bytes;
    } else {
      P.table = static_cast<const char*>(P.table) + P.n * P.table_stride * (TDT == DT_MX4 ? 1 : ElemBytes<TDT>::value);
      if (P.scales) P.scales += P.n * P.scales_stride;
    }
  }
  return hipSuccess;
}
template <int TDT>
hipError_t dispatch_gather(int out_dtype, const GatherParams& P, hipStream_t s) {
  switch (out_dtype) {
    case LPS_DTYPE_F32: return launch_gather<TDT, LPS_DTYPE_F32>(P, s);
    case LPS_DTYPE_BF16: return launch_gather<TDT, LPS_DTYPE_BF16>(P, s);
    default: return launch_gather<TDT, LPS_DTYPE_F16>(P, s);
  }
}

template <int DT>
hipError_t launch_quantize(Mx4Params P, hipStream_t s) {
  P.lg_tpr = lg_threads_per_row(4 * P.blocks);
  const bool past = (int64_t)P.rows * P.blocks * 16 > MX4_STREAM;
  // (rows that outgrow a launch: the next ones in another)
  const int64_t most = kMaxGroups << (8 - P.lg_tpr);
  for (int64_t left = P.rows; left > 0; left -= most) {
    P.rows = (int)(left < most ? left : most);
    const dim3 grid((unsigned)(((int64_t)P.rows + (256 >> P.lg_tpr) - 1) >> (8 - P.lg_tpr)));
    if (past) hipLaunchKernelGGL((mx4_quantize_kernel<DT, true>), grid, dim3(256), 0, s, P);
    else hipLaunchKernelGGL((mx4_quantize_kernel<DT, false>), grid, dim3(256), 0, s, P);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    P.x = static_cast<const char*>(P.x) + P.rows * P.x_stride * ElemBytes<DT>::value;
    P.codes += P.rows * P.codes_stride;
    P.scales += P.rows * P.scales_stride;
  }
  return hipSuccess;
}

int check_mx4(const lps_mx4_args* a) {
  if (!a) return LPS_EINVAL;
  if (!dtype_ok(a->dtype)) return LPS_EUNSUPPORTED_DTYPE;
  if (a->rows < 0 || a->hidden < 1 || a->hidden > MX4_MAX_HIDDEN) return LPS_EINVAL;
  if (a->rows == 0) return LPS_OK;
  if (!a->x || !a->codes || !a->scales || !aligned_to(a->x, elem_bytes(a->dtype))) return LPS_EINVAL;
  if (!aligned_to(a->codes, 4) || a->codes_stride % 4) return LPS_EINVAL;
  const int64_t nb = blocks_of(a->hidden);
  if (a->rows > 1 && (a->x_stride < a->hidden || a->codes_stride < 16 * nb || a->scales_stride < nb)) return LPS_EINVAL;
  return LPS_OK;
}

struct EgWs {
  size_t count, sid, spos, tmp_id, tmp_pos, part, bytes;
};
// Positions of a tile: about 2048 tiles, so that a frequent token's rows spread
// over the card and a tile's loads are in flight together.
int eg_tile(int n) {
  int s = 8;
  while (s < EG_SMAX && (int64_t)s * 2048 < n) s *= 2;
  return s;
}
// Without a sort and a workspace: few positions (a new fp32 gradient of 1000 to 4000 rows: 517
// positions about 12 us against 17, 1000 22 to 35 against 17 to 28, even at 768), and
// ids that 4096 workgroups can own.
bool eg_small(int n, int vocab) { return n == 0 || (n <= EG_SMALL && vocab <= 4096 * EG_OWN); }
EgWs eg_workspace(int n, int vocab, int hidden) {
  EgWs w{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  if (eg_small(n, vocab)) return w;
  const int S = eg_tile(n);
  const size_t tiles = ((size_t)n + S - 1) / S;
  w.count = take(4);
  w.sid = take((size_t)n * 4);
  w.spos = take((size_t)n * 4);
  w.tmp_id = take((size_t)n * 4);
  w.tmp_pos = take((size_t)n * 4);
  w.part = take(tiles * 2 * (((size_t)hidden + 7) / 8 * 8) * 4);
  w.bytes = at;
  return w;
}

// Workgroups of `threads` that zero all rows: 16 bytes a thread, whole eights, up to
// EG_FILL (a launch has fewer than 2^32 threads, the sort's at most 2^21 workgroups
// of 1024 among them).
unsigned fill_wgs(const EmbGradParams& P, int threads) {
  const int64_t eights = (P.fill_rows * P.fill_lines + 8 * threads - 1) / (8 * threads);
  return eights < EG_FILL / 8 ? 8 * (unsigned)eights : (unsigned)EG_FILL;
}

template <int GDT, int ODT>
hipError_t launch_grad(EmbGradParams P, hipStream_t s) {
  const int64_t bytes = P.accumulate ? 0 : (int64_t)P.vocab * P.hidden * ElemBytes<ODT>::value;
  if (eg_small(P.n, P.vocab)) {
    // more zeros than the L2s hold: in a launch before; of no positions the zeros are all
    P.zero = !P.accumulate && bytes <= MX4_STREAM && P.n > 0;
    if (bytes > 0 && !P.zero) {
      hipLaunchKernelGGL((grad_zero_kernel<ODT>), dim3(fill_wgs(P, 256)), dim3(256), 0, s, P);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess || P.n == 0) return e;
    }
    // about eight positions and 64 thousand values of zeros a workgroup, up to one on
    // each CU; more where it would own more ids than it can count
    const int64_t values = P.zero ? (int64_t)P.vocab * (P.hidden < 256 ? P.hidden : 256) : 0;
    int lg = 4;
    while (lg < 8 && ((8 << lg) < P.n || (values >> lg) > 65536)) lg++;
    while (((int64_t)P.vocab + (1 << lg) - 1) >> lg > EG_OWN) lg++;
    P.lg_groups = lg;
    hipLaunchKernelGGL((grad_small_kernel<GDT, ODT>), dim3(1u << lg, (unsigned)((P.hidden + 255) / 256)), dim3(256), 0, s, P);
    return hipGetLastError();
  }
  // (each reads what the one before wrote: none follows a failed one)
  hipLaunchKernelGGL((grad_sort_kernel<ODT>), dim3((1u << P.lg_groups) + (P.accumulate ? 0 : fill_wgs(P, EG_NT))), dim3(EG_NT), 0, s, P);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((grad_tiles_kernel<GDT, ODT>), dim3((unsigned)((int64_t)P.tiles * P.slices)), dim3(256), 0, s, P);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (P.tiles > 1)
    hipLaunchKernelGGL((grad_join_kernel<ODT>), dim3((unsigned)((P.tiles - 1 + EG_JOIN - 1) / EG_JOIN), (unsigned)((P.hidden + 255) / 256)), dim3(256), 0, s, P);
  return hipGetLastError();
}
template <int GDT>
hipError_t dispatch_grad(int out_dtype, const EmbGradParams& P, hipStream_t s) {
  switch (out_dtype) {
    case LPS_DTYPE_F32: return launch_grad<GDT, LPS_DTYPE_F32>(P, s);
    case LPS_DTYPE_BF16: return launch_grad<GDT, LPS_DTYPE_BF16>(P, s);
    default: return launch_grad<GDT, LPS_DTYPE_F16>(P, s);
  }
}

}  // namespace

extern "C" {

int lps_mx4_quantize(const lps_mx4_args* a, void* stream) {
  const int rc = check_mx4(a);
  if (rc != LPS_OK || a->rows == 0) return rc;
  Mx4Params P{};
  P.x = a->x;
  P.codes = static_cast<uint8_t*>(a->codes);
  P.scales = static_cast<uint8_t*>(a->scales);
  P.rows = a->rows;
  P.hidden = a->hidden;
  P.blocks = blocks_of(a->hidden);
  P.x_stride = a->rows > 1 ? a->x_stride : 0;
  P.codes_stride = a->rows > 1 ? a->codes_stride : 0;
  P.scales_stride = a->rows > 1 ? a->scales_stride : 0;
  P.words = aligned_to(a->scales, 4) && P.scales_stride % 4 == 0;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e = a->dtype == LPS_DTYPE_F32 ? launch_quantize<LPS_DTYPE_F32>(P, s)
                       : a->dtype == LPS_DTYPE_BF16 ? launch_quantize<LPS_DTYPE_BF16>(P, s)
                                                    : launch_quantize<LPS_DTYPE_F16>(P, s);
  return e == hipSuccess ? LPS_OK : LPS_ELAUNCH;
}

int lps_mx4_dequantize(const lps_mx4_args* a, void* stream) {
  const int rc = check_mx4(a);
  if (rc != LPS_OK || a->rows == 0) return rc;
  GatherParams P{};
  P.table = a->codes;
  P.scales = static_cast<const uint8_t*>(a->scales);
  P.out = a->x;
  P.table_stride = a->rows > 1 ? a->codes_stride : 0;
  P.scales_stride = a->rows > 1 ? a->scales_stride : 0;
  P.out_stride = a->rows > 1 ? a->x_stride : 0;
  P.n = P.vocab = a->rows;
  P.hidden = a->hidden;
  P.scale = 1.0f;
  return dispatch_gather<DT_MX4>(a->dtype, P, reinterpret_cast<hipStream_t>(stream)) == hipSuccess ? LPS_OK : LPS_ELAUNCH;
}

int lps_embedding(const lps_embedding_args* a, void* stream) {
  if (!a) return LPS_EINVAL;
  const bool mx4 = a->dtype == LPS_DTYPE_MX4;
  if ((!mx4 && !dtype_ok(a->dtype)) || !dtype_ok(a->out_dtype)) return LPS_EUNSUPPORTED_DTYPE;
  if (a->n < 0 || a->vocab < 1 || a->hidden < 1 || a->hidden > MX4_MAX_HIDDEN || (a->id_bytes != 4 && a->id_bytes != 8)) return LPS_EINVAL;
  if (a->n == 0) return LPS_OK;
  if (!a->ids || !a->table || !a->out || (mx4 && !a->scales)) return LPS_EINVAL;
  if (!aligned_to(a->ids, a->id_bytes) || !aligned_to(a->table, mx4 ? 4 : elem_bytes(a->dtype)) ||
      !aligned_to(a->out, elem_bytes(a->out_dtype)))
    return LPS_EINVAL;
  const int64_t nb = blocks_of(a->hidden);
  if (a->vocab > 1 && (mx4 ? a->table_stride < 16 * nb || a->scales_stride < nb : a->table_stride < a->hidden)) return LPS_EINVAL;
  if (a->n > 1 && a->out_stride < a->hidden) return LPS_EINVAL;
  GatherParams P{};
  P.ids = a->ids;
  P.table = a->table;
  P.scales = static_cast<const uint8_t*>(a->scales);
  P.out = a->out;
  P.table_stride = a->vocab > 1 ? a->table_stride : 0;
  P.scales_stride = a->vocab > 1 ? a->scales_stride : 0;
  P.out_stride = a->n > 1 ? a->out_stride : 0;
  if (mx4 && P.table_stride % 4) return LPS_EINVAL;
  P.n = a->n;
  P.vocab = a->vocab;
  P.hidden = a->hidden;
  P.id_bytes = a->id_bytes;
  P.scale = a->scale;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  hipError_t e;
  switch (a->dtype) {
    case LPS_DTYPE_F32: e = dispatch_gather<LPS_DTYPE_F32>(a->out_dtype, P, s); break;
    case LPS_DTYPE_BF16: e = dispatch_gather<LPS_DTYPE_BF16>(a->out_dtype, P, s); break;
    case LPS_DTYPE_F16: e = dispatch_gather<LPS_DTYPE_F16>(a->out_dtype, P, s); break;
    default: e = dispatch_gather<DT_MX4>(a->out_dtype, P, s); break;
  }
  return e == hipSuccess ? LPS_OK : LPS_ELAUNCH;
}

size_t lps_embedding_grad_workspace_bytes(int n, int vocab, int hidden) {
  if (n < 0 || n > kMaxPositions || vocab < 1 || hidden < 1 || hidden > MX4_MAX_HIDDEN) return 0;
  return eg_workspace(n, vocab, hidden).bytes;
}

int lps_embedding_grad(const lps_embedding_grad_args* a, void* stream) {
  if (!a) return LPS_EINVAL;
  if (!dtype_ok(a->dtype) || !dtype_ok(a->out_dtype)) return LPS_EUNSUPPORTED_DTYPE;
  if (a->n < 0 || a->n > kMaxPositions || a->vocab < 1 || a->hidden < 1 || a->hidden > MX4_MAX_HIDDEN) return LPS_EINVAL;
  if (a->id_bytes != 4 && a->id_bytes != 8) return LPS_EINVAL;
  if (a->n == 0 && a->accumulate) return LPS_OK;
  if (!a->out || (a->n > 0 && (!a->ids || !a->grad))) return LPS_EINVAL;
  if (!aligned_to(a->ids, a->id_bytes) || !aligned_to(a->grad, elem_bytes(a->dtype)) ||
      !aligned_to(a->out, elem_bytes(a->out_dtype)))
    return LPS_EINVAL;
  if ((a->n > 1 && a->grad_stride < a->hidden) || (a->vocab > 1 && a->out_stride < a->hidden)) return LPS_EINVAL;
  const EgWs w = eg_workspace(a->n, a->vocab, a->hidden);
  if (w.bytes && (!a->workspace || a->workspace_bytes < w.bytes)) return LPS_EWORKSPACE;
  if (w.bytes && !aligned_to(a->workspace, 16)) return LPS_EINVAL;
  char* ws = static_cast<char*>(a->workspace);
  EmbGradParams P{};
  P.ids = a->ids;
  P.grad = a->grad;
  P.out = a->out;
  P.grad_stride = a->n > 1 ? a->grad_stride : 0;
  P.out_stride = a->vocab > 1 ? a->out_stride : 0;
  P.n = a->n;
  P.vocab = a->vocab;
  P.hidden = a->hidden;
  P.id_bytes = a->id_bytes;
  P.scale = a->scale;
  P.accumulate = a->accumulate ? 1 : 0;
  // workgroups of the sort: about 64 positions each, up to one on each CU; more where
  // a workgroup would own more ids than it can count
  int lg = 3;
  while (lg < 8 && ((int64_t)64 << lg) < a->n) lg++;
  while (((int64_t)a->vocab + ((int64_t)1 << lg) - 1) >> lg > EG_OWN) lg++;
  P.lg_groups = lg;
  P.S = eg_tile(a->n);
  P.tiles = (int)(((int64_t)a->n + P.S - 1) / P.S);
  P.slices = (a->hidden + 2047) / 2048;
  const int64_t row_bytes = (int64_t)a->hidden * elem_bytes(a->out_dtype);
  P.zero = !P.accumulate;
  const bool whole = P.out_stride == a->hidden;
  P.fill_rows = whole ? 1 : a->vocab;
  P.fill_bytes = whole ? a->vocab * row_bytes : row_bytes;
  P.fill_lines = aligned_to(a->out, 16) && P.out_stride * elem_bytes(a->out_dtype) % 16 == 0 ? (P.fill_bytes + 15) / 16
                                                                                            : (P.fill_bytes + 14) / 16 + 1;
  if ((int64_t)P.tiles * P.slices > kMaxGroups || (a->hidden + 255) / 256 > 65535) return LPS_EINVAL;
  P.count = reinterpret_cast<int*>(ws + w.count);
  P.sid = reinterpret_cast<int*>(ws + w.sid);
  P.spos = reinterpret_cast<int*>(ws + w.spos);
  P.tmp_id = reinterpret_cast<int*>(ws + w.tmp_id);
  P.tmp_pos = reinterpret_cast<int*>(ws + w.tmp_pos);
  P.part = reinterpret_cast<float*>(ws + w.part);
  P.part_stride = ((int64_t)a->hidden + 7) / 8 * 8;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  hipError_t e;
  switch (a->dtype) {
    case LPS_DTYPE_F32: e = dispatch_grad<LPS_DTYPE_F32>(a->out_dtype, P, s); break;
    case LPS_DTYPE_BF16: e = dispatch_grad<LPS_DTYPE_BF16>(a->out_dtype, P, s); break;
    default: e = dispatch_grad<LPS_DTYPE_F16>(a->out_dtype, P, s); break;
  }
  return e == hipSuccess ? LPS_OK : LPS_ELAUNCH;
}

}  // extern "C"
