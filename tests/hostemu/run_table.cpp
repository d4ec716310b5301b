// Host build of the vocabulary table's C ABI (llm-pipeline_amd/csrc/lps_table.hip
// and lps_mx4head.hip, unchanged) over the HIP emulation, under AddressSanitizer and
// UndefinedBehaviorSanitizer: test infrastructure for tests/test_hostemu_table.py.
//
//   run_table IN OUT
//
// IN holds one call's inputs (header int32[16], then the arrays, little-endian),
// OUT receives its outputs.  Every array is its own heap allocation of exactly
// its size.
#include "mx4_ops.h"

// The emulated device's compute units (LPS_EMU_CUS, 256 by default).
inline hipError_t emu_cus(int* v) {
  const char* e = getenv("LPS_EMU_CUS");
  *v = e ? atoi(e) : 256;
  return hipSuccess;
}
#define hipDeviceGetAttribute(v, attribute, device) emu_cus(v)

#include "../../llm-pipeline_amd/csrc/lps_table.hip"
#include "../../llm-pipeline_amd/csrc/lps_mx4head.hip"

#include <vector>

namespace {

template <typename T>
T* rd(FILE* f, size_t n) {
  T* p = static_cast<T*>(malloc(n * sizeof(T)));
  if (n && fread(p, sizeof(T), n, f) != n) {
    fprintf(stderr, "run_table: short input\n");
    exit(2);
  }
  return p;
}
uint8_t* filled(size_t n, int v) {
  uint8_t* p = static_cast<uint8_t*>(malloc(n));
  memset(p, v, n);
  return p;
}
size_t elem(int dtype) { return dtype == LPS_DTYPE_F32 ? 4 : 2; }
int ended(const char* entry, int rc) {
  if (rc) fprintf(stderr, "run_table: %s returned %d\n", entry, rc);
  return rc ? 3 : 0;
}

// {1, dtype, out_dtype, rows, hidden, x_stride, scales_stride}: x; codes, scales
// (0x5A where nothing was written), then their values.
int quantise(const int32_t* h, FILE* f, FILE* o) {
  const int rows = h[3], H = h[4], nb = (H + 31) / 32;
  const size_t n = (size_t)(rows - 1) * h[5] + H, ns = (size_t)(rows - 1) * h[6] + nb;
  uint8_t* x = rd<uint8_t>(f, n * elem(h[1]));
  uint8_t *codes = filled((size_t)rows * nb * 16, 0x5A), *scales = filled(ns, 0x5A);
  lps_mx4_args a{};
  a.x = x;
  a.codes = codes;
  a.scales = scales;
  a.dtype = h[1];
  a.rows = rows;
  a.hidden = H;
  a.x_stride = h[5];
  a.codes_stride = 16 * nb;
  a.scales_stride = h[6];
  if (int rc = ended("lps_mx4_quantize", lps_mx4_quantize(&a, nullptr))) return rc;
  const size_t on = (size_t)rows * H * elem(h[2]);
  uint8_t* v = filled(on, 0x5A);
  a.x = v;
  a.dtype = h[2];
  a.x_stride = H;
  if (int rc = ended("lps_mx4_dequantize", lps_mx4_dequantize(&a, nullptr))) return rc;
  fwrite(codes, 1, (size_t)rows * nb * 16, o);
  fwrite(scales, 1, ns, o);
  fwrite(v, 1, on, o);
  free(x); free(codes); free(scales); free(v);
  return 0;
}

// {2, dtype (3: 4-bit), out_dtype, n, vocab, hidden, id_bytes, scale's bits}:
// ids, table (codes, scales); out.
int lookup(const int32_t* h, FILE* f, FILE* o) {
  const int n = h[3], V = h[4], H = h[5], nb = (H + 31) / 32;
  uint8_t* ids = rd<uint8_t>(f, (size_t)n * h[6]);
  uint8_t* table = rd<uint8_t>(f, h[1] == 3 ? (size_t)V * nb * 16 : (size_t)V * H * elem(h[1]));
  uint8_t* scales = h[1] == 3 ? rd<uint8_t>(f, (size_t)V * nb) : nullptr;
  const size_t on = (size_t)n * H * elem(h[2]);
  uint8_t* out = filled(on, 0x5A);
  lps_embedding_args a{};
  a.ids = ids;
  a.table = table;
  a.scales = scales;
  a.out = out;
  a.id_bytes = h[6];
  a.dtype = h[1];
  a.out_dtype = h[2];
  a.n = n;
  a.vocab = V;
  a.hidden = H;
  a.table_stride = h[1] == 3 ? 16 * nb : H;
  a.scales_stride = nb;
  a.out_stride = H;
  memcpy(&a.scale, &h[7], 4);
  if (int rc = ended("lps_embedding", lps_embedding(&a, nullptr))) return rc;
  fwrite(out, 1, on, o);
  free(ids); free(table); free(scales); free(out);
  return 0;
}

// {3, dtype, out_dtype, n, vocab, hidden, id_bytes, scale's bits, accumulate}:
// ids, grad, out; out.
int gradient(const int32_t* h, FILE* f, FILE* o) {
  const int n = h[3], V = h[4], H = h[5];
  uint8_t* ids = rd<uint8_t>(f, (size_t)n * h[6]);
  uint8_t* grad = rd<uint8_t>(f, (size_t)n * H * elem(h[1]));
  uint8_t* out = rd<uint8_t>(f, (size_t)V * H * elem(h[2]));
  lps_embedding_grad_args a{};
  a.ids = ids;
  a.grad = grad;
  a.out = out;
  a.id_bytes = h[6];
  a.dtype = h[1];
  a.out_dtype = h[2];
  a.n = n;
  a.vocab = V;
  a.hidden = H;
  a.grad_stride = a.out_stride = H;
  memcpy(&a.scale, &h[7], 4);
  a.accumulate = h[8];
  a.workspace_bytes = lps_embedding_grad_workspace_bytes(n, V, H);
  a.workspace = filled(a.workspace_bytes, 0xA5);
  if (int rc = ended("lps_embedding_grad", lps_embedding_grad(&a, nullptr))) return rc;
  fwrite(out, 1, (size_t)V * H * elem(h[2]), o);
  free(ids); free(grad); free(out); free(a.workspace);
  return 0;
}

// {4, dtype (3: 4-bit), out_dtype, rows, vocab, hidden, x_stride, scales_stride}:
// x (x scales), w, w scales; out, stats.
int head(const int32_t* h, FILE* f, FILE* o) {
  const int M = h[3], V = h[4], H = h[5], nb = (H + 31) / 32, G = (V + 127) / 128;
  const bool x4 = h[1] == 3;
  uint8_t* x = rd<uint8_t>(f, x4 ? (size_t)M * nb * 16 : ((size_t)(M - 1) * h[6] + H) * 2);
  uint8_t* xs = x4 ? rd<uint8_t>(f, (size_t)(M - 1) * h[7] + nb) : nullptr;
  uint8_t* w = rd<uint8_t>(f, (size_t)V * nb * 16);
  uint8_t* ws = rd<uint8_t>(f, (size_t)(V - 1) * h[7] + nb);
  const size_t on = (size_t)M * V * elem(h[2]), sn = (size_t)M * G * 8;
  uint8_t *out = filled(on, 0x5A), *stats = filled(sn, 0x5A);
  lps_lm_head_mx4_args a{};
  a.x = x;
  a.x_scales = xs;
  a.w = w;
  a.w_scales = ws;
  a.out = out;
  a.stats = reinterpret_cast<float*>(stats);
  a.dtype = h[1];
  a.out_dtype = h[2];
  a.rows = M;
  a.vocab = V;
  a.hidden = H;
  a.x_stride = x4 ? 16 * nb : h[6];
  a.x_scales_stride = a.w_scales_stride = h[7];
  a.w_stride = 16 * nb;
  a.out_stride = V;
  if (int rc = ended("lps_lm_head_mx4", lps_lm_head_mx4(&a, nullptr))) return rc;
  fwrite(out, 1, on, o);
  fwrite(stats, 1, sn, o);
  free(x); free(xs); free(w); free(ws); free(out); free(stats);
  return 0;
}

// {5, entry (1 to 4 as above, 5 dequantises), dtype, out_dtype, rows or n, vocab, hidden, accumulate}: the
// entry point's launches alone (LPS_EMU_LAUNCHES), over addresses that nothing is at;
// its return code.
int launches(const int32_t* h, FILE* o) {
  if (!getenv("LPS_EMU_LAUNCHES")) return 2;
  char* const at = reinterpret_cast<char*>((uintptr_t)1 << 40);
  const int dtype = h[2], out_dtype = h[3], n = h[4], V = h[5], H = h[6], nb = (H + 31) / 32;
  int32_t rc = -1;
  if (h[1] == 1 || h[1] == 5) {
    lps_mx4_args a{at, at, at, dtype, n, H, H, 16 * nb, nb};
    rc = h[1] == 1 ? lps_mx4_quantize(&a, nullptr) : lps_mx4_dequantize(&a, nullptr);
  } else if (h[1] == 2) {
    lps_embedding_args a{at, at, at, at, 8, dtype, out_dtype, n, V, H, dtype == 3 ? 16 * nb : H, nb, H, 1.0f};
    rc = lps_embedding(&a, nullptr);
  } else if (h[1] == 3) {
    lps_embedding_grad_args a{at, at, at, 8, dtype, out_dtype, n, V, H, H, H, 1.0f, h[7], at,
                              lps_embedding_grad_workspace_bytes(n, V, H)};
    rc = lps_embedding_grad(&a, nullptr);
  } else if (h[1] == 4) {
    const int ss = (nb + 3) & ~3;
    lps_lm_head_mx4_args a{at, at, at, at, at, nullptr, dtype, out_dtype, n, V, H,
                           dtype == 3 ? 16 * nb : (H + 7) & ~7, ss, 16 * nb, ss, V};
    rc = lps_lm_head_mx4(&a, nullptr);
  }
  fwrite(&rc, 4, 1, o);
  return 0;
}

}  // namespace

int main(int argc, char** argv) {
  if (argc != 3) return 2;
  FILE* f = fopen(argv[1], "rb");
  FILE* o = fopen(argv[2], "wb");
  if (!f || !o) return 2;
  int32_t h[16];
  if (fread(h, 4, 16, f) != 16) return 2;
  const int rc = h[0] == 1 ? quantise(h, f, o) : h[0] == 2 ? lookup(h, f, o) : h[0] == 3 ? gradient(h, f, o) : h[0] == 4 ? head(h, f, o) : h[0] == 5 ? launches(h, o) : 2;
  fclose(f);
  fclose(o);
  return rc;
}
