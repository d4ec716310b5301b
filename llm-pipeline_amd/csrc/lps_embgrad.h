// Gradient of the embedding lookup, without atomics on values:
//   out[v] = scale * sum over the positions i with id_i = v of grad[i]
// (added to out[v] when accumulating), summed in fp32 in one fixed order, so a
// call's result never depends on timing.
//
// 1. grad_sort_kernel groups the positions by id.  Workgroup w of G takes the
//    ids with id % G == w (neighbouring frequent ids land apart); it reads all
//    ids, counts its own and those of the workgroups before it (its place in
//    the order, so no workgroup waits for another), and places its positions by
//    id, in their own order.
// 2. grad_tiles_kernel cuts that order into tiles of S positions (a frequent id
//    costs no one workgroup more than another) and adds the gradient rows of
//    each run of one id.  A run inside a tile is written at once; a run's part
//    in a tile that it enters or leaves goes to that tile's partial rows.  For a
//    new gradient more workgroups of the launch zero the rows without a token.
// 3. grad_join_kernel adds the partial rows of each run that crosses tiles.
#pragma once

#include "lps_common.h"
#include "lps_mx4.h"
#include "lps_wave.h"

namespace lps {

constexpr int EG_NT = 1024;         // threads of the sort
constexpr int EG_NW = EG_NT / 64;
constexpr int EG_HIST = 16384;      // ids a workgroup of the sort can own
constexpr int EG_LIST = 4096;       // positions it keeps in LDS
constexpr int EG_SMAX = 256;        // positions of a tile, at most
constexpr int EG_FILL_ROWS = 16;    // rows a zeroing workgroup looks at

struct EmbGradParams {
  const void* ids;
  const void* grad;      // [n, hidden]
  void* out;             // [vocab, hidden]
  int64_t grad_stride, out_stride;   // elements
  int n, vocab, hidden, id_bytes;
  float scale;
  int accumulate;
  int lg_groups;         // log2 G
  int S, tiles, slices;  // positions of a tile; tiles; workgroups on a tile
  // workspace
  int* count;            // [1] positions with a valid id
  int* sid;              // [n] ids in the order
  int* spos;             // [n] positions in the order
  int* tmp_id;           // [n] lists that outgrow LDS
  int* tmp_pos;          // [n]
  uint8_t* touched;      // [vocab], new gradients
  float* part;           // [2 tiles, part_stride]: runs entering, runs leaving
  int64_t part_stride;
};

__global__ __launch_bounds__(EG_NT) void grad_sort_kernel(EmbGradParams P) {
  __shared__ uint32_t hist[EG_HIST];
  __shared__ int list_id[EG_LIST], list_pos[EG_LIST];
  __shared__ int wcnt[EG_NW], wless[EG_NW], wall[EG_NW];
  __shared__ uint32_t wsum[EG_NW];
  const int tid = (int)threadIdx.x, wv = tid >> 6, l = tid & 63;
  const int w = (int)blockIdx.x, lg = P.lg_groups, mask = (1 << lg) - 1;
  const int own = w < P.vocab ? (P.vocab - 1 - w) / (mask + 1) + 1 : 0;   // ids w, w + G, ..
  for (int k = tid; k < own; k += EG_NT) hist[k] = 0;
  __syncthreads();
  // each wave takes a run of positions, 64 at a time
  const int per = ((P.n + EG_NW - 1) / EG_NW + 63) & ~63;
  const int64_t a64 = (int64_t)wv * per;
  const int a = a64 < P.n ? (int)a64 : P.n, b = P.n - a < per ? P.n : a + per;
  constexpr int U = 8;
  int cnt = 0, less = 0, all = 0;
  for (int i0 = a; i0 < b; i0 += 64 * U) {
    int64_t id[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t i = (int64_t)i0 + 64 * u + l;
      id[u] = i < b ? load_id(P.ids, P.id_bytes, i) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const bool valid = id[u] >= 0 && id[u] < P.vocab;
      const int g = (int)id[u] & mask;
      const bool mine = valid && g == w;
      cnt += __builtin_popcountll(wballot(mine));
      less += __builtin_popcountll(wballot(valid && g < w));
      all += __builtin_popcountll(wballot(valid));
      if (mine) atomicAdd(&hist[(int)id[u] >> lg], 1u);
    }
  }
  if (l == 0) { wcnt[wv] = cnt; wless[wv] = less; wall[wv] = all; }
  __syncthreads();
  int start = 0, total = 0, mine0 = 0, every = 0;
  for (int k = 0; k < EG_NW; k++) {
    start += wless[k];
    mine0 += k < wv ? wcnt[k] : 0;
    total += wcnt[k];
    every += wall[k];
  }
  if (w == 0 && tid == 0) *P.count = every;
  if (P.touched)
    for (int k = tid; k < own; k += EG_NT) P.touched[w + ((int64_t)k << lg)] = hist[k] != 0;
  if (total == 0) return;                          // (uniform over the workgroup)
  // the ids' first places: an exclusive scan of the counts, a run of them per thread
  {
    const int run = (own + EG_NT - 1) / EG_NT, k0 = tid * run;
    uint32_t s = 0;
    for (int k = k0; k < k0 + run && k < own; k++) s += hist[k];
    const uint32_t incl = wscan_incl(s);
    if (l == 63) wsum[wv] = incl;
    __syncthreads();
    uint32_t at = incl - s;
    for (int k = 0; k < wv; k++) at += wsum[k];
    for (int k = k0; k < k0 + run && k < own; k++) {
      const uint32_t c = hist[k];
      hist[k] = at;
      at += c;
    }
  }
  // the workgroup's positions in their own order
  const bool in_lds = total <= EG_LIST;
  int* const gid = P.tmp_id + start;
  int* const gpos = P.tmp_pos + start;
  int at = mine0;
  for (int i0 = a; i0 < b; i0 += 64 * U) {
    int64_t id[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t i = (int64_t)i0 + 64 * u + l;
      id[u] = i < b ? load_id(P.ids, P.id_bytes, i) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const bool mine = id[u] >= 0 && id[u] < P.vocab && ((int)id[u] & mask) == w;
      const uint64_t m = wballot(mine);
      if (mine) {
        const int k = at + (int)lanes_below(m), i = i0 + 64 * u + l;
        if (in_lds) { list_id[k] = (int)id[u] >> lg; list_pos[k] = i; }
        else { gid[k] = (int)id[u] >> lg; gpos[k] = i; }
      }
      at += __builtin_popcountll(m);
    }
  }
  __syncthreads();
  if (wv != 0) return;
  // 64 at a time: a position's place is its id's next one, after the lower
  // lanes of the same id (found bit by bit of the id)
  const int bits = 32 - __builtin_clz((uint32_t)own);
  for (int k0 = 0; k0 < total; k0 += 64) {
    const int k = k0 + l;
    const bool on = k < total;
    const int id = on ? (in_lds ? list_id[k] : gid[k]) : 0;
    const int pos = on ? (in_lds ? list_pos[k] : gpos[k]) : 0;
    uint64_t same = wballot(on);
    for (int q = 0; q < bits; q++) {
      const bool one = (id >> q) & 1;
      const uint64_t m = wballot(one);
      same &= one ? m : ~m;
    }
    const int rank = (int)lanes_below(same), first = same ? __builtin_ctzll(same) : l;
    uint32_t base = 0;
    if (on && rank == 0) base = atomicAdd(&hist[id], (uint32_t)__builtin_popcountll(same));
    base = (uint32_t)__shfl((int)base, first, 64);
    if (on) {
      P.sid[start + (int)base + rank] = (id << lg) + w;
      P.spos[start + (int)base + rank] = pos;
    }
  }
}

// scale * acc to row id of the gradient, on top of it when accumulating.
template <int ODT>
__device__ __forceinline__ void grad_write(const EmbGradParams& P, int id, int e0, const float (&acc)[8]) {
  char* row = static_cast<char*>(P.out) + (int64_t)id * P.out_stride * ElemBytes<ODT>::value;
  float v[8];
  if (P.accumulate) {
    piece_values(load_piece<ODT>(row, e0, P.hidden), v);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = __builtin_fmaf(P.scale, acc[e], v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = __fmul_rn(P.scale, acc[e]);
  }
  store_piece<ODT>(row, e0, P.hidden, v);
}

template <int GDT, int ODT>
__global__ __launch_bounds__(256) void grad_tiles_kernel(EmbGradParams P) {
  __shared__ int s_id[EG_SMAX + 2], s_pos[EG_SMAX];
  const int tid = (int)threadIdx.x;
  const int64_t work = (int64_t)P.tiles * P.slices;
  if (blockIdx.x >= work) {
    // rows without a token
    const int64_t r0 = ((int64_t)blockIdx.x - work) * EG_FILL_ROWS;
    const float zero[8] = {};
    for (int r = 0; r < EG_FILL_ROWS; r++) {
      const int64_t row = r0 + r;
      if (row >= P.vocab || P.touched[row]) continue;
      char* o = static_cast<char*>(P.out) + row * P.out_stride * ElemBytes<ODT>::value;
      for (int e0 = 8 * tid; e0 < P.hidden; e0 += 8 * 256) store_piece<ODT>(o, e0, P.hidden, zero);
    }
    return;
  }
  const int t = (int)(blockIdx.x / (unsigned)P.slices), sl = (int)(blockIdx.x % (unsigned)P.slices);
  const int nv = *P.count;
  const int64_t base64 = (int64_t)t * P.S;
  if (base64 >= nv) return;                        // (uniform over the workgroup)
  const int base = (int)base64, m = nv - base < P.S ? nv - base : P.S;
  // ids base - 1 .. base + m (-1 past the order's ends)
  for (int k = tid; k < m + 2; k += 256) {
    const int j = base - 1 + k;
    s_id[k] = j >= 0 && j < nv ? P.sid[j] : -1;
    if (k < m) s_pos[k] = P.spos[base + k];
  }
  __syncthreads();
  const int e0 = 8 * (sl * 256 + tid);
  if (e0 >= P.hidden) return;
  float acc[8] = {};
  int run0 = 0;
  auto flush = [&](int id, int end) {              // the run of positions run0 .. end - 1
    const bool enters = run0 == 0 && s_id[0] == id;
    const bool leaves = end == m && s_id[m + 1] == id;
    if (enters || leaves) {
      float* d = P.part + ((int64_t)2 * t + (enters ? 0 : 1)) * P.part_stride + e0;
#pragma unroll
      for (int e = 0; e < 8; e += 4) *reinterpret_cast<u32x4*>(d + e) = u32x4{__float_as_uint(acc[e]),
          __float_as_uint(acc[e + 1]), __float_as_uint(acc[e + 2]), __float_as_uint(acc[e + 3])};
    } else {
      grad_write<ODT>(P, id, e0, acc);
    }
  };
  constexpr int U = GDT == LPS_DTYPE_F32 ? 4 : 8;
  int cur = __builtin_amdgcn_readfirstlane(s_id[1]);
  for (int i0 = 0; i0 < m; i0 += U) {
    Piece<GDT> g[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t pos = __builtin_amdgcn_readfirstlane(s_pos[i0 + u < m ? i0 + u : m - 1]);
      if (i0 + u < m)
        g[u] = load_piece<GDT, true>(static_cast<const char*>(P.grad) + pos * P.grad_stride * ElemBytes<GDT>::value, e0, P.hidden);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (i0 + u < m) {
        const int id = __builtin_amdgcn_readfirstlane(s_id[1 + i0 + u]);
        if (id != cur) {
          flush(cur, i0 + u);
          cur = id;
          run0 = i0 + u;
#pragma unroll
          for (int e = 0; e < 8; e++) acc[e] = 0.0f;
        }
        float v[8];
        piece_values(g[u], v);
#pragma unroll
        for (int e = 0; e < 8; e++) acc[e] = __fadd_rn(acc[e], v[e]);
      }
    }
  }
  flush(cur, m);
}

// One workgroup per tile and 256 columns: 32 threads of eight columns, eight of
// them on every eighth partial row, added in order at the end.
template <int ODT>
__global__ __launch_bounds__(256) void grad_join_kernel(EmbGradParams P) {
  __shared__ float red[8][256 + 8];
  const int t = (int)blockIdx.x, nv = *P.count;
  const int64_t end = ((int64_t)t + 1) * P.S;
  if (end >= nv) return;                           // the order's last tile: no run leaves it
  const int id = P.sid[end - 1];
  if (P.sid[end] != id) return;
  const int64_t base = end - P.S;
  if (base > 0 && P.sid[base] == id && P.sid[base - 1] == id) return;   // the run began in an earlier tile
  const int c = (int)threadIdx.x & 31, k = (int)threadIdx.x >> 5;
  const int e0 = 256 * (int)blockIdx.y + 8 * c;
  float acc[8] = {};
  if (e0 < P.hidden) {
    auto add = [&](int64_t row) {
      const u32x4* p = reinterpret_cast<const u32x4*>(P.part + row * P.part_stride + e0);
      const u32x4 x = p[0], y = p[1];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        acc[e] = __fadd_rn(acc[e], __uint_as_float(x[e]));
        acc[4 + e] = __fadd_rn(acc[4 + e], __uint_as_float(y[e]));
      }
    };
    if (k == 0) add(2 * (int64_t)t + 1);
    for (int64_t q = (int64_t)t + 1 + k; q * P.S < nv && P.sid[q * P.S] == id; q += 8) add(2 * q);
  }
#pragma unroll
  for (int e = 0; e < 8; e++) red[k][8 * c + e] = acc[e];
  __syncthreads();
  if (k == 0 && e0 < P.hidden) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      float s = acc[e];
#pragma unroll
      for (int q = 1; q < 8; q++) s = __fadd_rn(s, red[q][8 * c + e]);
      acc[e] = s;
    }
    grad_write<ODT>(P, id, e0, acc);
  }
}

}  // namespace lps
