// Gradient of the embedding lookup, without atomics on values:
//   out[v] = scale * sum over the positions i with id_i = v of grad[i]
// (added to out[v] when accumulating), summed in fp32 in one fixed order, so a
// call's result never depends on timing.
//
// Up to EG_SMALL positions grad_small_kernel, after grad_zero_kernel where there are
// many zeros to write; of none grad_zero_kernel alone.  More, three launches:
// 1. grad_sort_kernel groups the positions by id.  Workgroup w of G takes the
//    ids with id % G == w (neighbouring frequent ids land apart); it reads all
//    ids, counts its own and those of the workgroups before it (its place in
//    the order, so no workgroup waits for another), and places its positions by
//    id, in their own order.  For a new gradient more workgroups of the launch write
//    zeros to all rows meanwhile.
// 2. grad_tiles_kernel cuts that order into tiles of S positions (a frequent id
//    costs no one workgroup more than another) and adds the gradient rows of
//    each run of one id.  A run inside a tile is written at once; a run's part
//    in a tile that it enters or leaves goes to that tile's partial rows.
// 3. grad_join_kernel adds the partial rows of each run that crosses tiles.
#pragma once

#include "lps_common.h"
#include "lps_mx4.h"
#include "lps_wave.h"

namespace lps {

constexpr int EG_NT = 1024;         // threads of the sort
constexpr int EG_NW = EG_NT / 64;
constexpr int EG_OWN = 1024;        // ids a workgroup of the sort can own
constexpr int EG_LIST = 3968;       // positions it keeps in LDS: as many as leave room for two workgroups a CU
constexpr int EG_POS_BITS = 22;     // .. whose ids take the other 10
constexpr int EG_SMAX = 1024;       // positions of a tile, at most
constexpr int EG_FILL = (1 << 21) - 8;   // workgroups that write zeros: at most
constexpr int EG_JOIN = 8;          // tiles a joining workgroup looks at
constexpr int EG_SMALL = 768;       // positions of the form without a sort

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
  int zero;              // grad_small_kernel: rows without a token become zero
  // zeros: rows of the output, or all of it as one where they are neighbours (8192
  // positions into 151936 rows of 1601 fp32: 193 us against 271)
  int64_t fill_bytes;    // of such a row
  int fill_rows;
  int64_t fill_lines;    // 16-byte lines that it can lie in
  // workspace
  int* count;            // [1] positions with a valid id
  int* sid;              // [n] ids in the order
  int* spos;             // [n] positions in the order
  int* tmp_id;           // [n] lists that outgrow LDS
  int* tmp_pos;          // [n]
  float* part;           // [2 tiles, part_stride]: runs entering, runs leaving
  int64_t part_stride;
};

// Zeros to all rows of a new gradient, those with a token among them: they are
// written again by a later launch, and leaving them out costs more (1.2 GB 250 us).
// Chunk c is 256 of the 16-byte lines that the rows lie in, one of them a thread's.
template <int ODT>
__device__ __forceinline__ void grad_zero_chunk(const EmbGradParams& P, int64_t c, int t) {
  constexpr int ES = ElemBytes<ODT>::value;
  int64_t row = 0, q = c * 256;                    // (the row and its line: by scalar divisions up to the chunk's first)
  if (P.fill_rows > 1) {                           // (fewer than 2^32 lines a row)
    const uint32_t lines = (uint32_t)P.fill_lines;
    uint32_t k;
    if (q >> 32) {
      row = q / lines;
      k = (uint32_t)(q - row * lines);
    } else {
      row = (uint32_t)q / lines;
      k = (uint32_t)q % lines;
    }
    k += t;
    row += k / lines;
    q = k % lines;
  } else {
    q += t;
  }
  if (row >= P.fill_rows) return;
  // the line whole, or the row's part of it
  const int64_t bytes = P.fill_bytes;
  const uintptr_t p = reinterpret_cast<uintptr_t>(P.out) + row * P.out_stride * ES;
  const uintptr_t line = (p & ~(uintptr_t)15) + (uintptr_t)q * 16;
  if (line >= p && line + 16 <= p + bytes) {
    *reinterpret_cast<u32x4*>(line) = u32x4{};
  } else {
#pragma unroll
    for (int e = 0; e < 16; e += ES) {
      if (line + e >= p && line + e < p + bytes) {
        if constexpr (ES == 4) *reinterpret_cast<uint32_t*>(line + e) = 0;
        else *reinterpret_cast<uint16_t*>(line + e) = 0;
      }
    }
  }
}
// Workgroup wg of wgs, NT threads: NT / 256 chunks at a time.  Memory takes zeros best
// in its order, and where chunks of 4 KB go to the XCDs in turn, as workgroups do:
// 1.2 GB in workgroups of 256 take 181 us with a chunk each and 195 with two
// neighbouring ones; beside the sort, in workgroups of 1024, 195 with every eighth
// chunk, 217 with four neighbouring ones and 250 in a loop of 512 workgroups.
template <int ODT, int NT>
__device__ __forceinline__ void grad_zero(const EmbGradParams& P, int wg, int wgs) {
  const int64_t chunks = (P.fill_rows * P.fill_lines + 255) >> 8;
  constexpr int C = NT / 256;
  const int part = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 8);
  for (int64_t w = wg; (w >> 3) * (8 * C) < chunks; w += wgs)
    grad_zero_chunk<ODT>(P, (w >> 3) * (8 * C) + 8 * part + (w & 7), (int)threadIdx.x & 255);
}
template <int ODT>
__global__ __launch_bounds__(256) void grad_zero_kernel(EmbGradParams P) {
  grad_zero<ODT, 256>(P, (int)blockIdx.x, (int)gridDim.x);
}

// What bounds the sort is latency: every workgroup reads all ids (from its L2), lists
// its own in order (waves take runs of positions), and cuts the list into a run per
// wave: counts by id and wave, one scan over both, and each wave places its run.
// 8192 ids 9 us, 32768 15.5 us (with one wave that places the whole list 17 and 27).
// 64 VGPRs and half of a CU's LDS, so that a workgroup that writes zeros runs beside it.
template <int ODT>
__global__ __launch_bounds__(EG_NT, 8) void grad_sort_kernel(EmbGradParams P) {
  __shared__ uint32_t count[EG_NW][EG_OWN];        // positions of an id in a wave's run; then their next place
  __shared__ uint32_t list[EG_LIST];
  __shared__ int wcnt[EG_NW], wless[EG_NW], wall[EG_NW];
  __shared__ uint32_t wsum[EG_NW];
  const int tid = (int)threadIdx.x, wv = tid >> 6, l = tid & 63;
  const int w = (int)blockIdx.x, lg = P.lg_groups, mask = (1 << lg) - 1;
  if (w > mask) {
    grad_zero<ODT, EG_NT>(P, w - mask - 1, (int)gridDim.x - mask - 1);
    return;
  }
  const int own = w < P.vocab ? (P.vocab - 1 - w) / (mask + 1) + 1 : 0;   // ids w, w + G, ..
  // each wave takes a run of positions, 64 U at a time
  const int per = ((P.n + EG_NW - 1) / EG_NW + 63) & ~63;
  const int64_t a64 = (int64_t)wv * per;
  const int a = a64 < P.n ? (int)a64 : P.n, b = P.n - a < per ? P.n : a + per;
  static_assert(EG_OWN == 1 << (32 - EG_POS_BITS), "an id and a position to a word");
  constexpr int U = 4, R = 8;
  constexpr int NONE = 0xFFFF;                     // an id of another workgroup's
  uint32_t kept[R][U / 2];                         // R batches for the second pass: ids' places among the own ones
  int cnt = 0, less = 0, all = 0;                  // this lane's
  auto fetch = [&](int i0, int (&place)[U], bool tally) {
    int64_t v[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t i = (int64_t)i0 + 64 * u + l;
      v[u] = i < b ? load_id(P.ids, P.id_bytes, i) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const bool valid = v[u] >= 0 && v[u] < P.vocab;
      const int g = (int)v[u] & mask;
      place[u] = valid && g == w ? (int)v[u] >> lg : NONE;
      if (tally) {
        cnt += valid && g == w;
        less += valid && g < w;
        all += valid;
      }
    }
  };
  for (int k = l; k < own; k += 64) count[wv][k] = 0;
#pragma unroll
  for (int r = 0; r < R; r++) {
    if ((int64_t)a + 64 * U * r < b) {
      int place[U];
      fetch(a + 64 * U * r, place, true);
#pragma unroll
      for (int u = 0; u < U; u += 2) kept[r][u / 2] = (uint32_t)place[u] | (uint32_t)place[u + 1] << 16;
    }
  }
  for (int64_t i0 = (int64_t)a + 64 * U * R; i0 < b; i0 += 64 * U) {
    int place[U];
    fetch((int)i0, place, true);
  }
  cnt = lps::wsum(cnt);
  less = lps::wsum(less);
  all = lps::wsum(all);
  if (l == 0) { wcnt[wv] = cnt; wless[wv] = less; wall[wv] = all; }
  __syncthreads();
  int start = 0, total = 0, at = 0, every = 0;
  for (int k = 0; k < EG_NW; k++) {
    start += wless[k];
    at += k < wv ? wcnt[k] : 0;
    total += wcnt[k];
    every += wall[k];
  }
  if (w == 0 && tid == 0) *P.count = every;
  // the workgroup's positions in their own order
  const bool in_lds = total <= EG_LIST && P.n <= 1 << EG_POS_BITS;
  int* const gid = P.tmp_id + start;
  int* const gpos = P.tmp_pos + start;
  auto append = [&](int i0, const int (&place)[U]) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const bool mine = place[u] != NONE;
      const uint64_t m = wballot(mine);
      if (mine) {
        const int k = at + (int)lanes_below(m), i = i0 + 64 * u + l;
        if (in_lds) list[k] = (uint32_t)place[u] << EG_POS_BITS | (uint32_t)i;
        else { gid[k] = place[u]; gpos[k] = i; }
      }
      at += __builtin_popcountll(m);
    }
  };
#pragma unroll
  for (int r = 0; r < R; r++) {
    if ((int64_t)a + 64 * U * r < b) {
      int place[U];
#pragma unroll
      for (int u = 0; u < U; u++) place[u] = (int)(kept[r][u / 2] >> (16 * (u & 1)) & 0xFFFF);
      append(a + 64 * U * r, place);
    }
  }
  for (int64_t i0 = (int64_t)a + 64 * U * R; i0 < b; i0 += 64 * U) {
    int place[U];
    fetch((int)i0, place, false);
    append((int)i0, place);
  }
  __syncthreads();
  // this wave's run of the list
  const int run = ((total + EG_NW - 1) / EG_NW + 63) & ~63;
  const int k0 = wv * run < total ? wv * run : total, k1 = total - k0 < run ? total : k0 + run;
  for (int k = k0 + l; k < k1; k += 64) atomicAdd(&count[wv][in_lds ? (int)(list[k] >> EG_POS_BITS) : gid[k]], 1u);
  __syncthreads();
  {
    // a thread's id: its positions over the waves, its place over the ids
    uint32_t s = 0;
    if (tid < own) {
#pragma unroll
      for (int k = 0; k < EG_NW; k++) s += count[k][tid];
    }
    const uint32_t incl = wscan_incl(s);
    if (l == 63) wsum[wv] = incl;
    __syncthreads();
    uint32_t p = incl - s;
    for (int k = 0; k < wv; k++) p += wsum[k];
    if (tid < own) {
#pragma unroll
      for (int k = 0; k < EG_NW; k++) {
        const uint32_t c = count[k][tid];
        count[k][tid] = p;
        p += c;
      }
    }
  }
  __syncthreads();
  // 64 positions at a time: a position's place is its id's next one in this run, after
  // the lower lanes of the same id (found bit by bit of the id)
  const int bits = 32 - __builtin_clz((uint32_t)own | 1u);
  for (int q = k0; q < k1; q += 64) {
    const int k = q + l;
    const bool on = k < k1;
    int id = 0, pos = 0;
    if (on) {
      const uint32_t x = in_lds ? list[k] : 0;
      id = in_lds ? (int)(x >> EG_POS_BITS) : gid[k];
      pos = in_lds ? (int)(x & ((1u << EG_POS_BITS) - 1)) : gpos[k];
    }
    uint64_t same = wballot(on);
    for (int i = 0; i < bits; i++) {
      const bool one = (id >> i) & 1;
      const uint64_t m = wballot(one);
      same &= one ? m : ~m;
    }
    const int rank = (int)lanes_below(same), first = same ? __builtin_ctzll(same) : l;
    uint32_t base = 0;
    if (on && rank == 0) base = atomicAdd(&count[wv][id], (uint32_t)__builtin_popcountll(same));
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

// Columns e0 .. e0 + 7 of the eight threads that share them added in order: true in
// the first of the eight, with the sum in acc.
__device__ __forceinline__ bool grad_reduce8(float (&red)[8][256 + 8], int c, int k, float (&acc)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e++) red[k][8 * c + e] = acc[e];
  __syncthreads();
  if (k == 0) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      float s = acc[e];
#pragma unroll
      for (int q = 1; q < 8; q++) s = __fadd_rn(s, red[q][8 * c + e]);
      acc[e] = s;
    }
  }
  __syncthreads();
  return k == 0;
}

// One workgroup per EG_JOIN tiles and 256 columns, 32 threads of eight columns to a
// tile: they add the partial rows of the run that begins in it and leaves it, or,
// where it goes through more than EG_LONG tiles, all 256 do, every eighth row each
// and those eight sums in order.
constexpr int EG_LONG = 16;
template <int ODT>
__global__ __launch_bounds__(256) void grad_join_kernel(EmbGradParams P) {
  static_assert(EG_JOIN == 8, "a group of threads to a tile");
  __shared__ float red[8][256 + 8];
  __shared__ int s_id[EG_JOIN], s_tiles[EG_JOIN];
  const int nv = *P.count;
  const int c = (int)threadIdx.x & 31, k = (int)threadIdx.x >> 5;
  const int e0 = 256 * (int)blockIdx.y + 8 * c;
  auto add = [&](int64_t row, float (&acc)[8]) {
    const u32x4* p = reinterpret_cast<const u32x4*>(P.part + row * P.part_stride + e0);
    const u32x4 x = p[0], y = p[1];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      acc[e] = __fadd_rn(acc[e], __uint_as_float(x[e]));
      acc[4 + e] = __fadd_rn(acc[4 + e], __uint_as_float(y[e]));
    }
  };
  const int64_t t0 = (int64_t)blockIdx.x * EG_JOIN;
  {
    // tile t0 + k: not the order's last one, not one inside a run
    const int64_t t = t0 + k, base = t * P.S, end = base + P.S;
    int id = 0, tiles = 0;                         // (of the run: after this one)
    bool open = false;
    if (end < nv) {
      id = P.sid[end - 1];
      open = P.sid[end] == id && !(base > 0 && P.sid[base] == id && P.sid[base - 1] == id);
    }
    // the next tiles that begin with the id, 32 looked at at a time (two tiles a wave)
    while (wballot(open)) {
      const int64_t q = (t + 1 + tiles + c) * P.S;
      const uint64_t all = wballot(open && q < nv && P.sid[q < nv ? q : 0] == id);
      const uint32_t m = ~(uint32_t)(all >> (32 * (k & 1)));
      if (open) tiles += m ? __builtin_ctz(m) : 32;
      open = open && m == 0;
    }
    if (c == 0) {
      s_id[k] = id;
      s_tiles[k] = tiles;
    }
    if (tiles > 0 && tiles <= EG_LONG && e0 < P.hidden) {
      float acc[8] = {};
      add(2 * t + 1, acc);
#pragma unroll 4
      for (int q = 0; q < tiles; q++) add(2 * (t + 1 + q), acc);
      grad_write<ODT>(P, id, e0, acc);
    }
  }
  __syncthreads();
  for (int j = 0; j < EG_JOIN; j++) {
    const int tiles = s_tiles[j];
    if (tiles <= EG_LONG) continue;                // (uniform over the workgroup)
    const int64_t t = t0 + j;
    float acc[8] = {};
    if (e0 < P.hidden) {
      if (k == 0) add(2 * t + 1, acc);
#pragma unroll 4
      for (int q = k; q < tiles; q += 8) add(2 * (t + 1 + q), acc);
    }
    if (grad_reduce8(red, c, k, acc) && e0 < P.hidden) grad_write<ODT>(P, s_id[j], e0, acc);
  }
}

// ---------------------------------------------------------------------------
// Few positions, one launch.  Workgroup (w, y) owns the ids with id % G == w and
// 256 columns; it lists its positions in order and adds their rows: an id of few
// positions by 32 threads (eight ids at a time), of more by all eight such
// groups, every eighth listed position each.  Its other rows become zero.
// ---------------------------------------------------------------------------
template <int GDT, int ODT>
__global__ __launch_bounds__(256) void grad_small_kernel(EmbGradParams P) {
  __shared__ int first[EG_OWN];              // an id's first place in the list, and how often it is there
  __shared__ uint32_t times[EG_OWN];
  __shared__ unsigned short list_id[EG_SMALL], list_pos[EG_SMALL];
  __shared__ int wcnt[4];
  __shared__ float red[8][256 + 8];
  const int tid = (int)threadIdx.x, wv = tid >> 6, l = tid & 63;
  const int w = (int)blockIdx.x, lg = P.lg_groups, mask = (1 << lg) - 1;
  const int own = w < P.vocab ? (P.vocab - 1 - w) / (mask + 1) + 1 : 0;
  constexpr int U = EG_SMALL / 256;
  const int per = EG_SMALL / 4, a = wv * per;      // this wave's positions, 64 at a time
  int id[U], cnt = 0;
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int i = a + 64 * u + l;
    const int64_t v = i < P.n ? load_id(P.ids, P.id_bytes, i) : -1;
    id[u] = v >= 0 && v < P.vocab && ((int)v & mask) == w ? (int)v >> lg : -1;
    cnt += __builtin_popcountll(wballot(id[u] >= 0));
  }
  for (int k = tid; k < own; k += 256) {
    first[k] = EG_SMALL;
    times[k] = 0;
  }
  if (l == 0) wcnt[wv] = cnt;
  __syncthreads();
  int at = 0, total = 0;
  for (int k = 0; k < 4; k++) {
    at += k < wv ? wcnt[k] : 0;
    total += wcnt[k];
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint64_t m = wballot(id[u] >= 0);
    if (id[u] >= 0) {
      const int k = at + (int)lanes_below(m);
      list_id[k] = (unsigned short)id[u];
      list_pos[k] = (unsigned short)(a + 64 * u + l);
      atomicMin(&first[id[u]], k);
      atomicAdd(&times[id[u]], 1u);
    }
    at += __builtin_popcountll(m);
  }
  __syncthreads();
  const int c = tid & 31, k = tid >> 5;
  const int e0 = 256 * (int)blockIdx.y + 8 * c;
  const bool in = e0 < P.hidden;
  constexpr uint32_t FEW = 16;
  // the rows of list places j0, j0 + step, .. that hold the id
  auto add = [&](int want, int j0, int step, float (&acc)[8]) {
    constexpr int B = 4;
    for (int j = j0; j < total; j += step * B) {
      Piece<GDT> g[B];
      bool on[B];
#pragma unroll
      for (int u = 0; u < B; u++) {
        const int p = j + u * step;
        on[u] = p < total && list_id[p] == want;
        if (on[u])
          g[u] = load_piece<GDT>(static_cast<const char*>(P.grad) + (int64_t)list_pos[p] * P.grad_stride * ElemBytes<GDT>::value,
                                 e0, P.hidden);
      }
#pragma unroll
      for (int u = 0; u < B; u++) {
        if (on[u]) {
          float v[8];
          piece_values(g[u], v);
#pragma unroll
          for (int e = 0; e < 8; e++) acc[e] = __fadd_rn(acc[e], v[e]);
        }
      }
    }
  };
  if (in) {
    for (int j = k; j < total; j += 8) {
      const int x = list_id[j];
      if (first[x] != j || times[x] > FEW) continue;
      float acc[8] = {};
      add(x, j, 1, acc);
      grad_write<ODT>(P, (x << lg) + w, e0, acc);
    }
    if (P.zero) {
      const float zero[8] = {};
      for (int x = k; x < own; x += 8)
        if (times[x] == 0)
          store_piece<ODT, true>(static_cast<char*>(P.out) + (((int64_t)x << lg) + w) * P.out_stride * ElemBytes<ODT>::value,
                                 e0, P.hidden, zero);
    }
  }
  for (int j = 0; j < total; j++) {                // (uniform over the workgroup)
    const int x = list_id[j];
    if (first[x] != j || times[x] <= FEW) continue;
    float acc[8] = {};
    if (in) add(x, j + k, 8, acc);
    if (grad_reduce8(red, c, k, acc) && in) grad_write<ODT>(P, (x << lg) + w, e0, acc);
  }
}

}  // namespace lps
