// Sliding-window attention with sinks: what its kernels share.
//
//   key j is seen by query i, at position p = i + Lk - Lq, iff  j <= p + right  and  (j >= p - left  or  j < sinks)  and its mask is set.
//
// So the keys of a tile of queries are a run of tiles around it and a run of tiles at the front, and the queries of a tile of
// keys are one run: around it, or from it to the end where the tile holds a sink.
//
// A tile of queries holds the rows of all heads that share a key head: row r is query r / pack, head r % pack of the group (pack = G, or
// 1 where more heads share a key head than a tile has rows).  Keys are then read once for the group, the tile's window
// is only as wide as its few queries need, and a single token fills G rows instead of one.
#pragma once

#include "common.cuh"

namespace mf {
namespace win {

struct WinP {
  int B, N, Lq, Lk, H, Hk, D, G;         // G = H / Hk query heads share a key head
  int pack;                              // heads in a tile of queries
  int left, right, sinks, off;           // off = Lk - Lq: position of query 0
  float scale;                           // D^-1/2
  const void *q, *k, *v;
  int64_t qs[5], ks[5], vs[5];
  const uint8_t* mask; int64_t ms[3];    // NULL: every key is kept
  void* o; float* lse;                   // o, d_o, dq, dk, dv: contiguous; lse [B, N, H, Lq], may be NULL on the forward
  const void* d_o; const float* delta;
  void *dq, *dk, *dv;
  bool q_vec, k_vec, v_vec, g_vec;       // CUDA-core kernels: rows can be read four elements at a time
};

__device__ __forceinline__ bool in_window(const WinP& p, int i, int j) {
  const int at = i + p.off;
  return j <= at + p.right && (j >= at - p.left || j < p.sinks);
}
__device__ __forceinline__ bool kept(const WinP& p, int b, int n, int j) {
  return !p.mask || p.mask[b * p.ms[0] + n * p.ms[1] + j * p.ms[2]];
}

__host__ __device__ __forceinline__ int clamp_i(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// Key tiles (of KT keys) that hold a key some query of [i0, i1) sees: tiles [0, front) and [w0, w1), front <= w0.
struct KeyTiles {
  int front, w0, w1;
  __host__ __device__ __forceinline__ int count() const { return front + w1 - w0; }
  __host__ __device__ __forceinline__ int at(int t) const { return t < front ? t : w0 + t - front; }
};
template <int KT>
__host__ __device__ __forceinline__ KeyTiles key_tiles(const WinP& p, int i0, int i1) {
  const int hi = clamp_i(i1 + p.off + p.right, 0, p.Lk);            // one past the last
  const int lo = clamp_i(i0 + p.off - p.left, 0, hi);
  KeyTiles t;
  t.w0 = lo / KT; t.w1 = (hi + KT - 1) / KT;
  if (t.w1 < t.w0) t.w1 = t.w0;
  const int s = p.sinks < hi ? p.sinks : hi;
  t.front = (s + KT - 1) / KT;
  if (t.front > t.w0) t.front = t.w0;
  return t;
}
// Keys that some query of [i0, i1) may see: [lo, hi) and [0, front).  The others in a tile are read as zeros: a cache may hold anything
// where the window has passed.
struct KeyRange { int lo, hi, front; };
__host__ __device__ __forceinline__ KeyRange key_range(const WinP& p, int i0, int i1) {
  KeyRange r;
  r.hi = clamp_i(i1 + p.off + p.right, 0, p.Lk);
  r.lo = clamp_i(i0 + p.off - p.left, 0, r.hi);
  r.front = p.sinks < r.hi ? p.sinks : r.hi;
  return r;
}
__device__ __forceinline__ bool in_range(const KeyRange& r, int j) { return j < r.hi && (j >= r.lo || j < r.front); }
// Queries [lo, hi) that see a key of [j0, j1)
__host__ __device__ __forceinline__ void query_range(const WinP& p, int j0, int j1, int& lo, int& hi) {
  lo = clamp_i(j0 - p.right - p.off, 0, p.Lq);
  hi = j0 < p.sinks ? p.Lq : clamp_i(j1 + p.left - p.off, lo, p.Lq);
}

// ---- the work on dK and dV ------------------------------------------------------------------------------------------
// A tile of KT keys sums over a list of (pack of heads, block of QB rows).  The list of a tile with sinks runs to the last
// query, however narrow the window, and a short sequence has few tiles: lists are cut into chunks of `chunk` entries, a block
// of threads each, whose fp32 sums are added in a fixed order by a second kernel.  x enumerates (tile, chunk), tiles with
// sinks first; the first split_x of them are parts.
// queries of a tile of ROWS rows; groups of `pack` heads; lists of a key head
template <int ROWS> __host__ __device__ __forceinline__ int queries_of(const WinP& p) { return ROWS / p.pack; }
__host__ __device__ __forceinline__ int head_groups(const WinP& p) { return p.H / p.pack; }

struct KeyPlan {
  int n_tiles, n_sink, chunk, nc_sink, nc_rest, x_total, split_x;
};
template <int KT, int QB>
__host__ __device__ __forceinline__ int list_length(const WinP& p, int tile) {
  int lo, hi;
  query_range(p, tile * KT, tile * KT + KT < p.Lk ? tile * KT + KT : p.Lk, lo, hi);
  const int q = queries_of<QB>(p);
  return hi > lo ? p.G / p.pack * ((hi + q - 1) / q - lo / q) : 0;
}
template <int KT, int QB>
KeyPlan key_plan(const WinP& p, int blocks_wanted) {
  KeyPlan c;
  c.n_tiles = (p.Lk + KT - 1) / KT;
  c.n_sink = (p.sinks + KT - 1) / KT;
  if (c.n_sink > c.n_tiles) c.n_sink = c.n_tiles;
  int most_sink = 0, most_rest = 0;
  int64_t all = 0;
  for (int t = 0; t < c.n_tiles; ++t) {
    const int n = list_length<KT, QB>(p, t);
    all += n;
    int& m = t < c.n_sink ? most_sink : most_rest;
    if (n > m) m = n;
  }
  // an even share of all entries for each block that the processors hold, as long as that cuts no list needlessly; never below a few
  // entries, which would not pay for the partial sums
  const int64_t heads = (int64_t)p.B * p.N * p.Hk, most = most_sink > most_rest ? most_sink : most_rest;
  int64_t chunk = (all * heads + blocks_wanted - 1) / blocks_wanted;
  if (chunk > most) chunk = most;
  if (chunk < 6) chunk = 6;
  c.chunk = (int)chunk;
  auto chunks = [&](int n) { const int k = (n + c.chunk - 1) / c.chunk; return k > 1 ? k : 1; };
  c.nc_sink = chunks(most_sink); c.nc_rest = chunks(most_rest);
  c.x_total = c.n_sink * c.nc_sink + (c.n_tiles - c.n_sink) * c.nc_rest;
  c.split_x = c.nc_rest > 1 ? c.x_total : c.nc_sink > 1 ? c.n_sink * c.nc_sink : 0;
  return c;
}
__device__ __forceinline__ void plan_item(const KeyPlan& c, int x, int& tile, int& part) {
  const int front = c.n_sink * c.nc_sink;
  if (x < front) { tile = x / c.nc_sink; part = x - tile * c.nc_sink; }
  else { tile = (x - front) / c.nc_rest; part = x - front - tile * c.nc_rest; tile += c.n_sink; }
}
// partial sums of item x of (b, n, key head): dk and dv rows of D floats
template <int KT>
__host__ __device__ __forceinline__ size_t part_floats(const KeyPlan& c, const WinP& p) { return (size_t)2 * KT * p.D * c.split_x * p.B * p.N * p.Hk; }
template <int KT>
__device__ __forceinline__ float* part_of(float* parts, const KeyPlan& c, const WinP& p, int64_t head, int x) {
  return parts + (size_t)2 * KT * p.D * (head * c.split_x + x);
}

// Adds the parts of the tiles that were split, a thread an element; blockIdx.x enumerates (head of all sequences, tile, piece of 256 elements).
// (With a block a tile a long sequence's tile of sinks, 28 parts of it, took 163 us.)
template <typename T, int KT, int QB>
__global__ void __launch_bounds__(256) window_join_kernel(const __grid_constant__ WinP p, const KeyPlan c, const float* __restrict__ parts, int tiles, int pieces) {
  const int unit = blockIdx.x / pieces, tile = unit % tiles, nc = tile < c.n_sink ? c.nc_sink : c.nc_rest;
  const int x0 = tile < c.n_sink ? tile * c.nc_sink : c.n_sink * c.nc_sink + (tile - c.n_sink) * c.nc_rest;
  const int e = (blockIdx.x - unit * pieces) * 256 + threadIdx.x;
  if (x0 >= c.split_x || nc == 1 || e >= 2 * KT * p.D) return;
  const int which = e / (KT * p.D), r = e - which * KT * p.D, row = r / p.D, d = r - row * p.D, j = tile * KT + row;
  if (j >= p.Lk) return;
  int used = (list_length<KT, QB>(p, tile) + c.chunk - 1) / c.chunk;
  if (used < 1) used = 1;
  const int64_t head = unit / tiles, bn = head / p.Hk;
  const float* src = part_of<KT>(const_cast<float*>(parts), c, p, head, x0) + e;
  const size_t step = (size_t)2 * KT * p.D;
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < used; ++k) s += src[k * step];
  if (which == 0) s *= p.scale;
  static_cast<T*>(which ? p.dv : p.dk)[((bn * p.Lk + j) * p.Hk + (head - bn * p.Hk)) * p.D + d] = from_f<T>(s);
}
template <typename T, int KT, int QB>
int window_join(const WinP& p, const KeyPlan& c, const float* parts, cudaStream_t st) {
  if (!c.split_x) return MF_OK;
  const int tiles = c.nc_rest > 1 ? c.n_tiles : c.n_sink, pieces = (2 * KT * p.D + 255) / 256;
  const int64_t blocks = (int64_t)p.B * p.N * p.Hk * tiles * pieces;
  MF_REQUIRE(blocks <= 0x7fffffff, MF_ERR_UNSUPPORTED, "%d tiles of keys in parts are more than one launch takes", tiles);
  window_join_kernel<T, KT, QB><<<(unsigned)blocks, 256, 0, st>>>(p, c, parts, tiles, pieces);
  MF_LAUNCHED("window_join_kernel");
  return MF_OK;
}

// ---- few queries ------------------------------------------------------------------------------------------------------
// Where the tiles of queries do not occupy the processors, the key tiles of each are split over `splits` blocks.  Each leaves its
// normalised fp32 row and the row's log-sum-exp in `parts` ([splits][B, N, Lq, H][D], then [splits][B, N, Lq, H]), and a second kernel
// weighs them.
struct Split {
  int splits;
  float* parts;
  int64_t rows;             // B * N * Lq * H
  __device__ __forceinline__ float* row(int s, int64_t r, int D) const { return parts + ((int64_t)s * rows + r) * D; }
  __device__ __forceinline__ float& lse(int s, int64_t r, int D) const { return parts[(int64_t)splits * rows * D + (int64_t)s * rows + r]; }
};
template <int ROWS, int KT>
int split_count(const WinP& p, int blocks_wanted) {
  const int q = queries_of<ROWS>(p);
  const int64_t tiles = (p.Lq + q - 1) / q, blocks = tiles * p.B * p.N * head_groups(p);
  if (4 * blocks > blocks_wanted) return 1;                // joining costs some 5 us
  int most = 0;                                            // key tiles of a tile of queries; few of them, or blocks would be many
  for (int64_t t = 0; t < tiles; ++t) {
    const int i0 = (int)t * q, n = key_tiles<KT>(p, i0, i0 + q < p.Lq ? i0 + q : p.Lq).count();
    if (n > most) most = n;
  }
  int64_t s = blocks_wanted / blocks;
  if (s > most / 2) s = most / 2;                          // two tiles at least, or the joining costs more than it saves
  if (s > 64) s = 64;
  return s < 1 ? 1 : (int)s;
}
inline size_t split_bytes(const WinP& p, int splits) { return splits == 1 ? 0 : sizeof(float) * (size_t)splits * p.B * p.N * p.Lq * p.H * (p.D + 1); }
int window_split_join(const WinP& p, int dtype, const Split& s, cudaStream_t st);

WinP window_params(const mf_window_args& a);
int window_delta(const WinP& p, int dtype, float* delta, cudaStream_t st);       // delta [B, N, H, Lq] = sum over d of d_o * o

}  // namespace win
}  // namespace mf
