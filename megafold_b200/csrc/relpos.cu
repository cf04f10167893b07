// Learned relative position bias by buckets:  bias[b, 0, h, i, j] = weight[row(b, i, j), h]  and its gradient,
// d_weight[r, h] = sum of d_bias[b, 0, h, i, j] over the pairs of row r.
//
// The row of a pair is a function of the distance d = k_pos[j] - q_pos[i], or the table's last row where the two belong to
// different segments.  Buckets are given as ascending distances at which |d| enters the next one ("edges"), so that the borders
// of logarithmic buckets are whole numbers computed by the host and no logarithm is rounded here.  A block lays the rows of
// all distances up to the last edge out in shared memory once; a pair then costs a subtraction, a clamp and a look-up,
// shared by the heads of the block, and a second look-up a head.
//
// Bound: HBM writes (forward with aligned rows), four- or two-byte stores (other rows), issue slots for the look-ups (backward).
#include "common.cuh"

namespace mf {
namespace {

constexpr int kThreads = 256;

struct RelP {
  int B, H, Lq, Lk, rows, w_dtype;
  int n_edges, base_pos, step_pos, base_neg, step_neg, reach;      // reach = the last edge
  const void *q_pos, *k_pos, *q_seg, *k_seg;
  int64_t qp_b, kp_b, qs_b, ks_b;
  bool pos64, seg64;
  int log_tpr;                       // threads of a block that share a row of the bias
  int strips;                        // blocks along the queries of a batch element
  uint16_t edges[MF_RELPOS_MAX_EDGES];
};
static_assert(MF_RELPOS_MAX_EDGES == MF_RELPOS_MAX_ROWS - 1 && MF_RELPOS_MAX_DISTANCE <= 65535, "one direction has a border between any two rows");

__device__ __forceinline__ int64_t load_int(const void* p, int64_t i, bool wide) {
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}
__device__ __forceinline__ int64_t q_position(const RelP& p, int b, int i) { return p.q_pos ? load_int(p.q_pos, b * p.qp_b + i, p.pos64) : (int64_t)i + (p.Lk - p.Lq); }
__device__ __forceinline__ int64_t k_position(const RelP& p, int b, int j) { return p.k_pos ? load_int(p.k_pos, b * p.kp_b + j, p.pos64) : (int64_t)j; }

// Positions (and segments) in 32 bits, as differences from the first key's where all that a block sees lie within 2^30 of that; a block that
// finds others reads them again where it needs them.
constexpr int kFar = 1 << 30;
struct Origin { int64_t pos, seg; };
__device__ __forceinline__ Origin origin(const RelP& p, int b) { return Origin{k_position(p, b, 0), p.k_seg ? load_int(p.k_seg, b * p.ks_b, p.seg64) : 0}; }
__device__ __forceinline__ int near_to(int64_t x, int64_t from, bool& near) {
  const int64_t d = x - from;
  near = near && d > -kFar && d < kFar;
  return (int)d;
}

// Rows of the distances -reach .. reach.  The edges go through shared memory (`tmp`): read at an index that differs by lane from the
// kernel's parameters, 1600 distances took each block some 5 us.
__device__ __forceinline__ void fill_rows(const RelP& p, uint16_t* lut, uint16_t* tmp, int tid, int nt) {
  for (int x = tid; x < p.n_edges; x += nt) tmp[x] = p.edges[x];
  __syncthreads();
  // a thread fills adjacent distances of both signs, with one search among the edges
  const auto row = [&](int base, int by, int k) { const int r = base + by * k; return (uint16_t)(r < 0 ? 0 : r >= p.rows ? p.rows - 1 : r); };
  const int run = (p.reach + nt) / nt, to = run * (tid + 1) <= p.reach ? run * (tid + 1) : p.reach + 1;
  int n = run * tid, k = 0;                      // k edges are not above n
  for (int hi = p.n_edges; n < to && k < hi;) {
    const int mid = (k + hi) >> 1;
    if (tmp[mid] <= n) k = mid + 1; else hi = mid;
  }
  for (; n < to; ++n) {
    while (k < p.n_edges && tmp[k] <= n) ++k;
    if (n) lut[p.reach + n] = row(p.base_pos, p.step_pos, k);
    lut[p.reach - n] = row(p.base_neg, p.step_neg, k);
  }
}
__device__ __forceinline__ int row_of(const RelP& p, const uint16_t* lut, int d) { return lut[(d < -p.reach ? -p.reach : d > p.reach ? p.reach : d) + p.reach]; }
__device__ __forceinline__ int row_of_far(const RelP& p, const uint16_t* lut, int b, int i, int j) {
  if (p.q_seg && load_int(p.q_seg, b * p.qs_b + i, p.seg64) != load_int(p.k_seg, b * p.ks_b + j, p.seg64)) return p.rows - 1;
  const int64_t d = k_position(p, b, j) - q_position(p, b, i);
  return row_of(p, lut, d < -p.reach ? -p.reach : d > p.reach ? p.reach : (int)d);
}

// Forward: blockIdx = (column tile, batch element and strip of queries, group of heads).  A thread's columns: 16 bytes of adjacent ones where
// rows are 16-byte aligned, else eight, 32 apart, of its warp's 256 (a store of the warp then writes adjacent elements).
template <typename T, bool VEC> struct Cols {
  static constexpr int kC = VEC ? 16 / (int)sizeof(T) : 8, kStep = VEC ? 1 : 32;
  static __device__ __forceinline__ int first(int j0, int lane) { return VEC ? j0 + lane * kC : j0 + (lane & ~31) * 8 + (lane & 31); }
};
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) relpos_fwd_kernel(const __grid_constant__ RelP p, const void* __restrict__ weight, T* __restrict__ bias, int heads) {
  using C = Cols<T, VEC>;
  constexpr int kC = C::kC;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint16_t tmp[MF_RELPOS_MAX_EDGES];
  uint16_t* lut = reinterpret_cast<uint16_t*>(smem);
  T* table = reinterpret_cast<T*>(smem + ((2 * (2 * p.reach + 1) + 15) & ~15));       // [head of the group][row]
  const int tpr = 1 << p.log_tpr, lane = threadIdx.x & (tpr - 1), slot = threadIdx.x >> p.log_tpr, slots = kThreads >> p.log_tpr;
  const int j = C::first(blockIdx.x * tpr * kC, lane), b = blockIdx.y / p.strips, strip = blockIdx.y - b * p.strips;
  const int h0 = blockIdx.z * heads, nh = h0 + heads <= p.H ? heads : p.H - h0;
  const Origin o = origin(p, b);
  int kp[kC], ks[kC];
  bool near = true;
#pragma unroll
  for (int e = 0; e < kC; ++e) {
    const int je = j + e * C::kStep;
    kp[e] = je < p.Lk ? near_to(k_position(p, b, je), o.pos, near) : 0;
    ks[e] = je < p.Lk && p.k_seg ? near_to(load_int(p.k_seg, b * p.ks_b + je, p.seg64), o.seg, near) : 0;
  }
  fill_rows(p, lut, tmp, threadIdx.x, kThreads);
  for (int x = threadIdx.x; x < p.rows * nh; x += kThreads) {
    const int r = x / nh, h = x - r * nh;
    table[h * p.rows + r] = from_f<T>(load_rt(weight, (int64_t)r * p.H + h0 + h, p.w_dtype));
  }
  __syncthreads();
  const int end = (int)((int64_t)p.Lq * (strip + 1) / p.strips);
  for (int i = (int)((int64_t)p.Lq * strip / p.strips) + slot; i < end; i += slots) {
    bool close = near;
    const int qp = near_to(q_position(p, b, i), o.pos, close), qs = p.q_seg ? near_to(load_int(p.q_seg, b * p.qs_b + i, p.seg64), o.seg, close) : 0;
    int row[kC];
    if (close) {
#pragma unroll
      for (int e = 0; e < kC; ++e) {
        row[e] = row_of(p, lut, kp[e] - qp);
        if (ks[e] != qs) row[e] = p.rows - 1;              // without segments both are 0
      }
    } else {
#pragma unroll
      for (int e = 0; e < kC; ++e) row[e] = j + e * C::kStep < p.Lk ? row_of_far(p, lut, b, i, j + e * C::kStep) : 0;
    }
    T* out = bias + (((int64_t)b * p.H + h0) * p.Lq + i) * p.Lk + j;
    const T* t = table;
    const int left = p.Lk - j;
    for (int h = 0; h < nh; ++h, out += (int64_t)p.Lq * p.Lk, t += p.rows) {
      if constexpr (VEC) {
        __align__(16) T v[kC];
#pragma unroll
        for (int e = 0; e < kC; ++e) v[e] = t[row[e]];
        if (left > 0) __stcs(reinterpret_cast<uint4*>(out), *reinterpret_cast<const uint4*>(v));
      } else {
#pragma unroll
        for (int e = 0; e < kC; ++e)
          if (e * C::kStep < left) out[e * C::kStep] = t[row[e]];
      }
    }
  }
}

// Backward: blockIdx = (column tile, batch element and strip of queries, head).  A thread walks down diagonals: from one query to the next its
// columns move by one too (around the tile's end to its start), so that the distance, and with it the table's row, stays the same
// where positions run on.  It sums in registers and adds a sum to a column of its own of the block's table in shared memory when the row
// changes (no atomics: the sums' order is fixed); walking down columns instead, a warp met such a change in most of its
// steps and [2, 8, 1531, 1531] took 173 us.  The block's table goes to `parts` [gridDim.y * gridDim.x][H][rows].
// Bound by issue slots (the look-ups).  Where a block's positions run on without a gap it looks up what comes around the tile's end only: [2, 8, 1531, 1531] fp32
// 51 us instead of 75, [1, 16, 4096, 4096] bf16 248 instead of 432 (buckets = 32).
// Two rows of a thread are in registers, two more on their way into L2, and 512 threads of an SM have 128 registers each: with gaps and 64 rows of the
// table 78 us (before tiles were fitted to the rows 102), six rows ahead instead of four 103; three blocks of 80 registers 112, without the way into L2 120.
constexpr int kBwdCols = 8, kBwdAhead = 4, kBwdResident = 512;
template <typename T>
__global__ void __launch_bounds__(kThreads, kBwdResident / kThreads) relpos_bwd_kernel(const __grid_constant__ RelP p, const T* __restrict__ d_bias, float* __restrict__ parts) {
  constexpr int kC = kBwdCols;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint16_t tmp[MF_RELPOS_MAX_EDGES];
  const int nt = blockDim.x, tid = threadIdx.x;
  const int tpr = 1 << p.log_tpr, lane = tid & (tpr - 1), slot = tid >> p.log_tpr, slots = nt >> p.log_tpr, width_max = tpr * kC;
  int32_t* kpos = reinterpret_cast<int32_t*>(smem);                                            // positions of the tile's keys
  int32_t* kseg = kpos + width_max;
  uint16_t* lut = reinterpret_cast<uint16_t*>(kseg + (p.k_seg ? width_max : 0));
  float* table = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(lut) + ((2 * (2 * p.reach + 1) + 15) & ~15));       // [row][thread]
  const int j0 = blockIdx.x * width_max, h = blockIdx.z, b = blockIdx.y / p.strips, strip = blockIdx.y - b * p.strips;
  const int width = p.Lk - j0 < width_max ? p.Lk - j0 : width_max;
  const Origin o = origin(p, b);
  bool near = true;
  for (int x = tid; x < width; x += nt) {
    kpos[x] = near_to(k_position(p, b, j0 + x), o.pos, near);
    if (p.k_seg) kseg[x] = near_to(load_int(p.k_seg, b * p.ks_b + j0 + x, p.seg64), o.seg, near);
  }
  fill_rows(p, lut, tmp, tid, nt);
  for (int x = tid; x < p.rows * nt; x += nt) table[x] = 0.f;
  const int i0 = (int)((int64_t)p.Lq * strip / p.strips), end = (int)((int64_t)p.Lq * (strip + 1) / p.strips);
  // run_on: each position is the one before and one, of the tile's keys and of the strip's queries
  bool run_on = !p.k_seg && width > slots;
  for (int i = i0 + tid; i < end; i += nt) {
    const int64_t x = q_position(p, b, i);
    near_to(x, o.pos, near);
    if (p.q_seg) near_to(load_int(p.q_seg, b * p.qs_b + i, p.seg64), o.seg, near);
    if (i + 1 < end) run_on = run_on && q_position(p, b, i + 1) - x == 1;
  }
  near = __syncthreads_and(near);
  for (int x = tid; x + 1 < width; x += nt) run_on = run_on && kpos[x + 1] - kpos[x] == 1;
  run_on = __syncthreads_and(run_on && near);
  bool begun = false;
  float* mine = table + tid;                       // the only column that this thread touches before the last barrier
  const T* in = d_bias + (((int64_t)b * p.H + h) * p.Lq) * p.Lk + j0;
  // column e of this thread at query i is lane + e * tpr + (i - i0), around the width
  const int columns = (width - lane + tpr - 1) >> p.log_tpr;       // of the tile's width; at most kC
  int cur[kC];
  float acc[kC];
#pragma unroll
  for (int e = 0; e < kC; ++e) { cur[e] = 0; acc[e] = 0.f; }
  const int step = slots % width;
  auto wrap = [&](int c) { return c >= width ? c - width : c; };
  auto wrap_in = [&](int c, int e) { return e < columns ? wrap(c) : 0; };
  struct Cursor { int i, first; const T* row; };                   // of the loads, and of the sums two rows behind
  auto start = [&]() { return Cursor{i0 + slot, (lane + slot) % width, in + (int64_t)(i0 + slot) * p.Lk}; };
  auto next = [&](Cursor& c) { c.i += slots; c.first = wrap(c.first + step); c.row += (int64_t)slots * p.Lk; };
  auto load = [&](Cursor& c, T (&x)[kC]) {
#pragma unroll
    for (int e = 0; e < kC; ++e) {
      const bool there = c.i < end && e < columns;
      const T* at = c.row + wrap(c.first + e * tpr);
      x[e] = there ? *at : from_f<T>(0.f);
    }
    next(c);
  };
  auto add = [&](Cursor& c, const T (&x)[kC]) {
    const auto q_at = [&]() { return (int)q_position(p, b, c.i) - (int)o.pos; };
    // where positions run on, only the columns that came around in this step have another distance: the first, and the one behind which
    // the tile ends (a bit a column; two at most, as they lie further apart than a step but for the last and the first)
    uint32_t around = 0;
    if (run_on && begun) {
      const int k = width - c.first, e = (k + tpr - 1) >> p.log_tpr;
      around = (c.first < step ? 1u : 0u) | (e < columns && (e << p.log_tpr) - k < step ? 1u << e : 0u);
    }
    if (!(run_on && begun)) {
      int row[kC];
      if (near) {
        const int qp = q_at(), qs = p.q_seg ? (int)load_int(p.q_seg, b * p.qs_b + c.i, p.seg64) - (int)o.seg : 0;
#pragma unroll
        for (int e = 0; e < kC; ++e) row[e] = kpos[wrap_in(c.first + e * tpr, e)];
#pragma unroll
        for (int e = 0; e < kC; ++e) row[e] = row_of(p, lut, row[e] - qp);
        if (p.q_seg) {
#pragma unroll
          for (int e = 0; e < kC; ++e)
            if (kseg[wrap_in(c.first + e * tpr, e)] != qs) row[e] = p.rows - 1;
        }
      } else {
#pragma unroll
        for (int e = 0; e < kC; ++e) row[e] = row_of_far(p, lut, b, c.i, j0 + wrap_in(c.first + e * tpr, e));
      }
      bool moved = false;
#pragma unroll
      for (int e = 0; e < kC; ++e) moved = moved || row[e] != cur[e];
      if (__any_sync(0xffffffffu, moved)) {        // a warp is in one row of the bias: tpr is 32 at least
#pragma unroll
        for (int e = 0; e < kC; ++e)
          if (row[e] != cur[e]) { mine[cur[e] * nt] += acc[e]; cur[e] = row[e]; acc[e] = 0.f; }
      }
      begun = true;
    } else if (__any_sync(0xffffffffu, around != 0)) {
      const int qp = q_at();
#pragma unroll
      for (int e = 0; e < kC; ++e)
        if (around >> e & 1) {
          mine[cur[e] * nt] += acc[e];
          acc[e] = 0.f;
          cur[e] = row_of(p, lut, kpos[wrap(c.first + e * tpr)] - qp);
        }
    }
#pragma unroll
    for (int e = 0; e < kC; ++e) acc[e] += to_f(x[e]);             // zeros for columns that are not there
    next(c);
  };
  // a row of the tile is no more than tpr lines of 128 bytes
  const bool asks = lane * 128 < width * (int)sizeof(T);
  auto ahead = [&](int i, const T* row) {
    if (asks && i < end) asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(row) + lane * 128));
  };
  Cursor in_at = start(), sum_at = start();
  const int64_t row_step = (int64_t)slots * p.Lk;
#pragma unroll
  for (int k = 2; k < kBwdAhead; ++k) ahead(in_at.i + k * slots, in_at.row + k * row_step);
  T x0[kC], x1[kC];                                // two rows under way
  load(in_at, x0);
  load(in_at, x1);
  while (sum_at.i < end) {
    add(sum_at, x0);
    ahead(in_at.i + (kBwdAhead - 2) * slots, in_at.row + (kBwdAhead - 2) * row_step);
    load(in_at, x0);
    if (sum_at.i >= end) break;
    add(sum_at, x1);
    ahead(in_at.i + (kBwdAhead - 2) * slots, in_at.row + (kBwdAhead - 2) * row_step);
    load(in_at, x1);
  }
#pragma unroll
  for (int e = 0; e < kC; ++e) mine[cur[e] * nt] += acc[e];
  __syncthreads();
  const int warp = tid >> 5, l = tid & 31;
  float* out = parts + ((int64_t)(blockIdx.y * gridDim.x + blockIdx.x) * p.H + h) * p.rows;
  for (int x = warp; x < p.rows; x += nt >> 5) {
    float s = 0.f;
    for (int y = l; y < nt; y += 32) s += table[x * nt + y];
    s = warp_sum(s);
    if (l == 0) out[x] = s;
  }
}

// d_weight[r, h] = sum of the blocks' tables, a warp each
__global__ void __launch_bounds__(kThreads) relpos_join_kernel(const float* __restrict__ parts, int n_parts, int H, int rows, void* __restrict__ d_weight, int w_dtype) {
  const int x = (blockIdx.x * kThreads + threadIdx.x) >> 5, l = threadIdx.x & 31;
  if (x >= rows * H) return;
  const int h = x / rows, r = x - h * rows;
  double s = 0.;
  for (int k = l; k < n_parts; k += 32) s += parts[((int64_t)k * H + h) * rows + r];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (l == 0) store_rt(d_weight, (int64_t)r * H + h, w_dtype, (float)s);
}

RelP relpos_params(const mf_relpos_args& a) {
  RelP p{};
  p.B = a.B; p.H = a.H; p.Lq = a.Lq; p.Lk = a.Lk; p.rows = a.rows; p.w_dtype = a.w_dtype;
  p.n_edges = a.n_edges; p.base_pos = a.base_pos; p.step_pos = a.step_pos; p.base_neg = a.base_neg; p.step_neg = a.step_neg;
  for (int i = 0; i < a.n_edges; ++i) p.edges[i] = (uint16_t)a.edges[i];
  p.reach = a.n_edges ? a.edges[a.n_edges - 1] : 0;
  if (p.reach < 1) p.reach = 1;
  p.q_pos = a.q_pos; p.k_pos = a.k_pos; p.q_seg = a.q_seg; p.k_seg = a.k_seg;
  p.qp_b = a.q_pos_stride; p.kp_b = a.k_pos_stride; p.qs_b = a.q_seg_stride; p.ks_b = a.k_seg_stride;
  p.pos64 = a.pos_bytes == 8; p.seg64 = a.seg_bytes == 8;
  return p;
}
size_t lut_bytes(const RelP& p) { return (2 * (2 * (size_t)p.reach + 1) + 15) & ~(size_t)15; }
int log_threads(int Lk, int cols, int least, int threads) {
  int l = least;
  while ((1 << l) < threads && (1 << l) * cols < Lk) ++l;
  return l;
}

struct BwdPlan { int threads, tiles, parts; size_t smem; };
BwdPlan bwd_plan(RelP& p) {
  BwdPlan b;
  b.threads = kThreads;
  while (b.threads > 32 && (size_t)p.rows * b.threads * 4 > 72 * 1024) b.threads /= 2;
  // threads of a row: those that leave the least of the columns' places empty, with a step more where a column wraps around (one a row)
  int64_t least = 0;
  for (int l = 5; (1 << l) <= b.threads; ++l) {
    const int64_t wide = (int64_t)kBwdCols << l, cost = (p.Lk + wide - 1) / wide * wide * (320 + (64 >> (l - 5)));
    if (l == 5 || cost < least) { least = cost; p.log_tpr = l; }
  }
  const int tpr = 1 << p.log_tpr, slots = b.threads >> p.log_tpr;
  b.smem = lut_bytes(p) + (size_t)p.rows * b.threads * 4 + (size_t)tpr * kBwdCols * (p.k_seg ? 8 : 4);
  b.tiles = (p.Lk + tpr * kBwdCols - 1) / (tpr * kBwdCols);
  // as many blocks as fit the processors at once, each with two steps of its rows at least
  int fit = (int)(220 * 1024 / (b.smem + 4096));
  if (fit > kBwdResident / b.threads) fit = kBwdResident / b.threads;
  const int64_t want = (int64_t)tcx::sm_count() * (fit < 1 ? 1 : fit), others = (int64_t)p.H * b.tiles * p.B;
  int64_t strips = want / others;
  const int64_t most = (p.Lq + 2 * slots - 1) / (2 * slots);
  if (strips > most) strips = most;
  if (strips > 65535 / p.B) strips = 65535 / p.B;
  p.strips = (int)(strips < 1 ? 1 : strips);
  b.parts = b.tiles * p.strips * p.B;
  return b;
}
bool vec_ok(const mf_relpos_args& a, const void* ptr) { return (a.Lk * dtype_size(a.dtype)) % 16 == 0 && (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; }

template <typename T, bool VEC>
int run_fwd(const mf_relpos_args& a, cudaStream_t st) {
  RelP p = relpos_params(a);
  constexpr int kC = Cols<T, VEC>::kC;
  p.log_tpr = log_threads(p.Lk, kC, VEC ? 0 : 5, kThreads);
  const int tpr = 1 << p.log_tpr, slots = kThreads >> p.log_tpr;
  const int tiles = (p.Lk + tpr * kC - 1) / (tpr * kC);
  // heads of a block: all of them, less where the table would take more than 48 KB or the rows do not occupy the processors
  int heads = p.H;
  while (heads > 1 && (size_t)heads * p.rows * sizeof(T) > 48 * 1024) heads = (heads + 1) / 2;
  const int64_t row_blocks = (p.Lq + slots - 1) / slots, want = 4 * (int64_t)tcx::sm_count();
  while (heads > 1 && row_blocks * tiles * p.B * ((p.H + heads - 1) / heads) < want) heads = (heads + 1) / 2;
  const int groups = (p.H + heads - 1) / heads;
  // one wave of blocks, or two where a block of one would write more than 384 KB: a wave begins with some 4 us of tables ([2, 8, 1531, 1531]
  // bf16 28 us instead of 33), two end more evenly ([4, 8, 1536, 1536] fp32 55 us instead of 65)
  const int64_t waves = (int64_t)p.B * p.H * p.Lq * p.Lk * (int)sizeof(T) > want * (384 << 10) ? 2 : 1;
  int64_t strips = (waves * want + (int64_t)tiles * groups * p.B - 1) / ((int64_t)tiles * groups * p.B);
  if (strips > row_blocks) strips = row_blocks;
  if (strips > 65535 / p.B) strips = 65535 / p.B;
  p.strips = (int)(strips < 1 ? 1 : strips);
  const size_t smem = lut_bytes(p) + (size_t)heads * p.rows * sizeof(T);
  constexpr auto kern = relpos_fwd_kernel<T, VEC>;
  if (int e = opt_in_smem<kern>(smem)) return e;
  kern<<<dim3(tiles, (unsigned)(p.strips * p.B), groups), kThreads, smem, st>>>(p, a.weight, static_cast<T*>(a.bias), heads);
  MF_LAUNCHED("relpos_fwd_kernel");
  return MF_OK;
}

template <typename T>
int run_bwd(const mf_relpos_args& a, cudaStream_t st) {
  RelP p = relpos_params(a);
  const BwdPlan b = bwd_plan(p);
  constexpr auto kern = relpos_bwd_kernel<T>;
  if (int e = opt_in_smem<kern>(b.smem)) return e;
  float* parts = static_cast<float*>(a.workspace);
  kern<<<dim3(b.tiles, p.strips * p.B, p.H), b.threads, b.smem, st>>>(p, static_cast<const T*>(a.d_bias), parts);
  MF_LAUNCHED("relpos_bwd_kernel");
  relpos_join_kernel<<<(p.rows * p.H + kThreads / 32 - 1) / (kThreads / 32), kThreads, 0, st>>>(parts, b.parts, p.H, p.rows, a.d_weight, a.dw_dtype);
  MF_LAUNCHED("relpos_join_kernel");
  return MF_OK;
}
}  // namespace

int relpos_fwd(const mf_relpos_args& a, cudaStream_t st) {
  int r = MF_OK;
  MF_DISPATCH_FLOAT(a.dtype, T, r = vec_ok(a, a.bias) ? run_fwd<T, true>(a, st) : run_fwd<T, false>(a, st));
  return r;
}
size_t relpos_bwd_workspace(const mf_relpos_args& a) {
  RelP p = relpos_params(a);
  return sizeof(float) * (size_t)bwd_plan(p).parts * p.H * p.rows;
}
int relpos_bwd(const mf_relpos_args& a, cudaStream_t st) {
  int r = MF_OK;
  MF_DISPATCH_FLOAT(a.dtype, T, r = run_bwd<T>(a, st));
  return r;
}

}  // namespace mf
