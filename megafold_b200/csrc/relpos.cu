// Learned relative position bias by buckets:  bias[b, 0, h, i, j] = weight[row(b, i, j), h]  and its gradient,
// d_weight[r, h] = sum of d_bias[b, 0, h, i, j] over the pairs of row r.
//
// The row of a pair is a function of the distance d = k_pos[j] - q_pos[i], or the table's last row where the two belong to
// different segments.  Buckets are given as ascending distances at which |d| enters the next one ("edges"), so that the borders
// of logarithmic buckets are whole numbers computed by the host and no logarithm is rounded here.  A block lays the rows of
// all distances up to the last edge out in shared memory once; a pair then costs a subtraction, a clamp and a look-up,
// shared by the heads of the block, and a second look-up a head.
//
// Bound: HBM writes (forward) and reads (backward).
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
  int edges[MF_RELPOS_MAX_EDGES];
};

__device__ __forceinline__ int64_t load_int(const void* p, int64_t i, bool wide) {
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}
__device__ __forceinline__ int64_t q_position(const RelP& p, int b, int i) { return p.q_pos ? load_int(p.q_pos, b * p.qp_b + i, p.pos64) : (int64_t)i + (p.Lk - p.Lq); }
__device__ __forceinline__ int64_t k_position(const RelP& p, int b, int j) { return p.k_pos ? load_int(p.k_pos, b * p.kp_b + j, p.pos64) : (int64_t)j; }

// Rows of the distances -reach .. reach.  The edges go through shared memory (`tmp`, before anything else uses it): read at an index
// that differs by lane from the kernel's parameters, 1600 distances took each block some 5 us.
__device__ __forceinline__ void fill_rows(const RelP& p, uint16_t* lut, int32_t* tmp, int tid, int nt) {
  for (int x = tid; x < p.n_edges; x += nt) tmp[x] = p.edges[x];
  __syncthreads();
  for (int x = tid; x <= 2 * p.reach; x += nt) {
    const int d = x - p.reach, n = d < 0 ? -d : d;
    int lo = 0, hi = p.n_edges;                  // edges not above n
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (tmp[mid] <= n) lo = mid + 1; else hi = mid;
    }
    const int r = d > 0 ? p.base_pos + p.step_pos * lo : p.base_neg + p.step_neg * lo;
    lut[x] = (uint16_t)(r < 0 ? 0 : r >= p.rows ? p.rows - 1 : r);
  }
  __syncthreads();
}
__device__ __forceinline__ int row_of(const RelP& p, const uint16_t* lut, int64_t d) {
  d = d < -p.reach ? -p.reach : d > p.reach ? p.reach : d;
  return lut[(int)d + p.reach];
}

// A thread's eight columns of a tile of rows: C adjacent ones where rows are 16-byte aligned (16 bytes a store), else one every
// tpr columns (a warp then covers adjacent elements).  Columns at and beyond Lk are left out.
template <typename T, bool VEC> struct Cols {
  static constexpr int kC = VEC ? 16 / (int)sizeof(T) : 8;
  static __device__ __forceinline__ int at(int j0, int lane, int tpr, int e) { return VEC ? j0 + lane * kC + e : j0 + e * tpr + lane; }
};

// Forward: blockIdx = (column tile, rows, group of heads).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) relpos_fwd_kernel(const __grid_constant__ RelP p, const void* __restrict__ weight, T* __restrict__ bias, int heads) {
  using C = Cols<T, VEC>;
  constexpr int kC = C::kC;
  extern __shared__ __align__(16) uint8_t smem[];
  uint16_t* lut = reinterpret_cast<uint16_t*>(smem);
  T* table = reinterpret_cast<T*>(smem + ((2 * (2 * p.reach + 1) + 15) & ~15));       // [head of the group][row]
  const int h0 = blockIdx.z * heads, nh = h0 + heads <= p.H ? heads : p.H - h0;
  __shared__ int32_t tmp[MF_RELPOS_MAX_EDGES];
  fill_rows(p, lut, tmp, threadIdx.x, kThreads);
  for (int x = threadIdx.x; x < p.rows * nh; x += kThreads) {
    const int r = x / nh, h = x - r * nh;
    table[h * p.rows + r] = from_f<T>(load_rt(weight, (int64_t)r * p.H + h0 + h, p.w_dtype));
  }
  __syncthreads();
  const int tpr = 1 << p.log_tpr, lane = threadIdx.x & (tpr - 1), slot = threadIdx.x >> p.log_tpr, slots = kThreads >> p.log_tpr;
  const int j0 = blockIdx.x * tpr * kC;
  const int64_t n_rows = (int64_t)p.B * p.Lq;
  int64_t kp[kC], ks[kC];
  int kb = -1;
  for (int64_t r = (int64_t)blockIdx.y * slots + slot; r < n_rows; r += (int64_t)gridDim.y * slots) {
    const int b = (int)(r / p.Lq), i = (int)(r - (int64_t)b * p.Lq);
    if (b != kb) {
      kb = b;
#pragma unroll
      for (int e = 0; e < kC; ++e) {
        const int j = C::at(j0, lane, tpr, e);
        kp[e] = j < p.Lk ? k_position(p, b, j) : 0;
        ks[e] = j < p.Lk && p.k_seg ? load_int(p.k_seg, b * p.ks_b + j, p.seg64) : 0;
      }
    }
    const int64_t qp = q_position(p, b, i), qs = p.q_seg ? load_int(p.q_seg, b * p.qs_b + i, p.seg64) : 0;
    int row[kC];
#pragma unroll
    for (int e = 0; e < kC; ++e) {
      row[e] = row_of(p, lut, kp[e] - qp);
      if (p.q_seg && ks[e] != qs) row[e] = p.rows - 1;
    }
    T* out = bias + (((int64_t)b * p.H + h0) * p.Lq + i) * p.Lk;
    const T* t = table;
    for (int h = 0; h < nh; ++h, out += (int64_t)p.Lq * p.Lk, t += p.rows) {
      if constexpr (VEC) {
        __align__(16) T v[kC];
#pragma unroll
        for (int e = 0; e < kC; ++e) v[e] = t[row[e]];
        const int j = C::at(j0, lane, tpr, 0);
        if (j < p.Lk) __stcs(reinterpret_cast<uint4*>(out + j), *reinterpret_cast<const uint4*>(v));
      } else {
#pragma unroll
        for (int e = 0; e < kC; ++e) {
          const int j = C::at(j0, lane, tpr, e);
          if (j < p.Lk) out[j] = t[row[e]];
        }
      }
    }
  }
}

// Backward: blockIdx = (column tile, strip of rows, head).  A thread keeps a row of the table and a sum in registers for each of its
// columns and walks down the rows of its strip: the distance of a column changes by one or so from row to row, so the table's
// row seldom does.  Where it does, the sum goes to a column of the thread's own in the block's table in shared memory (no
// atomics: the sums' order is fixed).  The block's table goes to `parts` [gridDim.x * gridDim.y][H][rows].
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) relpos_bwd_kernel(const __grid_constant__ RelP p, const T* __restrict__ d_bias, float* __restrict__ parts) {
  using C = Cols<T, VEC>;
  constexpr int kC = C::kC;
  extern __shared__ __align__(16) uint8_t smem[];
  const int nt = blockDim.x, tid = threadIdx.x;
  uint16_t* lut = reinterpret_cast<uint16_t*>(smem);
  float* table = reinterpret_cast<float*>(smem + ((2 * (2 * p.reach + 1) + 15) & ~15));       // [row][thread]
  __shared__ int32_t tmp[MF_RELPOS_MAX_EDGES];
  fill_rows(p, lut, tmp, tid, nt);
  for (int x = tid; x < p.rows * nt; x += nt) table[x] = 0.f;
  float* mine = table + tid;                       // the only column that this thread touches before the last barrier
  __syncthreads();
  const int tpr = 1 << p.log_tpr, lane = tid & (tpr - 1), slot = tid >> p.log_tpr, slots = nt >> p.log_tpr;
  const int j0 = blockIdx.x * tpr * kC, h = blockIdx.z;
  const int64_t n_rows = (int64_t)p.B * p.Lq, r_end = n_rows * (blockIdx.y + 1) / gridDim.y;
  int64_t kp[kC], ks[kC];
  int kb = -1, cur[kC];
  float acc[kC];
#pragma unroll
  for (int e = 0; e < kC; ++e) { cur[e] = 0; acc[e] = 0.f; }
  auto load = [&](int64_t r, T (&x)[kC]) {
    const int64_t b = r / p.Lq, i = r - b * p.Lq;
    const T* in = d_bias + ((b * p.H + h) * p.Lq + i) * p.Lk;
    if constexpr (VEC) {
      const int j = C::at(j0, lane, tpr, 0);
      *reinterpret_cast<uint4*>(x) = r < r_end && j < p.Lk ? __ldcs(reinterpret_cast<const uint4*>(in + j)) : make_uint4(0u, 0u, 0u, 0u);
    } else {
#pragma unroll
      for (int e = 0; e < kC; ++e) {
        const int j = C::at(j0, lane, tpr, e);
        x[e] = r < r_end && j < p.Lk ? in[j] : from_f<T>(0.f);
      }
    }
  };
  int64_t r = n_rows * blockIdx.y / gridDim.y + slot;
  __align__(16) T next[kC];
  load(r, next);
  for (; r < r_end; r += slots) {
    const int b = (int)(r / p.Lq), i = (int)(r - (int64_t)b * p.Lq);
    float v[kC];
#pragma unroll
    for (int e = 0; e < kC; ++e) v[e] = to_f(next[e]);
    load(r + slots, next);
    if (b != kb) {
      kb = b;
#pragma unroll
      for (int e = 0; e < kC; ++e) {
        const int j = C::at(j0, lane, tpr, e);
        kp[e] = j < p.Lk ? k_position(p, b, j) : 0;
        ks[e] = j < p.Lk && p.k_seg ? load_int(p.k_seg, b * p.ks_b + j, p.seg64) : 0;
      }
    }
    const int64_t qp = q_position(p, b, i), qs = p.q_seg ? load_int(p.q_seg, b * p.qs_b + i, p.seg64) : 0;
#pragma unroll
    for (int e = 0; e < kC; ++e) {
      int row = row_of(p, lut, kp[e] - qp);
      if (p.q_seg && ks[e] != qs) row = p.rows - 1;
      if (row != cur[e]) { mine[cur[e] * nt] += acc[e]; cur[e] = row; acc[e] = 0.f; }
      acc[e] += v[e];                              // zeros beyond Lk
    }
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
  for (int i = 0; i < a.n_edges; ++i) p.edges[i] = a.edges[i];
  p.reach = a.n_edges ? a.edges[a.n_edges - 1] : 0;
  if (p.reach < 1) p.reach = 1;
  p.q_pos = a.q_pos; p.k_pos = a.k_pos; p.q_seg = a.q_seg; p.k_seg = a.k_seg;
  p.qp_b = a.q_pos_stride; p.kp_b = a.k_pos_stride; p.qs_b = a.q_seg_stride; p.ks_b = a.k_seg_stride;
  p.pos64 = a.pos_bytes == 8; p.seg64 = a.seg_bytes == 8;
  return p;
}
size_t lut_bytes(const RelP& p) { return (2 * (2 * (size_t)p.reach + 1) + 15) & ~(size_t)15; }
int log_threads(int Lk, int cols, int threads) {
  int l = 0;
  while ((1 << l) < threads && (1 << l) * cols < Lk) ++l;
  return l;
}

struct BwdPlan { int threads, tiles, strips; size_t smem; };
BwdPlan bwd_plan(RelP& p, int cols) {
  BwdPlan b;
  b.threads = kThreads;
  while (b.threads > 32 && (size_t)p.rows * b.threads * 4 > 72 * 1024) b.threads /= 2;
  b.smem = lut_bytes(p) + (size_t)p.rows * b.threads * 4;
  p.log_tpr = log_threads(p.Lk, cols, b.threads);
  const int tpr = 1 << p.log_tpr, slots = b.threads >> p.log_tpr;
  b.tiles = (p.Lk + tpr * cols - 1) / (tpr * cols);
  // as many blocks as fit the processors, each with a few rows at least: a block's table costs about as much as four rows of it
  const int fit = (int)(220 * 1024 / (b.smem + 1024));
  const int64_t want = (int64_t)tcx::sm_count() * (fit < 1 ? 1 : fit > 2048 / b.threads ? 2048 / b.threads : fit);
  int64_t strips = (want + (int64_t)p.H * b.tiles - 1) / ((int64_t)p.H * b.tiles);
  const int64_t most = ((int64_t)p.B * p.Lq + 4 * slots - 1) / (4 * slots);
  if (strips > most) strips = most;
  b.strips = (int)(strips < 1 ? 1 : strips > 65535 ? 65535 : strips);
  return b;
}
bool vec_ok(const mf_relpos_args& a, const void* ptr) { return (a.Lk * dtype_size(a.dtype)) % 16 == 0 && (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; }

template <typename T, bool VEC>
int run_fwd(const mf_relpos_args& a, cudaStream_t st) {
  RelP p = relpos_params(a);
  constexpr int kC = Cols<T, VEC>::kC;
  p.log_tpr = log_threads(p.Lk, kC, kThreads);
  const int tpr = 1 << p.log_tpr, slots = kThreads >> p.log_tpr;
  const int tiles = (p.Lk + tpr * kC - 1) / (tpr * kC);
  // heads of a block: all of them, less where the table would take more than 48 KB or the rows do not occupy the processors
  int heads = p.H;
  while (heads > 1 && (size_t)heads * p.rows * sizeof(T) > 48 * 1024) heads = (heads + 1) / 2;
  const int64_t row_blocks = ((int64_t)p.B * p.Lq + slots - 1) / slots, want = 4 * (int64_t)tcx::sm_count();
  while (heads > 1 && row_blocks * tiles * ((p.H + heads - 1) / heads) < want) heads = (heads + 1) / 2;
  const int groups = (p.H + heads - 1) / heads;
  int64_t gy = (2 * want + (int64_t)tiles * groups - 1) / ((int64_t)tiles * groups);
  if (gy > row_blocks) gy = row_blocks;
  if (gy > 65535) gy = 65535;
  const size_t smem = lut_bytes(p) + (size_t)heads * p.rows * sizeof(T);
  constexpr auto kern = relpos_fwd_kernel<T, VEC>;
  if (int e = opt_in_smem<kern>(smem)) return e;
  kern<<<dim3(tiles, (unsigned)gy, groups), kThreads, smem, st>>>(p, a.weight, static_cast<T*>(a.bias), heads);
  MF_LAUNCHED("relpos_fwd_kernel");
  return MF_OK;
}

template <typename T, bool VEC>
int run_bwd(const mf_relpos_args& a, cudaStream_t st) {
  RelP p = relpos_params(a);
  const BwdPlan b = bwd_plan(p, Cols<T, VEC>::kC);
  constexpr auto kern = relpos_bwd_kernel<T, VEC>;
  if (int e = opt_in_smem<kern>(b.smem)) return e;
  float* parts = static_cast<float*>(a.workspace);
  kern<<<dim3(b.tiles, b.strips, p.H), b.threads, b.smem, st>>>(p, static_cast<const T*>(a.d_bias), parts);
  MF_LAUNCHED("relpos_bwd_kernel");
  relpos_join_kernel<<<(p.rows * p.H + kThreads / 32 - 1) / (kThreads / 32), kThreads, 0, st>>>(parts, b.tiles * b.strips, p.H, p.rows, a.d_weight, a.dw_dtype);
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
  size_t most = 0;
  for (bool vec : {true, false}) {                 // whichever the alignment of d_bias asks for
    RelP p = relpos_params(a);
    const BwdPlan b = bwd_plan(p, vec ? 16 / (int)dtype_size(a.dtype) : 8);
    const size_t n = sizeof(float) * (size_t)b.tiles * b.strips * p.H * p.rows;
    if (n > most) most = n;
  }
  return most;
}
int relpos_bwd(const mf_relpos_args& a, cudaStream_t st) {
  int r = MF_OK;
  MF_DISPATCH_FLOAT(a.dtype, T, r = vec_ok(a, a.d_bias) ? run_bwd<T, true>(a, st) : run_bwd<T, false>(a, st));
  return r;
}

}  // namespace mf
