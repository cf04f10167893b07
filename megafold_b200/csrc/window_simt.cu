// Sliding-window attention with sinks on CUDA cores, fp32 arithmetic throughout: fp32 tensors, and what the tensor-core kernels do
// not take (head sizes that are no multiple of 8, unaligned or non-adjacent elements).
//
// Tiles and products are those of the dense attention's CUDA-core kernels.  Forward: a block per (b, n, 64 rows of queries) walks the
// key tiles that its rows see, with the running maximum and sum of the softmax.  Backward, two kinds of blocks in one launch:
// dQ per 64 rows of queries, and dK / dV per 64 keys and chunk of their list of query blocks.  Nothing is added atomically: every
// result is a sum in a fixed order.  Bound: issue slots (62 to 65 % at [1, 2000, 8, 64], window 300 both ways) and reads of shared memory (63 to 72 % of
// the L1's rate), with the FP32 pipe busy 41 to 47 %.
//
// Masked keys, and those of a tile that none of its queries sees, are read as zeros: whatever their rows hold (NaN, too) reaches nothing.  A row that sees no key gives 0, and a
// log-sum-exp of -inf, and passes no gradient.
#include "simt_tiles.cuh"
#include "window_common.cuh"

namespace mf {
namespace win {

namespace {
using namespace simt;

// Rows of a tile of queries: query i0 + r / pack, head h0 + r % pack; `i` is past Lq where there is none.
struct Row { int i, h; };
__device__ __forceinline__ Row query_row(const WinP& p, int i0, int h0, int r) {
  const int l = r / p.pack;
  return Row{l < queries_of<kTile>(p) ? i0 + l : p.Lq, h0 + r - l * p.pack};
}
// kept, for any j; reads the mask without a branch on j
__device__ __forceinline__ bool there(const WinP& p, int b, int n, int j) { return j < p.Lk & kept(p, b, n, j < p.Lk ? j : p.Lk - 1); }

// 64 rows as fp32, zero outside D and where there is none: at(r) is row r's first element or NULL.  The addresses come first, then the loads, then
// the stores: with a mask's byte awaited before each load, the forward of [1, 2720, 16 : 4, 128] took 3.4 ms instead of 2.8.
template <typename T, int DP, typename At>
__device__ __forceinline__ void load_rows(float* dst, bool vec, int64_t sd, int D, At at) {
  constexpr int pitch = DP + 4, kAll = kTile * DP / 4 / kThreads, kOnce = kAll < 4 ? kAll : 4;
#pragma unroll
  for (int i0 = 0; i0 < kAll; i0 += kOnce) {
    const T* from[kOnce];
    float4 v[kOnce];
#pragma unroll
    for (int i = 0; i < kOnce; ++i) {
      const int idx = (i0 + i) * kThreads + threadIdx.x, d = idx % (DP / 4) * 4;
      const T* row = at(idx / (DP / 4));
      from[i] = row && d < D ? row + d * sd : nullptr;
    }
#pragma unroll
    for (int i = 0; i < kOnce; ++i) {
      const int d = ((i0 + i) * kThreads + threadIdx.x) % (DP / 4) * 4;
      const T* p = from[i];
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (vec) {
        if constexpr (sizeof(T) == 4) {
          if (p) v[i] = __ldg(reinterpret_cast<const float4*>(p));
        } else {
          uint2 w = make_uint2(0u, 0u);
          if (p) w = __ldg(reinterpret_cast<const uint2*>(p));
          __align__(8) T e[4];
          *reinterpret_cast<uint2*>(e) = w;
          v[i] = make_float4(to_f(e[0]), to_f(e[1]), to_f(e[2]), to_f(e[3]));
        }
      } else if (p) {
        v[i].x = to_f(p[0]);
        if (d + 1 < D) v[i].y = to_f(p[sd]);
        if (d + 2 < D) v[i].z = to_f(p[2 * sd]);
        if (d + 3 < D) v[i].w = to_f(p[3 * sd]);
      }
    }
#pragma unroll
    for (int i = 0; i < kOnce; ++i) {
      const int idx = (i0 + i) * kThreads + threadIdx.x;
      *reinterpret_cast<float4*>(dst + idx / (DP / 4) * pitch + idx % (DP / 4) * 4) = v[i];
    }
  }
}
template <typename T, int DP>
__device__ __forceinline__ void load_queries(float* dst, const void* src, const int64_t* s, bool vec, const WinP& p, int b, int n, int i0, int h0) {
  const T* base = static_cast<const T*>(src) + b * s[0] + n * s[1];
  load_rows<T, DP>(dst, vec, s[4], p.D, [&](int r) {
    const Row q = query_row(p, i0, h0, r);
    return q.i < p.Lq ? base + q.i * s[2] + q.h * s[3] : nullptr;
  });
}
template <typename T, int DP, typename Keep>
__device__ __forceinline__ void load_keys(float* dst, const void* src, const int64_t* s, bool vec, const WinP& p, int b, int n, int hk, int j0, Keep keep) {
  const T* base = static_cast<const T*>(src) + b * s[0] + n * s[1] + hk * s[3];
  load_rows<T, DP>(dst, vec, s[4], p.D, [&](int r) { return keep(j0 + r) ? base + (j0 + r) * s[2] : nullptr; });
}

template <typename T, int DP>
__device__ __forceinline__ void store_keys(void* out, const WinP& p, int64_t bn, int h, int row0, int ty, int tx, const float (&acc)[4][DP / 16], float f) {
  const int D = p.D;
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const int l = row0 + ty + 16 * a;
    if (l >= p.Lk) continue;
    T* row = static_cast<T*>(out) + ((bn * p.Lk + l) * p.Hk + h) * D;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) {
      const int d = column<DP>(tx, e);
      if (d < D) row[d] = from_f<T>(acc[a][e] * f);
    }
  }
}
template <typename T, int DP>
__device__ __forceinline__ void store_queries(void* out, const WinP& p, int64_t bn, int i0, int h0, int ty, int tx, const float (&acc)[4][DP / 16], const float (&f)[4]) {
  const int D = p.D;
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const Row q = query_row(p, i0, h0, ty + 16 * a);
    if (q.i >= p.Lq) continue;
    T* row = static_cast<T*>(out) + ((bn * p.Lq + q.i) * p.H + q.h) * D;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) {
      const int d = column<DP>(tx, e);
      if (d < D) row[d] = from_f<T>(acc[a][e] * f[a]);
    }
  }
}

// Heads of more than 64 have one buffer for a tile's keys and then its values, so that two blocks fit an SM
// ([1, 2720, 16 : 4, 128], window 2043: 2.83 -> 2.55 ms)
constexpr bool one_buffer(int DP) { return DP > 64; }
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 2) window_fwd_simt_kernel(const __grid_constant__ WinP p, const Split sp) {
  extern __shared__ __align__(16) float smem[];
  constexpr int kOp = kTile * (DP + 4);
  constexpr bool kOne = one_buffer(DP);
  float *Qs = smem, *Ks = Qs + kOp, *Vs = kOne ? Ks : Ks + kOp, *Ps = Vs + kOp;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int h0 = blockIdx.y * p.pack, hk = h0 / p.G, bn = blockIdx.z, b = bn / p.N, n = bn - b * p.N;
  const int part = blockIdx.x % sp.splits, i0 = blockIdx.x / sp.splits * queries_of<kTile>(p);
  const int i1 = i0 + queries_of<kTile>(p) < p.Lq ? i0 + queries_of<kTile>(p) : p.Lq;
  load_queries<T, DP>(Qs, p.q, p.qs, p.q_vec, p, b, n, i0, h0);
  const KeyRange range = key_range(p, i0, i1);
  const auto keep = [&](int j) { return in_range(range, j) & there(p, b, n, j); };
  float acc[4][DP / 16], m[4], l[4];
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    m[a] = -INFINITY; l[a] = 0.f;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) acc[a][e] = 0.f;
  }
  const KeyTiles tiles = key_tiles<kTile>(p, i0, i1);
  const int t_end = (int)((int64_t)tiles.count() * (part + 1) / sp.splits);
  int at[4];
#pragma unroll
  for (int a = 0; a < 4; ++a) at[a] = query_row(p, i0, h0, ty + 16 * a).i;
  for (int t = (int)((int64_t)tiles.count() * part / sp.splits); t < t_end; ++t) {
    const int j0 = tiles.at(t) * kTile;
    __syncthreads();
    load_keys<T, DP>(Ks, p.k, p.ks, p.k_vec, p, b, n, hk, j0, keep);
    if (!kOne) load_keys<T, DP>(Vs, p.v, p.vs, p.v_vec, p, b, n, hk, j0, keep);
    bool see[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) see[c] = keep(j0 + tx + 16 * c);
    __syncthreads();
    float s[4][4] = {};
    dot_tile<DP>(Qs, Ks, ty, tx, s);
#pragma unroll
    for (int a = 0; a < 4; ++a) {
#pragma unroll
      for (int c = 0; c < 4; ++c) s[a][c] = see[c] && in_window(p, at[a], j0 + tx + 16 * c) ? s[a][c] * p.scale : -INFINITY;
      const float m_new = fmaxf(m[a], row_max(fmaxf(fmaxf(s[a][0], s[a][1]), fmaxf(s[a][2], s[a][3]))));
      const float m_ref = m_new == -INFINITY ? 0.f : m_new;         // nothing seen so far
      const float corr = expf(m[a] - m_ref);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float pr = expf(s[a][c] - m_ref);
        sum += pr;
        Ps[(ty + 16 * a) * kPPitch + tx + 16 * c] = pr;
      }
      l[a] = l[a] * corr + row_sum(sum);
      m[a] = m_new;
#pragma unroll
      for (int e = 0; e < DP / 16; ++e) acc[a][e] *= corr;
    }
    if (kOne) {
      __syncthreads();
      load_keys<T, DP>(Vs, p.v, p.vs, p.v_vec, p, b, n, hk, j0, keep);
      __syncthreads();
    } else {
      __syncwarp();              // a row's probabilities are written and read by the same half warp
    }
    sum_tile<DP, true>(Ps, Vs, ty, tx, acc);
  }
  float inv[4];
#pragma unroll
  for (int a = 0; a < 4; ++a) inv[a] = l[a] > 0.f ? 1.f / l[a] : l[a] == 0.f ? 0.f : l[a];      // NaN stays
  if (sp.splits > 1) {
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const Row q = query_row(p, i0, h0, ty + 16 * a);
      if (q.i >= p.Lq) continue;
      const int64_t r = ((int64_t)bn * p.Lq + q.i) * p.H + q.h;
      float* row = sp.row(part, r, p.D);
#pragma unroll
      for (int e = 0; e < DP / 16; ++e)
        if (column<DP>(tx, e) < p.D) row[column<DP>(tx, e)] = acc[a][e] * inv[a];
      if (tx == 0) sp.lse(part, r, p.D) = m[a] + logf(l[a]);
    }
    return;
  }
  store_queries<T, DP>(p.o, p, bn, i0, h0, ty, tx, acc, inv);
  if (tx == 0 && p.lse)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const Row q = query_row(p, i0, h0, ty + 16 * a);
      if (q.i < p.Lq) p.lse[((int64_t)bn * p.H + q.h) * p.Lq + q.i] = m[a] + logf(l[a]);
    }
}

// P and dS of one logit from its product sums
__device__ __forceinline__ void p_ds(const WinP& p, bool see, float s, float dp, float lse, float dl, float& pr, float& ds) {
  pr = see ? expf(fmaf(s, p.scale, -lse)) : 0.f;
  ds = see ? pr * (dp - dl) : 0.f;
}

template <int DP>
__device__ __forceinline__ void add_tile(const float* P, const float* V, int ty, int tx, float (&acc)[4][DP / 16]) {
  float sum[4][DP / 16] = {};
  sum_tile<DP, true>(P, V, ty, tx, sum);
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) acc[a][e] += sum[a][e];
}

template <typename T, int DP>
__device__ __forceinline__ void bwd_dkv(const WinP& p, const KeyPlan& c, float* parts, float* smem, int bn, int hk, int x) {
  constexpr int kOp = kTile * (DP + 4);
  float *Ks = smem, *Vs = Ks + kOp, *Qs = Vs + kOp, *Gs = Qs + kOp, *Ps = Gs + kOp, *Ds = Ps + kTile * kPPitch;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, b = bn / p.N, n = bn - b * p.N;
  int tile, part;
  plan_item(c, x, tile, part);
  const int j0 = tile * kTile, len = list_length<kTile, kTile>(p, tile), e0 = part * c.chunk;
  if (part > 0 && e0 >= len) return;
  const auto keep = [&](int j) { return there(p, b, n, j); };
  load_keys<T, DP>(Ks, p.k, p.ks, p.k_vec, p, b, n, hk, j0, keep);
  load_keys<T, DP>(Vs, p.v, p.vs, p.v_vec, p, b, n, hk, j0, keep);
  int lo, hi;
  query_range(p, j0, j0 + kTile < p.Lk ? j0 + kTile : p.Lk, lo, hi);
  const int nq = queries_of<kTile>(p), first = lo / nq, per_head = hi > lo ? (hi + nq - 1) / nq - first : 1;
  float dk[4][DP / 16] = {}, dv[4][DP / 16] = {};
  bool see[4];
#pragma unroll
  for (int a = 0; a < 4; ++a) see[a] = keep(j0 + ty + 16 * a);
  for (int e = e0; e < len && e < e0 + c.chunk; ++e) {
    const int h0 = hk * p.G + e / per_head * p.pack, i0 = (first + e % per_head) * nq;
    __syncthreads();
    load_queries<T, DP>(Qs, p.q, p.qs, p.q_vec, p, b, n, i0, h0);
    const int64_t gs[5] = {(int64_t)p.N * p.Lq * p.H * p.D, (int64_t)p.Lq * p.H * p.D, (int64_t)p.H * p.D, p.D, 1};
    load_queries<T, DP>(Gs, p.d_o, gs, p.g_vec, p, b, n, i0, h0);
    float lse[4], dl[4];
    int at[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const Row q = query_row(p, i0, h0, tx + 16 * k);
      at[k] = q.i;
      const int64_t row = ((int64_t)bn * p.H + q.h) * p.Lq + q.i;
      lse[k] = q.i < p.Lq ? p.lse[row] : 0.f; dl[k] = q.i < p.Lq ? p.delta[row] : 0.f;
    }
    __syncthreads();
    float s[4][4] = {}, dp[4][4] = {};
    dot_tile<DP>(Ks, Qs, ty, tx, s);
    dot_tile<DP>(Vs, Gs, ty, tx, dp);
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = j0 + ty + 16 * a;
        float pr, ds;
        p_ds(p, see[a] && at[k] < p.Lq && in_window(p, at[k], j), s[a][k], dp[a][k], lse[k], dl[k], pr, ds);
        Ps[(ty + 16 * a) * kPPitch + tx + 16 * k] = pr;
        Ds[(ty + 16 * a) * kPPitch + tx + 16 * k] = ds;
      }
    __syncwarp();
    // a tile's sum on its own: a key with the sinks' list sums thousands of rows, and one running sum of [1, 2720, 16 : 4, 128] was 1.4e-6 off, this is 6e-7
    add_tile<DP>(Ps, Gs, ty, tx, dv);
    add_tile<DP>(Ds, Qs, ty, tx, dk);
  }
  if (x < c.split_x) {
    float* out = part_of<kTile>(parts, c, p, (int64_t)bn * p.Hk + hk, x);
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int e = 0; e < DP / 16; ++e) {
        const int d = column<DP>(tx, e), row = ty + 16 * a;
        if (d < p.D) { out[row * p.D + d] = dk[a][e]; out[(kTile + row) * p.D + d] = dv[a][e]; }
      }
    return;
  }
  store_keys<T, DP>(p.dk, p, bn, hk, j0, ty, tx, dk, p.scale);
  store_keys<T, DP>(p.dv, p, bn, hk, j0, ty, tx, dv, 1.f);
}

template <typename T, int DP>
__device__ __forceinline__ void bwd_dq(const WinP& p, float* smem, int bn, int h0, int i0) {
  constexpr int kOp = kTile * (DP + 4);
  float *Ks = smem, *Vs = Ks + kOp, *Qs = Vs + kOp, *Gs = Qs + kOp, *Ds = Gs + kOp;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, b = bn / p.N, n = bn - b * p.N, hk = h0 / p.G;
  const int i1 = i0 + queries_of<kTile>(p) < p.Lq ? i0 + queries_of<kTile>(p) : p.Lq;
  load_queries<T, DP>(Qs, p.q, p.qs, p.q_vec, p, b, n, i0, h0);
  const int64_t gs[5] = {(int64_t)p.N * p.Lq * p.H * p.D, (int64_t)p.Lq * p.H * p.D, (int64_t)p.H * p.D, p.D, 1};
  load_queries<T, DP>(Gs, p.d_o, gs, p.g_vec, p, b, n, i0, h0);
  const KeyRange range = key_range(p, i0, i1);
  const auto keep = [&](int j) { return in_range(range, j) & there(p, b, n, j); };
  float dq[4][DP / 16] = {}, lse[4], dl[4];
  int at[4];
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const Row q = query_row(p, i0, h0, ty + 16 * a);
    at[a] = q.i;
    const int64_t row = ((int64_t)bn * p.H + q.h) * p.Lq + q.i;
    lse[a] = q.i < p.Lq ? p.lse[row] : 0.f; dl[a] = q.i < p.Lq ? p.delta[row] : 0.f;
  }
  const KeyTiles tiles = key_tiles<kTile>(p, i0, i1);
  for (int t = 0; t < tiles.count(); ++t) {
    const int j0 = tiles.at(t) * kTile;
    __syncthreads();
    load_keys<T, DP>(Ks, p.k, p.ks, p.k_vec, p, b, n, hk, j0, keep);
    load_keys<T, DP>(Vs, p.v, p.vs, p.v_vec, p, b, n, hk, j0, keep);
    bool see[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) see[c] = keep(j0 + tx + 16 * c);
    __syncthreads();
    float s[4][4] = {}, dp[4][4] = {};
    dot_tile<DP>(Qs, Ks, ty, tx, s);
    dot_tile<DP>(Gs, Vs, ty, tx, dp);
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float pr, ds;
        p_ds(p, see[c] && at[a] < p.Lq && in_window(p, at[a], j0 + tx + 16 * c), s[a][c], dp[a][c], lse[a], dl[a], pr, ds);
        Ds[(ty + 16 * a) * kPPitch + tx + 16 * c] = ds;
      }
    __syncwarp();
    sum_tile<DP, true>(Ds, Ks, ty, tx, dq);
  }
  const float sc[4] = {p.scale, p.scale, p.scale, p.scale};
  store_queries<T, DP>(p.dq, p, bn, i0, h0, ty, tx, dq, sc);
}

// blocks [0, n_dkv) work on dK and dV (the longest first: tiles with sinks lead), the others on dQ
// R: blocks of an SM
template <typename T, int DP, int R>
__global__ void __launch_bounds__(kThreads, R) window_bwd_simt_kernel(const __grid_constant__ WinP p, const KeyPlan c, float* parts, int64_t n_dkv) {
  extern __shared__ __align__(16) float smem[];
  const int64_t u = blockIdx.x;
  const int64_t heads = (int64_t)p.B * p.N * p.Hk;
  if (u < n_dkv) {
    const int x = (int)(u / heads);
    const int64_t head = u - (int64_t)x * heads;
    bwd_dkv<T, DP>(p, c, parts, smem, (int)(head / p.Hk), (int)(head % p.Hk), x);
  } else {
    const int groups = head_groups(p);
    const int64_t w = u - n_dkv, all = (int64_t)p.B * p.N * groups;
    const int t = (int)(w / all);
    const int64_t g = w - t * all;
    bwd_dq<T, DP>(p, smem, (int)(g / groups), (int)(g % groups) * p.pack, t * queries_of<kTile>(p));
  }
}

template <typename T>
__global__ void __launch_bounds__(256) window_delta_kernel(const T* __restrict__ o, const T* __restrict__ d_o, float* __restrict__ delta, int64_t rows, int Lq, int H,
                                                           int D, bool vec) {
  // four threads per (b, n, i, h)
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 2;
  const int q = threadIdx.x & 3;
  float s = 0.f;
  if (row < rows) {
    const T *po = o + row * D, *pg = d_o + row * D;
    constexpr int V = 16 / sizeof(T);
    if (vec) {
      for (int d = q * V; d < D; d += 4 * V) {
        __align__(16) T a[V];
        __align__(16) T g[V];
        *reinterpret_cast<uint4*>(a) = __ldg(reinterpret_cast<const uint4*>(po + d));
        *reinterpret_cast<uint4*>(g) = __ldg(reinterpret_cast<const uint4*>(pg + d));
#pragma unroll
        for (int e = 0; e < V; ++e) s = fmaf(to_f(a[e]), to_f(g[e]), s);
      }
    } else {
      for (int d = q; d < D; d += 4) s = fmaf(to_f(po[d]), to_f(pg[d]), s);
    }
  }
  s += __shfl_xor_sync(0xffffffffu, s, 1);
  s += __shfl_xor_sync(0xffffffffu, s, 2);
  if (row < rows && q == 0) {
    const int h = (int)(row % H);
    const int64_t t = row / H, bn = t / Lq;
    delta[(bn * H + h) * Lq + (t - bn * Lq)] = s;
  }
}

// A warp a row: the parts weighed by exp(their log-sum-exp).  Lane s holds the weights of parts s and s + 32.
template <typename T>
__global__ void __launch_bounds__(256) window_split_join_kernel(const __grid_constant__ WinP p, const Split sp) {
  const int64_t r = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (r >= sp.rows) return;
  float w[2], m = -INFINITY, sum = 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    w[k] = lane + 32 * k < sp.splits ? sp.lse(lane + 32 * k, r, p.D) : -INFINITY;
    m = fmaxf(m, w[k]);                                    // a NaN stays in w
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
  for (int k = 0; k < 2; ++k) { w[k] = expf(w[k] - (m == -INFINITY ? 0.f : m)); sum += w[k]; }
  sum = warp_sum(sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  for (int d0 = 0; d0 < p.D; d0 += 32) {
    const int d = d0 + lane;
    float o = 0.f;
#pragma unroll 4
    for (int s = 0; s < sp.splits; ++s) {
      const float ws = __shfl_sync(0xffffffffu, s < 32 ? w[0] : w[1], s & 31);
      if (ws != 0.f && d < p.D) o = fmaf(ws, sp.row(s, r, p.D)[d], o);
    }
    if (d < p.D) static_cast<T*>(p.o)[r * p.D + d] = from_f<T>(o * inv);
  }
  if (lane == 0 && p.lse) {
    const int h = (int)(r % p.H);
    const int64_t t = r / p.H, bn = t / p.Lq;
    p.lse[(bn * p.H + h) * p.Lq + (t - bn * p.Lq)] = m + logf(sum);
  }
}

int simt_splits(const WinP& p) { return split_count<kTile, kTile>(p, 2 * tcx::sm_count()); }

template <typename T>
int run_fwd(const WinP& p, const Split& sp, cudaStream_t st) {
  const auto go = [&](auto dp) -> int {
    constexpr int DP = decltype(dp)::value;
    constexpr size_t smem = sizeof(float) * ((one_buffer(DP) ? 2 : 3) * kTile * (DP + 4) + kTile * kPPitch);
    constexpr auto kern = window_fwd_simt_kernel<T, DP>;
    if (int e = opt_in_smem<kern>(smem)) return e;
    const int q = queries_of<kTile>(p);
    const int64_t gx = (int64_t)((p.Lq + q - 1) / q) * sp.splits;
    MF_REQUIRE(gx <= 0x7fffffff, MF_ERR_UNSUPPORTED, "too many tiles of queries for one launch");
    kern<<<dim3((unsigned)gx, head_groups(p), p.B * p.N), kThreads, smem, st>>>(p, sp);
    MF_LAUNCHED("window_fwd_simt_kernel");
    return MF_OK;
  };
  return p.D <= 32 ? go(std::integral_constant<int, 32>{}) : p.D <= 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
}

template <typename T>
int run_bwd(const WinP& p, const KeyPlan& c, float* parts, cudaStream_t st) {
  const auto go = [&](auto dp) -> int {
    constexpr int DP = decltype(dp)::value;
    constexpr size_t smem = sizeof(float) * (4 * kTile * (DP + 4) + 2 * kTile * kPPitch);
    const int64_t n_dkv = (int64_t)c.x_total * p.B * p.N * p.Hk, q = queries_of<kTile>(p);
    const int64_t blocks = n_dkv + (int64_t)((p.Lq + q - 1) / q) * p.B * p.N * head_groups(p);
    MF_REQUIRE(blocks <= 0x7fffffff, MF_ERR_UNSUPPORTED, "%lld blocks of 64 rows are more than one launch takes", (long long)blocks);
    const auto launch = [&](auto resident) -> int {
      constexpr auto kern = window_bwd_simt_kernel<T, DP, decltype(resident)::value>;
      if (int e = opt_in_smem<kern>(smem)) return e;
      kern<<<(unsigned)blocks, kThreads, smem, st>>>(p, c, parts, n_dkv);
      MF_LAUNCHED("window_bwd_simt_kernel");
      return MF_OK;
    };
    // Two blocks an SM have 128 registers a thread and spill (332 bytes of stores and 440 of loads at DP = 64, 184 and 240 at DP = 32), too few for a block alone: [2, 517, 8 : 2, 24], window 100, 61 us instead of 50, but with 8 times as many tiles
    // ([1, 2000, 8 : 1, 32], window 300) 137 instead of 172 and [1, 2000, 8, 64] 382 instead of 435.
    if constexpr (DP <= 64) {
      if (blocks > 3 * (int64_t)tcx::sm_count()) return launch(std::integral_constant<int, 2>{});
    }
    return launch(std::integral_constant<int, 1>{});
  };
  int r = p.D <= 32 ? go(std::integral_constant<int, 32>{}) : p.D <= 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
  return r ? r : window_join<T, kTile, kTile>(p, c, parts, st);
}

bool rows_vec(const void* ptr, const int64_t* s, int D, size_t es) {
  const int64_t q = 4;
  return s[4] == 1 && D % 4 == 0 && (reinterpret_cast<uintptr_t>(ptr) % (4 * es)) == 0 && s[0] % q == 0 && s[1] % q == 0 && s[2] % q == 0 && s[3] % q == 0;
}

KeyPlan simt_plan(const WinP& p) { return key_plan<kTile, kTile>(p, 2 * tcx::sm_count()); }
}  // namespace

WinP window_params(const mf_window_args& a) {
  WinP p{};
  p.B = a.B; p.N = a.N; p.Lq = a.Lq; p.Lk = a.Lk; p.H = a.H; p.Hk = a.Hk; p.D = a.D; p.G = a.H / a.Hk;
  p.pack = p.G <= 64 ? p.G : 1;
  const int reach = a.Lq + a.Lk;                       // wider than that sees no more
  p.left = a.left < reach ? a.left : reach; p.right = a.right < reach ? a.right : reach;
  p.sinks = a.sinks < a.Lk ? a.sinks : a.Lk;
  p.off = a.Lk - a.Lq;
  p.scale = 1.f / sqrtf((float)a.D);
  p.q = a.q; p.k = a.k; p.v = a.v;
  for (int i = 0; i < 5; ++i) { p.qs[i] = a.q_strides[i]; p.ks[i] = a.k_strides[i]; p.vs[i] = a.v_strides[i]; }
  p.mask = static_cast<const uint8_t*>(a.mask);
  for (int i = 0; i < 3; ++i) p.ms[i] = a.mask_strides[i];
  p.o = a.o; p.lse = a.lse; p.d_o = a.d_o; p.dq = a.dq; p.dk = a.dk; p.dv = a.dv;
  const size_t es = dtype_size(a.dtype);
  const int64_t gs[5] = {0, 0, 0, a.D, 1};
  p.q_vec = rows_vec(a.q, p.qs, a.D, es); p.k_vec = rows_vec(a.k, p.ks, a.D, es); p.v_vec = rows_vec(a.v, p.vs, a.D, es);
  p.g_vec = rows_vec(a.d_o, gs, a.D, es);
  return p;
}

int window_split_join(const WinP& p, int dtype, const Split& s, cudaStream_t st) {
  MF_DISPATCH_FLOAT(dtype, T, {
    window_split_join_kernel<T><<<(unsigned)((s.rows + 7) / 8), 256, 0, st>>>(p, s);
    MF_LAUNCHED("window_split_join_kernel");
  });
  return MF_OK;
}

int window_delta(const WinP& p, int dtype, float* delta, cudaStream_t st) {
  const int64_t rows = (int64_t)p.B * p.N * p.Lq * p.H, blocks = (rows + 63) / 64;
  MF_REQUIRE(blocks <= 0x7fffffff, MF_ERR_UNSUPPORTED, "too many query rows");
  const size_t es = dtype_size(dtype);
  const bool vec = (p.D * es) % 16 == 0 && ((reinterpret_cast<uintptr_t>(p.o) | reinterpret_cast<uintptr_t>(p.d_o)) & 15) == 0;
  MF_DISPATCH_FLOAT(dtype, T, {
    window_delta_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(static_cast<const T*>(p.o), static_cast<const T*>(p.d_o), delta, rows, p.Lq, p.H, p.D, vec);
    MF_LAUNCHED("window_delta_kernel");
  });
  return MF_OK;
}

}  // namespace win

using namespace win;

size_t window_fwd_simt_workspace(const mf_window_args& a) {
  const WinP p = window_params(a);
  return split_bytes(p, simt_splits(p));
}

int window_fwd_simt(const mf_window_args& a, cudaStream_t st) {
  const WinP p = window_params(a);
  const Split sp{simt_splits(p), static_cast<float*>(a.workspace), (int64_t)p.B * p.N * p.Lq * p.H};
  int r = MF_OK;
  MF_DISPATCH_FLOAT(a.dtype, T, r = run_fwd<T>(p, sp, st));
  return r || sp.splits == 1 ? r : window_split_join(p, a.dtype, sp, st);
}

size_t window_bwd_simt_workspace(const mf_window_args& a) {
  const WinP p = window_params(a);
  return align_up(sizeof(float) * (size_t)p.B * p.N * p.H * p.Lq, 256) + sizeof(float) * part_floats<kTile>(simt_plan(p), p);
}

int window_bwd_simt(const mf_window_args& a, cudaStream_t st) {
  WinP p = window_params(a);
  float* delta = static_cast<float*>(a.workspace);
  float* parts = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + align_up(sizeof(float) * (size_t)p.B * p.N * p.H * p.Lq, 256));
  if (int r = window_delta(p, a.dtype, delta, st)) return r;
  p.delta = delta;
  int r = MF_OK;
  MF_DISPATCH_FLOAT(a.dtype, T, r = run_bwd<T>(p, simt_plan(p), parts, st));
  return r;
}

}  // namespace mf
