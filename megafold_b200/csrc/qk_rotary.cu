// RMS norm of every head of queries and keys and their rotation by position, in one pass, and its backward.
//
//   y = x * rstd * w,  rstd = (mean_d x^2 + eps)^-1/2;   out = the pairs of y's first R elements turned by pos * inv_freq, the rest of y
//   g = d_out turned back;  dx = rstd * (w g - hat * mean_d(w g hat)),  hat = x * rstd;   dw = sum over tokens (and heads) of g * hat
//
// A head's row is a few threads, each with V pairs: two pieces of V elements that turn together (R / 2 apart, or adjacent where
// pairs are interleaved), so that nothing but the sum of squares crosses threads.  Angles are formed and
// reduced in 64 bits (a position of a million times a frequency in 32 bits is off by 0.06); a thread computes its V angles once for all heads of its token that it goes through.  Sums and norms are
// fp32, the outputs are rounded once.  The weights' gradients are summed in a fixed order: a thread over its tokens, a block over its threads
// in shared memory, a second kernel over the blocks.
//
// Bound: HBM; for single tokens latency.
#include "evo_tc_common.cuh"

namespace mf {
namespace {
using tcx::add2; using tcx::fma2; using tcx::mul2; using tcx::sub2;

constexpr int kThreads = 256;

struct RotP {
  int N, L, H, Hk, D, R;
  int64_t tokens;                           // B * N * L
  const void *q, *k; int64_t qs[5], ks[5];
  const void *qw, *kw; int w_dtype; int64_t w_head;      // weights (NULL: ones); elements between heads, 0: shared
  const float* inv_freq;
  const void* pos; int64_t ps[3]; bool pos64;            // NULL: the index along L
  float eps;
  int heads_per;                            // heads that a thread goes through
  int log_lpr;                              // threads of a row
  void *q_out, *k_out;                      // contiguous
  const void *dq_out, *dk_out; void *dq, *dk;
  float* parts;                             // [gridDim.y][gridDim.x][2][D]
};

// Sine and cosine of pos * f, in half turns: the whole quarters are taken off in 64 bits, exactly but for the one rounding of the
// product with 1 / pi, and what is left, at most a quarter, goes to CUDA's sincospif.
__device__ __forceinline__ void turn_of(double pos, float f, float& s, float& c) {
  const double t = pos * (double)f * 0.31830988618379067154, k = rint(2. * t);
  float sr, cr;
  sincospif((float)fma(k, -0.5, t), &sr, &cr);
  const int quarter = (int)((long long)k & 3);
  const float s1 = quarter & 1 ? cr : sr, c1 = quarter & 1 ? sr : cr;
  s = quarter & 2 ? -s1 : s1;
  c = quarter == 1 || quarter == 2 ? -c1 : c1;
}

template <typename T, int V> struct alignas(sizeof(T) * V) Piece { T v[V]; };

// A thread's unit u of a row: V pairs, or, behind the rotated part, up to 2 V elements that are not turned.
template <int V, bool IL>
struct Unit {
  int a, b;                 // first elements of the two pieces
  bool turned, has_a, has_b;
  __device__ __forceinline__ Unit(int u, int R, int D) {
    const int nr = R / 2 / V;
    turned = u < nr;
    if (turned) { a = IL ? 2 * V * u : V * u; b = IL ? a + V : R / 2 + a; has_a = has_b = true; }
    else { a = R + 2 * V * (u - nr); b = a + V; has_a = a < D; has_b = b < D; }
  }
};
// the two pieces of a unit as they are in memory
template <typename T, int V> struct Raw { Piece<T, V> p, q; };
template <typename T, int V, bool IL>
__device__ __forceinline__ void load_unit(const T* row, int64_t sd, const Unit<V, IL>& u, Raw<T, V>& r) {
  if constexpr (V == 1) {
    r.p.v[0] = u.has_a ? row[u.a * sd] : from_f<T>(0.f);
    r.q.v[0] = u.has_b ? row[u.b * sd] : from_f<T>(0.f);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) r.p.v[e] = r.q.v[e] = from_f<T>(0.f);
    if (u.has_a) r.p = *reinterpret_cast<const Piece<T, V>*>(row + u.a);
    if (u.has_b) r.q = *reinterpret_cast<const Piece<T, V>*>(row + u.b);
  }
}
// The first and the second elements of a unit's V pairs (or the two pieces of an unturned unit), two to a register pair: packed fp32
// arithmetic takes half the issue slots, which bound these kernels (V = 1: the second of each two is 0).
template <int V> struct Vec {
  static constexpr int P = (V + 1) / 2;
  float2 a[P], b[P];
};
template <int V> __device__ __forceinline__ float get(const float2 (&x)[(V + 1) / 2], int e) { return e % 2 ? x[e / 2].y : x[e / 2].x; }
template <int V> __device__ __forceinline__ void put(float2 (&x)[(V + 1) / 2], int e, float v) { if (e % 2) x[e / 2].y = v; else x[e / 2].x = v; }
template <typename T, int V, bool IL>
__device__ __forceinline__ void unpack_unit(const Raw<T, V>& r, Vec<V>& x) {
  if constexpr (V == 1) x.a[0].y = x.b[0].y = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if constexpr (IL && V > 1) {
      put<V>(x.a, e, to_f(2 * e < V ? r.p.v[2 * e] : r.q.v[2 * e - V]));
      put<V>(x.b, e, to_f(2 * e + 1 < V ? r.p.v[2 * e + 1] : r.q.v[2 * e + 1 - V]));
    } else {
      put<V>(x.a, e, to_f(r.p.v[e])); put<V>(x.b, e, to_f(r.q.v[e]));
    }
  }
}
template <typename T, int V, bool IL>
__device__ __forceinline__ void store_unit(T* row, const Unit<V, IL>& u, const Vec<V>& x) {
  Piece<T, V> p, q;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if constexpr (IL && V > 1) {
      (2 * e < V ? p.v[2 * e] : q.v[2 * e - V]) = from_f<T>(get<V>(x.a, e));
      (2 * e + 1 < V ? p.v[2 * e + 1] : q.v[2 * e + 1 - V]) = from_f<T>(get<V>(x.b, e));
    } else {
      p.v[e] = from_f<T>(get<V>(x.a, e)); q.v[e] = from_f<T>(get<V>(x.b, e));
    }
  }
  if (u.has_a) *reinterpret_cast<Piece<T, V>*>(row + u.a) = p;
  if (u.has_b) *reinterpret_cast<Piece<T, V>*>(row + u.b) = q;
}
// index in a row of D elements of the e-th of the first / second elements
template <int V, bool IL>
__device__ __forceinline__ int element(const Unit<V, IL>& u, int e) {
  if constexpr (IL) { const int i = e < V ? 2 * e : 2 * (e - V) + 1; return u.a + i; }      // the pieces are adjacent
  else return e < V ? u.a + e : u.b + e - V;
}
// the weights of a unit from a row of fp32 in shared memory (any number where there is no element: x is 0 there)
template <int V, bool IL>
__device__ __forceinline__ void load_weight(const float* w, const Unit<V, IL>& u, Vec<V>& out) {
  const int a = u.has_a ? u.a : 0, b = u.has_b ? u.b : 0;
  if constexpr (V == 1) out.a[0].y = out.b[0].y = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if constexpr (IL && V > 1) {
      put<V>(out.a, e, 2 * e < V ? w[a + 2 * e] : w[b + 2 * e - V]);
      put<V>(out.b, e, 2 * e + 1 < V ? w[a + 2 * e + 1] : w[b + 2 * e + 1 - V]);
    } else {
      put<V>(out.a, e, w[a + e]); put<V>(out.b, e, w[b + e]);
    }
  }
}
__device__ __forceinline__ float row_sum(float v, int lpr) {
  for (int o = lpr >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// blockIdx.y = group of heads_per heads (of the H + Hk of queries and keys); threads of a block walk tokens.
// UPL: units of a thread.  (Every thread of a warp takes part in each sum: rows that do not exist are zeros.)
// The weights of the block's heads wait in shared memory as fp32: read from global memory for each row, converted from a type known
// at run time, they were most of the instructions (4 + 4 heads of 32, 147456 tokens: 96 us forward, 220 backward).
template <typename T, int V, int UPL, bool IL, bool BWD>
__global__ void __launch_bounds__(kThreads, UPL > 1 ? 2 : BWD ? 3 : 4) qk_rotary_kernel(const __grid_constant__ RotP p) {
  const int lpr = 1 << p.log_lpr, lane = threadIdx.x & (lpr - 1), slot = threadIdx.x >> p.log_lpr, slots = kThreads >> p.log_lpr;
  const int heads = p.H + p.Hk, g0 = blockIdx.y * p.heads_per, g1 = g0 + p.heads_per < heads ? g0 + p.heads_per : heads;
  const float inv_d = 1.f / p.D;
  extern __shared__ __align__(16) float shared[];
  float* const ws = shared;                                    // [1 (no weights), 2 (shared: q, k) or heads of the group][D]
  if (!p.qw) {
    for (int x = threadIdx.x; x < p.D; x += kThreads) ws[x] = 1.f;
  } else if (!p.w_head) {
    for (int x = threadIdx.x; x < 2 * p.D; x += kThreads) ws[x] = x < p.D ? load_rt(p.qw, x, p.w_dtype) : load_rt(p.kw, x - p.D, p.w_dtype);
  } else {
    for (int x = threadIdx.x; x < (g1 - g0) * p.D; x += kThreads) {
      const int64_t at = (int64_t)g0 * p.D + x, nq = (int64_t)p.H * p.D;
      ws[x] = at < nq ? load_rt(p.qw, at, p.w_dtype) : load_rt(p.kw, at - nq, p.w_dtype);
    }
  }
  __syncthreads();
  constexpr int P = Vec<V>::P;
  Vec<V> dwq[BWD ? UPL : 1] = {}, dwk[BWD ? UPL : 1] = {};
  const int64_t stride = (int64_t)gridDim.x * slots;
  for (int64_t t0 = (int64_t)blockIdx.x * slots; t0 < p.tokens; t0 += stride) {
    const int64_t tok = t0 + slot;
    const bool live = tok < p.tokens;
    const uint32_t bn = live ? (uint32_t)tok / (uint32_t)p.L : 0, l = live ? (uint32_t)tok - bn * p.L : 0, b = bn / (uint32_t)p.N, n = bn - b * p.N;
    const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + n * p.qs[1] + l * p.qs[2];
    const T* kk = static_cast<const T*>(p.k) + b * p.ks[0] + n * p.ks[1] + l * p.ks[2];
    auto unit = [&](int k) {
      Unit<V, IL> u(lane + k * lpr, p.R, p.D);
      u.has_a = u.has_a && live; u.has_b = u.has_b && live;
      return u;
    };
    auto fetch = [&](int g, Raw<T, V> (&x)[UPL], Raw<T, V> (&d)[BWD ? UPL : 1]) {
      const bool is_q = g < p.H;
      const int h = is_q ? g : g - p.H;
      const T* row = is_q ? q + h * p.qs[3] : kk + h * p.ks[3];
#pragma unroll
      for (int k = 0; k < UPL; ++k) load_unit<T, V, IL>(row, is_q ? p.qs[4] : p.ks[4], unit(k), x[k]);
      if constexpr (BWD) {
        const T* dr = static_cast<const T*>(is_q ? p.dq_out : p.dk_out) + (tok * (is_q ? p.H : p.Hk) + h) * p.D;
#pragma unroll
        for (int k = 0; k < UPL; ++k) load_unit<T, V, IL>(dr, 1, unit(k), d[k]);
      }
    };
    Raw<T, V> xr[UPL], dr[BWD ? UPL : 1];
    fetch(g0, xr, dr);                                         // on its way while the angles are formed
    double pos = (double)l;
    if (p.pos) {
      const int64_t at = b * p.ps[0] + n * p.ps[1] + l * p.ps[2];
      pos = p.pos64 ? (double)static_cast<const int64_t*>(p.pos)[at] : (double)static_cast<const int32_t*>(p.pos)[at];
    }
    Vec<V> turn[UPL];                                          // a: cosines, b: sines
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
      const int u = lane + k * lpr;
      const bool turned = u < p.R / 2 / V;
#pragma unroll
      for (int e = 0; e < P; ++e) { turn[k].a[e] = make_float2(1.f, 1.f); turn[k].b[e] = make_float2(0.f, 0.f); }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float sn, cs;
        if (turned && live) { turn_of(pos, p.inv_freq[u * V + e], sn, cs); put<V>(turn[k].a, e, cs); put<V>(turn[k].b, e, sn); }
      }
    }
    for (int g = g0; g < g1; ++g) {
      const bool is_q = g < p.H;
      const int h = is_q ? g : g - p.H;
      const int64_t out_at = (tok * (is_q ? p.H : p.Hk) + h) * p.D;
      const float* w = ws + (!p.qw ? 0 : !p.w_head ? (is_q ? 0 : p.D) : (g - g0) * p.D);
      Vec<V> x[UPL], d[BWD ? UPL : 1];
      float2 ss2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int k = 0; k < UPL; ++k) {
        unpack_unit<T, V, IL>(xr[k], x[k]);
        if constexpr (BWD) unpack_unit<T, V, IL>(dr[k], d[k]);
#pragma unroll
        for (int e = 0; e < P; ++e) ss2 = fma2(x[k].b[e], x[k].b[e], fma2(x[k].a[e], x[k].a[e], ss2));
      }
      if (g + 1 < g1) fetch(g + 1, xr, dr);
      const float rstd = rsqrtf(fmaf(row_sum(ss2.x + ss2.y, lpr), inv_d, p.eps));
      const float2 rstd2 = make_float2(rstd, rstd);
      if constexpr (!BWD) {
        T* out = static_cast<T*>(is_q ? p.q_out : p.k_out) + out_at;
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
          const Unit<V, IL> u = unit(k);
          Vec<V> wt;
          load_weight<V, IL>(w, u, wt);
#pragma unroll
          for (int e = 0; e < P; ++e) {
            const float2 ya = mul2(mul2(x[k].a[e], rstd2), wt.a[e]), yb = mul2(mul2(x[k].b[e], rstd2), wt.b[e]), c = turn[k].a[e], s = turn[k].b[e];
            x[k].a[e] = sub2(mul2(ya, c), mul2(yb, s));        // by 1 and 0 where nothing turns
            x[k].b[e] = fma2(ya, s, mul2(yb, c));
          }
          store_unit<T, V, IL>(out, u, x[k]);
        }
      } else {
        float2 dot2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
          Vec<V> wt;
          load_weight<V, IL>(w, unit(k), wt);
#pragma unroll
          for (int e = 0; e < P; ++e) {
            const float2 c = turn[k].a[e], s = turn[k].b[e], da = d[k].a[e], db = d[k].b[e];
            const float2 ga = fma2(db, s, mul2(da, c)), gb = sub2(mul2(db, c), mul2(da, s));
            x[k].a[e] = mul2(x[k].a[e], rstd2); x[k].b[e] = mul2(x[k].b[e], rstd2);        // hat
            const float2 ta = mul2(ga, x[k].a[e]), tb = mul2(gb, x[k].b[e]);
            if (is_q) { dwq[k].a[e] = add2(dwq[k].a[e], ta); dwq[k].b[e] = add2(dwq[k].b[e], tb); }
            else { dwk[k].a[e] = add2(dwk[k].a[e], ta); dwk[k].b[e] = add2(dwk[k].b[e], tb); }
            dot2 = fma2(tb, wt.b[e], fma2(ta, wt.a[e], dot2));
            d[k].a[e] = mul2(ga, wt.a[e]); d[k].b[e] = mul2(gb, wt.b[e]);
          }
        }
        const float dot = row_sum(dot2.x + dot2.y, lpr) * -inv_d;
        const float2 minus = make_float2(dot, dot);
        T* out = static_cast<T*>(is_q ? p.dq : p.dk) + out_at;
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
#pragma unroll
          for (int e = 0; e < P; ++e) {
            x[k].a[e] = mul2(rstd2, fma2(x[k].a[e], minus, d[k].a[e]));
            x[k].b[e] = mul2(rstd2, fma2(x[k].b[e], minus, d[k].b[e]));
          }
          store_unit<T, V, IL>(out, unit(k), x[k]);
        }
      }
    }
  }
  if constexpr (BWD) {
    if (!p.parts) return;
    float* const sum = shared;                                 // [slots][D]
    float* out = p.parts + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * p.D;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < UPL; ++k) {
        const Unit<V, IL> u(lane + k * lpr, p.R, p.D);
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) {
          const int i = element<V, IL>(u, e);
          const Vec<V>& dw = which ? dwk[k] : dwq[k];
          if (i < p.D && (u.turned || i >= p.R)) sum[slot * p.D + i] = e < V ? get<V>(dw.a, e) : get<V>(dw.b, e - V);
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < p.D; i += kThreads) {
        float s = 0.f;
        for (int k = 0; k < slots; ++k) s += sum[k * p.D + i];
        out[which * p.D + i] = s;
      }
    }
  }
}

// Weight gradients: blockIdx = (32 elements, row of [H or 1 + Hk or 1]); a row is the sum of its blocks' rows, 32 of them at a time.
__global__ void __launch_bounds__(1024) qk_rotary_join_kernel(const float* __restrict__ parts, int gx, int gy, int D, int H, int Hk, bool per_head, void* __restrict__ dqw,
                                                              void* __restrict__ dkw, int w_dtype) {
  __shared__ float sums[32][33];
  const int q_rows = per_head ? H : 1, row = blockIdx.y, i = blockIdx.x * 32 + (threadIdx.x & 31), warp = threadIdx.x >> 5;
  const bool is_k = row >= q_rows;
  const int64_t k0 = per_head ? (int64_t)row * gx : 0, k1 = per_head ? k0 + gx : (int64_t)gy * gx;        // per head: a group of blocks each, queries' heads first
  float s = 0.f;
  if (i < D) {
#pragma unroll 8
    for (int64_t k = k0 + warp; k < k1; k += 32) s += parts[(k * 2 + is_k) * D + i];
  }
  sums[warp][threadIdx.x & 31] = s;
  __syncthreads();
  if (warp || i >= D) return;
  s = 0.f;
  for (int k = 0; k < 32; ++k) s += sums[k][threadIdx.x];
  if (is_k) store_rt(dkw, (int64_t)(row - q_rows) * D + i, w_dtype, s);
  else store_rt(dqw, (int64_t)row * D + i, w_dtype, s);
}

RotP rot_params(const mf_qk_rotary_args& a) {
  RotP p{};
  p.N = a.N; p.L = a.L; p.H = a.H; p.Hk = a.Hk; p.D = a.D; p.R = a.R; p.tokens = (int64_t)a.B * a.N * a.L;
  p.q = a.q; p.k = a.k;
  for (int i = 0; i < 5; ++i) { p.qs[i] = a.q_strides[i]; p.ks[i] = a.k_strides[i]; }
  p.qw = a.q_weight; p.kw = a.k_weight; p.w_dtype = a.w_dtype; p.w_head = a.per_head ? a.D : 0;
  p.inv_freq = a.inv_freq; p.pos = a.positions; p.pos64 = a.pos_bytes == 8;
  for (int i = 0; i < 3; ++i) p.ps[i] = a.pos_strides[i];
  p.eps = a.eps; p.q_out = a.q_out; p.k_out = a.k_out;
  p.dq_out = a.dq_out; p.dk_out = a.dk_out; p.dq = a.dq; p.dk = a.dk;
  return p;
}

// Elements of a piece: the widest load that sizes, strides and addresses allow, 16 bytes on the forward and 8 on the backward, where a
// thread holds twice as much and the sums of the weights' gradients besides (with 16 bytes 176 registers, one block of
// 256 threads on an SM).
int piece_limit(int dtype, bool bwd) { return (bwd ? 8 : 16) / (int)dtype_size(dtype); }
int piece(const mf_qk_rotary_args& a, bool bwd) {
  const int es = (int)dtype_size(a.dtype);
  for (int v = piece_limit(a.dtype, bwd); v > 1; v /= 2) {
    bool ok = a.R / 2 % v == 0 && (a.D - a.R) % v == 0 && a.q_strides[4] == 1 && a.k_strides[4] == 1;
    for (int i = 0; i < 4; ++i) ok = ok && a.q_strides[i] % v == 0 && a.k_strides[i] % v == 0;
    const uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.k | (bwd ? (uintptr_t)a.dq_out | (uintptr_t)a.dk_out | (uintptr_t)a.dq | (uintptr_t)a.dk
                                                                : (uintptr_t)a.q_out | (uintptr_t)a.k_out);
    if (ok && at % (v * es) == 0) return v;
  }
  return 1;
}
int units_per(int V) { return V >= 4 ? 1 : V == 2 ? 2 : 4; }

struct Plan { int log_lpr, heads_per, gx, gy; };
Plan plan(const mf_qk_rotary_args& a, int V, bool bwd) {
  Plan c;
  const int units = a.R / 2 / V + (a.D - a.R + 2 * V - 1) / (2 * V), lanes = (units + units_per(V) - 1) / units_per(V);
  c.log_lpr = 0;
  while ((1 << c.log_lpr) < lanes) ++c.log_lpr;
  const int slots = kThreads >> c.log_lpr, heads = a.H + a.Hk;
  const int64_t tokens = (int64_t)a.B * a.N * a.L, blocks = (tokens + slots - 1) / slots, want = 8 * (int64_t)tcx::sm_count();
  // every head of a token in one thread, which computes the angles once; fewer where that leaves processors idle, and one where
  // each head has a weight of its own whose gradient a block sums
  c.heads_per = heads;
  if (bwd && a.per_head && a.dq_weight) c.heads_per = 1;
  if (a.per_head && a.q_weight)
    while (c.heads_per > 1 && (size_t)c.heads_per * a.D * sizeof(float) > 24 * 1024) c.heads_per = (c.heads_per + 1) / 2;
  while (c.heads_per > 1 && blocks * ((heads + c.heads_per - 1) / c.heads_per) < want) c.heads_per = (c.heads_per + 1) / 2;
  c.gy = (heads + c.heads_per - 1) / c.heads_per;
  int64_t gx = blocks;
  if (bwd) { const int64_t most = (want + c.gy - 1) / c.gy; if (gx > most) gx = most; }
  if (gx > 0x7fffffff) gx = 0x7fffffff;
  c.gx = (int)gx;
  return c;
}

template <typename T, int V, bool BWD>
int run(const mf_qk_rotary_args& a, cudaStream_t st) {
  constexpr int UPL = V >= 4 ? 1 : V == 2 ? 2 : 4;
  RotP p = rot_params(a);
  const Plan c = plan(a, V, BWD);
  p.log_lpr = c.log_lpr; p.heads_per = c.heads_per;
  size_t smem = sizeof(float) * a.D * (!a.q_weight ? 1 : !a.per_head ? 2 : c.heads_per);
  if (BWD && a.dq_weight) {
    p.parts = static_cast<float*>(a.workspace);
    const size_t sums = sizeof(float) * (kThreads >> c.log_lpr) * a.D;
    if (sums > smem) smem = sums;
  }
  const auto go = [&](auto il) -> int {
    constexpr auto kern = qk_rotary_kernel<T, V, UPL, decltype(il)::value, BWD>;
    if (int e = opt_in_smem<kern>(smem)) return e;
    kern<<<dim3(c.gx, c.gy), kThreads, smem, st>>>(p);
    MF_LAUNCHED("qk_rotary_kernel");
    return MF_OK;
  };
  if (int e = a.interleaved ? go(std::true_type{}) : go(std::false_type{})) return e;
  if (BWD && a.dq_weight) {
    const int rows = a.per_head ? a.H + a.Hk : 2;
    qk_rotary_join_kernel<<<dim3((a.D + 31) / 32, rows), 1024, 0, st>>>(p.parts, c.gx, c.gy, a.D, a.H, a.Hk, a.per_head != 0, a.dq_weight, a.dk_weight,
                                                                                                a.w_dtype);
    MF_LAUNCHED("qk_rotary_join_kernel");
  }
  return MF_OK;
}
template <typename T, bool BWD>
int dispatch(const mf_qk_rotary_args& a, cudaStream_t st) {
  constexpr int kMost = (BWD ? 8 : 16) / (int)sizeof(T);
  const int v = piece(a, BWD);
  if constexpr (kMost >= 8) if (v == 8) return run<T, 8, BWD>(a, st);
  if constexpr (kMost >= 4) if (v == 4) return run<T, 4, BWD>(a, st);
  return v == 2 ? run<T, 2, BWD>(a, st) : run<T, 1, BWD>(a, st);
}
}  // namespace

int qk_rotary_fwd(const mf_qk_rotary_args& a, cudaStream_t st) {
  int r = MF_OK;
  MF_DISPATCH_FLOAT(a.dtype, T, r = (dispatch<T, false>(a, st)));
  return r;
}
size_t qk_rotary_bwd_workspace(const mf_qk_rotary_args& a) {
  if (!a.dq_weight) return 0;
  size_t most = 0;
  for (int v = 1; v <= piece_limit(a.dtype, true); v *= 2) {       // whichever width the alignment allows
    if (a.R / 2 % v || (a.D - a.R) % v) break;
    const Plan c = plan(a, v, true);
    const size_t n = sizeof(float) * 2 * a.D * (size_t)c.gx * c.gy;
    if (n > most) most = n;
  }
  return most;
}
int qk_rotary_bwd(const mf_qk_rotary_args& a, cudaStream_t st) {
  int r = MF_OK;
  MF_DISPATCH_FLOAT(a.dtype, T, r = (dispatch<T, true>(a, st)));
  return r;
}

}  // namespace mf
