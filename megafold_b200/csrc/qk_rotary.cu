// RMS norm of every head of queries and keys and their rotation by position, in one pass, and its backward.
//
//   y = x * rstd * w,  rstd = (mean_d x^2 + eps)^-1/2;   out = the pairs of y's first R elements turned by pos * inv_freq, the rest of y
//   g = d_out turned back;  dx = rstd * (w g - hat * mean_d(w g hat)),  hat = x * rstd;   dw = sum over tokens (and heads) of g * hat
//
// A head's row is a few threads, each with V pairs: two pieces of V elements that turn together (R / 2 apart, or adjacent where
// pairs are interleaved), so that nothing but the sum of squares crosses threads.  Angles are formed and
// reduced in 64 bits (a position of a million times a frequency in 32 bits is off by 0.06), once a token and block.  Sums and norms are
// fp32, the outputs are rounded once.  The weights' gradients are summed in a fixed order: a thread over its tokens, a block over its
// threads in shared memory, a second kernel over the blocks.
//
// Bound: issue slots and the latency of the instructions (0.57 of the copy rate); for single tokens the latency of a launch.
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
  uint32_t pair_magic;                      // 2^20 / (R / 2), rounded up
  int hb, tb, mt;                           // a block's heads, its tokens at a time and its tokens in a chunk
  int spans;                                // chunks of a sequence where all sequences have the same positions, else 0
  int log_lpr;                              // threads of a row
  void *q_out, *k_out;                      // contiguous
  const void *dq_out, *dk_out; void *dq, *dk;
  float* parts;                             // sums of the blocks, for the weights' gradients
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
// The two pieces of a unit as they are in memory, in 32-bit words (arrays of 16-bit elements went through local memory).
template <typename T, int V> struct Raw {
  static constexpr int B = sizeof(T) * V, W = (B + 3) / 4;
  uint32_t p[W], q[W];
};
template <int B>
__device__ __forceinline__ void load_words(const void* at, uint32_t (&w)[(B + 3) / 4]) {
  if constexpr (B == 16) { const uint4 v = *static_cast<const uint4*>(at); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
  else if constexpr (B == 8) { const uint2 v = *static_cast<const uint2*>(at); w[0] = v.x; w[1] = v.y; }
  else if constexpr (B == 4) w[0] = *static_cast<const uint32_t*>(at);
  else w[0] = *static_cast<const uint16_t*>(at);
}
template <int B>
__device__ __forceinline__ void store_words(void* at, const uint32_t (&w)[(B + 3) / 4]) {
  if constexpr (B == 16) *static_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (B == 8) *static_cast<uint2*>(at) = make_uint2(w[0], w[1]);
  else if constexpr (B == 4) *static_cast<uint32_t*>(at) = w[0];
  else *static_cast<uint16_t*>(at) = (uint16_t)w[0];
}
template <typename T, int V, bool IL>
__device__ __forceinline__ void load_unit(const T* row, int64_t sd, const Unit<V, IL>& u, Raw<T, V>& r) {
#pragma unroll
  for (int e = 0; e < Raw<T, V>::W; ++e) r.p[e] = r.q[e] = 0u;
  if (u.has_a) load_words<Raw<T, V>::B>(row + (V == 1 ? u.a * sd : u.a), r.p);
  if (u.has_b) load_words<Raw<T, V>::B>(row + (V == 1 ? u.b * sd : u.b), r.q);
}
// element pair k (elements 2 k and 2 k + 1; of a single element the first) of a piece
template <typename T, int V> __device__ __forceinline__ float2 pair_of(const uint32_t (&w)[Raw<T, V>::W], int k) {
  if constexpr (sizeof(T) == 2) { const float2 v = tcx::Pack2<T>::unpack(w[k]); return V == 1 ? make_float2(v.x, 0.f) : v; }
  else return make_float2(__uint_as_float(w[2 * k]), V == 1 ? 0.f : __uint_as_float(w[(2 * k + 1) % Raw<T, V>::W]));
}
template <typename T, int V> __device__ __forceinline__ void set_pair(uint32_t (&w)[Raw<T, V>::W], int k, float2 v) {
  if constexpr (sizeof(T) == 2) w[k] = tcx::Pack2<T>::pack(v.x, v.y);
  else { w[2 * k] = __float_as_uint(v.x); if (V > 1) w[(2 * k + 1) % Raw<T, V>::W] = __float_as_uint(v.y); }
}

// The first and the second elements of a unit's V pairs (or the two pieces of an unturned unit), two to a register pair: packed fp32
// arithmetic takes half the issue slots (V = 1: the second of each two is 0).
template <int V> struct Vec {
  static constexpr int P = (V + 1) / 2;
  float2 a[P], b[P];
};
template <int V> __device__ __forceinline__ float get(const float2 (&x)[(V + 1) / 2], int e) { return e % 2 ? x[e / 2].y : x[e / 2].x; }
template <int V> __device__ __forceinline__ void put(float2 (&x)[(V + 1) / 2], int e, float v) { if (e % 2) x[e / 2].y = v; else x[e / 2].x = v; }
template <typename T, int V, bool IL>
__device__ __forceinline__ void unpack_unit(const Raw<T, V>& r, Vec<V>& x) {
  constexpr int P = Vec<V>::P;
#pragma unroll
  for (int k = 0; k < P; ++k) {
    const float2 p = pair_of<T, V>(r.p, k), q = pair_of<T, V>(r.q, k);
    if constexpr (IL && V > 1) {                 // a pair of memory is a first and a second element
      put<V>(x.a, k, p.x); put<V>(x.b, k, p.y);
      put<V>(x.a, P + k, q.x); put<V>(x.b, P + k, q.y);
    } else {
      x.a[k] = p; x.b[k] = q;
    }
  }
}
template <typename T, int V, bool IL>
__device__ __forceinline__ void store_unit(T* row, const Unit<V, IL>& u, const Vec<V>& x) {
  constexpr int P = Vec<V>::P;
  Raw<T, V> r;
#pragma unroll
  for (int k = 0; k < P; ++k) {
    if constexpr (IL && V > 1) {
      set_pair<T, V>(r.p, k, make_float2(get<V>(x.a, k), get<V>(x.b, k)));
      set_pair<T, V>(r.q, k, make_float2(get<V>(x.a, P + k), get<V>(x.b, P + k)));
    } else {
      set_pair<T, V>(r.p, k, x.a[k]); set_pair<T, V>(r.q, k, x.b[k]);
    }
  }
  if (u.has_a) store_words<Raw<T, V>::B>(row + u.a, r.p);
  if (u.has_b) store_words<Raw<T, V>::B>(row + u.b, r.q);
}
// index in a row of D elements of the e-th of the first / second elements
template <int V, bool IL>
__device__ __forceinline__ int element(const Unit<V, IL>& u, int e) {
  if constexpr (IL) { const int i = e < V ? 2 * e : 2 * (e - V) + 1; return u.a + i; }      // the pieces are adjacent
  else return e < V ? u.a + e : u.b + e - V;
}
__device__ __forceinline__ float row_sum(float v, int lpr) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < lpr) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A block takes `hb` heads (blockIdx.y; of the H + Hk of queries and keys) of `tb` tokens at a time and walks the tokens: the threads of a token's
// heads are neighbours, so that a warp reads and writes whole lines, and a thread keeps to its head, whose weights and whose sums of
// the weights' gradients stay in registers.  The angles of a chunk of tokens are formed by all threads together in shared memory.  A step's
// loads leave one step ahead (asynchronous copies three to six steps ahead were no faster: registers and warps bound it, not the way to memory).
// 4 + 4 heads of 32, 147456 tokens, forward and backward: a thread through all heads of its token 48 and 108 us; a thread a head in
// pieces of 8 bytes 50 and 71; pieces of 16 bytes, as many blocks as stay resident 42 and 63, with the same positions in all 384 sequences 39 and 58.
// UPL: units of a thread.  Every thread of a warp takes part in each sum over a row: rows that do not exist are zeros.
constexpr int units_per(int V) { return V >= 4 ? 1 : V == 2 ? 2 : 4; }
// blocks of an SM ([1, 32768, 16 + 4, 128] bf16 in pieces of 16 bytes: forward 2 blocks 113 us, 3 99, 4 110; backward 1 186, 2 133, 3 233.
// [1, 147456, 4 + 4, 32] fp32: forward 3 blocks 68, 4 60; backward 2 91, 3 93).  The registers that this leaves spill a little: 16-byte pieces of 16-bit
// elements 24 bytes of stack forward and 24 to 32 backward, 8-byte ones 40 to 48 backward, fp32 32 forward, single elements 88 to 120 backward.
constexpr int resident(int V, int es, bool bwd) { return units_per(V) > 1 ? 2 : V * es < 16 ? (bwd ? 3 : 4) : bwd ? 2 : es == 4 ? 4 : 3; }
template <typename T, int V, int UPL, bool IL, bool BWD>
__global__ void __launch_bounds__(kThreads, resident(V, sizeof(T), BWD)) qk_rotary_kernel(const __grid_constant__ RotP p) {
  constexpr int P = Vec<V>::P;
  const int lpr = 1 << p.log_lpr, lane = threadIdx.x & (lpr - 1), slot = threadIdx.x >> p.log_lpr;
  const int heads = p.H + p.Hk, tslot = slot / p.hb, g = blockIdx.y * p.hb + slot - tslot * p.hb;
  const bool head_ok = tslot < p.tb && g < heads, is_q = g < p.H;
  const int h = is_q ? g : g - p.H, pairs = p.R / 2;
  const float inv_d = 1.f / p.D;
  extern __shared__ __align__(16) float shared[];
  // [mt][pairs] cosines and sines (two pairs: both cosines, then both sines), then V pairs that turn nothing
  float* const angles = reinterpret_cast<float*>(shared);
  double* const positions = reinterpret_cast<double*>(angles + 2 * (p.mt * pairs + V));
  if (threadIdx.x < 2 * V) angles[2 * p.mt * pairs + threadIdx.x] = V > 1 ? (threadIdx.x & 2 ? 0.f : 1.f) : (threadIdx.x ? 0.f : 1.f);

  Vec<V> wt[UPL], dw[BWD ? UPL : 1] = {};
#pragma unroll
  for (int k = 0; k < UPL; ++k) {
    const Unit<V, IL> u(lane + k * lpr, p.R, p.D);
    const void* w = is_q ? p.qw : p.kw;
    if constexpr (V == 1) wt[k].a[0].y = wt[k].b[0].y = 0.f;
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) {
      const int i = element<V, IL>(u, e);
      const float x = !head_ok || i >= p.D ? 0.f : w ? load_rt(w, h * p.w_head + i, p.w_dtype) : 1.f;
      if (e < V) put<V>(wt[k].a, e, x); else put<V>(wt[k].b, e - V, x);
    }
  }
  const int64_t qs3 = is_q ? p.qs[3] : p.ks[3], sd = is_q ? p.qs[4] : p.ks[4];
  const int64_t sb = is_q ? p.qs[0] : p.ks[0], sn = is_q ? p.qs[1] : p.ks[1], sl = is_q ? p.qs[2] : p.ks[2];
  const T* const in = static_cast<const T*>(is_q ? p.q : p.k) + h * qs3;
  const int own = is_q ? p.H : p.Hk;                           // heads of a token in the contiguous arrays
  const T* const din = BWD ? static_cast<const T*>(is_q ? p.dq_out : p.dk_out) + (int64_t)h * p.D : nullptr;
  T* const out = static_cast<T*>(BWD ? (is_q ? p.dq : p.dk) : (is_q ? p.q_out : p.k_out)) + (int64_t)h * p.D;
  auto unit = [&](int k, bool live) {
    Unit<V, IL> u(lane + k * lpr, p.R, p.D);
    u.has_a = u.has_a && live; u.has_b = u.has_b && live;
    return u;
  };
  const uint32_t tokens = (uint32_t)p.tokens;
  // a thread's place among the tokens: stepped along, and found by divisions only where a sequence ends
  struct Place {
    uint32_t tok, l;
    const T* row;
  };
  auto place = [&](uint32_t tok) {
    Place c;
    const uint32_t t = head_ok && tok < tokens ? tok : 0, bn = t / (uint32_t)p.L, b = bn / (uint32_t)p.N, n = bn - b * p.N;
    c.tok = tok; c.l = t - bn * p.L;
    c.row = in + b * sb + n * sn + c.l * sl;
    return c;
  };
  const int64_t row_step = p.tb * sl, arr_step = (int64_t)p.tb * own * p.D;
  auto fetch = [&](const Place& c, const T* dp, bool live, Raw<T, V> (&x)[UPL], Raw<T, V> (&d)[BWD ? UPL : 1]) {
#pragma unroll
    for (int k = 0; k < UPL; ++k) load_unit<T, V, IL>(c.row, sd, unit(k, live), x[k]);
    if constexpr (BWD) {
#pragma unroll
      for (int k = 0; k < UPL; ++k) load_unit<T, V, IL>(dp, 1, unit(k, live), d[k]);
    }
  };
  // This block's chunks, mt tokens at most each.  Where all sequences have the same positions, a block keeps to one span of them and
  // walks the sequences, with one set of angles; else the chunks are gridDim.x apart.
  const uint32_t span = p.spans ? blockIdx.x % p.spans : 0, leap = p.spans ? gridDim.x / p.spans : gridDim.x, n_rows = p.spans ? tokens / p.L : 0;
  struct Chunk { uint32_t c0, c1; };                           // none left: c0 = c1
  auto chunk = [&](uint32_t x) {
    Chunk c;
    uint32_t end = tokens;
    if (p.spans) {
      if (x >= n_rows) return Chunk{tokens, tokens};
      end = (x + 1) * p.L;
      c.c0 = x * p.L + span * p.mt;
    } else {
      if (x >= (tokens + p.mt - 1) / p.mt) return Chunk{tokens, tokens};
      c.c0 = x * p.mt;
    }
    c.c1 = end - c.c0 < (uint32_t)p.mt ? end : c.c0 + p.mt;
    return c;
  };
  uint32_t at_chunk = p.spans ? blockIdx.x / p.spans : blockIdx.x;
  Chunk rest = chunk(at_chunk);                                // what is left of the chunk
  Place at = place(rest.c0 + tslot);
  bool live = head_ok && at.tok < rest.c1, fresh = true, angles_left = true;
  Raw<T, V> xr[UPL], dr[BWD ? UPL : 1];
  const T* dp = BWD ? din + (int64_t)(live ? at.tok : 0) * own * p.D : nullptr;
  T* to = out + (int64_t)(live ? at.tok : 0) * own * p.D;
  int first_turn[UPL], turn_step[UPL];
#pragma unroll
  for (int k = 0; k < UPL; ++k) {
    const bool turned = unit(k, true).turned;
    first_turn[k] = 2 * (turned ? tslot * pairs + (lane + k * lpr) * V : p.mt * pairs);
    turn_step[k] = turned ? 2 * p.tb * pairs : 0;
  }
  fetch(at, dp, live, xr, dr);                                 // on its way while the angles are formed
  const float* turns[UPL];
  while (rest.c0 < rest.c1) {
    if (fresh && angles_left) {
      for (uint32_t i = threadIdx.x; i < rest.c1 - rest.c0; i += kThreads) {
        const uint32_t t = rest.c0 + i, bn = t / (uint32_t)p.L, l = t - bn * p.L, b = bn / (uint32_t)p.N, n = bn - b * p.N;
        double pos = (double)l;
        if (p.pos) {
          const int64_t x = b * p.ps[0] + n * p.ps[1] + l * p.ps[2];
          pos = p.pos64 ? (double)static_cast<const int64_t*>(p.pos)[x] : (double)static_cast<const int32_t*>(p.pos)[x];
        }
        positions[i] = pos;
      }
      __syncthreads();                                         // besides: the last chunk's angles have been read
      for (uint32_t x = threadIdx.x; x < (rest.c1 - rest.c0) * pairs; x += kThreads) {
        const uint32_t i = x * p.pair_magic >> 20, f = x - i * pairs;          // x / pairs, for the few thousand angles of a chunk
        float* const at_turn = angles + (V > 1 ? 4 * (x >> 1) + (x & 1) : 2 * x);
        turn_of(positions[i], p.inv_freq[f], at_turn[V > 1 ? 2 : 1], at_turn[0]);
      }
      __syncthreads();
      angles_left = !p.spans;
    }
    if (fresh) {
#pragma unroll
      for (int k = 0; k < UPL; ++k) turns[k] = angles + (live ? first_turn[k] : 2 * p.mt * pairs);      // a dead thread's row is zeros and turns nothing
    }
    // every thread takes every step: the sums over rows take whole warps
    Vec<V> x[UPL], d[BWD ? UPL : 1];
    float2 ss2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
      unpack_unit<T, V, IL>(xr[k], x[k]);
      if constexpr (BWD) unpack_unit<T, V, IL>(dr[k], d[k]);
#pragma unroll
      for (int e = 0; e < P; ++e) ss2 = fma2(x[k].b[e], x[k].b[e], fma2(x[k].a[e], x[k].a[e], ss2));
    }
    const bool now = live;
    T* const row_out = to;
    rest.c0 += p.tb;
    fresh = rest.c0 >= rest.c1;
    if (!fresh) {
      at.tok += p.tb; at.l += p.tb; at.row += row_step;
      live = head_ok && at.tok < rest.c1;
      if (BWD) dp += arr_step;
      to += arr_step;
      if (live && at.l >= (uint32_t)p.L) at = place(at.tok);
    } else {                                                 // to the next chunk
      at_chunk += leap;
      rest = chunk(at_chunk);
      at = place(rest.c0 + tslot);
      live = head_ok && at.tok < rest.c1;
      const int64_t arr = (int64_t)(live ? at.tok : 0) * own * p.D;
      if (BWD) dp = din + arr;
      to = out + arr;
    }
    fetch(at, dp, live, xr, dr);
    const float ss = row_sum(ss2.x + ss2.y, lpr);              // of every lane, whether its row exists or not
    float rstd = rsqrtf(fmaf(ss, inv_d, p.eps));
    if (BWD && !now) rstd = 0.f;                               // adds nothing to the weights' gradients, also without an eps: 0 * inf would
    const float2 rstd2 = make_float2(rstd, rstd);
    float2 dot2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
      const Unit<V, IL> u = unit(k, now);
      Vec<V> turn;                                           // a: cosines, b: sines; 1 and 0 where nothing turns
      if constexpr (V == 1) {
        const float2 t = *reinterpret_cast<const float2*>(turns[k]);
        turn.a[0] = make_float2(t.x, 0.f); turn.b[0] = make_float2(t.y, 0.f);
      } else {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const float4 t = reinterpret_cast<const float4*>(turns[k])[e];
          turn.a[e] = make_float2(t.x, t.y); turn.b[e] = make_float2(t.z, t.w);
        }
      }
      if constexpr (!BWD) {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const float2 ya = mul2(mul2(x[k].a[e], rstd2), wt[k].a[e]), yb = mul2(mul2(x[k].b[e], rstd2), wt[k].b[e]), c = turn.a[e], s = turn.b[e];
          x[k].a[e] = sub2(mul2(ya, c), mul2(yb, s));
          x[k].b[e] = fma2(ya, s, mul2(yb, c));
        }
        store_unit<T, V, IL>(row_out, u, x[k]);
      } else {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const float2 c = turn.a[e], s = turn.b[e], da = d[k].a[e], db = d[k].b[e];
          const float2 ga = fma2(db, s, mul2(da, c)), gb = sub2(mul2(db, c), mul2(da, s));
          x[k].a[e] = mul2(x[k].a[e], rstd2); x[k].b[e] = mul2(x[k].b[e], rstd2);        // hat
          const float2 ta = mul2(ga, x[k].a[e]), tb = mul2(gb, x[k].b[e]);
          dw[k].a[e] = add2(dw[k].a[e], ta); dw[k].b[e] = add2(dw[k].b[e], tb);
          dot2 = fma2(tb, wt[k].b[e], fma2(ta, wt[k].a[e], dot2));
          d[k].a[e] = mul2(ga, wt[k].a[e]); d[k].b[e] = mul2(gb, wt[k].b[e]);
        }
      }
    }
    if constexpr (BWD) {
      const float dot = row_sum(dot2.x + dot2.y, lpr) * -inv_d;
      const float2 minus = make_float2(dot, dot);
#pragma unroll
      for (int k = 0; k < UPL; ++k) {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          x[k].a[e] = mul2(rstd2, fma2(x[k].a[e], minus, d[k].a[e]));
          x[k].b[e] = mul2(rstd2, fma2(x[k].b[e], minus, d[k].b[e]));
        }
        store_unit<T, V, IL>(row_out, unit(k, now), x[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < UPL; ++k)
      if (live) turns[k] += turn_step[k];
  }
  if constexpr (BWD) {
    if (!p.parts) return;
    float* const sum = shared;                                 // [token][head of the block][D]
    __syncthreads();
    if (head_ok) {
#pragma unroll
      for (int k = 0; k < UPL; ++k) {
        const Unit<V, IL> u(lane + k * lpr, p.R, p.D);
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) {
          const int i = element<V, IL>(u, e);
          if (i < p.D && (u.turned || i >= p.R)) sum[slot * p.D + i] = e < V ? get<V>(dw[k].a, e) : get<V>(dw[k].b, e - V);
        }
      }
    }
    __syncthreads();
    const int here = heads - (int)blockIdx.y * p.hb < p.hb ? heads - (int)blockIdx.y * p.hb : p.hb, q_here = p.H - (int)blockIdx.y * p.hb;
    if (p.w_head) {                                            // a row a head: parts [gridDim.x][heads][D]
      for (int x = threadIdx.x; x < here * p.D; x += kThreads) {
        float s = 0.f;
        for (int t = 0; t < p.tb; ++t) s += sum[t * p.hb * p.D + x];
        p.parts[((int64_t)blockIdx.x * heads + blockIdx.y * p.hb) * p.D + x] = s;
      }
    } else {                                                   // queries and keys: parts [gridDim.y][gridDim.x][2][D]
      for (int x = threadIdx.x; x < 2 * p.D; x += kThreads) {
        const int which = x / p.D, i = x - which * p.D;
        float s = 0.f;
        for (int t = 0; t < p.tb; ++t)
          for (int y = 0; y < here; ++y)
            if ((y >= q_here) == which) s += sum[(t * p.hb + y) * p.D + i];
        p.parts[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * p.D + x] = s;
      }
    }
  }
}

// Weight gradients: blockIdx = (32 elements, row of [H or 1 + Hk or 1]); a row is the sum of `n` parts, `step` floats apart from `first`, 32
// of them at a time.
__global__ void __launch_bounds__(1024) qk_rotary_join_kernel(const float* __restrict__ parts, int n, int step, int D, int q_rows, void* __restrict__ dqw, void* __restrict__ dkw,
                                                              int w_dtype) {
  __shared__ float sums[32][33];
  const int row = blockIdx.y, i = blockIdx.x * 32 + (threadIdx.x & 31), warp = threadIdx.x >> 5;
  float s = 0.f;
  if (i < D) {
#pragma unroll 8
    for (int k = warp; k < n; k += 32) s += parts[(int64_t)k * step + row * D + i];
  }
  sums[warp][threadIdx.x & 31] = s;
  __syncthreads();
  if (warp || i >= D) return;
  s = 0.f;
  for (int k = 0; k < 32; ++k) s += sums[k][threadIdx.x];
  if (row >= q_rows) store_rt(dkw, (int64_t)(row - q_rows) * D + i, w_dtype, s);
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

// Elements of a piece: the widest load that sizes, strides and addresses allow, 16 bytes at most, and 8 where 16 would leave processors
// without a block (32 tokens of 32 + 8 heads of 128: 4.0 us instead of 4.9; 32768 tokens of 16 + 4 heads 117 forward, 187 backward instead of 99 and 133).
int piece_limit(const mf_qk_rotary_args& a) {
  const int v = 16 / (int)dtype_size(a.dtype);
  const int64_t elements = (int64_t)a.B * a.N * a.L * (a.H + a.Hk) * a.D;
  return elements / (2 * v) < (int64_t)kThreads * tcx::sm_count() ? v / 2 : v;
}
int piece(const mf_qk_rotary_args& a, bool bwd) {
  const int es = (int)dtype_size(a.dtype);
  for (int v = piece_limit(a); v > 1; v /= 2) {
    bool ok = a.R / 2 % v == 0 && (a.D - a.R) % v == 0 && a.q_strides[4] == 1 && a.k_strides[4] == 1;
    for (int i = 0; i < 4; ++i) ok = ok && a.q_strides[i] % v == 0 && a.k_strides[i] % v == 0;
    const uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.k | (bwd ? (uintptr_t)a.dq_out | (uintptr_t)a.dk_out | (uintptr_t)a.dq | (uintptr_t)a.dk
                                                                : (uintptr_t)a.q_out | (uintptr_t)a.k_out);
    if (ok && at % (v * es) == 0) return v;
  }
  return 1;
}

struct Plan { int log_lpr, hb, tb, mt, spans, gx, gy; size_t smem; };
Plan plan(const mf_qk_rotary_args& a, int V, bool bwd) {
  Plan c;
  const int units = a.R / 2 / V + (a.D - a.R + 2 * V - 1) / (2 * V), lanes = (units + units_per(V) - 1) / units_per(V), heads = a.H + a.Hk;
  c.log_lpr = 0;
  while ((1 << c.log_lpr) < lanes) ++c.log_lpr;
  const int slots = kThreads >> c.log_lpr, pairs = a.R / 2;
  // as few groups of heads as leave few threads without a row (20 heads, 32 rows a block: two groups, three tokens at a time)
  int used = 0;
  for (int least = (heads + slots - 1) / slots, gy = least; gy <= 4 * least && gy <= heads; ++gy) {
    const int hb = (heads + gy - 1) / gy, tb = slots / hb, of_all = (int)((int64_t)1000 * heads * tb / ((int64_t)(heads + hb - 1) / hb * slots));
    if (of_all > used + used / 10) { used = of_all; c.hb = hb; c.tb = tb; }
  }
  c.gy = (heads + c.hb - 1) / c.hb;
  while (c.tb > 1 && c.tb * pairs * 8 > 32 * 1024) c.tb /= 2;
  // Steps of a chunk, 16 KB of angles and positions at most: those that take the blocks of one wave the least time.  Where all sequences have the same positions (and
  // are no shorter than eight ninths of their steps), a block forms the angles of one chunk of them once; else it waits for new ones at each chunk.
  const int64_t tokens = (int64_t)a.B * a.N * a.L, rows = (int64_t)a.B * a.N;
  int64_t places = (int64_t)resident(V, (int)dtype_size(a.dtype), bwd) * tcx::sm_count() / c.gy, best = 0;
  if (places < 1) places = 1;
  const int64_t steps = (a.L + c.tb - 1) / c.tb;
  const bool same = rows > 1 && steps * c.tb * 8 <= (int64_t)9 * a.L &&
                    (!a.positions || ((a.B == 1 || a.pos_strides[0] == 0) && (a.N == 1 || a.pos_strides[1] == 0)));
  for (int n = 1; n <= 64 && (n == 1 || n * c.tb * (pairs + 1) * 8 <= 16 * 1024); ++n) {
    const int mt = c.tb * n;
    int64_t time, spans = same ? (steps + n - 1) / n : 0, gx;
    if (spans > places) spans = 0;
    if (spans) {
      const int64_t leap = places / spans < rows ? places / spans : rows;
      gx = spans * leap;
      time = ((rows + leap - 1) / leap + 1) * n;
    } else {
      const int64_t chunks = (tokens + mt - 1) / mt;
      gx = chunks < places ? chunks : places;
      time = (chunks + gx - 1) / gx * (n + 1);
    }
    if (n == 1 || time < best) { best = time; c.mt = mt; c.spans = (int)spans; c.gx = (int)gx; }
  }
  c.smem = sizeof(float2) * ((size_t)c.mt * pairs + V) + sizeof(double) * c.mt;
  const size_t sums = bwd && a.dq_weight ? sizeof(float) * (size_t)c.tb * c.hb * a.D : 0;
  if (sums > c.smem) c.smem = sums;
  return c;
}
size_t part_floats(const mf_qk_rotary_args& a, const Plan& c) { return (size_t)c.gx * a.D * (a.per_head ? a.H + a.Hk : 2 * c.gy); }

template <typename T, int V, bool BWD>
int run(const mf_qk_rotary_args& a, cudaStream_t st) {
  constexpr int UPL = units_per(V);
  RotP p = rot_params(a);
  const Plan c = plan(a, V, BWD);
  p.log_lpr = c.log_lpr; p.hb = c.hb; p.tb = c.tb; p.mt = c.mt; p.spans = c.spans;
  p.pair_magic = a.R > 1 ? ((1u << 20) + a.R / 2 - 1) / (a.R / 2) : 1u << 20;
  const bool sums = BWD && a.dq_weight;
  if (sums) p.parts = static_cast<float*>(a.workspace);
  const auto go = [&](auto il) -> int {
    constexpr auto kern = qk_rotary_kernel<T, V, UPL, decltype(il)::value, BWD>;
    if (int e = opt_in_smem<kern>(c.smem)) return e;
    kern<<<dim3(c.gx, c.gy), kThreads, c.smem, st>>>(p);
    MF_LAUNCHED("qk_rotary_kernel");
    return MF_OK;
  };
  if (int e = a.interleaved ? go(std::true_type{}) : go(std::false_type{})) return e;
  if (sums) {
    const int rows = a.per_head ? a.H + a.Hk : 2;
    qk_rotary_join_kernel<<<dim3((a.D + 31) / 32, rows), 1024, 0, st>>>(p.parts, a.per_head ? c.gx : c.gx * c.gy, rows * a.D, a.D, a.per_head ? a.H : 1, a.dq_weight, a.dk_weight,
                                                                      a.w_dtype);
    MF_LAUNCHED("qk_rotary_join_kernel");
  }
  return MF_OK;
}
template <typename T, bool BWD>
int dispatch(const mf_qk_rotary_args& a, cudaStream_t st) {
  const int v = piece(a, BWD);
  if constexpr (sizeof(T) == 2) if (v == 8) return run<T, 8, BWD>(a, st);
  if (v == 4) return run<T, 4, BWD>(a, st);
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
  for (int v = 1; v <= piece_limit(a); v *= 2) {       // whichever width the alignment allows
    if (a.R / 2 % v || (a.D - a.R) % v) break;
    const size_t n = sizeof(float) * part_floats(a, plan(a, v, true));
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
