// Tiles of the attention kernels on CUDA cores: 64 rows x 64 columns of the logits for 256 threads; thread (ty, tx) owns the rows
// ty + 16 a and the columns tx + 16 b (a, b = 0..3).  Operands are fp32 rows of pitch DP + 4 floats in shared memory, so that the
// 16-byte reads of neighbouring rows touch different banks.
#pragma once

#include "common.cuh"

namespace mf {
namespace simt {

constexpr int kThreads = 256;
constexpr int kTile = 64;
constexpr int kPPitch = kTile + 4;

// Rows [row0, row0 + 64) x [0, DP) of a [.., L, H, D] operand as fp32, zero outside L and D.
template <typename T, int DP>
__device__ __forceinline__ void load_tile(float* dst, const void* src, const int64_t* s, bool vec, int b, int n, int h, int row0, int L, int D) {
  constexpr int pitch = DP + 4;
  const T* base = static_cast<const T*>(src) + b * s[0] + n * s[1] + h * s[3];
#pragma unroll
  for (int it = 0; it < kTile * DP / 4 / kThreads; ++it) {
    const int idx = it * kThreads + threadIdx.x;
    const int r = idx / (DP / 4), d = (idx - r * (DP / 4)) * 4;
    const int l = row0 + r;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (l < L && d < D) {
      const T* p = base + l * s[2];
      if (vec) {
        __align__(16) T e[4];
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(e) = __ldg(reinterpret_cast<const uint4*>(p + d));
        else *reinterpret_cast<uint2*>(e) = __ldg(reinterpret_cast<const uint2*>(p + d));
        v = make_float4(to_f(e[0]), to_f(e[1]), to_f(e[2]), to_f(e[3]));
      } else {
        v.x = to_f(p[d * s[4]]);
        if (d + 1 < D) v.y = to_f(p[(d + 1) * s[4]]);
        if (d + 2 < D) v.z = to_f(p[(d + 2) * s[4]]);
        if (d + 3 < D) v.w = to_f(p[(d + 3) * s[4]]);
      }
    }
    *reinterpret_cast<float4*>(dst + r * pitch + d) = v;
  }
}

// acc[a][b] += sum_d A[ty + 16 a][d] B[tx + 16 b][d]
template <int DP>
__device__ __forceinline__ void dot_tile(const float* A, const float* B, int ty, int tx, float (&acc)[4][4]) {
  constexpr int pitch = DP + 4;
#pragma unroll 2
  for (int d = 0; d < DP; d += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) x[a] = *reinterpret_cast<const float4*>(A + (ty + 16 * a) * pitch + d);
#pragma unroll
    for (int b = 0; b < 4; ++b) y[b] = *reinterpret_cast<const float4*>(B + (tx + 16 * b) * pitch + d);
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        acc[a][b] = fmaf(x[a].x, y[b].x, acc[a][b]);
        acc[a][b] = fmaf(x[a].y, y[b].y, acc[a][b]);
        acc[a][b] = fmaf(x[a].z, y[b].z, acc[a][b]);
        acc[a][b] = fmaf(x[a].w, y[b].w, acc[a][b]);
      }
  }
}

// The DP / 16 head columns of a thread: adjacent ones, or (SPREAD) fours of them, 64 apart, so that eight threads read 128 adjacent bytes
template <int DP> __device__ __forceinline__ int column(int tx, int e) { return DP <= 64 ? tx * (DP / 16) + e : e / 4 * 64 + tx * 4 + e % 4; }

// acc[a][e] += sum_c P[ty + 16 a][c] V[c][d], d = tx * DP / 16 + e or (SPREAD) column(tx, e)
template <int DP, bool SPREAD = false>
__device__ __forceinline__ void sum_tile(const float* P, const float* V, int ty, int tx, float (&acc)[4][DP / 16]) {
  constexpr int pitch = DP + 4, E = DP / 16;
#pragma unroll 4
  for (int c = 0; c < kTile; c += 4) {
    float4 pr[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) pr[a] = *reinterpret_cast<const float4*>(P + (ty + 16 * a) * kPPitch + c);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float v[E];
      const float* row = V + (c + k) * pitch + (SPREAD && E > 4 ? tx * 4 : tx * E);
      if constexpr (E == 2) { const float2 t = *reinterpret_cast<const float2*>(row); v[0] = t.x; v[1] = t.y; }
      else {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
          const float4 t = *reinterpret_cast<const float4*>(row + (SPREAD ? e * 16 : e));
          v[e] = t.x; v[e + 1] = t.y; v[e + 2] = t.z; v[e + 3] = t.w;
        }
      }
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const float w = k == 0 ? pr[a].x : k == 1 ? pr[a].y : k == 2 ? pr[a].z : pr[a].w;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[a][e] = fmaf(w, v[e], acc[a][e]);
      }
    }
  }
}

// reductions over the 16 threads that share a row
__device__ __forceinline__ float row_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace simt
}  // namespace mf
