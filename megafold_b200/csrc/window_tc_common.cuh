// What the tensor-core kernels of the sliding-window attention share: operand tiles, masks of visible keys, tensor maps.
//
// Operand tiles hold 16-bit rows of DP elements (32, 64 or 128; smaller heads are filled up with zeros by TMA) as panels of
// up to 64 columns: 64-byte rows with 64B swizzle for DP = 32, 128-byte rows with 128B swizzle otherwise, two panels for DP = 128.
#pragma once

#include "evo_tc_common.cuh"
#include "window_common.cuh"

namespace mf {
namespace win {
using namespace tcx;

template <int DP> struct Geo {
  static constexpr int ROWB = DP == 32 ? 64 : 128;            // bytes of a row of a panel
  static constexpr int COLS = ROWB / 2, PANELS = DP / COLS;
  static constexpr Swizzle SW = DP == 32 ? kSw64 : kSw128;
  static constexpr uint32_t HI = desc_hi(8 * ROWB, SW);
  static constexpr int TILE(int rows) { return rows * DP * 2; }
};
// descriptor offset (in 16-byte units) of the 16 columns [16 ks, 16 ks + 16) of a K-major tile of `rows` rows
template <int DP>
__device__ __forceinline__ constexpr uint32_t k_step(int ks, int rows) {
  using G = Geo<DP>;
  return (uint32_t)(ks / (G::COLS / 16) * (rows * G::ROWB / 16) + ks % (G::COLS / 16) * 2);
}

// Maps of a [B, N, L, H, D] operand; a batch or sequence stride of 0 (a broadcast view) becomes an extent of 1 that every
// coordinate is 0 in.  A copy fetches `rows` tokens of `heads` heads: the tile's rows are the heads of one token after the other.
struct Coords { int n_mul, b_mul; };
inline int operand_map(CUtensorMap* m, Coords* c, const void* ptr, int dtype, int B, int N, int L, int H, int D, const int64_t* s, int cols, int heads, int rows) {
  c->n_mul = s[1] == 0 ? 0 : 1; c->b_mul = s[0] == 0 ? 0 : 1;
  const int64_t dims[5] = {D, H, L, c->n_mul ? N : 1, c->b_mul ? B : 1};
  const int64_t str[5] = {1, s[3], s[2], s[1], s[0]};
  const int box[5] = {cols, heads, rows, 1, 1};
  return make_tiled_map(m, ptr, dtype, 5, dims, str, box, cols * 2);
}
inline bool operand_ok(const void* p, const int64_t* s, int B, int N, int L, int H) {
  if ((reinterpret_cast<uintptr_t>(p) & 15) != 0 || s[4] != 1) return false;
  const int64_t sizes[4] = {B, N, L, H};
  for (int i = 0; i < 4; ++i)
    if (sizes[i] > 1 && (s[i] % 8 != 0 || s[i] < 0 || (i >= 2 && s[i] == 0) || s[i] >= (int64_t)1 << 38)) return false;
  return true;
}
// One tile from token l0 and head h: a copy a panel, panels `rows` rows apart.
template <int DP>
__device__ __forceinline__ void load_tile_tma(uint8_t* dst, const CUtensorMap* m, uint64_t* bar, int rows, int h, int l0, int n, int b) {
  using G = Geo<DP>;
#pragma unroll
  for (int pn = 0; pn < G::PANELS; ++pn) tma_load_5d(dst + pn * rows * G::ROWB, m, bar, pn * G::COLS, h, l0, n, b);
}

__device__ __forceinline__ uint32_t ones32(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// Bits of the 32 keys from j0 that a query at position `at` sees
__device__ __forceinline__ uint32_t seen32(const WinP& p, int at, int j0) {
  int hi = at + p.right + 1 - j0;
  if (hi > p.Lk - j0) hi = p.Lk - j0;
  return ones32(hi) & (~ones32(at - p.left - j0) | ones32(p.sinks - j0));
}
// Bits of the 32 keys from j0 that are in a range
__device__ __forceinline__ uint32_t range32(const KeyRange& r, int j0) { return ones32(r.hi - j0) & (~ones32(r.lo - j0) | ones32(r.front - j0)); }
// Does every query of positions [at0, at1] see every key of [j0, j1)?  (the mask aside)
__device__ __forceinline__ bool all_seen(const WinP& p, int at0, int at1, int j0, int j1) {
  return j1 <= p.Lk && j1 - 1 <= at0 + p.right && (j0 >= at1 - p.left || j1 <= p.sinks);
}

// store_rows for rows at addresses of their own: 32 fp32 columns of a TMEM accumulator, scaled; `row` is where the first of them goes of
// this lane's row (NULL: nowhere), of which `left` (a multiple of 8) are there.
template <typename T>
__device__ __forceinline__ void store_rows_at(uint32_t tacc, float sc, T* row, int left) {
  uint32_t w[4][4];                            // [piece of eight columns][word]
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    uint32_t o16[16];
    tmem_ld16(tacc + hf * 16, o16);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 8; ++e) w[hf * 2 + e / 4][e % 4] = Pack2<T>::pack(__uint_as_float(o16[2 * e]) * sc, __uint_as_float(o16[2 * e + 1]) * sc);
  }
  const int q = threadIdx.x & 3;
#pragma unroll
  for (int s2 = 2; s2 > 0; s2 >>= 1) {         // 4 x 4 transposition over lanes q
    const bool up = q & s2;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (c & s2) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? w[c][e] : w[c + s2][e], s2);
        if (up) w[c][e] = got; else w[c + s2][e] = got;
      }
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {                // w[c]: piece q of the row of lane c of these four
    T* to = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), (threadIdx.x & 28) + c));
    if (to && q * 8 < left) *reinterpret_cast<uint4*>(to + q * 8) = make_uint4(w[c][0], w[c][1], w[c][2], w[c][3]);
  }
}

bool window_tc_supported(const mf_window_args& a);

}  // namespace win
}  // namespace mf
