// Sliding-window attention with sinks, backward, on the tensor cores (tcgen05 + TMEM + TMA): 16-bit tensors, head sizes that are
// multiples of 8 up to 128.  Three kernels, each result a sum in a fixed order:
//
// window_terms_kernel   delta_i = sum_d dO_i O_i, and per block of 64 rows of queries a [64 x 16] bf16 tile of the terms -lse_i sqrt(D)
//                       and -delta_i, each as three bf16 that sum to it (evo_tc_common.cuh, "rank-one terms").
//
// window_dkv_tc_kernel  a CTA keeps 128 keys of one key head and walks its list of blocks of 64 rows of queries (or a chunk of
//                       it: window_common.cuh), keys on the TMEM lanes:
//                         S^T = K Q^T - 1 (lse sqrt(D))^T     dP^T = V dO^T - 1 delta^T      the subtrahends by one K = 16 product each
//                         P^T = 2^(c1 S^T)                    dS^T = P^T dP^T                written over S^T and dP^T as 16 bits, read from TMEM by
//                         dV += P^T dO                        dK += dS^T Q                   (B operands MN-major, as the tiles are)
//
// window_dq_tc_kernel   a CTA keeps 128 rows of queries and walks the blocks of 64 keys that they see, queries on the lanes:
//                         S = Q K^T   dP = dO V^T   dS = P (dP - delta)   dQ += dS K
//                       (a narrow window: a walk that sums P dP to delta before that one, instead of the sum of dO O)
//
// Scores are formed twice (7 products instead of 5): a single pass would add dQ or dK and dV atomically, in an order that changes, and
// a window leaves few tiles to carry an accumulator over.  In both walking kernels eight compute warps take a block, two to a
// set of lanes with 32 columns each; one warp copies, one issues products.  TMEM lets two CTAs share an SM and fill each other's
// waits (dK and dV at DP = 128: one CTA, two score buffers).  In the dQ kernel S and dP have barriers of their own besides, so that
// the next S is formed while the compute warps exponentiate (184 -> 168 us at 16384 tokens, 16 heads of 64, window 1024);
// in the other one, where each barrier stands between two products, that cost more than it gave (199 -> 233).
//
// Two CTAs an SM leave a thread 96 registers: dK and dV at DP = 64 spill 12 bytes of stores, dQ at DP = 128 spills 8 (bf16) or 16.
//
// Rows of masked keys: their lanes give zeros (dK, dV); as B operand of dQ they, and those that no query of the tile sees, are overwritten
// with zeros in shared memory.
// P and dS are rounded to the operands' type, the matrix instruction's; all sums are fp32.  Waits are bounded as in the forward.
//
// fp16 has five bits of exponent: with the gradients of a scaled loss dS overflowed up to sqrt(D) before dQ and dK did, and at small gradients and wide windows it
// lost bits below 2^-14.  There dS is rounded with a power of two that the accumulator's write-out takes back, so that nothing else changes: in dQ one
// a row, from the row's largest |dO|; in dK and dV's kernel one a CTA, from the largest |dS| of the rows that it walks, which the dQ kernel leaves in
// `tops` (it runs before).  [1, 1, 3000, 2, 128] fp16, window 2048, error of dQ's norm at gradients of 1e-4 8.5e-3 -> 2.5e-3 (that of rounding the result), of 1e-3
// 8.9e-4 -> 4e-4, of 1 3.1e-4 as before; [1, 1, 8192, 16 on 4 heads, 128], window 1024, forward and backward 551 -> 557 us.  Giving dS its factor D^-1/2 before it
// is rounded, instead, left the small gradients ten times as far off.
#include <type_traits>

#include "window_tc_common.cuh"

namespace mf {
namespace win {
namespace {

constexpr int kThreads = 320, kCompute = 256;
constexpr int kKeys = 128;          // dK/dV kernel: keys of a CTA
constexpr int kQB = 64;             // ... and rows of queries of a block
constexpr int kRows = 128;          // dQ kernel: rows of queries of a CTA
constexpr int kKB = 64;             // ... and keys of a block
constexpr int kXB = kQB * 32;       // bytes of a block's term tile

template <typename T> constexpr bool kNarrow = std::is_same<T, __half>::value;          // dS needs a power of two
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ float back(float up) { return __int_as_float((254 << 23) - __float_as_int(up)); }      // 1 / up, a power of two

struct BwdP {
  WinP w;
  KeyPlan plan;
  Coords cq, ck, cv;
  int n_blocks;             // blocks of kQB rows of queries of a pack of heads
  int n_qt, groups;         // dQ: tiles of queries; packs of heads in all sequences
  int q_bytes, qt_bytes;    // bytes of the rows of a block / a tile of queries (copies leave the rest of it alone)
  float c1;
  uint32_t fmt;
  int two_walks;            // dQ: a walk for delta first
  float* delta;             // ... which it writes here
  const uint8_t* terms;     // [packs of heads][n_blocks][kXB]
  int* tops;                // fp16: the largest |dS| of each CTA of the dQ kernel, as bits of a float
  float* parts;
  int* status;
};

// ---------------------------------------------------------------------------------------------------------------- terms
// blockIdx = (block of rows, pack of heads, b * N + n); four threads a row.  GIVEN: delta has been written by the dQ kernel.
template <typename T, bool GIVEN>
__global__ void __launch_bounds__(256) window_terms_kernel(const __grid_constant__ WinP p, float* __restrict__ delta, uint8_t* __restrict__ terms, float sqrt_d) {
  const int r = threadIdx.x >> 2, q = threadIdx.x & 3;
  const int l = r / p.pack, nq = queries_of<kQB>(p), i = blockIdx.x * nq + l, h = blockIdx.y * p.pack + r - l * p.pack;
  const bool live = l < nq && i < p.Lq;
  const int64_t bn = blockIdx.z, row = (bn * p.Lq + i) * p.H + h;
  float s = 0.f;
  if (!GIVEN && live) {
    const T *po = static_cast<const T*>(p.o) + row * p.D, *pg = static_cast<const T*>(p.d_o) + row * p.D;
    for (int d = q * 8; d < p.D; d += 32) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(po + d)), g = __ldg(reinterpret_cast<const uint4*>(pg + d));
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x = Pack2<T>::unpack(aw[e]), y = Pack2<T>::unpack(gw[e]);
        s = fmaf(x.x, y.x, fmaf(x.y, y.y, s));
      }
    }
  }
  s += __shfl_xor_sync(0xffffffffu, s, 1);
  s += __shfl_xor_sync(0xffffffffu, s, 2);
  if (q) return;
  float lse = -INFINITY;
  if (live) {
    const int64_t at = (bn * p.H + h) * p.Lq + i;
    lse = p.lse[at];
    if (GIVEN) s = delta[at]; else delta[at] = s;
  }
  // a row that sees nothing, or is none, gets probability 0 from a finite term
  __nv_bfloat16 a[3], d[3];
  split3(lse == -INFINITY ? kMinusBig : -lse * sqrt_d, a);
  split3(live ? -s : 0.f, d);
  const __nv_bfloat16 z = __float2bfloat16_rn(0.f);
  uint8_t* tile = terms + ((bn * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * kXB;
  *reinterpret_cast<uint4*>(tile + swz_offset(r, 0, 32)) = make_uint4(0u, pack_bf(z, a[0]), pack_bf(a[1], a[2]), pack_bf(d[0], d[1]));
  *reinterpret_cast<uint4*>(tile + swz_offset(r, 1, 32)) = make_uint4(pack_bf(d[2], z), 0u, 0u, 0u);
}

__device__ __forceinline__ void bulk_load_1d(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// ------------------------------------------------------------------------------------------------------------- dK and dV
template <int DP> struct KvCfg {
  static constexpr int NB = DP == 128 ? 2 : 1;                  // score buffers (S^T and dP^T, 64 columns each)
  static constexpr int NS = DP == 128 ? 3 : 2;                  // stages of Q, dO and terms
  static constexpr int CTAS = DP == 128 ? 1 : 2;
  static constexpr uint32_t COLS = DP == 128 ? 512 : 256;
  static constexpr int KB = Geo<DP>::TILE(kKeys), QB = Geo<DP>::TILE(kQB);
  static constexpr size_t SMEM = 1024 + 2 * KB + NS * (2 * QB + kXB) + 2 * kKeys * 32;
};
template <int NS, int NB> struct KvBars {
  uint64_t kv_full, qd_full[NS], qd_empty[NS], sd_ready[NB], pd_ready[NB], done;
};

template <int DP, typename T>
__global__ void __launch_bounds__(kThreads, KvCfg<DP>::CTAS)
window_dkv_tc_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mq,
                     const __grid_constant__ CUtensorMap mg, const __grid_constant__ BwdP f) {
  using C = KvCfg<DP>;
  using G = Geo<DP>;
  constexpr int NS = C::NS, NB = C::NB;
  const WinP& p = f.w;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *sK = smem, *sV = sK + C::KB, *sQ = sV + C::KB, *sG = sQ + NS * C::QB, *sX = sG + NS * C::QB;
  uint8_t *sOneS = sX + NS * kXB, *sOneD = sOneS + kKeys * 32;        // ones in the columns of the lse / delta terms
  __shared__ KvBars<NS, NB> bar;
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;

  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  // blockIdx.x walks the heads fastest: all the heads' longest items (tiles with sinks) start first
  const int heads = p.B * p.N * p.Hk;
  const int x = blockIdx.x / heads, head = blockIdx.x - x * heads, bn = head / p.Hk, hk = head - bn * p.Hk, n = bn % p.N, b = bn / p.N;
  int tile, part;
  plan_item(f.plan, x, tile, part);
  const int j0 = tile * kKeys, len = list_length<kKeys, kQB>(p, tile), e0 = part * f.plan.chunk;
  if (part > 0 && e0 >= len) return;
  const int T_ = len - e0 < f.plan.chunk ? len - e0 : f.plan.chunk;
  int lo, hi;
  query_range(p, j0, j0 + kKeys < p.Lk ? j0 + kKeys : p.Lk, lo, hi);
  const int nq = queries_of<kQB>(p), first = lo / nq, per_pack = hi > lo ? (hi + nq - 1) / nq - first : 1;

  if (tid == 0) {
    abort_s = 0;
    mbar_init(&bar.kv_full, 1);
    for (int i = 0; i < NS; ++i) { mbar_init(&bar.qd_full[i], 1); mbar_init(&bar.qd_empty[i], 1); }
    for (int i = 0; i < NB; ++i) { mbar_init(&bar.sd_ready[i], 1); mbar_init(&bar.pd_ready[i], kCompute); }
    mbar_init(&bar.done, 1);
    mbar_fence_init();
    prefetch_tmap(&mk); prefetch_tmap(&mv); prefetch_tmap(&mq); prefetch_tmap(&mg);
  }
  if (warp == 0) { tmem_alloc(&tmem_base_s, C::COLS); tmem_relinquish(); }
  if (tid < kKeys) {
    const uint32_t one = 0x3f80u;      // bf16 1.0
    *reinterpret_cast<uint4*>(sOneS + swz_offset(tid, 0, 32)) = make_uint4(0u, one << 16, one | (one << 16), 0u);
    *reinterpret_cast<uint4*>(sOneS + swz_offset(tid, 1, 32)) = make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4*>(sOneD + swz_offset(tid, 0, 32)) = make_uint4(0u, 0u, 0u, one | (one << 16));
    *reinterpret_cast<uint4*>(sOneD + swz_offset(tid, 1, 32)) = make_uint4(one, 0u, 0u, 0u);
  }
  // rows that no copy fills (64 is no multiple of the pack) have to be numbers: their probability is 0
  const int filled = nq * p.pack;
  for (int e = tid; e < (kQB - filled) * NS * 2 * G::PANELS * (G::ROWB / 16); e += kThreads) {
    const int piece = e % (G::ROWB / 16), row = filled + e / (G::ROWB / 16) % (kQB - filled), tl = e / (G::ROWB / 16) / (kQB - filled);
    *reinterpret_cast<uint4*>(sQ + tl * kQB * G::ROWB + row * G::ROWB + piece * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  volatile int* abort_flag = &abort_s;
  const uint32_t t0 = uniform(tmem_base_s), tK = t0 + NB * 128, tV = tK + DP;       // buffer u: S^T at 128 u, dP^T at 128 u + 64

  if (warp == 8) {
    // ------------------------------------------------------------------------------------------------ copies
    if (elect_one() && T_ > 0) {
      mbar_expect_tx(&bar.kv_full, 2 * C::KB);
      load_tile_tma<DP>(sK, &mk, &bar.kv_full, kKeys, hk, j0, n * f.ck.n_mul, b * f.ck.b_mul);
      load_tile_tma<DP>(sV, &mv, &bar.kv_full, kKeys, hk, j0, n * f.cv.n_mul, b * f.cv.b_mul);
      int t = 0, pk = e0 / per_pack, blk = first + e0 % per_pack;
      for (; t < T_; ++t) {
        const int s = t % NS, h0 = hk * p.G + pk * p.pack;
        if (t >= NS) wait_or_flag(&bar.qd_empty[s], (t / NS - 1) & 1, abort_flag);
        if (*abort_flag) break;
        mbar_expect_tx(&bar.qd_full[s], 2 * f.q_bytes + kXB);
        load_tile_tma<DP>(sQ + s * C::QB, &mq, &bar.qd_full[s], kQB, h0, blk * nq, n * f.cq.n_mul, b * f.cq.b_mul);
        load_tile_tma<DP>(sG + s * C::QB, &mg, &bar.qd_full[s], kQB, h0, blk * nq, n, b);
        bulk_load_1d(sX + s * kXB, f.terms + (((int64_t)bn * head_groups(p) + h0 / p.pack) * f.n_blocks + blk) * kXB, kXB, &bar.qd_full[s]);
        if (++blk == first + per_pack) { blk = first; ++pk; }
      }
      drain_ring(&bar.kv_full, 1, 1); drain_ring(bar.qd_full, t, NS);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------------------------------------ products
    const uint32_t id_s = idesc_f16(128, kQB, f.fmt, 0, 0), id_x = idesc_f16(128, kQB, 1u, 0, 0), id_o = idesc_f16(128, DP, f.fmt, 0, 1);
    const uint32_t k_lo = desc_lo(smem_u32(sK), 16), v_lo = desc_lo(smem_u32(sV), 16), os_lo = desc_lo(smem_u32(sOneS), 16), od_lo = desc_lo(smem_u32(sOneD), 16);
    constexpr uint32_t kXHi = desc_hi(8 * 32, kSw32);
    auto scores = [&](int t) {
      const int s = t % NS;
      wait_or_flag(&bar.qd_full[s], (t / NS) & 1, abort_flag);
      if (__any_sync(0xffffffffu, *abort_flag)) return false;
      tc_fence_after();
      const uint32_t q_lo = desc_lo(smem_u32(sQ + s * C::QB), 16), g_lo = desc_lo(smem_u32(sG + s * C::QB), 16), x_lo = desc_lo(smem_u32(sX + s * kXB), 16);
      const uint32_t d = t0 + (t % NB) * 128;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) mma_ss_el(d, k_lo + k_step<DP>(ks, kKeys), G::HI, q_lo + k_step<DP>(ks, kQB), G::HI, id_s, ks > 0);
      mma_ss_el(d, os_lo, kXHi, x_lo, kXHi, id_x, true);
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) mma_ss_el(d + 64, v_lo + k_step<DP>(ks, kKeys), G::HI, g_lo + k_step<DP>(ks, kQB), G::HI, id_s, ks > 0);
      mma_ss_el(d + 64, od_lo, kXHi, x_lo, kXHi, id_x, true);
      tc_commit_el(&bar.sd_ready[t % NB]);
      return true;
    };
    if (T_ > 0) {
      wait_or_flag(&bar.kv_full, 0, abort_flag);
      bool ok = true;
      for (int t = 0; ok && t < NB && t < T_; ++t) ok = scores(t);
      for (int t = 0; ok && t < T_; ++t) {
        const int s = t % NS;
        wait_or_flag(&bar.pd_ready[t % NB], (t / NB) & 1, abort_flag);
        if (__any_sync(0xffffffffu, *abort_flag)) break;
        tc_fence_after();
        const uint32_t q_lo = desc_lo(smem_u32(sQ + s * C::QB), kQB * G::ROWB), g_lo = desc_lo(smem_u32(sG + s * C::QB), kQB * G::ROWB), a = t0 + (t % NB) * 128;
#pragma unroll
        for (int ks = 0; ks < kQB / 16; ++ks)        // the two halves of a block's columns keep their P^T where their scores were
          mma_ts_el(tV, a + (ks / 2) * 32 + (ks % 2) * 8, g_lo + ks * (16 * G::ROWB / 16), G::HI, id_o, t > 0 || ks > 0);
#pragma unroll
        for (int ks = 0; ks < kQB / 16; ++ks)
          mma_ts_el(tK, a + 64 + (ks / 2) * 32 + (ks % 2) * 8, q_lo + ks * (16 * G::ROWB / 16), G::HI, id_o, t > 0 || ks > 0);
        tc_commit_el(&bar.qd_empty[s]);
        if (t + 1 == T_) tc_commit_el(&bar.done);
        if (t + NB < T_) ok = scores(t + NB);
      }
    }
  } else {
    // ------------------------------------------------------------------------------------------------ P^T and dS^T
    const int half = warp >> 2, r = (warp & 3) * 32 + lane, j = j0 + r;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const bool keep = j < p.Lk && kept(p, b, n, j);
    const bool all_kept = __all_sync(0xffffffffu, keep);
    // queries [a, z] see key j
    const int a = j - p.right - p.off, z = j < p.sinks ? p.Lq : j + p.left - p.off;
    const int a_all = j0 + kKeys - 1 - p.right - p.off, z_all = j0 + kKeys <= p.sinks ? p.Lq : j0 + p.left - p.off;       // every key of the tile
    float up = 1.f;                               // dS's power of two: the largest |dS| comes to 2^13 .. 2^14
    if constexpr (kNarrow<T>) {
      const int nr = queries_of<kRows>(p), q0 = lo / nr, nt = hi > lo ? (hi + nr - 1) / nr - q0 : 0, packs = p.G / p.pack;
      int top = 0;
      for (int e = lane; e < nt * packs; e += 32)
        top = max(top, __ldg(f.tops + (int64_t)(f.n_qt - 1 - q0 - e % nt) * f.groups + bn * head_groups(p) + hk * packs + e / nt));
      top = __reduce_max_sync(0xffffffffu, top);
      if (top > 0 && top < 0x7f800000) up = pow2(13 - clamp_i((top >> 23) - 127, -40, 40));
    }
    int blk = first + e0 % per_pack;
    for (int t = 0; t < T_; ++t) {
      const int i0 = blk * nq;
      if (++blk == first + per_pack) blk = first;
      wait_or_flag(&bar.sd_ready[t % NB], (t / NB) & 1, abort_flag);
      if (__any_sync(0xffffffffu, *abort_flag)) break;
      tc_fence_after();
      const uint32_t tS = t0 + lanes + (t % NB) * 128 + half * 32, tD = tS + 64;
      uint32_t s[32], d[32];
      tmem_ld32(tS, s);
      tmem_ld32(tD, d);
      tmem_ld_wait(s, d);
      uint32_t bits = ~0u;
      const bool whole = all_kept && i0 >= a_all && i0 + nq - 1 <= z_all;
      if (!whole) {
        const int from = clamp_i(a - i0, 0, 64) * p.pack - half * 32, to = clamp_i(z - i0 + 1, 0, 64) * p.pack - half * 32;
        bits = keep ? ones32(to) & ~ones32(from) : 0u;
      }
      uint32_t pw[16];
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        float2 pr = mul2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), make_float2(f.c1, f.c1));
        pr = make_float2(ex2f(pr.x), ex2f(pr.y));
        float2 dp = make_float2(__uint_as_float(d[e]), __uint_as_float(d[e + 1]));
        if constexpr (kNarrow<T>) dp = mul2(dp, make_float2(up, up));
        float2 ds = mul2(pr, dp);
        if (!whole) {
          if (!(bits >> e & 1)) pr.x = ds.x = 0.f;
          if (!(bits >> (e + 1) & 1)) pr.y = ds.y = 0.f;
        }
        pw[e / 2] = Pack2<T>::pack(pr.x, pr.y);
        s[e / 2] = Pack2<T>::pack(ds.x, ds.y);
      }
      tmem_st16(tS, pw);
      tmem_st16(tD, *reinterpret_cast<uint32_t (*)[16]>(s));
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bar.pd_ready[t % NB]);
    }
    if (T_ > 0) wait_or_flag(&bar.done, 0, abort_flag);
    tc_fence_after();
    // write-out: warps 0-3 dK, 4-7 dV
    if (!__any_sync(0xffffffffu, *abort_flag)) {
      const uint32_t acc = (half ? tV : tK) + lanes;
      if (x < f.plan.split_x) {
        float* out = part_of<kKeys>(f.parts, f.plan, p, head, x) + (half * kKeys + r) * p.D;
        const float f1 = half ? 1.f : back(up);
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          if (c * 32 >= p.D) break;
          uint32_t o32[32];
          if (T_ > 0) { tmem_ld32(acc + c * 32, o32); tmem_ld_wait(); pin32(o32); }
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (c * 32 + e < p.D)
              *reinterpret_cast<float4*>(out + c * 32 + e) = T_ > 0 ? make_float4(__uint_as_float(o32[e]) * f1, __uint_as_float(o32[e + 1]) * f1,
                                                                                  __uint_as_float(o32[e + 2]) * f1, __uint_as_float(o32[e + 3]) * f1)
                                                                    : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      } else {
        T* out = static_cast<T*>(half ? p.dv : p.dk) + (((int64_t)bn * p.Lk + j) * p.Hk + hk) * p.D;
        if (T_ > 0) {
#pragma unroll
          for (int c = 0; c < DP / 32; ++c)
            if (c * 32 < p.D) store_rows<T>(acc + c * 32, half ? 1.f : p.scale * back(up), out + c * 32, (int64_t)p.Hk * p.D, j, p.Lk, p.D - c * 32);
        } else if (j < p.Lk) {
          for (int e = 0; e < p.D; e += 8) *reinterpret_cast<uint4*>(out + e) = make_uint4(0u, 0u, 0u, 0u);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && abort_s) *reinterpret_cast<volatile int*>(f.status) = 1;
  if (warp == 0) tmem_dealloc(t0, C::COLS);
}

// -------------------------------------------------------------------------------------------------------------------- dQ
template <int DP> struct QCfg {
  static constexpr int NS = DP == 128 ? 1 : 2;                  // stages of K and V
  static constexpr uint32_t COLS = 256;                         // S at 0, dP at 64, dQ at 128
  static constexpr int QB = Geo<DP>::TILE(kRows), KB = Geo<DP>::TILE(kKB);
  static constexpr size_t SMEM = 1024 + 2 * QB + 2 * NS * KB;
};
template <int NS> struct QBars {
  uint64_t q_full, kv_full[NS], kv_empty[NS], s_ready, d_ready, s_read, ds_written, summed, done;
};

template <int DP, typename T>
__global__ void __launch_bounds__(kThreads, 2)
window_dq_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mg, const __grid_constant__ CUtensorMap mk,
                    const __grid_constant__ CUtensorMap mv, const __grid_constant__ BwdP f) {
  using C = QCfg<DP>;
  using G = Geo<DP>;
  constexpr int NS = C::NS;
  const WinP& p = f.w;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *sQ = smem, *sG = sQ + C::QB, *sK = sG + C::QB, *sV = sK + NS * C::KB;
  __shared__ QBars<NS> bar;
  __shared__ float sums[2][kRows];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s, top_s;

  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  if (tid == 0) {
    abort_s = top_s = 0;
    mbar_init(&bar.q_full, 1);
    for (int i = 0; i < NS; ++i) { mbar_init(&bar.kv_full[i], 1); mbar_init(&bar.kv_empty[i], 1); }
    mbar_init(&bar.s_ready, 1); mbar_init(&bar.d_ready, 1); mbar_init(&bar.s_read, kCompute); mbar_init(&bar.ds_written, kCompute); mbar_init(&bar.summed, kCompute); mbar_init(&bar.done, 1);
    mbar_fence_init();
    prefetch_tmap(&mq); prefetch_tmap(&mg); prefetch_tmap(&mk); prefetch_tmap(&mv);
  }
  if (warp == 0) { tmem_alloc(&tmem_base_s, C::COLS); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  volatile int* abort_flag = &abort_s;
  const uint32_t t0 = uniform(tmem_base_s), tQ = t0 + 128;
  const int qt = f.n_qt - 1 - (int)(blockIdx.x / f.groups), group = blockIdx.x % f.groups;
  const int bn = group / head_groups(p), h0 = (group - bn * head_groups(p)) * p.pack, n = bn % p.N, b = bn / p.N, hk = h0 / p.G;
  const int nq = queries_of<kRows>(p), i0 = qt * nq, i1 = i0 + nq < p.Lq ? i0 + nq : p.Lq;
  const KeyTiles tiles = key_tiles<kKB>(p, i0, i1);
  const KeyRange range = key_range(p, i0, i1);
  // steps: the blocks of keys, or (f.two_walks) all of them for delta and then all of them for dQ
  const int blocks = tiles.count(), delta_steps = f.two_walks ? blocks : 0, T_ = delta_steps + blocks;
  auto key_block = [&](int t) { return tiles.at(t < blocks ? t : t - blocks) * kKB; };

  if (warp == 8) {
    // ------------------------------------------------------------------------------------------------ copies
    if (elect_one() && T_ > 0) {
      mbar_expect_tx(&bar.q_full, 2 * f.qt_bytes);
      load_tile_tma<DP>(sQ, &mq, &bar.q_full, kRows, h0, i0, n * f.cq.n_mul, b * f.cq.b_mul);
      load_tile_tma<DP>(sG, &mg, &bar.q_full, kRows, h0, i0, n, b);
      int t = 0;
      for (; t < T_; ++t) {
        const int s = t % NS, j0 = key_block(t);
        if (t >= NS) wait_or_flag(&bar.kv_empty[s], (t / NS - 1) & 1, abort_flag);
        if (*abort_flag) break;
        mbar_expect_tx(&bar.kv_full[s], 2 * C::KB);
        load_tile_tma<DP>(sK + s * C::KB, &mk, &bar.kv_full[s], kKB, hk, j0, n * f.ck.n_mul, b * f.ck.b_mul);
        load_tile_tma<DP>(sV + s * C::KB, &mv, &bar.kv_full[s], kKB, hk, j0, n * f.cv.n_mul, b * f.cv.b_mul);
      }
      drain_ring(&bar.q_full, 1, 1); drain_ring(bar.kv_full, t, NS);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------------------------------------ products
    const uint32_t id_s = idesc_f16(128, kKB, f.fmt, 0, 0), id_q = idesc_f16(128, DP, f.fmt, 0, 1);
    const uint32_t q_lo = desc_lo(smem_u32(sQ), 16), g_lo = desc_lo(smem_u32(sG), 16);
    auto s_scores = [&](int t) {                  // S(t); false: given up
      const int s = t % NS;
      wait_or_flag(&bar.kv_full[s], (t / NS) & 1, abort_flag);
      if (__any_sync(0xffffffffu, *abort_flag)) return false;
      tc_fence_after();
      const uint32_t k_lo = desc_lo(smem_u32(sK + s * C::KB), 16);
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) mma_ss_el(t0, q_lo + k_step<DP>(ks, kRows), G::HI, k_lo + k_step<DP>(ks, kKB), G::HI, id_s, ks > 0);
      tc_commit_el(&bar.s_ready);
      return true;
    };
    auto d_scores = [&](int t) {                  // dP(t), of the stage that S(t) waited for
      const uint32_t v_lo = desc_lo(smem_u32(sV + t % NS * C::KB), 16);
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) mma_ss_el(t0 + 64, g_lo + k_step<DP>(ks, kRows), G::HI, v_lo + k_step<DP>(ks, kKB), G::HI, id_s, ks > 0);
      tc_commit_el(&bar.d_ready);
    };
    if (T_ > 0) {
      wait_or_flag(&bar.q_full, 0, abort_flag);
      bool ok = s_scores(0);
      if (ok) d_scores(0);
      for (int t = 0; ok && t < T_; ++t) {
        const int s = t % NS;
        // S has been read: the next one, while the compute warps exponentiate (with one stage its keys are not there yet)
        wait_or_flag(&bar.s_read, t & 1, abort_flag);
        if (NS > 1 && t + 1 < T_) ok = s_scores(t + 1);
        wait_or_flag(&bar.ds_written, t & 1, abort_flag);
        if (!ok || __any_sync(0xffffffffu, *abort_flag)) break;
        tc_fence_after();
        if (t >= delta_steps) {
          const uint32_t k_lo = desc_lo(smem_u32(sK + s * C::KB), kKB * G::ROWB);
#pragma unroll
          for (int ks = 0; ks < kKB / 16; ++ks)
            mma_ts_el(tQ, t0 + 64 + (ks / 2) * 32 + (ks % 2) * 8, k_lo + ks * (16 * G::ROWB / 16), G::HI, id_q, t > delta_steps || ks > 0);
        }
        tc_commit_el(&bar.kv_empty[s]);
        if (t + 1 == T_) tc_commit_el(&bar.done);
        else {
          if (NS == 1) ok = s_scores(t + 1);
          if (ok) d_scores(t + 1);
        }
      }
    }
  } else {
    // ------------------------------------------------------------------------------------------------ dS
    const int half = warp >> 2, r = (warp & 3) * 32 + lane, l_ = r / p.pack, i = i0 + l_, h = h0 + r - l_ * p.pack, at = i + p.off;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const bool live = l_ < nq && i < p.Lq;
    float up = 1.f, top = 0.f;                    // dS's power of two; the largest |dS| so far, with it
    if constexpr (kNarrow<T>) {
      if (T_ > 0) {
        // the row's largest |dO| comes to 4 .. 8, so that V may be some hundreds before dS overflows; bytes of a row stay in it when they are swizzled
        wait_or_flag(&bar.q_full, 0, abort_flag);
        uint32_t most = 0;
#pragma unroll
        for (int pn = 0; pn < G::PANELS; ++pn)
#pragma unroll
          for (int e = 0; e < G::ROWB / 16; ++e) {
            // (each lane of eight begins at another piece: other banks)
            const int piece = (e + (G::ROWB == 128 ? lane : lane >> 1)) % (G::ROWB / 16);
            const uint4 g = *reinterpret_cast<const uint4*>(sG + pn * kRows * G::ROWB + r * G::ROWB + piece * 16);
            most = __vmaxu2(__vmaxu2(most, __vmaxu2(g.x & 0x7fff7fffu, g.y & 0x7fff7fffu)), __vmaxu2(g.z & 0x7fff7fffu, g.w & 0x7fff7fffu));
          }
        const int m = max((int)(most & 0xffffu), (int)(most >> 16));
        if (m > 0 && m < 0x7c00) up = pow2(2 - (m >= 0x400 ? (m >> 10) - 15 : 7 - __clz(m)));
      }
    }
    float lse = -INFINITY, minus = 0.f;           // minus: -delta, with dS's power of two
    const int64_t stat = ((int64_t)bn * p.H + h) * p.Lq + i;
    if (live) {
      lse = p.lse[stat];
      if (!f.two_walks) minus = -p.delta[stat] * up;
    }
    float sum = 0.f;                              // of P dP over this thread's columns
    const float off = lse == -INFINITY ? -INFINITY : -lse * kLog2e;       // a row that sees nothing: probability 0
    const uint8_t* mask = p.mask ? p.mask + b * p.ms[0] + n * p.ms[1] : nullptr;
    auto mask_byte = [&](int t, int hf) -> uint32_t {
      const int j = key_block(t) + hf * 32 + lane;
      return j < p.Lk && mask[(int64_t)j * p.ms[2]];
    };
    uint32_t mb = 1;
    if (mask && T_ > 0) mb = mask_byte(0, half);
    for (int t = 0; t < T_; ++t) {
      const int j0 = key_block(t) + half * 32;
      uint32_t keep = ~0u;
      if (mask) {
        keep = __ballot_sync(0xffffffffu, mb);
        if (t + 1 < T_) mb = mask_byte(t + 1, half);
      }
      if (f.two_walks && t == delta_steps) {      // the two halves' sums make delta
        sums[half][r] = sum;
        mbar_arrive(&bar.summed);
        wait_or_flag(&bar.summed, 0, abort_flag);
        if (__any_sync(0xffffffffu, *abort_flag)) break;
        const float delta = sum + sums[half ^ 1][r];
        if (half == 0 && live) f.delta[stat] = delta;
        minus = -delta * up;
      }
      wait_or_flag(&bar.s_ready, t & 1, abort_flag);
      if (__any_sync(0xffffffffu, *abort_flag)) break;
      tc_fence_after();
      const uint32_t tS = t0 + lanes + half * 32, tD = tS + 64;
      uint32_t s[32], d[32];
      tmem_ld32(tS, s);
      tmem_ld_wait();
      pin32(s);
      tc_fence_before();
      mbar_arrive(&bar.s_read);
      const bool whole = all_seen(p, i0 + p.off, i1 - 1 + p.off, j0, j0 + 32) && keep == ~0u;
      const uint32_t bits = whole ? ~0u : seen32(p, at, j0) & keep;
      const float2 c2 = make_float2(f.c1, f.c1), o2 = make_float2(off, off), u2 = make_float2(up, up), d2 = make_float2(minus, minus);
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const float2 x = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c2, o2);
        s[e] = __float_as_uint(ex2f(x.x)); s[e + 1] = __float_as_uint(ex2f(x.y));
      }
      wait_or_flag(&bar.d_ready, t & 1, abort_flag);
      if (__any_sync(0xffffffffu, *abort_flag)) break;
      tc_fence_after();
      tmem_ld32(tD, d);
      tmem_ld_wait();
      pin32(d);
      if (t < delta_steps) {
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float2 x = mul2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), make_float2(__uint_as_float(d[e]), __uint_as_float(d[e + 1])));
          if (!whole) {
            if (!(bits >> e & 1)) x.x = 0.f;
            if (!(bits >> (e + 1) & 1)) x.y = 0.f;
          }
          acc = add2(acc, x);
        }
        sum += acc.x + acc.y;
        tc_fence_before();
        mbar_arrive(&bar.ds_written);
        continue;
      }
      uint32_t w[16];
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        float2 ds = mul2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), fma2(make_float2(__uint_as_float(d[e]), __uint_as_float(d[e + 1])), u2, d2));
        if (!whole) {
          if (!(bits >> e & 1)) ds.x = 0.f;
          if (!(bits >> (e + 1) & 1)) ds.y = 0.f;
        }
        if constexpr (kNarrow<T>) top = max3f(top, fabsf(ds.x), fabsf(ds.y));
        w[e / 2] = Pack2<T>::pack(ds.x, ds.y);
      }
      tmem_st16(tD, w);
      if (!whole) {
        // rows of K of keys that are masked or that no query of the tile sees, this warp set's 32 keys of the block (the keys beyond Lk are
        // zeros already): S has been formed
        const uint32_t z = ~(keep & range32(range, j0)) & ones32(p.Lk - j0);
        if (z) {
          const int row = r >> 2;                 // four threads a row
          if (z >> row & 1) {
            uint8_t* at_row = sK + (t % NS) * C::KB + (half * 32 + row) * G::ROWB + (r & 3) * (G::ROWB / 4);
#pragma unroll
            for (int pn = 0; pn < G::PANELS; ++pn)
#pragma unroll
              for (int e = 0; e < G::ROWB / 64; ++e) *reinterpret_cast<uint4*>(at_row + pn * kKB * G::ROWB + e * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_async_smem();
        }
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bar.ds_written);
    }
    if (T_ > 0) wait_or_flag(&bar.done, 0, abort_flag);
    tc_fence_after();
    if (!__any_sync(0xffffffffu, *abort_flag)) {
      T* out = static_cast<T*>(p.dq) + (((int64_t)bn * p.Lq + i) * p.H + h) * p.D;
      if (T_ > 0) {
#pragma unroll
        for (int c = 0; c < DP / 32; ++c)            // the two warps of a set of lanes take alternate columns
          if (c % 2 == half % (DP / 32 > 1 ? 2 : 1) && (DP > 32 || half == 0) && c * 32 < p.D)
            store_rows_at<T>(tQ + lanes + c * 32, p.scale * back(up), live ? out + c * 32 : nullptr, p.D - c * 32);
      } else if (live && half == 0) {
        for (int e = 0; e < p.D; e += 8) *reinterpret_cast<uint4*>(out + e) = make_uint4(0u, 0u, 0u, 0u);
        if (f.two_walks) f.delta[stat] = 0.f;
      }
    }
    if constexpr (kNarrow<T>) {
      const int most = __reduce_max_sync(0xffffffffu, live ? __float_as_int(top * back(up)) : 0);
      if (lane == 0) atomicMax(&top_s, most);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && abort_s) *reinterpret_cast<volatile int*>(f.status) = 1;
  if (kNarrow<T> && tid == 0) f.tops[blockIdx.x] = top_s;
  if (warp == 0) tmem_dealloc(t0, C::COLS);
}

// ------------------------------------------------------------------------------------------------------------------ host
// processors' worth of CTAs; two share one
KeyPlan tc_plan(const WinP& p) { return key_plan<kKeys, kQB>(p, 2 * sm_count()); }
int block_count(const WinP& p) { const int q = queries_of<kQB>(p); return (p.Lq + q - 1) / q; }
size_t delta_bytes(const WinP& p) { return align_up(sizeof(float) * (size_t)p.B * p.N * p.H * p.Lq, 256); }
// dQ: tiles of queries of a pack of heads
int query_tiles(const WinP& p) { const int q = queries_of<kRows>(p); return (p.Lq + q - 1) / q; }
size_t top_bytes(const WinP& p, int dtype) {
  return dtype == MF_F16 ? align_up(sizeof(int) * (size_t)query_tiles(p) * p.B * p.N * head_groups(p), 256) : 0;
}
size_t term_bytes(const WinP& p) { return (size_t)p.B * p.N * head_groups(p) * block_count(p) * kXB; }

template <int DP, typename T>
int launch(const mf_window_args& a, cudaStream_t st) {
  using G = Geo<DP>;
  BwdP f{};
  WinP& p = f.w;
  p = window_params(a);
  f.plan = tc_plan(p);
  f.n_blocks = block_count(p);
  const int nq = queries_of<kRows>(p), nb = queries_of<kQB>(p);
  f.n_qt = query_tiles(p); f.groups = a.B * a.N * head_groups(p);
  f.q_bytes = nb * p.pack * DP * 2; f.qt_bytes = nq * p.pack * DP * 2;
  f.c1 = kLog2e / sqrtf((float)a.D);
  f.fmt = a.dtype == MF_BF16 ? 1u : 0u;
  float* delta = static_cast<float*>(a.workspace);
  uint8_t* terms = static_cast<uint8_t*>(a.workspace) + delta_bytes(p);
  // delta of a row is the sum of o d_o, o rounded to 16 bits, and dS = P (dP - delta) gets P times its error: with few keys a row, where P
  // is large, that is as much as dS's own rounding.  Up to 512 keys the dQ kernel forms it as the sum of P dP instead, in a walk of its
  // own, which is short there.  [1, 1, 3000, 2, 64] bf16, causal: dQ off by 2.4e-3 of its norm at 3, 5 and 129 keys a row; from o d_o 3.2e-3, 2.9e-3 and 2.4e-3
  // (2.40e-3 and 2.46e-3 at 129 keys and heads of 32), dK alike.
  f.two_walks = (int64_t)p.left + p.right + 1 + p.sinks <= 512 || p.Lk <= 512;
  p.delta = f.delta = delta; f.terms = terms;
  f.tops = reinterpret_cast<int*>(terms + term_bytes(p));
  f.parts = reinterpret_cast<float*>(terms + term_bytes(p) + top_bytes(p, a.dtype));
  f.status = status_word();
  MF_REQUIRE(f.status, MF_ERR_CUDA, "could not allocate the device status word");
  MF_REQUIRE(tc_async_status() == 0, MF_ERR_CUDA, "an earlier tensor-core kernel gave up on a bounded wait; results are invalid");
  const int64_t grid_kv = (int64_t)f.plan.x_total * a.B * a.N * a.Hk, grid_q = (int64_t)f.n_qt * f.groups;
  MF_REQUIRE(grid_kv <= 0x7fffffff && grid_q <= 0x7fffffff && (int64_t)a.B * a.N * a.H <= 0x7fffffff, MF_ERR_UNSUPPORTED, "too many tiles for one launch");

  CUtensorMap mq, mg, mk, mv, mq64, mg64, mk64, mv64;
  Coords cg;
  const int64_t gs[5] = {(int64_t)a.N * a.Lq * a.H * a.D, (int64_t)a.Lq * a.H * a.D, (int64_t)a.H * a.D, a.D, 1};
  int r;
  if ((r = operand_map(&mq, &f.cq, a.q, a.dtype, a.B, a.N, a.Lq, a.H, a.D, a.q_strides, G::COLS, p.pack, nq))) return r;
  if ((r = operand_map(&mg, &cg, a.d_o, a.dtype, a.B, a.N, a.Lq, a.H, a.D, gs, G::COLS, p.pack, nq))) return r;
  if ((r = operand_map(&mq64, &f.cq, a.q, a.dtype, a.B, a.N, a.Lq, a.H, a.D, a.q_strides, G::COLS, p.pack, nb))) return r;
  if ((r = operand_map(&mg64, &cg, a.d_o, a.dtype, a.B, a.N, a.Lq, a.H, a.D, gs, G::COLS, p.pack, nb))) return r;
  if ((r = operand_map(&mk, &f.ck, a.k, a.dtype, a.B, a.N, a.Lk, a.Hk, a.D, a.k_strides, G::COLS, 1, kKeys))) return r;
  if ((r = operand_map(&mv, &f.cv, a.v, a.dtype, a.B, a.N, a.Lk, a.Hk, a.D, a.v_strides, G::COLS, 1, kKeys))) return r;
  if ((r = operand_map(&mk64, &f.ck, a.k, a.dtype, a.B, a.N, a.Lk, a.Hk, a.D, a.k_strides, G::COLS, 1, kKB))) return r;
  if ((r = operand_map(&mv64, &f.cv, a.v, a.dtype, a.B, a.N, a.Lk, a.Hk, a.D, a.v_strides, G::COLS, 1, kKB))) return r;

  const auto terms_kernel = [&](auto given) -> int {
    window_terms_kernel<T, decltype(given)::value><<<dim3(f.n_blocks, head_groups(p), a.B * a.N), 256, 0, st>>>(p, delta, terms, sqrtf((float)a.D));
    MF_LAUNCHED("window_terms_kernel");
    return MF_OK;
  };
  constexpr auto dkv = window_dkv_tc_kernel<DP, T>;
  constexpr auto dq = window_dq_tc_kernel<DP, T>;
  if ((r = opt_in_smem<dkv>(KvCfg<DP>::SMEM))) return r;
  if ((r = opt_in_smem<dq>(QCfg<DP>::SMEM))) return r;
  const auto dq_kernel = [&]() -> int {
    dq<<<(unsigned)grid_q, kThreads, QCfg<DP>::SMEM, st>>>(mq, mg, mk64, mv64, f);
    MF_LAUNCHED("window_dq_tc_kernel");
    return MF_OK;
  };
  if (f.two_walks) {
    if ((r = dq_kernel())) return r;
    if ((r = terms_kernel(std::true_type{}))) return r;
  } else {
    if ((r = terms_kernel(std::false_type{}))) return r;
    if ((r = dq_kernel())) return r;
  }
  dkv<<<(unsigned)grid_kv, kThreads, KvCfg<DP>::SMEM, st>>>(mk, mv, mq64, mg64, f);
  MF_LAUNCHED("window_dkv_tc_kernel");
  return window_join<T, kKeys, kQB>(p, f.plan, f.parts, st);
}
template <typename T>
int by_size(const mf_window_args& a, cudaStream_t st) {
  return a.D <= 32 ? launch<32, T>(a, st) : a.D <= 64 ? launch<64, T>(a, st) : launch<128, T>(a, st);
}
}  // namespace
}  // namespace win

bool window_bwd_tc_supported(const mf_window_args& a) {
  const uintptr_t align = (uintptr_t)a.o | (uintptr_t)a.d_o | (uintptr_t)a.dq | (uintptr_t)a.dk | (uintptr_t)a.dv;
  return win::window_tc_supported(a) && (align & 15) == 0;
}
size_t window_bwd_tc_workspace(const mf_window_args& a) {
  const win::WinP p = win::window_params(a);
  return win::delta_bytes(p) + win::term_bytes(p) + win::top_bytes(p, a.dtype) + sizeof(float) * win::part_floats<win::kKeys>(win::tc_plan(p), p);
}
int window_bwd_tc(const mf_window_args& a, cudaStream_t st) {
  return a.dtype == MF_BF16 ? win::by_size<__nv_bfloat16>(a, st) : win::by_size<__half>(a, st);
}

}  // namespace mf
