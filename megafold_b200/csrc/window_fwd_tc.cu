// Sliding-window attention with sinks, forward, on the tensor cores (tcgen05 + TMEM + TMA): 16-bit tensors, head sizes that are
// multiples of 8 up to 128.
//
// A CTA takes 128 rows of queries (of the heads that share a key head) and walks the blocks of 64 keys that they see.  Warps 0-7: two
// threads share a query row (a TMEM lane), 32 columns each; running maximum (the two exchange theirs) and sum, P over the
// scores in TMEM.  Warp 8 fetches Q, K and V by TMA, warp 9 issues the products
//
//   S(t) = Q K(t)^T into one of two buffers          O += P(t) V(t)   (P as TMEM A operand, V MN-major)
//
// in the order S(0) S(1) PV(0) S(2) PV(1) ..., so that a buffer's P has been read when the next scores go over it, and the next scores are
// there while this block's are exponentiated.  O stays in TMEM and is brought to a new maximum only when that grew by more than
// 2^8 in the exponent.  A window makes short walks (5 blocks at 64 + 64 keys), so nothing is pipelined across items: two CTAs share
// an SM instead.  Tried at [1, 1, 16384, 16 on 4 heads, 64], window 1024 / [2, 1, 2048 of 6001, 16 on 4, 128], window 2048 / one token of 64
// sequences, 32 on 8 heads of 128, window 1024 / [1, 1, 4603, 4, 32], window 65: twenty calls in a row 158 / 88 / 56 / 8.7 us a call,
// one call with its operands out of L2 168 / 97 / 72 / 14.  One thread a row, one score buffer, four CTAs (two at 128 columns): 131 / 89 / 81 / 9.8 and
// 140 / 108 / 96 / 16, so ahead by a fifth where many tiles of up to 64 columns fill the processors four times over, and behind elsewhere: one form
// serves all sizes, and long sequences of such heads pay for it.  One score buffer with two threads a row, and blocks of 128 keys, were no
// better at the first size and behind at the next two (159 / 127 / 87 and 168 / 102 / 77, measured beside 160 / 88 / 68 for this).
// Bound: the exponentials, half of the time at 64 columns (16 a clock and SM), and the waits between a block's steps.
//
// Blocks that a row does not see whole go through a 64-bit mask a row (window, sinks, end of the keys, key mask); rows of V whose
// key is masked, or seen by no query of the tile, are overwritten with zeros in shared memory, since 0 * NaN would reach the sum.  P is rounded to the
// operands' type (the matrix instruction's), its sum is of the unrounded fp32 values.
//
// All waits are bounded; on expiry the CTA leaves without touching its outputs and the host sees mf_async_status() != 0.
#include "window_tc_common.cuh"

namespace mf {
namespace win {
namespace {

constexpr int kQ = 128, kK = 64;
constexpr int NB = 2;                                           // score buffers of 64 columns
constexpr int kSoft = 256, kThreads = kSoft + 64;
constexpr uint32_t kCols = 256;                                 // TMEM: scores at 0 and 64, O at 128

template <int DP> struct Cfg {
  static constexpr int NS = DP == 128 ? 2 : 3;                  // K and V stages
  static constexpr int QB = Geo<DP>::TILE(kQ), KB = Geo<DP>::TILE(kK);
  static constexpr size_t SMEM = 1024 + QB + 2 * NS * KB;
};

struct FwdP {
  WinP w;
  Coords cq, ck, cv;
  Split sp;
  int n_qt, groups;         // tiles of queries; groups of heads in all sequences
  int q_bytes;              // of a tile's rows of queries
  float c1;                 // D^-1/2 * log2(e)
  uint32_t fmt;
  int* status;
};

template <int NS> struct Bars {
  uint64_t q_full, k_full[NS], k_empty[NS], v_full[NS], v_empty[NS], s_ready[NB], p_ready[NB], pv_done;
};

template <int DP, typename T>
__global__ void __launch_bounds__(kThreads, 2)
window_fwd_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                     const __grid_constant__ FwdP f) {
  using C = Cfg<DP>;
  using G = Geo<DP>;
  constexpr int NS = C::NS;
  const WinP& p = f.w;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *sQ = smem, *sK = sQ + C::QB, *sV = sK + NS * C::KB;
  __shared__ Bars<NS> bar;
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;
  __shared__ float other[2][2][kQ];               // [parity of the block][half of the columns][row]: maxima, at the end sums

  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  if (tid == 0) {
    abort_s = 0;
    mbar_init(&bar.q_full, 1);
    for (int i = 0; i < NS; ++i) { mbar_init(&bar.k_full[i], 1); mbar_init(&bar.k_empty[i], 1); mbar_init(&bar.v_full[i], 1); mbar_init(&bar.v_empty[i], 1); }
    for (int i = 0; i < NB; ++i) { mbar_init(&bar.s_ready[i], 1); mbar_init(&bar.p_ready[i], kSoft); }
    mbar_init(&bar.pv_done, 1);
    mbar_fence_init();
    prefetch_tmap(&mq); prefetch_tmap(&mk); prefetch_tmap(&mv);
  }
  if (warp == 0) { tmem_alloc(&tmem_base_s, kCols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  volatile int* abort_flag = &abort_s;
  const uint32_t t0 = uniform(tmem_base_s);
  const uint32_t tO = t0 + NB * 64;

  // the last queries first: where windows are cut off at the start of the keys those have the most to do
  const int part = blockIdx.x % f.sp.splits, item = blockIdx.x / f.sp.splits;
  const int qt = f.n_qt - 1 - item / f.groups, group = item % f.groups;
  const int bn = group / head_groups(p), h0 = (group - bn * head_groups(p)) * p.pack, n = bn % p.N, b = bn / p.N, hk = h0 / p.G;
  const int nq = queries_of<kQ>(p), i0 = qt * nq, i1 = i0 + nq < p.Lq ? i0 + nq : p.Lq;
  const KeyTiles tiles = key_tiles<kK>(p, i0, i1);
  const KeyRange range = key_range(p, i0, i1);
  const int first = (int)((int64_t)tiles.count() * part / f.sp.splits), T_ = (int)((int64_t)tiles.count() * (part + 1) / f.sp.splits) - first;

  if (warp == 8) {
    // ------------------------------------------------------------------------------------------------ copies
    // A copy a panel, each from a lane of its own: one instruction for two copies costs the warp little more than one copy.  K goes ahead of V:
    // S(t) has left the stage of K(t) one product before V(t) is done with.
    const bool leader = elect_one();
    auto ask = [&](uint8_t* dst, const CUtensorMap* m, uint64_t* full, int t, const Coords& c) {
      __syncwarp();
      if (lane < G::PANELS) tma_load_5d(dst + lane * kK * G::ROWB, m, full, lane * G::COLS, hk, tiles.at(first + t) * kK, n * c.n_mul, b * c.b_mul);
      __syncwarp();
    };
    int k_asked = 0, v_asked = 0;
    if (T_ > 0) {
      if (leader) mbar_expect_tx(&bar.q_full, f.q_bytes);
      __syncwarp();
      if (lane < G::PANELS) tma_load_5d(sQ + lane * kQ * G::ROWB, &mq, &bar.q_full, lane * G::COLS, h0, i0, n * f.cq.n_mul, b * f.cq.b_mul);
      __syncwarp();
      for (; v_asked < T_; ++v_asked) {
        const int t = v_asked, s = t % NS;
        if (t >= NS) wait_or_flag(&bar.k_empty[s], (t / NS - 1) & 1, abort_flag);
        if (__any_sync(0xffffffffu, *abort_flag)) break;
        if (leader) mbar_expect_tx(&bar.k_full[s], C::KB);
        ask(sK + s * C::KB, &mk, &bar.k_full[s], t, f.ck);
        ++k_asked;
        if (t >= NS) wait_or_flag(&bar.v_empty[s], (t / NS - 1) & 1, abort_flag);
        if (__any_sync(0xffffffffu, *abort_flag)) break;
        if (leader) mbar_expect_tx(&bar.v_full[s], C::KB);
        ask(sV + s * C::KB, &mv, &bar.v_full[s], t, f.cv);
      }
      // none may land after this CTA has left
      drain_ring(&bar.q_full, 1, 1); drain_ring(bar.k_full, k_asked, NS); drain_ring(bar.v_full, v_asked, NS);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------------------------------------ products
    const uint32_t id_s = idesc_f16(128, kK, f.fmt, 0, 0), id_o = idesc_f16(128, DP, f.fmt, 0, 1);
    const uint32_t q_lo = desc_lo(smem_u32(sQ), 16);
    auto scores = [&](int t) {                    // false: given up
      const int s = t % NS;
      wait_or_flag(&bar.k_full[s], (t / NS) & 1, abort_flag);
      if (__any_sync(0xffffffffu, *abort_flag)) return false;
      tc_fence_after();
      const uint32_t k_lo = desc_lo(smem_u32(sK + s * C::KB), 16), d = t0 + t % NB * 64;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) mma_ss_el(d, q_lo + k_step<DP>(ks, kQ), G::HI, k_lo + k_step<DP>(ks, kK), G::HI, id_s, ks > 0);
      tc_commit_el(&bar.s_ready[t % NB]);
      tc_commit_el(&bar.k_empty[s]);
      return true;
    };
    if (T_ > 0) {
      wait_or_flag(&bar.q_full, 0, abort_flag);
      bool ok = true;
      for (int t = 0; ok && t < NB && t < T_; ++t) ok = scores(t);
      for (int t = 0; ok && t < T_; ++t) {
        const int s = t % NS;
        wait_or_flag(&bar.v_full[s], (t / NS) & 1, abort_flag);
        wait_or_flag(&bar.p_ready[t % NB], (t / NB) & 1, abort_flag);
        if (__any_sync(0xffffffffu, *abort_flag)) break;
        tc_fence_after();
        const uint32_t v_lo = desc_lo(smem_u32(sV + s * C::KB), kK * G::ROWB), a = t0 + t % NB * 64;
#pragma unroll
        for (int ks = 0; ks < kK / 16; ++ks)      // each half of the columns keeps its P where its scores were
          mma_ts_el(tO, a + ks / 2 * 32 + ks % 2 * 8, v_lo + ks * (16 * G::ROWB / 16), G::HI, id_o, t > 0 || ks > 0);
        tc_commit_el(&bar.pv_done);
        tc_commit_el(&bar.v_empty[s]);
        if (t + NB < T_) ok = scores(t + NB);
      }
    }
  } else {
    // ------------------------------------------------------------------------------------------------ softmax
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int half = warp >> 2, r = (warp & 3) * 32 + lane, l_ = r / p.pack, i = i0 + l_, h = h0 + r - l_ * p.pack, at = i + p.off;
    const bool live = l_ < nq && i < p.Lq, any_live = __any_sync(0xffffffffu, live);       // a warp without rows (a few queries) only takes part
    const uint8_t* mask = p.mask ? p.mask + b * p.ms[0] + n * p.ms[1] : nullptr;
    auto mask_bytes = [&](int t, uint32_t (&mb)[2]) {
      const int j = tiles.at(first + t) * kK + lane;
      mb[0] = j < p.Lk && mask[(int64_t)j * p.ms[2]]; mb[1] = j + 32 < p.Lk && mask[(int64_t)(j + 32) * p.ms[2]];
    };
    uint32_t mb[2] = {1, 1};
    if (mask && T_ > 0) mask_bytes(0, mb);
    float m = -INFINITY, l = 0.f;                 // m: the maximum that the sums refer to
    for (int t = 0; t < T_; ++t) {
      const int j0 = tiles.at(first + t) * kK;
      uint32_t keep[2] = {~0u, ~0u};
      if (mask) {
        keep[0] = __ballot_sync(0xffffffffu, mb[0]); keep[1] = __ballot_sync(0xffffffffu, mb[1]);
        if (t + 1 < T_) mask_bytes(t + 1, mb);
      }
      wait_or_flag(&bar.s_ready[t % NB], (t / NB) & 1, abort_flag);
      tc_fence_after();
      const uint32_t tS = t0 + lanes + t % NB * 64 + half * 32;
      const bool whole = all_seen(p, i0 + p.off, i1 - 1 + p.off, j0, j0 + kK) && (keep[0] & keep[1]) == ~0u;
      uint32_t s[32];
      tmem_ld32(tS, s);
      tmem_ld_wait();
      pin32(s);
      float corr = 1.f, mx = m;
      if (any_live) {
        if (!whole) {
          const uint32_t bits = seen32(p, at, j0 + half * 32) & (half ? keep[1] : keep[0]);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(bits >> e & 1)) s[e] = 0xff800000u;
        }
        float m4[4] = {m, m, m, m};
#pragma unroll
        for (int e = 0; e < 32; e += 2) m4[e / 2 % 4] = max3f(m4[e / 2 % 4], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
        mx = fmaxf(max3f(m4[0], m4[1], m4[2]), m4[3]);
      }
      other[t & 1][half][r] = mx;
      if (named_sync_or(1 + (warp & 3), 64, *abort_flag)) break;          // the two warps of these rows, which leave together
      if (any_live) {
        mx = fmaxf(mx, other[t & 1][half ^ 1][r]);
        if ((mx - m) * f.c1 > 8.f) {              // also from -inf
          corr = ex2f((m - mx) * f.c1);
          m = mx;
          l *= corr;
        }
        const float off = m == -INFINITY ? 0.f : -m * f.c1;     // nothing seen so far: every logit is -inf
        const float2 c2 = make_float2(f.c1, f.c1), o2 = make_float2(off, off);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 x = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c2, o2);
          const float2 pr = make_float2(ex2f(x.x), ex2f(x.y));
          sum[e / 2 % 2] = add2(sum[e / 2 % 2], pr);
          w[e / 2] = Pack2<T>::pack(pr.x, pr.y);
        }
        tmem_st16(tS, w);
        const float2 s2 = add2(sum[0], sum[1]);
        l += s2.x + s2.y;
      }
      // P V of the block before: O may be changed, and has to be complete to be
      if (t > 0) {
        wait_or_flag(&bar.pv_done, (t - 1) & 1, abort_flag);
        if (__any_sync(0xffffffffu, corr != 1.f)) {
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < DP / 32; ++c) {     // warps that share rows take alternate columns
            if (c % 2 != half) continue;
            uint32_t o32[32];
            tmem_ld32(tO + lanes + c * 32, o32);
            tmem_ld_wait();
            pin32(o32);
#pragma unroll
            for (int e = 0; e < 32; ++e) o32[e] = __float_as_uint(__uint_as_float(o32[e]) * corr);
            tmem_st32(tO + lanes + c * 32, o32);
          }
        }
      }
      if (!whole) {
        // rows of V of keys that are masked or that no query of the tile sees (the keys beyond Lk are zeros already)
        const int left = p.Lk - j0;
        const uint32_t z0 = ~(keep[0] & range32(range, j0)) & ones32(left), z1 = ~(keep[1] & range32(range, j0 + 32)) & ones32(left - 32);
        if (z0 | z1) {
          const int s = t % NS;
          wait_or_flag(&bar.v_full[s], (t / NS) & 1, abort_flag);
          const int row = tid / 4;                // four threads a row
          if ((row < 32 ? z0 >> row : z1 >> (row - 32)) & 1) {
            uint8_t* at_row = sV + s * C::KB + row * G::ROWB + tid % 4 * (G::ROWB / 4);
#pragma unroll
            for (int pn = 0; pn < G::PANELS; ++pn)
#pragma unroll
              for (int x = 0; x < G::ROWB / 64; ++x) *reinterpret_cast<uint4*>(at_row + pn * kK * G::ROWB + x * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_async_smem();
        }
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bar.p_ready[t % NB]);
    }
    if (T_ > 0) wait_or_flag(&bar.pv_done, (T_ - 1) & 1, abort_flag);
    tc_fence_after();
    other[T_ & 1][half][r] = l;                   // the last maxima were of the other parity
    if (!named_sync_or(1 + (warp & 3), 64, *abort_flag)) {
      l += other[T_ & 1][half ^ 1][r];
      const int64_t row = ((int64_t)bn * p.Lq + i) * p.H + h;
      const float inv = l == 0.f ? 0.f : 1.f / l, lse = l == 0.f ? -INFINITY : (m * f.c1 + lg2f(l)) * kLn2;
      if (f.sp.splits > 1) {
        float* out = f.sp.row(part, row, p.D);
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          if (c * 32 >= p.D) break;
          if (c % 2 != half) continue;
          uint32_t o32[32];
          if (T_ > 0) { tmem_ld32(tO + lanes + c * 32, o32); tmem_ld_wait(); pin32(o32); }
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (live && c * 32 + e < p.D) out[c * 32 + e] = T_ > 0 ? __uint_as_float(o32[e]) * inv : 0.f;
        }
        if (live && half == 0) f.sp.lse(part, row, p.D) = lse;
      } else {
        T* out = static_cast<T*>(p.o) + row * p.D;
        if (T_ > 0) {
#pragma unroll
          for (int c = 0; c < DP / 32; ++c)
            if (c % 2 == half && c * 32 < p.D) store_rows_at<T>(tO + lanes + c * 32, inv, live ? out + c * 32 : nullptr, p.D - c * 32);
        } else if (live && half == 0) {
          for (int d = 0; d < p.D; d += 8) *reinterpret_cast<uint4*>(out + d) = make_uint4(0u, 0u, 0u, 0u);
        }
        if (p.lse && live && half == 0) p.lse[((int64_t)bn * p.H + h) * p.Lq + i] = lse;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && abort_s) *reinterpret_cast<volatile int*>(f.status) = 1;
  if (warp == 0) tmem_dealloc(t0, kCols);
}

int tc_splits(const WinP& p) { return split_count<kQ, kK>(p, 2 * sm_count()); }

template <int DP, typename T>
int launch(const mf_window_args& a, cudaStream_t st) {
  using C = Cfg<DP>;
  using G = Geo<DP>;
  FwdP f{};
  f.w = window_params(a);
  CUtensorMap mq, mk, mv;
  if (int r = operand_map(&mq, &f.cq, a.q, a.dtype, a.B, a.N, a.Lq, a.H, a.D, a.q_strides, G::COLS, f.w.pack, queries_of<kQ>(f.w))) return r;
  if (int r = operand_map(&mk, &f.ck, a.k, a.dtype, a.B, a.N, a.Lk, a.Hk, a.D, a.k_strides, G::COLS, 1, kK)) return r;
  if (int r = operand_map(&mv, &f.cv, a.v, a.dtype, a.B, a.N, a.Lk, a.Hk, a.D, a.v_strides, G::COLS, 1, kK)) return r;
  const int nq = queries_of<kQ>(f.w);
  f.n_qt = (a.Lq + nq - 1) / nq; f.groups = a.B * a.N * head_groups(f.w);
  f.q_bytes = nq * f.w.pack * DP * 2;
  f.sp = Split{tc_splits(f.w), static_cast<float*>(a.workspace), (int64_t)a.B * a.N * a.Lq * a.H};
  f.c1 = kLog2e / sqrtf((float)a.D);
  f.fmt = a.dtype == MF_BF16 ? 1u : 0u;
  f.status = status_word();
  MF_REQUIRE(f.status, MF_ERR_CUDA, "could not allocate the device status word");
  MF_REQUIRE(tc_async_status() == 0, MF_ERR_CUDA, "an earlier tensor-core kernel gave up on a bounded wait; results are invalid");
  const int64_t grid = (int64_t)f.n_qt * f.groups * f.sp.splits;
  MF_REQUIRE((int64_t)a.B * a.N * a.H <= 0x7fffffff && grid <= 0x7fffffff, MF_ERR_UNSUPPORTED, "%lld tiles of 128 queries are more than one launch takes", (long long)grid);
  constexpr auto kern = window_fwd_tc_kernel<DP, T>;
  if (int e = opt_in_smem<kern>(C::SMEM)) return e;
  kern<<<(unsigned)grid, kThreads, C::SMEM, st>>>(mq, mk, mv, f);
  MF_LAUNCHED("window_fwd_tc_kernel");
  return f.sp.splits > 1 ? window_split_join(f.w, a.dtype, f.sp, st) : MF_OK;
}
template <typename T>
int by_size(const mf_window_args& a, cudaStream_t st) {
  return a.D <= 32 ? launch<32, T>(a, st) : a.D <= 64 ? launch<64, T>(a, st) : launch<128, T>(a, st);
}
}  // namespace

bool window_tc_supported(const mf_window_args& a) {
  return !(a.flags & MF_FLAG_FORCE_SIMT) && (a.dtype == MF_BF16 || a.dtype == MF_F16) && a.D % 8 == 0 && operand_ok(a.q, a.q_strides, a.B, a.N, a.Lq, a.H) &&
         operand_ok(a.k, a.k_strides, a.B, a.N, a.Lk, a.Hk) && operand_ok(a.v, a.v_strides, a.B, a.N, a.Lk, a.Hk);
}
}  // namespace win

bool window_fwd_tc_supported(const mf_window_args& a) { return win::window_tc_supported(a) && ((uintptr_t)a.o & 15) == 0; }
size_t window_fwd_tc_workspace(const mf_window_args& a) {
  const win::WinP p = win::window_params(a);
  return win::split_bytes(p, win::tc_splits(p));
}
int window_fwd_tc(const mf_window_args& a, cudaStream_t st) {
  return a.dtype == MF_BF16 ? win::by_size<__nv_bfloat16>(a, st) : win::by_size<__half>(a, st);
}

}  // namespace mf
