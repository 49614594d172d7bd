// Gradients of cross attention (h3b_cross_attention_bwd) on tcgen05.
//
//   P = 2^(scale log2e S - lse log2e),  delta_i = do_i . o_i
//   dP = dO V^T,  dS = P (dP - delta)
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO   (a key head's query heads summed)
//
// Two kernels, each the owner of what it sums, so no sum crosses CTAs through
// atomics and the result does not depend on scheduling:
//   xattn_dq_kernel   a unit is 128 query rows of one head; it runs over the
//                     key tiles (three products a tile).
//   xattn_dkv_kernel  a unit is 128 keys of one key head and a range of the
//                     query tiles of all heads that share it (four products a
//                     tile), in the transposed form: TMEM lanes are keys.
//                     Ranges exist because an encoder's keys are few (512 keys
//                     x 24 heads are 96 units for 148 SMs); their fp32 sums
//                     are joined in order by xattn_dkv_join_kernel.
// That is seven products where five would do if dQ were summed across key
// tiles in memory; the five-product form needs fp32 atomics on dQ (one 64 KB
// tile per 128 x 128 block) or a cluster exchange of them.
// P and dS go back to TMEM as 16-bit values and are the A operands; Q, dO and
// K tiles are read from shared memory both ways (K-major for S and dP,
// MN-major for the sums) through two descriptors of the same bytes.
// Work of a 128 x 128 block on the other pipes: 16384 exponentials and ~10
// fp32 operations a value, two warpgroups of 64 columns each.  (Four of 32
// columns: dq 182 -> 201 us, dk and dv 190 -> 200.)
// 24 heads of 128, bf16, 16384 queries x 512 keys: delta 36 us (memory), dq 182,
// dk and dv 190, join 7.  Both large kernels wait on their chains: of a block's
// 3500 cycles in the second, 2048 are products, because TMEM holds one S^T and
// one dP^T beside the sums (128 x 512 columns are full).
// In f16, P is held times 2^8 (P <= 1), which lowers the point where small
// weights lose bits.  dS has the size of the caller's gradients, which may be
// anything, so it is held times a power of two, of its row in dq, of its sample
// and key head in dk (whose sums run over the rows), which the fp32 result is
// divided by: |dP - delta| <= 2 |do| |v|, and the factor brings that bound to
// 2^14 .. 2^15.  Without it do ~ 1e-4 lost 1 % of dq and dk over 1024 keys in
// f16's smallest numbers, several thousands passed its largest, and left-out
// keys (dS = -delta P in dq, see warp 10) made infinities, so NaN, of delta
// above 65504.  (In dk, rows whose |do| is below some 1e-4 of the largest of
// their key head still lose bits, in sums that the others mostly make.)  The
// norms cost a pass over do (delta's, where that is taken) and one over v: 2 x
// 2049 x 1025, 24 heads on 6 of 128, 5 us and a launch (330 -> 341 with the
// forward); 16384 x 77, 24 heads of 128, 32 us of 226.
#include "h3b_common.cuh"
#include "h3b_host.hpp"
#include "xattn.hpp"

H3B_DECLARE_STATUS();
H3B_REGISTER_STATUS_READER(xattn_bwd);

namespace {

using h3b::XAttnGrad;

constexpr int THREADS = 384;  // two compute warpgroups; TMA, MMA, statistics, idle
constexpr int REGS_LAUNCH = 168;
constexpr int REGS_CONTROL = 88;
constexpr int REGS_COMPUTE = 208;
static_assert(128 * (REGS_CONTROL + 2 * REGS_COMPUTE) <= THREADS * REGS_LAUNCH, "register split exceeds launch");
constexpr float LOG2E = 1.4426950408889634f;

template <int D>
struct Cfg {
  static constexpr int HALVES = D / 64;
  static constexpr int TILE_BYTES = 128 * D * 2;
  static constexpr int HALF_BYTES = 128 * 64 * 2;
};

H3B_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The smaller of two, NaN if one is.
H3B_DEV float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

template <bool SPIN = false>
H3B_DEV bool warp_wait(uint64_t* bar, uint32_t parity, int site, volatile int* abort_flag) {
  const bool ok = mbar_wait<SPIN, false, true>(bar, parity, &g_status, site, abort_flag);
  return __all_sync(0xffffffffu, ok);
}

// The tiles need 1024-byte alignment; the same answer for the whole CTA,
// before it has started anything.
H3B_DEV bool misaligned(const uint8_t* smem) {
  if ((smem_u32(smem) & 1023u) == 0) return false;
  if (threadIdx.x == 0 && atomicCAS(&g_status.code, 0, H3B_ERR_DEVICE) == 0) g_status.site = 30;
  return true;
}

// log2-domain row statistic; a row without kept keys (-inf) gives +inf, so
// that all its weights are 2^-inf = 0.
H3B_DEV float lse2_of(float lse) { return lse == -INFINITY ? INFINITY : lse * LOG2E; }

// Products of one 128-row tile: D (+)= A B^T with both operands K-major in
// shared memory (contraction over the head dim), and D (+)= A B with A in
// TMEM (two pieces of 64 columns' worth, at a0 and a1) and B MN-major.
template <int D>
H3B_DEV void issue_ss(uint32_t d, uint32_t a_s, uint32_t b_s, uint32_t idesc) {
  const uint64_t ad = sdesc_kmajor_sw128(a_s), bd = sdesc_kmajor_sw128(b_s);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const uint32_t at = static_cast<uint32_t>((kk >> 2) * (Cfg<D>::HALF_BYTES >> 4) + (kk & 3) * 2);
    mma_f16_ss(d, desc_add_lo(ad, at), desc_add_lo(bd, at), idesc, kk > 0);
  }
}
template <int D>
H3B_DEV void issue_ts_half(uint32_t d, uint32_t a_tmem, uint32_t b_s, int half, uint32_t idesc, bool fresh) {
  const uint64_t bd = sdesc_mnmajor_sw128(b_s, Cfg<D>::HALF_BYTES, 1024);
#pragma unroll
  for (int kk = 0; kk < 4; ++kk)
    mma_f16_ts(d, a_tmem + kk * 8, desc_add_lo(bd, static_cast<uint32_t>((4 * half + kk) * (2048 >> 4))), idesc,
               (fresh && kk == 0) ? 0u : 1u);
}

// The power of two that f16 dS is held times, from |do|^2 |v|^2 (see the top of
// the file): 2^14 / (|do| |v|), rounded down by at most 2.  (0 gives 2^77, and
// dS is 0 then; infinities and NaN give 2^-51 and stay.)
H3B_DEV float ds_factor(float sq) {
  const int e = static_cast<int>((__float_as_uint(sq) >> 23) & 0xffu) - 127;  // sq < 2^(e + 1)
  return __uint_as_float(static_cast<uint32_t>(127 + 14 - ((e + 2) >> 1)) << 23);
}
H3B_DEV float inverse_of_power(float p) { return __uint_as_float((254u << 23) - __float_as_uint(p)); }

struct GradArgs {
  XAttnGrad a;
  int q_tiles;   // of 128 rows
  int k_tiles;   // of 128 keys
  int group;
  int units;
  int step_q, step_head, step_b;  // gridDim.x units of the dq kernel further, digit by digit
  float scale_log2;
};

// Kept-key words of a tile (see xattn_tile.cu).
H3B_DEV uint32_t mask_bytes(const XAttnGrad& a, int b, int key0, int len, int lane) {
  uint32_t m = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int key = key0 + c * 32 + lane;
    if (key < len && __ldg(a.key_mask + b * a.mask_stride + key) != 0) m |= 1u << c;
  }
  return m;
}
H3B_DEV void keep_words(bool masked, uint32_t bytes, int valid, uint32_t (&w)[4]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int v = valid - 32 * c;
    w[c] = v >= 32 ? 0xffffffffu : (v <= 0 ? 0u : (1u << v) - 1u);
    if (masked) w[c] = __ballot_sync(0xffffffffu, (bytes >> c) & 1u);
  }
}
H3B_DEV int len_of(const XAttnGrad& a, int b) {
  return a.kv_lens == nullptr ? a.s_kv : max(0, min(a.s_kv, __ldg(a.kv_lens + b)));
}

// ============================================================== dQ (and delta)
// TMEM: SA | SB | dP | dQ.  S of tile j goes to SA or SB by turns, dS(j) over
// it.  Issue order: dP(j+1) when dP(j) has been read; dQ += dS(j) K(j); S(j+2)
// over dS(j).  So S is two tiles ahead and dP one, and the compute warps find
// both when they come to a tile.  (With S one tile ahead, K in a ring of two
// and the walk over the units in the issuing warp a tile took 8000 cycles,
// its products 1536: the next K was loaded only after dQ.)
// Warp 10 walks the units ahead of the issuing warp: what tile j is of its
// unit, and that K, V and Q are there; it zeroes the left-out rows of K and V.
constexpr int KST = 3, VST = 2;
constexpr int INFOS = 4;  // entry j + 4 is written after dQ(j + 1), so after entry j has been read
enum : uint32_t { T_FIRST = 1, T_LAST = 2, T_END = 4 };

struct __align__(16) DqBars {
  uint32_t flags[INFOS];  // T_* of a tile
  uint64_t ready[INFOS];
  uint64_t x_full[2], x_free[2];  // Q, dO
  uint64_t k_full[KST], k_free[KST];
  uint64_t v_full[VST], v_free[VST];
  uint64_t s_full[2];   // by step parity
  uint64_t dp_full;
  uint64_t dp_free;     // 8 warps have read dP
  // [step parity][warpgroup], 4 warps each.  By parity, because S and dP run
  // a tile ahead of dQ: a fast warp may deliver tile j + 1 before a slow one
  // of its warpgroup has delivered tile j (but not j + 2, which waits for dQ(j)).
  uint64_t ds_half[2][2];
  uint64_t dq_full;
  uint64_t delta_ready; // 8 warps
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
};

// No slack for alignment: seven tiles and the statistics fill the shared
// memory, whose start is aligned (checked by the kernels).
template <int D>
constexpr size_t dq_smem() {
  return (2 + KST + VST) * Cfg<D>::TILE_BYTES + 2 * 256 * sizeof(float) + sizeof(DqBars);
}

static_assert(dq_smem<128>() <= 232448, "shared memory of a CTA");

// The units of one CTA (sample, head, 128 rows; rows fastest), the digits
// carried from unit to unit.  WARP: called by whole warps (the reduction makes
// the length uniform for the compiler).
struct DqUnit {
  int x, qt, head, b;
  int q0, len, n;

  template <bool WARP>
  H3B_DEV void settle(const GradArgs& args) {
    q0 = qt * 128;
    len = args.a.s_kv;
    if (args.a.kv_lens != nullptr && x < args.units) {
      len = len_of(args.a, b);
      if constexpr (WARP) len = __reduce_max_sync(0xffffffffu, len);
    }
    n = (len + 127) / 128;
  }
  H3B_DEV void first(const GradArgs& args) {
    x = blockIdx.x;
    qt = x % args.q_tiles;
    const int u = x / args.q_tiles;
    head = u % args.a.heads;
    b = u / args.a.heads;
    settle<true>(args);
  }
  template <bool WARP = true>
  H3B_DEV void next(const GradArgs& args) {
    x += gridDim.x;
    qt += args.step_q;
    head += args.step_head;
    b += args.step_b;
    if (qt >= args.q_tiles) qt -= args.q_tiles, ++head;
    if (head >= args.a.heads) head -= args.a.heads, ++b;
    settle<WARP>(args);
  }
};

template <int D, bool F16>
__global__ void __launch_bounds__(THREADS, 1)
    xattn_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                    const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ GradArgs args) {
  using C = Cfg<D>;
  constexpr uint32_t IDESC_S = F16 ? idesc_f16_f32(128, 128, 0, 0) : idesc_bf16_f32(128, 128, 0, 0);
  constexpr uint32_t IDESC_G = F16 ? idesc_f16_f32(128, D, 0, 1) : idesc_bf16_f32(128, D, 0, 1);
  extern __shared__ __align__(1024) uint8_t smem_tiles[];
  uint8_t* smem = smem_tiles;
  if (misaligned(smem)) return;
  uint8_t* sX = smem;  // Q | dO
  uint8_t* sK = sX + 2 * C::TILE_BYTES;
  uint8_t* sV = sK + KST * C::TILE_BYTES;
  float* s_delta = reinterpret_cast<float*>(sV + VST * C::TILE_BYTES);  // [unit parity][256]
  DqBars* bars = reinterpret_cast<DqBars*>(s_delta + 2 * 256);
  const XAttnGrad& a = args.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &bars->abort_flag;
  const bool masked = a.key_mask != nullptr;

  if (threadIdx.x == 0) {
    for (int i = 0; i < INFOS; ++i) mbar_init(&bars->ready[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bars->x_full[i], 1), mbar_init(&bars->x_free[i], 1);
    for (int i = 0; i < KST; ++i) mbar_init(&bars->k_full[i], 1), mbar_init(&bars->k_free[i], 1);
    for (int i = 0; i < VST; ++i) mbar_init(&bars->v_full[i], 1), mbar_init(&bars->v_free[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->ds_half[i][0], 4);
      mbar_init(&bars->ds_half[i][1], 4);
    }
    mbar_init(&bars->dp_full, 1);
    mbar_init(&bars->dp_free, 8);
    mbar_init(&bars->dq_full, 1);
    mbar_init(&bars->delta_ready, 8);
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // all 512 columns are this CTA's (a constant keeps operands in uniform registers)
  if (bars->tmem_base != 0) {   // (cannot happen; the same for the whole CTA)
    if (threadIdx.x == 0 && atomicCAS(&g_status.code, 0, H3B_ERR_DEVICE) == 0) g_status.site = 31;
    if (warp == 9) tmem_dealloc(bars->tmem_base, 512);
    return;
  }
  constexpr uint32_t DP_COL = 256, DQ_COL = 384;
  DqUnit u;  // each role walks the CTA's units on its own
  u.first(args);

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CONTROL));
    if (warp == 8 && lane == 0) {
      // ---------------------------------------------------------- TMA
      // A slot's free barrier completed phase (c / ring) - 1 when the tile
      // before it was read, and its next phase needs this load.
      prefetch_tmap(&tm_q);
      prefetch_tmap(&tm_do);
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
      int xc = 0, t = 0, loaded = 0;
      bool ok = true;
      // c-th tile of a ring of `stages`
      auto load = [&](const CUtensorMap* tm, uint8_t* ring, uint64_t* full, uint64_t* free_, int stages, int c, int row,
                      int head, int b) {
        const int s = c % stages;
        if (c >= stages && !mbar_wait<false, false, true>(&free_[s], (c / stages - 1) & 1, &g_status, 1, abort_flag))
          return false;
        mbar_arrive_expect_tx(&full[s], C::TILE_BYTES);
        for (int h = 0; h < C::HALVES; ++h)
          tma_load_4d(ring + s * C::TILE_BYTES + h * C::HALF_BYTES, tm, h * 64, row, head, b, &full[s]);
        return true;
      };
#pragma unroll 1
      for (; u.x < args.units && ok; u.next<false>(args)) {
        const int kvh = args.group == 1 ? u.head : u.head / args.group;
#pragma unroll 1
        for (int j = 0; j < u.n && ok; ++j, ++t) {
          // (Q and dO: rings of one, so the c-th use is the unit's)
          if (j == 0) ok = load(&tm_q, sX, &bars->x_full[0], &bars->x_free[0], 1, xc, u.q0, u.head, u.b);
          if (ok && (ok = load(&tm_k, sK, bars->k_full, bars->k_free, KST, t, j * 128, kvh, u.b))) loaded = 2 * t + 1;
          if (ok && j == 0) {
            ok = load(&tm_do, sX + C::TILE_BYTES, &bars->x_full[1], &bars->x_free[1], 1, xc, u.q0, u.head, u.b);
            ++xc;
          }
          if (ok && (ok = load(&tm_v, sV, bars->v_full, bars->v_free, VST, t, j * 128, kvh, u.b))) loaded = 2 * t + 2;
        }
      }
      if (!ok || *abort_flag) {
        // let the copies in flight land (bounded) before the CTA goes
        for (int c = max(0, (loaded + 1) / 2 - KST); c < (loaded + 1) / 2; ++c)
          mbar_wait<false, false, true>(&bars->k_full[c % KST], (c / KST) & 1, &g_status, 11, nullptr);
        for (int c = max(0, loaded / 2 - VST); c < loaded / 2; ++c)
          mbar_wait<false, false, true>(&bars->v_full[c % VST], (c / VST) & 1, &g_status, 12, nullptr);
        for (int i = 0; i < 2; ++i)
          if (xc > 0) mbar_wait<false, false, true>(&bars->x_full[i], (xc - 1) & 1, &g_status, 10, nullptr);
      }
    } else if (warp == 9) {
      // ---------------------------------------------------------- MMA
      // The warp runs the schedule converged: all lanes poll, one elected lane
      // issues.  Every barrier waited on here completes once per use and its
      // next use depends on what this warp issues after the wait.
      bool ok = true;
      uint32_t uc = 0;  // units whose dO has been waited for
      auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
        ok = mbar_wait<true, false, true>(bar, parity, &g_status, site, abort_flag) && ok;
      };
      auto next_tile = [&](int j) -> uint32_t {  // flags of tile j, once it is there
        wait(&bars->ready[j % INFOS], (j / INFOS) & 1, 4);
        const uint32_t f = ok ? *const_cast<volatile uint32_t*>(&bars->flags[j % INFOS]) : static_cast<uint32_t>(T_END);
        return __reduce_or_sync(0xffffffffu, f);
      };
      auto issue_s = [&](int j, uint32_t f) {
        __syncwarp();
        tc_fence_after();
        if (elect_one()) {
          issue_ss<D>(tmem + (j & 1) * 128, smem_u32(sX), smem_u32(sK + (j % KST) * C::TILE_BYTES), IDESC_S);
          tc_commit(&bars->s_full[j & 1]);
          if (f & T_LAST) tc_commit(&bars->x_free[0]);
        }
        __syncwarp();
      };
      auto issue_dp = [&](int j, uint32_t f) {
        if (f & T_FIRST) {
          wait(&bars->x_full[1], uc & 1, 5);
          ++uc;
        }
        // dP(j - 1) has been read: the barrier's next phase follows this dP
        if (j > 0) wait(&bars->dp_free, (j - 1) & 1, 7);
        __syncwarp();
        tc_fence_after();
        if (elect_one()) {
          issue_ss<D>(tmem + DP_COL, smem_u32(sX + C::TILE_BYTES), smem_u32(sV + (j % VST) * C::TILE_BYTES), IDESC_S);
          tc_commit(&bars->dp_full);
          tc_commit(&bars->v_free[j % VST]);
          if (f & T_LAST) tc_commit(&bars->x_free[1]);
        }
        __syncwarp();
      };
      uint32_t f0 = next_tile(0), f1 = T_END, f2;  // tiles j, j + 1, j + 2
      if (!(f0 & T_END)) {
        issue_s(0, f0);
        issue_dp(0, f0);
        f1 = next_tile(1);
        if (!(f1 & T_END)) issue_s(1, f1);
      }
#pragma unroll 1
      for (int j = 0; !(f0 & T_END); ++j) {
        if (!(f1 & T_END)) issue_dp(j + 1, f1);
        // dQ (+)= dS K, the first of a unit after both warpgroups are past
        // the last unit's stores of it
        uint64_t* ds = bars->ds_half[j & 1];
        wait(&ds[0], (j >> 1) & 1, 8);
        wait(&ds[1], (j >> 1) & 1, 8);
        __syncwarp();
        tc_fence_after();
        if (elect_one()) {
          const uint32_t k_s = smem_u32(sK + (j % KST) * C::TILE_BYTES);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            issue_ts_half<D>(tmem + DQ_COL, tmem + (j & 1) * 128 + h * 64, k_s, h, IDESC_G, (f0 & T_FIRST) != 0 && h == 0);
          tc_commit(&bars->k_free[j % KST]);
          if (f0 & T_LAST) tc_commit(&bars->dq_full);
        }
        __syncwarp();
        f2 = T_END;
        if (!(f1 & T_END)) {
          f2 = next_tile(j + 2);
          if (!(f2 & T_END)) issue_s(j + 2, f2);
        }
        if (!__all_sync(0xffffffffu, ok)) break;
        f0 = f1;
        f1 = f2;
      }
      if (elect_one()) tc_commit(&bars->drain);
      __syncwarp();
      warp_wait(&bars->drain, 0, 9, nullptr);
    } else if (warp == 10) {
      // ---------------------------------------------------------- tiles
      // Ahead of the issuing warp by the K ring; every barrier is waited for
      // once per use, so the parity waits are one phase behind.
      bool ok = true;
      int t = 0;
      uint32_t uc = 0;
#pragma unroll 1
      for (; u.x < args.units && ok; u.next(args)) {
#pragma unroll 1
        for (int j = 0; j < u.n; ++j, ++t) {
          const int key0 = j * 128;
          const uint32_t mb = masked ? mask_bytes(a, u.b, key0, u.len, lane) : 0u;
          ok = (j > 0 || warp_wait(&bars->x_full[0], uc & 1, 3, abort_flag)) &&
               warp_wait(&bars->k_full[t % KST], (t / KST) & 1, 14, abort_flag) &&
               warp_wait(&bars->v_full[t % VST], (t / VST) & 1, 15, abort_flag);
          if (!ok) break;
          uint32_t w[4];
          keep_words(masked, mb, u.len - key0, w);
          if ((w[0] & w[1] & w[2] & w[3]) != ~0u) {
            // Left-out rows of K and V are zeroed: S and dP are 0 there, so P
            // is held to 1, dS to delta (f16: and its factor), both finite,
            // and dS K adds nothing.
            zero_left_out<C::HALVES>(smem_u32(sK + (t % KST) * C::TILE_BYTES), w, lane);
            zero_left_out<C::HALVES>(smem_u32(sV + (t % VST) * C::TILE_BYTES), w, lane);
            fence_proxy_async_smem();
          }
          if (lane == 0)
            *const_cast<volatile uint32_t*>(&bars->flags[t % INFOS]) = (j == 0 ? T_FIRST : 0u) | (j == u.n - 1 ? T_LAST : 0u);
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->ready[t % INFOS]);
        }
        if (u.n > 0) ++uc;
      }
      if (ok) {
        // entry t - INFOS has been read by all: this wait ends after dQ(t - INFOS)
        if (t >= INFOS) ok = warp_wait(&bars->k_free[(t - INFOS) % KST], ((t - INFOS) / KST) & 1, 16, abort_flag);
        if (lane == 0 && ok) {
          *const_cast<volatile uint32_t*>(&bars->flags[t % INFOS]) = T_END;
          mbar_arrive(&bars->ready[t % INFOS]);
        }
      }
    }
  } else {
    // ------------------------------------------------------------ compute
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_COMPUTE));
    const int wg = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    uint32_t step = 0, dc = 0, qc = 0;
    bool ok = true;
    float lse_next = -INFINITY, delta_next = 0.0f, sq_next = 0.0f;
    auto fetch = [&](const DqUnit& v) {
      const int r = v.q0 + row;
      lse_next = -INFINITY;
      delta_next = sq_next = 0.0f;
      if (v.x < args.units && r < a.s_q) {
        const int64_t at = (static_cast<int64_t>(v.b) * a.heads + v.head) * a.s_q + r;
        lse_next = __ldg(a.lse + at);
        if (args.k_tiles > 1) delta_next = a.delta[at];
        if (F16 && args.k_tiles > 0)
          sq_next = a.do_sq[at] * a.v_sq[v.b * a.kv_heads + (args.group == 1 ? v.head : v.head / args.group)];
      }
    };
    fetch(u);
#pragma unroll 1
    for (; u.x < args.units && ok; u.next(args)) {
      const int q_row = u.q0 + row;
      const int64_t stat = (static_cast<int64_t>(u.b) * a.heads + u.head) * a.s_q;
      // The rows' statistics, fetched a unit ahead.
      const float neg_lse2 = -lse2_of(lse_next);
      float delta = delta_next;
      const float factor = F16 ? ds_factor(sq_next) : 1.0f;
      {
        DqUnit v = u;
        v.next(args);
        fetch(v);
      }
#pragma unroll 1
      for (int j = 0; j < u.n; ++j, ++step) {
        const uint32_t s_tmem = tmem + (step & 1) * 128 + wg * 64 + lane_off;
        // S of this parity again only after this tile's dS has been read
        if (!warp_wait<true>(&bars->s_full[step & 1], (step >> 1) & 1, 21, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[64], d[64];
        tmem_ld32p(s_tmem, s);
        tmem_ld32p(s_tmem + 32, s + 32);
        tmem_wait_fence<2>(s);
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          const float2 t = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])),
                                make_float2(args.scale_log2, args.scale_log2), make_float2(neg_lse2, neg_lse2));
          // (P <= 1 but for rounding; a left-out key's score of 0 may be far above lse; a NaN stays one)
          s[e] = __float_as_uint(ex2(min_nan(t.x, 0.0f)));
          s[e + 1] = __float_as_uint(ex2(min_nan(t.y, 0.0f)));
        }
        if (!warp_wait<true>(&bars->dp_full, step & 1, 22, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        tmem_ld32p(tmem + DP_COL + wg * 64 + lane_off, d);
        tmem_ld32p(tmem + DP_COL + wg * 64 + lane_off + 32, d + 32);
        tmem_wait_fence<2>(d);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->dp_free);
        if (u.n == 1) {
          // One tile holds all keys: delta = sum_j P_j dP_j, both halves.  With
          // few keys dP is close to delta, and the 16-bit rounding of o would
          // cost dS bits (1.6 to 2.3 times the error of dq and dk at 2 to 26 keys).
          float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int e = 0; e < 64; e += 2)
            acc[(e >> 1) & 1] = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])),
                                     make_float2(__uint_as_float(d[e]), __uint_as_float(d[e + 1])), acc[(e >> 1) & 1]);
          const float2 t = add2(acc[0], acc[1]);
          float* part = s_delta + (dc & 1) * 256;
          part[wg * 128 + row] = t.x + t.y;
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->delta_ready);
          // (completes once a unit of one tile; no warp can be two such units ahead)
          if (!warp_wait(&bars->delta_ready, dc & 1, 24, abort_flag)) {
            ok = false;
            break;
          }
          ++dc;
          delta = part[row] + part[128 + row];
          if (wg == 0 && q_row < a.s_q) a.delta[stat + q_row] = delta;
        }
        const float2 nd = make_float2(-delta * factor, -delta * factor);
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          float2 t = make_float2(__uint_as_float(d[e]), __uint_as_float(d[e + 1]));
          t = F16 ? fma2(t, make_float2(factor, factor), nd) : add2(t, nd);
          t = mul2(t, make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])));
          d[e] = __float_as_uint(t.x);
          d[e + 1] = __float_as_uint(t.y);
        }
#pragma unroll
        for (int e = 0; e < 32; ++e)
          d[e] = pack16x2<F16>(__uint_as_float(d[2 * e]), __uint_as_float(d[2 * e + 1]));
        tmem_st32(s_tmem, *reinterpret_cast<uint32_t(*)[32]>(d));
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->ds_half[step & 1][wg]);
      }
      if (!ok) break;
      // ---- dQ: this warpgroup's D / 2 columns
      if (u.n > 0) {
        if (!warp_wait(&bars->dq_full, qc & 1, 23, abort_flag)) {
          ok = false;
          break;
        }
        ++qc;
        tc_fence_after();
      }
      const float out_scale = F16 ? a.scale * inverse_of_power(factor) : a.scale;
      uint16_t* out = static_cast<uint16_t*>(a.dq) +
                      ((static_cast<int64_t>(u.b) * a.s_q + q_row) * a.heads + u.head) * D + wg * (D / 2);
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        uint32_t r[32];
        if (u.n > 0) {
          tmem_ld32p(tmem + DQ_COL + wg * (D / 2) + c * 32 + lane_off, r);
          tmem_wait_fence<1>(r);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = 0u;
        }
        if (q_row < a.s_q) {
#pragma unroll
          for (int e = 0; e < 32; e += 16) {
            uint32_t v[8];
#pragma unroll
            for (int t = 0; t < 8; ++t)
              v[t] = pack16x2<F16>(__uint_as_float(r[e + 2 * t]) * out_scale, __uint_as_float(r[e + 2 * t + 1]) * out_scale);
            st_global_v8(out + c * 32 + e, v);
          }
        }
        __syncwarp();  // the next tcgen05.ld is for the whole warp
      }
      tc_fence_before();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// delta = do . o of every row, where the keys take more than one tile (DELTA):
// one pass over o and do at memory rate.  (In the dq kernel, at the start of
// each unit, its loads were waited for: 7 us a unit of 128 rows x 512 keys,
// whose tiles take 8.)  In f16 |do|^2 too, and the maxima set to 0 for the
// kernel below.  D / 8 lanes a row.
template <int D, bool F16, bool DELTA>
__global__ void __launch_bounds__(256) xattn_delta_kernel(const __grid_constant__ XAttnGrad a) {
  constexpr int LPR = D / 8;
  constexpr int ROWS = 4;  // a thread's loads in flight
  // (32-bit row numbers: 2^31 rows would be 274 GB of q)
  const uint32_t first = blockIdx.x * (256 / LPR) * ROWS + threadIdx.x / LPR;
  const int col = (threadIdx.x % LPR) * 8;
  const uint32_t rows = static_cast<uint32_t>(a.batch) * a.s_q * a.heads;
  if (F16 && blockIdx.x == 0)
    for (int64_t i = threadIdx.x; i < 2ll * a.batch * a.kv_heads; i += 256) a.v_sq[i] = 0.0f;  // (and do_top)
  uint4 ov[ROWS], gv[ROWS];
  int64_t at[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const uint32_t i = first + k * (256 / LPR);  // (b, token, head)
    at[k] = -1;
    ov[k] = gv[k] = make_uint4(0, 0, 0, 0);
    if (i < rows) {
      const uint32_t bt = i / static_cast<uint32_t>(a.heads);
      const int64_t head = i - bt * a.heads;
      const uint32_t b32 = bt / static_cast<uint32_t>(a.s_q);
      const int64_t b = b32, tok = bt - b32 * a.s_q;
      if constexpr (DELTA)
        ov[k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.o) + b * a.o_stride[0] +
                                                     tok * a.o_stride[1] + head * a.o_stride[2] + col));
      gv[k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.d_o) + b * a.do_stride[0] +
                                                   tok * a.do_stride[1] + head * a.do_stride[2] + col));
      at[k] = (b * a.heads + head) * a.s_q + tok;
    }
  }
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const uint32_t ow[4] = {ov[k].x, ov[k].y, ov[k].z, ov[k].w}, gw[4] = {gv[k].x, gv[k].y, gv[k].z, gv[k].w};
    float s = 0.0f, sq = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (F16) {
        const float2 of = __half22float2(*reinterpret_cast<const __half2*>(&ow[e]));
        const float2 gf = __half22float2(*reinterpret_cast<const __half2*>(&gw[e]));
        s = fmaf(of.x, gf.x, fmaf(of.y, gf.y, s));
        sq = fmaf(gf.x, gf.x, fmaf(gf.y, gf.y, sq));
      } else {
        s = fmaf(bf16lo_to_f32(ow[e]), bf16lo_to_f32(gw[e]), s);
        s = fmaf(bf16hi_to_f32(ow[e]), bf16hi_to_f32(gw[e]), s);
      }
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) {
      if constexpr (DELTA) s += __shfl_xor_sync(0xffffffffu, s, o);
      if constexpr (F16) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    }
    if (at[k] >= 0 && threadIdx.x % LPR == 0) {
      if constexpr (DELTA) a.delta[at[k]] = s;
      if constexpr (F16) a.do_sq[at[k]] = sq;
    }
  }
}

// f16: the largest |v|^2 of a sample's kept keys (the first blocks, NORM_KEYS
// keys of a key head each) and the largest |do|^2 of the rows that share the key
// head (the others, NORM_ROWS rows each).  (As unsigned numbers: a NaN is the
// largest.  The maximum does not depend on the order of the blocks.)
constexpr int NORM_KEYS = 64, NORM_ROWS = 2048;
template <int D>
__global__ void __launch_bounds__(256) xattn_norms_kernel(const __grid_constant__ XAttnGrad a, int key_blocks) {
  constexpr int LPR = D / 8;
  __shared__ uint32_t s_top[8];
  const bool keys = static_cast<int>(blockIdx.x) < key_blocks;
  const int x = keys ? blockIdx.x : blockIdx.x - key_blocks;
  const int rows = a.heads / a.kv_heads * a.s_q;  // the group's heads lie one behind the other
  const int chunks = keys ? (a.s_kv + NORM_KEYS - 1) / NORM_KEYS : (rows + NORM_ROWS - 1) / NORM_ROWS;
  const int chunk = x % chunks, slab = x / chunks;  // slab: (sample, key head)
  const int kvh = slab % a.kv_heads, b = slab / a.kv_heads;
  const int len = len_of(a, b);
  const uint16_t* v = static_cast<const uint16_t*>(a.v) + b * a.kv_stride[0] + kvh * a.kv_stride[2] + (threadIdx.x % LPR) * 8;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NORM_ROWS / 256; ++i) {
    const int row = chunk * NORM_ROWS + i * 256 + static_cast<int>(threadIdx.x);
    if (!keys && row < rows)
      top = max(top, __float_as_uint(a.do_sq[static_cast<int64_t>(slab) * rows + row]) & 0x7fffffffu);
  }
#pragma unroll
  for (int i = 0; i < NORM_KEYS * LPR / 256 && keys; ++i) {
    const int key = chunk * NORM_KEYS + i * (256 / LPR) + static_cast<int>(threadIdx.x) / LPR;
    float sq = 0.0f;
    if (key < len && (a.key_mask == nullptr || __ldg(a.key_mask + b * a.mask_stride + key) != 0)) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(v + key * a.kv_stride[1]));
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
        sq = fmaf(f.x, f.x, fmaf(f.y, f.y, sq));
      }
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    top = max(top, __float_as_uint(sq) & 0x7fffffffu);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) top = max(top, s_top[i]);
    if (top != 0) atomicMax(reinterpret_cast<uint32_t*>(keys ? a.v_sq : a.do_top) + slab, top);
  }
}

// ============================================================== dK and dV
// TMEM lanes are keys: S^T | dP^T | dV | dK.  P^T goes over S^T, dS^T over
// dP^T.  Issue order a tile: dV += P^T(j) dO(j), S^T(j+1); dK += dS^T(j) Q(j), dP^T(j+1).
constexpr int RST = 5;    // ring of Q and dO tiles, by turns
constexpr int STATS = 2;  // ring of the rows' lse and delta

struct __align__(8) DkvBars {
  uint64_t r_full[RST], r_free[RST];
  uint64_t k_full, v_full, k_free, v_free;
  uint64_t stat_full[STATS], stat_free[STATS];
  uint64_t s_full, dp_full;
  uint64_t p_half[2], ds_half[2];
  uint64_t out_full;
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
};

template <int D>
constexpr size_t dkv_smem() {
  return (RST + 2) * Cfg<D>::TILE_BYTES + STATS * 2 * 128 * sizeof(float) + sizeof(DkvBars);
}

static_assert(dkv_smem<128>() <= 232448, "shared memory of a CTA");

// What dP - delta is multiplied by: f16, dS's factor without P's 2^P_SHIFT.
template <bool F16>
H3B_DEV float dp_factor(const XAttnGrad& a, int b, int kvh) {
  if constexpr (!F16) return 1.0f;
  const int64_t at = static_cast<int64_t>(b) * a.kv_heads + kvh;
  return ds_factor(a.v_sq[at] * a.do_top[at]) * 0.00390625f;
}

struct DkvUnit {
  int b, kvh, key0, split, len;
  int t0, n;  // first (head of the group, query tile), tiles
};
H3B_DEV DkvUnit dkv_unit(const GradArgs& args, int u) {
  DkvUnit x;
  x.key0 = (u % args.k_tiles) * 128;  // fastest: units that run together share Q and dO in L2
  u /= args.k_tiles;
  x.split = u % args.a.splits;
  u /= args.a.splits;
  x.kvh = u % args.a.kv_heads;
  x.b = u / args.a.kv_heads;
  x.len = len_of(args.a, x.b);
  const int all = args.group * args.q_tiles;
  const int per = (all + args.a.splits - 1) / args.a.splits;
  x.t0 = x.split * per;
  x.n = x.key0 < x.len ? max(0, min(all, x.t0 + per) - x.t0) : 0;
  return x;
}

template <int D, bool F16>
__global__ void __launch_bounds__(THREADS, 1)
    xattn_dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                     const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ GradArgs args) {
  using C = Cfg<D>;
  constexpr uint32_t IDESC_S = F16 ? idesc_f16_f32(128, 128, 0, 0) : idesc_bf16_f32(128, 128, 0, 0);
  constexpr uint32_t IDESC_G = F16 ? idesc_f16_f32(128, D, 0, 1) : idesc_bf16_f32(128, D, 0, 1);
  constexpr float P_SHIFT = F16 ? 8.0f : 0.0f;             // P held times 2^P_SHIFT
  constexpr float P_UNIT = F16 ? 0.00390625f : 1.0f;       // 2^-P_SHIFT
  extern __shared__ __align__(1024) uint8_t smem_tiles[];
  uint8_t* smem = smem_tiles;
  if (misaligned(smem)) return;
  uint8_t* sR = smem;
  uint8_t* sK = sR + RST * C::TILE_BYTES;
  uint8_t* sV = sK + C::TILE_BYTES;
  float* s_stat = reinterpret_cast<float*>(sV + C::TILE_BYTES);  // [STATS][shift - lse2 | -delta scaled][128]
  DkvBars* bars = reinterpret_cast<DkvBars*>(s_stat + STATS * 2 * 128);
  const XAttnGrad& a = args.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &bars->abort_flag;

  if (threadIdx.x == 0) {
    for (int i = 0; i < RST; ++i) mbar_init(&bars->r_full[i], 1), mbar_init(&bars->r_free[i], 1);
    for (int i = 0; i < STATS; ++i) mbar_init(&bars->stat_full[i], 1), mbar_init(&bars->stat_free[i], 8);
    mbar_init(&bars->k_full, 1);
    mbar_init(&bars->v_full, 1);
    mbar_init(&bars->k_free, 1);
    mbar_init(&bars->v_free, 1);
    mbar_init(&bars->s_full, 1);
    mbar_init(&bars->dp_full, 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bars->p_half[i], 4), mbar_init(&bars->ds_half[i], 4);
    mbar_init(&bars->out_full, 1);
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  constexpr uint32_t DP_COL = 128, DV_COL = 256, DK_COL = 384;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CONTROL));
    if (warp == 8 && lane == 0) {
      // ---------------------------------------------------------- TMA
      prefetch_tmap(&tm_q);
      prefetch_tmap(&tm_do);
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
      int rc = 0, uc = 0;
      bool ok = true;
      auto tile = [&](const CUtensorMap* tm, uint8_t* dst, uint64_t* full, int row, int head, int b) {
        mbar_arrive_expect_tx(full, C::TILE_BYTES);
        for (int h = 0; h < C::HALVES; ++h) tma_load_4d(dst + h * C::HALF_BYTES, tm, h * 64, row, head, b, full);
      };
      auto load_r = [&](const CUtensorMap* tm, int row, int head, int b) {
        const int s = rc % RST;
        if (rc >= RST && !mbar_wait<false, false, true>(&bars->r_free[s], (rc / RST - 1) & 1, &g_status, 1, abort_flag)) return false;
        tile(tm, sR + s * C::TILE_BYTES, &bars->r_full[s], row, head, b);
        ++rc;
        return true;
      };
      for (int x = blockIdx.x; x < args.units && ok; x += gridDim.x) {
        const DkvUnit u = dkv_unit(args, x);
        if (u.n == 0) continue;
        // K and V are held for the unit; the unit before releases them (one
        // phase a unit)
        if (uc > 0 && !mbar_wait<false, false, true>(&bars->k_free, (uc - 1) & 1, &g_status, 2, abort_flag)) ok = false;
        if (ok) tile(&tm_k, sK, &bars->k_full, u.key0, u.kvh, u.b);
        for (int i = 0; i < u.n && ok; ++i) {
          const int head = u.kvh * args.group + (u.t0 + i) / args.q_tiles;
          const int q0 = ((u.t0 + i) % args.q_tiles) * 128;
          ok = load_r(&tm_q, q0, head, u.b);
          if (ok && i == 0) {
            if (uc > 0 && !mbar_wait<false, false, true>(&bars->v_free, (uc - 1) & 1, &g_status, 3, abort_flag)) ok = false;
            if (ok) {
              tile(&tm_v, sV, &bars->v_full, u.key0, u.kvh, u.b);
              ++uc;
            }
          }
          ok = ok && load_r(&tm_do, q0, head, u.b);
        }
      }
      if (!ok || *abort_flag) {
        for (int c = max(0, rc - RST); c < rc; ++c)
          mbar_wait<false, false, true>(&bars->r_full[c % RST], (c / RST) & 1, &g_status, 10, nullptr);
        if (uc > 0) {
          mbar_wait<false, false, true>(&bars->k_full, (uc - 1) & 1, &g_status, 11, nullptr);
          mbar_wait<false, false, true>(&bars->v_full, (uc - 1) & 1, &g_status, 12, nullptr);
        }
      }
    } else if (warp == 9) {
      // ---------------------------------------------------------- MMA
      bool ok = true;
      int step = 0, uc = 0;
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) tc_commit(bar);
        __syncwarp();
      };
      auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
        if (!warp_wait<true>(bar, parity, site, abort_flag)) return false;
        tc_fence_after();
        return true;
      };
      auto ring = [&](int c) { return smem_u32(sR + (c % RST) * C::TILE_BYTES); };
      auto issue_s = [&](int t) -> bool {  // S^T(t) = K Q^T
        if (!wait(&bars->r_full[(2 * t) % RST], (2 * t / RST) & 1, 4)) return false;
        if (elect_one()) {
          issue_ss<D>(tmem, smem_u32(sK), ring(2 * t), IDESC_S);
          tc_commit(&bars->s_full);
        }
        __syncwarp();
        return true;
      };
      auto issue_dp = [&](int t) -> bool {  // dP^T(t) = V dO^T
        if (!wait(&bars->r_full[(2 * t + 1) % RST], ((2 * t + 1) / RST) & 1, 5)) return false;
        if (elect_one()) {
          issue_ss<D>(tmem + DP_COL, smem_u32(sV), ring(2 * t + 1), IDESC_S);
          tc_commit(&bars->dp_full);
        }
        __syncwarp();
        return true;
      };
      for (int x = blockIdx.x; x < args.units && ok; x += gridDim.x) {
        const DkvUnit u = dkv_unit(args, x);
        if (u.n == 0) continue;
        ok = wait(&bars->k_full, uc & 1, 6) && issue_s(step) && wait(&bars->v_full, uc & 1, 7) && issue_dp(step);
        for (int i = 0; i < u.n && ok; ++i, ++step) {
          const bool last = i == u.n - 1;
          for (int h = 0; h < 2 && ok; ++h) {  // dV += P^T dO
            ok = wait(&bars->p_half[h], step & 1, 8);
            if (ok && elect_one())
              issue_ts_half<D>(tmem + DV_COL, tmem + h * 64, ring(2 * step + 1), h, IDESC_G, i == 0 && h == 0);
            __syncwarp();
          }
          if (!ok) break;
          commit(&bars->r_free[(2 * step + 1) % RST]);
          if (last) {
            commit(&bars->k_free);  // every S^T of the unit is behind this
          } else {
            ok = issue_s(step + 1);
          }
          for (int h = 0; h < 2 && ok; ++h) {  // dK += dS^T Q
            ok = wait(&bars->ds_half[h], step & 1, 9);
            if (ok && elect_one())
              issue_ts_half<D>(tmem + DK_COL, tmem + DP_COL + h * 64, ring(2 * step), h, IDESC_G, i == 0 && h == 0);
            __syncwarp();
          }
          if (!ok) break;
          commit(&bars->r_free[(2 * step) % RST]);
          if (last) {
            commit(&bars->v_free);
            commit(&bars->out_full);
          } else {
            ok = issue_dp(step + 1);
          }
        }
        ++uc;
      }
      commit(&bars->drain);
      warp_wait(&bars->drain, 0, 13, nullptr);
    } else if (warp == 10) {
      // ---------------------------------------------------------- row statistics
      int step = 0;
      bool ok = true;
      for (int x = blockIdx.x; x < args.units && ok; x += gridDim.x) {
        const DkvUnit u = dkv_unit(args, x);
        const float factor = dp_factor<F16>(a, u.b, u.kvh);
        for (int i = 0; i < u.n; ++i, ++step) {
          const int head = u.kvh * args.group + (u.t0 + i) / args.q_tiles;
          const int q0 = ((u.t0 + i) % args.q_tiles) * 128;
          const int64_t at = (static_cast<int64_t>(u.b) * a.heads + head) * a.s_q;
          float lse[4], del[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int r = q0 + c * 32 + lane;
            const bool in = r < a.s_q;
            lse[c] = in ? P_SHIFT - lse2_of(__ldg(a.lse + at + r)) : -INFINITY;
            del[c] = in ? -a.delta[at + r] * factor : 0.0f;
          }
          const int s = step % STATS;
          if (step >= STATS && !warp_wait(&bars->stat_free[s], (step / STATS - 1) & 1, 14, abort_flag)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s_stat[s * 256 + c * 32 + lane] = lse[c];
            s_stat[s * 256 + 128 + c * 32 + lane] = del[c];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->stat_full[s]);
        }
      }
    }
  } else {
    // ------------------------------------------------------------ compute
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_COMPUTE));
    const int wg = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + wg * 64 + lane_off;
    const uint32_t dp_tmem = tmem + DP_COL + wg * 64 + lane_off;
    uint32_t step = 0, oc = 0;
    bool ok = true;
    for (int x = blockIdx.x; x < args.units && ok; x += gridDim.x) {
      const DkvUnit u = dkv_unit(args, x);
      const int key = u.key0 + row;
      const float factor = dp_factor<F16>(a, u.b, u.kvh);
      const bool kept = key < u.len && (a.key_mask == nullptr || __ldg(a.key_mask + u.b * a.mask_stride + key) != 0);
      for (int i = 0; i < u.n; ++i, ++step) {
        const int slot = step % STATS;
        const float4* lse = reinterpret_cast<const float4*>(s_stat + slot * 256 + wg * 64);
        const float4* del = reinterpret_cast<const float4*>(s_stat + slot * 256 + 128 + wg * 64);
        if (!warp_wait(&bars->stat_full[slot], (step / STATS) & 1, 20, abort_flag) ||
            !warp_wait<true>(&bars->s_full, step & 1, 21, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[64], d[64];
        tmem_ld32p(s_tmem, s);
        tmem_ld32p(s_tmem + 32, s + 32);
        tmem_wait_fence<2>(s);
        const float2 sc = make_float2(args.scale_log2, args.scale_log2);
#pragma unroll
        for (int e = 0; e < 64; e += 4) {
          const float4 l = lse[e / 4];
          const float2 t0 = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), sc, make_float2(l.x, l.y));
          const float2 t1 = fma2(make_float2(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3])), sc, make_float2(l.z, l.w));
          s[e] = __float_as_uint(kept ? ex2(t0.x) : 0.0f);
          s[e + 1] = __float_as_uint(kept ? ex2(t0.y) : 0.0f);
          s[e + 2] = __float_as_uint(kept ? ex2(t1.x) : 0.0f);
          s[e + 3] = __float_as_uint(kept ? ex2(t1.y) : 0.0f);
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) d[e] = pack16x2<F16>(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
        tmem_st32(s_tmem, *reinterpret_cast<uint32_t(*)[32]>(d));
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_half[wg]);
        if (!warp_wait<true>(&bars->dp_full, step & 1, 22, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        tmem_ld32p(dp_tmem, d);
        tmem_ld32p(dp_tmem + 32, d + 32);
        tmem_wait_fence<2>(d);
        const float2 pu = make_float2(factor, factor);
#pragma unroll
        for (int e = 0; e < 64; e += 4) {
          const float4 l = del[e / 4];
          float2 t0 = make_float2(__uint_as_float(d[e]), __uint_as_float(d[e + 1]));
          float2 t1 = make_float2(__uint_as_float(d[e + 2]), __uint_as_float(d[e + 3]));
          if constexpr (F16) {
            t0 = fma2(t0, pu, make_float2(l.x, l.y));
            t1 = fma2(t1, pu, make_float2(l.z, l.w));
          } else {
            t0 = add2(t0, make_float2(l.x, l.y));
            t1 = add2(t1, make_float2(l.z, l.w));
          }
          t0 = mul2(t0, make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])));
          t1 = mul2(t1, make_float2(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3])));
          d[e / 2] = kept ? pack16x2<F16>(t0.x, t0.y) : 0u;
          d[e / 2 + 1] = kept ? pack16x2<F16>(t1.x, t1.y) : 0u;
        }
        tmem_st32(dp_tmem, *reinterpret_cast<uint32_t(*)[32]>(d));
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars->ds_half[wg]);
          mbar_arrive(&bars->stat_free[slot]);
        }
      }
      if (!ok) break;
      // ---- warpgroup 0 writes dV, warpgroup 1 dK
      if (u.n > 0) {
        if (!warp_wait(&bars->out_full, oc & 1, 23, abort_flag)) {
          ok = false;
          break;
        }
        ++oc;
        tc_fence_after();
      }
      const float f = wg ? (F16 ? a.scale * inverse_of_power(factor) * P_UNIT : a.scale) : P_UNIT;
      const int64_t key_row = (static_cast<int64_t>(u.b) * a.s_kv + key) * a.kv_heads + u.kvh;
      const int64_t per_split = static_cast<int64_t>(a.batch) * a.s_kv * a.kv_heads;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        if (u.n > 0) {
          tmem_ld32p(tmem + (wg ? DK_COL : DV_COL) + c * 32 + lane_off, r);
          tmem_wait_fence<1>(r);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = 0u;
        }
        if (key < a.s_kv && a.splits > 1) {
          float* dst = a.part + ((wg * static_cast<int64_t>(a.splits) + u.split) * per_split + key_row) * D + c * 32;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t v[8];
#pragma unroll
            for (int t = 0; t < 8; ++t) v[t] = __float_as_uint(__uint_as_float(r[e + t]) * f);
            st_global_v8(dst + e, v);
          }
        } else if (key < a.s_kv) {
          uint16_t* dst = static_cast<uint16_t*>(wg ? a.dk : a.dv) + key_row * D + c * 32;
#pragma unroll
          for (int e = 0; e < 32; e += 16) {
            uint32_t v[8];
#pragma unroll
            for (int t = 0; t < 8; ++t)
              v[t] = pack16x2<F16>(__uint_as_float(r[e + 2 * t]) * f, __uint_as_float(r[e + 2 * t + 1]) * f);
            st_global_v8(dst + e, v);
          }
        }
        __syncwarp();  // the next tcgen05.ld is for the whole warp
      }
      tc_fence_before();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dv (blockIdx.y 0) and dk (1): the ranges' fp32 sums added in order, rounded
// once.  One thread = 8 values.
template <bool F16>
__global__ void __launch_bounds__(256) xattn_dkv_join_kernel(const float* part, uint16_t* dv, uint16_t* dk, int splits,
                                                             int64_t n) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8;
  if (i >= n) return;
  const float* p = part + blockIdx.y * splits * n + i;
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = 0; k < splits; ++k) {
    const float4 x = *reinterpret_cast<const float4*>(p + k * n), y = *reinterpret_cast<const float4*>(p + k * n + 4);
    s[0] += x.x, s[1] += x.y, s[2] += x.z, s[3] += x.w;
    s[4] += y.x, s[5] += y.y, s[6] += y.z, s[7] += y.w;
  }
  *reinterpret_cast<uint4*>((blockIdx.y ? dk : dv) + i) =
      make_uint4(pack16x2<F16>(s[0], s[1]), pack16x2<F16>(s[2], s[3]), pack16x2<F16>(s[4], s[5]), pack16x2<F16>(s[6], s[7]));
}

int encode_tiles(CUtensorMap* m, const void* p, bool f16, int d, const int64_t (&st)[3], int seq, int heads, int batch) {
  const uint64_t dims[4] = {static_cast<uint64_t>(d), static_cast<uint64_t>(seq > 0 ? seq : 1),
                            static_cast<uint64_t>(heads), static_cast<uint64_t>(batch)};
  const uint64_t sb[3] = {static_cast<uint64_t>(st[1]) * 2, static_cast<uint64_t>(st[2]) * 2,
                          static_cast<uint64_t>(st[0]) * 2};
  const uint32_t box[4] = {64, 128, 1, 1};
  return h3b::encode_4d(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p, dims, sb, box,
                        CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int D, bool F16>
int launch(const XAttnGrad& a, cudaStream_t stream) {
  CUtensorMap tq, tdo, tk, tv;
  int rc = encode_tiles(&tq, a.q, F16, D, a.q_stride, a.s_q, a.heads, a.batch);
  if (rc == H3B_OK) rc = encode_tiles(&tdo, a.d_o, F16, D, a.do_stride, a.s_q, a.heads, a.batch);
  if (rc == H3B_OK) rc = encode_tiles(&tk, a.k, F16, D, a.kv_stride, a.s_kv, a.kv_heads, a.batch);
  if (rc == H3B_OK) rc = encode_tiles(&tv, a.v, F16, D, a.kv_stride, a.s_kv, a.kv_heads, a.batch);
  if (rc != H3B_OK) return rc;
  auto dq = xattn_dq_kernel<D, F16>;
  auto dkv = xattn_dkv_kernel<D, F16>;
  static h3b::OncePerDevice attr;
  rc = attr.run(h3b::device(), [=] {
    const int e = h3b::allow_smem(dq, dq_smem<D>());
    return e == H3B_OK ? h3b::allow_smem(dkv, dkv_smem<D>()) : e;
  });
  if (rc != H3B_OK) return rc;
  GradArgs args{};
  args.a = a;
  args.group = a.heads / a.kv_heads;
  args.q_tiles = (a.s_q + 127) / 128;
  args.k_tiles = (a.s_kv + 127) / 128;
  args.scale_log2 = a.scale * LOG2E;
  const int sms = h3b::num_sms();
  const int64_t qu = static_cast<int64_t>(a.batch) * a.heads * args.q_tiles;
  const int64_t ku = static_cast<int64_t>(a.batch) * a.kv_heads * args.k_tiles * a.splits;
  if (qu > 0x3fffffff || ku > 0x3fffffff) return H3B_ERR_SHAPE;
  if (args.k_tiles > 1 || (F16 && args.k_tiles > 0)) {
    const int64_t per = 4 * 256 / (D / 8);  // rows of a block
    const int64_t blocks = (static_cast<int64_t>(a.batch) * a.s_q * a.heads + per - 1) / per;
    if (blocks > 0x7fffffff) return H3B_ERR_SHAPE;
    if (args.k_tiles > 1) {
      xattn_delta_kernel<D, F16, true><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a);
    } else {
      xattn_delta_kernel<D, true, false><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a);
    }
    rc = h3b::launch_status();
    if (rc != H3B_OK) return rc;
  }
  if (F16 && args.k_tiles > 0) {
    const int64_t slabs = static_cast<int64_t>(a.batch) * a.kv_heads, rows = static_cast<int64_t>(args.group) * a.s_q;
    const int64_t key_blocks = slabs * ((a.s_kv + NORM_KEYS - 1) / NORM_KEYS);
    const int64_t blocks = key_blocks + slabs * ((rows + NORM_ROWS - 1) / NORM_ROWS);
    if (blocks > 0x7fffffff) return H3B_ERR_SHAPE;
    xattn_norms_kernel<D><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a, static_cast<int>(key_blocks));
    rc = h3b::launch_status();
    if (rc != H3B_OK) return rc;
  }
  args.units = static_cast<int>(qu);
  int step = static_cast<int>(qu < sms ? qu : sms);
  args.step_q = step % args.q_tiles;
  step /= args.q_tiles;
  args.step_head = step % a.heads;
  args.step_b = step / a.heads;
  dq<<<static_cast<unsigned>(qu < sms ? qu : sms), THREADS, dq_smem<D>(), stream>>>(tq, tdo, tk, tv, args);
  rc = h3b::launch_status();
  if (rc != H3B_OK || ku == 0) return rc;
  args.units = static_cast<int>(ku);
  dkv<<<static_cast<unsigned>(ku < sms ? ku : sms), THREADS, dkv_smem<D>(), stream>>>(tq, tdo, tk, tv, args);
  rc = h3b::launch_status();
  if (rc != H3B_OK || a.splits == 1) return rc;
  const int64_t n = static_cast<int64_t>(a.batch) * a.s_kv * a.kv_heads * D;
  const dim3 grid(static_cast<unsigned>((n / 8 + 255) / 256), 2);
  xattn_dkv_join_kernel<F16><<<grid, 256, 0, stream>>>(a.part, static_cast<uint16_t*>(a.dv),
                                                       static_cast<uint16_t*>(a.dk), a.splits, n);
  return h3b::launch_status();
}

}  // namespace

namespace h3b {

int xattn_bwd_splits(const XAttnGrad& a) {
  // Ranges of the query tiles: rounds of units over the SMs times the tiles
  // of a unit, a unit's own start and end counted as three tiles.
  const int64_t base = static_cast<int64_t>(a.batch) * a.kv_heads * ((a.s_kv + 127) / 128);
  const int64_t tiles = static_cast<int64_t>(a.heads / a.kv_heads) * ((a.s_q + 127) / 128);
  const int sms = num_sms();
  int best = 1;
  double cost = 1e30;
  for (int s = 1; s <= 64 && s <= tiles; ++s) {
    const double c = static_cast<double>((base * s + sms - 1) / sms) *
                     (static_cast<double>((tiles + s - 1) / s) + 3.0 + (s > 1 ? 1.0 : 0.0));
    if (c < cost * 0.98) {
      cost = c;
      best = s;
    }
  }
  return best;
}

int xattn_bwd_launch(const XAttnGrad& a, cudaStream_t stream) {
  if (a.head_dim == 128) return a.dtype == H3B_F16 ? launch<128, true>(a, stream) : launch<128, false>(a, stream);
  return a.dtype == H3B_F16 ? launch<64, true>(a, stream) : launch<64, false>(a, stream);
}

}  // namespace h3b
