// The orthogonal factor of an update matrix, approached by Newton-Schulz
// steps: X <- a X + (b G + c G G) X, G = X X^T, from X = x / (|x| + eps), the
// smaller side first (x of more rows than columns is taken transposed and
// given back so).
//
// A step is three matrix products on tcgen05 (kind::f16, fp32 accumulators in
// TMEM), each with its arithmetic in the epilogue:
//   GRAM  G = X X^T            symmetric: only tiles on or below the diagonal,
//   POLY  B = b G + c G G      stored to both sides
//   MUL   X' = a X + B X       (X is read K-major by GRAM, N-major by MUL)
//
// Precision.  A step multiplies small singular values by a, five steps by
// 480: what a rounding spills from the large directions into the small ones
// grows with them, and one plane of 16-bit operands (2^-12 a rounding) leaves
// 1.4 % of the result wrong for an update dominated by a few directions, bf16
// operands 13 %.  So operands are pairs of f16 planes, v = hi + lo (22 bits),
// and a product is hi hi + lo hi + hi lo in one accumulator (what is left out
// is 2^-22).  That is as near as 32-bit arithmetic comes at a fifth of its
// time on CUDA cores.  Two products are exact or late enough to save on:
// x in 16 bits is one plane as it is (its 8 or 11 bits are kept by a scale of
// a power of two; the norm's fraction goes into the first epilogues), and the
// last step of a bf16 result, after which nothing grows, takes one plane.
// That step is written about G = 1, where X is by then: with H = G - 1,
// X' = (a + b + c) X + ((b + 2c) H + c H H) X, so that what is rounded to 11
// bits is small beside what it is added to.
//
// Planes hold SCALE * value: f16 has its full precision between 2^-24 and 64
// of the value then.  Elements are below the largest singular value, 1.2 for
// coefficients that converge; beyond 64 they become infinite and the result
// NaN.
//
// The tensor cores' sums drop what falls below their last bit at every 16
// elements of K; over a long row that is a bias (2^-25 for each of 768 sums
// at K = 4096: 1e-5 of G's diagonal, 3e-5 of the result).  An accumulator
// therefore takes 128 elements of K, the small products before the large
// ones (512 where a plane of 11 bits decides), and the storing warps add
// accumulators in registers, rounding to nearest.
//
// Tiles: 256 x 256 by CTA pairs (cta_group::2, each CTA stages 128 rows of
// both operands) or, where those are too few for the SMs, 128 x 128 by one
// CTA (its operand reads and copies share the shared-memory port: a tile
// costs 0.8 of the pair's time for half the work).  Warp 0 loads (TMA, zero
// beyond the matrix), warp 1 issues the products, eight warps add and store;
// two accumulators in turn, so that products go on meanwhile.  Every wait is
// bounded.
#include "h3b_common.cuh"
#include "h3b_host.hpp"

H3B_DECLARE_STATUS();
H3B_REGISTER_STATUS_READER(ortho);

namespace {

constexpr float SCALE = 1024.0f;
constexpr int BM = 128;            // accumulator rows of a CTA
constexpr int KB = 64;             // elements of K a stage (128 bytes a row)
constexpr int PLANE_BYTES = BM * 128;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 128 + 32 * EPI_WARPS;  // a warpgroup to load and issue (two of its warps idle), two to store

// Registers a thread: 384 threads launch with 168; the storing warpgroups,
// which hold 128 sums a thread, take over what the first one does not need.
constexpr int LAUNCH_REGS = 168;
constexpr int REGS_CTL = 72;
constexpr int REGS_EPI = 216;
static_assert(4 * REGS_CTL + 8 * REGS_EPI <= 12 * LAUNCH_REGS, "register split exceeds launch");

enum Op { GRAM = 0, POLY = 1, MUL = 2 };

template <int PAIR, int OP, int SPLIT>
struct Cfg {
  static constexpr int BN = 128 * PAIR;
  static constexpr int PLANES = SPLIT ? 2 : 1;
  static constexpr int STAGE_BYTES = 2 * PLANES * PLANE_BYTES;  // A planes, then B planes
  static constexpr int STAGES = SPLIT ? 3 : 6;
  static constexpr int TMEM_COLS = 2 * BN;  // two accumulators
  static constexpr int CHUNK = SPLIT ? 2 : 8;  // stages of K an accumulator takes
  static constexpr uint32_t IDESC = idesc_f16_f32(BM * PAIR, BN, 0, OP == MUL ? 1 : 0);
};

struct Planes {
  __half* hi;
  __half* lo;
};

struct Args {
  int rows, cols, k;       // of the product, per matrix
  int batch;
  int b_lo;                // SPLIT: the B operand has a second plane
  Planes add;              // POLY: G, MUL: X (rows x cols, row stride add_ld), lo may be null
  int64_t add_ld, add_batch;
  Planes out;              // rows x cols planes; lo may be null (nothing reads it)
  int64_t out_ld, out_batch;
  const float* factor;     // [batch], x's scale: value = factor * plane (the first step), or null
  float alpha, beta;       // result = alpha * add + beta * product
  float diagonal;          // GRAM: added to the planes' diagonal
  void* result;            // MUL's last: the caller's matrix instead of planes
  int result_dtype, result_t, result_wide;  // transposed; rows in 16-byte words
  int64_t result_batch, result_ld;
};

struct __align__(8) Barriers {
  uint64_t full[6];
  uint64_t empty[6];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
  int consumed;
};

template <int PAIR, int OP, int SPLIT>
constexpr size_t smem_bytes() {
  using C = Cfg<PAIR, OP, SPLIT>;
  return 1024 + static_cast<size_t>(C::STAGES) * C::STAGE_BYTES + sizeof(Barriers);
}

template <bool SPIN = false, bool CLUSTER = false>
H3B_DEV bool warp_wait(uint64_t* bar, uint32_t parity, int site, volatile int* abort_flag) {
  const bool ok = mbar_wait<SPIN, CLUSTER>(bar, parity, &g_status, site, abort_flag);
  return __all_sync(0xffffffffu, ok);
}

H3B_DEV void tma_load_3d_pair(void* smem_dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z,
                              uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(leader_bar)
      : "memory");
}

H3B_DEV void mma_f16_ss_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

struct Tile {
  int batch, i, j;  // tile row, tile column
};
// Symmetric products: tile t of the lower triangle, row by row.
template <bool SYMMETRIC>
H3B_DEV Tile tile_at(int t, int per_matrix, int col_tiles) {
  Tile r;
  r.batch = t / per_matrix;
  const int u = t - r.batch * per_matrix;
  if constexpr (SYMMETRIC) {
    int i = static_cast<int>((sqrtf(8.0f * static_cast<float>(u) + 1.0f) - 1.0f) * 0.5f);
    while (i * (i + 1) / 2 > u) --i;
    while ((i + 1) * (i + 2) / 2 <= u) ++i;
    r.i = i;
    r.j = u - i * (i + 1) / 2;
  } else {
    r.i = u / col_tiles;
    r.j = u - r.i * col_tiles;
  }
  return r;
}

H3B_DEV void unpack8(const uint4& w, float* v) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

template <class T>
H3B_DEV T from_f32(float v);
template <>
H3B_DEV float from_f32<float>(float v) { return v; }
template <>
H3B_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
H3B_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Sixteen columns of a row of the caller's matrix.
template <class T>
H3B_DEV void store_row(const Args& args, int batch, int row, int col0, const float (&v)[16]) {
  T* base = static_cast<T*>(args.result) + batch * args.result_batch;
  constexpr int N = 16 / sizeof(T);
  if (args.result_t) {  // consecutive lanes, consecutive columns
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (col0 + j < args.cols) base[(col0 + j) * args.result_ld + row] = from_f32<T>(v[j]);
    return;
  }
  T* dst = base + row * args.result_ld + col0;
  if (args.result_wide && col0 + 16 <= args.cols) {
#pragma unroll
    for (int j = 0; j < 16; j += N) {
      T w[N];
#pragma unroll
      for (int e = 0; e < N; ++e) w[e] = from_f32<T>(v[j + e]);
      *reinterpret_cast<uint4*>(dst + j) = *reinterpret_cast<const uint4*>(w);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (col0 + j < args.cols) dst[j] = from_f32<T>(v[j]);
}
H3B_DEV void store_result(const Args& args, int batch, int row, int col0, const float (&v)[16]) {
  if (args.result_dtype == H3B_F32)
    store_row<float>(args, batch, row, col0, v);
  else if (args.result_dtype == H3B_F16)
    store_row<__half>(args, batch, row, col0, v);
  else
    store_row<__nv_bfloat16>(args, batch, row, col0, v);
}

template <int PAIR, int OP, int SPLIT>
__global__ void __launch_bounds__(THREADS, 1)
    ortho_product(const __grid_constant__ CUtensorMap a_hi, const __grid_constant__ CUtensorMap a_lo,
                  const __grid_constant__ CUtensorMap b_hi, const __grid_constant__ CUtensorMap b_lo, const Args args) {
  using C = Cfg<PAIR, OP, SPLIT>;
  constexpr int STAGES = C::STAGES, BN = C::BN;
  constexpr bool SYMMETRIC = OP != MUL;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Barriers* bars = reinterpret_cast<Barriers*>(smem + STAGES * C::STAGE_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR == 2 ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int cluster = static_cast<int>(blockIdx.x) / PAIR, n_clusters = static_cast<int>(gridDim.x) / PAIR;
  const int row_tiles = (args.rows + BN - 1) / BN, col_tiles = (args.cols + BN - 1) / BN;  // tiles are square
  const int per_matrix = SYMMETRIC ? row_tiles * (row_tiles + 1) / 2 : row_tiles * col_tiles;
  const int num_tiles = per_matrix * args.batch;
  const int nk = (args.k + KB - 1) / KB;
  volatile int* abort_flag = &bars->abort_flag;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc_full[b], 1);
      mbar_init(&bars->acc_empty[b], EPI_WARPS * PAIR);
    }
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    bars->consumed = 0;
    fence_barrier_init();
    prefetch_tmap(&a_hi);
    prefetch_tmap(&b_hi);
  }
  if (warp == 1) {
    if constexpr (PAIR == 2) {
      tmem_alloc_pair(&bars->tmem_base, C::TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&bars->tmem_base, C::TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (PAIR == 2)
    cluster_sync();
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;

  if (warp < 4) {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CTL));
  if (warp == 0) {
    // ---------------------------------------------------------- loads
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      const bool two_b = SPLIT && args.b_lo;
      const uint32_t bytes = PAIR * PLANE_BYTES * (C::PLANES + (two_b ? 2 : 1));
      for (int t = cluster; t < num_tiles && ok; t += n_clusters) {
        const Tile tile = tile_at<SYMMETRIC>(t, per_matrix, col_tiles);
        const int m0 = tile.i * BN + static_cast<int>(rank) * BM;
        const int n0 = tile.j * BN + static_cast<int>(rank) * BM;  // this CTA's 128 of the tile's columns
        for (int kb = 0; kb < nk; ++kb, ++it) {
          const int s = it % STAGES, round = it / STAGES;
          if (round > 0 && !mbar_wait(&bars->empty[s], (round - 1) & 1, &g_status, 1, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* stage = smem + s * C::STAGE_BYTES;
          uint32_t full = 0;
          if constexpr (PAIR == 2) full = mapa_shared(smem_u32(&bars->full[s]), 0);
          if (leader) mbar_arrive_expect_tx(&bars->full[s], bytes);
          auto load = [&](uint8_t* dst, const CUtensorMap* map, int x, int y) {
            if constexpr (PAIR == 2)
              tma_load_3d_pair(dst, map, x, y, tile.batch, full);
            else
              tma_load_3d(dst, map, x, y, tile.batch, &bars->full[s]);
          };
          load(stage, &a_hi, kb * KB, m0);
          if constexpr (SPLIT != 0) load(stage + PLANE_BYTES, &a_lo, kb * KB, m0);
          auto load_b = [&](uint8_t* dst, const CUtensorMap* map) {
            if constexpr (OP == MUL) {  // boxes of 64 columns x 64 rows of K
              load(dst, map, n0, kb * KB);
              load(dst + PLANE_BYTES / 2, map, n0 + 64, kb * KB);
            } else {
              load(dst, map, kb * KB, n0);
            }
          };
          load_b(stage + C::PLANES * PLANE_BYTES, &b_hi);
          if (two_b) load_b(stage + (C::PLANES + 1) * PLANE_BYTES, &b_lo);
        }
      }
      if (!ok || *abort_flag) {
        // No copy may still be in flight when the CTA leaves: wait (bounded)
        // for the stages issued and not seen by the products; the peer, whose
        // copies complete on the leader's barriers, gives them 200 us.
        if (leader) {
          const int consumed = *reinterpret_cast<volatile int*>(&bars->consumed);
          for (int j = consumed; j < it; ++j) mbar_wait(&bars->full[j % STAGES], (j / STAGES) & 1, &g_status, 9, nullptr);
        } else {
          const uint64_t t0 = globaltimer_ns();
          while (globaltimer_ns() - t0 < 200000ull) {
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------- products
    if (leader) {
      int it = 0, local = 0, s = 0, ph = 0;  // local: accumulators filled
      bool ok = true;
      const bool two_b = SPLIT && args.b_lo;
      for (int t = cluster; t < num_tiles && ok; t += n_clusters) {
        for (int kb = 0; kb < nk; ++kb, ++it) {
          const int buf = local & 1;
          if (kb % C::CHUNK == 0) {
            const int use = local >> 1;
            if (use > 0 && !warp_wait<false, PAIR == 2>(&bars->acc_empty[buf], (use - 1) & 1, 2, abort_flag)) {
              ok = false;
              break;
            }
          }
          if (!warp_wait<true>(&bars->full[s], static_cast<uint32_t>(ph), 3, abort_flag)) {
            ok = false;
            break;
          }
          if (lane == 0) *reinterpret_cast<volatile int*>(&bars->consumed) = it + 1;
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + buf * BN;
          const uint32_t stage = smem_u32(smem + s * C::STAGE_BYTES);
          const uint64_t ad = sdesc_kmajor_sw128(stage);
          const uint32_t sb = stage + C::PLANES * PLANE_BYTES;
          const uint64_t bd = OP == MUL ? sdesc_mnmajor_sw128(sb, PLANE_BYTES / 2, 1024) : sdesc_kmajor_sw128(sb);
          constexpr uint32_t B_STEP = OP == MUL ? 2048 >> 4 : 2;  // 16 elements of K
          constexpr uint32_t NEXT = PLANE_BYTES >> 4;             // the second plane
          const bool last = kb % C::CHUNK == C::CHUNK - 1 || kb == nk - 1;
          if (elect_one()) {
            auto mma = [&](uint64_t x, uint64_t y, bool add) {
              if constexpr (PAIR == 2)
                mma_f16_ss_pair(d_tmem, x, y, C::IDESC, add);
              else
                mma_f16_ss(d_tmem, x, y, C::IDESC, add);
            };
            const bool add = kb % C::CHUNK != 0;
            if constexpr (SPLIT != 0) {
#pragma unroll
              for (int j = 0; j < 4; ++j) mma(ad + NEXT + 2 * j, bd + B_STEP * j, add || j != 0);
              if (two_b) {
#pragma unroll
                for (int j = 0; j < 4; ++j) mma(ad + 2 * j, bd + NEXT + B_STEP * j, true);
              }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) mma(ad + 2 * j, bd + B_STEP * j, SPLIT || add || j != 0);
            if constexpr (PAIR == 2) {
              tc_commit_pair_mc(&bars->empty[s], 0x3);
              if (last) tc_commit_pair_mc(&bars->acc_full[buf], 0x3);
            } else {
              tc_commit(&bars->empty[s]);
              if (last) tc_commit(&bars->acc_full[buf]);
            }
          }
          __syncwarp();
          if (last) ++local;
          if (++s == STAGES) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (elect_one()) {
        if constexpr (PAIR == 2)
          tc_commit_pair(&bars->drain);
        else
          tc_commit(&bars->drain);
      }
      __syncwarp();
      warp_wait(&bars->drain, 0, 8, nullptr);
    }
  }
  } else {
    // --------------------------------------------------------- stores
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_EPI));
    const int quad = warp & 3, half = (warp - 4) >> 2;  // TMEM lane quadrant; alternate 32-column chunks
    constexpr int MINE = BN / 64;                         // this warp's chunks of 32 columns
    int local = 0;
    bool ok = true;
    for (int t = cluster; t < num_tiles && ok; t += n_clusters) {
      float acc[2 * MINE][16];
      for (int kb = 0; kb < nk; kb += C::CHUNK, ++local) {
        const int buf = local & 1, use = local >> 1;
        if (!warp_wait<true>(&bars->acc_full[buf], use & 1, 4, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t t_row = tmem_base + buf * BN + (static_cast<uint32_t>(quad * 32) << 16);
#pragma unroll
        for (int i = 0; i < 2 * MINE; ++i) {
          uint32_t r[16];
          tmem_ld16(t_row + (half + 2 * (i >> 1)) * 32 + (i & 1) * 16, r);
          tc_wait_ld();
          reg_fence16(r);
          if (i == 2 * MINE - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (PAIR == 2)
                mbar_arrive_cluster(mapa_shared(smem_u32(&bars->acc_empty[buf]), 0));
              else
                mbar_arrive(&bars->acc_empty[buf]);
            }
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[i][j] = kb == 0 ? __uint_as_float(r[j]) : acc[i][j] + __uint_as_float(r[j]);
        }
      }
      if (!ok) break;
      const Tile tile = tile_at<SYMMETRIC>(t, per_matrix, col_tiles);
      const int row = tile.i * BN + static_cast<int>(rank) * BM + quad * 32 + lane;
      const bool row_ok = row < args.rows;
      const float f = args.factor != nullptr ? args.factor[tile.batch] : 1.0f;
      const float beta = (OP == GRAM ? f * f : OP == MUL ? f : 1.0f) * args.beta;
      const float alpha = (OP == MUL ? f : 1.0f) * args.alpha;
      const int64_t add_at = tile.batch * args.add_batch + row * args.add_ld;
      const int64_t out_at = tile.batch * args.out_batch;
      if (row_ok) {
        // Sixteen columns at a time.  Rows of the planes are multiples of 32
        // elements apart, so whole pieces are read and written; what lies
        // behind the last column is never used.
#pragma unroll
        for (int i = 0; i < 2 * MINE; ++i) {
          const int col0 = tile.j * BN + (half + 2 * (i >> 1)) * 32 + (i & 1) * 16;
          if (col0 >= args.cols) continue;
          float v[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = acc[i][j] * beta;
          if (OP == GRAM && tile.i == tile.j) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (col0 + j == row) v[j] += args.diagonal;
          }
          if (OP != GRAM) {
#pragma unroll
            for (int j = 0; j < 16; j += 8) {
              float h[8];
              unpack8(*reinterpret_cast<const uint4*>(args.add.hi + add_at + col0 + j), h);
#pragma unroll
              for (int e = 0; e < 8; ++e) v[j + e] = fmaf(alpha, h[e], v[j + e]);
              if (args.add.lo != nullptr) {
                unpack8(*reinterpret_cast<const uint4*>(args.add.lo + add_at + col0 + j), h);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[j + e] = fmaf(alpha, h[e], v[j + e]);
              }
            }
          }
          if (OP == MUL && args.result != nullptr) {
            store_result(args, tile.batch, row, col0, v);
            continue;
          }
          uint32_t hi[8], lo[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            hi[j] = pack_f16x2(v[2 * j], v[2 * j + 1]);
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[j]));
            lo[j] = pack_f16x2(v[2 * j] - h.x, v[2 * j + 1] - h.y);
          }
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            __half* plane = p == 0 ? args.out.hi : args.out.lo;
            if (plane == nullptr) continue;
            const uint32_t* w = p == 0 ? hi : lo;
            uint4* dst = reinterpret_cast<uint4*>(plane + out_at + row * args.out_ld + col0);
            dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
            dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
            if (SYMMETRIC && tile.i != tile.j) {  // the other side: consecutive lanes, consecutive columns
              __half* mirror = plane + out_at + col0 * args.out_ld + row;
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                if (col0 + j < args.cols)
                  *mirror = __ushort_as_half(static_cast<unsigned short>(w[j >> 1] >> (16 * (j & 1))));
                mirror += args.out_ld;
              }
            }
          }
        }
      }
      __syncwarp();  // before the next tile's TMEM loads
    }
  }

  tc_fence_before();
  if constexpr (PAIR == 2)
    cluster_sync();
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR == 2)
      tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
    else
      tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

// ------------------------------------------------------- norm and planes

H3B_DEV float to_f32(float v) { return v; }
H3B_DEV float to_f32(__half v) { return __half2float(v); }
H3B_DEV float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

constexpr int MAX_PARTS = 256;

// Sums of squares in 64 bits (a 32-bit square of a gradient of 10^-20 is
// nothing); part p of matrix b: rows p, p + parts, ...
template <class T>
__global__ void __launch_bounds__(256) ortho_squares(const T* x, int64_t batch_stride, int64_t ld, int m, int n,
                                                     double* parts) {
  const T* base = x + blockIdx.y * batch_stride;
  double s = 0.0;
  for (int r = blockIdx.x; r < m; r += gridDim.x) {
    const T* row = base + r * ld;
    for (int c = threadIdx.x; c < n; c += 256) {
      const double v = to_f32(row[c]);
      s = fma(v, v, s);
    }
  }
  __shared__ double warp_sums[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) s += warp_sums[i];
    parts[blockIdx.y * gridDim.x + blockIdx.x] = s;
  }
}

// Planes of SCALE * x / 2^e, 2^e <= |x| < 2^(e+1), and the factor
// 2^e / (|x| + eps) that is left; 32 x 32 elements a CTA, transposed if asked.
template <class T>
__global__ void __launch_bounds__(256) ortho_planes(const T* x, int64_t batch_stride, int64_t ld, int m, int n,
                                                    int transposed, const double* parts, int n_parts, float eps,
                                                    float* factor, __half* hi, __half* lo, int64_t out_batch,
                                                    int64_t out_ld) {
  __shared__ float tile[32][33];
  __shared__ double total;
  const int b = blockIdx.z;
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int i = 0; i < n_parts; ++i) s += parts[b * n_parts + i];
    total = s;
  }
  __syncthreads();
  const double norm = sqrt(total);
  const int e = norm > 0.0 && norm < 1e300 ? ilogb(norm) : 0;
  const int up = 10 - e;  // 2^10 = SCALE
  const float s1 = ldexpf(1.0f, up / 2), s2 = ldexpf(1.0f, up - up / 2);
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0)
    factor[b] = static_cast<float>(scalbn(1.0, e) / (norm + static_cast<double>(eps)));
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32;
  const T* base = x + b * batch_stride;
  auto put = [&](int r, int c, float v) {
    const int64_t at = b * out_batch + r * out_ld + c;
    const __half h = __float2half_rn(v);
    hi[at] = h;
    if (lo != nullptr) lo[at] = __float2half_rn(v - __half2float(h));
  };
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const int r = r0 + ty + i, c = c0 + tx;
    if (r < m && c < n) {
      const float v = to_f32(base[r * ld + c]) * s1 * s2;
      if (transposed)
        tile[ty + i][tx] = v;
      else
        put(r, c, v);
    }
  }
  if (!transposed) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const int r = c0 + ty + i, c = r0 + tx;
    if (r < n && c < m) put(r, c, tile[tx][ty + i]);
  }
}

// No steps: x / (|x| + eps).
template <class T>
__global__ void __launch_bounds__(256) ortho_scale(const T* x, int64_t batch_stride, int64_t ld, int m, int n,
                                                   const double* parts, int n_parts, float eps, T* out) {
  double s = 0.0;
  for (int i = 0; i < n_parts; ++i) s += parts[blockIdx.y * n_parts + i];
  const double inv = 1.0 / (sqrt(s) + static_cast<double>(eps));
  for (int r = blockIdx.x; r < m; r += gridDim.x)
    for (int c = threadIdx.x; c < n; c += 256)
      out[(static_cast<int64_t>(blockIdx.y) * m + r) * n + c] =
          static_cast<T>(static_cast<float>(to_f32(x[blockIdx.y * batch_stride + r * ld + c]) * inv));
}

// ---------------------------------------------------------------- hosts

struct Layout {
  int64_t small, large;      // sides of X
  int64_t x_ld, g_ld;        // row strides of the planes of X and of G, B
  int64_t x_plane, g_plane;  // elements of a plane, all matrices
  int64_t bytes;
};

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Planes of X (two, in turn), G and B, two each; sums of squares; factors.
Layout layout(int64_t batch, int64_t m, int64_t n) {
  Layout l;
  l.small = m < n ? m : n;
  l.large = m < n ? n : m;
  l.x_ld = up(l.large, 32);
  l.g_ld = up(l.small, 32);
  l.x_plane = up(batch * l.small * l.x_ld, 128);
  l.g_plane = up(batch * l.small * l.g_ld, 128);
  l.bytes = (4 * l.x_plane + 4 * l.g_plane) * 2 + batch * (MAX_PARTS * 8) + up(batch * 4, 256);
  return l;
}

int check(int64_t batch, int64_t m, int64_t n) {
  if (batch < 0 || batch > 65535 || m < 1 || n < 1 || m > 65536 || n > 65536) return H3B_ERR_SHAPE;
  if (batch * m > (1ll << 31) / 4 || batch * n > (1ll << 31) / 4) return H3B_ERR_SHAPE;
  return H3B_OK;
}

struct Maps {
  CUtensorMap hi, lo;
};

// rows x cols planes for tiles of 128 rows by 64 columns, or (by_rows) for
// boxes of 64 columns by 64 rows.
int encode(Maps* maps, const Planes& p, int64_t batch, int64_t rows, int64_t cols, int64_t ld, bool boxes) {
  const uint32_t high = boxes ? 64 : 128;
  for (int i = 0; i < 2; ++i) {
    const __half* base = i == 0 || p.lo == nullptr ? p.hi : p.lo;
    const int rc = h3b::encode_3d(i == 0 ? &maps->hi : &maps->lo, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, base, cols, rows,
                                  batch, ld * 2, rows * ld * 2, 64, high, 1, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != H3B_OK) return rc;
  }
  return H3B_OK;
}

template <int PAIR, int OP, int SPLIT>
int launch(const Maps& a, const Maps& b, const Args& args, int64_t tiles, cudaStream_t stream) {
  constexpr size_t smem = smem_bytes<PAIR, OP, SPLIT>();
  static_assert(smem <= 227 * 1024, "shared memory budget");
  static h3b::OncePerDevice once;
  const auto kernel = ortho_product<PAIR, OP, SPLIT>;
  const int rc = once.run(h3b::device(), [&] {
    // the register split waits for good in a launch with fewer registers than it adds up to
    cudaFuncAttributes attr;
    if (cudaFuncGetAttributes(&attr, kernel) != cudaSuccess || attr.numRegs < LAUNCH_REGS) return static_cast<int>(H3B_ERR_LAUNCH);
    return h3b::allow_smem(kernel, smem);
  });
  if (rc != H3B_OK) return rc;
  const int64_t most = h3b::num_sms() / PAIR;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((tiles < most ? tiles : most) * PAIR));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PAIR;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR == 2 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a.hi, a.lo, b.hi, b.lo, args) == cudaSuccess ? H3B_OK : H3B_ERR_LAUNCH;
}

// Tiles of side `t`, all matrices.
int64_t tiles_of(int64_t rows, int64_t cols, int64_t batch, int64_t t, bool symmetric) {
  const int64_t r = (rows + t - 1) / t, c = (cols + t - 1) / t;
  return batch * (symmetric ? r * (r + 1) / 2 : r * c);
}

template <int OP, int SPLIT>
int product(const Maps& a, const Maps& b, const Args& args, cudaStream_t stream) {
  const int64_t sms = h3b::num_sms();
  const int64_t t1 = tiles_of(args.rows, args.cols, args.batch, 128, OP != MUL);
  const int64_t t2 = tiles_of(args.rows, args.cols, args.batch, 256, OP != MUL);
  // Rounds of tiles, a 128 x 128 tile counted 0.8 of a pair's 256 x 256 one.
  const int64_t single = (t1 + sms - 1) / sms * 4, pair = (t2 + sms / 2 - 1) / (sms / 2) * 5;
  return single <= pair ? launch<1, OP, SPLIT>(a, b, args, t1, stream) : launch<2, OP, SPLIT>(a, b, args, t2, stream);
}

template <int OP>
int product(bool split, const Maps& a, const Maps& b, const Args& args, cudaStream_t stream) {
  return split ? product<OP, 1>(a, b, args, stream) : product<OP, 0>(a, b, args, stream);
}

template <class T>
int run(const T* x, T* out, int dtype, int64_t batch, int64_t m, int64_t n, int64_t batch_stride, int64_t ld, int steps,
        const float* coefficients, float eps, uint8_t* ws, cudaStream_t stream) {
  const Layout l = layout(batch, m, n);
  __half* at = reinterpret_cast<__half*>(ws);
  auto take = [&](int64_t plane) {
    Planes p{at, at + plane};
    at += 2 * plane;
    return p;
  };
  Planes xs[2] = {take(l.x_plane), take(l.x_plane)};
  const Planes g = take(l.g_plane), b = take(l.g_plane);
  double* parts = reinterpret_cast<double*>(at);
  float* factor = reinterpret_cast<float*>(parts + batch * MAX_PARTS);
  const int n_parts = static_cast<int>(m < MAX_PARTS ? m : MAX_PARTS);
  const int mi = static_cast<int>(m), ni = static_cast<int>(n);
  ortho_squares<T><<<dim3(n_parts, static_cast<unsigned>(batch)), 256, 0, stream>>>(x, batch_stride, ld, mi, ni, parts);
  if (steps == 0) {
    ortho_scale<T><<<dim3(n_parts, static_cast<unsigned>(batch)), 256, 0, stream>>>(x, batch_stride, ld, mi, ni, parts,
                                                                                 n_parts, eps, out);
    return h3b::launch_status();
  }
  const bool tall = m > n;
  const bool exact = dtype != H3B_F32;  // one plane holds x
  const dim3 grid(static_cast<unsigned>((n + 31) / 32), static_cast<unsigned>((m + 31) / 32), static_cast<unsigned>(batch));
  ortho_planes<T><<<grid, 256, 0, stream>>>(x, batch_stride, ld, mi, ni, tall ? 1 : 0, parts, n_parts, eps, factor,
                                            xs[0].hi, exact ? nullptr : xs[0].lo, l.small * l.x_ld, l.x_ld);
  int rc = h3b::launch_status();
  if (rc != H3B_OK) return rc;

  Maps x_k[2], x_n[2], gm, bm;  // X by rows (K-major) and by boxes (N-major)
  for (int i = 0; i < 2 && rc == H3B_OK; ++i) {
    rc = encode(&x_k[i], xs[i], batch, l.small, l.large, l.x_ld, false);
    if (rc == H3B_OK) rc = encode(&x_n[i], xs[i], batch, l.small, l.large, l.x_ld, true);
  }
  if (rc == H3B_OK) rc = encode(&gm, g, batch, l.small, l.small, l.g_ld, false);
  if (rc == H3B_OK) rc = encode(&bm, b, batch, l.small, l.small, l.g_ld, false);

  for (int s = 0; s < steps && rc == H3B_OK; ++s) {
    const bool first = s == 0, last = s == steps - 1;
    const bool pairs = !(last && dtype == H3B_BF16);  // planes in pairs: all steps but a bf16 result's last
    const bool x_lo = pairs && !(first && exact);
    const int cur = s & 1;
    Args a{};
    a.batch = static_cast<int>(batch);
    a.rows = a.cols = static_cast<int>(l.small);
    a.k = static_cast<int>(l.large);
    a.factor = first ? factor : nullptr;
    a.b_lo = x_lo;
    a.beta = 1.0f / SCALE;
    a.diagonal = pairs ? 0.0f : -SCALE;
    a.out = {g.hi, pairs ? g.lo : nullptr};
    a.out_ld = l.g_ld;
    a.out_batch = l.small * l.g_ld;
    rc = product<GRAM>(x_lo, x_k[cur], x_k[cur], a, stream);
    if (rc != H3B_OK) break;

    a.factor = nullptr;
    a.k = a.rows;
    a.b_lo = pairs;
    a.add = a.out;
    a.add_ld = l.g_ld;
    a.add_batch = a.out_batch;
    a.out = b;
    if (!pairs) a.out.lo = nullptr;
    a.alpha = pairs ? coefficients[1] : coefficients[1] + 2.0f * coefficients[2];
    a.beta = coefficients[2] / SCALE;
    rc = product<POLY>(pairs, gm, gm, a, stream);
    if (rc != H3B_OK) break;

    a.factor = first ? factor : nullptr;
    a.cols = static_cast<int>(l.large);
    a.b_lo = x_lo;
    a.add = xs[cur];
    if (first && exact) a.add.lo = nullptr;
    a.add_ld = l.x_ld;
    a.add_batch = l.small * l.x_ld;
    a.out = xs[cur ^ 1];
    a.out_ld = l.x_ld;
    a.out_batch = a.add_batch;
    a.alpha = pairs ? coefficients[0] : coefficients[0] + coefficients[1] + coefficients[2];
    a.beta = 1.0f / SCALE;
    if (last) {
      a.alpha /= SCALE;
      a.beta /= SCALE;
      a.result = out;
      a.result_dtype = dtype;
      a.result_t = tall;
      a.result_batch = m * n;
      a.result_ld = n;
      a.result_wide = !tall && h3b::aligned16(out) && n * static_cast<int64_t>(sizeof(T)) % 16 == 0;
    }
    rc = product<MUL>(pairs, bm, x_n[cur], a, stream);
  }
  return rc;
}

}  // namespace

extern "C" int h3b_orthogonalize_workspace(int64_t batch, int64_t m, int64_t n, int64_t* bytes) {
  if (bytes == nullptr) return H3B_ERR_ARG;
  const int rc = check(batch, m, n);
  if (rc != H3B_OK) return rc;
  *bytes = layout(batch, m, n).bytes;
  return H3B_OK;
}

extern "C" int h3b_orthogonalize(const void* x, void* out, int dtype, int64_t batch, int64_t m, int64_t n,
                                 int64_t batch_stride, int64_t ld, int64_t steps, float a, float b, float c, float eps,
                                 void* workspace, int64_t workspace_bytes, h3b_stream_t stream) {
  if (dtype != H3B_BF16 && dtype != H3B_F16 && dtype != H3B_F32) return H3B_ERR_DTYPE;
  const int rc = check(batch, m, n);
  if (rc != H3B_OK) return rc;
  if (batch == 0) return H3B_OK;
  if (x == nullptr || out == nullptr || workspace == nullptr || steps < 0 || steps > 1000 || !(eps >= 0.0f))
    return H3B_ERR_ARG;
  if (!h3b::aligned16(workspace)) return H3B_ERR_ALIGN;
  if (workspace_bytes < layout(batch, m, n).bytes) return H3B_ERR_ARG;
  const float coefficients[3] = {a, b, c};
  const auto st = reinterpret_cast<cudaStream_t>(stream);
  auto* ws = static_cast<uint8_t*>(workspace);
  const int k = static_cast<int>(steps);
  if (dtype == H3B_F32)
    return run(static_cast<const float*>(x), static_cast<float*>(out), dtype, batch, m, n, batch_stride, ld, k,
               coefficients, eps, ws, st);
  if (dtype == H3B_F16)
    return run(static_cast<const __half*>(x), static_cast<__half*>(out), dtype, batch, m, n, batch_stride, ld, k,
               coefficients, eps, ws, st);
  return run(static_cast<const __nv_bfloat16*>(x), static_cast<__nv_bfloat16*>(out), dtype, batch, m, n, batch_stride,
             ld, k, coefficients, eps, ws, st);
}
