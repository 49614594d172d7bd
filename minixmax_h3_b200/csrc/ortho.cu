// The orthogonal factor of an update matrix, approached by Newton-Schulz
// steps: X <- a X + (b G + c G G) X, G = X X^T, from X = x / (|x| + eps), the
// smaller side first (x of more rows than columns is taken transposed and
// given back so).
//
// A step is three matrix products on tcgen05 (kind::f16, fp32 accumulators in
// TMEM), arranged so that none has a second matrix to add where it stores.
// Results in 16 bits complete the polynomial's square:
//   GRAM  H = X X^T + (b / 2c) 1         symmetric: only tiles on or below the
//   POLY  B = c H H + (a - b^2 / 4c) 1   diagonal, stored to both sides
//   MUL   X' = B X    (X is read K-major by GRAM, N-major by MUL)
// Results in 32 bits, whose first steps the constants would cost a bit or two
// (G is small there), and coefficients with |b / 2c| above 4 take a second
// factor instead, K = c G + b 1, for B = G K + a 1 (at 4096 GRAM takes 180 us
// with it and 156 without).
//
// Precision.  A step multiplies small singular values by a, five steps by
// 480: what a rounding spills from the large directions into the small ones
// grows with them, and one plane of 16-bit operands (2^-12 a rounding) leaves
// 1.4 % of the result wrong for an update dominated by a few directions, bf16
// operands 13 %.  So operands are pairs of f16 planes, v = hi + lo (22 bits),
// and a product is hi hi + lo hi + hi lo in one accumulator (what is left out
// is 2^-22).  That is as near as 32-bit arithmetic comes at a fifth of its
// time on CUDA cores, for every step of every type: a bf16 result's last steps
// in one plane were a fifth faster (4096 x 4096 in 2.73 ms, so 3.40), but off
// by 0.0006 to 0.0015, up to what the result's own rounding is (0.0017).  One product saves a plane without a loss: x in 16 bits is one as it
// is, by a scale of a power of two (the norm's fraction goes into the first
// epilogues; its 8 or 11 bits are whole down to 2^-24 of the norm, smaller
// elements are off by 2^-35 of the norm at most, as any element of a pair is).
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
// ones, and the storing warps add accumulators in registers, rounding to
// nearest.
//
// Tiles: 256 x 256 by CTA pairs (cta_group::2, each CTA stages 128 rows of
// both operands); where those are too few for the SMs, 128 x 128 by one CTA;
// where those are, too, 128 x 64 or 128 x 32 (a launch takes 1 us by itself and
// the stores of 128 columns 3.4: five steps of 200 x 200 bf16 in 92 us, with
// 128 columns 121), or, over a long K, 128 x 128 by a cluster of two to four,
// each with a part of K, that hand each other their sums through distributed
// shared memory.
// Warp 0 loads (TMA, zero beyond the matrix), warp 1 issues the products,
// eight warps add and store; two accumulators in turn, so that products go on
// meanwhile.  Stores go through shared memory as TMA blocks of 32 x 32 (lanes
// that stored their rows' 16-byte pieces themselves took 20 us a tile, a third
// of a product's time at 4096).  Every wait is bounded.
//
// A launch's setup overlaps the end of the one before it (programmatic
// dependent launch); every kernel waits for it before it touches memory.
#include <algorithm>

#include "h3b_common.cuh"
#include "h3b_host.hpp"
#include "ortho.hpp"

H3B_DECLARE_STATUS();
H3B_REGISTER_STATUS_READER(ortho);

namespace {

constexpr float SCALE = 1024.0f;
constexpr int BM = 128;            // accumulator rows of a CTA
constexpr int KB = 64;             // elements of K a stage (128 bytes a row)
constexpr int CHUNK = 2;           // stages of K an accumulator takes
constexpr int PLANE_BYTES = BM * 128;
constexpr int BLOCK_BYTES = 32 * 64;  // a block on its way out: 32 rows of 64 bytes
constexpr int BLOCKS = 2;             // of each storing warp
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 128 + 32 * EPI_WARPS;  // a warpgroup to load and issue (two of its warps idle), two to store

// Registers a thread: 384 threads launch with 168; the storing warpgroups,
// which hold 128 sums a thread, take over what the first one does not need.
constexpr int LAUNCH_REGS = 168;
constexpr int REGS_CTL = 72;
constexpr int REGS_EPI = 216;
static_assert(4 * REGS_CTL + 8 * REGS_EPI <= 12 * LAUNCH_REGS, "register split exceeds launch");

enum Op { GRAM = 0, POLY = 1, MUL = 2 };

// PAIR: CTAs of a 256 x 256 tile.  PARTS: CTAs that share the K of a 128 x 128
// tile (PAIR = 1).  COLS: columns of a CTA's part of a 128 x 128 tile (where
// all three are 1, 1 and less than 128).
template <int PAIR, int PARTS, int OP, int SPLIT, int COLS>
struct Cfg {
  static_assert(PAIR == 1 || PARTS == 1, "pairs take all of K");
  static_assert(COLS == 128 || (PAIR * PARTS == 1 && (COLS == 64 || (COLS == 32 && OP != MUL))), "narrow tiles");
  static constexpr int SIDE = 128 * PAIR;      // of a tile
  static constexpr int SLICES = 128 / COLS;    // of a tile, a CTA's work each
  static constexpr int BN = COLS * PAIR;
  static constexpr int B_BYTES = COLS * 128;   // a plane of B
  static constexpr int PLANES = SPLIT ? 2 : 1;
  static constexpr int STAGE_BYTES = PLANES * (PLANE_BYTES + B_BYTES);  // A planes, then B planes
  static constexpr int STAGES = SPLIT ? (COLS == 128 ? 3 : 4) : 6;
  static constexpr int TMEM_COLS = 2 * BN;  // two accumulators
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
  int with_k;              // GRAM: K is stored beside G
  const float* factor;     // [batch], x's scale: value = factor * plane (the first step), or null
  float beta, diagonal;    // beta * product + diagonal * 1
  float k_beta, k_diagonal;  // GRAM's K: of the former
  void* result;            // MUL's last: the caller's matrix instead of planes
  int result_dtype, result_t, result_tma;  // transposed; out_hi is its map
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

template <int PAIR, int PARTS, int OP, int SPLIT, int COLS>
constexpr size_t smem_bytes() {
  using C = Cfg<PAIR, PARTS, OP, SPLIT, COLS>;
  return 1024 + static_cast<size_t>(C::STAGES) * C::STAGE_BYTES + EPI_WARPS * BLOCKS * BLOCK_BYTES + sizeof(Barriers);
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

H3B_DEV void tma_store_3d(const CUtensorMap* map, const void* smem_src, int32_t x, int32_t y, int32_t z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(z), "r"(smem_u32(smem_src))
               : "memory");
}

// A storing warp's blocks.  Lane l holds row y0 + l, columns x0 .. x0 + 31 (16
// bits) or x0 .. x0 + 15 (32 bits); `turned` stores the block transposed.
struct Blocks {
  uint8_t* smem;
  int lane, at;

  // 16-byte piece c of row r in the 64-byte swizzle
  H3B_DEV static uint32_t swz(int r, int c) { return static_cast<uint32_t>(r * 64 + ((c ^ ((r >> 1) & 3)) << 4)); }
  H3B_DEV uint8_t* next() {
    uint8_t* p = smem + (at++ % BLOCKS) * BLOCK_BYTES;
    if (lane == 0) bulk_wait_group_read<BLOCKS - 1>();  // the store from here has read it
    __syncwarp();
    return p;
  }
  H3B_DEV void send(const CUtensorMap* map, const uint8_t* p, int x, int y, int z) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_3d(map, p, x, y, z);
      bulk_commit_group();
    }
  }
  // w: 32 columns of 16 bits
  H3B_DEV void put(const CUtensorMap* map, const uint32_t (&w)[16], bool turned, int x0, int y0, int z) {
    uint8_t* p = next();
    if (!turned) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<uint4*>(p + swz(lane, c)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
      send(map, p, x0, y0, z);
      return;
    }
    // A pair of lanes trades halves: the even one takes the even column of
    // both rows, the odd one the odd column; a row of the block is a column.
    const uint32_t pick = lane & 1 ? 0x3276 : 0x5410;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, w[j], 1);
      *reinterpret_cast<uint32_t*>(p + swz(2 * j + (lane & 1), lane >> 3) + ((lane >> 1) & 3) * 4) =
          __byte_perm(w[j], other, pick);
    }
    send(map, p, y0, x0, z);
  }
  // v: 32 columns of 32 bits, as two blocks of 16 (columns, or, turned, lanes)
  H3B_DEV void put(const CUtensorMap* map, const float (&v)[32], bool turned, int x0, int y0, int z) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint8_t* p = next();
      if (!turned) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<float4*>(p + swz(lane, c)) =
              make_float4(v[16 * h + 4 * c], v[16 * h + 4 * c + 1], v[16 * h + 4 * c + 2], v[16 * h + 4 * c + 3]);
        send(map, p, x0 + 16 * h, y0, z);
      } else {
        if ((lane >> 4) == h) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            *reinterpret_cast<float*>(p + swz(j, (lane & 15) >> 2) + (lane & 3) * 4) = v[j];
        }
        send(map, p, y0 + 16 * h, x0, z);
      }
    }
  }
};

// 32 columns of a row of the caller's matrix, element by element (rows that
// are no multiple of 16 bytes).
H3B_DEV void store_elements(const Args& args, int batch, int row, int col0, const float (&v)[32]) {
  const int64_t base = batch * args.result_batch + (args.result_t ? col0 * args.result_ld + row : row * args.result_ld + col0);
  const int64_t step = args.result_t ? args.result_ld : 1;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    if (col0 + j < args.cols) {
      const int64_t at = base + j * step;
      if (args.result_dtype == H3B_F32)
        static_cast<float*>(args.result)[at] = v[j];
      else if (args.result_dtype == H3B_F16)
        static_cast<__half*>(args.result)[at] = __float2half_rn(v[j]);
      else
        static_cast<__nv_bfloat16*>(args.result)[at] = __float2bfloat16_rn(v[j]);
    }
  }
}

// Lets the next launch set itself up; waits for the one before to end.
H3B_DEV void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
H3B_DEV void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <int PAIR, int PARTS, int OP, int SPLIT, int COLS>
__global__ void __launch_bounds__(THREADS, 1)
    ortho_product(const __grid_constant__ CUtensorMap a_hi, const __grid_constant__ CUtensorMap a_lo,
                  const __grid_constant__ CUtensorMap b_hi, const __grid_constant__ CUtensorMap b_lo,
                  const __grid_constant__ CUtensorMap out_hi, const __grid_constant__ CUtensorMap out_lo,
                  const __grid_constant__ CUtensorMap k_hi, const __grid_constant__ CUtensorMap k_lo,
                  const Args args) {
  using C = Cfg<PAIR, PARTS, OP, SPLIT, COLS>;
  constexpr int STAGES = C::STAGES, BN = C::BN, SIDE = C::SIDE, SLICES = C::SLICES;
  constexpr bool SYMMETRIC = OP != MUL;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* blocks = smem + STAGES * C::STAGE_BYTES;
  Barriers* bars = reinterpret_cast<Barriers*>(blocks + EPI_WARPS * BLOCKS * BLOCK_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR == 2 ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int part = PARTS > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int cluster = static_cast<int>(blockIdx.x) / (PAIR * PARTS), n_clusters = static_cast<int>(gridDim.x) / (PAIR * PARTS);
  const int row_tiles = (args.rows + SIDE - 1) / SIDE, col_tiles = (args.cols + SIDE - 1) / SIDE;  // tiles are square
  const int per_matrix = SYMMETRIC ? row_tiles * (row_tiles + 1) / 2 : row_tiles * col_tiles;
  const int num_tiles = per_matrix * args.batch * SLICES;  // or slices
  // stages of K: this CTA's (PARTS > 1: a launch has a cluster for each tile)
  const int all_k = (args.k + KB - 1) / KB, share_k = (all_k + PARTS - 1) / PARTS;
  const int first_k = part * share_k, nk = max(0, min(share_k, all_k - first_k));
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
    prefetch_tmap(&out_hi);
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
  if constexpr (PAIR * PARTS > 1)
    cluster_sync();
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  launch_next();
  wait_previous();

  if (warp < 4) {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CTL));
  if (warp == 0) {
    // ---------------------------------------------------------- loads
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      const bool two_b = SPLIT && args.b_lo;
      const uint32_t bytes = PAIR * (PLANE_BYTES * C::PLANES + C::B_BYTES * (two_b ? 2 : 1));
      for (int t = cluster; t < num_tiles && ok; t += n_clusters) {
        const Tile tile = tile_at<SYMMETRIC>(t / SLICES, per_matrix, col_tiles);
        const int m0 = tile.i * SIDE + static_cast<int>(rank) * BM;
        const int n0 = tile.j * SIDE + static_cast<int>(rank) * BM + t % SLICES * COLS;  // this CTA's of the tile's columns
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
          load(stage, &a_hi, (first_k + kb) * KB, m0);
          if constexpr (SPLIT != 0) load(stage + PLANE_BYTES, &a_lo, (first_k + kb) * KB, m0);
          auto load_b = [&](uint8_t* dst, const CUtensorMap* map) {
            if constexpr (OP == MUL) {  // boxes of 64 columns x 64 rows of K
              load(dst, map, n0, (first_k + kb) * KB);
              if constexpr (COLS == 128) load(dst + PLANE_BYTES / 2, map, n0 + 64, (first_k + kb) * KB);
            } else {
              load(dst, map, (first_k + kb) * KB, n0);
            }
          };
          load_b(stage + C::PLANES * PLANE_BYTES, &b_hi);
          if (two_b) load_b(stage + C::PLANES * PLANE_BYTES + C::B_BYTES, &b_lo);
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
          if (kb % CHUNK == 0) {
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
          constexpr uint32_t NEXT = PLANE_BYTES >> 4, NEXT_B = C::B_BYTES >> 4;  // the second planes
          const bool last = kb % CHUNK == CHUNK - 1 || kb == nk - 1;
          if (elect_one()) {
            auto mma = [&](uint64_t x, uint64_t y, bool add) {
              if constexpr (PAIR == 2)
                mma_f16_ss_pair(d_tmem, x, y, C::IDESC, add);
              else
                mma_f16_ss(d_tmem, x, y, C::IDESC, add);
            };
            const bool add = kb % CHUNK != 0;
            if constexpr (SPLIT != 0) {
#pragma unroll
              for (int j = 0; j < 4; ++j) mma(ad + NEXT + 2 * j, bd + B_STEP * j, add || j != 0);
              if (two_b) {
#pragma unroll
                for (int j = 0; j < 4; ++j) mma(ad + 2 * j, bd + NEXT_B + B_STEP * j, true);
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
  if constexpr (PARTS > 1) {  // the storing warps' hand-over
    __syncwarp();
    cluster_sync();
    cluster_sync();
  }
  } else {
    // --------------------------------------------------------- stores
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_EPI));
    const int quad = warp & 3, half = (warp - 4) >> 2;  // TMEM lane quadrant; alternate 32-column chunks
    constexpr int MINE = BN > 32 ? BN / 64 : 1;           // this warp's chunks of 32 columns
    // (both halves take a single chunk, and share its planes)
    const auto chunk = [&](int i) { return COLS == 32 ? 0 : half + 2 * i; };
    Blocks out{blocks + (warp - 4) * BLOCKS * BLOCK_BYTES, lane, 0};
    int local = 0;
    bool ok = true;
    for (int t = cluster; t < num_tiles && ok; t += n_clusters) {
      float acc[2 * MINE][16];
      if (PARTS > 1 && nk == 0) {  // a part without any of K
#pragma unroll
        for (int i = 0; i < 2 * MINE; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;
      }
      for (int kb = 0; kb < nk; kb += CHUNK, ++local) {
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
          tmem_ld16(t_row + chunk(i >> 1) * 32 + (i & 1) * 16, r);
          tc_wait_ld();
          reg_fence16(r);
          if (i == 2 * MINE - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              // (a release of cluster scope would hold this warp for 1000 cycles)
              if (leader)
                mbar_arrive(&bars->acc_empty[buf]);
              else
                mbar_arrive_remote(mapa_shared(smem_u32(&bars->acc_empty[buf]), 0));
            }
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[i][j] = kb == 0 ? __uint_as_float(r[j]) : acc[i][j] + __uint_as_float(r[j]);
        }
      }
      if constexpr (PARTS == 1) {
        if (!ok) break;
      }
      const Tile tile = tile_at<SYMMETRIC>(t / SLICES, per_matrix, col_tiles);
      const int row0 = tile.i * SIDE + static_cast<int>(rank) * BM + quad * 32, row = row0 + lane;
      const float f = args.factor != nullptr ? args.factor[tile.batch] : 1.0f;
      const float beta = (OP == GRAM ? f * f : OP == MUL ? f : 1.0f) * args.beta;
      // Stores 32 columns from col0 of the sums that sums(v) puts into v; of
      // the planes (G's, then K's two) those in `planes`.
      auto store = [&](auto sums, int col0, int planes) {
        float v[32];
        sums(v);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] *= beta;
        if (SYMMETRIC && tile.i == tile.j) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (col0 + j == row) v[j] += args.diagonal;
        }
        uint32_t w[16];
        if (OP == MUL && args.result != nullptr) {
          if ((planes & 1) == 0) return;
          if (!args.result_tma) {
            if (row < args.rows) store_elements(args, tile.batch, row, col0, v);
            __syncwarp();
          } else if (args.result_dtype == H3B_F32) {
            out.put(&out_hi, v, args.result_t, col0, row0, tile.batch);
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              w[j] = args.result_dtype == H3B_F16 ? pack_f16x2(v[2 * j], v[2 * j + 1]) : pack_bf16x2(v[2 * j], v[2 * j + 1]);
            out.put(&out_hi, w, args.result_t, col0, row0, tile.batch);
          }
          return;
        }
        const bool mirror = SYMMETRIC && tile.i != tile.j;
#pragma unroll
        for (int m = 0; m < (OP == GRAM ? 2 : 1); ++m) {
          if (m == 1) {  // K, from the sums once more (fewer registers than keeping G)
            if (!args.with_k) break;
            sums(v);
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              v[j] *= beta;
              if (!mirror && col0 + j == row) v[j] += args.diagonal;
              v[j] = v[j] * args.k_beta + (col0 + j == row ? args.k_diagonal : 0.0f);
            }
          }
          const CUtensorMap *hi = m == 0 ? &out_hi : &k_hi, *lo = m == 0 ? &out_lo : &k_lo;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            w[j] = pack_f16x2(v[2 * j], v[2 * j + 1]);
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            v[2 * j] -= h.x;
            v[2 * j + 1] -= h.y;
          }
          if (planes & (1 << (2 * m))) {
            out.put(hi, w, false, col0, row0, tile.batch);
            if (mirror) out.put(hi, w, true, col0, row0, tile.batch);
          }
          if (planes & (2 << (2 * m))) {
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = pack_f16x2(v[2 * j], v[2 * j + 1]);
            out.put(lo, w, false, col0, row0, tile.batch);
            if (mirror) out.put(lo, w, true, col0, row0, tile.batch);
          }
        }
      };
      // where both halves' warps store a chunk: G's planes and K's, or first and second
      const int shared_planes = OP == GRAM && args.with_k ? (half ? 12 : 3) : (half ? 2 : 1);
      if constexpr (PARTS == 1) {
        if (row0 >= args.rows) continue;  // warp-uniform, as all that follows
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
          const int col0 = tile.j * SIDE + t % SLICES * COLS + chunk(i) * 32;
          if (col0 < args.cols)
            store([&](float(&v)[32]) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = acc[2 * i + (j >> 4)][j & 15];
            }, col0, COLS > 32 ? 15 : shared_planes);
        }
      } else {
        // Each part gets the parts' sums of one or two of the four blocks of
        // 32 columns (of three parts the first gets two), four columns of
        // all rows after the other (a warp writes 512 bytes at once), where
        // the operands' stages were.
        static_assert(PARTS >= 1 && PARTS <= 4, "a block for each part");
        constexpr int OWN = PARTS == 4 ? 1 : 2;  // blocks of a part, at most
        const auto owner = [](int block) { return PARTS == 3 ? max(block - 1, 0) : block / OWN; };
        const int first = PARTS == 3 ? (part == 0 ? 0 : part + 1) : part * OWN;
        const bool two = OWN == 2 && (PARTS != 3 || part == 0);
        auto share = [&](int from, int block, int p) {
          return static_cast<uint32_t>((((from * OWN + block) * 8 + p) * BM + quad * 32 + lane) * 16);
        };
        __syncwarp();
        cluster_sync();  // every part's products have read their stages
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
          const int block = half + 2 * i;
          const int to_part = owner(block), at = block == 0 ? 0 : owner(block - 1) == to_part ? 1 : 0;
          const uint32_t to = mapa_shared(smem_u32(smem), static_cast<uint32_t>(to_part));
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            const float* x = &acc[2 * i + (p >> 2)][4 * (p & 3)];
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + share(part, at, p)), "f"(x[0]), "f"(x[1]),
                         "f"(x[2]), "f"(x[3])
                         : "memory");
          }
        }
        cluster_sync();
        const int block = two ? half : 0, col0 = tile.j * SIDE + (first + block) * 32;
        const int planes = two ? 15 : shared_planes;
        if (row0 < args.rows && col0 < args.cols)
          store([&](float(&v)[32]) {
#pragma unroll
            for (int p = 0; p < 8; ++p) {
              float4 s = *reinterpret_cast<const float4*>(smem + share(0, block, p));
#pragma unroll
              for (int q = 1; q < PARTS; ++q) {
                const float4 x = *reinterpret_cast<const float4*>(smem + share(q, block, p));
                s.x += x.x;
                s.y += x.y;
                s.z += x.z;
                s.w += x.w;
              }
              v[4 * p] = s.x;
              v[4 * p + 1] = s.y;
              v[4 * p + 2] = s.z;
              v[4 * p + 3] = s.w;
            }
          }, col0, planes);
      }
    }
    if (lane == 0) bulk_wait_group<0>();  // the blocks are in place before the CTA leaves
    __syncwarp();
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

constexpr int MAX_PARTS = 256;  // of a matrix's sum of squares; the threads of a CTA

// Eight elements, from 16-byte words where `wide`; those at and behind `n` are 0.
template <class T>
H3B_DEV void load8(const T* p, int n, bool wide, float (&v)[8]) {
  if (wide) {  // n is a multiple of 8 then
    T e[8];
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.0f;
  }
}

// CTA-wide sum of 256 threads' values, in a fixed order.
H3B_DEV double block_sum(double s) {
  __shared__ double sums[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += sums[i];
  return s;
}

struct Input {
  const void* x;
  int64_t batch_stride, ld;
  int m, n;
  int wide;       // rows in 16-byte words
  double* parts;  // [batch][n_parts]
  int n_parts;
};

// Sums of squares, in 64 bits: a 32-bit square of a gradient of 10^-20 is
// nothing.
template <class T>
__global__ void __launch_bounds__(MAX_PARTS) ortho_squares(const Input in) {
  launch_next();
  const T* base = static_cast<const T*>(in.x) + blockIdx.y * in.batch_stride;
  const unsigned vectors = (in.n + 7) / 8;
  const int64_t items = static_cast<int64_t>(vectors) * in.m, step = static_cast<int64_t>(gridDim.x) * MAX_PARTS;
  double s = 0.0;
#pragma unroll 4
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * MAX_PARTS + threadIdx.x; i < items; i += step) {
    const unsigned r = static_cast<unsigned>(i / vectors), c = static_cast<unsigned>(i - r * static_cast<int64_t>(vectors)) * 8;
    float v[8];
    load8(base + r * in.ld + c, in.n - static_cast<int>(c), in.wide, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fma(static_cast<double>(v[e]), static_cast<double>(v[e]), s);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) in.parts[blockIdx.y * gridDim.x + blockIdx.x] = s;
}

// Planes of SCALE * x / 2^e, 2^e <= |x| < 2^(e+1), and the factor
// 2^e / (|x| + eps) that is left.
struct Output {
  float eps;
  float* factor;
  __half *hi, *lo;  // lo null: one plane holds x
  int64_t batch, ld;
};

struct Scales {
  float s1, s2;  // x * s1 * s2
};
template <class T>
H3B_DEV Scales scales(const Input& in, const Output& out, bool first) {
  const double total = block_sum(threadIdx.x < static_cast<unsigned>(in.n_parts)
                                     ? in.parts[blockIdx.z * in.n_parts + threadIdx.x] : 0.0);
  const double norm = sqrt(total);
  const int e = norm > 0.0 && norm < 1e300 ? ilogb(norm) : 0;
  const int up = 10 - e;  // 2^10 = SCALE; two factors, as one would leave the range of 32 bits
  // (a zero matrix times 1 / eps would be NaN where that, or its square, is infinite)
  const double all = norm > 0.0 || out.eps == 0.0f ? norm + static_cast<double>(out.eps) : 1.0;
  if (first && threadIdx.x == 0) out.factor[blockIdx.z] = static_cast<float>(scalbn(1.0, e) / all);
  return {ldexpf(1.0f, up / 2), ldexpf(1.0f, up - up / 2)};
}

template <class T>
__global__ void __launch_bounds__(MAX_PARTS) ortho_planes(const Input in, const Output out) {
  launch_next();
  wait_previous();
  const Scales k = scales<T>(in, out, blockIdx.x == 0);
  const T* base = static_cast<const T*>(in.x) + blockIdx.z * in.batch_stride;
  const unsigned vectors = (in.n + 7) / 8;
  const int64_t items = static_cast<int64_t>(vectors) * in.m, step = static_cast<int64_t>(gridDim.x) * MAX_PARTS;
#pragma unroll 2
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * MAX_PARTS + threadIdx.x; i < items; i += step) {
    const unsigned r = static_cast<unsigned>(i / vectors), c = static_cast<unsigned>(i - r * static_cast<int64_t>(vectors)) * 8;
    float v[8];
    load8(base + r * in.ld + c, in.n - static_cast<int>(c), in.wide, v);
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = v[2 * e] * k.s1 * k.s2, y = v[2 * e + 1] * k.s1 * k.s2;
      hi[e] = pack_f16x2(x, y);
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[e]));
      lo[e] = pack_f16x2(x - h.x, y - h.y);
    }
    // the planes' rows are multiples of 32 elements apart
    const int64_t at = blockIdx.z * out.batch + r * out.ld + c;
    *reinterpret_cast<uint4*>(out.hi + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if (out.lo != nullptr) *reinterpret_cast<uint4*>(out.lo + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

// The same of x transposed, 64 x 64 elements a CTA.
template <class T>
__global__ void __launch_bounds__(MAX_PARTS) ortho_planes_t(const Input in, const Output out) {
  __shared__ float tile[64][65];
  launch_next();
  wait_previous();
  const Scales k = scales<T>(in, out, blockIdx.x == 0 && blockIdx.y == 0);
  const T* base = static_cast<const T*>(in.x) + blockIdx.z * in.batch_stride;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = warp; i < 64; i += 8)
#pragma unroll
    for (int h = 0; h < 64; h += 32) {
      const int r = r0 + i, c = c0 + h + lane;
      tile[i][h + lane] = r < in.m && c < in.n ? to_f32(base[r * in.ld + c]) * k.s1 * k.s2 : 0.0f;
    }
  __syncthreads();
#pragma unroll
  for (int i = warp; i < 64; i += 8) {
    const int r = c0 + i, c = r0 + 2 * lane;  // of the transposed
    if (r < in.n && c < in.m) {  // a pair may reach into the padding of the plane's row
      const float x = tile[2 * lane][i], y = tile[2 * lane + 1][i];
      const uint32_t hi = pack_f16x2(x, y);
      const int64_t at = blockIdx.z * out.batch + r * out.ld + c;
      *reinterpret_cast<uint32_t*>(out.hi + at) = hi;
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
      if (out.lo != nullptr) *reinterpret_cast<uint32_t*>(out.lo + at) = pack_f16x2(x - h.x, y - h.y);
    }
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

// No steps: x / (|x| + eps).
template <class T>
__global__ void __launch_bounds__(MAX_PARTS) ortho_scale(const Input in, float eps, T* out) {
  wait_previous();
  const double norm = sqrt(block_sum(threadIdx.x < static_cast<unsigned>(in.n_parts)
                                         ? in.parts[blockIdx.z * in.n_parts + threadIdx.x] : 0.0));
  const double inv = 1.0 / (norm + static_cast<double>(eps));
  const T* base = static_cast<const T*>(in.x) + blockIdx.z * in.batch_stride;
  for (int r = blockIdx.x; r < in.m; r += gridDim.x)
    for (int c = threadIdx.x; c < in.n; c += MAX_PARTS)
      out[(static_cast<int64_t>(blockIdx.z) * in.m + r) * in.n + c] =
          from_f32<T>(static_cast<float>(to_f32(base[r * in.ld + c]) * inv));
}

// ---------------------------------------------------------------- hosts

struct Layout {
  int64_t small, large;      // sides of X
  int64_t x_ld, g_ld;        // row strides of the planes of X and of G, K, B
  int64_t x_plane, g_plane;  // elements of a plane, all matrices
  int64_t planes, bytes;     // where the planes begin; all
};

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Sums of squares, factors; planes of X (two, in turn), G, K and B, two each
// (none for matrices that ortho_small takes).
Layout layout(int64_t batch, int64_t m, int64_t n) {
  Layout l;
  l.small = m < n ? m : n;
  l.large = m < n ? n : m;
  l.x_ld = up(l.large, 32);
  l.g_ld = up(l.small, 32);
  l.x_plane = up(batch * l.small * l.x_ld, 128);
  l.g_plane = up(batch * l.small * l.g_ld, 128);
  l.planes = batch * (MAX_PARTS * 8) + up(batch * 4, 256);
  l.bytes = l.planes + (h3b::ortho_small_fits(m, n) ? 0 : (4 * l.x_plane + 6 * l.g_plane) * 2);
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

// Boxes of a map of planes: an operand whose rows are K (128 rows by 64
// elements of K; 64 and 32 for narrow tiles), one whose columns are K (64 rows
// of K by 64), stores.
enum Boxes { BY_ROWS, BY_ROWS_64, BY_ROWS_32, BY_COLUMNS, STORES };

int encode(Maps* maps, const Planes& p, int64_t batch, int64_t rows, int64_t cols, int64_t ld, Boxes boxes) {
  const uint32_t high = boxes == BY_ROWS ? 128 : boxes == BY_COLUMNS || boxes == BY_ROWS_64 ? 64 : 32;
  for (int i = 0; i < 2; ++i) {
    const int rc = h3b::encode_3d(i == 0 ? &maps->hi : &maps->lo, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, i == 0 ? p.hi : p.lo,
                                  cols, rows, batch, ld * 2, rows * ld * 2, boxes == STORES ? 32 : 64, high, 1,
                                  boxes == STORES ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != H3B_OK) return rc;
  }
  return H3B_OK;
}

template <int PAIR, int PARTS, int OP, int SPLIT, int COLS = 128>
int launch(const Maps& a, const Maps& b, const Maps& out, const Maps& k, const Args& args, int64_t tiles, cudaStream_t stream) {
  constexpr size_t smem = smem_bytes<PAIR, PARTS, OP, SPLIT, COLS>();
  static_assert(smem <= 227 * 1024, "shared memory budget");
  static h3b::OncePerDevice once;
  const auto kernel = ortho_product<PAIR, PARTS, OP, SPLIT, COLS>;
  const int rc = h3b::prepare(once, kernel, smem, LAUNCH_REGS);
  if (rc != H3B_OK) return rc;
  // every tile has a cluster of its own where parts share it
  const int64_t most = PARTS > 1 ? tiles : h3b::num_sms() / PAIR;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((tiles < most ? tiles : most) * PAIR * PARTS));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = PAIR * PARTS;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR * PARTS > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a.hi, a.lo, b.hi, b.lo, out.hi, out.lo, k.hi, k.lo, args) == cudaSuccess ? H3B_OK : H3B_ERR_LAUNCH;
}

// Tiles of side `t`, all matrices.
int64_t tiles_of(int64_t rows, int64_t cols, int64_t batch, int64_t t, bool symmetric) {
  const int64_t r = (rows + t - 1) / t, c = (cols + t - 1) / t;
  return batch * (symmetric ? r * (r + 1) / 2 : r * c);
}

// The second operand of a product, for tiles of 128 columns and narrow ones.
struct Operand {
  Maps all, narrow;
};

// Columns of narrow tiles, if they are taken (one round of them): as few as
// there are SMs for.
int narrow_columns(int64_t tiles, bool symmetric) { return symmetric && 4 * tiles <= h3b::num_sms() ? 32 : 64; }

template <int OP, int SPLIT>
int product(const Maps& a, const Operand& b, const Maps& out, const Maps& k, const Args& args, cudaStream_t stream) {
  const int64_t sms = h3b::num_sms();
  const int64_t t1 = tiles_of(args.rows, args.cols, args.batch, 128, OP != MUL);
  const int64_t t2 = tiles_of(args.rows, args.cols, args.batch, 256, OP != MUL);
  // Rounds of tiles times what one takes, in cycles (fitted to 200 x 200 up to
  // 4096 x 4096): a stage of K in three products 1280 (one CTA; its operand
  // reads and copies share the shared-memory port), 1540 (a pair's tile of
  // four times the size), 1100 and 900 (64 and 32 columns), a third of it in
  // one; the beginning and the stores 8000, 14000, 4500 and 3800, and 10000
  // where CTAs hand their sums over.  Of clusters of three with a whole SM
  // for each CTA 45 run at once on 148 SMs, of four 33.
  const int64_t stages = (args.k + KB - 1) / KB, stage = SPLIT ? 1281 : 427;
  const auto rounds = [](int64_t n, int64_t at_once) { return (n + at_once - 1) / at_once; };
  const int64_t single = rounds(t1, sms) * (stages * stage + 8000);
  const int64_t pair = rounds(t2, sms / 2) * (stages * stage * 6 / 5 + 14000);
  const int64_t halves = rounds(t1, sms / 2) * ((stages + 1) / 2 * stage + 10000);
  const int64_t thirds = rounds(t1, sms * 45 / 148) * ((stages + 2) / 3 * stage + 10000);
  const int64_t quarters = rounds(t1, sms * 9 / 40) * ((stages + 3) / 4 * stage + 10000);
  const int narrow = narrow_columns(t1, OP != MUL);
  const int64_t slices = 128 / narrow * t1 > sms ? INT64_MAX
                         : narrow == 64          ? stages * stage * 6 / 7 + 4500
                                                 : stages * stage * 7 / 10 + 3800;
  const int64_t best = std::min({single, pair, halves, thirds, quarters, slices});
  if (single == best) return launch<1, 1, OP, SPLIT>(a, b.all, out, k, args, t1, stream);
  if (pair == best) return launch<2, 1, OP, SPLIT>(a, b.all, out, k, args, t2, stream);
  if (slices == best) {
    if constexpr (OP != MUL)
      if (narrow == 32) return launch<1, 1, OP, SPLIT, 32>(a, b.narrow, out, k, args, 4 * t1, stream);
    return launch<1, 1, OP, SPLIT, 64>(a, b.narrow, out, k, args, 2 * t1, stream);
  }
  if (halves == best) return launch<1, 2, OP, SPLIT>(a, b.all, out, k, args, t1, stream);
  if (thirds == best) return launch<1, 3, OP, SPLIT>(a, b.all, out, k, args, t1, stream);
  return launch<1, 4, OP, SPLIT>(a, b.all, out, k, args, t1, stream);
}

// A small kernel that starts while the one before it ends.
template <class... Params, class... Values>
int launch_after(void (*kernel)(Params...), dim3 grid, cudaStream_t stream, Values... values) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(MAX_PARTS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, values...) == cudaSuccess ? H3B_OK : H3B_ERR_LAUNCH;
}

template <class T>
int run(const h3b::OrthoCall& call, uint8_t* ws, cudaStream_t stream) {
  const T* x = static_cast<const T*>(call.x);
  T* out = static_cast<T*>(call.out);
  const int dtype = call.dtype, steps = call.steps;
  const int64_t batch = call.batch, m = call.m, n = call.n, batch_stride = call.batch_stride, ld = call.ld;
  const float eps = call.eps;
  const Layout l = layout(batch, m, n);
  double* parts = reinterpret_cast<double*>(ws);
  float* factor = reinterpret_cast<float*>(parts + batch * MAX_PARTS);
  __half* at = reinterpret_cast<__half*>(ws + l.planes);
  auto take = [&](int64_t plane) {
    Planes p{at, at + plane};
    at += 2 * plane;
    return p;
  };
  Planes xs[2] = {take(l.x_plane), take(l.x_plane)};
  const Planes g = take(l.g_plane), k = take(l.g_plane), b = take(l.g_plane);
  const int64_t row_bytes = n * static_cast<int64_t>(sizeof(T));
  const bool wide = n % 8 == 0 && h3b::aligned16(x) && ld * static_cast<int64_t>(sizeof(T)) % 16 == 0 &&
                    (batch == 1 || batch_stride * static_cast<int64_t>(sizeof(T)) % 16 == 0);
  // 2048 elements a CTA at least, and CTAs for two an SM together
  const int64_t pieces = ((n + 7) / 8 * m + MAX_PARTS - 1) / MAX_PARTS;
  const int64_t share = (2 * h3b::num_sms() + batch - 1) / batch;
  const int64_t most = pieces < share ? pieces : share;
  const int n_parts = static_cast<int>(most < MAX_PARTS ? most : MAX_PARTS);
  const unsigned nb = static_cast<unsigned>(batch);
  const Input in{x, batch_stride, ld, static_cast<int>(m), static_cast<int>(n), wide ? 1 : 0, parts, n_parts};
  ortho_squares<T><<<dim3(n_parts, nb), MAX_PARTS, 0, stream>>>(in);
  if (steps == 0) return launch_after(ortho_scale<T>, dim3(n_parts, 1, nb), stream, in, eps, out);
  const bool tall = m > n;
  const bool exact = dtype != H3B_F32;  // one plane holds x
  const Output planes{eps, factor, xs[0].hi, exact ? nullptr : xs[0].lo, l.small * l.x_ld, l.x_ld};
  int rc = tall ? launch_after(ortho_planes_t<T>, dim3(static_cast<unsigned>((n + 63) / 64), static_cast<unsigned>((m + 63) / 64), nb),
                               stream, in, planes)
                : launch_after(ortho_planes<T>, dim3(static_cast<unsigned>(pieces < 4 * share ? pieces : 4 * share), 1, nb), stream,
                               in, planes);
  if (rc != H3B_OK) return rc;

  // X by rows and by columns, both sets of planes; G, K (where the square is
  // not completed) and B by rows; all as stores
  const double ca = call.a, cb = call.b, cc = call.c;
  Maps x_out[2], g_out, k_out, b_k, b_out, result;
  Operand x_k[2], x_n[2], g_k, k_k;
  const auto enc = [&](Maps* maps, const Planes& p, int64_t cols, int64_t pitch, Boxes boxes) {
    if (rc == H3B_OK) rc = encode(maps, p, batch, l.small, cols, pitch, boxes);
  };
  const bool square = dtype != H3B_F32 && cc != 0.0 && cb * cb <= 64.0 * cc * cc;
  const int64_t tiles = tiles_of(l.small, l.small, batch, 128, true);  // of the symmetric products
  const Boxes narrow = narrow_columns(tiles, true) == 32 ? BY_ROWS_32 : BY_ROWS_64;
  const auto enc_second = [&](Operand* o, const Planes& p, int64_t cols, int64_t pitch) {
    enc(&o->all, p, cols, pitch, BY_ROWS);
    if (2 * tiles <= h3b::num_sms()) enc(&o->narrow, p, cols, pitch, narrow);
  };
  for (int i = 0; i < (steps > 1 ? 2 : 1); ++i) {
    enc_second(&x_k[i], xs[i], l.large, l.x_ld);
    enc(&x_n[i].all, xs[i], l.large, l.x_ld, BY_COLUMNS);
    x_n[i].narrow = x_n[i].all;
    if (steps > 1) enc(&x_out[i], xs[i], l.large, l.x_ld, STORES);
  }
  enc_second(&g_k, g, l.small, l.g_ld);
  enc(&g_out, g, l.small, l.g_ld, STORES);
  k_k = g_k;
  k_out = g_out;
  if (!square) {
    enc_second(&k_k, k, l.small, l.g_ld);
    enc(&k_out, k, l.small, l.g_ld, STORES);
  }
  enc(&b_k, b, l.small, l.g_ld, BY_ROWS);
  enc(&b_out, b, l.small, l.g_ld, STORES);
  const bool result_tma = row_bytes % 16 == 0 && h3b::aligned16(out);
  if (rc == H3B_OK && result_tma) {
    rc = h3b::encode_3d(&result.hi,
                        dtype == H3B_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                        : dtype == H3B_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                           : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                        out, n, m, batch, row_bytes, m * row_bytes, 64 / sizeof(T), 32, 1, CU_TENSOR_MAP_SWIZZLE_64B);
    result.lo = result.hi;
  } else {
    result = g_out;  // not used
  }

  for (int s = 0; s < steps && rc == H3B_OK; ++s) {
    const bool first = s == 0, last = s == steps - 1;
    const bool x_exact = first && exact;
    const int cur = s & 1;
    Args p{};
    p.batch = static_cast<int>(batch);
    p.rows = p.cols = static_cast<int>(l.small);
    p.k = static_cast<int>(l.large);
    p.factor = first ? factor : nullptr;
    p.b_lo = 1;
    p.beta = 1.0f / SCALE;
    p.diagonal = square ? static_cast<float>(SCALE * cb / (2.0 * cc)) : 0.0f;
    p.k_beta = call.c;
    p.k_diagonal = static_cast<float>(SCALE * cb);
    p.with_k = !square;
    rc = x_exact ? product<GRAM, 0>(x_k[cur].all, x_k[cur], g_out, k_out, p, stream)
                 : product<GRAM, 1>(x_k[cur].all, x_k[cur], g_out, k_out, p, stream);
    if (rc != H3B_OK) break;

    p.factor = nullptr;
    p.k = p.rows;
    if (square) p.beta *= call.c;
    p.diagonal = static_cast<float>(SCALE * (square ? ca - cb * cb / (4.0 * cc) : ca));
    rc = product<POLY, 1>(g_k.all, k_k, b_out, b_out, p, stream);
    if (rc != H3B_OK) break;

    p.factor = first ? factor : nullptr;
    p.beta = 1.0f / SCALE;
    p.cols = static_cast<int>(l.large);
    p.b_lo = !x_exact;
    if (last) {
      p.beta /= SCALE;
      p.result = out;
      p.result_dtype = dtype;
      p.result_t = tall;
      p.result_tma = result_tma;
      p.result_batch = m * n;
      p.result_ld = n;
    }
    const Maps& to = last ? result : x_out[cur ^ 1];
    rc = product<MUL, 1>(b_k, x_n[cur], to, to, p, stream);
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
  const h3b::OrthoCall call{x, out, dtype, batch, m, n, batch_stride, ld, static_cast<int>(steps), a, b, c, eps};
  const auto st = reinterpret_cast<cudaStream_t>(stream);
  if (steps > 0 && h3b::ortho_small_fits(m, n)) return h3b::ortho_small(call, st);
  auto* ws = static_cast<uint8_t*>(workspace);
  if (dtype == H3B_F32) return run<float>(call, ws, st);
  if (dtype == H3B_F16) return run<__half>(call, ws, st);
  return run<__nv_bfloat16>(call, ws, st);
}
