// Newton-Schulz steps (ortho.cu has the formulas) for matrices of which one
// side is at most 128 and the other at most 2048, all steps in one launch.
//
// A cluster of 1 to 8 CTAs holds X [128 rows, zero below the smaller side] in
// shared memory for good: each CTA 256 columns at most, as two f16 planes in
// tiles of 64 columns with the 128-byte swizzle.  The same tile is GRAM's
// operand, K along the row, and MUL's, K down the rows.  A step:
//   G = X X^T over this CTA's columns, into TMEM.  With several CTAs, CTA q
//     gets columns q of the others' sums through distributed shared memory,
//     adds them in order and gives the result to all.
//   B = b G + c G G in every CTA (128^3 products cost less than a hand-over)
//   X = a X + B X over this CTA's columns, in two halves: one is stored while
//     the other's product runs, and the next G begins while that is stored.
// a X and b G are added in fp32 from the planes, which a thread reads and
// overwrites at its own elements.  A launch a product takes 17 launches of 8
// to 18 us here, bound by their beginnings and ends: 24 matrices of
// 128 x 1024 took 165 us.
//
// Planes hold SCALE times the value, as in ortho.cu; the result is read back
// from them (22 bits) so that it leaves in whole rows.  A sum over K stays in
// one accumulator, up to 256 elements long (128 in ortho.cu), which the tensor
// core cuts as often: 96 x 250 in 32 bits is off by 1.4e-6, plain 32-bit
// products by 1.2e-6.
#include <type_traits>

#include "h3b_common.cuh"
#include "h3b_host.hpp"
#include "ortho.hpp"

H3B_DECLARE_STATUS();
H3B_REGISTER_STATUS_READER(ortho_small);

namespace {

constexpr float SCALE = 1024.0f;
constexpr int ROWS = 128;
constexpr int MAX_W = 256;               // columns of a CTA
constexpr int MAX_CTAS = 8;
constexpr int TILE = ROWS * 128;         // bytes of a tile of 64 columns
constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr uint32_t TMEM_COLS = 512;      // B X (columns 0 .. 255), G and G G
constexpr uint32_t G_COL = 256, GG_COL = 384;
enum { GRAM = 0, POLY = 1, MUL = 2, MUL_2 = 3 };  // products, each once a step

struct Args {
  const void* x;
  void* out;
  int64_t batch_stride, ld;
  int m, n, tall;    // tall: X is x transposed
  int rows, cols;    // of X
  int width;         // columns of a CTA, a multiple of 64
  int wide, out_wide;  // rows of x, of the result in 16-byte words of eight elements
  int steps;
  float a, b, c, eps;
};

struct Shared {
  double squares[MAX_CTAS];
  double warp_sums[WARPS];
  uint64_t done[4];
  uint32_t tmem;
  int abort_flag;
};

H3B_DEV float to_f32(float v) { return v; }
H3B_DEV float to_f32(__half v) { return __half2float(v); }
H3B_DEV float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
H3B_DEV T from_f32(float v);
template <>
H3B_DEV float from_f32<float>(float v) { return v; }
template <>
H3B_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
H3B_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Byte offset of columns 8p .. 8p + 7 of row r in tiles of 64 columns.
H3B_DEV uint32_t piece(int r, int p) { return static_cast<uint32_t>((p >> 3) * TILE + r * 128 + (((p & 7) ^ (r & 7)) << 4)); }

H3B_DEV void st_cluster(uint32_t addr, const uint4& v) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}
// The two halves of cluster_sync, in turn; no other barrier of the cluster between.
H3B_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
H3B_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
H3B_DEV void fence_async() { asm volatile("fence.proxy.async;" ::: "memory"); }

// Eight values as pieces of the two planes, and back.
H3B_DEV void split8(const float* v, uint4* hi, uint4* lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = pack_f16x2(v[2 * i], v[2 * i + 1]);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    l[i] = pack_f16x2(v[2 * i] - f.x, v[2 * i + 1] - f.y);
  }
  *hi = make_uint4(h[0], h[1], h[2], h[3]);
  *lo = make_uint4(l[0], l[1], l[2], l[3]);
}
H3B_DEV void join8(const uint4& hi, const uint4& lo, float* v) {
  const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w}, l[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&l[i]));
    v[2 * i] = f.x + g.x;
    v[2 * i + 1] = f.y + g.y;
  }
}

template <class T, int CTAS>
__global__ void __launch_bounds__(THREADS, 1) ortho_small_kernel(const Args args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tiles = args.width / 64;
  // X's planes, then G's (two tiles each); G's bytes also take the other
  // CTAs' sums, and B
  uint8_t* x_hi = smem;
  uint8_t* x_lo = x_hi + tiles * TILE;
  uint8_t* g_hi = x_lo + tiles * TILE;
  uint8_t* g_lo = g_hi + 2 * TILE;
  Shared* sh = reinterpret_cast<Shared*>(g_lo + 2 * TILE);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = CTAS > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int matrix = static_cast<int>(blockIdx.x) / CTAS;
  const int col0 = rank * args.width;
  const int quad = warp & 3, part = warp >> 2, row = quad * 32 + lane;  // this thread's row and columns of an accumulator
  volatile int* abort_flag = &sh->abort_flag;

  if (tid == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(&sh->done[i], 1);
    sh->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(&sh->tmem, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem;
  const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16);
  // Everything in the cluster: shared memory written so far is seen by all,
  // the products' reads of it included.
  auto all_sync = [&] {
    fence_async();
    __syncwarp();
    if constexpr (CTAS > 1)
      cluster_sync();
    else
      __syncthreads();
    fence_async();
  };
  auto local_sync = [&] {
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  };

  // ------------------------------------------------- norm, planes of X
  // First x as it is: the upper 16 bits of an element (as 32 bits) where its
  // first plane will be, the lower ones where the second; 32 elements of a
  // thread in flight, in loops (code that runs once comes from L2: unrolled
  // whole it took longer than the loads).  Then the norm, and each piece in
  // its place.  Where rows of x are whole 16-byte words an item is eight
  // elements, neighbouring threads taking neighbouring items of a row of X, or
  // of a column of it where x is its transpose; else a warp takes rows of x.
  const T* x = static_cast<const T*>(args.x) + matrix * args.batch_stride;
  const int cols = max(0, min(args.width, args.cols - col0));
  const int lines = args.tall ? cols : args.rows, length = args.tall ? args.rows : cols;
  const int per_line = (length + 7) / 8, items = lines * per_line;
  auto item = [&](int i, int* line, int* at) {
    if (args.tall) {
      *line = i % lines;
      *at = i / lines * 8;
    } else {
      *line = i / per_line;
      *at = (i - *line * per_line) * 8;
    }
  };
  auto put_raw = [&](int r, int c, T v) {
    const uint32_t to = piece(r, c >> 3) + (c & 7) * 2;
    const uint32_t bits = __float_as_uint(to_f32(v));
    *reinterpret_cast<uint16_t*>(x_hi + to) = static_cast<uint16_t>(bits >> 16);
    *reinterpret_cast<uint16_t*>(x_lo + to) = static_cast<uint16_t>(bits);
  };
  // zero planes: rows and columns behind the matrix stay so
  for (int i = tid; i < tiles * TILE * 2 / 16; i += THREADS) reinterpret_cast<uint4*>(x_hi)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  double sums[2] = {0.0, 0.0};  // 64 bits: a 32-bit square of 10^-20 is nothing
  auto square_of = [&](T v, int i) { sums[i] = fma(static_cast<double>(to_f32(v)), static_cast<double>(to_f32(v)), sums[i]); };
  x += args.tall ? col0 * args.ld : col0;
  if (args.wide) {
    for (int i0 = tid; i0 < items; i0 += 4 * THREADS) {
      T e[4][8];
      int line[4], at[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + k * THREADS;
        if (i < items) {
          item(i, &line[k], &at[k]);
          const T* p = x + line[k] * args.ld + at[k];
#pragma unroll
          for (int j = 0; j < static_cast<int>(sizeof(T)) / 2; ++j)
            reinterpret_cast<uint4*>(e[k])[j] = reinterpret_cast<const uint4*>(p)[j];
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k * THREADS < items) {
#pragma unroll
          for (int j = 0; j < 8; ++j) square_of(e[k][j], j & 1);
          if (args.tall) {
#pragma unroll
            for (int j = 0; j < 8; ++j) put_raw(at[k] + j, line[k], e[k][j]);
          } else {
            uint32_t h[4], l[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t u = __float_as_uint(to_f32(e[k][2 * j])), v = __float_as_uint(to_f32(e[k][2 * j + 1]));
              h[j] = __byte_perm(u, v, 0x7632);
              l[j] = __byte_perm(u, v, 0x5410);
            }
            *reinterpret_cast<uint4*>(x_hi + piece(line[k], at[k] >> 3)) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(x_lo + piece(line[k], at[k] >> 3)) = make_uint4(l[0], l[1], l[2], l[3]);
          }
        }
    }
  } else {
    auto rows_of_x = [&](auto transposed, auto across) {  // rows of 32 * across elements at most
      constexpr bool T_ = decltype(transposed)::value;
      constexpr int N = decltype(across)::value, L = 32 / N;
      for (int line0 = warp; line0 < lines; line0 += WARPS * L) {
        T e[L][N];
#pragma unroll
        for (int l = 0; l < L; ++l) {
          const int line = line0 + WARPS * l;
          const T* p = x + line * args.ld + lane;
#pragma unroll
          for (int j = 0; j < N; ++j) e[l][j] = line < lines && lane + 32 * j < length ? p[32 * j] : from_f32<T>(0.0f);
        }
#pragma unroll
        for (int l = 0; l < L; ++l)
#pragma unroll
          for (int j = 0; j < N; ++j) square_of(e[l][j], j & 1);
#pragma unroll
        for (int l = 0; l < L; ++l) {
          const int line = line0 + WARPS * l;
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (line < lines && lane + 32 * j < length)
              put_raw(T_ ? lane + 32 * j : line, T_ ? line : lane + 32 * j, e[l][j]);
        }
      }
    };
    if (args.tall)
      rows_of_x(std::true_type{}, std::integral_constant<int, ROWS / 32>{});
    else
      rows_of_x(std::false_type{}, std::integral_constant<int, MAX_W / 32>{});
  }
  double s = sums[0] + sums[1];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) sh->warp_sums[warp] = s;
  __syncthreads();
  if (CTAS > 1) cluster_sync();  // every CTA runs: its shared memory can be written
  if (tid < CTAS) {
    s = 0.0;
    for (int i = 0; i < WARPS; ++i) s += sh->warp_sums[i];
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_shared(smem_u32(&sh->squares[rank]), tid)), "d"(s) : "memory");
  }
  all_sync();
  s = 0.0;
  for (int i = 0; i < CTAS; ++i) s += sh->squares[i];
  // x * SCALE / (norm + eps), as a factor below 2 and two powers of two (one
  // would leave the range of 32 bits)
  const double divisor = sqrt(s) + static_cast<double>(args.eps);
  const int e = divisor > 0.0 && divisor < 1e300 ? ilogb(divisor) : 0;
  const float f = static_cast<float>(static_cast<double>(SCALE) * scalbn(1.0, e) / divisor);
  const float s1 = ldexpf(1.0f, -e / 2), s2 = ldexpf(1.0f, -e + e / 2);
  const int pieces = tiles * 8;
  for (int i = tid; i < args.rows * pieces; i += THREADS) {
    const uint32_t at = piece(i / pieces, i % pieces);
    uint4* hi = reinterpret_cast<uint4*>(x_hi + at);
    uint4* lo = reinterpret_cast<uint4*>(x_lo + at);
    const uint32_t h[4] = {hi->x, hi->y, hi->z, hi->w}, l[4] = {lo->x, lo->y, lo->z, lo->w};
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(__byte_perm(l[j], h[j], 0x5410)) * s1 * s2 * f;
      v[2 * j + 1] = __uint_as_float(__byte_perm(l[j], h[j], 0x7632)) * s1 * s2 * f;
    }
    split8(v, hi, lo);
  }
  local_sync();

  // ------------------------------------------------------------- steps
  // Products stop at the last 16 rows and columns that hold anything; what the
  // planes get behind those is never read.  X is worked on in halves of 128
  // columns: while the second one's product runs the first one is stored, and
  // while the second one is stored the next G takes the first.
  const int k_rows = (args.rows + 15) / 16, k_cols = max(1, (cols + 15) / 16);  // of 16
  const int k_first = min(k_cols, 8), k_second = k_cols - k_first;
  const uint32_t square_d = idesc_f16_f32(ROWS, 16 * static_cast<uint32_t>(k_rows), 0, 0);
  uint32_t parity = 0;
  auto wait_for = [&](int product) {
    mbar_wait<false, false, true>(&sh->done[product], parity, &g_status, 1 + product, abort_flag);  // out of time: noted, and on to the barriers
    __syncwarp();
    tc_fence_after();
  };
  // A A^T over K from 16 `from` to 16 `to` along the planes' rows, the small products first
  auto square = [&](uint32_t d, const uint8_t* hi, const uint8_t* lo, int from, int to, bool add) {
    const uint64_t h = sdesc_kmajor_sw128(smem_u32(hi)), l = sdesc_kmajor_sw128(smem_u32(lo));
    for (int p = 0; p < 3; ++p)
      for (int k = from; k < to; ++k) {
        const uint32_t at = (k >> 2) * (TILE >> 4) + 2 * (k & 3);
        mma_f16_ss(d, (p == 0 ? l : h) + at, (p == 1 ? l : h) + at, square_d, add || p != 0 || k != from);
      }
  };
  // columns 128 i .. of B X, K down the rows of X
  auto product = [&](int i, int n) {
    const uint32_t wide_d = idesc_f16_f32(ROWS, 16 * static_cast<uint32_t>(n), 0, 1);
    const uint64_t bh = sdesc_kmajor_sw128(smem_u32(g_hi)), bl = sdesc_kmajor_sw128(smem_u32(g_lo));
    const uint64_t xh = sdesc_mnmajor_sw128(smem_u32(x_hi + i * 2 * TILE), TILE, 1024);
    const uint64_t xl = sdesc_mnmajor_sw128(smem_u32(x_lo + i * 2 * TILE), TILE, 1024);
    for (int p = 0; p < 3; ++p)
      for (int k = 0; k < k_rows; ++k)
        mma_f16_ss(tmem + 128 * i, (p == 0 ? bl : bh) + (k >> 2) * (TILE >> 4) + 2 * (k & 3),
                   (p == 1 ? xl : xh) + k * (2048 >> 4), wide_d, (p | k) != 0);
    tc_commit(&sh->done[MUL + i]);
  };
  // 32 of its columns: X = a X + B X
  auto store_half = [&](int i, int n) {
    const int c = i * 128 + part * 32;
    if (part * 32 >= 16 * n) return;
    uint32_t r[32];
    tmem_ld32p(t_row + c, r);
    tmem_wait_fence<1>(r);
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
      uint4* hi = reinterpret_cast<uint4*>(x_hi + piece(row, (c + j) >> 3));
      uint4* lo = reinterpret_cast<uint4*>(x_lo + piece(row, (c + j) >> 3));
      float v[8];
      join8(*hi, *lo, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fmaf(args.a, v[e], __uint_as_float(r[j + e]) * (1.0f / SCALE));
      split8(v, hi, lo);
    }
  };
  const bool mine = part * 32 < 16 * k_rows;  // columns of G and B

  if constexpr (CTAS > 1) cluster_arrive();
  if (warp == 0 && elect_one()) square(tmem + G_COL, x_hi, x_lo, 0, k_first, false);
  __syncwarp();
  for (int step = 0; step < args.steps; ++step, parity ^= 1) {
    if (warp == 0 && elect_one()) {
      square(tmem + G_COL, x_hi, x_lo, k_first, k_cols, true);
      tc_commit(&sh->done[GRAM]);
    }
    __syncwarp();
    wait_for(GRAM);
    uint32_t r[32];
    if constexpr (CTAS == 1) {
      if (mine) {
        tmem_ld32p(t_row + G_COL + part * 32, r);
        tmem_wait_fence<1>(r);
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]) * (1.0f / SCALE);
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          uint4 h, l;
          split8(v + j, &h, &l);
          *reinterpret_cast<uint4*>(g_hi + piece(row, part * 4 + (j >> 3))) = h;
          *reinterpret_cast<uint4*>(g_lo + piece(row, part * 4 + (j >> 3))) = l;
        }
      }
      local_sync();
    } else {
      constexpr int OWN = ROWS / CTAS;      // columns of G that a CTA adds up
      constexpr int PART = ROWS * OWN * 4;  // bytes of one CTA's share
      // A share holds four columns of all rows after the other: a warp writes
      // 512 bytes at once (rows 128 bytes apart crossed at a third of that).
      auto share = [](int r, int p) { return static_cast<uint32_t>((p * ROWS + r) * 16); };
      cluster_wait();  // every CTA is done with B
      if (mine) {
        tmem_ld32p(t_row + G_COL + part * 32, r);
        tmem_wait_fence<1>(r);
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const int c = part * 32 + j, owner = c / OWN, p = c % OWN / 4;
          st_cluster(mapa_shared(smem_u32(g_hi) + rank * PART + share(row, p), owner),
                     make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]));
        }
      }
      __syncwarp();
      tc_fence_before();
      cluster_sync();
      // a thread adds eight columns of a row, its neighbours the next eight
      constexpr int ITEMS = ROWS * OWN / 8, SUMS = (ITEMS + THREADS - 1) / THREADS;
      float v[SUMS][8];
#pragma unroll
      for (int k = 0; k < SUMS; ++k) {
        const int i = (tid + k * THREADS) % ITEMS, r = i / (OWN / 8), p = i % (OWN / 8) * 2;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[k][j] = 0.0f;
#pragma unroll
        for (int q = 0; q < CTAS; ++q)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 t = *reinterpret_cast<const float4*>(g_hi + q * PART + share(r, p + h));
            v[k][4 * h] += t.x;
            v[k][4 * h + 1] += t.y;
            v[k][4 * h + 2] += t.z;
            v[k][4 * h + 3] += t.w;
          }
      }
      __syncwarp();
      cluster_arrive();  // the shares have been read: G takes their place
      cluster_wait();
#pragma unroll
      for (int k = 0; k < SUMS; ++k) {
        const int i = tid + k * THREADS, r = i / (OWN / 8), p = i % (OWN / 8);
        if (i < ITEMS) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[k][j] *= 1.0f / SCALE;
          uint4 h, l;
          split8(v[k], &h, &l);
          const uint32_t at = piece(r, rank * (OWN / 8) + p);
#pragma unroll
          for (int q = 0; q < CTAS; ++q) {
            st_cluster(mapa_shared(smem_u32(g_hi) + at, q), h);
            st_cluster(mapa_shared(smem_u32(g_lo) + at, q), l);
          }
        }
      }
      all_sync();
      tc_fence_after();
    }

    if (warp == 0 && elect_one()) {
      square(tmem + GG_COL, g_hi, g_lo, 0, k_rows, false);
      tc_commit(&sh->done[POLY]);
    }
    __syncwarp();
    wait_for(POLY);
    if (mine) {
      tmem_ld32p(t_row + GG_COL + part * 32, r);
      tmem_wait_fence<1>(r);
#pragma unroll
      for (int j = 0; j < 32; j += 8) {
        uint4* hi = reinterpret_cast<uint4*>(g_hi + piece(row, part * 4 + (j >> 3)));
        uint4* lo = reinterpret_cast<uint4*>(g_lo + piece(row, part * 4 + (j >> 3)));
        float v[8];
        join8(*hi, *lo, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(args.b, v[e], __uint_as_float(r[j + e]) * (args.c / SCALE));
        split8(v, hi, lo);
      }
    }
    local_sync();

    if (warp == 0 && elect_one()) {
      product(0, k_first);
      if (k_second > 0) product(1, k_second);
    }
    __syncwarp();
    wait_for(MUL);
    store_half(0, k_first);
    local_sync();
    if (step + 1 < args.steps && warp == 0 && elect_one()) square(tmem + G_COL, x_hi, x_lo, 0, k_first, false);
    __syncwarp();
    if (k_second > 0) {
      wait_for(MUL_2);
      store_half(1, k_second);
      local_sync();
    }
    if (CTAS > 1 && step + 1 < args.steps) cluster_arrive();
  }

  // ------------------------------------------------------------ result
  T* out = static_cast<T*>(args.out) + static_cast<int64_t>(matrix) * args.m * args.n +
           (args.tall ? static_cast<int64_t>(col0) * args.n : col0);
  auto get = [&](int r, int c) {
    const uint32_t from = piece(r, c >> 3) + (c & 7) * 2;
    return (__half2float(*reinterpret_cast<const __half*>(x_hi + from)) +
            __half2float(*reinterpret_cast<const __half*>(x_lo + from))) * (1.0f / SCALE);
  };
  if (!args.out_wide) {
    auto rows_of_x = [&](auto transposed, auto across) {
      constexpr bool T_ = decltype(transposed)::value;
#pragma unroll 2
      for (int line = warp; line < lines; line += WARPS) {
        T* p = out + static_cast<int64_t>(line) * args.n + lane;
#pragma unroll
        for (int j = 0; j < decltype(across)::value; ++j)
          if (lane + 32 * j < length) p[32 * j] = from_f32<T>(T_ ? get(lane + 32 * j, line) : get(line, lane + 32 * j));
      }
    };
    if (args.tall)
      rows_of_x(std::true_type{}, std::integral_constant<int, ROWS / 32>{});
    else
      rows_of_x(std::false_type{}, std::integral_constant<int, MAX_W / 32>{});
  } else {
#pragma unroll 2
    for (int i = tid; i < items; i += THREADS) {
      int line, at;
      item(i, &line, &at);
      float v[8];
      if (!args.tall) {
        join8(*reinterpret_cast<const uint4*>(x_hi + piece(line, at >> 3)),
              *reinterpret_cast<const uint4*>(x_lo + piece(line, at >> 3)), v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= 1.0f / SCALE;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = get(at + j, line);
      }
      T e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = from_f32<T>(v[j]);
      T* p = out + static_cast<int64_t>(line) * args.n + at;
#pragma unroll
      for (int j = 0; j < static_cast<int>(sizeof(T)) / 2; ++j)
        reinterpret_cast<uint4*>(p)[j] = reinterpret_cast<const uint4*>(e)[j];
    }
  }
  // (the last writes between CTAs were G, before the step's last barrier)
  if (warp == 0) tmem_dealloc(tmem, TMEM_COLS);
}

// More than half of an SM's at least: a CTA takes all of TMEM, and of two
// clusters that share SMs each could hold what the other waits for.
size_t smem_bytes(int width) {
  const size_t need = 1024 + static_cast<size_t>(width / 64) * TILE * 2 + 4 * TILE + sizeof(Shared);
  const size_t alone = 116 * 1024;
  return need > alone ? need : alone;
}
static_assert(1024 + MAX_W / 64 * TILE * 2 + 4 * TILE + sizeof(Shared) <= 227 * 1024, "shared memory budget");

template <class T, int CTAS>
int launch(const Args& args, int64_t batch, cudaStream_t stream) {
  const auto kernel = ortho_small_kernel<T, CTAS>;
  static h3b::OncePerDevice once;
  const int rc = h3b::prepare(once, kernel, smem_bytes(MAX_W));
  if (rc != H3B_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(batch * CTAS));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem_bytes(args.width);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CTAS;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CTAS > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args) == cudaSuccess ? H3B_OK : H3B_ERR_LAUNCH;
}

template <class T>
int run(const h3b::OrthoCall& c, cudaStream_t stream) {
  Args a{};
  a.x = c.x;
  a.out = c.out;
  a.batch_stride = c.batch_stride;
  a.ld = c.ld;
  a.m = static_cast<int>(c.m);
  a.n = static_cast<int>(c.n);
  a.tall = c.m > c.n;
  a.rows = a.tall ? a.n : a.m;
  a.cols = a.tall ? a.m : a.n;
  const int64_t size = sizeof(T);
  a.wide = c.n % 8 == 0 && h3b::aligned16(c.x) && c.ld * size % 16 == 0 && (c.batch == 1 || c.batch_stride * size % 16 == 0);
  a.out_wide = c.n % 8 == 0 && h3b::aligned16(c.out);
  a.steps = c.steps;
  a.a = c.a;
  a.b = c.b;
  a.c = c.c;
  a.eps = c.eps;
  // as few CTAs as hold the columns, each with as many
  const int ctas = a.cols <= MAX_W ? 1 : a.cols <= 2 * MAX_W ? 2 : a.cols <= 4 * MAX_W ? 4 : 8;
  a.width = ((a.cols + ctas - 1) / ctas + 63) / 64 * 64;
  if (ctas == 1) return launch<T, 1>(a, c.batch, stream);
  if (ctas == 2) return launch<T, 2>(a, c.batch, stream);
  if (ctas == 4) return launch<T, 4>(a, c.batch, stream);
  return launch<T, 8>(a, c.batch, stream);
}

}  // namespace

namespace h3b {

bool ortho_small_fits(int64_t m, int64_t n) {
  return (m < n ? m : n) <= ROWS && (m < n ? n : m) <= MAX_CTAS * MAX_W;
}

int ortho_small(const OrthoCall& call, cudaStream_t stream) {
  if (call.dtype == H3B_F32) return run<float>(call, stream);
  if (call.dtype == H3B_F16) return run<__half>(call, stream);
  return run<__nv_bfloat16>(call, stream);
}

}  // namespace h3b
