// Layer norm over the last axis of x [m, n], forward and backward.
//
//   y = xhat w + b,   xhat = (x - mean) rstd,   rstd = 1 / sqrt(var + eps)
//   g = dy w,   dx = rstd (g - mean(g) - xhat mean(g xhat))
//   dw = sum_rows dy xhat,   db = sum_rows dy
//
// Both directions are bound by HBM: x is read and y written once; backward, x
// and dy are read and dx written once.  Arithmetic is packed, two elements an
// instruction, or it would bind first.  Rows are held in registers, each by a
// group of threads (forward mostly four rows by a few warps together), so the
// variance is taken about the mean in a second pass over registers, and what
// rounding the mean left over is taken off with it: var = mean(d^2) -
// mean(d)^2, d = x - mean, with mean(d) of the size of a rounding.  Forward
// that keeps the accuracy of 32 bits for any mean.  Backward x - mean comes
// from the mean as it is stored, one 32-bit number: xhat is off by 2^-24 |mean|
// rstd in the whole row (5e-4 where the mean is 10^4 deviations away, as in
// plain 32-bit arithmetic).
//
// The weights' gradients are sums over all rows.  Each CTA walks rows with a
// stride and keeps its threads' columns of both sums in registers (32-bit),
// adds its groups' sums in order through shared memory and writes one partial
// row; a second launch adds the partial rows of a column in order.  No
// atomics: results do not depend on scheduling.
#include <type_traits>

#include "h3b_common.cuh"
#include "h3b_host.hpp"

H3B_DECLARE_STATUS();
H3B_REGISTER_STATUS_READER(layer_norm);

namespace {

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

// VEC consecutive elements: one 16-byte word, or one element.
template <class T, int VEC>
struct Pack {
  T e[VEC];
};
template <class T, int VEC>
H3B_DEV Pack<T, VEC> load_pack(const T* p) {
  Pack<T, VEC> r;
  if constexpr (VEC == 1) {
    r.e[0] = *p;
  } else {
    static_assert(VEC * sizeof(T) == 16, "one 16-byte word");
    *reinterpret_cast<uint4*>(r.e) = *reinterpret_cast<const uint4*>(p);
  }
  return r;
}
template <class T, int VEC>
H3B_DEV void store_pack(T* p, const Pack<T, VEC>& r) {
  if constexpr (VEC == 1)
    *p = r.e[0];
  else
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(r.e);
}
// Pairs of elements, for packed fp32 arithmetic.
H3B_DEV float2 pair_of(uint32_t w, __nv_bfloat16) { return make_float2(bf16lo_to_f32(w), bf16hi_to_f32(w)); }
H3B_DEV float2 pair_of(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <class T, int VEC>
H3B_DEV float2 get2(const Pack<T, VEC>& p, int i) {  // elements 2 i, 2 i + 1
  if constexpr (sizeof(T) == 4)
    return make_float2(p.e[2 * i], p.e[2 * i + 1]);
  else
    return pair_of(reinterpret_cast<const uint32_t*>(p.e)[i], T());
}
template <class T, int VEC>
H3B_DEV void set2(Pack<T, VEC>& p, int i, float2 v) {
  if constexpr (sizeof(T) == 4) {
    p.e[2 * i] = v.x;
    p.e[2 * i + 1] = v.y;
  } else if constexpr (std::is_same<T, __half>::value) {
    reinterpret_cast<uint32_t*>(p.e)[i] = pack_f16x2(v.x, v.y);
  } else {
    reinterpret_cast<uint32_t*>(p.e)[i] = pack_bf16x2(v.x, v.y);
  }
}
H3B_DEV float2 both(float v) { return make_float2(v, v); }
// Pair q of a thread's elements: of a vector, or of two vectors of one.
template <class T, int VEC, int N>
H3B_DEV float2 pair_at(const Pack<T, VEC> (&v)[N], int q) {
  if constexpr (VEC == 1)
    return make_float2(to_f32(v[2 * q].e[0]), to_f32(v[2 * q + 1].e[0]));
  else
    return get2(v[2 * q / VEC], 2 * q % VEC / 2);
}
template <class T, int VEC, int N>
H3B_DEV void set_pair(Pack<T, VEC> (&v)[N], int q, float2 x) {
  if constexpr (VEC == 1) {
    v[2 * q].e[0] = from_f32<T>(x.x);
    v[2 * q + 1].e[0] = from_f32<T>(x.y);
  } else {
    set2(v[2 * q / VEC], 2 * q % VEC / 2, x);
  }
}

// VEC weights of type WT (float beside a 16-bit T takes two words).
template <class WT, int VEC>
struct Weights {
  static constexpr int N = VEC == 1 ? 1 : 16 / sizeof(WT);
  Pack<WT, N> p[VEC / N];
  H3B_DEV void load(const WT* at) {
#pragma unroll
    for (int i = 0; i < VEC / N; ++i) p[i] = load_pack<WT, N>(at + i * N);
  }
  H3B_DEV void fill(float v) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[i / N].e[i % N] = from_f32<WT>(v);
  }
  H3B_DEV float operator[](int i) const { return to_f32(p[i / N].e[i % N]); }
  H3B_DEV float2 pair(int i) const { return get2(p[2 * i / N], 2 * i % N / 2); }
};
template <class WT, int VEC, int N>
H3B_DEV float2 pair_at(const Weights<WT, VEC> (&w)[N], int q) {
  if constexpr (VEC == 1)
    return make_float2(w[2 * q][0], w[2 * q + 1][0]);
  else
    return w[2 * q / VEC].pair(2 * q % VEC / 2);
}

// Sums of two values over a group of TPR threads (a row), the same in all of
// them.  Groups of up to a warp by shuffles; larger ones are a whole CTA and
// alternate between two sets of slots, so one barrier a sum is enough.
template <int TPR>
struct RowSum {
  static_assert(TPR <= 32 || TPR % 32 == 0, "whole warps");
  float2 (*slots)[32];
  int set = 0;
  H3B_DEV float2 operator()(float a, float b) {
    constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if constexpr (TPR > 32) {
      float2* s = slots[set];
      set ^= 1;
      if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = make_float2(a, b);
      __syncthreads();
      a = b = 0.0f;
#pragma unroll
      for (int i = 0; i < TPR / 32; ++i) {
        const float2 t = s[i];
        a += t.x;
        b += t.y;
      }
    }
    return make_float2(a, b);
  }
};

// Both sums of each of N rows over their group of TPR threads, behind one
// barrier; `slots` are used by every other call.
template <int TPR, int N>
H3B_DEV void row_sums(float (&a)[N], float (&b)[N], float2 (*slots)[32]) {
  constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      a[k] += __shfl_xor_sync(0xffffffffu, a[k], o);
      b[k] += __shfl_xor_sync(0xffffffffu, b[k], o);
    }
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) slots[k][threadIdx.x >> 5] = make_float2(a[k], b[k]);
    __syncthreads();
    const int first = threadIdx.x / TPR * (TPR / 32);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      a[k] = b[k] = 0.0f;
#pragma unroll
      for (int i = 0; i < TPR / 32; ++i) {
        const float2 t = slots[k][first + i];
        a[k] += t.x;
        b[k] += t.y;
      }
    }
  }
}

template <int N>
H3B_DEV float half_of(const float2 (&p)[N], int j) { return j & 1 ? p[j / 2].y : p[j / 2].x; }

// Rows of a warp or less share a CTA; larger groups are a CTA (RowSum).
constexpr int EPT = 16;  // elements of a row that a thread holds, backward
constexpr int block_threads(int tpr) { return tpr <= 32 ? 128 : tpr; }

// From mean(d^2) and mean(d).  A rounding must not leave less than nothing; a
// NaN stays one (fmaxf would drop it).
H3B_DEV float inverse_std(float d2, float dm, float eps) {
  const float var = fmaf(-dm, dm, d2);
  return __frsqrt_rn((var < 0.0f ? 0.0f : var) + eps);
}

// ----------------------------------------------------------------- forward

struct FwdArgs {
  const void *x, *w, *b;
  void* y;
  float *mean, *rstd;
  int64_t m, n, ldx, ldy;
  float eps;
};

// TPR threads a row, HELD elements a thread at most.
template <class T, class WT, int VEC, int TPR, int HELD>
__global__ void __launch_bounds__(block_threads(TPR)) ln_fwd_kernel(const FwdArgs a) {
  constexpr int MAXV = HELD / VEC;
  constexpr int GROUPS = block_threads(TPR) / TPR;
  __shared__ float2 slots[2][32];
  RowSum<TPR> sum{slots};
  const int t = threadIdx.x % TPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + threadIdx.x / TPR;
  const bool live = row < a.m;  // a group without a row still takes part in its warp's shuffles
  const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.ldx;
  const int n = static_cast<int>(a.n);
  const int nv = (n + VEC - 1) / VEC;
  const float inv_n = 1.0f / static_cast<float>(n);

  Pack<T, VEC> v[MAXV];
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int c = t + i * TPR;
    if (c < nv) v[i] = load_pack<T, VEC>(x + static_cast<int64_t>(c) * VEC);
  }
  float2 s = both(0.0f);
#pragma unroll
  for (int i = 0; i < MAXV; ++i)
    if (t + i * TPR < nv) {
      if constexpr (VEC == 1) {
        s.x += to_f32(v[i].e[0]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) s = add2(s, get2(v[i], j));
      }
    }
  const float m0 = sum(s.x + s.y, 0.0f).x * inv_n;
  float2 s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
  for (int i = 0; i < MAXV; ++i)
    if (t + i * TPR < nv) {
      if constexpr (VEC == 1) {
        const float d = to_f32(v[i].e[0]) - m0;
        s1.x += d;
        s2.x = fmaf(d, d, s2.x);
      } else {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
          const float2 d = add2(get2(v[i], j), both(-m0));
          s1 = add2(s1, d);
          s2 = fma2(d, d, s2);
        }
      }
    }
  const float2 r = sum(s1.x + s1.y, s2.x + s2.y);
  const float dm = r.x * inv_n;
  const float rstd = inverse_std(r.y * inv_n, dm, a.eps);
  if (!live) return;
  if (a.mean != nullptr && t == 0) {
    a.mean[row] = m0 + dm;
    a.rstd[row] = rstd;
  }
  T* y = static_cast<T*>(a.y) + row * a.ldy;
  const WT* w = static_cast<const WT*>(a.w);
  const WT* b = static_cast<const WT*>(a.b);
  const float shift = -dm * rstd;
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int c = t + i * TPR;
    if (c < nv) {
      Weights<WT, VEC> wv, bv;
      if (w != nullptr) wv.load(w + c * VEC);
      if (b != nullptr) bv.load(b + c * VEC);
      if constexpr (VEC == 1) {
        float h = fmaf(to_f32(v[i].e[0]) - m0, rstd, shift);
        if (w != nullptr) h *= wv[0];
        if (b != nullptr) h += bv[0];
        v[i].e[0] = from_f32<T>(h);
      } else {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
          float2 h = fma2(add2(get2(v[i], j), both(-m0)), both(rstd), both(shift));
          if (w != nullptr)
            h = b != nullptr ? fma2(h, wv.pair(j), bv.pair(j)) : mul2(h, wv.pair(j));
          else if (b != nullptr)
            h = add2(h, bv.pair(j));
          set2(v[i], j, h);
        }
      }
      store_pack<T, VEC>(y + static_cast<int64_t>(c) * VEC, v[i]);
    }
  }
}

// N values of every lane, summed over the warp: lane l gets the sum of value
// l N / 32 in v[0].  Halves of the values change sides while there are several.
template <int N>
H3B_DEV void fold(float (&v)[N]) {
  int have = N;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (have > 1) {
      have /= 2;
      const bool upper = threadIdx.x & o;
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        if (i < have) {
          const float other = __shfl_xor_sync(0xffffffffu, upper ? v[i] : v[i + have], o);
          v[i] = (upper ? v[i + have] : v[i]) + other;
        }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
}

// WARPS warps hold R rows together, PACKS 16-byte words of each a thread: the
// weights of its columns are loaded once for the R.
template <class T, class WT, int VEC, int WARPS, int R, int PACKS>
__global__ void __launch_bounds__(32 * WARPS) ln_fwd_rows_kernel(const FwdArgs a) {
  constexpr int THREADS = 32 * WARPS;
  __shared__ float means[R][WARPS], squares[2 * R][WARPS];
  auto total = [](const float (&of_warps)[WARPS]) {
    float s = of_warps[0];
#pragma unroll
    for (int i = 1; i < WARPS; ++i) s += of_warps[i];
    return s;
  };
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * R;
  const int rows = static_cast<int>(a.m - row0 < R ? a.m - row0 : R);
  const T* x = static_cast<const T*>(a.x) + row0 * a.ldx;
  const int n = static_cast<int>(a.n), nv = n / VEC;
  const float inv_n = 1.0f / static_cast<float>(n);
  Pack<T, VEC> v[R][PACKS];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      const int c = t + i * THREADS;
      if (c < nv && r < rows) {
        v[r][i] = load_pack<T, VEC>(x + r * a.ldx + c * VEC);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[r][i].e[j] = from_f32<T>(0.0f);
      }
    }
  float m0[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float2 s = both(0.0f);
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) s = add2(s, get2(v[r][i], j));
    m0[r] = s.x + s.y;
  }
  fold(m0);
  if (lane % (32 / R) == 0) means[lane / (32 / R)][warp] = m0[0];
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) m0[r] = total(means[r]) * inv_n;
  float s[2 * R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float2 s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
      if (t + i * THREADS < nv) {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
          const float2 d = add2(get2(v[r][i], j), both(-m0[r]));
          s1 = add2(s1, d);
          s2 = fma2(d, d, s2);
        }
      }
    s[r] = s1.x + s1.y;
    s[R + r] = s2.x + s2.y;
  }
  fold(s);
  if (lane % (16 / R) == 0) squares[lane / (16 / R)][warp] = s[0];
  __syncthreads();
  float rstd[R], shift[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float dm = total(squares[r]) * inv_n;
    rstd[r] = inverse_std(total(squares[R + r]) * inv_n, dm, a.eps);
    shift[r] = -dm * rstd[r];
    if (a.mean != nullptr && t == r && r < rows) {
      a.mean[row0 + r] = m0[r] + dm;
      a.rstd[row0 + r] = rstd[r];
    }
  }
  T* y = static_cast<T*>(a.y) + row0 * a.ldy;
  const WT* w = static_cast<const WT*>(a.w);
  const WT* b = static_cast<const WT*>(a.b);
#pragma unroll
  for (int i = 0; i < PACKS; ++i) {
    const int c = t + i * THREADS;
    if (c < nv) {
      Weights<WT, VEC> wv, bv;
      if (w != nullptr) wv.load(w + c * VEC);
      if (b != nullptr) bv.load(b + c * VEC);
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
          float2 h = fma2(add2(get2(v[r][i], j), both(-m0[r])), both(rstd[r]), both(shift[r]));
          if (w != nullptr)
            h = b != nullptr ? fma2(h, wv.pair(j), bv.pair(j)) : mul2(h, wv.pair(j));
          else if (b != nullptr)
            h = add2(h, bv.pair(j));
          set2(v[r][i], j, h);
        }
        if (r < rows) store_pack<T, VEC>(y + r * a.ldy + c * VEC, v[r][i]);
      }
    }
  }
}

// Rows longer than 32 x 1024 elements: a CTA a row, read three times (from L2
// after the first), element by element.
template <class T, class WT>
__global__ void __launch_bounds__(1024) ln_fwd_long_kernel(const FwdArgs a) {
  __shared__ float2 slots[2][32];
  RowSum<1024> sum{slots};
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const float inv_n = 1.0f / static_cast<float>(a.n);
  float s = 0.0f;
  for (int64_t c = threadIdx.x; c < a.n; c += 1024) s += to_f32(x[c]);
  const float m0 = sum(s, 0.0f).x * inv_n;
  float s1 = 0.0f, s2 = 0.0f;
  for (int64_t c = threadIdx.x; c < a.n; c += 1024) {
    const float d = to_f32(x[c]) - m0;
    s1 += d;
    s2 = fmaf(d, d, s2);
  }
  const float2 r = sum(s1, s2);
  const float dm = r.x * inv_n;
  const float rstd = inverse_std(r.y * inv_n, dm, a.eps);
  if (a.mean != nullptr && threadIdx.x == 0) {
    a.mean[row] = m0 + dm;
    a.rstd[row] = rstd;
  }
  T* y = static_cast<T*>(a.y) + row * a.ldy;
  for (int64_t c = threadIdx.x; c < a.n; c += 1024) {
    float h = ((to_f32(x[c]) - m0) - dm) * rstd;
    if (a.w != nullptr) h *= to_f32(static_cast<const WT*>(a.w)[c]);
    if (a.b != nullptr) h += to_f32(static_cast<const WT*>(a.b)[c]);
    y[c] = from_f32<T>(h);
  }
}

// ---------------------------------------------------------------- backward

struct BwdArgs {
  const void *dy, *x, *w;
  const float *mean, *rstd;
  void *dx, *dw, *db;
  float* partial;  // [ctas][2][n]: sums of dy xhat, of dy
  int64_t m, n, lddy, ldx, lddx;
  int sums;        // write partials
};

// Backward, groups of any size share a CTA of 256 threads: their sums of the
// columns are joined before they are written.  Two such CTAs an SM (three and
// four, with fewer registers each, are slower).
constexpr int bwd_threads(int tpr) { return tpr < 256 ? 256 : tpr; }
constexpr int bwd_ctas_per_sm(int tpr) { return bwd_threads(tpr) == 256 ? 2 : 1; }

// 16-bit rows come through a ring of RING rounds in shared memory, fetched by
// bulk copies while earlier ones are worked on: 16384 x 4096 without the sums
// takes 70 us, with four rounds 77, with loads into registers 78.  Rows of a
// warp would wait for each other (131072 x 512: 84, without the ring 71).
// 32-bit rows have twice the bytes for the same arithmetic, and two CTAs'
// loads in turn are enough.
constexpr int RING = 6;
constexpr bool bwd_ring(int element, int vec, int tpr) { return element == 2 && vec > 1 && tpr >= 64 && tpr <= 512; }

template <class T, class WT, int VEC, int TPR>
__global__ void __launch_bounds__(bwd_threads(TPR), VEC > 1 ? bwd_ctas_per_sm(TPR) : 1) ln_bwd_kernel(const BwdArgs a) {
  constexpr int MAXV = EPT / VEC;
  constexpr int THREADS = bwd_threads(TPR);
  constexpr int GROUPS = THREADS / TPR;
  // Rows that a group works on together, their sums behind one barrier: two
  // of 16 bits (32768 x 2048 in 77 us, one 86), one of 32 (8192 x 4096 in 70
  // us, two are a sixth slower).  CTAs of 1024 threads have 64 registers a
  // thread: one row, and the weights again for each (from L1).
  constexpr bool SMALL = THREADS == 1024;
  constexpr int ROWS = SMALL || sizeof(T) == 4 || VEC == 1 ? 1 : 2;
  constexpr bool FETCHED = bwd_ring(sizeof(T), VEC, TPR);
  __shared__ float2 slots[2][ROWS][32];
  __shared__ uint64_t full[RING];
  // the ring, [RING][x, dy][GROUPS][n]; then groups' sums, where there are several, [GROUPS][TPR * EPT]
  extern __shared__ __align__(128) uint8_t smem[];
  float2* joined = reinterpret_cast<float2*>(smem);
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const int n = static_cast<int>(a.n);
  const int nv = (n + VEC - 1) / VEC;
  const float inv_n = 1.0f / static_cast<float>(n);
  const WT* w = static_cast<const WT*>(a.w);

  Weights<WT, VEC> wv[MAXV];
  auto load_weights = [&] {
#pragma unroll
    for (int i = 0; i < MAXV; ++i) {
      const int c = t + i * TPR;
      wv[i].fill(c < nv ? 1.0f : 0.0f);  // beyond the row there is nothing
      if (w != nullptr && c < nv) wv[i].load(w + c * VEC);
    }
  };
  if (!SMALL) load_weights();
  constexpr int PAIRS = EPT / 2;
  float2 sw[PAIRS], sb[PAIRS];
#pragma unroll
  for (int q = 0; q < PAIRS; ++q) sw[q] = sb[q] = both(0.0f);
  int set = 0;
  // Every group of the CTA makes the same number of rounds (the row sums need
  // whole warps); one without a row adds zeros and writes nothing.
  const int64_t step = static_cast<int64_t>(gridDim.x) * GROUPS;
  const uint32_t row_bytes = static_cast<uint32_t>(n * sizeof(T)), tensor_bytes = GROUPS * row_bytes;
  auto fetch = [&](int64_t first, int slot) {  // a round's rows; warp 0
    const int rows = static_cast<int>(a.m - first < GROUPS ? a.m - first : GROUPS);
    if (threadIdx.x == 0) mbar_arrive_expect_tx(&full[slot], 2 * static_cast<uint32_t>(rows) * row_bytes);
    __syncwarp();
    const int r = static_cast<int>(threadIdx.x);
    if (r < rows) {
      uint8_t* to = smem + 2 * slot * tensor_bytes + r * row_bytes;
      bulk_load(to, static_cast<const T*>(a.x) + (first + r) * a.ldx, row_bytes, &full[slot]);
      bulk_load(to + tensor_bytes, static_cast<const T*>(a.dy) + (first + r) * a.lddy, row_bytes, &full[slot]);
    }
  };
  int slot = 0;
  uint32_t parity = 0;
  if constexpr (FETCHED) {
    static_assert(RING % ROWS == 0, "whole iterations");
    if (threadIdx.x == 0) {
      for (int i = 0; i < RING; ++i) mbar_init(&full[i], 1);
      fence_barrier_init();
    }
    __syncthreads();
    if (threadIdx.x < 32)
      for (int i = 0; i < RING; ++i) {
        const int64_t first = static_cast<int64_t>(blockIdx.x) * GROUPS + i * step;
        if (first < a.m) fetch(first, i);
      }
  }
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * GROUPS; base < a.m; base += ROWS * step) {
    Pack<T, VEC> vx[ROWS][MAXV], vg[ROWS][MAXV];
    float rstd[ROWS], shift[ROWS];
    bool live[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const int64_t row = base + k * step + group;
      live[k] = row < a.m;
      rstd[k] = shift[k] = 0.0f;
      if (FETCHED && live[k]) {
        shift[k] = -a.mean[row];
        rstd[k] = a.rstd[row];
      }
    }
    auto load_row = [&](int k) {
      const int64_t row = base + k * step + group;
      const T* x = static_cast<const T*>(a.x) + row * a.ldx;
      const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
      if constexpr (FETCHED) {
        x = reinterpret_cast<const T*>(smem + 2 * (slot + k) * tensor_bytes + group * row_bytes);
        dy = reinterpret_cast<const T*>(smem + (2 * (slot + k) + 1) * tensor_bytes + group * row_bytes);
      }
#pragma unroll
      for (int i = 0; i < MAXV; ++i) {
        const int c = t + i * TPR;
        if (live[k] && c < nv) {
          vx[k][i] = load_pack<T, VEC>(x + static_cast<int64_t>(c) * VEC);
          vg[k][i] = load_pack<T, VEC>(dy + static_cast<int64_t>(c) * VEC);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) vx[k][i].e[j] = vg[k][i].e[j] = from_f32<T>(0.0f);
        }
      }
    };
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      if (FETCHED && base + k * step < a.m) mbar_wait(&full[slot + k], parity, &g_status, 1, nullptr);  // out of time: noted
      load_row(k);
      if (!FETCHED && live[k]) {
        shift[k] = -a.mean[base + k * step + group];
        rstd[k] = a.rstd[base + k * step + group];
      }
    }
    if (SMALL) load_weights();
    float s1[ROWS], s2[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      float2 p1 = both(0.0f), p2 = both(0.0f);
#pragma unroll
      for (int q = 0; q < PAIRS; ++q) {
        const float2 xm = add2(pair_at(vx[k], q), both(shift[k]));  // x - mean = xhat / rstd
        const float2 d = pair_at(vg[k], q), w = pair_at(wv, q);
        const float2 e = mul2(d, xm);
        p1 = fma2(d, w, p1);
        p2 = fma2(e, w, p2);
        sw[q] = fma2(e, both(rstd[k]), sw[q]);
        sb[q] = add2(sb[q], d);
      }
      s1[k] = p1.x + p1.y;
      s2[k] = p2.x + p2.y;
    }
    row_sums<TPR, ROWS>(s1, s2, slots[set]);
    set ^= 1;
    if constexpr (FETCHED) {
      // a barrier was among the sums: all threads are done with the rounds before these
      if (threadIdx.x < 32 && base >= ROWS * step)
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
          const int64_t next = base + (RING - ROWS + k) * step;
          if (next < a.m) fetch(next, (slot == 0 ? RING : slot) - ROWS + k);
        }
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      // dx = rstd (g - c1) - rstd^2 c2 (x - mean), with c2 = rstd mean(g (x - mean))
      const float c1 = -s1[k] * inv_n * rstd[k], c2 = -s2[k] * inv_n * rstd[k] * rstd[k] * rstd[k];
      if (FETCHED) load_row(k);  // once more: both rows' would not fit in registers beside the sums
#pragma unroll
      for (int q = 0; q < PAIRS; ++q) {
        const float2 xm = add2(pair_at(vx[k], q), both(shift[k]));
        const float2 g = mul2(pair_at(vg[k], q), pair_at(wv, q));
        set_pair(vx[k], q, fma2(g, both(rstd[k]), fma2(xm, both(c2), both(c1))));
      }
      T* dx = static_cast<T*>(a.dx) + (base + k * step + group) * a.lddx;
#pragma unroll
      for (int i = 0; i < MAXV; ++i) {
        const int c = t + i * TPR;
        if (live[k] && c < nv) store_pack<T, VEC>(dx + static_cast<int64_t>(c) * VEC, vx[k][i]);
      }
    }
    if constexpr (FETCHED) {
      slot += ROWS;
      if (slot == RING) {
        slot = 0;
        parity ^= 1;
      }
    }
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (!a.sums) return;
  float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.n;
  if constexpr (GROUPS > 1) {
    if constexpr (FETCHED) __syncthreads();  // the ring's last rows have been read
#pragma unroll
    for (int i = 0; i < MAXV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        joined[group * TPR * EPT + (t + i * TPR) * VEC + j] = make_float2(half_of(sw, i * VEC + j), half_of(sb, i * VEC + j));
    __syncthreads();
    for (int c = threadIdx.x; c < n; c += THREADS) {
      float2 s = joined[c];
      for (int g = 1; g < GROUPS; ++g) s = add2(s, joined[g * TPR * EPT + c]);
      out[c] = s.x;
      out[n + c] = s.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < MAXV; ++i) {
      const int c = t + i * TPR;
      if (c < nv) {
        if constexpr (VEC == 1) {
          out[c] = half_of(sw, i);
          out[n + c] = half_of(sb, i);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; j += 4) {
            const int q = (i * VEC + j) / 2;
            *reinterpret_cast<float4*>(out + c * VEC + j) = make_float4(sw[q].x, sw[q].y, sw[q + 1].x, sw[q + 1].y);
            *reinterpret_cast<float4*>(out + n + c * VEC + j) = make_float4(sb[q].x, sb[q].y, sb[q + 1].x, sb[q + 1].y);
          }
        }
      }
    }
  }
}

// Rows longer than 16 x 1024 elements: dx, a CTA a row.
template <class T, class WT>
__global__ void __launch_bounds__(1024) ln_bwd_long_kernel(const BwdArgs a) {
  __shared__ float2 slots[2][32];
  RowSum<1024> sum{slots};
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
  const WT* w = static_cast<const WT*>(a.w);
  const float mean = a.mean[row], rstd = a.rstd[row];
  const float inv_n = 1.0f / static_cast<float>(a.n);
  float s1 = 0.0f, s2 = 0.0f;
  for (int64_t c = threadIdx.x; c < a.n; c += 1024) {
    const float g = to_f32(dy[c]) * (w != nullptr ? to_f32(w[c]) : 1.0f);
    s1 += g;
    s2 = fmaf(g, (to_f32(x[c]) - mean) * rstd, s2);
  }
  const float2 r = sum(s1, s2);
  const float c1 = r.x * inv_n, c2 = r.y * inv_n;
  T* dx = static_cast<T*>(a.dx) + row * a.lddx;
  for (int64_t c = threadIdx.x; c < a.n; c += 1024) {
    const float g = to_f32(dy[c]) * (w != nullptr ? to_f32(w[c]) : 1.0f);
    dx[c] = from_f32<T>(rstd * (fmaf(-(to_f32(x[c]) - mean) * rstd, c2, g) - c1));
  }
}

// The column sums of such rows: 256 columns and every gridDim.y-th row a CTA.
template <class T>
__global__ void __launch_bounds__(256) ln_bwd_long_sums_kernel(const BwdArgs a) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= a.n) return;
  float sw = 0.0f, sb = 0.0f;
  for (int64_t row = blockIdx.y; row < a.m; row += gridDim.y) {
    const float d = to_f32(static_cast<const T*>(a.dy)[row * a.lddy + c]);
    sw = fmaf(d, (to_f32(static_cast<const T*>(a.x)[row * a.ldx + c]) - a.mean[row]) * a.rstd[row], sw);
    sb += d;
  }
  float* out = a.partial + static_cast<int64_t>(blockIdx.y) * 2 * a.n;
  out[c] = sw;
  out[a.n + c] = sb;
}

// dw and db from the partial rows, in order: each of a CTA's 32 warps reads 32
// columns of every 32nd partial row, the first one adds the warps' sums.
template <class WT>
__global__ void __launch_bounds__(1024) ln_bwd_join_kernel(const float* partial, int ctas, int64_t n, WT* dw, WT* db) {
  __shared__ float part[32][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // for the partial rows
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  const int64_t which = dw == nullptr ? 1 : blockIdx.y;
  float s = 0.0f;
  if (c < n)
    for (int p0 = warp; p0 < ctas; p0 += 32 * 10) {  // (two CTAs an SM: once, all loads in flight)
      float v[10];
#pragma unroll
      for (int i = 0; i < 10; ++i) {
        const int p = p0 + 32 * i;
        v[i] = p < ctas ? partial[(static_cast<int64_t>(p) * 2 + which) * n + c] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 10; ++i) s += v[i];
    }
  part[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < n) {
#pragma unroll
    for (int i = 1; i < 32; ++i) s += part[i][lane];
    (which == 0 ? dw : db)[c] = from_f32<WT>(s);
  }
}

// ------------------------------------------------------------------- hosts

// Threads that a row of n elements takes, backward.
int row_threads(int64_t n) {
  for (int tpr : {8, 32, 64, 128, 256, 512, 1024})
    if (n <= static_cast<int64_t>(tpr) * EPT) return tpr;
  return 0;  // longer
}

int element_bytes(int dtype) { return dtype == H3B_F32 ? 4 : 2; }

// CTAs of a backward pass, each of which leaves a partial row.
int64_t bwd_ctas(int64_t m, int64_t n) {
  const int tpr = row_threads(n);
  if (tpr == 0) {
    const int64_t most = 64;
    return m < most ? m : most;
  }
  const int64_t groups = bwd_threads(tpr) / tpr;
  const int64_t ctas = static_cast<int64_t>(h3b::num_sms()) * bwd_ctas_per_sm(tpr);
  const int64_t need = (m + groups - 1) / groups;
  return need < ctas ? need : ctas;
}

template <class T, class WT, int VEC>
int run_fwd(const FwdArgs& a, cudaStream_t st) {
#define H3B_LN_FWD(TPR, HELD)                                                                             \
  if (a.n <= static_cast<int64_t>(TPR) * HELD) {                                                          \
    constexpr int64_t groups = block_threads(TPR) / TPR;                                                  \
    const unsigned blocks = static_cast<unsigned>((a.m + groups - 1) / groups);                           \
    ln_fwd_kernel<T, WT, VEC, TPR, HELD><<<blocks, block_threads(TPR), 0, st>>>(a);                         \
    return h3b::launch_status();                                                                          \
  }
  H3B_LN_FWD(8, 32)
  if constexpr (VEC == 1) {
    H3B_LN_FWD(32, 32)
    H3B_LN_FWD(64, 32)
    H3B_LN_FWD(128, 32)
  } else {
    // Weights in fp32 are twice the bytes of a 16-bit row, and L1 would bind:
    // as many warps as hold four rows (two longer ones) in 64 registers of
    // each thread.  16384 x 4096 bf16 takes 48.7 us, with a warp a row 57.4;
    // 131072 x 512 47, 62; 8192 x 8192 54, a CTA a row 60; fp32 within 2 us of
    // those.  Few rows would be a little quicker with more threads; a row's
    // result does not depend on how many others there are.
#define H3B_LN_FWD_ROWS(WARPS, R, PACKS)                                                                                    \
  if (a.n <= 32 * WARPS * PACKS * VEC) {                                                                                   \
    ln_fwd_rows_kernel<T, WT, VEC, WARPS, R, PACKS><<<static_cast<unsigned>((a.m + R - 1) / R), 32 * WARPS, 0, st>>>(a);    \
    return h3b::launch_status();                                                                                           \
  }
    H3B_LN_FWD_ROWS(1, 4, 2)
    H3B_LN_FWD_ROWS(1, 4, 3)
    H3B_LN_FWD_ROWS(1, 4, 4)
    H3B_LN_FWD_ROWS(2, 4, 3)
    H3B_LN_FWD_ROWS(2, 4, 4)
    H3B_LN_FWD_ROWS(4, 4, 3)
    H3B_LN_FWD_ROWS(4, 4, 4)
    H3B_LN_FWD_ROWS(4, 2, 5)
    H3B_LN_FWD_ROWS(4, 2, 6)
    H3B_LN_FWD_ROWS(4, 2, 8)
    H3B_LN_FWD_ROWS(8, 2, 6)
#undef H3B_LN_FWD_ROWS
  }
  if constexpr (VEC < 8) H3B_LN_FWD(256, 32)
  H3B_LN_FWD(512, 32)
  H3B_LN_FWD(1024, 32)
#undef H3B_LN_FWD
  ln_fwd_long_kernel<T, WT><<<static_cast<unsigned>(a.m), 1024, 0, st>>>(a);
  return h3b::launch_status();
}

template <class T, class WT, int VEC>
int run_bwd(const BwdArgs& a, cudaStream_t st) {
  const int tpr = row_threads(a.n);
  const unsigned ctas = static_cast<unsigned>(bwd_ctas(a.m, a.n));
#define H3B_LN_BWD(TPR)                                                                                             \
  case TPR: {                                                                                                       \
    constexpr int threads = bwd_threads(TPR), joined = threads > TPR ? threads * EPT * 8 : 0;                       \
    constexpr int ring = bwd_ring(sizeof(T), VEC, TPR) ? RING * 2 * threads * EPT * static_cast<int>(sizeof(T)) : 0; \
    constexpr int most = ring > joined ? ring : joined;                                                             \
    static_assert(bwd_ctas_per_sm(TPR) * (most + 3 * 1024) <= 227 * 1024, "shared memory of the CTAs of an SM");    \
    if constexpr (most > 40 * 1024) {                                                                               \
      static h3b::OncePerDevice once;                                                                               \
      const int rc = h3b::prepare(once, ln_bwd_kernel<T, WT, VEC, TPR>, most);                                      \
      if (rc != H3B_OK) return rc;                                                                                  \
    }                                                                                                               \
    const int used = ring > 0 ? static_cast<int>(RING * 2 * (threads / TPR) * a.n * sizeof(T)) : 0;                 \
    ln_bwd_kernel<T, WT, VEC, TPR><<<ctas, threads, used > joined ? used : joined, st>>>(a);                        \
    break;                                                                                                          \
  }
  switch (tpr) {
    H3B_LN_BWD(8)
    H3B_LN_BWD(32)
    H3B_LN_BWD(64)
    H3B_LN_BWD(128)
    H3B_LN_BWD(256)
    H3B_LN_BWD(512)
    H3B_LN_BWD(1024)
    default:
      ln_bwd_long_kernel<T, WT><<<static_cast<unsigned>(a.m), 1024, 0, st>>>(a);
      if (a.sums) {
        const dim3 grid(static_cast<unsigned>((a.n + 255) / 256), ctas);
        ln_bwd_long_sums_kernel<T><<<grid, 256, 0, st>>>(a);
      }
  }
#undef H3B_LN_BWD
  if (a.sums) {
    const dim3 grid(static_cast<unsigned>((a.n + 31) / 32), a.dw != nullptr && a.db != nullptr ? 2 : 1);
    // (set up while the kernel before it ends, and waiting for it)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(1024);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, ln_bwd_join_kernel<WT>, static_cast<const float*>(a.partial), static_cast<int>(ctas), a.n,
                           static_cast<WT*>(a.dw), static_cast<WT*>(a.db)) != cudaSuccess)
      return H3B_ERR_LAUNCH;
  }
  return h3b::launch_status();
}

// F(T, WT, VEC) for the types, with 16-byte words where `wide`.
#define H3B_LN_TYPES(F, ...)                                                                            \
  do {                                                                                                  \
    if (dtype == H3B_F32) return wide ? F<float, float, 4>(__VA_ARGS__) : F<float, float, 1>(__VA_ARGS__); \
    if (dtype == H3B_BF16 && wdtype == H3B_F32)                                                         \
      return wide ? F<__nv_bfloat16, float, 8>(__VA_ARGS__) : F<__nv_bfloat16, float, 1>(__VA_ARGS__);  \
    if (dtype == H3B_BF16)                                                                              \
      return wide ? F<__nv_bfloat16, __nv_bfloat16, 8>(__VA_ARGS__)                                     \
                  : F<__nv_bfloat16, __nv_bfloat16, 1>(__VA_ARGS__);                                    \
    if (wdtype == H3B_F32) return wide ? F<__half, float, 8>(__VA_ARGS__) : F<__half, float, 1>(__VA_ARGS__); \
    return wide ? F<__half, __half, 8>(__VA_ARGS__) : F<__half, __half, 1>(__VA_ARGS__);                \
  } while (0)

int check(int dtype, int wdtype, int64_t m, int64_t n) {
  if (dtype != H3B_BF16 && dtype != H3B_F16 && dtype != H3B_F32) return H3B_ERR_DTYPE;
  if (wdtype != dtype && wdtype != H3B_F32) return H3B_ERR_DTYPE;
  if (m < 0 || m > 0x7FFFFFFF || n < 1 || n > (1ll << 30)) return H3B_ERR_SHAPE;
  return H3B_OK;
}

}  // namespace

extern "C" int h3b_layer_norm_fwd(const h3b_layer_norm_args* p, h3b_stream_t stream) {
  if (p == nullptr) return H3B_ERR_ARG;
  const int dtype = p->dtype, wdtype = p->wdtype;
  const int64_t m = p->m, n = p->n;
  const int rc = check(dtype, wdtype, m, n);
  if (rc != H3B_OK) return rc;
  if (m == 0) return H3B_OK;
  if (p->x == nullptr || p->y == nullptr || (p->mean == nullptr) != (p->rstd == nullptr) || !(p->eps >= 0.0))
    return H3B_ERR_ARG;
  const FwdArgs a{p->x, p->w, p->b, p->y, p->mean, p->rstd, m, n, p->ldx, p->ldy, static_cast<float>(p->eps)};
  const int64_t vec = 16 / element_bytes(dtype);
  const bool wide = n % vec == 0 && (m == 1 || (a.ldx % vec == 0 && a.ldy % vec == 0)) && h3b::aligned16(a.x) &&
                    h3b::aligned16(a.y) && h3b::aligned16(a.w) && h3b::aligned16(a.b);
  const auto st = reinterpret_cast<cudaStream_t>(stream);
  H3B_LN_TYPES(run_fwd, a, st);
}

extern "C" int h3b_layer_norm_bwd_workspace(int64_t m, int64_t n, int64_t* bytes) {
  if (bytes == nullptr) return H3B_ERR_ARG;
  if (m < 0 || m > 0x7FFFFFFF || n < 1 || n > (1ll << 30)) return H3B_ERR_SHAPE;
  *bytes = bwd_ctas(m, n) * 2 * n * static_cast<int64_t>(sizeof(float));
  return H3B_OK;
}

extern "C" int h3b_layer_norm_bwd(const h3b_layer_norm_bwd_args* p, h3b_stream_t stream) {
  if (p == nullptr) return H3B_ERR_ARG;
  const int dtype = p->dtype, wdtype = p->wdtype;
  const int64_t m = p->m, n = p->n;
  const int rc = check(dtype, wdtype, m, n);
  if (rc != H3B_OK) return rc;
  if (m == 0) return H3B_OK;
  if (p->dy == nullptr || p->x == nullptr || p->mean == nullptr || p->rstd == nullptr || p->dx == nullptr)
    return H3B_ERR_ARG;
  const bool sums = p->dw != nullptr || p->db != nullptr;
  if (sums && (p->workspace == nullptr || p->workspace_bytes < bwd_ctas(m, n) * 2 * n * static_cast<int64_t>(sizeof(float))))
    return H3B_ERR_ARG;
  if (sums && !h3b::aligned16(p->workspace)) return H3B_ERR_ALIGN;
  const BwdArgs a{p->dy,   p->x, p->w,    p->mean, p->rstd, p->dx,        p->dw, p->db, static_cast<float*>(p->workspace),
                  m,       n,    p->lddy, p->ldx,  p->lddx, sums ? 1 : 0};
  const int64_t vec = 16 / element_bytes(dtype);
  const bool wide = n % vec == 0 && (m == 1 || (a.ldx % vec == 0 && a.lddy % vec == 0 && a.lddx % vec == 0)) &&
                    h3b::aligned16(a.x) && h3b::aligned16(a.dy) && h3b::aligned16(a.dx) && h3b::aligned16(a.w);
  const auto st = reinterpret_cast<cudaStream_t>(stream);
  H3B_LN_TYPES(run_bwd, a, st);
}
