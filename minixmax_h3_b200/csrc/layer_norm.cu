// Layer norm over the last axis of x [m, n], forward and backward.
//
//   y = xhat w + b,   xhat = (x - mean) rstd,   rstd = 1 / sqrt(var + eps)
//   g = dy w,   dx = rstd (g - mean(g) - xhat mean(g xhat))
//   dw = sum_rows dy xhat,   db = sum_rows dy
//
// Both directions are bound by HBM: x is read and y written once; backward, x
// and dy are read and dx written once.  A group of threads holds a row in
// registers (forward 32 elements a thread at most, backward 16), so the
// variance is taken about the mean in a second pass over registers, and what
// rounding the mean left over is taken off with it: var = mean(d^2) -
// mean(d)^2, d = x - mean, with mean(d) of the size of a rounding.
//
// The weights' gradients are sums over all rows.  Each CTA walks rows with a
// stride and keeps its threads' columns of both sums in registers (32-bit),
// adds its groups' sums in order through shared memory and writes one partial
// row; a second launch adds the partial rows of a column in order.  No
// atomics: results do not depend on scheduling.
#include "h3b_common.cuh"
#include "h3b_host.hpp"

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
// VEC values of the weight's type WT (float beside a 16-bit T takes two words).
template <class WT, int VEC>
H3B_DEV void load_weights(const WT* p, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = to_f32(*p);
  } else {
    constexpr int N = 16 / sizeof(WT);
#pragma unroll
    for (int i = 0; i < VEC; i += N) {
      const Pack<WT, N> r = load_pack<WT, N>(p + i);
#pragma unroll
      for (int j = 0; j < N; ++j) v[i + j] = to_f32(r.e[j]);
    }
  }
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

// Rows of a warp or less share a CTA; larger groups are a CTA (RowSum).
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

template <class T, class WT, int VEC, int TPR>
__global__ void __launch_bounds__(block_threads(TPR)) ln_fwd_kernel(const FwdArgs a) {
  constexpr int MAXV = 32 / VEC;
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
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int c = t + i * TPR;
    if (c < nv) v[i] = load_pack<T, VEC>(x + static_cast<int64_t>(c) * VEC);
  }
#pragma unroll
  for (int i = 0; i < MAXV; ++i)
    if (t + i * TPR < nv)
#pragma unroll
      for (int j = 0; j < VEC; ++j) s += to_f32(v[i].e[j]);
  const float m0 = sum(s, 0.0f).x * inv_n;
  float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
  for (int i = 0; i < MAXV; ++i)
    if (t + i * TPR < nv)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = to_f32(v[i].e[j]) - m0;
        s1 += d;
        s2 = fmaf(d, d, s2);
      }
  const float2 r = sum(s1, s2);
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
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int c = t + i * TPR;
    if (c < nv) {
      float wv[VEC], bv[VEC];
      if (w != nullptr) load_weights<WT, VEC>(w + c * VEC, wv);
      if (b != nullptr) load_weights<WT, VEC>(b + c * VEC, bv);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float h = ((to_f32(v[i].e[j]) - m0) - dm) * rstd;
        if (w != nullptr) h *= wv[j];
        if (b != nullptr) h += bv[j];
        v[i].e[j] = from_f32<T>(h);
      }
      store_pack<T, VEC>(y + static_cast<int64_t>(c) * VEC, v[i]);
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

template <class T, class WT, int VEC, int TPR>
__global__ void __launch_bounds__(block_threads(TPR)) ln_bwd_kernel(const BwdArgs a) {
  constexpr int MAXV = 16 / VEC;
  constexpr int THREADS = block_threads(TPR);
  constexpr int GROUPS = THREADS / TPR;
  __shared__ float2 slots[2][32];
  // groups' sums meet here (only groups of less than a CTA)
  __shared__ float2 joined[GROUPS > 1 ? TPR * 16 : 1];
  RowSum<TPR> sum{slots};
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const int n = static_cast<int>(a.n);
  const int nv = (n + VEC - 1) / VEC;
  const float inv_n = 1.0f / static_cast<float>(n);
  const WT* w = static_cast<const WT*>(a.w);

  float wv[MAXV][VEC];
  float sw[MAXV][VEC], sb[MAXV][VEC];
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) wv[i][j] = 1.0f, sw[i][j] = sb[i][j] = 0.0f;
    const int c = t + i * TPR;
    if (w != nullptr && c < nv) load_weights<WT, VEC>(w + c * VEC, wv[i]);
  }
  // Every group of the CTA makes the same number of rounds (the row sums need
  // whole warps); one without a row adds zeros and writes nothing.
  const int64_t step = static_cast<int64_t>(gridDim.x) * GROUPS;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * GROUPS; base < a.m; base += step) {
    const int64_t row = base + group;
    const bool live = row < a.m;
    Pack<T, VEC> vx[MAXV], vg[MAXV];
    float mean = 0.0f, rstd = 0.0f;
    if (live) {
      const T* x = static_cast<const T*>(a.x) + row * a.ldx;
      const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
#pragma unroll
      for (int i = 0; i < MAXV; ++i) {
        const int c = t + i * TPR;
        if (c < nv) {
          vx[i] = load_pack<T, VEC>(x + static_cast<int64_t>(c) * VEC);
          vg[i] = load_pack<T, VEC>(dy + static_cast<int64_t>(c) * VEC);
        }
      }
      mean = a.mean[row];
      rstd = a.rstd[row];
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < MAXV; ++i)
      if (live && t + i * TPR < nv)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float xhat = (to_f32(vx[i].e[j]) - mean) * rstd;
          const float d = to_f32(vg[i].e[j]);
          const float g = d * wv[i][j];
          s1 += g;
          s2 = fmaf(g, xhat, s2);
          sw[i][j] = fmaf(d, xhat, sw[i][j]);
          sb[i][j] += d;
        }
    const float2 r = sum(s1, s2);
    if (live) {
      const float c1 = r.x * inv_n, c2 = r.y * inv_n;
      T* dx = static_cast<T*>(a.dx) + row * a.lddx;
#pragma unroll
      for (int i = 0; i < MAXV; ++i) {
        const int c = t + i * TPR;
        if (c < nv) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float xhat = (to_f32(vx[i].e[j]) - mean) * rstd;
            const float g = to_f32(vg[i].e[j]) * wv[i][j];
            vx[i].e[j] = from_f32<T>(rstd * (fmaf(-xhat, c2, g) - c1));
          }
          store_pack<T, VEC>(dx + static_cast<int64_t>(c) * VEC, vx[i]);
        }
      }
    }
  }
  if (!a.sums) return;
  float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.n;
  if constexpr (GROUPS > 1) {
    for (int g = 0; g < GROUPS; ++g) {
      if (group == g) {
#pragma unroll
        for (int i = 0; i < MAXV; ++i) {
          const int c = t + i * TPR;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int at = c * VEC + j;
            const float2 before = g == 0 ? make_float2(0.0f, 0.0f) : joined[at];
            joined[at] = make_float2(before.x + sw[i][j], before.y + sb[i][j]);
          }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < n; c += THREADS) {
      out[c] = joined[c].x;
      out[n + c] = joined[c].y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < MAXV; ++i) {
      const int c = t + i * TPR;
      if (c < nv)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          out[c * VEC + j] = sw[i][j];
          out[n + c * VEC + j] = sb[i][j];
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

// dw and db from the partial rows, in order: a warp reads 32 columns of every
// eighth partial row, the CTA's eight warps' sums are added in order.
template <class WT>
__global__ void __launch_bounds__(256) ln_bwd_join_kernel(const float* partial, int ctas, int64_t n, WT* dw, WT* db) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  const int64_t which = blockIdx.y;
  float s = 0.0f;
  if (c < n)
#pragma unroll 4
    for (int p = warp; p < ctas; p += 8) s += partial[(static_cast<int64_t>(p) * 2 + which) * n + c];
  part[warp][lane] = s;
  __syncthreads();
  WT* out = which == 0 ? dw : db;
  if (warp == 0 && c < n && out != nullptr) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += part[i][lane];
    out[c] = from_f32<WT>(s);
  }
}

// ------------------------------------------------------------------- hosts

// Threads a row of n elements takes at `ept` elements a thread.
int row_threads(int64_t n, int ept) {
  for (int tpr : {8, 32, 64, 128, 256, 512, 1024})
    if (n <= static_cast<int64_t>(tpr) * ept) return tpr;
  return 0;  // longer
}

int element_bytes(int dtype) { return dtype == H3B_F32 ? 4 : 2; }

// CTAs of a backward pass: two waves of 1024 threads an SM at most, so that a
// CTA's partial row stands for many rows.
int64_t bwd_ctas(int64_t m, int64_t n) {
  const int tpr = row_threads(n, 16);
  if (tpr == 0) {
    const int64_t most = 64;
    return m < most ? m : most;
  }
  const int threads = block_threads(tpr);
  const int64_t groups = threads / tpr;
  const int64_t ctas = static_cast<int64_t>(h3b::num_sms()) * (threads >= 512 ? 1 : 512 / threads);
  const int64_t need = (m + groups - 1) / groups;
  return need < ctas ? need : ctas;
}

template <class T, class WT, int VEC>
int run_fwd(const FwdArgs& a, cudaStream_t st) {
  const int tpr = row_threads(a.n, 32);
#define H3B_LN_FWD(TPR)                                                                              \
  case TPR: {                                                                                        \
    const int64_t groups = block_threads(TPR) / TPR, blocks = (a.m + groups - 1) / groups;           \
    ln_fwd_kernel<T, WT, VEC, TPR><<<static_cast<unsigned>(blocks), block_threads(TPR), 0, st>>>(a); \
    break;                                                                                           \
  }
  switch (tpr) {
    H3B_LN_FWD(8)
    H3B_LN_FWD(32)
    H3B_LN_FWD(64)
    H3B_LN_FWD(128)
    H3B_LN_FWD(256)
    H3B_LN_FWD(512)
    H3B_LN_FWD(1024)
    default:
      ln_fwd_long_kernel<T, WT><<<static_cast<unsigned>(a.m), 1024, 0, st>>>(a);
  }
#undef H3B_LN_FWD
  return h3b::launch_status();
}

template <class T, class WT, int VEC>
int run_bwd(const BwdArgs& a, cudaStream_t st) {
  const int tpr = row_threads(a.n, 16);
  const unsigned ctas = static_cast<unsigned>(bwd_ctas(a.m, a.n));
#define H3B_LN_BWD(TPR)                                                        \
  case TPR:                                                                    \
    ln_bwd_kernel<T, WT, VEC, TPR><<<ctas, block_threads(TPR), 0, st>>>(a);    \
    break;
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
    const dim3 grid(static_cast<unsigned>((a.n + 31) / 32), a.db != nullptr ? 2 : 1);
    ln_bwd_join_kernel<WT><<<grid, 256, 0, st>>>(a.partial, static_cast<int>(ctas), a.n, static_cast<WT*>(a.dw),
                                                 static_cast<WT*>(a.db));
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

extern "C" int h3b_layer_norm_fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd,
                                  int dtype, int wdtype, int64_t m, int64_t n, int64_t ldx, int64_t ldy, float eps,
                                  h3b_stream_t stream) {
  const int rc = check(dtype, wdtype, m, n);
  if (rc != H3B_OK) return rc;
  if (m == 0) return H3B_OK;
  if (x == nullptr || y == nullptr || (mean == nullptr) != (rstd == nullptr) || !(eps >= 0.0f)) return H3B_ERR_ARG;
  const FwdArgs a{x, w, b, y, mean, rstd, m, n, ldx, ldy, eps};
  const int64_t vec = 16 / element_bytes(dtype);
  const bool wide = n % vec == 0 && (m == 1 || (ldx % vec == 0 && ldy % vec == 0)) && h3b::aligned16(x) &&
                    h3b::aligned16(y) && h3b::aligned16(w) && h3b::aligned16(b);
  const auto st = reinterpret_cast<cudaStream_t>(stream);
  H3B_LN_TYPES(run_fwd, a, st);
}

extern "C" int h3b_layer_norm_bwd_workspace(int64_t m, int64_t n, int64_t* bytes) {
  if (bytes == nullptr) return H3B_ERR_ARG;
  if (m < 0 || m > 0x7FFFFFFF || n < 1 || n > (1ll << 30)) return H3B_ERR_SHAPE;
  *bytes = bwd_ctas(m, n) * 2 * n * static_cast<int64_t>(sizeof(float));
  return H3B_OK;
}

extern "C" int h3b_layer_norm_bwd(const void* dy, const void* x, const void* w, const float* mean, const float* rstd,
                                  void* dx, void* dw, void* db, int dtype, int wdtype, int64_t m, int64_t n,
                                  int64_t lddy, int64_t ldx, int64_t lddx, void* workspace, int64_t workspace_bytes,
                                  h3b_stream_t stream) {
  const int rc = check(dtype, wdtype, m, n);
  if (rc != H3B_OK) return rc;
  if (m == 0) return H3B_OK;
  if (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr || dx == nullptr) return H3B_ERR_ARG;
  const bool sums = dw != nullptr || db != nullptr;
  if (sums && (workspace == nullptr || workspace_bytes < bwd_ctas(m, n) * 2 * n * static_cast<int64_t>(sizeof(float))))
    return H3B_ERR_ARG;
  const BwdArgs a{dy, x, w, mean, rstd, dx, dw, db, static_cast<float*>(workspace), m, n, lddy, ldx, lddx, sums ? 1 : 0};
  const int64_t vec = 16 / element_bytes(dtype);
  const bool wide = n % vec == 0 && (m == 1 || (ldx % vec == 0 && lddy % vec == 0 && lddx % vec == 0)) &&
                    h3b::aligned16(x) && h3b::aligned16(dy) && h3b::aligned16(dx) && h3b::aligned16(w);
  const auto st = reinterpret_cast<cudaStream_t>(stream);
  H3B_LN_TYPES(run_bwd, a, st);
}
