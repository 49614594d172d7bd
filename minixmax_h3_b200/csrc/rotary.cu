// Rotary positions of q [B, S, H, D] and k [B, S, Hkv, D] in one launch.
//
//   (x1, x2) -> f (x1 cos a - x2 sin a, x2 cos a + x1 sin a),   a = position * w[pair],
//
// over the first `rot` channels of a head, as pairs (i, i + rot/2) or
// (2i, 2i + 1); the other channels are copied.  `inverse` turns by -a, which
// is also the transpose of the map: the gradients' pass.
//
// The angle is kept in turns, as a 64-bit binary fraction: w[pair] / 2 pi
// arrives as a multiple of 2^-64 and the product with the integer position
// wraps exactly, so a position of 2^31 loses 2^-33 turns and no whole turns
// have to be removed from a float (a 32-bit float's angle at position 10^6
// is off by 0.06 rad).  The fraction's nearest quarter turn is taken off as
// an integer; sincospif sees at most an eighth of a turn to either side.
//
// Bound by HBM: every channel is read and written once.  A thread owns VEC
// pairs of one token (two vectors of VEC elements, 16 bytes where the
// alignment allows) and walks a range of heads with their sines and cosines
// in registers, four heads' loads in flight; a few tokens are spread over
// the heads too.
#include "h3b_common.cuh"
#include "h3b_host.hpp"

namespace {

constexpr int THREADS = 256;

struct Operand {
  const void* in;
  void* out;
  int64_t in_b, in_s, in_h;     // strides in elements
  int64_t out_b, out_s, out_h;
};

struct RotaryArgs {
  Operand q, k;
  const void* pos;
  int64_t pos_b, pos_s, pos_a;
  const uint64_t* turns;  // [rot / 2]
  int64_t tokens;         // b * s
  int s, heads, all_heads;  // all_heads = heads + kv_heads
  int heads_per_group;
  int units, rot_units;   // units of 2 * VEC channels: all of a head (or the turned ones, in place), the turned ones
  int half;               // rot / 2
  int end0, end1;         // pairs of axis 0, of axes 0 and 1
  int pos64;
  float factor, sign;
};

template <int BYTES>
struct Word;
template <>
struct Word<2> { using T = uint16_t; };
template <>
struct Word<4> { using T = uint32_t; };
template <>
struct Word<8> { using T = uint2; };
template <>
struct Word<16> { using T = uint4; };

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

template <class T, int VEC>
union Pack {
  typename Word<VEC * sizeof(T)>::T w;
  T e[VEC];
  H3B_DEV Pack() {}
};

// sin and cos of `turn` / 2^64 turns.
H3B_DEV void sincos_turns(uint64_t turn, float* s, float* c) {
  const uint32_t quarter = static_cast<uint32_t>((turn + (1ull << 61)) >> 62);
  const uint64_t rest = turn - (static_cast<uint64_t>(quarter) << 62);  // as int64: [-2^61, 2^61)
  // 2^-63: half turns.  A small high word converts exactly, so the low word still counts.
  const float x = fmaf(__uint2float_rn(static_cast<uint32_t>(rest)), 0x1p-63f,
                       __int2float_rn(static_cast<int32_t>(rest >> 32)) * 0x1p-31f);
  float sn, cs;
  sincospif(x, &sn, &cs);
  const bool swap = quarter & 1;
  const float a = swap ? cs : sn, b = swap ? sn : cs;
  *s = (quarter & 2) ? -a : a;
  *c = ((quarter + 1) & 2) ? -b : b;
}

template <class T, int VEC, bool NEIGHBOURS>
__global__ void __launch_bounds__(THREADS) rotary_kernel(const RotaryArgs a) {
  const int64_t item = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x;
  const int64_t token = item / a.units;
  if (token >= a.tokens) return;
  const int unit = static_cast<int>(item - token * a.units);
  const int64_t b = token / a.s, s = token - b * a.s;
  const int h0 = static_cast<int>(blockIdx.y) * a.heads_per_group;
  const int h1 = min(h0 + a.heads_per_group, a.all_heads);
  const bool turned = unit < a.rot_units;

  // first channels of the unit's two vectors
  const int c0 = NEIGHBOURS || !turned ? unit * 2 * VEC : unit * VEC;
  const int c1 = NEIGHBOURS || !turned ? c0 + VEC : c0 + a.half;

  float sn[VEC], cs[VEC];
  if (turned) {
    int64_t p[3];
    const int64_t at = b * a.pos_b + s * a.pos_s;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const bool used = i == 0 || (i == 1 ? a.end0 < a.half : a.end1 < a.half);
      p[i] = !used ? 0
                   : a.pos64 ? static_cast<const int64_t*>(a.pos)[at + i * a.pos_a]
                             : static_cast<const int32_t*>(a.pos)[at + i * a.pos_a];
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int pair = unit * VEC + i;
      const int64_t pp = pair < a.end0 ? p[0] : (pair < a.end1 ? p[1] : p[2]);
      sincos_turns(static_cast<uint64_t>(pp) * a.turns[pair], &sn[i], &cs[i]);
      sn[i] *= a.sign * a.factor;
      cs[i] *= a.factor;
    }
  }

  using P = Pack<T, VEC>;
  auto in_of = [&](int h) {
    return h < a.heads ? static_cast<const T*>(a.q.in) + b * a.q.in_b + s * a.q.in_s + h * a.q.in_h
                       : static_cast<const T*>(a.k.in) + b * a.k.in_b + s * a.k.in_s + (h - a.heads) * a.k.in_h;
  };
  auto out_of = [&](int h) {
    return h < a.heads ? static_cast<T*>(a.q.out) + b * a.q.out_b + s * a.q.out_s + h * a.q.out_h
                       : static_cast<T*>(a.k.out) + b * a.k.out_b + s * a.k.out_s + (h - a.heads) * a.k.out_h;
  };
  auto load = [&](int h, P& x, P& y) {
    const T* in = in_of(h);
    x.w = *reinterpret_cast<const decltype(x.w)*>(in + c0);
    y.w = *reinterpret_cast<const decltype(y.w)*>(in + c1);
  };
  auto finish = [&](int h, P& x, P& y) {
    if (turned) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        T* e1 = NEIGHBOURS ? (2 * i < VEC ? &x.e[2 * i] : &y.e[2 * i - VEC]) : &x.e[i];
        T* e2 = NEIGHBOURS ? (2 * i + 1 < VEC ? &x.e[2 * i + 1] : &y.e[2 * i + 1 - VEC]) : &y.e[i];
        const float v1 = to_f32(*e1), v2 = to_f32(*e2);
        *e1 = from_f32<T>(fmaf(v1, cs[i], -v2 * sn[i]));
        *e2 = from_f32<T>(fmaf(v2, cs[i], v1 * sn[i]));
      }
    }
    T* out = out_of(h);
    *reinterpret_cast<decltype(x.w)*>(out + c0) = x.w;
    *reinterpret_cast<decltype(y.w)*>(out + c1) = y.w;
  };
  int h = h0;
  for (; h + 4 <= h1; h += 4) {
    P x[4], y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) load(h + j, x[j], y[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) finish(h + j, x[j], y[j]);
  }
  for (; h < h1; ++h) {
    P x, y;
    load(h, x, y);
    finish(h, x, y);
  }
}

template <class T, int VEC>
int launch(RotaryArgs& a, int64_t d, int64_t rot, int neighbours, cudaStream_t stream) {
  // in place, the channels behind the turned ones are there already
  const auto same = [](const Operand& o) {
    return o.in == o.out && o.in_b == o.out_b && o.in_s == o.out_s && o.in_h == o.out_h;
  };
  const bool in_place = same(a.q) && (a.k.in == nullptr || same(a.k));
  a.rot_units = static_cast<int>(rot / (2 * VEC));
  a.units = in_place ? a.rot_units : static_cast<int>(d / (2 * VEC));
  if (a.units == 0) return H3B_OK;
  const int64_t items = a.tokens * a.units;
  // Heads are split into groups until there are threads for two waves of
  // half-full SMs; a group recomputes its pairs' sines (about three heads'
  // work for eight pairs).
  const int64_t want = static_cast<int64_t>(h3b::num_sms()) * 2048;
  int64_t groups = (want + items - 1) / items;
  if (groups > a.all_heads) groups = a.all_heads;
  a.heads_per_group = static_cast<int>((a.all_heads + groups - 1) / groups);
  groups = (a.all_heads + a.heads_per_group - 1) / a.heads_per_group;
  const int64_t blocks = (items + THREADS - 1) / THREADS;
  if (blocks > 0x7FFFFFFF || groups > 65535) return H3B_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(groups));
  if (neighbours)
    rotary_kernel<T, VEC, true><<<grid, THREADS, 0, stream>>>(a);
  else
    rotary_kernel<T, VEC, false><<<grid, THREADS, 0, stream>>>(a);
  return h3b::launch_status();
}

// Whether every vector of `vec` elements of `bytes` each is aligned.
bool fits(const Operand& o, int64_t b, int64_t s, int64_t h, int64_t vec, int64_t bytes) {
  const auto ok = [&](const void* p, int64_t sb, int64_t ss, int64_t sh) {
    return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(vec * bytes) == 0 && (b == 1 || sb % vec == 0) &&
           (s == 1 || ss % vec == 0) && (h == 1 || sh % vec == 0);
  };
  return ok(o.in, o.in_b, o.in_s, o.in_h) && ok(o.out, o.out_b, o.out_s, o.out_h);
}

}  // namespace

extern "C" int h3b_rotary(const h3b_rotary_args* r, h3b_stream_t stream) {
  if (r == nullptr) return H3B_ERR_ARG;
  const int dtype = r->dtype;
  const int64_t b = r->b, s = r->s, heads = r->heads, kv_heads = r->kv_heads, d = r->d, rot = r->rot;
  if (dtype != H3B_BF16 && dtype != H3B_F16 && dtype != H3B_F32) return H3B_ERR_DTYPE;
  if (b < 0 || s < 0 || heads < 0 || kv_heads < 0 || heads + kv_heads > 65535) return H3B_ERR_SHAPE;
  if (d < 1 || d > 65536 || rot < 0 || rot > d || (rot & 1)) return H3B_ERR_SHAPE;
  if (r->axis0_pairs < 0 || r->axis1_pairs < 0 || r->axis0_pairs + r->axis1_pairs > rot / 2) return H3B_ERR_SHAPE;
  if (b == 0 || s == 0 || heads + kv_heads == 0) return H3B_OK;
  if ((heads > 0 && (r->q == nullptr || r->q_out == nullptr)) || (kv_heads > 0 && (r->k == nullptr || r->k_out == nullptr)))
    return H3B_ERR_ARG;
  if (rot > 0 && (r->positions == nullptr || r->turns == nullptr)) return H3B_ERR_ARG;
  if (s > 0x7FFFFFFF || b > 0x7FFFFFFF || b * s > (1ll << 40)) return H3B_ERR_SHAPE;
  const auto operand = [](const void* in, void* out, const int64_t (&i)[3], const int64_t (&o)[3]) {
    return Operand{in, out, i[0], i[1], i[2], o[0], o[1], o[2]};
  };
  RotaryArgs a{};
  a.q = operand(r->q, r->q_out, r->q_stride, r->q_out_stride);
  a.k = operand(r->k, r->k_out, r->k_stride, r->k_out_stride);
  if (heads == 0) a.q = a.k;
  if (kv_heads == 0) a.k = a.q;
  a.pos = r->positions;
  a.pos_b = r->pos_stride[0];
  a.pos_s = r->pos_stride[1];
  a.pos_a = r->pos_stride[2];
  a.turns = r->turns;
  a.tokens = b * s;
  a.s = static_cast<int>(s);
  a.heads = static_cast<int>(heads);
  a.all_heads = static_cast<int>(heads + kv_heads);
  a.half = static_cast<int>(rot / 2);
  a.end0 = static_cast<int>(r->axis0_pairs);
  a.end1 = static_cast<int>(r->axis0_pairs + r->axis1_pairs);
  a.pos64 = r->positions64;
  a.factor = static_cast<float>(r->factor);
  a.sign = r->inverse ? -1.0f : 1.0f;
  const int64_t bytes = dtype == H3B_F32 ? 4 : 2;
  int64_t vec = 16 / bytes;
  while (vec > 1 && (rot % (2 * vec) != 0 || d % (2 * vec) != 0 ||
                     (heads > 0 && !fits(a.q, b, s, heads, vec, bytes)) ||
                     (kv_heads > 0 && !fits(a.k, b, s, kv_heads, vec, bytes))))
    vec /= 2;
  if (vec == 1 && (d & 1)) return H3B_ERR_SHAPE;
  const auto st = reinterpret_cast<cudaStream_t>(stream);
#define H3B_ROTARY(T, V) return launch<T, V>(a, d, rot, r->interleaved, st)
#define H3B_ROTARY16(T)      \
  if (vec == 8) H3B_ROTARY(T, 8); \
  if (vec == 4) H3B_ROTARY(T, 4); \
  if (vec == 2) H3B_ROTARY(T, 2); \
  H3B_ROTARY(T, 1)
  if (dtype == H3B_BF16) {
    H3B_ROTARY16(__nv_bfloat16);
  }
  if (dtype == H3B_F16) {
    H3B_ROTARY16(__half);
  }
  if (vec == 4) H3B_ROTARY(float, 4);
  if (vec == 2) H3B_ROTARY(float, 2);
  H3B_ROTARY(float, 1);
#undef H3B_ROTARY16
#undef H3B_ROTARY
}
