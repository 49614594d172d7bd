// Attention of many query rows on tcgen05 (h3b_cross_attention_fwd): 256 query
// rows of one head at a time, in 128-key tiles.
//
//   S = Q K^T;  P = 2^(scale log2e S - M);  O = O 2^(M_old - M) + P V;  o = O / l
//
// An encoder's states are few (77 to some thousand keys), so a call is many
// short pieces of work: 256 rows x 512 keys are 4 tiles and take 10.4 us (24
// heads of 128: 1.9 us a tile, 3 for the border between units); the first unit
// of a launch takes 3 more for barriers, TMEM allocation and the first loads.  So the kernel is persistent: one CTA
// per SM runs through units (sample, head, 256 rows, range of keys) with one
// continuous pipeline of matrix instructions; the next unit's Q and first K
// are loaded, and its first scores computed, while the last one's softmax and
// stores are under way.
//   warps 0-3   softmax of rows 0-127 (thread = row = TMEM lane)
//   warps 4-7   softmax of rows 128-255
//   warp 8      TMA: Q through a ring of 3 tiles, K and V through one of 4
//   warp 9      TMEM allocation and matrix instructions
//   warp 10     what the next round of products consists of, and that its
//               tiles are there; zeroes the left-out rows of V
//   warp 11     idle
//   warps 12-15 stores: O / l of a finished unit, while the softmax warps are
//               at the next one; over a cache whose codes are not written out
//               beforehand they convert the codes too, tile by tile
// TMEM: S0 | S1 | O0 | O1, 128 columns each (O: D).  P goes back to TMEM as
// 16-bit values over the S it came from and is the A operand of P V.  One
// warp issues round after round, across the units' borders too:
//   P V0(t-1)  S0(t)  P V1(t-1)  S1(t)
// so the tensor pipe has one 128-row tile's products while the other's softmax
// runs.  The stream executes in order: S_i(t) cannot overwrite P_i(t-1) before
// P V_i has read it, and the commit behind S_i(t) says that O_i is settled as
// well.
// The running maximum is raised lazily, by steps of more than 2^8, so P <=
// 2^8: exact in fp32 sums.  f16 weights are held times 2^7 (UP), so that they
// fill f16's range up to 2^15 and down to 2^-31 of the largest (a long tail of
// small ones is in l, and has to be in the products).
// Left-out keys: a score column is replaced (-inf) whatever it holds, and the
// row of V is zeroed in shared memory before P V reads it (0 * NaN is NaN).
// What bounds it is the chain softmax -> P V -> S -> softmax of a row tile and
// its hand-offs, of which two are interleaved: 24 heads of 128, bf16, 16384 x
// 4096 673 us (1230 TFLOP/s), 32768 x 512 218 us (950; the border counts for
// a fourth), x 128 102 us (500); of 64, 32768 x 512 185 us.  These are short
// runs: under sustained load, at the power limit, 32768 x 512 of 128 takes 246 us.
#include "h3b_common.cuh"
#include "h3b_host.hpp"
#include "xattn.hpp"

H3B_DECLARE_STATUS();
H3B_REGISTER_STATUS_READER(xattn_tile);

namespace {

using h3b::KV_DENSE;
using h3b::KV_E4M3;
using h3b::KV_INT8;
using h3b::KV8_SCALE_MIN;
using h3b::KvKind;
using h3b::XAttn;

constexpr int BQ = 128, BKV = 128;
constexpr int KVST = 4;  // K/V ring (K_s in slots 0, 2, V_s in 1, 3)
constexpr int THREADS = 512;
constexpr int REGS_LAUNCH = 128;
constexpr int REGS_CONTROL = 64;
constexpr float RESCALE_THRESHOLD = 8.0f;
template <bool F16>
constexpr float UP = F16 ? 7.0f : 0.0f;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.69314718055994531f;

// PRE: a cache whose codes a kernel before this one has written out as 16-bit
// operands (kv8.cu), for calls of many query tiles; else its codes are
// converted here, once a tile and unit.
template <int D, KvKind KIND, bool PRE>
struct Cfg {
  static constexpr bool SCALED = KIND != KV_DENSE;
  static constexpr bool CODES = SCALED && !PRE;  // converted here
  // Registers of the storing and the softmax warps.  (Where no codes are
  // converted the storing warps leave enough that no score is spilled: masked 2
  // x 2049 x 1025, 24 heads of 128 95 -> 89 us, 32768 x 512 of 64 191 -> 186.)
  static constexpr int REGS_STORE = CODES ? 112 : 80;
  static constexpr int REGS_SOFTMAX = CODES ? 168 : 184;
  static_assert(128 * (REGS_CONTROL + REGS_STORE + 2 * REGS_SOFTMAX) <= THREADS * REGS_LAUNCH, "register split exceeds launch");
  // Q ring (128-row tiles).  Over a cache a unit is long, and the codes' own
  // two tiles take the room of the third slot.
  static constexpr int QST = CODES ? 2 : (D == 128 ? 3 : 6);
  static constexpr int RAW_BYTES = CODES ? 128 * D : 0;  // codes of a K or V tile
  static constexpr int HALVES = D / 64;            // 64-column TMA boxes of a tile
  static constexpr int TILE_BYTES = 128 * D * 2;   // Q, K or V
  static constexpr int HALF_BYTES = 128 * 64 * 2;  // 16 KB
};

// What a round of products consists of, written by warp 10 for the issuing warp.
enum : uint32_t {
  R_S0 = 1,        // S_0, S_1 of a tile
  R_S1 = 2,
  R_S_LAST = 4,    // the unit's last: Q is free after it
  R_PV0 = 8,       // P V of the tile before
  R_PV1 = 16,
  R_PV_FIRST = 32, // of its unit: O starts anew
  R_PV_LAST = 64,  // O is complete after it
  R_END = 128,     // the last round
  R_S_FIRST = 256, // of its unit: Q_1 has to be waited for, at
  R_Q1_PHASE = 512,  // this parity
  R_Q0_SHIFT = 10, // Q slots of S_0, S_1
  R_Q1_SHIFT = 13
};

// What the softmax warps of a row tile have to know of a tile, by warp 10.
struct __align__(16) TileInfo {
  uint32_t keep[4];  // kept columns
  uint32_t flags;    // T_*
  int causal;        // row 0 of the 128 sees columns < causal (T_CAUSAL)
  uint32_t pad[2];
  // cache, by 32 columns: score factor (log2 domain), log2 and reciprocal of
  // the values' scale
  float k_factor[4], v_log2[4], v_inv[4];
};
enum : uint32_t { T_FIRST = 1, T_LAST = 2, T_WHOLE = 4, T_CAUSAL = 8, T_END = 16 };
constexpr int INFOS = 4;  // ring: entry s + 4 is written after round s + 2, so after P(s + 1)

struct __align__(16) Bars {
  TileInfo info[2][INFOS];
  uint64_t q_full[6];
  uint64_t q_free[6];
  uint64_t raw_full[2];   // codes of K, of V
  uint64_t raw_free[2];   // converted (4 warps)
  uint64_t kv_full[KVST];
  uint64_t kv_free[2];    // by round parity: round t of the products has read V_{t-1} and K_t
  uint64_t s_full[2];
  uint64_t p_half[2][2];  // one arrival per softmax warp
  uint64_t o_full[2];
  uint64_t o_free[2];     // the 4 storing warps have read O_i
  uint64_t ml_full[2];    // the row statistics of O_i: one arrival per softmax warp
  uint64_t ml_free[2];    // read by the 4 storing warps
  uint64_t ready[2];      // by round parity: what round t reads is in shared memory, and todo[] says what to do
  uint64_t drain;
  uint32_t todo[2];       // by round parity: R_* bits and Q slots
  uint32_t tmem_base;
  int abort_flag;
};

template <int D, KvKind KIND, bool PRE>
constexpr size_t smem_bytes() {
  using C = Cfg<D, KIND, PRE>;
  return (C::QST + KVST) * C::TILE_BYTES + 2 * C::RAW_BYTES + 2 * 128 * sizeof(float2) + sizeof(Bars);
}
static_assert(smem_bytes<128, KV_DENSE, false>() <= 232448 && smem_bytes<128, KV_INT8, false>() <= 232448, "shared memory of a CTA");

struct TileArgs {
  XAttn a;
  int q_tiles;  // units of 256 rows per (sample, head)
  int units;
  int group;
  int o_wide;   // 32-byte stores of o allowed
  int step_q, step_split, step_head, step_b;  // gridDim.x units further, digit by digit
  float scale_log2;
};

// The units of one CTA, x = blockIdx.x, + gridDim.x, ...  x counts query tile
// (fastest: units that run together share K and V in L2), split, head, sample.
// The digits are carried from unit to unit: four divisions cost the issuing
// warp and the softmax warps ~2000 cycles a unit.
struct Unit {
  int x;
  int qt, split, head, b;
  int q0;
  int len;    // the sample's kept prefix
  int j0, n;  // first tile, tiles
  bool two;   // rows 128-255 exist

  // WARP: called by whole warps; a reduction tells the compiler that the
  // length, and with it all control flow, is the same for the warp (uniform
  // registers, no convergence code: the issuing warp's rounds need it).
  template <bool WARP>
  H3B_DEV void settle(const TileArgs& args) {
    const XAttn& a = args.a;
    q0 = qt * 2 * BQ;
    two = q0 + BQ < a.s_q;
    len = a.s_kv;
    if (a.kv_lens != nullptr && x < args.units) {
      len = max(0, min(len, __ldg(a.kv_lens + b)));
      if constexpr (WARP) len = __reduce_max_sync(0xffffffffu, len);
    }
    int end = len;
    if (a.causal) end = max(0, min(end, len - a.s_q + min(q0 + 2 * BQ, a.s_q)));
    const int tiles = (len + BKV - 1) / BKV;
    const int per = a.splits == 1 ? tiles : (tiles + a.splits - 1) / a.splits;
    j0 = split * per;
    n = max(0, min((end + BKV - 1) / BKV, j0 + per) - j0);
  }
  H3B_DEV void first(const TileArgs& args) {
    x = blockIdx.x;
    int u = x;
    qt = u % args.q_tiles;
    u /= args.q_tiles;
    split = u % args.a.splits;
    u /= args.a.splits;
    head = u % args.a.heads;
    b = u / args.a.heads;
    settle<true>(args);
  }
  template <bool WARP = true>
  H3B_DEV void next(const TileArgs& args) {
    x += gridDim.x;
    qt += args.step_q;
    split += args.step_split;
    head += args.step_head;
    b += args.step_b;
    if (qt >= args.q_tiles) qt -= args.q_tiles, ++split;
    if (split >= args.a.splits) split -= args.a.splits, ++head;
    if (head >= args.a.heads) head -= args.a.heads, ++b;
    settle<WARP>(args);
  }
};

// (compact: the roles share instruction caches)
template <bool SPIN>
H3B_DEV bool lane_wait(uint64_t* bar, uint32_t parity, int site, volatile int* abort_flag) {
  return mbar_wait<SPIN, false, true>(bar, parity, &g_status, site, abort_flag);
}
template <bool SPIN = false>
H3B_DEV bool warp_wait(uint64_t* bar, uint32_t parity, int site, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, lane_wait<SPIN>(bar, parity, site, abort_flag));
}

H3B_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Which keys of a tile are kept, one bit each: first the bytes (or 1s), then
// the words, so that a wait can stand between the load and its use.
H3B_DEV uint32_t mask_bytes(const XAttn& a, int b, int key0, int len, int lane) {
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

H3B_DEV void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
H3B_DEV void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

H3B_DEV float4 lds4(const volatile void* p) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(smem_u32(const_cast<const void*>(p))));
  return v;
}
H3B_DEV float2 lds2(const volatile void* p) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(smem_u32(const_cast<const void*>(p))));
  return v;
}

H3B_DEV float row_max32(const uint32_t* r) {
  float mx[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) mx[c] = __uint_as_float(r[c]);
#pragma unroll
  for (int e = 4; e < 28; e += 8)
#pragma unroll
    for (int c = 0; c < 4; ++c) mx[c] = fmax3(mx[c], __uint_as_float(r[e + c]), __uint_as_float(r[e + 4 + c]));
#pragma unroll
  for (int c = 0; c < 4; ++c) mx[c] = fmaxf(mx[c], __uint_as_float(r[28 + c]));
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}
H3B_DEV float row_max64(const uint32_t* r) {
  float mx[8];
#pragma unroll
  for (int c = 0; c < 8; ++c)
    mx[c] = fmax3(__uint_as_float(r[c]), __uint_as_float(r[c + 8]), __uint_as_float(r[c + 16]));
#pragma unroll
  for (int e = 24; e < 56; e += 16)
#pragma unroll
    for (int c = 0; c < 8; ++c) mx[c] = fmax3(mx[c], __uint_as_float(r[e + c]), __uint_as_float(r[e + 8 + c]));
#pragma unroll
  for (int c = 0; c < 8; ++c) mx[c] = fmaxf(mx[c], __uint_as_float(r[56 + c]));
  return fmax3(fmax3(mx[0], mx[1], mx[2]), fmax3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7]));
}

// 64 scores r[0..63] -> weights 2^(s * scale + neg_m), packed into dst[0..31];
// returns their sum and, with MAX, the largest of the 128 scores r[0..127].
template <bool F16, bool MAX>
H3B_DEV float2 exp_pack64(uint32_t* r, uint32_t* dst, float scale_log2, float neg_m) {
  const float2 sc = make_float2(scale_log2, scale_log2);
  const float2 nm = make_float2(neg_m, neg_m);
  float mx[8];
  if constexpr (MAX) {
#pragma unroll
    for (int c = 0; c < 8; ++c) mx[c] = -INFINITY;
  }
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    const float sa = __uint_as_float(r[2 * e]), sb = __uint_as_float(r[2 * e + 1]);
    if constexpr (MAX) {
      mx[e & 7] = fmax3(mx[e & 7], sa, sb);
      mx[e & 7] = fmax3(mx[e & 7], __uint_as_float(r[64 + 2 * e]), __uint_as_float(r[64 + 2 * e + 1]));
    }
    const float2 x = fma2(make_float2(sa, sb), sc, nm);
    r[2 * e] = __float_as_uint(ex2(x.x));
    r[2 * e + 1] = __float_as_uint(ex2(x.y));
  }
  float2 acc[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    const float2 p = make_float2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]));
    acc[e & 3] = add2(acc[e & 3], p);
    dst[e] = pack16x2<F16>(p.x, p.y);
  }
  const float2 t = add2(add2(acc[0], acc[1]), add2(acc[2], acc[3]));
  float m = 0.0f;
  if constexpr (MAX) m = fmax3(fmax3(mx[0], mx[1], mx[2]), fmax3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7]));
  return make_float2(t.x + t.y, m);
}

// The same for a cache's columns, whose factor and exponent offset change
// every 32: sc and nm are those of the two groups of r[0..63], the sum is
// weighted by inv.  With MAX the largest exponent of the 128 scores is found
// (factors fx, offsets ox of the four groups).
template <bool F16, bool MAX>
H3B_DEV float2 exp_codes64(uint32_t* r, uint32_t* dst, float2 sc, float2 nm, float2 inv, const float (&fx)[4],
                           const float (&ox)[4]) {
  float top = -INFINITY;
  if constexpr (MAX) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 32; e += 2)
        mx[(e >> 1) & 3] = fmax3(mx[(e >> 1) & 3], __uint_as_float(r[32 * g + e]), __uint_as_float(r[32 * g + e + 1]));
      top = fmaxf(top, fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fx[g], ox[g]));
    }
  }
  float sum = 0.0f;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const float f = g ? sc.y : sc.x, o = g ? nm.y : nm.x;
    float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int e = 16 * g; e < 16 * g + 16; ++e) {
      const float2 x = fma2(make_float2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), make_float2(f, f),
                            make_float2(o, o));
      const float2 w = make_float2(ex2(x.x), ex2(x.y));
      acc[e & 1] = add2(acc[e & 1], w);
      dst[e] = pack16x2<F16>(w.x, w.y);
    }
    const float2 t = add2(acc[0], acc[1]);
    sum = fmaf(t.x + t.y, g ? inv.y : inv.x, sum);
  }
  return make_float2(sum, top);
}

// Four codes -> two packed pairs of the operands' type, exactly.
template <KvKind KIND, bool F16>
H3B_DEV void codes4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (KIND == KV_INT8) {
    w ^= 0x80808080u;
    if constexpr (F16) {  // 0x6400 | u is 1024 + u in f16
      const uint32_t a = __byte_perm(w, 0x64646464u, 0x5140), b = __byte_perm(w, 0x64646464u, 0x5342);
      const __half2 c = __half2half2(__ushort_as_half(0x6480));  // 1152
      const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), c);
      const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), c);
      lo = *reinterpret_cast<const uint32_t*>(&x);
      hi = *reinterpret_cast<const uint32_t*>(&y);
    } else {  // 0x4B000000 | u is 2^23 + u in fp32
      const float2 c = make_float2(-8388736.0f, -8388736.0f);
      const float2 x = add2(make_float2(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440)),
                                        __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7441))), c);
      const float2 y = add2(make_float2(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7442)),
                                        __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7443))), c);
      lo = pack_bf16x2(x.x, x.y);
      hi = pack_bf16x2(y.x, y.y);
    }
  } else {
    uint32_t a, b;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(a), "=r"(b)
        : "r"(w));
    if constexpr (F16) {
      lo = a;
      hi = b;
    } else {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a));
      const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&b));
      lo = pack_bf16x2(x.x, x.y);
      hi = pack_bf16x2(y.x, y.y);
    }
  }
}

// One row of a tile of codes (128 rows, TMA swizzle) as 16-bit operands in
// the two 64-column halves that the products read (128-byte swizzle), 64
// codes at a time: four loads in flight, then the conversions.
template <int D, KvKind KIND, bool F16>
H3B_DEV void convert_row(uint32_t raw, uint32_t dst, int row) {
#pragma unroll 1
  for (int h = 0; h < D / 64; ++h) {
    uint32_t w[4][4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int x = 4 * h + c;
      const uint32_t at = D == 128 ? row * 128 + ((x ^ (row & 7)) << 4) : row * 64 + ((x ^ ((row >> 1) & 3)) << 4);
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(w[c][0]), "=r"(w[c][1]), "=r"(w[c][2]), "=r"(w[c][3])
                   : "r"(raw + at)
                   : "memory");
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t v[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) codes4<KIND, F16>(w[c][k], v[2 * k], v[2 * k + 1]);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst + h * (128 * 128) + row * 128 +
                                                                   (((2 * c + k) ^ (row & 7)) << 4)),
                     "r"(v[4 * k]), "r"(v[4 * k + 1]), "r"(v[4 * k + 2]), "r"(v[4 * k + 3])
                     : "memory");
    }
  }
}
template <int D>
H3B_DEV void zero_row(uint32_t dst, int row) {
#pragma unroll 1
  for (int c = 0; c < D / 8; ++c)
    asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(dst + (c >> 3) * (128 * 128) + row * 128 + (c & 7) * 16),
                 "r"(0u)
                 : "memory");
}

// The cache's block of a key, -1 if there is none.
H3B_DEV int block_of(const XAttn& a, int b, int key) {
  const int j = key >> (31 - __clz(a.block_tokens));  // (a power of two)
  if (j >= a.max_blocks) return -1;
  const int id = __ldg(a.table + static_cast<int64_t>(b) * a.max_blocks + j);
  return id >= 0 && id < a.num_blocks ? id : -1;
}

template <int D, bool F16, KvKind KIND, bool MASKED, bool PRE>
__global__ void __launch_bounds__(THREADS, 1)
    xattn_tile_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ TileArgs args) {
  using C = Cfg<D, KIND, PRE>;
  constexpr bool CODES = C::CODES, SCALED = C::SCALED;
  constexpr int QST = C::QST;
  constexpr uint32_t IDESC_S = F16 ? idesc_f16_f32(128, BKV, 0, 0) : idesc_bf16_f32(128, BKV, 0, 0);
  constexpr uint32_t IDESC_O = F16 ? idesc_f16_f32(128, D, 0, 1) : idesc_bf16_f32(128, D, 0, 1);
  extern __shared__ __align__(1024) uint8_t smem_tiles[];
  if ((smem_u32(smem_tiles) & 1023u) != 0) {  // the same for the whole CTA; nothing has been started
    if (threadIdx.x == 0 && atomicCAS(&g_status.code, 0, H3B_ERR_DEVICE) == 0) g_status.site = 30;
    return;
  }
  uint8_t* sQ = smem_tiles;
  uint8_t* sKV = sQ + QST * C::TILE_BYTES;
  uint8_t* sRaw = sKV + KVST * C::TILE_BYTES;  // codes of K | V
  float2* s_ml = reinterpret_cast<float2*>(sRaw + 2 * C::RAW_BYTES);  // [2][128]
  Bars* bars = reinterpret_cast<Bars*>(s_ml + 2 * 128);
  const XAttn& a = args.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &bars->abort_flag;
  constexpr bool masked = MASKED;  // a.key_mask is given

  if (threadIdx.x == 0) {
    for (int i = 0; i < QST; ++i) {
      mbar_init(&bars->q_full[i], 1);
      mbar_init(&bars->q_free[i], 1);
    }
    for (int i = 0; i < KVST; ++i) mbar_init(&bars->kv_full[i], CODES ? 4 : 1);  // 4 converting warps, or TMA
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->raw_full[i], 1);
      mbar_init(&bars->raw_free[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->kv_free[i], 1);
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_half[i][0], 4);
      mbar_init(&bars->p_half[i][1], 4);
      mbar_init(&bars->o_full[i], 1);
      mbar_init(&bars->o_free[i], 4);
      mbar_init(&bars->ml_full[i], 4);
      mbar_init(&bars->ml_free[i], 4);
    }
    mbar_init(&bars->ready[0], 1);
    mbar_init(&bars->ready[1], 1);
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
  // All 512 columns are this CTA's, so they start at 0: a constant, which
  // keeps the products' operands in uniform registers.
  constexpr uint32_t tmem = 0;
  if (bars->tmem_base != 0) {  // (cannot happen; the same for the whole CTA)
    if (threadIdx.x == 0 && atomicCAS(&g_status.code, 0, H3B_ERR_DEVICE) == 0) g_status.site = 31;
    if (warp == 9) tmem_dealloc(bars->tmem_base, 512);
    return;
  }
  auto s_col = [](int i) { return static_cast<uint32_t>(i * 128); };
  auto o_col = [](int i) { return static_cast<uint32_t>(256 + i * 128); };

  Unit u;  // each role walks the CTA's units on its own
  u.first(args);

  if (warp >= 8 && warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CONTROL));
    if (warp == 8 && lane == 0) {
      // ------------------------------------------------------------ TMA
      // Slot of the c-th Q tile: c % ring; its free barrier has completed
      // phase (c / ring) - 1 when the tile before it is read, and its next
      // phase needs this very load: a parity wait is one phase behind.  So it
      // is for K and V: round t + 1 of the products needs V_t, round t needs K_t.
      prefetch_tmap(&tm_q);
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
      int qc = 0;
      bool ok = true;
      auto load_q = [&](const Unit& u, int i) {
        const int s = qc % QST;
        if (qc >= QST && !lane_wait<false>(&bars->q_free[s], (qc / QST - 1) & 1, 1, abort_flag)) return false;
        mbar_arrive_expect_tx(&bars->q_full[s], C::TILE_BYTES);
        for (int h = 0; h < C::HALVES; ++h)
          tma_load_4d(sQ + s * C::TILE_BYTES + h * C::HALF_BYTES, &tm_q, h * 64, u.q0 + i * BQ, u.head, u.b,
                      &bars->q_full[s]);
        ++qc;
        return true;
      };
      // K_t overwrites K_{t-2}, released with round t - 2 of the products; V_t
      // overwrites V_{t-2}, released with round t - 1 (see the matrix warp).
      // Cache: the blocks of a tile, looked up a tile ahead (an absent block
      // loads block 0: it may hold anything, see warp 10).
      int ids[4] = {0, 0, 0, 0};
      auto look_up = [&](const Unit& u, int j) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (g * a.block_tokens < BKV) ids[g] = max(block_of(a, u.b, (u.j0 + j) * BKV + g * a.block_tokens), 0);
      };
      auto load_kv = [&](const CUtensorMap* tm, const Unit& u, int j, int t, int v) {
        const int kvh = args.group == 1 ? u.head : u.head / args.group;
        const int key0 = (u.j0 + j) * BKV;
        if constexpr (CODES) {
          // codes: slot v, converted once a tile
          if (t > 0 && !lane_wait<false>(&bars->raw_free[v], (t - 1) & 1, 2, abort_flag)) return false;
          mbar_arrive_expect_tx(&bars->raw_full[v], C::RAW_BYTES);
          const int rows = a.block_tokens;
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if (g * rows < BKV)
              tma_load_3d(sRaw + v * C::RAW_BYTES + g * rows * D, tm, 0, 0, ids[g] * a.kv_heads + kvh, &bars->raw_full[v]);
        } else {
          const int s = 2 * (t & 1) + v, round = t < 2 ? -1 : t - 2 + v;
          if (round >= 0 && !lane_wait<false>(&bars->kv_free[round & 1], (round >> 1) & 1, 2, abort_flag)) return false;
          mbar_arrive_expect_tx(&bars->kv_full[s], C::TILE_BYTES);
          for (int h = 0; h < C::HALVES; ++h)
            tma_load_4d(sKV + s * C::TILE_BYTES + h * C::HALF_BYTES, tm, h * 64, key0, kvh, u.b, &bars->kv_full[s]);
        }
        return true;
      };
      int t = 0, loaded = 0;
#pragma unroll 1
      for (; u.x < args.units && ok; u.next<false>(args)) {
#pragma unroll 1
        for (int j = 0; j < u.n && ok; ++j, ++t) {
          if (CODES && j == 0) look_up(u, 0);
          if (!CODES && j == 0) {  // the next unit's Q into L2: its slots come free late
            Unit v = u;
            v.next<false>(args);
            if (v.x < args.units && v.n > 0) {
              for (int h = 0; h < C::HALVES; ++h) {
                tma_prefetch_4d(&tm_q, h * 64, v.q0, v.head, v.b);
                if (v.two) tma_prefetch_4d(&tm_q, h * 64, v.q0 + BQ, v.head, v.b);
              }
            }
          }
          if (j == 0) ok = load_q(u, 0);
          if (ok && (ok = load_kv(&tm_k, u, j, t, 0))) loaded = 2 * t + 1;
          if (ok && j == 0 && u.two) ok = load_q(u, 1);
          if (ok && (ok = load_kv(&tm_v, u, j, t, 1))) loaded = 2 * t + 2;
          if (CODES && j + 1 < u.n) look_up(u, j + 1);
        }
      }
      if (!ok || *abort_flag) {
        // let the copies in flight land (bounded) before the CTA goes
        for (int c = max(0, qc - QST); c < qc; ++c)
          lane_wait<false>(&bars->q_full[c % QST], (c / QST) & 1, 10, nullptr);
        for (int c = max(0, loaded - 2); CODES && c < loaded; ++c)
          lane_wait<false>(&bars->raw_full[c & 1], (c >> 1) & 1, 12, nullptr);
        for (int c = max(0, loaded - KVST); !CODES && c < loaded; ++c)
          lane_wait<false>(&bars->kv_full[c % KVST], (c / KVST) & 1, 11, nullptr);
      }
    } else if (warp == 9) {
      // ------------------------------------------------------------ MMA
      // The warp runs the schedule converged: all lanes poll, one elected
      // lane issues.  Round t of the products is
      //   P V_0(t-1)  S_0(t)  P V_1(t-1)  S_1(t)
      // What stands between a P tile and the products behind it is on every
      // tile's critical path (softmax -> P V -> S -> softmax), and this warp
      // shares its scheduler and instruction cache with softmax warps that
      // stream through 10 KB of code a tile.  So it only waits for `ready` and
      // for P, and issues; warp 10 does everything else ahead of it.  (With
      // the bookkeeping here a round took 5000 cycles, 3000 of them with the
      // softmax warps idle.)
      // Every barrier waited on completes once per use and its next use
      // depends on what this warp issues after the wait.
      uint32_t phases = 0;  // bit i: parity of row tile i's P; bit 2 + i: of its O; bit 4 + i: O begun once
      bool ok = true;
#pragma unroll 1
      for (int t = 0; ok; ++t) {
        ok = lane_wait<true>(&bars->ready[t & 1], (t >> 1) & 1, 4, abort_flag);
        // (the reduction makes the word uniform for the compiler too)
        const uint32_t todo = ok ? *const_cast<volatile uint32_t*>(&bars->todo[t & 1]) : static_cast<uint32_t>(R_END);
        const uint32_t r = __reduce_or_sync(0xffffffffu, todo);
        const uint64_t kd = sdesc_kmajor_sw128(smem_u32(sKV + 2 * (t & 1) * C::TILE_BYTES));
        const uint64_t vd =
            sdesc_mnmajor_sw128(smem_u32(sKV + (2 * ((t + 1) & 1) + 1) * C::TILE_BYTES), C::HALF_BYTES, 1024);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool do_pv = (r & (i ? R_PV1 : R_PV0)) != 0, do_s = (r & (i ? R_S1 : R_S0)) != 0;
          const uint32_t qs = (r >> (i ? R_Q1_SHIFT : R_Q0_SHIFT)) & 7u;
          const uint64_t qd = sdesc_kmajor_sw128(smem_u32(sQ + qs * C::TILE_BYTES));
          const uint32_t s_tmem = tmem + s_col(i), o_tmem = tmem + o_col(i);
          if (do_pv) {
            if (r & R_PV_FIRST) {  // O_i of the unit before has been read (its phase: one a unit)
              if ((phases >> (4 + i)) & 1) {
                ok = lane_wait<true>(&bars->o_free[i], (phases >> (2 + i)) & 1, 6, abort_flag) && ok;
                phases ^= 4u << i;
              }
              phases |= 16u << i;
            }
            // as the softmax delivers: 64 keys a half
            ok = lane_wait<true>(&bars->p_half[i][0], (phases >> i) & 1, 5, abort_flag) && ok;
            __syncwarp();
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_f16_ts(o_tmem, s_tmem + kk * 8, desc_add_lo(vd, static_cast<uint32_t>(kk * (2048 >> 4))), IDESC_O,
                           kk == 0 ? (~r & R_PV_FIRST) : 1u);
            }
            ok = lane_wait<true>(&bars->p_half[i][1], (phases >> i) & 1, 5, abort_flag) && ok;
            phases ^= 1u << i;
          }
          // (Q_1 is loaded half a round later than Q_0: its slot is Q_0's of the unit before)
          if (i == 1 && do_s && (r & R_S_FIRST))
            ok = lane_wait<true>(&bars->q_full[qs], (r & R_Q1_PHASE) ? 1u : 0u, 3, abort_flag) && ok;
          __syncwarp();
          tc_fence_after();
          if (elect_one()) {
            if (do_pv) {
#pragma unroll
              for (int kk = 4; kk < 8; ++kk)
                mma_f16_ts(o_tmem, s_tmem + kk * 8, desc_add_lo(vd, static_cast<uint32_t>(kk * (2048 >> 4))), IDESC_O, 1u);
              if (r & R_PV_LAST) tc_commit(&bars->o_full[i]);
            }
            if (do_s) {
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk) {
                const uint32_t at = static_cast<uint32_t>((kk >> 2) * (C::HALF_BYTES >> 4) + (kk & 3) * 2);
                mma_f16_ss(s_tmem, desc_add_lo(qd, at), desc_add_lo(kd, at), IDESC_S, kk > 0);
              }
              tc_commit(&bars->s_full[i]);
              if (r & R_S_LAST) tc_commit(&bars->q_free[qs]);
            }
            if (r & R_END) tc_commit(&bars->s_full[i]);  // info says that there is no tile
            if (i == 1) tc_commit(&bars->kv_free[t & 1]);
          }
          __syncwarp();
        }
        ok = __all_sync(0xffffffffu, ok) && (r & R_END) == 0;
      }
      if (elect_one()) tc_commit(&bars->drain);
      __syncwarp();
      warp_wait(&bars->drain, 0, 8, nullptr);
    } else if (warp == 10) {
      // ------------------------------------------------------------ rounds
      // Ahead of the issuing warp: says what round t consists of, waits for
      // K_t, V_{t-1} and at a unit's start its Q_0, and zeroes the rows of
      // V_{t-1} that are left out.  It is at most two rounds ahead (K_t
      // overwrites K_{t-2}, released with round t - 2), so todo[] and ready[]
      // of that parity are free again, and every tile's barrier is waited for
      // once: one phase behind.
      int qc = 0;
      uint32_t pv = 0;                  // R_PV* of the tile before
      uint32_t vw[4] = {0, 0, 0, 0};    // its kept columns
      uint32_t ic[2] = {0, 0};          // infos written, per row tile
      int id_here = 0, id_ahead = 0;    // cache: blocks of this tile and the next, scales of this
      float k_here = 1.0f, v_here = 1.0f;
      int kvh = 0;                      // the unit's key head
      bool ok = true;
      while (u.x < args.units && u.n == 0) u.next(args);
      int j = 0;
      bool end = false;
#pragma unroll 1
      for (int t = 0; !end; ++t) {
        const bool more = u.x < args.units;
        const int key0 = (u.j0 + j) * BKV;
        uint32_t r = pv;
        uint32_t w[4] = {~0u, ~0u, ~0u, ~0u};
        if (more) {
          const uint32_t mb = masked ? mask_bytes(a, u.b, key0, u.len, lane) : 0u;
          r |= R_S0 | (u.two ? R_S1 : 0u) | (j == u.n - 1 ? R_S_LAST : 0u) | ((qc % QST) << R_Q0_SHIFT) |
               (((qc + 1) % QST) << R_Q1_SHIFT) | (j == 0 ? R_S_FIRST : 0u) |
               ((((qc + 1) / QST) & 1) ? R_Q1_PHASE : 0u);
          if constexpr (SCALED) {
            if (lane < 4) {
              if (j == 0) {
                id_ahead = block_of(a, u.b, key0 + 32 * lane);
                kvh = args.group == 1 ? u.head : u.head / args.group;
              }
              id_here = id_ahead;
              if (j + 1 < u.n) id_ahead = block_of(a, u.b, key0 + BKV + 32 * lane);
              const int at = max(id_here, 0) * a.kv_heads + kvh;  // (below 2^31: checked on the host)
              k_here = __ldg(a.k_scale + at);
              v_here = __ldg(a.v_scale + at);
            }
          }
          ok = warp_wait(&bars->kv_full[2 * (t & 1)], (t >> 1) & 1, 9, abort_flag);
          if (j == 0) ok = ok && warp_wait(&bars->q_full[qc % QST], (qc / QST) & 1, 3, abort_flag);
          keep_words(masked, mb, u.len - key0, w);
        }
        float kf = 1.0f, vs = 1.0f;
        if constexpr (SCALED) {
          // lane g (of four): the block of columns 32 g .., its scales, looked
          // up while the tile was awaited (the block of the next one, too)
          int id = 0;
          if (more && lane < 4) {
            id = id_here;
            kf = k_here;
            vs = v_here;
          }
          const uint32_t there = __ballot_sync(0xffffffffu, id >= 0);
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (((there >> c) & 1u) == 0) w[c] = 0u;
          // (columns that are all left out: their scales may be anything, and an
          // infinity would make NaN of -inf)
          if (((lane & 2) ? (lane & 1) ? w[3] : w[2] : (lane & 1) ? w[1] : w[0]) == 0) kf = vs = 1.0f;
          kf = fmaxf(kf * args.scale_log2, 1e-37f);  // (a factor of 0 would make NaN of -inf)
          vs = fmaxf(vs, KV8_SCALE_MIN);
        }
        if (pv != 0) {
          ok = ok && warp_wait(&bars->kv_full[2 * ((t + 1) & 1) + 1], ((t - 1) >> 1) & 1, 7, abort_flag);
          if (!CODES && ok && (vw[0] & vw[1] & vw[2] & vw[3]) != ~0u) {
            zero_left_out<C::HALVES>(smem_u32(sKV + (2 * ((t + 1) & 1) + 1) * C::TILE_BYTES), vw, lane);
            fence_proxy_async_smem();
          }
        }
        if (!ok) break;
        const int causal = a.causal ? u.len - a.s_q + u.q0 + 1 - key0 : BKV;
        const uint32_t flags = (j == 0 ? T_FIRST : 0u) | (j == u.n - 1 ? T_LAST : 0u) |
                               ((w[0] & w[1] & w[2] & w[3]) == ~0u ? T_WHOLE : 0u);
        pv = 0;
        const bool two = u.two;
        if (more) {
          pv = R_PV0 | (two ? R_PV1 : 0u) | (j == 0 ? R_PV_FIRST : 0u) | (j == u.n - 1 ? R_PV_LAST : 0u);
        }
        end = pv == 0;
        if (lane < 2 && (lane == 0 || two || end)) {
          volatile TileInfo* info = &bars->info[lane][(lane ? ic[1] : ic[0]) % INFOS];
          const int sees = causal + lane * BQ;
          info->keep[0] = w[0];
          info->keep[1] = w[1];
          info->keep[2] = w[2];
          info->keep[3] = w[3];
          info->causal = sees;
          info->flags = end ? static_cast<uint32_t>(T_END) : sees < BKV ? (flags & ~T_WHOLE) | T_CAUSAL : flags;
        }
        if constexpr (SCALED) {
          if (lane < 4) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              volatile TileInfo* info = &bars->info[i][ic[i] % INFOS];
              info->k_factor[lane] = kf;
              info->v_log2[lane] = __log2f(vs);
              info->v_inv[lane] = __fdividef(1.0f, vs);  // (a call of the IEEE division is fetched anew each tile)
            }
          }
        }
        ++ic[0];
        if (two) ++ic[1];
        if (lane == 0) *const_cast<volatile uint32_t*>(&bars->todo[t & 1]) = r | (end ? R_END : 0u);
#pragma unroll
        for (int c = 0; c < 4; ++c) vw[c] = w[c];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->ready[t & 1]);
        if (more && ++j == u.n) {
          j = 0;
          qc += two ? 2 : 1;
          do {
            u.next(args);
          } while (u.x < args.units && u.n == 0);
        }
      }
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_SOFTMAX));
    const int wg = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + s_col(wg) + lane_off;
    const uint32_t o_tmem = tmem + o_col(wg) + lane_off;
    float m_run = -INFINITY;  // running max, log2 domain
    float l_run = 0.0f;
    uint32_t oc = 0;  // units seen
#pragma unroll 1
    for (uint32_t sc = 0;; ++sc) {
      {
        // S_i of the next tile is published only after this tile's P_i
        if (!warp_wait<true>(&bars->s_full[wg], sc & 1, 20, abort_flag)) break;
        tc_fence_after();
        const volatile TileInfo* info = &bars->info[wg][sc % INFOS];
        const uint32_t flags = info->flags;
        if (flags & T_END) break;
        const bool first = (flags & T_FIRST) != 0;
        if (first) {
          m_run = -INFINITY;
          l_run = 0.0f;
        }
        if (!MASKED && (flags & T_WHOLE) == 0) {
          // Left-out columns become -inf in TMEM, 32 at a time in a loop that
          // stays out of the instruction cache of whole tiles.  (With a mask
          // every tile has some: there they are replaced in registers below.)
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t keep = info->keep[c];
            if (flags & T_CAUSAL) {
              const int v = info->causal + row - 32 * c;
              keep &= v >= 32 ? 0xffffffffu : (v <= 0 ? 0u : (1u << v) - 1u);
            }
            if (__all_sync(0xffffffffu, keep == 0xffffffffu)) continue;
            uint32_t o[32];
            tmem_ld32p(s_tmem + c * 32, o);
            tmem_wait_fence<1>(o);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if ((keep & (1u << e)) == 0) o[e] = __float_as_uint(-INFINITY);
            __syncwarp();
            tmem_st32(s_tmem + c * 32, o);
          }
          tc_wait_st();
        }
        // The first tile looks for its maximum first.  After it, half 0 is
        // exponentiated against the running maximum while the tile's is found;
        // only where that outgrew it by more than the threshold the warp goes
        // round again (P is not written over S yet).
        uint32_t r[128];
        float m_use = m_run;
        float sum = 0.0f;
        bool slow = first;
#pragma unroll 1
        for (int round = 0; round < 2; ++round) {
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32p(s_tmem + c * 32, r + 32 * c);
          tmem_wait_fence<4>(r);
          if constexpr (MASKED) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint32_t keep = info->keep[c];
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if ((keep & (1u << e)) == 0) r[32 * c + e] = __float_as_uint(-INFINITY);
            }
          }
          float fx[4], ox[4];
          if constexpr (SCALED) {
            const float4 f = lds4(info->k_factor), o = lds4(info->v_log2);
            fx[0] = f.x, fx[1] = f.y, fx[2] = f.z, fx[3] = f.w;
            ox[0] = o.x, ox[1] = o.y, ox[2] = o.z, ox[3] = o.w;
          }
          if (slow) {
            float m_tile;
            if constexpr (SCALED) {
              m_tile = -INFINITY;
#pragma unroll
              for (int g = 0; g < 4; ++g) m_tile = fmaxf(m_tile, fmaf(row_max32(r + 32 * g), fx[g], ox[g]));
            } else {
              m_tile = fmaxf(row_max64(r), row_max64(r + 64)) * args.scale_log2;
            }
            const bool rescale = m_tile > m_run + RESCALE_THRESHOLD;
            if (rescale) m_use = m_tile;
            if (__any_sync(0xffffffffu, rescale)) {
              const float factor = rescale ? ex2(m_run - m_use) : 1.0f;
              l_run *= factor;
              if (!first) {
#pragma unroll 1
                for (int c = 0; c < D / 8; ++c) {  // (few registers: the tile's scores stay live)
                  uint32_t o[8];
                  tmem_ld8(o_tmem + c * 8, o);
                  tc_wait_ld();
#pragma unroll
                  for (int e = 0; e < 8; ++e) {
                    asm volatile("" : "+r"(o[e]));
                    o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
                  }
                  tmem_st8(o_tmem + c * 8, o);
                }
              }
              if (rescale) m_run = m_use;
            }
          }
          const float neg_m = m_use == -INFINITY ? 0.0f : UP<F16> - m_use;
          float2 sm;
          if constexpr (SCALED) {
            sm = exp_codes64<F16, true>(r, r, make_float2(fx[0], fx[1]), make_float2(ox[0] + neg_m, ox[1] + neg_m),
                                        lds2(info->v_inv), fx, ox);
          } else {
            sm = exp_pack64<F16, true>(r, r, args.scale_log2, neg_m);
            sm.y *= args.scale_log2;
          }
          sum = sm.x;
          if (slow) break;
          slow = __any_sync(0xffffffffu, sm.y > m_run + RESCALE_THRESHOLD);
          if (!slow) break;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h == 1) {
            const float neg_m = m_use == -INFINITY ? 0.0f : UP<F16> - m_use;
            if constexpr (SCALED) {
              const float f[4] = {0.f, 0.f, 0.f, 0.f};
              const float2 o = lds2(info->v_log2 + 2);
              sum += exp_codes64<F16, false>(r + 64, r + 32, lds2(info->k_factor + 2),
                                             make_float2(o.x + neg_m, o.y + neg_m), lds2(info->v_inv + 2), f, f).x;
            } else {
              sum += exp_pack64<F16, false>(r + 64, r + 32, args.scale_log2, neg_m).x;
            }
          }
          tmem_st32(s_tmem + 32 * h, *reinterpret_cast<uint32_t(*)[32]>(r + 32 * h));
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->p_half[wg][h]);
        }
        l_run += sum;
        if (flags & T_LAST) {
          // ---- the row statistics, to the storing warps
          if (oc > 0 && !warp_wait<true>(&bars->ml_free[wg], (oc - 1) & 1, 22, abort_flag)) break;
          ++oc;
          s_ml[wg * 128 + row] = make_float2(m_run - UP<F16>, l_run);
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->ml_full[wg]);
        }
      }
    }
  } else {
    // ------------------------------------------------------------ stores
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_STORE));
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int64_t total_rows = static_cast<int64_t>(a.batch) * a.heads * a.s_q;
    uint32_t oc0 = 0, oc1 = 0;
    bool ok = true;
    auto store = [&](const Unit& u) {  // a unit's rows
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        if (!ok || (i == 1 && !u.two)) continue;
        float2 ml = make_float2(-INFINITY, 0.0f);
        const uint32_t phase = (i ? oc1 : oc0) & 1;
        if (u.n > 0) {
          // both complete once a unit, and again only after this warp's arrivals below
          ok = warp_wait(&bars->ml_full[i], phase, 23, abort_flag) &&
               warp_wait(&bars->o_full[i], phase, 24, abort_flag);
          if (!ok) continue;
          if (i) ++oc1; else ++oc0;
          tc_fence_after();
          ml = s_ml[i * 128 + row];
        }
        const int q_row = u.q0 + i * BQ + row;
        const bool in = q_row < a.s_q;
        const int64_t lse_row = (static_cast<int64_t>(u.b) * a.heads + u.head) * a.s_q + q_row;
        const float inv_l = ml.y == 0.0f ? 0.0f : 1.0f / ml.y;  // (0: no key; a NaN stays one)
        // 32 columns at a time in a rolled loop: this code runs once a unit, so
        // it is fetched anew each time (unrolled, a 128-row tile took 4500
        // cycles).  O is given back before its last columns are stored.
        uint16_t* orow =
            static_cast<uint16_t*>(a.o) + u.b * a.o_stride[0] + q_row * a.o_stride[1] + u.head * a.o_stride[2];
        float* prow = a.part_o + (u.split * total_rows + lse_row) * D;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          if (u.n > 0) {
            tmem_ld32p(tmem + o_col(i) + c * 32 + lane_off, r);
            tmem_wait_fence<1>(r);
            if (c == D / 32 - 1) {  // O_i and the statistics are read
              tc_fence_before();
              __syncwarp();
              if (lane == 0) {
                mbar_arrive(&bars->o_free[i]);
                mbar_arrive(&bars->ml_free[i]);
              }
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) r[e] = 0u;
          }
          if (a.splits > 1) {
            if (in) {
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                uint32_t v[8];
#pragma unroll
                for (int t = 0; t < 8; ++t) v[t] = r[e + t];
                st_global_v8(prow + c * 32 + e, v);
              }
            }
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float2 x = mul2(make_float2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])),
                                    make_float2(inv_l, inv_l));
              r[e] = pack16x2<F16>(x.x, x.y);
            }
            if (in && args.o_wide) {
#pragma unroll
              for (int e = 0; e < 16; e += 8) {
                uint32_t v[8];
#pragma unroll
                for (int t = 0; t < 8; ++t) v[t] = r[e + t];
                st_global_v8(orow + c * 32 + 2 * e, v);
              }
            } else if (in) {
#pragma unroll
              for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<uint4*>(orow + c * 32 + 2 * e) = make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3]);
            }
          }
          __syncwarp();  // the next tcgen05.ld is for the whole warp
        }
        if (in) {
          if (a.splits > 1) {
            a.part_ml[u.split * total_rows + lse_row] = ml;
          } else if (a.lse != nullptr) {
            a.lse[lse_row] = ml.y == 0.0f ? -INFINITY : (ml.x + __log2f(ml.y)) * LN2;
          }
        }
      }
    };
    if constexpr (CODES) {
      // These warps also turn the codes into operands: K_t, then V_t, row
      // `row` each thread.  A finished unit is stored between the next one's
      // first K and first V: its last P V runs in the round that has that K.
      int t = 0;
      Unit done = u;
      bool have = false;
      const int shift = a.block_tokens == 32 ? 5 : (a.block_tokens == 64 ? 6 : 7);
      // table entry of the thread's row of tile j, fetched a tile ahead of its use
      auto entry = [&](int j) -> int {
        const int x = ((u.j0 + j) * BKV + row) >> shift;
        return j < u.n && x < a.max_blocks ? __ldg(a.table + static_cast<int64_t>(u.b) * a.max_blocks + x) : -1;
      };
#pragma unroll 1
      for (; u.x < args.units && ok; u.next(args)) {
        if (u.n == 0) {
          store(u);
          continue;
        }
        int id = entry(0);
#pragma unroll 1
        for (int j = 0; j < u.n && ok; ++j, ++t) {
          const int id_next = entry(j + 1);
#pragma unroll 1
          for (int v = 0; v < 2 && ok; ++v) {
            if (v == 1 && j == 0 && have) store(done);
            const int round = t < 2 ? -1 : t - 2 + v;  // K_t overwrites K_{t-2}, V_t V_{t-2}
            ok = ok && (round < 0 || warp_wait(&bars->kv_free[round & 1], (round >> 1) & 1, 26, abort_flag)) &&
                 warp_wait(&bars->raw_full[v], t & 1, 25, abort_flag);
            if (!ok) break;
            const int slot = 2 * (t & 1) + v;
            const uint32_t dst = smem_u32(sKV + slot * C::TILE_BYTES);
            convert_row<D, KIND, F16>(smem_u32(sRaw + v * C::RAW_BYTES), dst, row);
            if (v == 1 && !((u.j0 + j) * BKV + row < u.len && id >= 0 && id < a.num_blocks)) zero_row<D>(dst, row);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&bars->kv_full[slot]);
              mbar_arrive(&bars->raw_free[v]);
            }
          }
          id = id_next;
        }
        done = u;
        have = true;
      }
      if (have && ok) store(done);
    } else {
#pragma unroll 1
      for (; u.x < args.units && ok; u.next(args)) store(u);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, bool F16, KvKind KIND, bool MASKED = false, bool PRE = false>
int launch(const XAttn& a, cudaStream_t stream) {
  const CUtensorMapDataType dt = F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap tq, tk, tv;
  auto encode = [&](CUtensorMap* m, const void* p, const int64_t (&st)[3], int seq, int heads) {
    const uint64_t dims[4] = {D, static_cast<uint64_t>(seq > 0 ? seq : 1), static_cast<uint64_t>(heads),
                              static_cast<uint64_t>(a.batch)};
    const uint64_t sb[3] = {static_cast<uint64_t>(st[1]) * 2, static_cast<uint64_t>(st[2]) * 2,
                            static_cast<uint64_t>(st[0]) * 2};
    const uint32_t box[4] = {64, 128, 1, 1};
    return h3b::encode_4d(m, dt, p, dims, sb, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  int rc = encode(&tq, a.q, a.q_stride, a.s_q, a.heads);
  if constexpr (PRE) {  // [batch, kv_heads, s_kv, D]
    const int64_t st[3] = {static_cast<int64_t>(a.kv_heads) * a.s_kv * D, D, static_cast<int64_t>(a.s_kv) * D};
    if (rc == H3B_OK) rc = encode(&tk, a.pre_k, st, a.s_kv, a.kv_heads);
    if (rc == H3B_OK) rc = encode(&tv, a.pre_v, st, a.s_kv, a.kv_heads);
  } else if constexpr (KIND == KV_DENSE) {
    if (rc == H3B_OK) rc = encode(&tk, a.k, a.kv_stride, a.s_kv, a.kv_heads);
    if (rc == H3B_OK) rc = encode(&tv, a.v, a.kv_stride, a.s_kv, a.kv_heads);
  } else {
    const uint64_t slabs = static_cast<uint64_t>(a.num_blocks) * a.kv_heads;
    const uint64_t slab = static_cast<uint64_t>(a.block_tokens) * D;
    const uint32_t rows = static_cast<uint32_t>(a.block_tokens < BKV ? a.block_tokens : BKV);
    constexpr CUtensorMapSwizzle sw = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    for (int i = 0; i < 2 && rc == H3B_OK; ++i)
      rc = h3b::encode_3d(i ? &tv : &tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, i ? a.v : a.k, D, a.block_tokens, slabs, D, slab,
                          D, rows, 1, sw);
  }
  if (rc != H3B_OK) return rc;
  auto kernel = xattn_tile_kernel<D, F16, KIND, MASKED, PRE>;
  static h3b::OncePerDevice attr;
  rc = attr.run(h3b::device(), [=] { return h3b::allow_smem(kernel, smem_bytes<D, KIND, PRE>()); });
  if (rc != H3B_OK) return rc;
  TileArgs args{};
  args.a = a;
  args.group = a.heads / a.kv_heads;
  args.q_tiles = (a.s_q + 2 * BQ - 1) / (2 * BQ);
  const int64_t units = static_cast<int64_t>(a.batch) * a.heads * a.splits * args.q_tiles;
  if (units > 0x3fffffff) return H3B_ERR_SHAPE;
  args.units = static_cast<int>(units);
  args.scale_log2 = a.scale * LOG2E;
  args.o_wide = (reinterpret_cast<uintptr_t>(a.o) & 31u) == 0 && a.o_stride[0] % 16 == 0 && a.o_stride[1] % 16 == 0 &&
                a.o_stride[2] % 16 == 0;
  const int sms = h3b::num_sms();
  int step = static_cast<int>(units < sms ? units : sms);
  args.step_q = step % args.q_tiles;
  step /= args.q_tiles;
  args.step_split = step % a.splits;
  step /= a.splits;
  args.step_head = step % a.heads;
  args.step_b = step / a.heads;
  kernel<<<static_cast<unsigned>(units < sms ? units : sms), THREADS, smem_bytes<D, KIND, PRE>(), stream>>>(tq, tk, tv, args);
  return h3b::launch_status();
}

}  // namespace

namespace h3b {

int xattn_tile_splits(const XAttn& a) {
  // Ranges of keys per row tile: units run in rounds of one per SM, so the
  // call takes about ceil(units / SMs) / splits of a whole unit; a split
  // costs the write and the second read of its fp32 rows, about as much as
  // half a tile of 128 keys of work.
  const int64_t tiles = (static_cast<int64_t>(a.s_kv) + BKV - 1) / BKV;
  const int64_t base = static_cast<int64_t>(a.batch) * a.heads * ((a.s_q + 2 * BQ - 1) / (2 * BQ));
  const int sms = num_sms();
  int best = 1;
  double cost = 1e30;
  for (int s = 1; s <= 32 && s <= tiles; ++s) {
    const double per = static_cast<double>((tiles + s - 1) / s) + 1.0 + (s > 1 ? 2.0 : 0.0);
    const double c = static_cast<double>((base * s + sms - 1) / sms) * per;
    if (c < cost * 0.97) {
      cost = c;
      best = s;
    }
  }
  return best;
}

namespace {
template <int D, bool F16>
int launch_kind(const XAttn& a, cudaStream_t stream) {
  switch (a.kind) {
    case KV_INT8:
    case KV_E4M3:
      if (a.pre_k != nullptr) {  // written out: the kinds are the same then
        const int rc = kv8_expand_launch(a, stream);
        return rc == H3B_OK ? launch<D, F16, KV_INT8, false, true>(a, stream) : rc;
      }
      return a.kind == KV_INT8 ? launch<D, F16, KV_INT8>(a, stream) : launch<D, F16, KV_E4M3>(a, stream);
    default:
      return a.key_mask != nullptr ? launch<D, F16, KV_DENSE, true>(a, stream) : launch<D, F16, KV_DENSE>(a, stream);
  }
}
}  // namespace

int xattn_tile_launch(const XAttn& a, cudaStream_t stream) {
  int rc;
  if (a.head_dim == 128) {
    rc = a.dtype == H3B_F16 ? launch_kind<128, true>(a, stream) : launch_kind<128, false>(a, stream);
  } else {
    rc = a.dtype == H3B_F16 ? launch_kind<64, true>(a, stream) : launch_kind<64, false>(a, stream);
  }
  return rc != H3B_OK || a.splits == 1 ? rc : xattn_combine_launch(a, stream);
}

}  // namespace h3b
