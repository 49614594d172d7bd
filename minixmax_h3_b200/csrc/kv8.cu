// The 8-bit key/value cache: new rows quantised into its blocks, and the
// values read back.
//
// The pool holds, for K and for V, codes [num_blocks, kv_heads, block_tokens,
// D] (int8 or e4m3) and one fp32 scale per (block, head); token j of sequence
// b is row j % block_tokens of block table[b, j / block_tokens].  A row's
// value is code * scale.
//
// Append (positions start .. start + n): for each touched (block, head),
//   s' = max(amax of the new rows, 1e-12) / top         (top = 127 or 448)
//   s  = max(s_old, s') if the block held tokens before start, else s'
//   new rows:  code = round(x / s), rows held before: code = round(code s_old / s)
// in IEEE fp32 (round half even, int8 clamped to +-127, e4m3 saturating), so
// a block's codes do not depend on how its rows are spread over threads.  A
// held row is touched only when the block's scale grows: each of its values
// is then off by at most half a step more per growth.  Rows of the block
// behind the last token are zeroed.
//
// What bounds them is memory: append reads 2 bytes and writes 1 per value of
// the new rows (one CTA per touched block and head, the block's rows in
// registers between the maximum and the codes), read does 1 and 2 or 4.  4 x
// 4001 tokens x 8 heads of 128, e4m3: append 27 us (3.6 TB/s: each CTA loads,
// meets, and stores once, so its lengths, its rows and its table entry are
// waited for in turn; 32 us with the table's before the rows'), read of 4 x 5001
// tokens 21.5 us (5.7 TB/s).  The expansion for the tile kernel writes 16-bit
// operands without the scales: 24 heads x 32768 tokens 93 us (6.5 TB/s).
#include "h3b_common.cuh"
#include "h3b_host.hpp"
#include "xattn.hpp"

namespace {

constexpr int THREADS = 256;

// log2 of a block's tokens (32, 64 or 128)
__host__ __device__ constexpr int shift_of(int block_tokens) {
  return block_tokens == 32 ? 5 : (block_tokens == 64 ? 6 : 7);
}

struct AppendArgs {
  const void* src[2];      // new K, new V: [batch, n, kv_heads, D]
  int64_t src_stride[3];   // batch, token, head (elements)
  uint8_t* codes[2];
  float* scale[2];
  const int32_t* table;
  const int32_t* start;    // [batch]
  const int32_t* count;    // [batch] or null: n rows each
  int n, kv_heads, max_blocks, num_blocks, block_tokens;
};

template <bool F16>
H3B_DEV void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (F16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = bf16lo_to_f32(u[i]);
      x[2 * i + 1] = bf16hi_to_f32(u[i]);
    }
  }
}

// x / s, correctly rounded: from the correctly rounded reciprocal r of s,
// q = x r is within an ulp or so, the FMA gives its residual exactly, and one
// more FMA rounds the corrected quotient (Markstein's division; bits as
// __fdiv_rn for results that are not subnormal, and smaller ones are code 0
// either way).  s lies between 1e-12 / 448 and 3.4e38 / 127, so r is normal.
// Three operations against some ten of a division.
H3B_DEV float quotient(float x, float s, float r) {
  const float q = __fmul_rn(x, r);
  return __fmaf_rn(__fmaf_rn(-q, s, x), r, q);
}

// Four values -> four codes of one register, and back.
template <bool E4M3>
H3B_DEV uint32_t to_codes4(float a, float b, float c, float d) {
  if constexpr (E4M3) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
  } else {
    auto q = [](float v) -> uint32_t {
      return static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(v, -127.0f), 127.0f))) & 0xffu;
    };
    return q(a) | (q(b) << 8) | (q(c) << 16) | (q(d) << 24);
  }
}
template <bool E4M3>
H3B_DEV void from_codes4(uint32_t w, float (&x)[4]) {
  if constexpr (E4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t h;
      asm("{\n\t.reg .b16 two;\n\tcvt.u16.u32 two, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, two;\n\t}" : "=r"(h) : "r"(w >> (16 * i)));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int8_t>((w >> (8 * i)) & 0xffu));
  }
}

// The larger magnitudes of two pairs (a NaN gives way to a number).
template <bool F16>
H3B_DEV uint32_t max_abs2(uint32_t a, uint32_t b) {
  b &= 0x7fff7fffu;
  if constexpr (F16) {
    const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  } else {
    const __nv_bfloat162 m =
        __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
}

// One CTA = one touched block of one sequence, one head, K or V.
template <int D, bool F16, bool E4M3>
__global__ void __launch_bounds__(THREADS) kv8_append_kernel(const __grid_constant__ AppendArgs args) {
  constexpr int VPR = D / 8;             // 8-value pieces of a row
  constexpr int RPP = THREADS / VPR;     // rows per pass
  constexpr int PASSES = 128 / RPP;      // of the largest block
  constexpr float TOP = E4M3 ? 448.0f : 127.0f;
  __shared__ float s_max[THREADS / 32];
  const int b = blockIdx.z >> 1, which = blockIdx.z & 1, head = blockIdx.y;
  const int start = max(args.start[b], 0);
  int n = args.n;
  if (args.count != nullptr) n = max(0, min(n, args.count[b]));
  const int bt = args.block_tokens;
  const int j = (start >> shift_of(bt)) + static_cast<int>(blockIdx.x);
  const int lo = j * bt, end = start + n;
  if (j >= args.max_blocks || end <= max(lo, start)) return;
  const int id = args.table[static_cast<int64_t>(b) * args.max_blocks + j];
  const int first = max(start - lo, 0);          // first new row of the block
  const int last = min(end - lo, bt);            // one behind the last
  const uint16_t* src = static_cast<const uint16_t*>(args.src[which]) + b * args.src_stride[0] +
                        head * args.src_stride[2];
  const int row0 = threadIdx.x / VPR, col = (threadIdx.x % VPR) * 8;

  // (the rows' loads are under way before the table's entry is looked at)
  uint4 raw[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int r = p * RPP + row0;
    raw[p] = make_uint4(0, 0, 0, 0);
    if (r >= first && r < last)
      raw[p] = __ldcs(reinterpret_cast<const uint4*>(src + static_cast<int64_t>(lo + r - start) * args.src_stride[1] + col));
  }
  if (id < 0 || id >= args.num_blocks) return;
  const int64_t slab = static_cast<int64_t>(id) * args.kv_heads + head;
  uint8_t* codes = args.codes[which] + slab * bt * D;
  uint32_t top2 = 0;  // two running maxima, in the rows' type: exact
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    if (p * RPP < bt) top2 = max_abs2<F16>(max_abs2<F16>(max_abs2<F16>(max_abs2<F16>(top2, raw[p].x), raw[p].y), raw[p].z), raw[p].w);
  }
  float mx = F16 ? fmaxf(__half2float(__ushort_as_half(top2 & 0xffffu)), __half2float(__ushort_as_half(top2 >> 16)))
                 : fmaxf(bf16lo_to_f32(top2), bf16hi_to_f32(top2));
  mx = warp_max(mx);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = mx;
  const float held = first > 0 ? args.scale[which][slab] : 0.0f;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) mx = fmaxf(mx, s_max[w]);
  const float scale = fmaxf(held, __fdiv_rn(fmaxf(mx, 1e-12f), TOP));
  if (threadIdx.x == 0) args.scale[which][slab] = scale;
  const float recip = __frcp_rn(scale);
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    if (p * RPP >= bt) break;
    const int r = p * RPP + row0;
    uint2* dst = reinterpret_cast<uint2*>(codes + r * D + col);
    uint2 w = make_uint2(0, 0);
    if (r >= first && r < last) {
      float x[8];
      unpack8<F16>(raw[p], x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = quotient(x[e], scale, recip);
      w.x = to_codes4<E4M3>(x[0], x[1], x[2], x[3]);
      w.y = to_codes4<E4M3>(x[4], x[5], x[6], x[7]);
    } else if (r < first) {
      if (scale == held) continue;
      w = *dst;
      float x[8], y[4];
      from_codes4<E4M3>(w.x, y);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = quotient(__fmul_rn(y[e], held), scale, recip);
      from_codes4<E4M3>(w.y, y);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 + e] = quotient(__fmul_rn(y[e], held), scale, recip);
      w.x = to_codes4<E4M3>(x[0], x[1], x[2], x[3]);
      w.y = to_codes4<E4M3>(x[4], x[5], x[6], x[7]);
    }
    *dst = w;
  }
}

struct ReadArgs {
  const uint8_t* codes[2];
  const float* scale[2];
  void* dst[2];  // [batch, max_len, kv_heads, D] dense
  const int32_t* table;
  const int32_t* lens;
  int batch, max_len, kv_heads, max_blocks, num_blocks, block_shift;
};

// OUT: 0 bf16, 1 f16, 2 f32.  One thread = 16 codes of one token's head.
template <int D, bool E4M3, int OUT>
__global__ void __launch_bounds__(THREADS) kv8_read_kernel(const __grid_constant__ ReadArgs args) {
  constexpr int VPR = D / 16;
  const int which = blockIdx.y;
  const int col = static_cast<int>(threadIdx.x % VPR) * 16;
  // (32-bit row numbers: 2^31 rows of 64 values are 274 GB)
  const uint32_t row = blockIdx.x * (THREADS / VPR) + threadIdx.x / VPR;  // (b, token, head)
  const uint32_t bt_row = row / static_cast<uint32_t>(args.kv_heads);
  const int head = static_cast<int>(row - bt_row * args.kv_heads);
  const uint32_t b32 = bt_row / static_cast<uint32_t>(args.max_len);
  const int tok = static_cast<int>(bt_row - b32 * args.max_len);
  const int64_t b = b32;
  if (b >= args.batch) return;
  float x[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = 0.0f;
  const int blk = tok >> args.block_shift;
  if (tok < args.lens[b] && blk < args.max_blocks) {
    const int id = args.table[b * args.max_blocks + blk];
    if (id >= 0 && id < args.num_blocks) {
      const int64_t slab = static_cast<int64_t>(id) * args.kv_heads + head;
      const float s = args.scale[which][slab];
      const uint4 w = __ldcs(reinterpret_cast<const uint4*>(
          args.codes[which] + ((slab << args.block_shift) + tok - (blk << args.block_shift)) * D + col));
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float y[4];
        from_codes4<E4M3>(u[k], y);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * k + e] = __fmul_rn(y[e], s);
      }
    }
  }
  const int64_t at = static_cast<int64_t>(row) * D + col;
  if constexpr (OUT == 2) {
    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(args.dst[which]) + at);
#pragma unroll
    for (int k = 0; k < 4; ++k) __stcs(dst + k, make_float4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]));
  } else {
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (OUT == 1) {
        const __half2 h = __floats2half2_rn(x[2 * k], x[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        w[k] = pack_bf16x2(x[2 * k], x[2 * k + 1]);
      }
    }
    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(args.dst[which]) + at);
    __stcs(dst, make_uint4(w[0], w[1], w[2], w[3]));
    __stcs(dst + 1, make_uint4(w[4], w[5], w[6], w[7]));
  }
}

// The codes themselves (no scale) as 16-bit numbers in the order of the
// tokens, heads first: each is exact.  Tokens up to the next 128 behind a
// sequence's length, and absent blocks, are 0; what lies further is not written.
template <int D, bool E4M3, bool F16>
__global__ void __launch_bounds__(THREADS) kv8_expand_kernel(const __grid_constant__ h3b::XAttn a) {
  constexpr int VPR = D / 16;
  const int col = static_cast<int>(threadIdx.x % VPR) * 16;
  const int tok = static_cast<int>(blockIdx.x * (THREADS / VPR) + threadIdx.x / VPR);
  const int head = blockIdx.y >> 1;
  const int64_t b = blockIdx.z;
  const bool values = (blockIdx.y & 1) != 0;
  if (tok >= a.s_kv) return;
  const int64_t row = (b * a.kv_heads + head) * static_cast<int64_t>(a.s_kv) + tok;
  const int shift = shift_of(a.block_tokens);
  const int len = max(0, min(a.s_kv, a.kv_lens[b]));
  if (tok >= (len + 127) / 128 * 128) return;
  const int id = a.table[b * a.max_blocks + (tok >> shift)];
  uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (tok < len && id >= 0 && id < a.num_blocks) {
    const int64_t slab = static_cast<int64_t>(id) * a.kv_heads + head;
    const uint4 c = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(values ? a.v : a.k) +
                                                          ((slab << shift) + (tok & (a.block_tokens - 1))) * D + col));
    const uint32_t u[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float y[4];
      from_codes4<E4M3>(u[k], y);
      w[2 * k] = pack16x2<F16>(y[0], y[1]);
      w[2 * k + 1] = pack16x2<F16>(y[2], y[3]);
    }
  }
  st_global_v8(static_cast<uint16_t*>(values ? a.pre_v : a.pre_k) + row * D + col, w);
}

bool block_ok(int64_t bt) { return bt == 32 || bt == 64 || bt == 128; }

}  // namespace

namespace h3b {

int kv8_expand_launch(const XAttn& a, cudaStream_t stream) {
  const int per = THREADS / (a.head_dim / 16);
  if (a.kv_heads > 32767) return H3B_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>((a.s_kv + per - 1) / per), static_cast<unsigned>(2 * a.kv_heads),
                  static_cast<unsigned>(a.batch));
  const bool f16 = a.dtype == H3B_F16, e4 = a.kind == KV_E4M3;
#define H3B_EXPAND(DD)                                                                       \
  (e4 ? (f16 ? kv8_expand_kernel<DD, true, true><<<grid, THREADS, 0, stream>>>(a)            \
             : kv8_expand_kernel<DD, true, false><<<grid, THREADS, 0, stream>>>(a))          \
      : (f16 ? kv8_expand_kernel<DD, false, true><<<grid, THREADS, 0, stream>>>(a)           \
             : kv8_expand_kernel<DD, false, false><<<grid, THREADS, 0, stream>>>(a)))
  if (a.head_dim == 128) H3B_EXPAND(128); else H3B_EXPAND(64);
#undef H3B_EXPAND
  return launch_status();
}

}  // namespace h3b

extern "C" int h3b_kv8_append(const void* k, const void* v, int x_dtype, int64_t batch, int64_t n, int64_t kv_heads,
                              int64_t head_dim, int64_t batch_stride, int64_t seq_stride, int64_t head_stride,
                              uint8_t* k_codes, uint8_t* v_codes, float* k_scale, float* v_scale, int code_type,
                              int64_t num_blocks, int64_t block_tokens, const int32_t* table, int64_t max_blocks,
                              const int32_t* start, const int32_t* count, h3b_stream_t stream) {
  if (batch < 0 || n < 0 || kv_heads <= 0 || kv_heads > 65535 || batch > 32767 || n > (1ll << 30) ||
      (head_dim != 64 && head_dim != 128) || !block_ok(block_tokens) || num_blocks <= 0 || max_blocks <= 0 ||
      num_blocks * kv_heads > 0x7fffffffll || max_blocks * block_tokens > (1ll << 30))
    return H3B_ERR_SHAPE;
  if (x_dtype != H3B_BF16 && x_dtype != H3B_F16) return H3B_ERR_DTYPE;
  if (code_type != H3B_KV_INT8 && code_type != H3B_KV_E4M3) return H3B_ERR_DTYPE;
  if (batch == 0 || n == 0) return H3B_OK;
  if (!k || !v || !k_codes || !v_codes || !k_scale || !v_scale || !table || !start) return H3B_ERR_ARG;
  // (an axis of extent 1 may carry any stride)
  const int64_t strides[3] = {batch > 1 ? batch_stride : 0, n > 1 ? seq_stride : 0, kv_heads > 1 ? head_stride : 0};
  for (int64_t st : strides)
    if (st < 0 || st % 8 != 0) return H3B_ERR_ALIGN;
  for (const void* p : {k, v, static_cast<const void*>(k_codes), static_cast<const void*>(v_codes)})
    if (!h3b::aligned16(p)) return H3B_ERR_ALIGN;
  AppendArgs a{};
  a.src[0] = k, a.src[1] = v;
  for (int i = 0; i < 3; ++i) a.src_stride[i] = strides[i];
  a.codes[0] = k_codes, a.codes[1] = v_codes;
  a.scale[0] = k_scale, a.scale[1] = v_scale;
  a.table = table, a.start = start, a.count = count;
  a.n = static_cast<int>(n), a.kv_heads = static_cast<int>(kv_heads), a.max_blocks = static_cast<int>(max_blocks);
  a.num_blocks = static_cast<int>(num_blocks), a.block_tokens = static_cast<int>(block_tokens);
  // n rows touch at most ceil((n - 1) / block) + 1 blocks, wherever they start
  const dim3 grid(static_cast<unsigned>((n - 1 + block_tokens - 1) / block_tokens + 1),
                  static_cast<unsigned>(kv_heads), static_cast<unsigned>(2 * batch));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool f16 = x_dtype == H3B_F16, e4 = code_type == H3B_KV_E4M3;
#define H3B_APPEND(DD, FF, EE) kv8_append_kernel<DD, FF, EE><<<grid, THREADS, 0, st>>>(a)
  if (head_dim == 128) {
    if (f16) { if (e4) H3B_APPEND(128, true, true); else H3B_APPEND(128, true, false); }
    else { if (e4) H3B_APPEND(128, false, true); else H3B_APPEND(128, false, false); }
  } else {
    if (f16) { if (e4) H3B_APPEND(64, true, true); else H3B_APPEND(64, true, false); }
    else { if (e4) H3B_APPEND(64, false, true); else H3B_APPEND(64, false, false); }
  }
#undef H3B_APPEND
  return h3b::launch_status();
}

extern "C" int h3b_kv8_read(const uint8_t* k_codes, const uint8_t* v_codes, const float* k_scale, const float* v_scale,
                            int code_type, int64_t num_blocks, int64_t kv_heads, int64_t block_tokens,
                            int64_t head_dim, const int32_t* table, int64_t max_blocks, const int32_t* lens,
                            int64_t batch, int64_t max_len, void* k_out, void* v_out, int out_dtype,
                            h3b_stream_t stream) {
  if (batch < 0 || max_len < 0 || kv_heads <= 0 || (head_dim != 64 && head_dim != 128) || !block_ok(block_tokens) ||
      num_blocks <= 0 || max_blocks <= 0 || num_blocks * kv_heads > 0x7fffffffll || max_len > (1ll << 30) ||
      max_blocks * block_tokens > (1ll << 30))
    return H3B_ERR_SHAPE;
  if (code_type != H3B_KV_INT8 && code_type != H3B_KV_E4M3) return H3B_ERR_DTYPE;
  if (out_dtype != H3B_BF16 && out_dtype != H3B_F16 && out_dtype != H3B_F32) return H3B_ERR_DTYPE;
  if (batch == 0 || max_len == 0) return H3B_OK;
  if (!k_codes || !v_codes || !k_scale || !v_scale || !table || !lens || !k_out || !v_out) return H3B_ERR_ARG;
  for (const void* p : {static_cast<const void*>(k_codes), static_cast<const void*>(v_codes),
                        static_cast<const void*>(k_out), static_cast<const void*>(v_out)})
    if (!h3b::aligned16(p)) return H3B_ERR_ALIGN;
  ReadArgs a{};
  a.codes[0] = k_codes, a.codes[1] = v_codes;
  a.scale[0] = k_scale, a.scale[1] = v_scale;
  a.dst[0] = k_out, a.dst[1] = v_out;
  a.table = table, a.lens = lens;
  a.batch = static_cast<int>(batch), a.max_len = static_cast<int>(max_len), a.kv_heads = static_cast<int>(kv_heads);
  a.max_blocks = static_cast<int>(max_blocks), a.num_blocks = static_cast<int>(num_blocks);
  a.block_shift = shift_of(static_cast<int>(block_tokens));
  const int64_t rows = batch * max_len * kv_heads, per = THREADS / (head_dim / 16);
  if (rows > 0x7fffffffll) return H3B_ERR_SHAPE;
  const int64_t gx = (rows + per - 1) / per;
  const dim3 grid(static_cast<unsigned>(gx), 2);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool e4 = code_type == H3B_KV_E4M3;
#define H3B_READ(DD, EE)                                                                            \
  (out_dtype == H3B_BF16  ? kv8_read_kernel<DD, EE, 0><<<grid, THREADS, 0, st>>>(a)                 \
   : out_dtype == H3B_F16 ? kv8_read_kernel<DD, EE, 1><<<grid, THREADS, 0, st>>>(a)                 \
                          : kv8_read_kernel<DD, EE, 2><<<grid, THREADS, 0, st>>>(a))
  if (head_dim == 128) {
    if (e4) H3B_READ(128, true); else H3B_READ(128, false);
  } else {
    if (e4) H3B_READ(64, true); else H3B_READ(64, false);
  }
#undef H3B_READ
  return h3b::launch_status();
}
