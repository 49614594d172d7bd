// Attention of few query rows over many keys (h3b_cross_attention_fwd and
// h3b_kv8_attention when a key head serves few rows): one pass over K and V.
//
//   o_r = sum_j p_rj v_j,  p_rj = exp(scale q_r.k_j - lse_r) over the kept j
//
// with the running max M and sum l of a softmax per row, in fp32.  For the
// 8-bit cache k_j = sk K_j and v_j = sv V_j with one sk, sv per block of
// tokens and head: sk goes into the factor of the score, and sv into its
// exponent: w_j = 2^(x_j + log2 sv - M) is what multiplies the codes V_j, and l
// += w_j / sv.  M lies 14 below the running maximum where the weights are f16 (any
// call over the cache, bf16 queries too): w is at most 2^14, and a weight keeps
// its bits down to 2^-28 of the largest.  (At most 1, those below 2^-25 were 0 in
// the product but not in l, which a long tail beside one large key makes visible.)  The codes themselves go
// into the matrix instructions, exactly (|int8| <= 128 and every e4m3 value
// are f16 numbers), so nothing is rounded between the cache and the product.
//
// The work has to move the bytes of K and V.  A CTA is one range of keys x one
// key head x 16 or 32 query rows (tokens x the heads that share the key
// head).  Its 4 warps take the range's tiles in turn and never meet before
// the end: each has its own ring of TMA tiles (16 KB at 16 rows, so that three
// CTAs fit an SM; 24 KB at 32) and its own running softmax, and the four join
// through shared memory at the end.  A tile is 32 keys of the cache or 16 keys
// of a dense tensor.  m16n8k16 matrix instructions do both products: 16 rows
// fill one, and the conversion of the codes is shared by all rows of the CTA.
// (tcgen05 needs 128 rows per instruction; few-row calls have 1 to 32.)
// What bounds it over a long cache is issue slots, about half of them taken in
// every cycle by the conversion and the softmax: 131072 tokens x 24 heads of
// 128 e4m3 145 us (5.6 TB/s), int8, whose conversion is longer, 161 (5.0 TB/s).
//
// Lane layout of the codes.  The contraction order of a product is free as
// long as both operands use it, so K is read 16 bytes at a time: lane (g, t)
// (g = lane / 4, t = lane % 4) holds row key(g), bytes [16 t, 16 t + 16) of
// each 64 (D = 128: and 64 + the same), and q is loaded in the same order.  V
// is read by rows too: lane (g, t) reads D/8 bytes at d = g D/8 of the four
// keys of its k slots and interleaves them by byte permutes.  perm() maps the
// column n of a score tile to the key row so that both reads touch each bank
// once under the TMA swizzle.
#include <type_traits>

#include "h3b_common.cuh"
#include "h3b_host.hpp"
#include "xattn.hpp"

H3B_DECLARE_STATUS();
H3B_REGISTER_STATUS_READER(xattn_rows);

namespace {

using h3b::KV_DENSE;
using h3b::KV_E4M3;
using h3b::KV_INT8;
using h3b::KV8_SCALE_MIN;
using h3b::KvKind;
using h3b::XAttn;

constexpr int WARPS = 4;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.69314718055994531f;

template <int D, KvKind KIND, int MT>
struct Tile {
  static constexpr int RING_BYTES = (MT == 1 ? 16 : 24) * 1024;  // per warp
  static constexpr int KEYS = KIND == KV_DENSE ? 16 : 32;
  static constexpr int ELT = KIND == KV_DENSE ? 2 : 1;
  static constexpr int ROW = D * ELT < 128 ? D * ELT : 128;  // bytes of a row inside one TMA box
  static constexpr int BOXES = D * ELT / ROW;                // 2 for 16-bit, D = 128
  static constexpr int BOX_BYTES = KEYS * ROW;
  static constexpr int BYTES = KEYS * D * ELT;  // K (V follows)
  static constexpr int STAGES = RING_BYTES / (2 * BYTES);
};

struct RowsArgs {
  XAttn a;
  int row_tiles;
  int group;      // heads / kv_heads
  int rows;       // s_q * group
};

H3B_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool F16>
H3B_DEV void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

H3B_DEV void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
H3B_DEV void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
H3B_DEV uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
H3B_DEV uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

// Two codes -> f16x2.  int8 (bytes biased by 128 by the caller): 0x6400 | u is
// 1024 + u in f16, minus 1152 leaves u - 128.
H3B_DEV uint32_t i8_pair(uint32_t biased, uint32_t sel) {
  const uint32_t u = __byte_perm(biased, 0x64646464u, sel);
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&v);
}
H3B_DEV uint32_t e4m3_pair(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo;\n\tcvt.u16.u32 lo, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
// Four codes of one register -> f16x2 of bytes (0, 1) and (2, 3).
template <KvKind KIND>
H3B_DEV void codes4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (KIND == KV_INT8) {
    w ^= 0x80808080u;
    lo = i8_pair(w, 0x5140);
    hi = i8_pair(w, 0x5342);
  } else {
    lo = e4m3_pair(w);
    hi = e4m3_pair(w >> 16);
  }
}

// Column n of a score tile of 8 -> key row of the tile's 8 rows.  D = 128
// (rows of 128 bytes, 16-byte chunk c stored at c ^ (row & 7)): rows of
// columns 2i and 2i+1 differ by 4, rows of even columns differ in row >> 1.
// D = 64 (rows of 64 bytes, chunk c at c ^ ((row >> 1) & 3)): rows of columns
// 2i and 2i+1 differ in bit 0, rows of even columns in (bit 0, bit 2).
template <int D>
H3B_DEV int perm(int n) {
  return static_cast<int>(((D == 128 ? 0x37156240u : 0x65742130u) >> (4 * n)) & 7u);
}
// Byte offset of 16-byte chunk c of row r of a code tile.
template <int D>
H3B_DEV uint32_t code_off(int r, int c) {
  return D == 128 ? static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4))
                  : static_cast<uint32_t>(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

template <int D, KvKind KIND, bool QF16, int MT>
__global__ void __launch_bounds__(WARPS * 32, MT == 1 ? 3 : 2)
    xattn_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ RowsArgs args) {
  using T = Tile<D, KIND, MT>;
  constexpr bool CODES = KIND != KV_DENSE;
  constexpr bool F16 = CODES || QF16;  // operand type of the matrix instructions
  constexpr float UP = F16 ? 14.0f : 0.0f;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + WARPS * T::RING_BYTES);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + WARPS * T::STAGES);
  float2* s_ml = reinterpret_cast<float2*>(bars + WARPS * T::STAGES + 2);  // [WARPS][16 MT]

  const XAttn& a = args.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  int bx = blockIdx.x;
  const int split = bx % a.splits;
  bx /= a.splits;
  const int row_tile = bx % args.row_tiles;
  bx /= args.row_tiles;
  const int kvh = bx % a.kv_heads;
  const int b = bx / a.kv_heads;

  if (threadIdx.x == 0) {
    for (int i = 0; i < WARPS * T::STAGES; ++i) mbar_init(&bars[i], 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();

  int len = a.s_kv;
  if (a.kv_lens != nullptr) len = max(0, min(len, a.kv_lens[b]));
  // This split's range of keys: the sample's own length in equal parts of
  // whole tiles, so that every split has work whatever the longest sample is.
  const int n_tiles = (len + T::KEYS - 1) / T::KEYS;
  const int per = (n_tiles + a.splits - 1) / a.splits;
  const int tile0 = split * per, tile1 = min(n_tiles, tile0 + per);
  const int mine = tile1 - tile0 > warp ? (tile1 - tile0 - warp + WARPS - 1) / WARPS : 0;  // tiles of this warp

  uint8_t* ring = smem + warp * T::RING_BYTES;
  uint64_t* full = bars + warp * T::STAGES;
  // Cache: the block of a tile, -1 if the table has none (its keys are left out).
  auto block_of = [&](int tile) -> int {
    const int id = a.table[static_cast<int64_t>(b) * a.max_blocks + tile * T::KEYS / a.block_tokens];
    return id >= 0 && id < a.num_blocks ? id : -1;
  };
  auto issue = [&](int i) {  // lane 0: load the warp's i-th tile
    const int tile = tile0 + warp + i * WARPS;
    const int s = i % T::STAGES;
    uint8_t* dst = ring + s * 2 * T::BYTES;
    mbar_arrive_expect_tx(&full[s], 2 * T::BYTES);
    if constexpr (CODES) {
      // an absent block loads block 0 (it may hold anything: masked below)
      const int id = max(block_of(tile), 0);
      const int row = (tile * T::KEYS) % a.block_tokens;
      tma_load_3d(dst, &tm_k, 0, row, id * a.kv_heads + kvh, &full[s]);
      tma_load_3d(dst + T::BYTES, &tm_v, 0, row, id * a.kv_heads + kvh, &full[s]);
    } else {
#pragma unroll
      for (int x = 0; x < T::BOXES; ++x) {
        tma_load_4d(dst + x * T::BOX_BYTES, &tm_k, x * 64, tile * T::KEYS, kvh, b, &full[s]);
        tma_load_4d(dst + T::BYTES + x * T::BOX_BYTES, &tm_v, x * 64, tile * T::KEYS, kvh, b, &full[s]);
      }
    }
  };
  int issued = 0;
  if (lane == 0) {
    for (; issued < min(mine, T::STAGES); ++issued) issue(issued);
  }

  // ---- q fragments, row factors, causal limits
  uint32_t qa[MT][D / 16][4];
  float mult[MT][2];  // score -> log2 domain
  int limit[MT][2];   // keys a row sees
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = row_tile * 16 * MT + m * 16 + hf * 8 + g;
      const int tok = r / args.group, head = kvh * args.group + r % args.group;
      const bool in = r < args.rows;
      limit[m][hf] = !in ? 0 : a.causal ? len - a.s_q + tok + 1 : len;
      const uint32_t* qrow = reinterpret_cast<const uint32_t*>(
          static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + tok * a.q_stride[1] + head * a.q_stride[2]);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          // codes: chunk t (+4 for the second half of the steps), bytes 4 (kk % 4) + 2 p
          const int d = CODES ? 16 * (t + 4 * (kk >> 2)) + 4 * (kk & 3) + 2 * p : 16 * kk + 2 * t + 8 * p;
          qa[m][kk][hf + 2 * p] = in ? __ldg(qrow + d / 2) : 0u;
        }
      float e = 1.0f;
      if constexpr (CODES && !QF16) {
        // bf16 q in f16 products: a power of two brings the row's largest
        // value into [1, 2); 8 significant bits then fit f16 exactly down to
        // 2^-17 of it, and what is smaller is off by 2^-25 of it at most.
        float mx = 0.0f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const uint32_t w = qa[m][kk][hf + 2 * p];
            mx = fmaxf(mx, fmaxf(fabsf(bf16lo_to_f32(w)), fabsf(bf16hi_to_f32(w))));
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const int ex = min(max(static_cast<int>(__float_as_uint(mx) >> 23), 1), 253);  // biased exponent
        const float inv = __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
        e = __uint_as_float(static_cast<uint32_t>(ex) << 23);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const uint32_t w = qa[m][kk][hf + 2 * p];
            qa[m][kk][hf + 2 * p] = pack_f16x2(bf16lo_to_f32(w) * inv, bf16hi_to_f32(w) * inv);
          }
      }
      mult[m][hf] = a.scale * LOG2E * e;
    }
  }

  // Keys that every row of the CTA sees (rows past the last one are never stored).
  const int full_to = a.causal ? len - a.s_q + (row_tile * 16 * MT) / args.group + 1 : len;

  float acc[MT][D / 8][4];
  float M[MT][2], L[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    M[m][0] = M[m][1] = -INFINITY;
    L[m][0] = L[m][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][i][e] = 0.0f;
  }

  // What a tile needs beside its rows is fetched ahead: the block two tiles,
  // its scales (or its mask bytes) one tile before they are used.
  auto fetch_block = [&](int i) -> int { return CODES && i < mine ? block_of(tile0 + warp + i * WARPS) : -1; };
  auto fetch_scale = [&](const float* p, int id) -> float {
    return CODES && id >= 0 ? __ldg(p + static_cast<int64_t>(id) * a.kv_heads + kvh) : 1.0f;
  };
  auto fetch_mask = [&](int i) -> bool {
    const int key = (tile0 + warp + i * WARPS) * T::KEYS + (lane & 15);
    return i < mine && key < len && a.key_mask[b * a.mask_stride + key] != 0;
  };
  const bool masked = !CODES && a.key_mask != nullptr;
  int id0 = fetch_block(0), id1 = fetch_block(1);
  float sk0 = fetch_scale(a.k_scale, id0), sv0 = fetch_scale(a.v_scale, id0);
  bool mask0 = masked ? fetch_mask(0) : true;

  bool ok = true;
  for (int i = 0; i < mine; ++i) {
    const int tile = tile0 + warp + i * WARPS;
    const int s = i % T::STAGES;
    const int key0 = tile * T::KEYS;
    // kept keys of the tile, one bit each
    uint32_t keep = len - key0 >= 32 ? 0xffffffffu : (1u << (len - key0)) - 1u;
    if constexpr (T::KEYS == 16) keep &= 0xffffu;
    const float sk = sk0, sv = sv0;
    if constexpr (CODES) {
      if (id0 < 0) keep = 0;
      id0 = id1;
      id1 = fetch_block(i + 2);
      sk0 = fetch_scale(a.k_scale, id0);
      sv0 = fetch_scale(a.v_scale, id0);
    } else if (masked) {
      keep &= __ballot_sync(0xffffffffu, mask0);
      mask0 = fetch_mask(i + 1);
    }
    // One parity bit per use of the slot: the next use is issued only after
    // the __syncwarp below, so the wait is never more than a phase behind.
    if (!__all_sync(0xffffffffu, mbar_wait(&full[s], (i / T::STAGES) & 1, &g_status, 1, abort_flag))) {
      ok = false;
      break;
    }
    const uint32_t k_s = smem_u32(ring + s * 2 * T::BYTES);
    const uint32_t v_s = k_s + T::BYTES;
    const uint32_t all = T::KEYS == 32 ? 0xffffffffu : 0xffffu;
    if (keep != all) {
      // A left-out value may be anything, NaN included, and 0 * NaN is NaN:
      // its row is zeroed before the product reads it.
      for (int c = lane; c < T::KEYS * D * T::ELT / 16; c += 32) {
        const int r = (c * 16 % T::BOX_BYTES) / T::ROW;
        if (((keep >> r) & 1u) == 0)
          asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(v_s + c * 16), "r"(0u) : "memory");
      }
      __syncwarp();
    }

    // ---- scores of 8-key column tiles
    constexpr int NT = T::KEYS / 8;
    float sc[MT][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[m][n][e] = 0.0f;
      if constexpr (CODES) {
        const int r = 8 * n + perm<D>(g);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const uint4 w = lds128(k_s + code_off<D>(r, t + 4 * c));
          const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t b0, b1;
            codes4<KIND>(ws[j], b0, b1);
#pragma unroll
            for (int m = 0; m < MT; ++m) mma16816<F16>(sc[m][n], qa[m][4 * c + j], b0, b1);
          }
        }
      } else {
        // matrices: 8 keys x 8 d, four consecutive d groups
        const int r = 8 * n + (lane & 7);
#pragma unroll
        for (int kk = 0; kk < D / 16; kk += 2) {
          uint32_t w[4];
          const int c = 2 * kk + (lane >> 3);  // 16-byte chunk of the row
          ldsm_x4(k_s + (c >> 3) * T::BOX_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4), w);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma16816<F16>(sc[m][n], qa[m][kk], w[0], w[1]);
            mma16816<F16>(sc[m][n], qa[m][kk + 1], w[2], w[3]);
          }
        }
      }
    }

    // ---- running softmax; x = score * mult * sk + log2 sv
    const float lsv = CODES ? __log2f(fmaxf(sv, KV8_SCALE_MIN)) : 0.0f;
    const float inv_sv = CODES ? 1.0f / fmaxf(sv, KV8_SCALE_MIN) : 1.0f;
    if (keep != all || key0 + T::KEYS > full_to) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int col = 2 * t + (e & 1);
            const int key = 8 * n + (CODES ? perm<D>(col) : col);
            if (((keep >> key) & 1u) == 0 || key0 + key >= limit[m][e >> 1]) sc[m][n][e] = -INFINITY;
          }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float f[2], off[2], corr[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        float top = fmaxf(sc[m][0][2 * hf], sc[m][0][2 * hf + 1]);
#pragma unroll
        for (int n = 1; n < NT; ++n) top = fmax3(top, sc[m][n][2 * hf], sc[m][n][2 * hf + 1]);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // (a factor of 0 would make NaN of -inf: a row of zeros has e = 2^-126, zero keys sk = 1e-14)
        f[hf] = CODES ? fmaxf(mult[m][hf] * sk, 1e-37f) : mult[m][hf];
        const float mn = fmaxf(M[m][hf], fmaf(top, f[hf], lsv - UP));
        const float base = mn == -INFINITY ? 0.0f : mn;  // nothing kept so far: every weight is 2^-inf = 0
        corr[hf] = ex2(M[m][hf] - base);
        off[hf] = lsv - base;
        M[m][hf] = mn;
      }
      if (__any_sync(0xffffffffu, corr[0] != 1.0f || corr[1] != 1.0f)) {
#pragma unroll
        for (int i2 = 0; i2 < D / 8; ++i2) {
          acc[m][i2][0] *= corr[0];
          acc[m][i2][1] *= corr[0];
          acc[m][i2][2] *= corr[1];
          acc[m][i2][3] *= corr[1];
        }
      }
      float sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float w = ex2(fmaf(sc[m][n][e], f[e >> 1], off[e >> 1]));
          sc[m][n][e] = w;
          sum[e >> 1] += w;
        }
      L[m][0] = fmaf(sum[0], inv_sv, L[m][0] * corr[0]);
      L[m][1] = fmaf(sum[1], inv_sv, L[m][1] * corr[1]);
    }

    // ---- o += w v, 16 keys at a time
#pragma unroll
    for (int h = 0; h < T::KEYS / 16; ++h) {
      uint32_t pa[MT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // a0: row g, columns 2t, 2t+1 of key tile 2h; a1: row g+8; a2, a3: key tile 2h+1
          const float lo = sc[m][2 * h + (j >> 1)][2 * (j & 1)], hi = sc[m][2 * h + (j >> 1)][2 * (j & 1) + 1];
          pa[m][j] = F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
        }
      if constexpr (CODES) {
        constexpr int W = D / 32;  // words of a row piece (D / 8 codes)
        uint32_t w[4][W];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 16 * h + 8 * (j >> 1) + perm<D>(2 * t + (j & 1));
          if constexpr (W == 4) {
            const uint4 x = lds128(v_s + code_off<D>(r, g));
            w[j][0] = x.x, w[j][1] = x.y, w[j][2] = x.z, w[j][3] = x.w;
          } else {
            const uint2 x = lds64(v_s + code_off<D>(r, g >> 1) + (g & 1) * 8);
            w[j][0] = x.x, w[j][1] = x.y;
          }
        }
#pragma unroll
        for (int x = 0; x < W; ++x) {
          // bytes (key 2t, key 2t+1) and (2t+8, 2t+9) of d = g D/8 + 4 x + (0..3)
          const uint32_t lo01 = __byte_perm(w[0][x], w[1][x], 0x5140), lo23 = __byte_perm(w[0][x], w[1][x], 0x7362);
          const uint32_t hi01 = __byte_perm(w[2][x], w[3][x], 0x5140), hi23 = __byte_perm(w[2][x], w[3][x], 0x7362);
          uint32_t b0[4], b1[4];
          codes4<KIND>(lo01, b0[0], b0[1]);
          codes4<KIND>(lo23, b0[2], b0[3]);
          codes4<KIND>(hi01, b1[0], b1[1]);
          codes4<KIND>(hi23, b1[2], b1[3]);
#pragma unroll
          for (int y = 0; y < 4; ++y)
#pragma unroll
            for (int m = 0; m < MT; ++m) mma16816<F16>(acc[m][4 * x + y], pa[m], b0[y], b1[y]);
        }
      } else {
        // matrices: (keys 0-7, keys 8-15) x (d group i, d group i + 1)
        const int r = 16 * h + (lane & 15);
#pragma unroll
        for (int i2 = 0; i2 < D / 8; i2 += 2) {
          uint32_t w[4];
          const int c = i2 + (lane >> 4);
          ldsm_x4_trans(v_s + (c >> 3) * T::BOX_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4), w);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma16816<F16>(acc[m][i2], pa[m], w[0], w[1]);
            mma16816<F16>(acc[m][i2 + 1], pa[m], w[2], w[3]);
          }
        }
      }
    }
    if (keep != all) fence_proxy_async_smem();  // the zeroed rows, before the slot's next copy
    __syncwarp();                               // every lane has read the slot
    if (lane == 0 && issued < mine) issue(issued++);
  }
  if (!ok && lane == 0) {
    // let the copies in flight land (bounded) before the CTA goes
    for (int i = max(0, issued - T::STAGES); i < issued; ++i)
      mbar_wait(&full[i % T::STAGES], (i / T::STAGES) & 1, &g_status, 2, nullptr);
  }

  // ---- the four warps' results, joined
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      L[m][hf] += __shfl_xor_sync(0xffffffffu, L[m][hf], 1);
      L[m][hf] += __shfl_xor_sync(0xffffffffu, L[m][hf], 2);
      if (t == 0) s_ml[warp * 16 * MT + m * 16 + hf * 8 + g] = make_float2(M[m][hf], L[m][hf]);
    }
  __syncthreads();  // rings are free: every warp has read its last tile
  constexpr int PAD = D + 4;
  float* s_o = reinterpret_cast<float*>(smem);  // [WARPS][16 MT][PAD]
  static_assert(WARPS * 16 * MT * PAD * 4 <= WARPS * T::RING_BYTES, "join buffer");
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = 2 * t + (e & 1);
        const int d = CODES ? n * (D / 8) + i : 8 * i + n;
        s_o[(warp * 16 * MT + m * 16 + (e >> 1) * 8 + g) * PAD + d] = acc[m][i][e];
      }
  __syncthreads();
  if (*abort_flag) return;
  const int64_t total_rows = static_cast<int64_t>(a.batch) * a.heads * a.s_q;
  for (int x = threadIdx.x; x < 16 * MT * (D / 4); x += WARPS * 32) {
    const int r16 = x / (D / 4), d = (x % (D / 4)) * 4;
    const int r = row_tile * 16 * MT + r16;
    if (r >= args.rows) continue;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, s_ml[w * 16 * MT + r16].x);
    const float base = mx == -INFINITY ? 0.0f : mx;
    float l = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float2 ml = s_ml[w * 16 * MT + r16];
      const float f = ex2(ml.x - base);
      const float4 v = *reinterpret_cast<const float4*>(&s_o[(w * 16 * MT + r16) * PAD + d]);
      l = fmaf(ml.y, f, l);
      o.x = fmaf(v.x, f, o.x);
      o.y = fmaf(v.y, f, o.y);
      o.z = fmaf(v.z, f, o.z);
      o.w = fmaf(v.w, f, o.w);
    }
    const int tok = r / args.group, head = kvh * args.group + r % args.group;
    const int64_t row = (static_cast<int64_t>(b) * a.heads + head) * a.s_q + tok;
    if (a.splits > 1) {
      *reinterpret_cast<float4*>(a.part_o + (split * total_rows + row) * D + d) = o;
      if (d == 0) a.part_ml[split * total_rows + row] = make_float2(mx, l);
    } else {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (0: no key; a NaN stays one)
      uint2 w;
      if (a.dtype == H3B_F16) {
        w = make_uint2(pack_f16x2(o.x * inv, o.y * inv), pack_f16x2(o.z * inv, o.w * inv));
      } else {
        w = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
      }
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + b * a.o_stride[0] + tok * a.o_stride[1] +
                                head * a.o_stride[2] + d) = w;
      if (d == 0 && a.lse != nullptr) a.lse[row] = l == 0.0f ? -INFINITY : (mx + __log2f(l)) * LN2;
    }
  }
}

// Joins the split ranges of each row: o = sum_i 2^(M_i - M) o_i / sum_i
// 2^(M_i - M) l_i.  One warp per row, D/32 values per lane; the sums run in
// the order of the ranges.  Eight ranges' values are under way at a time, the
// first eight before the maxima arrive (1560 x 24 rows of 6 ranges: 36 us with
// the maxima first, 28 so; 4.5 TB/s, much of it from L2).  (Row numbers have 32 bits: 2^31 rows
// of two ranges would be a workspace of 1 TB.)
template <int D>
__global__ void __launch_bounds__(128) xattn_combine_kernel(const __grid_constant__ XAttn a) {
  constexpr int E = D / 32, DEEP = 8;
  using Vec = typename std::conditional<E == 4, float4, float2>::type;
  const uint32_t total = static_cast<uint32_t>(a.batch) * a.heads * a.s_q;
  const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= total) return;
  const int lane = threadIdx.x & 31;
  const Vec* src = reinterpret_cast<const Vec*>(a.part_o + static_cast<int64_t>(row) * D) + lane;
  const int64_t step = static_cast<int64_t>(total) * 32;  // (Vecs from range to range)
  Vec v[DEEP];
#pragma unroll
  for (int k = 0; k < DEEP; ++k)
    if (k < a.splits) v[k] = src[k * step];
  float2 ml = lane < a.splits ? a.part_ml[static_cast<int64_t>(lane) * total + row] : make_float2(-INFINITY, 0.0f);
  float mx = ml.x;
  for (int i = lane + 32; i < a.splits; i += 32) mx = fmaxf(mx, a.part_ml[static_cast<int64_t>(i) * total + row].x);
  mx = warp_max(mx);
  const float base = mx == -INFINITY ? 0.0f : mx;
  float l = 0.0f;
  float o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
  for (int i = 0; i < a.splits; i += DEEP) {
    if (i > 0) {
#pragma unroll
      for (int k = 0; k < DEEP; ++k)
        if (i + k < a.splits) v[k] = src[(i + k) * step];
      if ((i & 31) == 0)
        ml = i + lane < a.splits ? a.part_ml[static_cast<int64_t>(i + lane) * total + row] : make_float2(-INFINITY, 0.0f);
    }
    const float w = ex2(ml.x - base);
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
      if (i + k < a.splits) {
        const float f = __shfl_sync(0xffffffffu, w, (i + k) & 31);
        l = fmaf(__shfl_sync(0xffffffffu, ml.y, (i + k) & 31), f, l);
        const float x[4] = {v[k].x, v[k].y, E == 4 ? reinterpret_cast<const float*>(&v[k])[E - 2] : 0.0f,
                            E == 4 ? reinterpret_cast<const float*>(&v[k])[E - 1] : 0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(x[e], f, o[e]);
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (0: no key; a NaN stays one)
  const uint32_t bh = row / static_cast<uint32_t>(a.s_q);
  const int64_t tok = row - bh * a.s_q, b = bh / static_cast<uint32_t>(a.heads);
  const int64_t head = bh - static_cast<uint32_t>(b) * a.heads;
  uint16_t* dst = static_cast<uint16_t*>(a.o) + b * a.o_stride[0] + tok * a.o_stride[1] + head * a.o_stride[2] + lane * E;
  uint32_t w[E / 2];
#pragma unroll
  for (int e = 0; e < E; e += 2)
    w[e / 2] = a.dtype == H3B_F16 ? pack_f16x2(o[e] * inv, o[e + 1] * inv) : pack_bf16x2(o[e] * inv, o[e + 1] * inv);
  if constexpr (E == 4) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  } else {
    *reinterpret_cast<uint32_t*>(dst) = w[0];
  }
  if (lane == 0 && a.lse != nullptr) a.lse[row] = l == 0.0f ? -INFINITY : (mx + __log2f(l)) * LN2;
}

template <int D, KvKind KIND, bool QF16, int MT>
int launch(const XAttn& a, cudaStream_t stream) {
  using T = Tile<D, KIND, MT>;
  CUtensorMap tk, tv;
  int rc;
  if constexpr (KIND == KV_DENSE) {
    const uint64_t dims[4] = {D, static_cast<uint64_t>(a.s_kv > 0 ? a.s_kv : 1), static_cast<uint64_t>(a.kv_heads),
                              static_cast<uint64_t>(a.batch)};
    const uint64_t st[3] = {static_cast<uint64_t>(a.kv_stride[1]) * 2, static_cast<uint64_t>(a.kv_stride[2]) * 2,
                            static_cast<uint64_t>(a.kv_stride[0]) * 2};
    const uint32_t box[4] = {64, T::KEYS, 1, 1};
    const CUtensorMapDataType dt = QF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    rc = h3b::encode_4d(&tk, dt, a.k, dims, st, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc == H3B_OK) rc = h3b::encode_4d(&tv, dt, a.v, dims, st, box, CU_TENSOR_MAP_SWIZZLE_128B);
  } else {
    const uint64_t slabs = static_cast<uint64_t>(a.num_blocks) * a.kv_heads;
    const uint64_t slab = static_cast<uint64_t>(a.block_tokens) * D;
    constexpr CUtensorMapSwizzle sw = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    rc = h3b::encode_3d(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.k, D, a.block_tokens, slabs, D, slab, D, T::KEYS, 1, sw);
    if (rc == H3B_OK)
      rc = h3b::encode_3d(&tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.v, D, a.block_tokens, slabs, D, slab, D, T::KEYS, 1, sw);
  }
  if (rc != H3B_OK) return rc;
  constexpr size_t smem = 1024 + WARPS * T::RING_BYTES + (WARPS * T::STAGES + 2) * 8 + WARPS * 16 * MT * sizeof(float2);
  auto kernel = xattn_rows_kernel<D, KIND, QF16, MT>;
  static h3b::OncePerDevice attr;
  rc = attr.run(h3b::device(), [=] { return h3b::allow_smem(kernel, smem); });
  if (rc != H3B_OK) return rc;
  RowsArgs args{};
  args.a = a;
  args.group = a.heads / a.kv_heads;
  args.rows = a.s_q * args.group;
  args.row_tiles = (args.rows + 16 * MT - 1) / (16 * MT);
  const int64_t grid = static_cast<int64_t>(a.splits) * args.row_tiles * a.kv_heads * a.batch;
  if (grid > 0x7fffffff) return H3B_ERR_SHAPE;
  kernel<<<static_cast<unsigned>(grid), WARPS * 32, smem, stream>>>(tk, tv, args);
  return h3b::launch_status();
}

template <int D, KvKind KIND, bool QF16>
int launch_mt(const XAttn& a, cudaStream_t stream) {
  return static_cast<int64_t>(a.s_q) * (a.heads / a.kv_heads) <= 16 ? launch<D, KIND, QF16, 1>(a, stream)
                                                                    : launch<D, KIND, QF16, 2>(a, stream);
}

template <int D, KvKind KIND>
int launch_dt(const XAttn& a, cudaStream_t stream) {
  return a.dtype == H3B_F16 ? launch_mt<D, KIND, true>(a, stream) : launch_mt<D, KIND, false>(a, stream);
}

template <int D>
int launch_kind(const XAttn& a, cudaStream_t stream) {
  switch (a.kind) {
    case KV_INT8: return launch_dt<D, KV_INT8>(a, stream);
    case KV_E4M3: return launch_dt<D, KV_E4M3>(a, stream);
    default: return launch_dt<D, KV_DENSE>(a, stream);
  }
}

}  // namespace

namespace h3b {

int xattn_rows_splits(const XAttn& a) {
  const int64_t rows = static_cast<int64_t>(a.s_q) * (a.heads / a.kv_heads);
  const int64_t ctas = (rows <= 16 ? 1 : (rows + 31) / 32) * a.kv_heads * a.batch;
  // Rounds of CTAs (two or three fit an SM) times the steps of one (its four
  // warps' tiles), its own start and end counted as two steps.  131072 int8
  // keys x 24 heads: 18 splits (one round) 179 us, 37 (two) 183, 74 (four)
  // 202; 32 x 16384 e4m3 keys x 8 heads: 1 split 253, 3 231, 6 220.
  const int64_t slots = static_cast<int64_t>(num_sms()) * (rows <= 16 ? 3 : 2);
  const int64_t keys = WARPS * (a.kind == KV_DENSE ? 16 : 32);
  const int64_t steps = (static_cast<int64_t>(a.s_kv) + keys - 1) / keys;
  int best = 1;
  int64_t cost = INT64_MAX;
  for (int64_t s = 1; s <= 128 && (s == 1 || s <= steps); ++s) {
    // (joining splits is a second launch: 2 us on the host, 4 on the GPU, or
    // about eight steps)
    const int64_t c = ((ctas * s + slots - 1) / slots) * ((steps + s - 1) / s + 2) + (s > 1 ? 8 : 0);
    if (c < cost) {
      cost = c;
      best = static_cast<int>(s);
    }
  }
  return best;
}

int xattn_rows_launch(const XAttn& a, cudaStream_t stream) {
  const int rc = a.head_dim == 128 ? launch_kind<128>(a, stream) : launch_kind<64>(a, stream);
  return rc != H3B_OK || a.splits == 1 ? rc : xattn_combine_launch(a, stream);
}

int xattn_combine_launch(const XAttn& a, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.batch) * a.heads * a.s_q;
  if (rows > 0x7fffffff) return H3B_ERR_SHAPE;
  const int64_t grid = (rows + 3) / 4;
  if (a.head_dim == 128) {
    xattn_combine_kernel<128><<<static_cast<unsigned>(grid), 128, 0, stream>>>(a);
  } else {
    xattn_combine_kernel<64><<<static_cast<unsigned>(grid), 128, 0, stream>>>(a);
  }
  return launch_status();
}

}  // namespace h3b
