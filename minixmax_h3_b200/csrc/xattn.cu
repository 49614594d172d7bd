// Entry points of cross attention and of attention over the 8-bit cache:
// argument checks, the choice of kernel and of splits, workspace sizes.
#include "h3b_host.hpp"
#include "xattn.hpp"

namespace {

using h3b::XAttn;

// A tensor of extent 1 along an axis may carry any stride there.
bool fix_strides(int64_t (&st)[3], int64_t batch, int64_t seq, int64_t heads, int64_t d) {
  const int64_t ext[3] = {batch, seq, heads};
  for (int i = 0; i < 3; ++i) {
    if (ext[i] <= 1) st[i] = d;
    if (st[i] <= 0 || st[i] % 8 != 0 || st[i] > (1ll << 38)) return false;
  }
  return true;
}

int check_sizes(int dtype, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t s_q,
                int64_t s_kv) {
  if (dtype != H3B_BF16 && dtype != H3B_F16) return H3B_ERR_DTYPE;
  if (batch < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || s_q < 0 || s_kv < 0 ||
      (head_dim != 64 && head_dim != 128) || batch > 65535 || heads > 65535 || s_q > (1ll << 30) ||
      s_kv > (1ll << 30) || s_q * (heads / kv_heads) > (1ll << 30) || batch * heads * s_q > (1ll << 40))
    return H3B_ERR_SHAPE;
  return H3B_OK;
}

int64_t rows_of(const XAttn& a) { return static_cast<int64_t>(a.batch) * a.heads * a.s_q; }

// Which kernel: the tile kernel works on 128 rows of one head whether they
// exist or not, the row kernel on 16 or 32 rows of the heads that share a key
// head.  GPU us, tiles / rows, at 32 and 48 tokens: 24 heads x 512 keys 10.7 /
// 14.9 and 11.1 / 14.9; 4 samples, 24 heads on 6, 2000 keys 33.8 / 26.1 and
// 34.0 / 32.7; 32768 int8 tokens x 24 heads 136 / 86 and 136 / 142; 4 x 4096, 32
// heads on 8 79 / 61 and 79 / 104.  Over at most 128 keys the row kernel's
// shorter start wins up to 128 tokens (2 samples, 8 heads of 64, 77 keys: 7.5 / 6.0).
bool by_tiles(const XAttn& a) { return a.s_q > 32 && (a.s_q > 128 || a.s_kv > 128); }

// The last call's splits are kept by its sizes: a model's layers repeat them,
// and the search is 2 us of divisions on calls of 10.
struct Sizes {
  int kind, batch, heads, kv_heads, head_dim, s_q, s_kv, sms;
  bool operator==(const Sizes& o) const {
    return kind == o.kind && batch == o.batch && heads == o.heads && kv_heads == o.kv_heads && head_dim == o.head_dim &&
           s_q == o.s_q && s_kv == o.s_kv && sms == o.sms;
  }
};
template <class A, class F>
int kept_splits(const A& a, int kind, Sizes& last, int& splits, F search) {
  const Sizes now{kind, a.batch, a.heads, a.kv_heads, a.head_dim, a.s_q, a.s_kv, h3b::num_sms()};
  if (splits == 0 || !(now == last)) {
    splits = search(a);
    last = now;
  }
  return splits;
}

void plan(XAttn& a) {
  static thread_local Sizes last{};
  static thread_local int splits = 0;
  a.splits = kept_splits(a, a.kind == h3b::KV_DENSE ? 0 : 1, last, splits, [](const XAttn& x) {
    return by_tiles(x) ? h3b::xattn_tile_splits(x) : h3b::xattn_rows_splits(x);
  });
}

// Whether a cache's codes are written out as 16-bit operands first; else each
// 256-row tile of each query head converts them anew.  32768 int8 tokens x 24
// heads, bf16, us with and without: 256 rows 212 / 167, 512 rows 294 / 306, 768
// rows 380 / 450, 1560 rows 798 / 1222.  At most 8 GB of workspace.
int64_t expand_bytes(const XAttn& a) {
  const int64_t times = static_cast<int64_t>(a.heads / a.kv_heads) * ((a.s_q + 255) / 256);
  if (a.kind == h3b::KV_DENSE || !by_tiles(a) || times < 2) return 0;
  const int64_t n = 2ll * a.batch * a.kv_heads * a.s_kv * a.head_dim * 2;
  return n <= (8ll << 30) ? n : 0;
}

int64_t part_bytes(const XAttn& a) {
  return a.splits > 1 ? rows_of(a) * a.splits * (a.head_dim + 2) * static_cast<int64_t>(sizeof(float)) : 0;
}

// Workspace: 16-bit operands of K and V, then the splits' partial rows.
int64_t workspace_of(const XAttn& a) { return expand_bytes(a) + part_bytes(a); }

int run(XAttn& a, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  plan(a);
  const int64_t need = workspace_of(a);
  if (need > 0) {
    if (workspace == nullptr) return H3B_ERR_ARG;
    if (workspace_bytes < need) return H3B_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(workspace) & 31u) != 0) return H3B_ERR_ALIGN;
    const int64_t pre = expand_bytes(a);
    if (pre > 0) {
      a.pre_k = workspace;
      a.pre_v = static_cast<uint8_t*>(workspace) + pre / 2;
    }
    a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + pre);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + rows_of(a) * a.splits * a.head_dim);
  }
  return by_tiles(a) ? h3b::xattn_tile_launch(a, stream) : h3b::xattn_rows_launch(a, stream);
}

XAttn sizes(int dtype, h3b::KvKind kind, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t s_q,
            int64_t s_kv) {
  XAttn a{};
  a.dtype = dtype;
  a.kind = kind;
  a.batch = static_cast<int>(batch);
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.head_dim = static_cast<int>(head_dim);
  a.s_q = static_cast<int>(s_q);
  a.s_kv = static_cast<int>(s_kv);
  a.splits = 1;
  return a;
}

}  // namespace

extern "C" int h3b_cross_attention_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                             int64_t s_q, int64_t s_kv, int64_t* bytes) {
  if (bytes == nullptr) return H3B_ERR_ARG;
  const int rc = check_sizes(H3B_BF16, batch, heads, kv_heads, head_dim, s_q, s_kv);
  if (rc != H3B_OK) return rc;
  XAttn a = sizes(H3B_BF16, h3b::KV_DENSE, batch, heads, kv_heads, head_dim, s_q, s_kv);
  plan(a);
  *bytes = workspace_of(a);
  return H3B_OK;
}

extern "C" int h3b_cross_attention_fwd(const void* q, const void* k, const void* v, void* o, float* lse, int dtype,
                                       int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t s_q,
                                       int64_t s_kv, int64_t q_batch_stride, int64_t q_seq_stride,
                                       int64_t q_head_stride, int64_t kv_batch_stride, int64_t kv_seq_stride,
                                       int64_t kv_head_stride, int64_t o_batch_stride, int64_t o_seq_stride,
                                       int64_t o_head_stride, const int32_t* kv_lens, const uint8_t* key_mask,
                                       int64_t mask_stride, float scale, void* workspace, int64_t workspace_bytes,
                                       h3b_stream_t stream) {
  const int rc = check_sizes(dtype, batch, heads, kv_heads, head_dim, s_q, s_kv);
  if (rc != H3B_OK) return rc;
  if (!(scale > 0.0f) || mask_stride < 0) return H3B_ERR_ARG;
  if (batch == 0 || s_q == 0) return H3B_OK;
  XAttn a = sizes(dtype, h3b::KV_DENSE, batch, heads, kv_heads, head_dim, s_q, s_kv);
  a.q = q, a.k = s_kv > 0 ? k : q, a.v = s_kv > 0 ? v : q, a.o = o, a.lse = lse;
  if (a.q == nullptr || a.k == nullptr || a.v == nullptr || o == nullptr) return H3B_ERR_ARG;
  a.q_stride[0] = q_batch_stride, a.q_stride[1] = q_seq_stride, a.q_stride[2] = q_head_stride;
  a.kv_stride[0] = kv_batch_stride, a.kv_stride[1] = kv_seq_stride, a.kv_stride[2] = kv_head_stride;
  a.o_stride[0] = o_batch_stride, a.o_stride[1] = o_seq_stride, a.o_stride[2] = o_head_stride;
  if (!fix_strides(a.q_stride, batch, s_q, heads, head_dim) ||
      !fix_strides(a.kv_stride, s_kv > 0 ? batch : 1, s_kv, s_kv > 0 ? kv_heads : 1, head_dim) ||
      !fix_strides(a.o_stride, batch, s_q, heads, head_dim))
    return H3B_ERR_ALIGN;
  for (const void* p : {a.q, a.k, a.v, static_cast<const void*>(o)})
    if (!h3b::aligned16(p)) return H3B_ERR_ALIGN;
  a.kv_lens = kv_lens;
  a.key_mask = s_kv > 0 ? key_mask : nullptr;
  a.mask_stride = mask_stride;
  a.scale = scale;
  return run(a, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

namespace {

// Workspace of a backward call: the ranges' sums (16-byte pieces), then delta,
// and the norms that f16 calls scale dS by (the query of the size does not say
// which type it is for).
int64_t grad_part_floats(const h3b::XAttnGrad& a) {
  return a.splits > 1 ? 2ll * a.splits * a.batch * a.s_kv * a.kv_heads * a.head_dim : 0;
}
int64_t grad_rows(const h3b::XAttnGrad& a) { return static_cast<int64_t>(a.batch) * a.heads * a.s_q; }
int64_t grad_workspace(const h3b::XAttnGrad& a) {
  return (grad_part_floats(a) + 2 * grad_rows(a) + 2ll * a.batch * a.kv_heads) *
         static_cast<int64_t>(sizeof(float));
}
h3b::XAttnGrad grad_sizes(int dtype, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t s_q,
                          int64_t s_kv) {
  h3b::XAttnGrad a{};
  a.dtype = dtype;
  a.batch = static_cast<int>(batch);
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.head_dim = static_cast<int>(head_dim);
  a.s_q = static_cast<int>(s_q);
  a.s_kv = static_cast<int>(s_kv);
  static thread_local Sizes last{};
  static thread_local int splits = 0;
  a.splits = kept_splits(a, 2, last, splits, h3b::xattn_bwd_splits);
  return a;
}

}  // namespace

extern "C" int h3b_cross_attention_bwd_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                 int64_t s_q, int64_t s_kv, int64_t* bytes) {
  if (bytes == nullptr) return H3B_ERR_ARG;
  const int rc = check_sizes(H3B_BF16, batch, heads, kv_heads, head_dim, s_q, s_kv);
  if (rc != H3B_OK) return rc;
  *bytes = grad_workspace(grad_sizes(H3B_BF16, batch, heads, kv_heads, head_dim, s_q, s_kv));
  return H3B_OK;
}

extern "C" int h3b_cross_attention_bwd(const void* d_o, const void* q, const void* k, const void* v, const void* o,
                                       const float* lse, void* dq, void* dk, void* dv, int dtype, int64_t batch,
                                       int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t s_q, int64_t s_kv,
                                       int64_t do_batch_stride, int64_t do_seq_stride, int64_t do_head_stride,
                                       int64_t q_batch_stride, int64_t q_seq_stride, int64_t q_head_stride,
                                       int64_t kv_batch_stride, int64_t kv_seq_stride, int64_t kv_head_stride,
                                       int64_t o_batch_stride, int64_t o_seq_stride, int64_t o_head_stride,
                                       const int32_t* kv_lens, const uint8_t* key_mask, int64_t mask_stride,
                                       float scale, void* workspace, int64_t workspace_bytes, h3b_stream_t stream) {
  const int rc = check_sizes(dtype, batch, heads, kv_heads, head_dim, s_q, s_kv);
  if (rc != H3B_OK) return rc;
  if (!(scale > 0.0f) || mask_stride < 0) return H3B_ERR_ARG;
  if (batch == 0) return H3B_OK;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (s_kv > 0 && (dk == nullptr || dv == nullptr)) return H3B_ERR_ARG;
  if (s_q == 0) {  // no query: the sums over queries are zero
    const size_t n = static_cast<size_t>(batch * s_kv * kv_heads * head_dim) * 2;
    if (n == 0) return H3B_OK;
    return cudaMemsetAsync(dk, 0, n, st) == cudaSuccess && cudaMemsetAsync(dv, 0, n, st) == cudaSuccess
               ? H3B_OK
               : H3B_ERR_LAUNCH;
  }
  if (batch * heads * s_q > 0x7fffffffll) return H3B_ERR_SHAPE;
  h3b::XAttnGrad a = grad_sizes(dtype, batch, heads, kv_heads, head_dim, s_q, s_kv);
  a.q = q, a.k = s_kv > 0 ? k : q, a.v = s_kv > 0 ? v : q, a.o = o, a.d_o = d_o, a.lse = lse;
  a.dq = dq, a.dk = dk, a.dv = dv;
  if (!a.q || !a.k || !a.v || !o || !d_o || !lse || !dq || !workspace) return H3B_ERR_ARG;
  const int64_t st4[4][3] = {{q_batch_stride, q_seq_stride, q_head_stride},
                             {kv_batch_stride, kv_seq_stride, kv_head_stride},
                             {o_batch_stride, o_seq_stride, o_head_stride},
                             {do_batch_stride, do_seq_stride, do_head_stride}};
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = st4[0][i];
    a.kv_stride[i] = st4[1][i];
    a.o_stride[i] = st4[2][i];
    a.do_stride[i] = st4[3][i];
  }
  if (!fix_strides(a.q_stride, batch, s_q, heads, head_dim) ||
      !fix_strides(a.kv_stride, s_kv > 0 ? batch : 1, s_kv, s_kv > 0 ? kv_heads : 1, head_dim) ||
      !fix_strides(a.o_stride, batch, s_q, heads, head_dim) || !fix_strides(a.do_stride, batch, s_q, heads, head_dim))
    return H3B_ERR_ALIGN;
  for (const void* p : {a.q, a.k, a.v, o, d_o})
    if (!h3b::aligned16(p)) return H3B_ERR_ALIGN;
  for (const void* p : {static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv),
                        static_cast<const void*>(workspace)})
    if ((reinterpret_cast<uintptr_t>(p) & 31u) != 0) return H3B_ERR_ALIGN;
  if (workspace_bytes < grad_workspace(a)) return H3B_ERR_SHAPE;
  a.part = static_cast<float*>(workspace);
  a.delta = a.part + grad_part_floats(a);
  a.do_sq = a.delta + grad_rows(a);
  a.v_sq = a.do_sq + grad_rows(a);
  a.do_top = a.v_sq + batch * kv_heads;
  a.kv_lens = kv_lens;
  a.key_mask = s_kv > 0 ? key_mask : nullptr;
  a.mask_stride = mask_stride;
  a.scale = scale;
  return h3b::xattn_bwd_launch(a, st);
}

extern "C" int h3b_kv8_attention_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                           int64_t s_q, int64_t block_tokens, int64_t max_blocks, int64_t* bytes) {
  if (bytes == nullptr) return H3B_ERR_ARG;
  const int rc = check_sizes(H3B_BF16, batch, heads, kv_heads, head_dim, s_q, 0);
  if (rc != H3B_OK) return rc;
  if (max_blocks <= 0 || block_tokens <= 0 || max_blocks * block_tokens > (1ll << 30)) return H3B_ERR_SHAPE;
  XAttn a = sizes(H3B_BF16, h3b::KV_INT8, batch, heads, kv_heads, head_dim, s_q, max_blocks * block_tokens);
  plan(a);
  *bytes = workspace_of(a);
  return H3B_OK;
}

extern "C" int h3b_kv8_attention(const void* q, void* o, float* lse, int dtype, int64_t batch, int64_t heads,
                                 int64_t kv_heads, int64_t head_dim, int64_t s_q, int64_t q_batch_stride,
                                 int64_t q_seq_stride, int64_t q_head_stride, int64_t o_batch_stride,
                                 int64_t o_seq_stride, int64_t o_head_stride, const uint8_t* k_codes,
                                 const uint8_t* v_codes, const float* k_scale, const float* v_scale, int code_type,
                                 int64_t num_blocks, int64_t block_tokens, const int32_t* table, int64_t max_blocks,
                                 const int32_t* lens, int causal, float scale, void* workspace,
                                 int64_t workspace_bytes, h3b_stream_t stream) {
  const int rc = check_sizes(dtype, batch, heads, kv_heads, head_dim, s_q, 0);
  if (rc != H3B_OK) return rc;
  if (code_type != H3B_KV_INT8 && code_type != H3B_KV_E4M3) return H3B_ERR_DTYPE;
  if ((block_tokens != 32 && block_tokens != 64 && block_tokens != 128) || num_blocks <= 0 || max_blocks <= 0 ||
      num_blocks * kv_heads > 0x7fffffffll || max_blocks * block_tokens > (1ll << 30))
    return H3B_ERR_SHAPE;
  if (!(scale > 0.0f)) return H3B_ERR_ARG;
  if (batch == 0 || s_q == 0) return H3B_OK;
  if (!q || !o || !k_codes || !v_codes || !k_scale || !v_scale || !table || !lens) return H3B_ERR_ARG;
  XAttn a = sizes(dtype, code_type == H3B_KV_INT8 ? h3b::KV_INT8 : h3b::KV_E4M3, batch, heads, kv_heads, head_dim, s_q,
                  max_blocks * block_tokens);
  a.q = q, a.k = k_codes, a.v = v_codes, a.o = o, a.lse = lse;
  a.q_stride[0] = q_batch_stride, a.q_stride[1] = q_seq_stride, a.q_stride[2] = q_head_stride;
  a.o_stride[0] = o_batch_stride, a.o_stride[1] = o_seq_stride, a.o_stride[2] = o_head_stride;
  if (!fix_strides(a.q_stride, batch, s_q, heads, head_dim) || !fix_strides(a.o_stride, batch, s_q, heads, head_dim))
    return H3B_ERR_ALIGN;
  for (const void* p : {q, static_cast<const void*>(o), a.k, a.v})
    if (!h3b::aligned16(p)) return H3B_ERR_ALIGN;
  a.table = table, a.max_blocks = static_cast<int>(max_blocks), a.block_tokens = static_cast<int>(block_tokens);
  a.num_blocks = static_cast<int>(num_blocks), a.k_scale = k_scale, a.v_scale = v_scale;
  a.kv_lens = lens;
  a.causal = causal != 0;
  a.scale = scale;
  return run(a, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}
