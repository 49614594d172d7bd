// What the kernels behind h3b_cross_attention_fwd / _bwd and h3b_kv8_attention
// share: the call's sizes and pointers, and the entry of each kernel family.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/h3b.h"

namespace h3b {

// Where keys and values come from: a dense 16-bit tensor of q's type, or the
// 8-bit cache (codes int8 or e4m3, one scale per block of tokens and head).
enum KvKind { KV_DENSE = 0, KV_INT8 = 1, KV_E4M3 = 2 };

// The smallest scale that a cache's block counts with: a scale of 0 (a block of
// zeros; an empty cache) has no logarithm.  Its values are then off by 4e-25 at
// most, and its tokens keep their share of the weights: an exponent lowered by
// log2 of this (90) does not vanish beside blocks of scale 2^10 and scores 15 nats
// above, and l = sum w / sv of 2^14 a token stays finite over 1.4e7 tokens.
constexpr float KV8_SCALE_MIN = 7e-28f;

// One attention call.  Strides are in elements, in the order (batch, token,
// head); o_* as q_*.  Element (b, s, h, d) of q lies at q + b*q_stride[0] +
// s*q_stride[1] + h*q_stride[2] + d.
struct XAttn {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* lse;  // [batch, heads, s_q] or null
  int dtype;   // H3B_BF16 / H3B_F16: q, o (and dense k, v)
  KvKind kind;
  int64_t q_stride[3];
  int64_t kv_stride[3];  // dense only
  int64_t o_stride[3];
  int batch, heads, kv_heads, head_dim, s_q;
  int s_kv;                  // dense: keys per sample; cache: max_blocks * block_tokens
  const int32_t* kv_lens;    // [batch] or null (all s_kv keys)
  const uint8_t* key_mask;   // dense: [batch, s_kv] bytes, 0 = left out; or null
  int64_t mask_stride;
  // cache
  const int32_t* table;  // [batch, max_blocks]
  int max_blocks, block_tokens, num_blocks;
  const float* k_scale;  // [num_blocks, kv_heads]
  const float* v_scale;
  void* pre_k;  // workspace [batch, kv_heads, s_kv, head_dim] of 16-bit operands, or null: see xattn_tile.cu
  void* pre_v;
  int causal;  // query i of s_q sees keys < kv_len - s_q + i + 1
  float scale;
  // split calls: partial results of `splits` key ranges per row
  int splits;
  float* part_o;   // [splits, batch*heads*s_q, head_dim], unnormalised
  float2* part_ml; // [splits, batch*heads*s_q]: running max (log2 domain), sum
};

// A backward call.  Outputs dq, dk, dv are dense [batch, tokens, heads, D].
struct XAttnGrad {
  const void* q;
  const void* k;
  const void* v;
  const void* o;
  const void* d_o;
  const float* lse;  // [batch, heads, s_q]
  void* dq;
  void* dk;
  void* dv;
  int dtype;
  int64_t q_stride[3], kv_stride[3], o_stride[3], do_stride[3];
  int batch, heads, kv_heads, head_dim, s_q, s_kv;
  const int32_t* kv_lens;
  const uint8_t* key_mask;
  int64_t mask_stride;
  float scale;
  float* delta;  // workspace [batch, heads, s_q]
  float* do_sq;  // f16: workspace [batch, heads, s_q], |do|^2 of a row
  float* v_sq;   // f16: workspace [batch, kv_heads], largest |v|^2 of a kept key
  float* do_top; // f16: behind it, [batch, kv_heads], largest |do|^2 of the rows that share a key head
  int splits;
  float* part;   // workspace [dv | dk][splits, batch, s_kv, kv_heads, D], if splits > 1
};
int xattn_bwd_splits(const XAttnGrad& a);
int xattn_bwd_launch(const XAttnGrad& a, cudaStream_t stream);

// Keys split over so many ranges by the row kernel / the tile kernel.
int xattn_rows_splits(const XAttn& a);
int xattn_tile_splits(const XAttn& a);

int xattn_rows_launch(const XAttn& a, cudaStream_t stream);
int xattn_tile_launch(const XAttn& a, cudaStream_t stream);
// Writes a cache's codes out as 16-bit numbers of q's type into pre_k, pre_v.
int kv8_expand_launch(const XAttn& a, cudaStream_t stream);
// Joins the ranges of a split call into o and lse.
int xattn_combine_launch(const XAttn& a, cudaStream_t stream);

}  // namespace h3b
