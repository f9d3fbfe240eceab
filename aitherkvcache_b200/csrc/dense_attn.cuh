// Arguments of the attention kernels over the dense (fp16 / bf16) paged cache: dense_decode.cu (single tokens) and
// dense_prefill.cu (chunks of new tokens).
#pragma once

#include "common.cuh"

namespace akv {

struct DenseArgs {
  const void* q; int64_t q_st, q_sh;
  const void* k; int64_t k_sb, k_sp, k_sh;
  const void* v; int64_t v_sb, v_sp, v_sh;
  const void* block_tables; int bt_dtype; int64_t bt_stride;
  const void* seq_lens; int sl_dtype;
  const void* starts; int qs_dtype;
  int num_seqs, n_tokens, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq;
  int64_t num_blocks;
  float scale_log2;             // scale * log2(e): scores are kept in log2 units
  int window;                   // keys a token sees, itself included; 0: all before it
  void* out; int64_t out_st, out_sh;
};

}  // namespace akv

// Mirror of akv_dense_attn_params in include/akv_b200.h.
struct akv_dense_attn_params {
  const void* query; int dtype; int64_t q_stride_tok, q_stride_head;
  const void* k_cache; int64_t k_stride_blk, k_stride_pos, k_stride_head;
  const void* v_cache; int64_t v_stride_blk, v_stride_pos, v_stride_head;
  const void* block_tables; int bt_dtype; int64_t bt_stride_seq;
  const void* seq_lens; int sl_dtype;
  const void* query_start_loc; int qs_dtype;
  int num_seqs, num_tokens, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq;
  int64_t num_blocks;
  float scale; int window;
  void* out; int64_t out_stride_tok, out_stride_head;
  int zero_tail;
  void* workspace; size_t workspace_bytes;
  void* stream;
};

namespace akv {

// Checks what both entry points share and fills the kernel arguments (dense_decode.cu).
int dense_common(const akv_dense_attn_params* p, const char* who, DenseArgs* a);

// Finite numbers only reach log2 units through this: 2^x, -inf gives 0.
__device__ __forceinline__ float dense_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row's reference m in log2 units: it moves when a score exceeds what the largest weight may be, to the score minus
// DENSE_SHIFT.  fp16 ends at 2^-24 below, so weights relative to the largest score itself would vanish from the product below
// 2^-25 of the largest weight while the sum still counts them: 40000 keys of 2^-26 each, 6e-4 of the result, came out as
// zeros.  With the factor 2^7 the largest weight stays at or below 2^15 (65504 is the end above) and what vanishes is 2^-32
// of it and less.  bf16 has the range of float32.
constexpr float DENSE_RESCALE = 8.0f;
template <bool BF> constexpr float DENSE_SHIFT = BF ? 0.0f : 7.0f;
template <bool BF> constexpr float DENSE_TOP = DENSE_RESCALE + DENSE_SHIFT<BF>;      // log2 of the largest weight

template <bool BF> __device__ __forceinline__ uint32_t dense_pack(float lo, float hi) {
  if (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool BF> __device__ __forceinline__ void dense_store(void* p, int64_t i, float v) {
  if (BF) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

// Block of the pool that holds key `key` of a sequence: entries outside the pool are clamped, so a stale or padded table
// entry never reads out of bounds.
__device__ __forceinline__ int64_t dense_block(const DenseArgs& a, int s, int idx) {
  if (idx >= a.max_blocks_per_seq) idx = a.max_blocks_per_seq - 1;
  const int64_t b = load_index(a.block_tables, a.bt_dtype, (int64_t)s * a.bt_stride + idx);
  return b < 0 ? 0 : (b >= a.num_blocks ? a.num_blocks - 1 : b);
}

}  // namespace akv
