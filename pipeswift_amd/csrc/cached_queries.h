// What the kernels that read queries against the paged FP8 cache and take a
// whole batch's lengths from the device share (tree_attention.hip,
// attention_weights.hip): the argument checks of their C entries.
#pragma once

#include <cmath>

#include "paged_attention.h"

namespace psk_detail {

// The arguments both entries take, as their callers gave them.
struct CachedQueries {
  const void* q;
  int64_t q_tok_stride, q_head_stride;
  int q_dtype;
  const void* k;
  const int64_t* k_strides;
  const int32_t* block_table;
  int64_t block_table_stride, block_table_width;
  const int32_t* seq_lens;
  int64_t num_seqs, num_q_heads, num_kv_heads, head_size, block_size, num_blocks, total_q, max_seqlen_q;
  const int32_t* cu_seqlens_q;
  float softmax_scale;
  const float* q_descale;
  const float* k_descale;
};

// PSK_OK with `a` filled in, or the refusal.  Pointers are looked at last, so
// that an empty step may leave them NULL (*empty).
inline int check_cached_queries(const CachedQueries& c, DecodeArgs& a, bool* empty) {
  *empty = false;
  if (c.num_seqs < 0 || c.num_kv_heads <= 0 || c.num_q_heads <= 0 || c.num_q_heads % c.num_kv_heads)
    return fail(PSK_E_ARG, "bad head counts (q %lld, kv %lld)", (long long)c.num_q_heads, (long long)c.num_kv_heads);
  if (c.num_q_heads > INT32_MAX / kHead) return fail(PSK_E_ARG, "%lld query heads", (long long)c.num_q_heads);
  const int64_t group = c.num_q_heads / c.num_kv_heads;
  if (c.num_seqs > INT32_MAX / 2 / c.num_kv_heads) return fail(PSK_E_ARG, "%lld sequences", (long long)c.num_seqs);
  if (c.max_seqlen_q <= 0 || c.max_seqlen_q > INT32_MAX / group)
    return fail(PSK_E_ARG, "max_seqlen_q %lld", (long long)c.max_seqlen_q);
  if (c.total_q < 0 || c.total_q > INT32_MAX / c.num_q_heads) return fail(PSK_E_ARG, "total_q %lld", (long long)c.total_q);
  if (!c.cu_seqlens_q && c.total_q != c.num_seqs * c.max_seqlen_q)
    return fail(PSK_E_ARG, "without cu_seqlens_q every sequence has max_seqlen_q rows (%lld != %lld x %lld)",
                (long long)c.total_q, (long long)c.num_seqs, (long long)c.max_seqlen_q);
  if (c.head_size != kHead) return fail(PSK_E_ARG, "head_size must be %d (got %lld)", kHead, (long long)c.head_size);
  if (c.block_size <= 0 || c.block_size > INT32_MAX || c.num_blocks <= 0 || c.num_blocks > INT32_MAX ||
      c.block_table_width <= 0)
    return fail(PSK_E_ARG, "bad cache geometry");
  if (c.q_dtype != PSK_DTYPE_FP8_E4M3FN && c.q_dtype != PSK_DTYPE_BF16 && c.q_dtype != PSK_DTYPE_F16 &&
      c.q_dtype != PSK_DTYPE_F32)
    return fail(PSK_E_DTYPE, "query dtype %d", c.q_dtype);
  if (!std::isfinite(c.softmax_scale)) return fail(PSK_E_ARG, "softmax_scale is not finite");
  if (c.num_seqs == 0) {
    *empty = true;
    return PSK_OK;
  }
  if ((c.total_q > 0 && !c.q) || !c.k || !c.k_strides || !c.block_table || !c.seq_lens)
    return fail(PSK_E_ARG, "NULL pointer");
  const uint64_t k_align[4] = {uint64_t(uintptr_t(c.k)), uint64_t(c.k_strides[0]), uint64_t(c.k_strides[1]),
                               uint64_t(c.k_strides[2])};
  if (common_align(k_align, 4, 16) < 16) return fail(PSK_E_ARG, "K/V caches need 16-byte aligned bases and strides");
  const int qsz = dtype_size(c.q_dtype);
  const uint64_t q_align[3] = {uint64_t(uintptr_t(c.q)), uint64_t(c.q_tok_stride * qsz), uint64_t(c.q_head_stride * qsz)};
  if (common_align(q_align, 3, 16) < 16) return fail(PSK_E_ARG, "query rows need 16-byte alignment");

  a.q = static_cast<const char*>(c.q);
  a.q_tok_stride = c.q_tok_stride * qsz;
  a.q_head_stride = c.q_head_stride * qsz;
  a.k = static_cast<const uint8_t*>(c.k);
  a.k_blk = c.k_strides[0];
  a.k_row = c.k_strides[1];
  a.k_head = c.k_strides[2];
  a.block_table = c.block_table;
  a.bt_stride = c.block_table_stride;
  a.bt_width = c.block_table_width;
  a.seq_lens = c.seq_lens;
  a.num_blocks = int32_t(c.num_blocks);
  a.block_size = int32_t(c.block_size);
  a.bs_shift = log2_exact(c.block_size);
  a.num_kv_heads = int32_t(c.num_kv_heads);
  a.group = int32_t(group);
  a.heads = int32_t(group);
  a.q_len = int32_t(c.max_seqlen_q);
  a.cu_q = c.cu_seqlens_q;
  a.scale_log2 = c.softmax_scale * 1.4426950408889634f;
  a.qd = c.q_descale;
  a.kd = c.k_descale;
  return PSK_OK;
}

// Sequence b's query rows: [first, first + n), inside the total_q rows of q
// whatever cu_seqlens_q says.
struct SeqRows {
  int32_t first, n;
};
__device__ __forceinline__ SeqRows seq_rows(const DecodeArgs& a, int32_t total_q, int b) {
  const int64_t f = q_first(a, b);
  if (f < 0 || f >= total_q) return SeqRows{0, 0};
  return SeqRows{int32_t(f), min(q_count(a, b), total_q - int32_t(f))};
}

// The 16-byte chunks of one cached row of a kv head, or nullptr where the page is missing.
__device__ __forceinline__ const uint8_t* cached_row(const DecodeArgs& a, const uint8_t* base, int64_t blk, int64_t row,
                                                     int b, int key) {
  const int pi = page_index(a, key);
  if (pi >= a.bt_width) return nullptr;
  const int32_t id = a.block_table[int64_t(b) * a.bt_stride + pi];
  if (id < 0 || id >= a.num_blocks) return nullptr;
  return base + id * blk + int64_t(key - pi * a.block_size) * row;
}

}  // namespace psk_detail
