// Attention of a tree of drafted tokens over the paged FP8 E4M3FN cache.
//
// Sequence b of L cached tokens has n drafted tokens, its last n; drafted token
// i sees every key before them and the drafted keys t whose bit of its mask is
// set.  Otherwise as the decode reader (paged_attention.hip): q~ = e4m3(q / qd),
// s = softmax_scale qd kd (q~ . K), out = vd softmax(s) V, lse = log sum exp s.
//
// A wave per query row: its lanes take 64 keys at a time for the scores, then
// two columns each for P V, with a running maximum and sum.
//
// C ABI: include/pipeswift_kv.h.  Nothing here allocates or synchronizes.

#include "cached_queries.h"

using namespace psk_detail;

namespace {

struct TreeArgs {
  DecodeArgs a;
  int32_t total_q;
  const int64_t* mask;
  int64_t mask_stride;  // words from a query token's mask to the next one's
  int32_t mask_words;
};

__device__ __forceinline__ float e4m3_value(uint32_t byte) { return e4m3_unpack2(byte, false).x; }

// Key position `key` of a sequence whose drafted tokens start at `ctx`, for a token with mask row `m`.
__device__ __forceinline__ bool sees(const TreeArgs& p, const int64_t* m, int ctx, int n, int key) {
  const int t = key - ctx;
  if (t < 0) return true;
  return t < n && (t >> 6) < p.mask_words && ((uint64_t(m[t >> 6]) >> (t & 63)) & 1);
}

__global__ void __launch_bounds__(256) tree_attention_kernel(TreeArgs p, int q_dtype, int out_dtype) {
  const DecodeArgs& a = p.a;
  __shared__ float s_q[4][kHead];
  __shared__ float s_p[4][64];
  const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) >> 6;
  const int hq = int(blockIdx.y), h = hq / a.heads, b = int(blockIdx.z);
  const SeqRows r = seq_rows(a, p.total_q, b);
  const int i = int(blockIdx.x) * 4 + wave;
  const bool live = i < r.n;
  const float qd = descale(a.qd, a.qd_b, a.qd_h, b, h);
  const float kd = descale(a.kd, a.kd_b, a.kd_h, b, h);
  const float vd = descale(a.vd, a.vd_b, a.vd_h, b, h);
  if (live && lane < 4) {
    uint32_t qw[8];
    const char* src = a.q + (int64_t(r.first) + i) * a.q_tok_stride + int64_t(hq) * a.q_head_stride;
    switch (q_dtype) {
      case PSK_DTYPE_FP8_E4M3FN: load_query_as<PSK_DTYPE_FP8_E4M3FN>(src, qd, 32 * lane, qw); break;
      case PSK_DTYPE_BF16: load_query_as<PSK_DTYPE_BF16>(src, qd, 32 * lane, qw); break;
      case PSK_DTYPE_F16: load_query_as<PSK_DTYPE_F16>(src, qd, 32 * lane, qw); break;
      default: load_query_as<PSK_DTYPE_F32>(src, qd, 32 * lane, qw); break;
    }
    for (int j = 0; j < 32; ++j) s_q[wave][32 * lane + j] = e4m3_value((qw[j / 4] >> (8 * (j % 4))) & 0xFFu);
  }
  __syncthreads();
  if (!live) return;
  const int L = max(a.seq_lens[b], 0), ctx = L - r.n;
  const int64_t* m = p.mask + (int64_t(r.first) + i) * p.mask_stride;
  const float sl = a.scale_log2 * qd * kd;
  float top = -__builtin_inff(), sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
  for (int k0 = 0; k0 < L; k0 += 64) {
    const int key = k0 + lane;
    const bool see = key < L && sees(p, m, ctx, r.n, key);
    float s = -__builtin_inff();
    if (see) {
      const uint8_t* row = cached_row(a, a.k + int64_t(h) * a.k_head, a.k_blk, a.k_row, b, key);
      float dot = 0.0f;
      for (int c = 0; row && c < 8; ++c) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(row + 16 * c);
        for (int j = 0; j < 16; ++j) dot += e4m3_value((w[j / 4] >> (8 * (j % 4))) & 0xFFu) * s_q[wave][16 * c + j];
      }
      s = dot * sl;
    }
    float mx = s;
    for (int x = 1; x < 64; x <<= 1) mx = __builtin_fmaxf(mx, __shfl_xor(mx, x));
    const float up = __builtin_fmaxf(top, mx);
    const uint64_t seen = __ballot(see);
    if (!seen) continue;
    const float f = top == up ? 1.0f : __builtin_amdgcn_exp2f(top - up);
    top = up;
    const float w = see ? __builtin_amdgcn_exp2f(s - top) : 0.0f;
    float ws = w;
    for (int x = 1; x < 64; x <<= 1) ws += __shfl_xor(ws, x);
    sum = sum * f + ws;
    o0 *= f;
    o1 *= f;
    for (int j = 0; j < 64; ++j) {
      if (!((seen >> j) & 1)) continue;
      const uint8_t* row = cached_row(a, a.v + int64_t(h) * a.v_head, a.v_blk, a.v_row, b, k0 + j);
      const float pj = __shfl(w, j);
      if (row) {
        const uint32_t v = *reinterpret_cast<const uint16_t*>(row + 2 * lane);
        const f32x2 f2 = e4m3_unpack2(v, false);
        o0 += pj * f2.x;
        o1 += pj * f2.y;
      }
    }
  }
  const bool any = sum != 0.0f;  // (a NaN sum counts)
  const float inv = any ? vd / sum : 0.0f;
  o0 = any ? o0 * inv : 0.0f;
  o1 = any ? o1 * inv : 0.0f;
  char* dst = a.out + (int64_t(r.first) + i) * a.out_tok_stride + int64_t(hq) * a.out_head_stride;
  if (out_dtype == PSK_DTYPE_BF16) {
    reinterpret_cast<uint16_t*>(dst)[2 * lane] = Elt<PSK_DTYPE_BF16>::from_f32(o0);
    reinterpret_cast<uint16_t*>(dst)[2 * lane + 1] = Elt<PSK_DTYPE_BF16>::from_f32(o1);
  } else {
    reinterpret_cast<float*>(dst)[2 * lane] = o0;
    reinterpret_cast<float*>(dst)[2 * lane + 1] = o1;
  }
  if (a.lse && lane == 0)
    a.lse[int64_t(hq) * a.lse_head_stride + r.first + i] =
        any ? (top + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f : -__builtin_inff();
  (void)s_p;
}

}  // namespace

extern "C" {

int64_t psk_paged_tree_workspace_len(int64_t num_seqs, int64_t total_q, int64_t max_seqlen_q, int64_t num_q_heads,
                                     int64_t num_kv_heads, int64_t max_seq_len) {
  if (num_seqs < 0 || total_q < 0 || max_seqlen_q <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 ||
      num_q_heads % num_kv_heads || max_seq_len < 0)
    return PSK_E_ARG;
  return 0;
}

int psk_paged_tree_attention(const void* q, int64_t q_tok_stride, int64_t q_head_stride, int q_dtype,
                             const void* k_cache, const void* v_cache, const int64_t* k_strides,
                             const int64_t* v_strides, const int32_t* block_table, int64_t block_table_stride,
                             int64_t block_table_width, const int32_t* seq_lens, int64_t num_seqs, int64_t num_q_heads,
                             int64_t num_kv_heads, int64_t head_size, int64_t block_size, int64_t num_blocks,
                             int64_t max_seq_len, int64_t total_q, int64_t max_seqlen_q, const int32_t* cu_seqlens_q,
                             const int64_t* tree_mask, int64_t tree_mask_stride, int64_t tree_mask_words,
                             float softmax_scale, const float* q_descale, const float* k_descale,
                             const float* v_descale, const int64_t* descale_strides, void* out,
                             int64_t out_tok_stride, int64_t out_head_stride, int out_dtype, float* lse,
                             int64_t lse_head_stride, float* workspace, int64_t workspace_len, void* stream) {
  begin_device_call();
  const CachedQueries c{q, q_tok_stride, q_head_stride, q_dtype, k_cache, k_strides, block_table, block_table_stride,
                        block_table_width, seq_lens, num_seqs, num_q_heads, num_kv_heads, head_size, block_size,
                        num_blocks, total_q, max_seqlen_q, cu_seqlens_q, softmax_scale, q_descale, k_descale};
  TreeArgs p{};
  DecodeArgs& a = p.a;
  bool empty = false;
  if (out_dtype != PSK_DTYPE_BF16 && out_dtype != PSK_DTYPE_F32)
    return fail(PSK_E_DTYPE, "output dtype %d (bf16 or f32)", out_dtype);
  if (tree_mask_words < 1 || tree_mask_words > INT32_MAX || max_seqlen_q > 64 * tree_mask_words)
    return fail(PSK_E_ARG, "%lld mask words of 64 tokens for up to %lld drafted tokens", (long long)tree_mask_words,
                (long long)max_seqlen_q);
  if (max_seq_len < 0) return fail(PSK_E_ARG, "max_seq_len %lld", (long long)max_seq_len);
  if (const int st = check_cached_queries(c, a, &empty); st != PSK_OK) return st;
  if (empty || total_q == 0) return PSK_OK;
  if (!v_cache || !v_strides || !tree_mask || !out) return fail(PSK_E_ARG, "NULL pointer");
  const uint64_t v_align[4] = {uint64_t(uintptr_t(v_cache)), uint64_t(v_strides[0]), uint64_t(v_strides[1]),
                               uint64_t(v_strides[2])};
  if (common_align(v_align, 4, 16) < 16) return fail(PSK_E_ARG, "K/V caches need 16-byte aligned bases and strides");
  const int osz = dtype_size(out_dtype);
  const uint64_t o_align[3] = {uint64_t(uintptr_t(out)), uint64_t(out_tok_stride * osz),
                               uint64_t(out_head_stride * osz)};
  if (common_align(o_align, 3, 4 * osz) < 4 * osz)
    return fail(PSK_E_ARG, "output rows need %d-byte alignment", 4 * osz);
  a.v = static_cast<const uint8_t*>(v_cache);
  a.v_blk = v_strides[0];
  a.v_row = v_strides[1];
  a.v_head = v_strides[2];
  const int64_t zero[6] = {0, 0, 0, 0, 0, 0};
  const int64_t* ds = descale_strides ? descale_strides : zero;
  a.qd_b = ds[0];
  a.qd_h = ds[1];
  a.kd_b = ds[2];
  a.kd_h = ds[3];
  a.vd = v_descale;
  a.vd_b = ds[4];
  a.vd_h = ds[5];
  a.out = static_cast<char*>(out);
  a.out_tok_stride = out_tok_stride * osz;
  a.out_head_stride = out_head_stride * osz;
  a.lse = lse;
  a.lse_head_stride = lse_head_stride;
  p.total_q = int32_t(total_q);
  p.mask = tree_mask;
  p.mask_stride = tree_mask_stride;
  p.mask_words = int32_t(tree_mask_words);
  (void)workspace;
  (void)workspace_len;
  if (num_seqs > 65535 || num_q_heads > 65535) return fail(PSK_E_ARG, "too many sequences or heads");
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(tree_attention_kernel, dim3(unsigned(ceil_div(max_seqlen_q, 4)), unsigned(num_q_heads), unsigned(num_seqs)),
                     dim3(256), 0, st, p, q_dtype, out_dtype);
  return check_launch("tree_attention_kernel launch");
}

}  // extern "C"
