// The attention weight every cached token received, summed over the queries of
// a step (the scores an eviction goes by):
//   A[b, h, j] = decay A[b, h, j] + sum over query tokens i that see j and heads g of
//                exp(s_ij - lse[h G + g, i]),     j < seq_lens[b],
// s as the readers compute it and lse as they return it.
//
// A thread per key: its K row stays in registers and the step's query rows of
// the kv head pass by it, so no sum leaves the thread.
//
// C ABI: include/pipeswift_kv.h.  Nothing here allocates or synchronizes.

#include "cached_queries.h"

using namespace psk_detail;

namespace {

struct WeightArgs {
  DecodeArgs a;
  int32_t total_q;
  const float* lse;
  int64_t lse_head_stride;
  float* scores;
  int64_t seq_stride, head_stride;  // elements
  int32_t width;
  float decay;
  double scale_log2;  // softmax_scale * log2(e)
};

__device__ __forceinline__ float e4m3_value(uint32_t byte) { return e4m3_unpack2(byte, false).x; }

__global__ void __launch_bounds__(256) attention_weights_kernel(WeightArgs p, int q_dtype) {
  const DecodeArgs& a = p.a;
  __shared__ float s_q[kHead];
  const int h = int(blockIdx.y), b = int(blockIdx.z);
  const SeqRows r = seq_rows(a, p.total_q, b);
  const int L = min(max(a.seq_lens[b], 0), p.width);
  const int full = max(a.seq_lens[b], 0);
  const float qd = descale(a.qd, a.qd_b, a.qd_h, b, h);
  const float kd = descale(a.kd, a.kd_b, a.kd_h, b, h);
  const float sl = score_scale(p.scale_log2, qd, kd);
  for (int k0 = int(blockIdx.x) * 256; k0 < L; k0 += int(gridDim.x) * 256) {
    const int key = k0 + int(threadIdx.x);
    const bool in = key < L;
    uint32_t kw[32];
    const uint8_t* row = in ? cached_row(a, a.k + int64_t(h) * a.k_head, a.k_blk, a.k_row, b, key) : nullptr;
    for (int c = 0; c < 8; ++c) {
      const u32x4 w = row ? *reinterpret_cast<const u32x4*>(row + 16 * c) : u32x4(0);
      for (int j = 0; j < 4; ++j) kw[4 * c + j] = w[j];
    }
    float total = 0.0f;
    for (int i = 0; i < r.n; ++i) {
      const bool see = in && (!a.causal || key <= full - r.n + i);
      for (int g = 0; g < a.heads; ++g) {
        const int hq = h * a.heads + g;
        __syncthreads();
        if (threadIdx.x < 4) {
          uint32_t qw[8];
          const int d0 = 32 * int(threadIdx.x);
          const char* src = a.q + (int64_t(r.first) + i) * a.q_tok_stride + int64_t(hq) * a.q_head_stride;
          switch (q_dtype) {
            case PSK_DTYPE_FP8_E4M3FN: load_query_as<PSK_DTYPE_FP8_E4M3FN>(src, qd, d0, qw); break;
            case PSK_DTYPE_BF16: load_query_as<PSK_DTYPE_BF16>(src, qd, d0, qw); break;
            case PSK_DTYPE_F16: load_query_as<PSK_DTYPE_F16>(src, qd, d0, qw); break;
            default: load_query_as<PSK_DTYPE_F32>(src, qd, d0, qw); break;
          }
          for (int j = 0; j < 32; ++j) s_q[d0 + j] = e4m3_value((qw[j / 4] >> (8 * (j % 4))) & 0xFFu);
        }
        __syncthreads();
        if (!see) continue;
        float dot = 0.0f;
        for (int j = 0; j < 128; ++j) dot += e4m3_value((kw[j / 4] >> (8 * (j % 4))) & 0xFFu) * s_q[j];
        const float lse2 = float(double(p.lse[int64_t(hq) * p.lse_head_stride + r.first + i]) * 1.4426950408889634);
        total += __builtin_amdgcn_exp2f(__builtin_fmaf(dot, sl, -lse2));
      }
    }
    if (in) {
      float* dst = p.scores + int64_t(b) * p.seq_stride + int64_t(h) * p.head_stride + key;
      *dst = p.decay == 0.0f ? total : *dst * p.decay + total;
    }
  }
}

}  // namespace

extern "C" {

int psk_accumulate_attention_weights(float* scores, int64_t scores_seq_stride, int64_t scores_head_stride,
                                     int64_t scores_width, const void* q, int64_t q_tok_stride, int64_t q_head_stride,
                                     int q_dtype, const void* k_cache, const int64_t* k_strides, const float* lse,
                                     int64_t lse_head_stride, const int32_t* block_table, int64_t block_table_stride,
                                     int64_t block_table_width, const int32_t* seq_lens, int64_t num_seqs,
                                     int64_t num_q_heads, int64_t num_kv_heads, int64_t head_size, int64_t block_size,
                                     int64_t num_blocks, int64_t max_seq_len, int64_t total_q, int64_t max_seqlen_q,
                                     const int32_t* cu_seqlens_q, int causal, float softmax_scale, float decay,
                                     const float* q_descale, const float* k_descale, const int64_t* descale_strides,
                                     void* stream) {
  begin_device_call();
  const CachedQueries c{q, q_tok_stride, q_head_stride, q_dtype, k_cache, k_strides, block_table, block_table_stride,
                        block_table_width, seq_lens, num_seqs, num_q_heads, num_kv_heads, head_size, block_size,
                        num_blocks, total_q, max_seqlen_q, cu_seqlens_q, softmax_scale, q_descale, k_descale};
  WeightArgs p{};
  DecodeArgs& a = p.a;
  bool empty = false;
  if (scores_width < 0 || scores_width > INT32_MAX) return fail(PSK_E_ARG, "scores_width %lld", (long long)scores_width);
  if (max_seq_len < 0) return fail(PSK_E_ARG, "max_seq_len %lld", (long long)max_seq_len);
  if (!std::isfinite(decay)) return fail(PSK_E_ARG, "decay is not finite");
  if (const int st = check_cached_queries(c, a, &empty); st != PSK_OK) return st;
  if (empty || scores_width == 0) return PSK_OK;
  if (!scores || (total_q > 0 && !lse)) return fail(PSK_E_ARG, "NULL pointer");
  const int64_t zero[4] = {0, 0, 0, 0};
  const int64_t* ds = descale_strides ? descale_strides : zero;
  a.qd_b = ds[0];
  a.qd_h = ds[1];
  a.kd_b = ds[2];
  a.kd_h = ds[3];
  a.causal = causal ? 1 : 0;
  p.total_q = int32_t(total_q);
  p.lse = lse;
  p.lse_head_stride = lse_head_stride;
  p.scores = scores;
  p.seq_stride = scores_seq_stride;
  p.head_stride = scores_head_stride;
  p.width = int32_t(scores_width);
  p.decay = decay;
  p.scale_log2 = double(softmax_scale) * 1.4426950408889634;
  if (num_seqs > 65535 || num_kv_heads > 65535) return fail(PSK_E_ARG, "too many sequences or heads");
  const int64_t keys = max_seq_len < scores_width ? max_seq_len : scores_width;
  const int64_t blocks = ceil_div(keys, 256) < 256 ? ceil_div(keys, 256) : 256;
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(attention_weights_kernel, dim3(unsigned(blocks > 0 ? blocks : 1), unsigned(num_kv_heads), unsigned(num_seqs)),
                     dim3(256), 0, st, p, q_dtype);
  return check_launch("attention_weights_kernel launch");
}

}  // extern "C"
