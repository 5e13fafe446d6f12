// What the two kernels of attention over the 4-bit cache share (mxfp4_attention.hip:
// a wave a tile of keys, for few query rows; mxfp4_prefill.hip: a workgroup a block
// of 256 query rows).
#pragma once

#include "cached_queries.h"
#include "mxfp4.h"

namespace psk_detail {

constexpr int kCodes = kHead / 2;    // bytes of a row's codes
constexpr int kRecord = kHead + 4;   // floats of a query row's partial result: accumulators, maximum, sum
constexpr float kShareMost = 32768.0f;  // a lane's share of a tile's weights before a row's maximum is raised
// The maximum of a row without a score yet: no finite one lies below it, so that the first raises it.
constexpr float kNoScore = -3.402823466e38f;
// From a maximum of this size on a wave rounds its scores' scaled values before it subtracts
// the maximum, so that the largest gives 0.  Below, an fma does both in one instruction and leaves
// the rounding of the maximum in the difference, 2^-5 and less, the same for every key; further on
// that grows with the score, and weights with it past what 16 bits and 32 hold.
constexpr float kFarScore = 0x1p20f;
// The size of the scale: a negative one is applied as -q (exact); one of 0 stays above it, for a hidden key's -inf.
__device__ __forceinline__ float scale_size(double scale_log2) {
  return __builtin_fmaxf(__builtin_fabsf(float(scale_log2)), 0x1p-126f);
}
__device__ __forceinline__ bool is_far(float m) { return __builtin_fabsf(m) > kFarScore && m != kNoScore; }

typedef u32x4 u32x4_any __attribute__((aligned(4)));

__device__ __forceinline__ void store4(char* dst, int dtype, f32x4 v) {
  if (dtype == PSK_DTYPE_F32) *reinterpret_cast<f32x4*>(dst) = v;
  else if (dtype == PSK_DTYPE_BF16) *reinterpret_cast<bf16x4*>(dst) = __builtin_convertvector(v, bf16x4);
  else *reinterpret_cast<u32x2*>(dst) = __builtin_bit_cast(u32x2, __builtin_convertvector(v, f16x4));
}

// Columns col .. col + 3 of query row `row` (token row / heads) of kv head h, and its
// lse with the first; zeros and -inf for a row that sees no key.  (A row whose scores are all
// past the largest float has a sum of 0 and is NaN, 0 / 0.)
__device__ __forceinline__ void finish(const DecodeArgs& a, int out_dtype, const SeqRows& r, int h, int row, int col,
                                       f32x4 o, float m, float sum, bool sees) {
  const int i = row / a.heads, hq = h * a.heads + row - i * a.heads;
  if (i >= r.n) return;
  const f32x4 v = sees ? o * (1.0f / sum) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int osz = out_dtype == PSK_DTYPE_F32 ? 4 : 2;
  store4(a.out + (int64_t(r.first) + i) * a.out_tok_stride + int64_t(hq) * a.out_head_stride + col * osz, out_dtype, v);
  if (a.lse && col == 0)
    a.lse[int64_t(hq) * a.lse_head_stride + r.first + i] =
        sees ? (m + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f : -__builtin_inff();
}

// Eight elements of a query row as bf16 and, for the wider types, what that leaves.
template <int Q_DT>
__device__ __forceinline__ void query8(const char* p, bool negate, bf16x8& hi, bf16x8& lo) {
  if constexpr (Q_DT == PSK_DTYPE_BF16) {
    u32x4 x = p ? *reinterpret_cast<const u32x4*>(p) : u32x4(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] ^= negate ? 0x80008000u : 0u;
    hi = __builtin_bit_cast(bf16x8, x);
  } else {
    typename Elt<Q_DT>::Bits e[8] = {};
    if (p) __builtin_memcpy(e, p, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = negate ? -Elt<Q_DT>::to_f32(e[i]) : Elt<Q_DT>::to_f32(e[i]);
      hi[i] = __bf16(x);
      lo[i] = __bf16(x - float(hi[i]));
    }
  }
}

// Sequences of more query tokens than `most` go to the blocks of mxfp4_prefill.hip.
struct Mx4Prefill {
  int64_t num_seqs, total_q, max_seqlen_q, max_seq_len;
  int32_t most;
  double scale_log2;
  int q_dtype, out_dtype;
};

// Floats of workspace (rows: `most`), and the launch (`a` filled in).
int64_t mx4_prefill_floats(int64_t num_seqs, int64_t total_q, int64_t max_seqlen_q, int64_t num_q_heads,
                           int64_t num_kv_heads, int64_t max_seq_len, int64_t rows);
int launch_mx4_prefill(const DecodeArgs& a, const Mx4Prefill& s, float* workspace, hipStream_t st);

}  // namespace psk_detail
