// Attention over the paged 4-bit KV cache for steps of many query tokens, MI355X
// (gfx950): the arithmetic of mxfp4_attention.hip, bound by the matrix cores.
//
// A workgroup takes a block of kBlock query rows (query tokens x heads of one kv head)
// and streams the keys that any of them sees once, 64 at a time, through two LDS
// stages that all its waves read:
//   * a thread loads one group of 32 elements (16 bytes) of K or of V and its scale
//     byte a stage ahead, and stores its values: K as bf16, V as fp16 rows of 256 bytes,
//     16-byte chunk c of key t at c ^ (t & 15) and at c ^ (2 (t & 7)), which spreads the
//     writes and both kinds of reads over the banks;
//   * S^T = K Q^T is eight v_mfma_f32_32x32x16_bf16 for 32 keys and a wave's 32 query
//     rows, and leaves each lane one row (l % 32) and keys 8 (i / 4) + 4 (l / 32) + i % 4;
//   * O^T = V^T P^T is eight v_mfma_f32_32x32x16_f16: the lane's weights are the P^T operand
//     as they stand, and ds_read_b64_tr_b16 gives V^T.  Into an fp16 or float32 out P is the sum
//     of two fp16 (2^-22) and P V runs twice.  Into a bf16 out P is rounded once (2^-11): the
//     error against 64 bits is 1.669e-3 of the values so, 1.658e-3 by the output's rounding
//     alone, and the second product takes 1410 us instead of 1050 for the chunk below.
//     (One rounding into fp16 left 2.8e-4 where the output's own is 2.1e-4.)
// V is exact in fp16 where its scales lie in [2^-23, 2^13]; a block that meets another
// one is computed again with V as bf16 and P as the sum of two bf16 (2^-17).
// A row's maximum is raised only when a tile's weights pass 2^15, to kHeadRoom below the
// largest, so that the common path has no rescale.
//
// Bound by the matrix cores and the softmax's vector work in turn: a chunk of 2048 tokens over
// 30000 keys (32 heads over 8) takes 1050 us, 1.0 PFLOP/s where large products reach 1.2 (8192^3) to
// 1.35 (16384^3); 8 prompts of 100 to 4000 tokens 474 us, 790 TFLOP/s.  Both halves of a stage at once need more registers than there
// are (1640 us); wave priorities around the products gain nothing.
//
// Where the blocks are fewer than the CUs, a block's keys are split over several
// workgroups, whose partial results a second kernel joins in order.
//
// C ABI: include/pipeswift_kv.h (psk_paged_mxfp4_attention).  Nothing here allocates or
// synchronizes.

#include <algorithm>

#include "mxfp4_attention.h"
#include "prefill_runs.h"

using namespace psk_detail;

namespace {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kBlock = 32 * kWaves;  // query rows of a workgroup
constexpr int kStage = 64;           // keys of a stage
constexpr int kMostSplit = 256;      // workgroups of a step that is split: a CU has one at a time (256
                                     // rows over 8000 keys 59 us, 74 with twice as many)
constexpr int kSplitKeys = 512;      // keys of a split, at least
constexpr int kFp16Low = 104, kFp16High = 140;  // scale bytes whose values fp16 holds

static_assert(kBlock == kBlockRows, "order_blocks counts blocks of as many rows");

struct PrefillArgs {
  DecodeArgs a;
  const int32_t* blocks;  // [num_seqs + 1]: blocks before launch position k; the total last
  const int32_t* order;   // [num_seqs]: the sequence at launch position k
  int32_t num_seqs, total_q;
  int32_t tq;             // query tokens of a block
  int32_t max_blocks;
  int32_t splits;         // workgroups that share a block's keys; 0: by the blocks that there are,
  int32_t most_splits;    // at most so many
  int32_t out_dtype;
  double scale_log2;
  float* records;         // [blocks][kv heads][splits][kBlock][kRecord]
};

// The splits of a step of `jobs` blocks and kv heads whose longest sequence can be cut into `most`.
__host__ __device__ constexpr int64_t splits_of(int64_t jobs, int64_t most) {
  const int64_t n = jobs < kMostSplit ? kMostSplit / int32_t(jobs > 0 ? jobs : 1) : 1;
  return n < most ? n : most > 1 ? most : 1;
}

// The step's blocks (max_blocks at most, whatever cu_seqlens_q says) and their splits.
__device__ __forceinline__ int blocks_here(const PrefillArgs& p) { return min(p.blocks[p.num_seqs], p.max_blocks); }
__device__ __forceinline__ int splits_here(const PrefillArgs& p) {
  return p.splits > 0 ? p.splits : int(splits_of(int64_t(blocks_here(p)) * p.a.num_kv_heads, p.most_splits));
}

// The launch order of the blocks of sequences with more than `most` query tokens.
__global__ void __launch_bounds__(1024) mx4_order_kernel(DecodeArgs a, int num_seqs, int total_q, int tq, int most,
                                                         int32_t* blocks, int32_t* order) {
  __shared__ OrderLds lds;
  const int b = int(threadIdx.x);
  if (num_seqs <= kOrderMax) {
    if (b < num_seqs) {
      const int n = seq_rows(a, total_q, b).n;
      put_sequence(lds, b, n > most ? n : 0, cached_len(a, b));
    }
    __syncthreads();
  }
  order_blocks<1024>(a, num_seqs, tq, blocks, order, lds);
}

// The launch position of block u (blocks[0] = 0 <= u < blocks[num_seqs]): the last k
// with blocks[k] <= u, 64 ways a round.
__device__ __forceinline__ int position_of(const int32_t* blocks, int num_seqs, int u, int lane) {
  int lo = 0, n = num_seqs;  // the answer lies in [lo, lo + n) and blocks[lo] <= u
  while (n > 1) {
    const int step = (n + 63) / 64;
    const bool le = lane * step < n && blocks[lo + lane * step] <= u;  // true on a prefix of the lanes
    const int last = 63 - __builtin_clzll(__ballot(le));
    lo += last * step;
    n = min(step, n - last * step);
  }
  return lo;
}

struct Stages {
  u32x4 k[2][kStage * 16];
  u32x4 v[2][kStage * 16];
};

struct Where {
  int b, h, i0, ni;  // sequence, kv head, the block's first query token and how many
  SeqRows r;
};
__device__ __forceinline__ bool block_of(const PrefillArgs& p, int idx, int lane, Where& w) {
  if (idx >= blocks_here(p)) return false;
  const int k = __builtin_amdgcn_readfirstlane(position_of(p.blocks, p.num_seqs, idx, lane));
  w.b = __builtin_amdgcn_readfirstlane(p.order[k]);
  // a sequence's blocks from its last (the most keys, when causal) to its first
  w.i0 = __builtin_amdgcn_readfirstlane((p.blocks[k + 1] - 1 - idx) * p.tq);
  w.r = seq_rows(p.a, p.total_q, w.b);
  w.ni = min(p.tq, w.r.n - w.i0);
  return w.ni > 0;
}

template <int Q_DT, bool P_PAIRS>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2))) mx4_prefill_kernel(PrefillArgs p) {
  constexpr bool kPairs = Q_DT != PSK_DTYPE_BF16;
  __shared__ Stages lds;
  __shared__ int32_t s_nan[4];  // of each group of columns the first key whose V is NaN there
  __shared__ int32_t s_wide;
  const DecodeArgs& a = p.a;
  const int tid = int(threadIdx.x), lane = tid & 63, half = lane >> 5, l31 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Hkv = a.num_kv_heads, G = a.heads;
  const int v0 = int(blockIdx.x) / Hkv, h = int(blockIdx.x) - v0 * Hkv;
  const int splits = splits_here(p), idx = v0 / splits, split = v0 - idx * splits;
  Where w;
  w.h = h;
  if (!block_of(p, idx, lane, w)) return;
  const int L = cached_len(a, w.b);
  const int base = a.causal ? L - w.r.n + 1 : L;
  auto limit = [&](int i) { return a.causal ? min(max(base + i, 0), L) : L; };
  const int key_end = limit(w.i0 + w.ni - 1);
  // this split's stages
  const int stages = (key_end + kStage - 1) / kStage;
  const int t_from = int(int64_t(stages) * split / splits), t_to = int(int64_t(stages) * (split + 1) / splits);

  // the wave's rows: which there are, what all and any of them see
  const int row = wave * 32 + l31, ti = row / G;
  const bool live = ti < w.ni;
  const int row_lim = live ? limit(w.i0 + ti) : 0;
  const bool wave_live = wave * 32 < w.ni * G;
  const int w_open = limit(w.i0 + wave * 32 / G), w_end = wave_live ? limit(w.i0 + min((wave * 32 + 31) / G, w.ni - 1)) : 0;

  const float sl_signed = float(p.scale_log2);
  bf16x8 qop[8], qlo[kPairs ? 8 : 1];
  {
    const char* src = live ? a.q + (int64_t(w.r.first) + w.i0 + ti) * a.q_tok_stride +
                                 int64_t(h * G + row - ti * G) * a.q_head_stride
                           : nullptr;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      query8<Q_DT>(src ? src + (16 * c + 8 * half) * Elt<Q_DT>::kSize : nullptr, sl_signed < 0.0f, qop[c], qlo[kPairs ? c : 0]);
  }

  // staging: waves 0..3 load K, 4..7 V; thread i of 256 group i % 4 of key i / 4
  const bool is_v = wave >= kWaves / 2;
  const int skey = (tid & 255) >> 2, sgroup = tid & 3;
  const uint8_t* sbase = is_v ? a.v + int64_t(h) * a.v_head : a.k + int64_t(h) * a.k_head;
  const int64_t sblk = is_v ? a.v_blk : a.k_blk, srow = is_v ? a.v_row : a.k_row;
  const int32_t* bt_row = a.block_table + int64_t(w.b) * a.bt_stride;
  auto page_id = [&](int t) -> int32_t {
    const int key = t * kStage + skey;
    if (key >= key_end) return -1;
    const int pi = page_index(a, key);
    return pi < a.bt_width ? bt_row[pi] : -1;
  };
  u32x4 raw;
  uint32_t byte;
  auto fetch = [&](int t, int32_t id) {
    raw = u32x4(0);
    byte = 127;
    if (id >= 0 && id < a.num_blocks) {
      const int key = t * kStage + skey;
      const uint8_t* at = sbase + int64_t(id) * sblk + int64_t(key - page_index(a, key) * a.block_size) * srow;
      raw = *reinterpret_cast<const u32x4_any*>(at + 16 * sgroup);
      byte = at[kCodes + sgroup];
    }
  };
  auto put_stage = [&](auto wide_tag, int st, int t) {
    constexpr bool WIDE = decltype(wide_tag)::value;
    if (is_v) {
      if (__builtin_expect(mx_not_finite(raw, byte), 0)) {  // (0 x NaN) zeros here, NaN at the end for the rows that see it
        atomicMin(&s_nan[sgroup], t * kStage + skey);
        byte = 127;
        raw = u32x4(0);
      }
      if (!WIDE && __builtin_expect(byte < kFp16Low || byte > kFp16High, 0)) s_wide = 1;
      const float s = mx_scale(byte);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        lds.v[st][skey * 16 + ((4 * sgroup + q) ^ (2 * (skey & 7)))] = WIDE ? mx_bf16x8(raw[q], s) : mx_f16x8(raw[q], s);
    } else {
      const float s = mx_scale(byte);
#pragma unroll
      for (int q = 0; q < 4; ++q) lds.k[st][skey * 16 + ((4 * sgroup + q) ^ (skey & 15))] = mx_bf16x8(raw[q], s);
    }
  };

  float m, l;
  // once a row's maximum is_far, the wave's tiles take the masked way, where the scale is applied first
  bool far;
  float mul;  // the scale, or 1
  int open;  // keys that all of the wave's rows see
  f32x16 o[4];
  // V^T reads: in each 16 lanes lane r addresses key r / 4 (of the four from 4 half) and columns 4 (r % 4)
  const int vr = lane & 15, vkey = 4 * half + (vr >> 2), vg = (lane >> 4) & 1;
  const char* const vbytes = reinterpret_cast<const char*>(&lds.v[0][0]);

  auto tile = [&](auto wide_tag, int st, int key0, int kb, bool masked) {
    constexpr bool WIDE = decltype(wide_tag)::value;
    f32x16 y = {};
    const u32x4* krow = &lds.k[st][(32 * kb + l31) * 16];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const bf16x8 kop = __builtin_bit_cast(bf16x8, krow[(2 * c + half) ^ (l31 & 15)]);
      if constexpr (kPairs) y = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kop, qlo[c], y, 0, 0, 0);
      y = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kop, qop[c], y, 0, 0, 0);
    }
    if (masked) {
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = key0 + 8 * (i >> 2) + 4 * half + (i & 3) < row_lim ? y[i] : -__builtin_inff();
      if (far) y *= scale_size(args_again<PrefillArgs>().scale_log2);
    }
    float e[16], sum = 0.0f;
    auto weigh = [&] {
      sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(y[i], mul, -m));
        sum += e[i];
      }
    };
    weigh();
    if (__builtin_expect(__any(!(sum <= kShareMost)), 0)) {  // (NaN scores come here too)
      float top = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, y[i]);
      top *= mul;
      top = __builtin_fmaxf(top, __shfl_xor(top, 32));
      if (!is_far(top)) top -= kHeadRoom;  // (a far one's steps may be wider than that)
      const float mn = __builtin_fmaxf(m, top);
      const float f = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] *= f;
      if (!far && __any(is_far(mn))) {
        far = true;
        open = 0;
        y *= mul;
        mul = 1.0f;
      }
      weigh();
    }
    l += sum;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      bf16x8 bh, bl;
      f16x8 fh, fl;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (WIDE) {
          bh[i] = __bf16(e[8 * u + i]);
          bl[i] = __bf16(e[8 * u + i] - float(bh[i]));
        } else {
          fh[i] = _Float16(e[8 * u + i]);
          if constexpr (P_PAIRS) fl[i] = _Float16(e[8 * u + i] - float(fh[i]));
        }
      }
      const int key = 32 * kb + 16 * u + vkey;
      const char* vrow = vbytes + st * int(sizeof(lds.v[0])) + 256 * key + 8 * (vr & 1);
      const int sw = 2 * (vkey & 7);
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        // (keys eight apart have the same swizzle)
        const char* at = vrow + 16 * ((4 * d + 2 * vg + ((vr & 3) >> 1)) ^ sw);
        const s16x4 t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
        const s16x4 t1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + 256 * 8));
        const auto v = __builtin_shufflevector(t0, t1, 0, 1, 2, 3, 4, 5, 6, 7);
        if constexpr (WIDE) {
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v), bl, o[d], 0, 0, 0);
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v), bh, o[d], 0, 0, 0);
        } else {
          if constexpr (P_PAIRS) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v), fl, o[d], 0, 0, 0);
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v), fh, o[d], 0, 0, 0);
        }
      }
    }
  };

  // The loads of stage t + 1 fly while stage t is computed, and the page ids of t + 2.
  auto stream = [&](auto wide_tag) {
    m = kNoScore;
    l = 0.0f;
    far = false;
    mul = scale_size(p.scale_log2);
    open = w_open;
#pragma unroll
    for (int d = 0; d < 4; ++d) o[d] = f32x16{};
    if (t_from >= t_to) return;
    fetch(t_from, page_id(t_from));
    int32_t next = t_from + 1 < t_to ? page_id(t_from + 1) : -1;
    put_stage(wide_tag, t_from & 1, t_from);
    __syncthreads();
    for (int t = t_from; t < t_to; ++t) {
      const bool more = t + 1 < t_to;
      if (more) {
        fetch(t + 1, next);
        next = t + 2 < t_to ? page_id(t + 2) : -1;
      }
#pragma unroll
      for (int kb = 0; kb < kStage / 32; ++kb) {
        const int key0 = t * kStage + 32 * kb;
        if (key0 < w_end) tile(wide_tag, t & 1, key0, kb, key0 + 32 > open);
      }
      if (more) put_stage(wide_tag, (t + 1) & 1, t + 1);
      __syncthreads();
    }
  };
  if (tid < 4) s_nan[tid] = INT32_MAX;
  if (tid == 4) s_wide = 0;
  __syncthreads();
  stream(std::false_type{});
  if (__builtin_expect(s_wide, 0)) stream(std::true_type{});  // (after the last stage's barrier)

  if (!wave_live) return;
  const float sum = l + __shfl_xor(l, 32);
  float* rec = splits > 1 ? p.records + (((int64_t(idx) * Hkv + h) * splits + split) * kBlock + row) * kRecord : nullptr;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const bool nan = s_nan[d] < row_lim;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f32x4 v = {o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
      if (__builtin_expect(nan, 0)) v = f32x4(__builtin_nanf(""));
      const int col = 32 * d + 8 * q + 4 * half;
      if (!live) continue;
      if (rec) {
        *reinterpret_cast<f32x4*>(rec + col) = v;
        if (col == 0) {
          rec[kHead] = m;
          rec[kHead + 1] = sum;
        }
      } else {
        finish(a, p.out_dtype, SeqRows{w.r.first + w.i0, w.ni}, h, row, col, v, m, sum, row_lim > 0);
      }
    }
  }
}

// The splits of a block joined: half a wave a query row.
__global__ void __launch_bounds__(256) mx4_prefill_merge_kernel(PrefillArgs p) {
  const DecodeArgs& a = p.a;
  const int lane = int(threadIdx.x) & 63;
  const int Hkv = a.num_kv_heads;
  const int job = int(blockIdx.x) / (kBlock / 8), row = (int(blockIdx.x) - job * (kBlock / 8)) * 8 + (int(threadIdx.x) >> 5);
  const int idx = job / Hkv, h = job - idx * Hkv, splits = splits_here(p);
  Where w;
  if (splits == 1 || !block_of(p, idx, lane, w) || row >= w.ni * a.heads) return;
  const int at4 = lane & 31;
  const float* rec = p.records + (int64_t(job) * splits * kBlock + row) * kRecord;
  float top = kNoScore, sum = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < splits; ++s, rec += int64_t(kBlock) * kRecord) {
    const float m = rec[kHead], l = rec[kHead + 1];
    const f32x4 v = *reinterpret_cast<const f32x4*>(rec + 4 * at4);
    const float up = __builtin_fmaxf(top, m);
    const float f0 = __builtin_amdgcn_exp2f(top - up), f1 = __builtin_amdgcn_exp2f(m - up);
    top = up;
    sum = sum * f0 + l * f1;
    o = o * f0 + v * f1;
  }
  const int L = cached_len(a, w.b);
  const bool sees = (a.causal ? L - w.r.n + 1 + w.i0 + row / a.heads : L) > 0;
  finish(a, p.out_dtype, SeqRows{w.r.first + w.i0, w.ni}, h, row, 4 * at4, o, top, sum, sees);
}

// Blocks at most: whole ones, and a partial one a sequence.
int64_t most_blocks(int64_t num_seqs, int64_t total_q, int64_t max_seqlen_q, int64_t tq) {
  return std::min(ceil_div(total_q, tq) + num_seqs - (num_seqs > 0 ? 1 : 0), num_seqs * ceil_div(max_seqlen_q, tq));
}

// How a step's blocks are split.  The host's bound on the blocks counts one for each
// sequence, also for those that go by rows (of up to `rows` query tokens); where fewer blocks
// could be split further, their number decides on the device (splits 0): a chunk of 256
// tokens over 32000 keys beside 31 decode sequences is 4 blocks of up to 36.
struct Splits {
  int64_t blocks, most, splits;
  int64_t groups;   // workgroups of the step
  int64_t joined;   // blocks and kv heads whose splits are joined, at most
  int64_t records;  // of blocks and kv heads, a split each
};
Splits splits_for(int64_t num_seqs, int64_t total_q, int64_t max_seqlen_q, int64_t heads, int64_t num_kv_heads,
                  int64_t max_seq_len, int64_t rows) {
  const int64_t tq = kBlock / heads;
  Splits s;
  s.blocks = most_blocks(num_seqs, total_q, max_seqlen_q, tq);
  s.most = std::min<int64_t>(max_seq_len / kSplitKeys, kMostSplit);
  const int64_t jobs = s.blocks * num_kv_heads;
  s.splits = splits_of(jobs, s.most);
  s.groups = jobs * s.splits;
  s.joined = s.splits > 1 ? jobs : 0;
  s.records = s.splits > 1 ? s.groups : 0;
  const int64_t least = std::max<int64_t>(ceil_div(total_q - num_seqs * rows, tq), 1) * num_kv_heads;
  if (rows > 0 && splits_of(least, s.most) > s.splits) {
    s.splits = 0;
    s.records = std::min<int64_t>(jobs * s.most, kMostSplit);
    s.groups = std::max(jobs, s.records);
    s.joined = std::min<int64_t>(jobs, kMostSplit / 2);
  }
  return s;
}

int64_t order_floats(int64_t num_seqs) { return (2 * num_seqs + 1 + 3) / 4 * 4; }

template <int Q_DT, bool P_PAIRS>
int launch(const PrefillArgs& p, const Splits& s, hipStream_t st) {
  hipLaunchKernelGGL((mx4_prefill_kernel<Q_DT, P_PAIRS>), dim3(unsigned(s.groups)), dim3(kThreads), 0, st, p);
  if (const int e = check_launch("mx4_prefill_kernel launch"); e != PSK_OK || s.joined == 0) return e;
  hipLaunchKernelGGL(mx4_prefill_merge_kernel, dim3(unsigned(s.joined * (kBlock / 8))), dim3(256), 0, st, p);
  return check_launch("mx4_prefill_merge_kernel launch");
}

}  // namespace

namespace psk_detail {

int64_t mx4_prefill_floats(int64_t num_seqs, int64_t total_q, int64_t max_seqlen_q, int64_t num_q_heads,
                           int64_t num_kv_heads, int64_t max_seq_len, int64_t rows) {
  const Splits s = splits_for(num_seqs, total_q, max_seqlen_q, num_q_heads / num_kv_heads, num_kv_heads, max_seq_len, rows);
  return 4 + order_floats(num_seqs) + s.records * kBlock * kRecord;
}

int launch_mx4_prefill(const DecodeArgs& a, const Mx4Prefill& s, float* workspace, hipStream_t st) {
  PrefillArgs p{};
  p.a = a;
  p.num_seqs = int32_t(s.num_seqs);
  p.total_q = int32_t(s.total_q);
  p.tq = kBlock / a.heads;
  p.out_dtype = s.out_dtype;
  p.scale_log2 = s.scale_log2;
  const Splits n = splits_for(s.num_seqs, s.total_q, s.max_seqlen_q, a.heads, a.num_kv_heads, s.max_seq_len, s.most);
  if (n.groups > INT32_MAX / kBlock)
    return fail(PSK_E_ARG, "too many query blocks (%lld x %d kv heads)", (long long)n.blocks, int(a.num_kv_heads));
  p.max_blocks = int32_t(n.blocks);
  p.splits = int32_t(n.splits);
  p.most_splits = int32_t(n.most);
  float* ws = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~uintptr_t(15));
  int32_t* order = reinterpret_cast<int32_t*>(ws);
  p.blocks = order;
  p.order = order + s.num_seqs + 1;
  p.records = ws + order_floats(s.num_seqs);
  hipLaunchKernelGGL(mx4_order_kernel, dim3(1), dim3(1024), 0, st, a, int(s.num_seqs), int(s.total_q), p.tq, s.most, order,
                     order + s.num_seqs + 1);
  if (const int e = check_launch("mx4_order_kernel launch"); e != PSK_OK) return e;
  const bool pairs = s.out_dtype != PSK_DTYPE_BF16;
  switch (s.q_dtype) {
    case PSK_DTYPE_BF16:
      return pairs ? launch<PSK_DTYPE_BF16, true>(p, n, st) : launch<PSK_DTYPE_BF16, false>(p, n, st);
    case PSK_DTYPE_F16: return pairs ? launch<PSK_DTYPE_F16, true>(p, n, st) : launch<PSK_DTYPE_F16, false>(p, n, st);
    default: return pairs ? launch<PSK_DTYPE_F32, true>(p, n, st) : launch<PSK_DTYPE_F32, false>(p, n, st);
  }
}

}  // namespace psk_detail
