// What the kernels that read queries against the paged FP8 cache and take a
// whole batch's lengths from the device share (tree_attention.hip,
// prefill_runs.hip's trees, attention_weights.hip).
#pragma once

#include <atomic>
#include <cmath>

#include "paged_attention.h"
#include "xcd_runs.h"

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
// `align`: bytes that cache rows start on (16 for FP8 rows, 4 for 4-bit ones, which take no FP8 query).
inline int check_cached_queries(const CachedQueries& c, DecodeArgs& a, bool* empty, int align = 16) {
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
  if ((c.q_dtype != PSK_DTYPE_FP8_E4M3FN || align < 16) && c.q_dtype != PSK_DTYPE_BF16 && c.q_dtype != PSK_DTYPE_F16 &&
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
  if (common_align(k_align, 4, align) < align)
    return fail(PSK_E_ARG, "K/V caches need %d-byte aligned bases and strides", align);
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
  a.qd = c.q_descale;
  a.kd = c.k_descale;
  return PSK_OK;
}

// CUs of the current device, asked for once each; 256 where it is not known.
inline int64_t device_cus() {
  static std::atomic<int> known[64];
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 256;
  const bool kept = dev >= 0 && dev < 64;
  if (kept && (cus = known[dev].load(std::memory_order_relaxed)) > 0) return cus;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) return 256;
  if (kept) known[dev].store(cus, std::memory_order_relaxed);
  return cus;
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

// A sequence's length, kept where the arithmetic on whole tiles of it stays in 31 bits.
__device__ __forceinline__ int32_t cached_len(const DecodeArgs& a, int b) {
  return min(max(a.seq_lens[b], 0), INT32_MAX - 1024);
}

// The scale from a product q~ . K to the exp2 domain, rounded once (each rounding
// of it is an error of every score in the same direction).
__device__ __forceinline__ float score_scale(double scale_log2, float qd, float kd) {
  return float(scale_log2 * double(qd) * double(kd));
}

// Visibility of keys key0 .. key0 + 31 (bit k: key0 + k) to a drafted token with mask m, of n after `ctx` keys.
__device__ __forceinline__ uint32_t visible(const int64_t* m, int ctx, int n, int key0) {
  const int j0 = key0 - ctx;  // the drafted index of key0
  if (j0 <= -32) return 0xFFFFFFFFu;
  if (j0 >= n) return 0u;
  const int left = n - j0;  // keys before the tree's end
  const uint32_t in = left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1u;
  if (j0 < 0) return ((uint32_t(m[0]) << -j0) | ((1u << -j0) - 1u)) & in;
  const int w = j0 >> 6, sh = j0 & 63;
  uint64_t bits = uint64_t(m[w]) >> sh;
  if (sh > 32 && left > 64 - sh) bits |= uint64_t(m[w + 1]) << (64 - sh);
  return uint32_t(bits) & in;
}

// A tree row's running maximum is raised to this much (log2) below the largest weight:
// its weights have to stay below 2^16 only, and those of keys far below count in fp16
// down to 2^-33 of the largest, not 2^-25 (the sum counts them all).
constexpr float kHeadRoom = 8.0f;

// Bit 0 of every byte of x that is an e4m3 NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t x) {
  return (((x & 0x7F7F7F7Fu) + 0x01010101u) >> 7) & 0x01010101u;
}

// Sixteen elements of a query row, loaded and then quantized to their e4m3 bytes
// (zeros without a row).
template <int Q_DT>
struct QueryBytes {
  static constexpr int kEsz = Q_DT == PSK_DTYPE_F32 ? 4 : Q_DT == PSK_DTYPE_FP8_E4M3FN ? 1 : 2;
  u32x4 x[kEsz];
  bool live;
  __device__ __forceinline__ void load(const char* src, int d0) {
    live = src != nullptr;
#pragma unroll
    for (int i = 0; i < kEsz; ++i) x[i] = live ? reinterpret_cast<const u32x4*>(src + d0 * kEsz)[i] : u32x4(0);
  }
  __device__ __forceinline__ u32x4 quantized(float qd, uint32_t sign) const {
    u32x4 y;
    if constexpr (Q_DT == PSK_DTYPE_FP8_E4M3FN) {
      y = x[0];
    } else {
      using QC = QuantConv<Q_DT, 16 / kEsz, kNanTorch>;
      const QScale qs = make_qscale(qd);
      uint8_t bytes[16];
#pragma unroll
      for (int i = 0; i < kEsz; ++i) {
        const typename QC::Out z = QC::apply(x[i], qs);
        __builtin_memcpy(bytes + 16 / kEsz * i, &z, 16 / kEsz);
      }
      __builtin_memcpy(&y, bytes, 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = live ? y[i] ^ sign : 0u;
    return y;
  }
};

// A kernel's only argument, read again from where the launch put it: what is used
// between two such calls alone takes no scalar registers outside.
template <class Args>
__device__ __forceinline__ const Args& args_again() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const Args*)p;
}

// ---------------------------------------------------------------------------
// a step's work cut into equal runs
// ---------------------------------------------------------------------------
//
// A job is a kv head of a sequence with query tokens; it costs `over` units and
// one for every step of 1 << step_shift keys.  Jobs follow each other by sequence and head, and
// run j takes the units [j q, (j + 1) q).  Every wave scans the lengths itself,
// 64 sequences at a time and a sequence a lane, so that no launch and no memory
// goes before the kernels and any number of sequences is taken.

struct JobSpace {
  int32_t num_seqs, total_q, heads;  // kv heads
  int32_t step_shift;
  int32_t over;                      // units a job costs beside its keys
  int32_t max_runs;
  int32_t min_run;                   // units a run has at least
  int32_t idle;                      // sequences without query tokens are jobs too
  int32_t width;                     // keys past it cost nothing
  int32_t most = INT32_MAX;          // sequences of more query tokens are no jobs
};

__device__ __forceinline__ int32_t key_steps(const JobSpace& s, int32_t len) {
  return (len + (1 << s.step_shift) - 1) >> s.step_shift;
}

template <class T>
__device__ __forceinline__ T lane_value(T x, int lane) {
  static_assert(sizeof(T) == 4 || sizeof(T) == 8, "");
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(u)), lane));
    const uint32_t hi = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(u >> 32)), lane));
    return __builtin_bit_cast(T, (uint64_t(hi) << 32) | lo);
  }
}

__device__ __forceinline__ int32_t wave_uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t wave_uniform(int64_t x) { return lane_value(x, 0); }

// x / y for 0 <= x, 0 < y, short where both fit 31 bits (they do, but for a huge step).
__device__ __forceinline__ int64_t uniform_div(int64_t x, int64_t y) {
  if (((x | y) >> 31) == 0) return int64_t(wave_uniform(int32_t(uint32_t(x) / uint32_t(y))));
  return wave_uniform(x / y);
}

// 64 consecutive sequences, one a lane: the lane's query rows and length, its
// units over all kv heads, and the units of the window's lanes before it.
struct SeqWindow {
  int32_t b0;
  int32_t first, n, len;
  int64_t cost, before, total;

  __device__ __forceinline__ void load(const DecodeArgs& a, const JobSpace& s, int from, int lane) {
    b0 = from;
    first = n = len = 0;
    if (from + lane < s.num_seqs) {
      const SeqRows r = seq_rows(a, s.total_q, from + lane);
      first = r.first;
      n = r.n <= s.most ? r.n : 0;
      len = cached_len(a, from + lane);
    }
    price(s, lane);
  }
  __device__ __forceinline__ void price(const JobSpace& s, int lane) {
    cost = n > 0 || (s.idle && b0 + lane < s.num_seqs) ? int64_t(s.over + key_steps(s, min(len, s.width))) * s.heads : 0;
    const int64_t v = int64_t(wave_prefix(uint64_t(cost)));
    before = v - cost;
    total = lane_value(v, 63);
  }
  __device__ __forceinline__ bool holds(int b) const { return b >= b0 && b < b0 + 64; }
};

struct StepRuns {
  int64_t total, run;  // units of the step and of a run
};

// The step's units.  `w` is left at the window of sequence 0 where there is but one.
__device__ __forceinline__ StepRuns step_runs(const DecodeArgs& a, const JobSpace& s, SeqWindow& w, int lane) {
  StepRuns c{0, 1};
  for (int b0 = 0; b0 < s.num_seqs; b0 += 64) {
    w.load(a, s, b0, lane);
    c.total += w.total;
  }
  const int64_t even = uniform_div(c.total + s.max_runs - 1, s.max_runs);
  c.run = even > s.min_run ? even : s.min_run;
  return c;
}

// The idx-th run of an XCD.  Workgroup w runs on XCD w % 8, and each XCD takes
// consecutive runs, so that its L2 sees every kv head of a few sequences (one
// head's rows lie a token apart and would fall on a part of its channels).  A run
// past the last comes back as one too.  max_runs is xcd_rounds() of something.
__device__ __forceinline__ int64_t xcd_run(const StepRuns& c, int xcd, int idx) {
  return run_of_xcd(uniform_div(c.total + c.run - 1, c.run), xcd, idx);
}

// The sequence that unit x (below the total) falls in, and the units before it.
__device__ __forceinline__ int seq_of_unit(const DecodeArgs& a, const JobSpace& s, int64_t x, SeqWindow& w, int lane,
                                           int64_t& before) {
  before = 0;
  for (int b0 = 0;; b0 += 64) {
    if (w.b0 != b0) w.load(a, s, b0, lane);
    const int64_t at = before + w.before;
    const uint64_t m = __ballot(at <= x && x < at + w.cost);
    if (m) {
      const int l = __builtin_ctzll(m);
      before = lane_value(at, l);
      return b0 + l;
    }
    before += w.total;
    if (b0 + 64 >= s.num_seqs) return s.num_seqs - 1;  // (not reached: x is below the total)
  }
}

// Units before sequence b; its window is left in `w`.
__device__ __forceinline__ int64_t units_before(const DecodeArgs& a, const JobSpace& s, int b, SeqWindow& w, int lane) {
  int64_t n = 0;
  for (int b0 = 0;; b0 += 64) {
    if (w.b0 != b0) w.load(a, s, b0, lane);
    if (w.holds(b)) return n + lane_value(w.before, b - b0);
    n += w.total;
  }
}

// Steps [from, to) of a job of `steps` that the units [lo, hi) of it pay for.
struct Piece {
  int32_t from, to;
};
__device__ __forceinline__ Piece piece_of(const JobSpace& s, int64_t lo, int64_t hi) {
  return Piece{int32_t(max(lo - s.over, int64_t(0))), int32_t(max(hi - s.over, int64_t(0)))};
}

}  // namespace psk_detail
