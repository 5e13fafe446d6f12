// Cached tokens chosen and moved: the eviction of a cache to a budget
// (selection by score, then the kept rows to fresh pages) and the commit of a
// drafted tree's accepted path.
//
// C ABI: include/pipeswift_kv.h.  Nothing here allocates or synchronizes.

#include <algorithm>

#include "psk_common.h"

using namespace psk_detail;

namespace {

// ---------------------------------------------------------------------------
// selection
// ---------------------------------------------------------------------------
//
// Of a row of scores (layer, sequence, head) the n = `budget` tokens of the
// largest keys stay: those above the n-th largest key and the first of those at
// it.  The keys are order-preserving integers, the first `sink` and the last
// `recent` tokens have the greatest of all, and the n-th is found a digit at a
// time (11, 11 and 10 bits): a histogram of the digit over the keys that agree
// in the digits before, and the bin that it falls in.  A workgroup holds up to
// kChunk keys in registers, sixteen a thread, each wave a contiguous part, so
// that the order is kept with ballots and one exchange between the waves.
//
//   * rows of at most kChunk: select_row_kernel, everything in one launch, with 64
//     registers, 8 values spilled, so that two workgroups of 1024 threads share a CU
//     (73 registers, one of them: 56 us).  512 rows of 12288: 27 us, bound by the histograms'
//     additions; 8 rows of 1100: 7.8 us, the barriers between the digits.
//     Rows of at most 4096 take 256 threads (80 registers, 10 spilled), which wait less at them: 512 rows of
//     4000 and their moves 29 us against 31 with 1024, 2048 of 2000, 74 against 95.
//   * longer ones, a workgroup a chunk: three launches of chunk_digit_kernel
//     leave each chunk's histogram of a digit, and every workgroup of the next
//     launch adds up those of its row; chunk_emit_kernel then has, from the
//     histograms of the chunks before its own, where its kept tokens go.  Four rows
//     of 131072: 34 us, bound by the launches and the histograms; with one workgroup
//     a row 337.  Chunks of 8192: the same, but 15 us more for a row of a million.

constexpr int kSelThreads = 1024;               // (256 for rows of at most 256 kPer)
constexpr int kPer = 16;                        // scores of a thread
constexpr int kChunk = kSelThreads * kPer;
constexpr int kSmallThreads = 256;
constexpr int kBins = 2048;                     // of the first two digits; half of the third's are used
constexpr int kDigits = 3;
constexpr int kCopies = 2;                      // counters of a bin in LDS (see digit_histogram)
using Copies = uint32_t __attribute__((ext_vector_type(kCopies)));
constexpr int kMaxChunks = 4096;                // of one round of launches: bounds the workspace

__device__ __forceinline__ constexpr int digit_shift(int d) { return d == 0 ? 21 : d == 1 ? 10 : 0; }

struct SelectArgs {
  const float* scores;
  int64_t s_layer, s_seq, s_head;
  float* out;
  int64_t o_layer, o_seq, o_head;
  int32_t out_width;
  int32_t width;
  const int32_t* seq_lens;
  int32_t num_seqs, heads;
  int32_t budget, sink, recent;
  int32_t* kept;      // [layers, num_seqs, heads, budget]
  int32_t* new_lens;  // [num_seqs]
  int32_t chunks;     // of a row, at its widest
  int32_t row0;       // first row of the round of launches
  uint16_t* hist;     // [rows of a round][chunks][kDigits][kBins]
  float* staged;      // kept scores where scores_out is scores itself: [rows of a round][budget], else nullptr
};

// Larger scores have larger keys, -0 and 0 the same one, a NaN the least of all;
// between 1 and 0xFF800001.  0: no token there; kForced: one that stays in any case.
constexpr uint32_t kForced = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t score_key(float f) {
  if (__builtin_isnan(f)) return 1u;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return (u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u)) + 1u;
}

struct SelectRow {
  const float* src;
  float* out;
  int32_t* kept;
  int32_t len, n;   // tokens, and how many stay
  int32_t lo, hi;   // the free ones
  uint32_t want;    // n where there is a choice, else 0
};

__device__ __forceinline__ SelectRow select_row(const SelectArgs& p, int row) {
  const int head = row % p.heads, rest = row / p.heads, b = rest % p.num_seqs, layer = rest / p.num_seqs;
  SelectRow r;
  r.src = p.scores + int64_t(layer) * p.s_layer + int64_t(b) * p.s_seq + int64_t(head) * p.s_head;
  r.out = p.out + int64_t(layer) * p.o_layer + int64_t(b) * p.o_seq + int64_t(head) * p.o_head;
  r.kept = p.kept + int64_t(row) * p.budget;
  r.len = min(max(p.seq_lens[b], 0), p.width);
  r.n = min(r.len, p.budget);
  const bool all = r.len <= p.budget;
  r.lo = all ? r.len : p.sink;
  r.hi = all ? r.len : r.len - p.recent;
  r.want = all ? 0u : uint32_t(p.budget);
  return r;
}

// The scores of positions [c0, c0 + kChunk) of a row: wave w's part is `part`
// positions long, lane l of it holds positions c0 + w part + 64 k + l.
template <int NT>
struct Held {
  static constexpr int kWaves = NT / 64;
  float f[kPer];
  uint32_t key[kPer];
  int32_t first, part, end;  // the wave's first position, its length, the chunk's end

  __device__ __forceinline__ void load(const SelectRow& r, int c0) {
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = int(threadIdx.x) & 63;
    end = min(r.len, c0 + NT * kPer);
    part = (max(end - c0, 0) + NT - 1) / NT * 64;
    first = c0 + wave * part;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int i = first + 64 * k + lane;
      f[k] = 0.0f;
      if (64 * k < part && i < end) f[k] = r.src[i];
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int i = first + 64 * k + lane;
      key[k] = 64 * k < part && i < end ? (i < r.lo || i >= r.hi ? kForced : score_key(f[k])) : 0u;
    }
  }
  // fn(k, position) of every place of the wave
  template <class F>
  __device__ __forceinline__ void each(const F& fn) const {
    const int lane = int(threadIdx.x) & 63;
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (64 * k < part) fn(k, first + 64 * k + lane);
  }
};

// The digit histogram of the held keys that agree with `prefix` above it (places
// without a token have the least key, which is never reached), kCopies counters a
// bin, lanes in turn: additions to one place wait for each other.  512 rows of 12288
// and their moves, scores apart / all equal, us: one counter 123 / 188, two 123 / 152,
// four 125 / 136, eight 134 / 137.  Ends with a barrier.
template <int NT>
__device__ __forceinline__ void digit_histogram(const Held<NT>& held, int digit, uint32_t prefix, Copies* hist) {
  const int shift = digit_shift(digit), over = digit == 0 ? 31 : digit_shift(digit - 1);
  const uint32_t mask = digit == 2 ? 1023u : 2047u, copy = threadIdx.x & (kCopies - 1);
  for (int i = int(threadIdx.x); i < kBins; i += NT) hist[i] = Copies(0);
  __syncthreads();
  held.each([&](int k, int) {
    const uint32_t key = held.key[k];
    if (digit == 0 || ((key ^ prefix) >> over) == 0)
      atomicAdd(reinterpret_cast<uint32_t*>(hist) + ((key >> shift) & mask) * kCopies + copy, 1u);
  });
  __syncthreads();
}
__device__ __forceinline__ uint32_t bin_count(const Copies& c) {
  uint32_t n = c[0];
#pragma unroll
  for (int i = 1; i < kCopies; ++i) n += c[i];
  return n;
}

// The bin, from the top, that the left-th key falls in, and the keys above it;
// thread t holds the PER bins from kBins - 1 - PER t down.  1 <= left <= all of them.
struct Digit {
  uint32_t bin, above;
};
// The sum of lanes 0 .. wave - 1's values.
__device__ __forceinline__ uint32_t waves_before(uint32_t x, int wave) {
  const uint32_t v = wave_prefix(x);
  return wave > 0 ? uint32_t(__builtin_amdgcn_readlane(int(v), wave - 1)) : 0u;
}
template <int NT>
__device__ __forceinline__ Digit find_digit(const uint32_t (&n)[kBins / NT], uint32_t left, uint32_t* s_wave,
                                            uint32_t* s_pick) {
  constexpr int PER = kBins / NT;
  const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint32_t own = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) own += n[i];
  const uint32_t x = wave_prefix(own);
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  uint32_t before = x - own + waves_before(lane < NT / 64 ? s_wave[lane] : 0u, wave);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (before < left && left <= before + n[i]) {
      s_pick[0] = uint32_t(kBins - 1 - PER * tid - i);
      s_pick[1] = before;
    }
    before += n[i];
  }
  __syncthreads();
  return Digit{s_pick[0], s_pick[1]};
}

// Lists the kept of the held positions: keys above `cut` and the first `ties` at
// it (of the whole row; `tied` of them and `done` kept tokens come before the
// chunk).  Writes kept positions and their scores.
template <int NT>
__device__ __forceinline__ void emit_kept(const SelectRow& r, const Held<NT>& held, uint32_t cut, uint32_t ties, uint32_t tied,
                                          uint32_t done, float* scores, int32_t scores_width, uint32_t (*s_count)[NT / 64]) {
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = int(threadIdx.x) & 63;
  uint32_t above = 0, at = 0;
  held.each([&](int k, int) {
    above += held.key[k] > cut;
    at += held.key[k] == cut;
  });
  above = wave_prefix(above);
  at = wave_prefix(at);
  if (lane == 63) {
    s_count[0][wave] = above;
    s_count[1][wave] = at;
  }
  __syncthreads();
  // the waves before: all their keys above the cut, and as many at it as there is room for
  const uint32_t room = ties > tied ? ties - tied : 0u;
  const uint32_t before = waves_before(lane < NT / 64 ? s_count[1][lane] : 0u, wave);
  done += waves_before(lane < NT / 64 ? s_count[0][lane] : 0u, wave) + min(before, room);
  tied += before;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  held.each([&](int k, int i) {
    const uint32_t key = held.key[k];
    const uint64_t t = __ballot(key == cut);
    bool keep = key > cut;
    if (t) {
      keep = keep || (key == cut && tied + __popcll(t & below) < ties);
      tied += __popcll(t);
    }
    const uint64_t m = __ballot(keep);
    const uint32_t rank = done + __popcll(m & below);
    done += __popcll(m);
    if (keep) {
      r.kept[rank] = i;
      if (int64_t(rank) < scores_width) scores[rank] = held.f[k];
    }
  });
}

template <int NT>
__global__ void __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(NT == kSelThreads ? 8 : 6)))
select_row_kernel(SelectArgs p) {
  constexpr int PER = kBins / NT;
  __shared__ Copies s_hist[kBins];
  __shared__ uint32_t s_wave[NT / 64], s_count[2][NT / 64], s_pick[2];
  const int tid = int(threadIdx.x), row = p.row0 + int(blockIdx.x);
  const SelectRow r = select_row(p, row);
  if (row < p.num_seqs * p.heads && row % p.heads == 0 && tid == 0) p.new_lens[row / p.heads] = r.n;
  Held<NT> held;
  held.load(r, 0);
  uint32_t prefix = 0, left = r.want;
#pragma unroll 1
  for (int d = 0; d < kDigits && r.want > 0; ++d) {
    digit_histogram<NT>(held, d, prefix, s_hist);
    uint32_t n[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) n[i] = bin_count(s_hist[kBins - 1 - PER * tid - i]);
    const Digit g = find_digit<NT>(n, left, s_wave, s_pick);
    prefix |= g.bin << digit_shift(d);
    left -= g.above;
  }
  __syncthreads();  // (scores_out may be scores: every score is held by now)
  emit_kept<NT>(r, held, prefix, left, 0, 0, r.out, p.out_width, s_count);
  for (int i = r.n + tid; i < min(r.len, p.out_width); i += NT) r.out[i] = 0.0f;
  for (int i = r.n + tid; i < p.budget; i += NT) r.kept[i] = -1;
}

// ---- rows of several chunks

__device__ __forceinline__ uint16_t* chunk_hist(const SelectArgs& p, int row, int chunk, int digit) {
  return p.hist + ((int64_t(row) * p.chunks + chunk) * kDigits + digit) * kBins;
}

// The row's histograms of its first N digits added up, all of them and those of the
// chunks before this one; thread t has bins 2047 - 2 t and 2046 - 2 t, which lie in
// one word.  (The loads of all the digits are in flight together.)
template <int N>
struct RowBins {
  uint32_t all[N][2], mine[N][2];

  __device__ __forceinline__ void load(const SelectArgs& p, const SelectRow& r, int row, int chunk) {
    const uint32_t* hist = reinterpret_cast<const uint32_t*>(chunk_hist(p, row, 0, 0)) + kBins / 2 - 1 - int(threadIdx.x);
    const int n = (r.len + kChunk - 1) / kChunk;
#pragma unroll
    for (int d = 0; d < N; ++d) all[d][0] = all[d][1] = mine[d][0] = mine[d][1] = 0;
#pragma unroll 8
    for (int c = 0; c < n; ++c) {
#pragma unroll
      for (int d = 0; d < N; ++d) {
        const uint32_t w = hist[(int64_t(c) * kDigits + d) * (kBins / 2)];
        all[d][0] += w >> 16;
        all[d][1] += w & 0xFFFFu;
        mine[d][0] += c < chunk ? w >> 16 : 0u;
        mine[d][1] += c < chunk ? w & 0xFFFFu : 0u;
      }
    }
  }
  // Finds digit d's bin of the left-th key; above and at: how many keys of the
  // chunks before this one are above that bin (added) and in it.
  __device__ __forceinline__ Digit find(int d, uint32_t left, uint32_t* s_wave, uint32_t* s_pick, uint32_t& above,
                                        uint32_t& at) const {
    const Digit g = find_digit<kSelThreads>(all[d], left, s_wave, s_pick);
    at = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t bin = uint32_t(kBins - 1 - 2 * int(threadIdx.x) - i);
      above += bin > g.bin ? mine[d][i] : 0u;
      at += bin == g.bin ? mine[d][i] : 0u;
    }
    __syncthreads();  // the pick is read by all before it is made again
    return g;
  }
};

template <int DIGIT>
__global__ void __launch_bounds__(kSelThreads) __attribute__((amdgpu_waves_per_eu(4))) chunk_digit_kernel(SelectArgs p) {
  __shared__ Copies s_hist[kBins];
  __shared__ uint32_t s_wave[kSelThreads / 64], s_pick[2];
  const int chunk = int(blockIdx.x), row = int(blockIdx.y);
  const SelectRow r = select_row(p, p.row0 + row);
  if (r.want == 0 || chunk * kChunk >= r.len) return;
  Held<kSelThreads> held;
  held.load(r, chunk * kChunk);
  uint32_t prefix = 0;
  if constexpr (DIGIT > 0) {
    RowBins<DIGIT> bins;
    bins.load(p, r, row, chunk);
    uint32_t left = r.want, above = 0, at;
#pragma unroll
    for (int d = 0; d < DIGIT; ++d) {
      const Digit g = bins.find(d, left, s_wave, s_pick, above, at);
      prefix |= g.bin << digit_shift(d);
      left -= g.above;
    }
  }
  digit_histogram<kSelThreads>(held, DIGIT, prefix, s_hist);
  const uint32_t w = (bin_count(s_hist[2 * threadIdx.x + 1]) << 16) | bin_count(s_hist[2 * threadIdx.x]);  // (at most kChunk each)
  reinterpret_cast<uint32_t*>(chunk_hist(p, row, chunk, DIGIT))[threadIdx.x] = w;
}

__global__ void __launch_bounds__(kSelThreads) __attribute__((amdgpu_waves_per_eu(4))) chunk_emit_kernel(SelectArgs p) {
  __shared__ uint32_t s_wave[kSelThreads / 64], s_count[2][kSelThreads / 64], s_pick[2];
  const int tid = int(threadIdx.x), chunk = int(blockIdx.x), row = int(blockIdx.y), c0 = chunk * kChunk;
  const SelectRow r = select_row(p, p.row0 + row);
  const int whole = p.row0 + row;
  if (chunk == 0) {
    if (whole < p.num_seqs * p.heads && whole % p.heads == 0 && tid == 0) p.new_lens[whole / p.heads] = r.n;
    for (int i = r.n + tid; i < p.budget; i += kSelThreads) r.kept[i] = -1;
  }
  if (c0 >= r.len) return;
  Held<kSelThreads> held;
  held.load(r, c0);
  // The cut, and of the chunks before this one the keys above it (in each digit
  // those of higher bins that agree before it) and at it.
  uint32_t prefix = 0, left = r.want, above = 0, at = 0;
  if (r.want > 0) {
    RowBins<kDigits> bins;
    bins.load(p, r, row, chunk);
#pragma unroll
    for (int d = 0; d < kDigits; ++d) {
      const Digit g = bins.find(d, left, s_wave, s_pick, above, at);
      prefix |= g.bin << digit_shift(d);
      left -= g.above;
    }
  }
  const int lane = tid & 63;
  above = wave_prefix(above);
  at = wave_prefix(at);
  if (lane == 63) {
    s_count[0][tid >> 6] = above;
    s_count[1][tid >> 6] = at;
  }
  __syncthreads();
  above = waves_before(lane < kSelThreads / 64 ? s_count[0][lane] : 0u, kSelThreads / 64);
  at = waves_before(lane < kSelThreads / 64 ? s_count[1][lane] : 0u, kSelThreads / 64);
  __syncthreads();
  if (r.want == 0) above = uint32_t(c0);  // every token before stays
  float* scores = p.staged ? p.staged + int64_t(row) * p.budget : r.out;
  emit_kept<kSelThreads>(r, held, prefix, left, at, above + min(at, left), scores,
                         p.staged ? p.budget : p.out_width, s_count);
  if (!p.staged)
    for (int i = max(r.n, c0) + tid; i < min(held.end, p.out_width); i += kSelThreads) r.out[i] = 0.0f;
}

// The staged scores to their rows, once every chunk has read its own, and zeros behind them.
__global__ void __launch_bounds__(256) unstage_scores_kernel(SelectArgs p) {
  const int row = int(blockIdx.y);
  const SelectRow r = select_row(p, p.row0 + row);
  const float* from = p.staged + int64_t(row) * p.budget;
  for (int i = int(blockIdx.x) * 256 + int(threadIdx.x); i < min(r.len, p.out_width); i += int(gridDim.x) * 256)
    r.out[i] = i < r.n ? from[i] : 0.0f;
}

// ---------------------------------------------------------------------------
// the kept rows to their new pages
// ---------------------------------------------------------------------------
//
// Row (slot, head) by row, heads first, V bytes a lane: the destination is
// written in order and every source row is read whole.  A thread takes kMoveRows
// rows at once, so that the chain to a row (kept position, page, row) is waited
// for once for all of them.  Bound by HBM: 2048 rows of 8 heads in each of 64
// (layer, sequence) pairs, 537 MB moved, 97 us, 5.5 TB/s (a row a thread through the
// caches: 20 us more).

constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 4;

struct MoveArgs {
  char* cache[2];
  int64_t layer_stride, blk, row, head_stride;  // bytes, of both caches
  int32_t heads, heads_shift;                   // shifts: log2, or -1
  int32_t kept_heads;
  int32_t chunks, chunks_shift;  // vectors of a head's row
  int32_t block_size, block_shift, num_blocks;
  const int32_t* table;
  int64_t table_stride, table_width;
  const int32_t* dst_table;
  int64_t dst_stride, dst_width;
  const int32_t* kept;
  int32_t budget, num_seqs;
};

__device__ __forceinline__ int32_t page_of(const int32_t* table, int64_t stride, int64_t width, int32_t num_blocks, int b,
                                           int64_t pi) {
  if (pi >= width) return -1;
  const int32_t id = table[int64_t(b) * stride + pi];
  return id >= 0 && id < num_blocks ? id : -1;
}

__device__ __forceinline__ uint32_t div_by(uint32_t x, int32_t by, int32_t shift) {
  return shift >= 0 ? x >> shift : x / uint32_t(by);
}

template <int V>
__global__ void __launch_bounds__(kMoveThreads) move_kept_kernel(MoveArgs p) {
  const int b = int(blockIdx.y), layer = int(blockIdx.z);
  const uint32_t rows = uint32_t(p.budget) * uint32_t(p.heads);  // (host: below 2^31)
  const uint32_t per = kMoveThreads;                             // vectors of a pass
  const int64_t items = int64_t(rows) * p.chunks;
  const int32_t* table = p.table + int64_t(b) * p.table_stride;
  const int32_t* dst_table = p.dst_table + int64_t(b) * p.dst_stride;
  const int32_t* lists = p.kept + (int64_t(layer) * p.num_seqs + b) * p.kept_heads * p.budget;
  char* const k = p.cache[0] + int64_t(layer) * p.layer_stride;
  char* const v = p.cache[1] ? p.cache[1] + int64_t(layer) * p.layer_stride : nullptr;
  using T = typename VecT<V>::T;
  for (int64_t x0 = int64_t(blockIdx.x) * per * kMoveRows; x0 < items; x0 += int64_t(gridDim.x) * per * kMoveRows) {
    int32_t from[kMoveRows], slot[kMoveRows];
    int64_t at[kMoveRows];
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      const int64_t x = x0 + u * int64_t(per) + threadIdx.x;
      from[u] = -1;
      slot[u] = 0;
      at[u] = 0;
      if (x < items) {
        // (items fit 32 bits but for budgets of many million tokens)
        const uint32_t r = items <= INT32_MAX ? div_by(uint32_t(x), p.chunks, p.chunks_shift) : uint32_t(x / p.chunks);
        const uint32_t c = uint32_t(x - int64_t(r) * p.chunks);
        const uint32_t i = div_by(r, p.heads, p.heads_shift), h = r - i * uint32_t(p.heads);
        slot[u] = int32_t(i);
        at[u] = int64_t(h) * p.head_stride + int64_t(c) * V;
        from[u] = lists[(p.kept_heads > 1 ? int64_t(h) * p.budget : 0) + i];
      }
    }
    int32_t sp[kMoveRows], dp[kMoveRows];
    uint32_t si[kMoveRows], di[kMoveRows];
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      sp[u] = dp[u] = -1;
      si[u] = di[u] = 0;
      if (from[u] >= 0) {
        si[u] = div_by(uint32_t(from[u]), p.block_size, p.block_shift);
        di[u] = div_by(uint32_t(slot[u]), p.block_size, p.block_shift);
        if (si[u] < p.table_width) sp[u] = table[si[u]];
        if (di[u] < p.dst_width) dp[u] = dst_table[di[u]];
      }
    }
    T kv[kMoveRows], vv[kMoveRows];
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      kv[u] = vv[u] = T(0);
      if (sp[u] >= 0 && sp[u] < p.num_blocks) {
        const int64_t src = at[u] + sp[u] * p.blk + int64_t(uint32_t(from[u]) - si[u] * uint32_t(p.block_size)) * p.row;
        kv[u] = vload_nt<V>(k + src);
        if (v) vv[u] = vload_nt<V>(v + src);
      }
    }
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      if (dp[u] >= 0 && dp[u] < p.num_blocks) {
        const int64_t dst = at[u] + dp[u] * p.blk + int64_t(uint32_t(slot[u]) - di[u] * uint32_t(p.block_size)) * p.row;
        vstore_nt<V>(k + dst, kv[u]);
        if (v) vstore_nt<V>(v + dst, vv[u]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// the accepted path of a drafted tree
// ---------------------------------------------------------------------------
//
// Rows starts[b] + path[b, i] become rows starts[b] + i, of every layer, as a
// snapshot: a workgroup owns some columns of all of a sequence's rows and reads
// every one of them before it writes any.  The shorter the paths, the more
// columns.  Bound by the chain of its three loads: paths of 6 in 32 sequences and 32
// layers (1 KB rows) 4.8 us, of 9 in 8 sequences and 61 layers the same.

constexpr int kCommitRows = 256;  // longest path
constexpr int kCommitThreads = 256;
constexpr int kCommitCols = 8;    // fewest vectors of a row a workgroup owns
constexpr int kCommitItems = kCommitRows * kCommitCols / kCommitThreads;

struct CommitArgs {
  char* cache[2];
  int64_t layer_stride, blk, row;  // bytes
  int32_t chunks;                  // vectors of a row
  int32_t cols_shift;              // log2 of the vectors of a row a workgroup owns
  int32_t block_size, num_blocks;
  const int32_t* table;
  int64_t table_stride, table_width;
  const int32_t* starts;
  const int32_t* path;
  int64_t path_stride;
  int32_t path_width;
  const int32_t* path_lens;
};

template <int V, int ITEMS>
__global__ void __launch_bounds__(kCommitThreads) commit_draft_kernel(CommitArgs p) {
  __shared__ int64_t s_from[kCommitRows], s_to[kCommitRows];
  const int b = int(blockIdx.y), layer = int(blockIdx.z);
  const int tid = int(threadIdx.x);
  const int n = min(max(p.path_lens[b], 0), p.path_width);
  const int64_t start = p.starts[b];
  if (tid < n) {
    const int64_t t = p.path[int64_t(b) * p.path_stride + tid];
    const int64_t s = start + t, d = start + tid;
    int64_t from = -1, to = -1;
    if (t >= 0 && start >= 0 && s != d) {
      const int64_t si = uint64_t(s) / uint32_t(p.block_size), di = uint64_t(d) / uint32_t(p.block_size);
      const int32_t sp = page_of(p.table, p.table_stride, p.table_width, p.num_blocks, b, si);
      const int32_t dp = page_of(p.table, p.table_stride, p.table_width, p.num_blocks, b, di);
      if (sp >= 0 && dp >= 0) {
        from = sp * p.blk + (s - si * p.block_size) * p.row;
        to = dp * p.blk + (d - di * p.block_size) * p.row;
      }
    }
    s_from[tid] = from;
    s_to[tid] = to;
  }
  __syncthreads();
  const int c = (int(blockIdx.x) << p.cols_shift) + (tid & ((1 << p.cols_shift) - 1));
  const int r0 = tid >> p.cols_shift, step = kCommitThreads >> p.cols_shift;
  typename VecT<V>::T v[2][ITEMS];
  const int64_t at = int64_t(layer) * p.layer_stride + int64_t(c) * V;
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int i = r0 + k * step;
    if (c < p.chunks && i < n && s_to[i] >= 0)
      for (int j = 0; j < 2; ++j)
        if (p.cache[j]) v[j][k] = vload<V>(p.cache[j] + at + s_from[i]);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int i = r0 + k * step;
    if (c < p.chunks && i < n && s_to[i] >= 0)
      for (int j = 0; j < 2; ++j)
        if (p.cache[j]) vstore<V>(p.cache[j] + at + s_to[i], v[j][k]);
  }
}

template <int V>
int launch_commit(CommitArgs p, int64_t num_layers, int64_t num_seqs, hipStream_t st) {
  // columns: a power of two, as many as the threads can take with a row each (a
  // row of one pass at least), and no more than the row has
  int shift = log2_exact(kCommitCols);
  while ((2 << shift) * int64_t(p.path_width) <= kCommitThreads && (1 << shift) < p.chunks) ++shift;
  p.cols_shift = shift;
  const dim3 grid{unsigned(ceil_div(p.chunks, 1 << shift)), unsigned(num_seqs), unsigned(num_layers)};
  if (int64_t(p.path_width) << shift <= kCommitThreads)
    hipLaunchKernelGGL((commit_draft_kernel<V, 1>), grid, dim3(kCommitThreads), 0, st, p);
  else
    hipLaunchKernelGGL((commit_draft_kernel<V, kCommitItems>), grid, dim3(kCommitThreads), 0, st, p);
  return check_launch("commit_draft_kernel launch");
}

template <int V>
int launch_move(const MoveArgs& p, int64_t num_layers, int64_t num_seqs, hipStream_t st) {
  const int64_t passes = ceil_div(int64_t(p.budget) * p.heads * p.chunks, kMoveThreads * kMoveRows);
  const dim3 grid{unsigned(std::min<int64_t>(passes, 65535)), unsigned(num_seqs), unsigned(num_layers)};
  hipLaunchKernelGGL((move_kept_kernel<V>), grid, dim3(kMoveThreads), 0, st, p);
  return check_launch("move_kept_kernel launch");
}

}  // namespace

extern "C" {

int64_t psk_select_tokens_workspace_bytes(int64_t num_layers, int64_t num_seqs, int64_t num_heads, int64_t scores_width,
                                          int64_t budget) {
  if (num_layers < 0 || num_seqs < 0 || num_heads <= 0 || scores_width < 0 || budget < 1 || budget > INT32_MAX ||
      scores_width > INT32_MAX || num_layers > INT32_MAX || num_seqs > INT32_MAX || num_heads > INT32_MAX)
    return PSK_E_ARG;
  if (scores_width <= kChunk) return 0;
  const int64_t chunks = ceil_div(scores_width, kChunk);
  const int64_t rows = std::min(std::max<int64_t>(kMaxChunks / chunks, 1), num_layers * num_seqs * num_heads);
  return 16 + rows * (chunks * kDigits * kBins * int64_t(sizeof(uint16_t)) + budget * int64_t(sizeof(float)));
}

int psk_select_tokens(const float* scores, const int64_t* scores_strides, int64_t scores_width, float* scores_out,
                      const int64_t* scores_out_strides, int64_t scores_out_width, const int32_t* seq_lens,
                      int64_t num_layers, int64_t num_seqs, int64_t num_heads, int64_t budget, int64_t sink,
                      int64_t recent, int32_t* kept, int32_t* new_lens, void* workspace, int64_t workspace_bytes,
                      void* stream) {
  begin_device_call();
  if (num_layers < 0 || num_seqs < 0 || num_heads <= 0 || scores_width < 0 || scores_width > INT32_MAX - 2 * kChunk ||
      scores_out_width < 0 || scores_out_width > INT32_MAX - 2 * kChunk)
    return fail(PSK_E_ARG, "bad sizes");
  if (budget < 1 || budget > INT32_MAX - 2 * kChunk) return fail(PSK_E_ARG, "budget %lld", (long long)budget);
  if (sink < 0 || recent < 0 || sink > budget || recent > budget - sink)
    return fail(PSK_E_ARG, "sink %lld and recent %lld do not fit a budget of %lld", (long long)sink, (long long)recent,
                (long long)budget);
  if (num_layers == 0 || num_seqs == 0) return PSK_OK;
  if (num_layers > INT32_MAX || num_seqs > INT32_MAX / num_layers || num_heads > INT32_MAX / (num_layers * num_seqs))
    return fail(PSK_E_ARG, "too many rows of scores");
  if (!scores_strides || !scores_out_strides || !seq_lens || !kept || !new_lens ||
      (scores_width > 0 && !scores) || (scores_out_width > 0 && !scores_out))
    return fail(PSK_E_ARG, "NULL pointer");
  const int64_t need = psk_select_tokens_workspace_bytes(num_layers, num_seqs, num_heads, scores_width, budget);
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(PSK_E_WORKSPACE, "workspace of %lld bytes, need %lld", (long long)workspace_bytes, (long long)need);
  SelectArgs p{};
  p.scores = scores;
  p.s_layer = scores_strides[0];
  p.s_seq = scores_strides[1];
  p.s_head = scores_strides[2];
  p.width = int32_t(scores_width);
  p.out = scores_out;
  p.o_layer = scores_out_strides[0];
  p.o_seq = scores_out_strides[1];
  p.o_head = scores_out_strides[2];
  p.out_width = int32_t(scores_out_width);
  p.seq_lens = seq_lens;
  p.num_seqs = int32_t(num_seqs);
  p.heads = int32_t(num_heads);
  p.budget = int32_t(budget);
  p.sink = int32_t(sink);
  p.recent = int32_t(recent);
  p.kept = kept;
  p.new_lens = new_lens;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t rows = num_layers * num_seqs * num_heads;
  if (need == 0) {
    constexpr int64_t kMostRows = 1 << 20;  // of a launch
    for (int64_t row = 0; row < rows; row += kMostRows) {
      p.row0 = int32_t(row);
      const dim3 grid{unsigned(std::min(kMostRows, rows - row)), 1u, 1u};
      if (scores_width <= kSmallThreads * kPer)
        hipLaunchKernelGGL(select_row_kernel<kSmallThreads>, grid, dim3(kSmallThreads), 0, st, p);
      else
        hipLaunchKernelGGL(select_row_kernel<kSelThreads>, grid, dim3(kSelThreads), 0, st, p);
    }
    return check_launch("select_row_kernel launch");
  }
  p.chunks = int32_t(ceil_div(scores_width, kChunk));
  const int64_t round = std::min(std::max<int64_t>(kMaxChunks / p.chunks, 1), rows);
  p.hist = reinterpret_cast<uint16_t*>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~uintptr_t(15));
  const bool in_place = scores == scores_out;
  if (in_place) p.staged = reinterpret_cast<float*>(p.hist + round * p.chunks * kDigits * kBins);
  for (int64_t row = 0; row < rows; row += round) {
    const unsigned n = unsigned(std::min(round, rows - row));
    p.row0 = int32_t(row);
    const dim3 grid{unsigned(p.chunks), n, 1u};
    hipLaunchKernelGGL(chunk_digit_kernel<0>, grid, dim3(kSelThreads), 0, st, p);
    hipLaunchKernelGGL(chunk_digit_kernel<1>, grid, dim3(kSelThreads), 0, st, p);
    hipLaunchKernelGGL(chunk_digit_kernel<2>, grid, dim3(kSelThreads), 0, st, p);
    hipLaunchKernelGGL(chunk_emit_kernel, grid, dim3(kSelThreads), 0, st, p);
    if (in_place)
      hipLaunchKernelGGL(unstage_scores_kernel, dim3(unsigned(4 * p.chunks), n, 1u), dim3(256), 0, st, p);
    if (const int e = check_launch("chunked selection launch"); e != PSK_OK) return e;
  }
  return PSK_OK;
}

int psk_move_kept_tokens(void* cache0, void* cache1, int64_t layer_stride, int64_t block_stride, int64_t row_stride,
                         int64_t head_stride, int64_t head_bytes, int64_t num_layers, int64_t num_heads,
                         int64_t block_size, int64_t num_blocks, const int32_t* block_table,
                         int64_t block_table_stride, int64_t block_table_width, const int32_t* dst_block_table,
                         int64_t dst_block_table_stride, int64_t dst_block_table_width, const int32_t* kept,
                         int64_t kept_heads, int64_t budget, int64_t num_seqs, void* stream) {
  begin_device_call();
  if (num_layers < 0 || num_layers > 65535 || num_seqs < 0 || num_seqs > 65535)
    return fail(PSK_E_ARG, "%lld layers, %lld sequences (at most 65535 each)", (long long)num_layers, (long long)num_seqs);
  if (num_heads <= 0 || num_heads > INT32_MAX || (kept_heads != 1 && kept_heads != num_heads))
    return fail(PSK_E_ARG, "kept lists of %lld heads for %lld", (long long)kept_heads, (long long)num_heads);
  if (head_bytes <= 0 || head_bytes > INT32_MAX || budget < 1 || budget > INT32_MAX || block_size <= 0 ||
      block_size > INT32_MAX || num_blocks <= 0 || num_blocks > INT32_MAX || block_table_width <= 0 ||
      dst_block_table_width <= 0)
    return fail(PSK_E_ARG, "bad sizes");
  if (num_layers == 0 || num_seqs == 0) return PSK_OK;
  if (!cache0 || !block_table || !dst_block_table || !kept) return fail(PSK_E_ARG, "NULL pointer");
  MoveArgs p{};
  p.cache[0] = static_cast<char*>(cache0);
  p.cache[1] = static_cast<char*>(cache1);
  p.layer_stride = layer_stride;
  p.blk = block_stride;
  p.row = row_stride;
  p.head_stride = head_stride;
  p.heads = int32_t(num_heads);
  p.kept_heads = int32_t(kept_heads);
  p.block_size = int32_t(block_size);
  p.num_blocks = int32_t(num_blocks);
  p.table = block_table;
  p.table_stride = block_table_stride;
  p.table_width = block_table_width;
  p.dst_table = dst_block_table;
  p.dst_stride = dst_block_table_stride;
  p.dst_width = dst_block_table_width;
  p.kept = kept;
  p.budget = int32_t(budget);
  p.num_seqs = int32_t(num_seqs);
  const uint64_t align[7] = {uint64_t(uintptr_t(cache0)), uint64_t(uintptr_t(cache1)), uint64_t(layer_stride),
                             uint64_t(block_stride), uint64_t(row_stride), uint64_t(head_stride), uint64_t(head_bytes)};
  const int v = common_align(align, 7, 16);
  p.chunks = int32_t(head_bytes / v);
  p.chunks_shift = log2_exact(p.chunks);
  p.heads_shift = log2_exact(num_heads);
  p.block_shift = log2_exact(block_size);
  if (budget > INT32_MAX / num_heads) return fail(PSK_E_ARG, "budget %lld of %lld heads", (long long)budget, (long long)num_heads);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (v) {
    case 16: return launch_move<16>(p, num_layers, num_seqs, st);
    case 8: return launch_move<8>(p, num_layers, num_seqs, st);
    case 4: return launch_move<4>(p, num_layers, num_seqs, st);
    case 2: return launch_move<2>(p, num_layers, num_seqs, st);
    default: return launch_move<1>(p, num_layers, num_seqs, st);
  }
}

int psk_commit_draft_tokens(void* cache0, void* cache1, int64_t layer_stride, int64_t block_stride, int64_t row_stride,
                            int64_t row_bytes, int64_t num_layers, int64_t block_size, int64_t num_blocks,
                            const int32_t* block_table, int64_t block_table_stride, int64_t block_table_width,
                            const int32_t* starts, const int32_t* path, int64_t path_stride, int64_t path_width,
                            const int32_t* path_lens, int64_t num_seqs, void* stream) {
  begin_device_call();
  if (num_layers < 0 || num_layers > 65535 || num_seqs < 0 || num_seqs > 65535)
    return fail(PSK_E_ARG, "%lld layers, %lld sequences (at most 65535 each)", (long long)num_layers, (long long)num_seqs);
  if (path_width < 0 || path_width > kCommitRows)
    return fail(PSK_E_ARG, "paths of at most %d tokens (got %lld)", kCommitRows, (long long)path_width);
  if (row_bytes <= 0 || row_bytes > INT32_MAX || block_size <= 0 || block_size > INT32_MAX || num_blocks <= 0 ||
      num_blocks > INT32_MAX || block_table_width <= 0)
    return fail(PSK_E_ARG, "bad sizes");
  if (num_layers == 0 || num_seqs == 0 || path_width == 0) return PSK_OK;
  if (!cache0 || !block_table || !starts || !path || !path_lens) return fail(PSK_E_ARG, "NULL pointer");
  CommitArgs p{};
  p.cache[0] = static_cast<char*>(cache0);
  p.cache[1] = static_cast<char*>(cache1);
  p.layer_stride = layer_stride;
  p.blk = block_stride;
  p.row = row_stride;
  p.block_size = int32_t(block_size);
  p.num_blocks = int32_t(num_blocks);
  p.table = block_table;
  p.table_stride = block_table_stride;
  p.table_width = block_table_width;
  p.starts = starts;
  p.path = path;
  p.path_stride = path_stride;
  p.path_width = int32_t(path_width);
  p.path_lens = path_lens;
  const uint64_t align[6] = {uint64_t(uintptr_t(cache0)), uint64_t(uintptr_t(cache1)), uint64_t(layer_stride),
                             uint64_t(block_stride), uint64_t(row_stride), uint64_t(row_bytes)};
  const int v = common_align(align, 6, 16);
  p.chunks = int32_t(row_bytes / v);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (v) {
    case 16: return launch_commit<16>(p, num_layers, num_seqs, st);
    case 8: return launch_commit<8>(p, num_layers, num_seqs, st);
    case 4: return launch_commit<4>(p, num_layers, num_seqs, st);
    case 2: return launch_commit<2>(p, num_layers, num_seqs, st);
    default: return launch_commit<1>(p, num_layers, num_seqs, st);
  }
}

}  // extern "C"
