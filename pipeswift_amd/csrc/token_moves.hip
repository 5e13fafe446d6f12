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
// One workgroup per row of scores (layer, sequence, head).  The k best of the
// free tokens are those above the k-th largest key and the first of those at
// it, found by a radix selection of four 8-bit digits over order-preserving
// integer keys; a scan in position order then lists the kept tokens.

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;

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
};

// Larger scores have larger keys, -0 and 0 the same one, a NaN the least of all.
__device__ __forceinline__ uint32_t score_key(float f) {
  if (__builtin_isnan(f)) return 0u;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix of `x` over the workgroup and its total.  Two barriers.
__device__ __forceinline__ uint32_t block_prefix(uint32_t x, uint32_t* s_wave, uint32_t& total) {
  const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) >> 6;
  uint32_t v = x;
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(v, o);
    if (lane >= o) v += y;
  }
  if (lane == 63) s_wave[wave] = v;
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (int w = 0; w < kSelWaves; ++w) {
    before += w < wave ? s_wave[w] : 0u;
    all += s_wave[w];
  }
  __syncthreads();
  total = all;
  return before + v - x;
}

__global__ void __launch_bounds__(kSelThreads) select_tokens_kernel(SelectArgs p) {
  __shared__ uint32_t s_hist[256];
  __shared__ uint32_t s_wave[kSelWaves];
  __shared__ uint32_t s_pick[2];
  const int tid = int(threadIdx.x);
  const int row = int(blockIdx.x);
  const int head = row % p.heads, b = (row / p.heads) % p.num_seqs, layer = row / p.heads / p.num_seqs;
  const float* src = p.scores + int64_t(layer) * p.s_layer + int64_t(b) * p.s_seq + int64_t(head) * p.s_head;
  float* out = p.out + int64_t(layer) * p.o_layer + int64_t(b) * p.o_seq + int64_t(head) * p.o_head;
  int32_t* kept = p.kept + int64_t(row) * p.budget;
  const int L = min(max(p.seq_lens[b], 0), p.width);
  const int n = min(L, p.budget);
  if (layer == 0 && head == 0 && tid == 0) p.new_lens[b] = n;

  // free tokens: [lo, hi); those before and after are kept
  int lo = L, hi = L;
  uint32_t want = 0;  // how many of the free tokens stay
  uint32_t cut = 0, ties = 0;  // keys above `cut` stay, and the first `ties` at it
  if (L > p.budget) {
    lo = p.sink;
    hi = L - p.recent;
    want = uint32_t(p.budget - p.sink - p.recent);
    uint32_t left = want, prefix = 0;
    for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
      if (tid < 256) s_hist[tid] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += kSelThreads) {
        const uint32_t key = score_key(src[i]);
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s_hist[(key >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        int d = 255;
        uint32_t above = 0;
        while (d > 0 && above + s_hist[d] < left) above += s_hist[d--];
        s_pick[0] = uint32_t(d);
        s_pick[1] = above;
      }
      __syncthreads();
      prefix |= s_pick[0] << shift;
      left -= s_pick[1];
      __syncthreads();
    }
    cut = prefix;
    ties = left;
  }
  uint32_t done = 0, tied = 0;
  for (int i0 = 0; i0 < L; i0 += kSelThreads) {
    const int i = i0 + tid;
    float f = 0.0f;
    uint32_t above = 0, at = 0;
    if (i < L) {
      f = src[i];
      if (i < lo || i >= hi) {
        above = 1;
      } else if (want > 0) {
        const uint32_t key = score_key(f);
        above = key > cut;
        at = key == cut;
      }
    }
    uint32_t tie_total, keep_total;
    const uint32_t tie_rank = tied + block_prefix(at, s_wave, tie_total);
    const uint32_t keep = above | (at & uint32_t(tie_rank < ties));
    const uint32_t rank = done + block_prefix(keep, s_wave, keep_total);
    // (a kept score moves down at most to its own place: the rows before it are read)
    if (keep) {
      kept[rank] = i;
      if (int(rank) < p.out_width) out[rank] = f;
    }
    tied += tie_total;
    done += keep_total;
  }
  __syncthreads();
  for (int i = n + tid; i < min(L, p.out_width); i += kSelThreads) out[i] = 0.0f;
  for (int i = n + tid; i < p.budget; i += kSelThreads) kept[i] = -1;
}

// ---------------------------------------------------------------------------
// the kept rows to their new pages
// ---------------------------------------------------------------------------
//
// Row (slot, head) by row, heads first, V bytes a lane: the destination is
// written in order and every source row is read whole.  A thread takes kMoveRows
// rows at once, so that the chain to a row (kept position, page, row) is waited
// for once for all of them.

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
// columns.

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

int psk_select_tokens(const float* scores, const int64_t* scores_strides, int64_t scores_width, float* scores_out,
                      const int64_t* scores_out_strides, int64_t scores_out_width, const int32_t* seq_lens,
                      int64_t num_layers, int64_t num_seqs, int64_t num_heads, int64_t budget, int64_t sink,
                      int64_t recent, int32_t* kept, int32_t* new_lens, void* stream) {
  begin_device_call();
  if (num_layers < 0 || num_seqs < 0 || num_heads <= 0 || scores_width < 0 || scores_width > INT32_MAX - kSelThreads ||
      scores_out_width < 0 || scores_out_width > INT32_MAX - kSelThreads)
    return fail(PSK_E_ARG, "bad sizes");
  if (budget < 1 || budget > INT32_MAX - kSelThreads) return fail(PSK_E_ARG, "budget %lld", (long long)budget);
  if (sink < 0 || recent < 0 || sink > budget || recent > budget - sink)
    return fail(PSK_E_ARG, "sink %lld and recent %lld do not fit a budget of %lld", (long long)sink, (long long)recent,
                (long long)budget);
  if (num_layers == 0 || num_seqs == 0) return PSK_OK;
  if (num_layers > INT32_MAX || num_seqs > INT32_MAX / num_layers || num_heads > INT32_MAX / (num_layers * num_seqs))
    return fail(PSK_E_ARG, "too many rows of scores");
  if (!scores_strides || !scores_out_strides || !seq_lens || !kept || !new_lens ||
      (scores_width > 0 && !scores) || (scores_out_width > 0 && !scores_out))
    return fail(PSK_E_ARG, "NULL pointer");
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
  hipLaunchKernelGGL(select_tokens_kernel, dim3(unsigned(num_layers * num_seqs * num_heads)), dim3(kSelThreads), 0,
                     static_cast<hipStream_t>(stream), p);
  return check_launch("select_tokens_kernel launch");
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
