// Attention of a tree of drafted tokens over the paged FP8 E4M3FN cache for
// MI355X (gfx950).
//
// Sequence b of L cached tokens has n drafted tokens, its last n; drafted token
// i sees every key before them and the drafted keys t whose bit of its mask is
// set.  Otherwise as the readers of paged_attention.hip and prefill_runs.hip:
// q~ = e4m3(q / qd), s = softmax_scale qd kd (q~ . K), out = vd softmax(s) V,
// lse = log sum exp s, Q K^T on the bf16 MFMA over exactly converted FP8
// operands, P V on the fp16 MFMA with V exact, float32 sums.  For a bf16 out P is
// rounded once (2^-11, below what the output's own rounding leaves); for a float32 one
// it is the sum of two fp16 (2^-22) and P V runs twice: 110 / 115 us for the 32 trees
// below, 148 / 197 for four wide ones (prefill_runs.hip).
//
// The n G query rows of a kv head (G query heads each) are rows of MFMA tiles,
// 32 to a workgroup.  Its four waves hold all of them and take the 32-key
// tiles of the keys in turn, each with a ring of LDS slots of its own that
// global_load_lds fills, so nothing but the merge of the four at the end of a
// piece of work waits on a barrier.
//   * S^T = K Q^T is eight v_mfma_f32_32x32x16_bf16 a tile and 32 rows: lane l
//     reads key l % 32's 64 bytes at d = 64 (l / 32), the query operand has the
//     same order of d, and the lane is left with query row l % 32 and keys
//     8 (i / 4) + 4 (l / 32) + i % 4, i < 16.
//   * P V is eight v_mfma_f32_32x32x16_f16: the lane's weights i = 8 u .. 8 u + 7
//     are the P^T operand of step u as they stand, and ds_read_b64_tr_b8 gives
//     the V^T operand of the same keys: in each 16-lane group, lane i's byte j is
//     byte i % 8 of the eight that lane 2 j + i / 8 addressed.
//   * a key's 128 bytes lie in a slot as eight 16-byte chunks, chunk c of key t at
//     c ^ (t & 7), which spreads both kinds of reads over the banks.
// A row's maximum is raised only when the weights of a tile pass 2^15 in sum, so
// that every weight is a finite fp16 value and the common path has no rescale, and to
// kHeadRoom below the tile's largest.
//
// The work is cut into equal runs over sequences and kv heads (cached_queries.h).
// A run's piece that is not all of a job's keys leaves a partial record (maxima,
// sums, float32 accumulators); merge_tree_kernel deals a job's records, in the order
// of their keys, to four waves in turn and joins the four sums.  Short contexts are
// not cut (kWholeKeys), and wide trees over much work run in prefill_runs.hip
// (kWideRows).
//
// What bounds it, and what it measured: 32 trees of 16 tokens over contexts of 512 to
// 16384 (32 query heads over 8), 113 us, the loads' latency (3.2 TB/s of K and V, each
// of which goes to LDS once for either row block, the second time from L2); 48 ragged trees over up to 6000 keys (8 heads over one)
// 27 us and one of 8 over 1000 15 us, the chain lengths - page ids - keys and the
// merge.  A tile of 32 keys and 32 rows costs 512 matrix cycles and 156 vector
// instructions, 64 of them the conversion of K and V to bf16 and fp16; the two hardly
// overlap at two waves a SIMD (1400 cycles a tile), and three do not fit the registers.
//
// C ABI: include/pipeswift_kv.h.  Nothing here allocates or synchronizes.

#include <algorithm>

#include "cached_queries.h"
#include "prefill_runs.h"

using namespace psk_detail;

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows = 32;                  // query rows of a workgroup
constexpr int kStepShift = 7;
constexpr int kTile = 32;                  // keys of a tile
constexpr uint32_t kHalfSlot = kTile * 128;  // bytes of a tile's K (its V follows)
constexpr uint32_t kSlot = 2 * kHalfSlot;
constexpr int kRing = 2;
// units (of kStepKeys keys) that a piece costs beside its keys: 1, 4, 6, 12 gave 35.5,
// 29.7, 28.4, 27.4 us for the ragged trees above and 113, 114, 114, 120 for the 32
constexpr int kOver = 6;
// units a run has at least: a shorter one is another record to merge.  4, 6, 8 gave 19,
// 20, 20 us for 8 tokens over 4000 keys (8 heads over one), 21, 21, 22 over 16000 (32
// over 8), 26, 25, 23 for 30 tokens over 30000 (8 over one) and 22, 28, 23 for 16
// trees of 8 over 100 to 4000
constexpr int kMinRun = 4;
// Up to this many keys a workgroup takes all of a job's and nothing is merged: four
// sequences of 8 tokens (32 query heads over 8), us, whole / cut: 1000 keys 17 / 19, 1600
// 19 / 19, 2500 24 / 21; 64 sequences of 1000, 32 / 38.
constexpr int kWholeKeys = 1536;
// Wide trees over much work go to prefill_runs.hip, whose waves share each key's
// conversion (here every 32 rows convert it again) at 15 us more for its start and
// end: from kWideRows rows a sequence on average and kWideWork query rows x keys on,
// by the bounds of both.  This kernel / that one, us (32 query heads): 4 sequences of 30000 keys over
// 4 kv heads, 24 tokens each 75 / 80, 32: 88 / 87, 48: 126 / 120, 64: 157 / 134; 16 of
// 8000 over 8, 32 tokens 95 / 110, 48: 157 / 138; 32 of 2000, 32 tokens 64 / 60, 48:
// 100 / 74; one of 16000, 64 tokens 38 / 55; uncut (kWholeKeys), 64 of 1500 over 4 kv
// heads, 24 tokens 73 / 74, 32: 87 / 72; 128 of 500 over 8, 60 tokens 216 / 141.
constexpr int kWideRows = 192;
constexpr int64_t kWideWork = 80000000;
constexpr int kPages = 1024;               // page ids a piece stages at a time
constexpr int kSlab = 4096 + 64;           // floats of 32 rows' partial result: accumulators, maxima, sums
constexpr int kMaxSlots = 512;             // resident workgroups the workspace is sized for
constexpr int kStepKeys = kTile * kWaves;  // of a step: a tile a wave
static_assert(kStepKeys == 1 << kStepShift, "");
static_assert(kPages >= kStepKeys + 1, "a step's pages fit, whatever the page size");

struct TreeArgs {
  DecodeArgs a;
  JobSpace s;
  double scale_log2;     // softmax_scale * log2(e)
  const int64_t* mask;
  int64_t mask_stride;   // words from a query token's mask to the next one's
  int32_t row_blocks;    // workgroups that share a run's keys, from max_seqlen_q (those past a job's own rows have nothing to do)
  int32_t whole;         // a workgroup takes all of a job's keys, and nothing is merged
  float* records;        // [max_runs][row_blocks][2][kSlab]
};

__device__ __forceinline__ float* record(const TreeArgs& p, int64_t run, int block, int slot) {
  return p.records + ((run * p.row_blocks + block) * 2 + slot) * kSlab;
}

// A tile's eight loads (see load_lds): K rows 8 u .. 8 u + 7 from kp[u] + 1024 u
// to slot + 1024 u, V rows behind them.  An instruction's offset counts for both
// its addresses, so the LDS base is set once for K and once for V.
__device__ __forceinline__ void load_tile(uint32_t slot, const uint8_t* const (&kp)[4], const uint8_t* const (&vp)[4],
                                          uint32_t offset) {
  uint32_t m0;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\ts_nop 0\n\t"
      "global_load_lds_dwordx4 %3, %4\n\t"
      "global_load_lds_dwordx4 %3, %5 offset:1024\n\t"
      "global_load_lds_dwordx4 %3, %6 offset:2048\n\t"
      "global_load_lds_dwordx4 %3, %7 offset:3072\n\t"
      "s_mov_b32 m0, %2\n\ts_nop 0\n\t"
      "global_load_lds_dwordx4 %3, %8\n\t"
      "global_load_lds_dwordx4 %3, %9 offset:1024\n\t"
      "global_load_lds_dwordx4 %3, %10 offset:2048\n\t"
      "global_load_lds_dwordx4 %3, %11 offset:3072\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(m0)
      : "s"(slot), "s"(slot + kHalfSlot), "v"(offset), "s"(kp[0]), "s"(kp[1]), "s"(kp[2]), "s"(kp[3]), "s"(vp[0]),
        "s"(vp[1]), "s"(vp[2]), "s"(vp[3])
      : "memory");
}

template <int OUT_DT>
__device__ __forceinline__ void store4(char* dst, f32x4 v) {
  if constexpr (OUT_DT == PSK_DTYPE_F32) {
    *reinterpret_cast<f32x4*>(dst) = v;
  } else {
    using E = Elt<PSK_DTYPE_BF16>;
    *reinterpret_cast<u32x2*>(dst) = u32x2{uint32_t(E::from_f32(v[0])) | (uint32_t(E::from_f32(v[1])) << 16),
                                           uint32_t(E::from_f32(v[2])) | (uint32_t(E::from_f32(v[3])) << 16)};
  }
}

// Four columns (of group c = 4 d + i: 32 d + 8 i + 4 (lane / 32)) of output row
// `row` of a job, and its lse once; zeros and -inf where the sum is 0.
template <int OUT_DT>
__device__ __forceinline__ void finish(const TreeArgs& p, const SeqRows& r, int b, int h, int row, int c, int lane, f32x4 o,
                                       float m, float sum) {
  const DecodeArgs& a = p.a;
  const int i = row / a.heads, hq = h * a.heads + row - i * a.heads;
  if (i >= r.n) return;
  const bool any = sum != 0.0f;  // (a NaN sum counts)
  const float f = any ? descale(a.vd, a.vd_b, a.vd_h, b, h) / sum : 0.0f;
  const f32x4 v = any ? o * f : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int col = 8 * c + 4 * (lane >> 5);
  store4<OUT_DT>(a.out + (int64_t(r.first) + i) * a.out_tok_stride + int64_t(hq) * a.out_head_stride +
                     col * Elt<OUT_DT>::kSize, v);
  if (a.lse && c == 0 && lane < 32)
    a.lse[int64_t(hq) * a.lse_head_stride + r.first + i] =
        any ? (m + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f : -__builtin_inff();
}

template <int Q_DT, int OUT_DT, bool GEN>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2)))
tree_attention_kernel(TreeArgs args) {
  constexpr bool kPairs = OUT_DT == PSK_DTYPE_F32;  // P as fp16 pairs
  __shared__ __attribute__((aligned(1024))) char s_ring[kWaves * kRing * kSlot];
  __shared__ int32_t s_pages[kPages];
  __shared__ u32x4 s_q[kRows * 8];  // the rows' e4m3 queries, chunk c of row r at c ^ (r & 7)
  __shared__ float s_m[kWaves][kRows], s_l[kWaves][kRows];
  __shared__ uint32_t s_nan[kHead];  // of each column the rows that see a NaN value
  __shared__ int s_nans;
  const int tid = int(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, kk = lane & 31;

  // the row blocks of a run, which read the same keys, are next to each other on its XCD
  const int w = int(blockIdx.x), idx = (w >> 3) / args.row_blocks, block = (w >> 3) - idx * args.row_blocks;
  SeqWindow seqs;
  int64_t j = 0, x, x_end, before = 0;  // the run, its units, the units before the sequence
  int b;
  if (args.whole) {  // a workgroup a job
    const int jobs = args.s.num_seqs * args.s.heads, per = (jobs + 7) >> 3;
    const int job = (w & 7) * per + idx;
    if (job >= jobs) return;
    b = job / args.s.heads;
    seqs.load(args.a, args.s, b & ~63, lane);
    if (lane_value(seqs.n, b - seqs.b0) == 0) return;
    const int64_t cost = args.s.over + key_steps(args.s, lane_value(seqs.len, b - seqs.b0));
    x = (job - b * args.s.heads) * cost;
    x_end = x + cost;
  } else {
    const StepRuns step_run = step_runs(args.a, args.s, seqs, lane);
    j = xcd_run(step_run, w & 7, idx);
    x = j * step_run.run;
    if (x >= step_run.total) return;
    x_end = min(x + step_run.run, step_run.total);
    b = seq_of_unit(args.a, args.s, x, seqs, lane, before);
  }

  const uint32_t ring = (uint32_t)(size_t)(lvoid*)s_ring + uint32_t(wave * kRing) * kSlot;
  // loads: lane l takes chunk position l % 8 of keys 8 u + l / 8
  const int lr = lane >> 3, lchunk = 16 * ((lane & 7) ^ lr);
  // reads (see above)
  uint32_t rd_k[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) rd_k[q] = uint32_t(128 * kk + 16 * ((4 * half + q) ^ (kk & 7)));
  const int vr = lane & 15, vg = (lane >> 4) & 1;
  const int vkey = 8 * (vr >> 3) + 4 * half + ((vr >> 1) & 3);  // of each 16
  uint32_t rd_v[4];
#pragma unroll
  for (int d = 0; d < 4; ++d)
    rd_v[d] = kHalfSlot + uint32_t(128 * vkey + 16 * ((2 * d + vg) ^ (vkey & 7)) + 8 * (vr & 1));

  while (x < x_end) {  // over the run's jobs
    const TreeArgs& p = args_again<TreeArgs>();
    const DecodeArgs& a = p.a;
    if (!seqs.holds(b)) seqs.load(a, p.s, b, lane);
    const SeqRows r{lane_value(seqs.first, b - seqs.b0), lane_value(seqs.n, b - seqs.b0)};
    const int L = lane_value(seqs.len, b - seqs.b0);
    const int steps = key_steps(p.s, L);
    const int64_t job_cost = p.s.over + steps;
    const int64_t seq_end = before + (r.n > 0 ? job_cost * p.s.heads : 0);
    if (x >= seq_end) {
      before = seq_end;
      ++b;
      continue;
    }
    const int h = int(uniform_div(x - before, job_cost));
    const int64_t at = before + h * job_cost;
    const int64_t hi = min(x_end, at + job_cost);
    const Piece c = piece_of(p.s, x - at, hi - at);
    x = hi;
    const int row0 = block * kRows;
    if ((c.from >= c.to && !p.whole) || row0 >= r.n * a.heads) continue;

    // The queries: every thread quantizes 16 elements of a row, and the waves
    // read the rows' bytes from LDS.  The pages of the first keys are on their
    // way meanwhile.
    const int first_page = page_index(a, c.from * kStepKeys);
    int32_t page0 = -1;
    if (first_page + tid < a.bt_width) page0 = a.block_table[int64_t(b) * a.bt_stride + first_page + tid];
    const int ctx = L - r.n;
    const int row = row0 + kk, i0 = row / a.heads;
    const bool live = i0 < r.n;
    const int64_t* mask = p.mask + (int64_t(r.first) + (live ? i0 : 0)) * p.mask_stride;
    QueryBytes<Q_DT> qb;
    {
      const int qr = row0 + (tid >> 3), qi = qr / a.heads;
      qb.load(qi < r.n ? a.q + (int64_t(r.first) + qi) * a.q_tok_stride +
                             int64_t(h * a.heads + qr - qi * a.heads) * a.q_head_stride
                       : nullptr, 16 * (tid & 7));
    }
    const float qd = descale(a.qd, a.qd_b, a.qd_h, b, h);
    const float sl_signed = score_scale(p.scale_log2, qd, descale(a.kd, a.kd_b, a.kd_h, b, h));
    const float sl = __builtin_fabsf(sl_signed);  // a negative scale is applied as -q~ (exact)
    __syncthreads();  // readers of the ring, the marks (the last piece's merge), the ids and the queries are done
    s_q[(tid >> 3) * 8 + ((tid & 7) ^ ((tid >> 3) & 7))] = qb.quantized(qd, sl_signed < 0.0f ? 0x80808080u : 0u);
    if (tid < kHead) s_nan[tid] = 0;
    if (tid == 0) s_nans = 0;

    float m = live ? kNegBig : -kNegBig, l = 0.0f;  // rows without a token keep every weight at 0
    f32x16 o[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) o[d] = f32x16{};
    bf16x8 qop[8];

    const uint8_t* kbase = a.k + int64_t(h) * a.k_head;
    const uint8_t* vbase = a.v + int64_t(h) * a.v_head;
    const int64_t v_from_k = vbase - kbase;
    const uint32_t off = uint32_t(lr * a.k_row) + lchunk;
    const int n_tiles = (L + kTile - 1) / kTile;
    const int t_mask = max(ctx, 0) / kTile;  // tiles from here on need masks
    const int steps_per_window = int(min(int64_t(kPages - 1) * a.block_size / kStepKeys, int64_t(1) << 24));

    for (int s0 = c.from; s0 < c.to; s0 += steps_per_window) {
      const int s1 = min(c.to, s0 + steps_per_window);
      // the pages of the window's keys, missing ones as -1
      const int p0 = page_index(a, s0 * kStepKeys);
      const int p1 = page_index(a, int(min(int64_t(L), int64_t(s1) * kStepKeys)) - 1);
      if (s0 > c.from) __syncthreads();  // the ids before these are done with
      for (int i = tid; i <= p1 - p0; i += kThreads) {
        int32_t id = page0;
        if (s0 > c.from || i >= kThreads) {
          id = -1;
          if (p0 + i < a.bt_width) id = a.block_table[int64_t(b) * a.bt_stride + p0 + i];
        }
        s_pages[i] = id < a.num_blocks ? id : -1;
      }
      __syncthreads();
      if (s0 == c.from) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const u32x4 x = s_q[kk * 8 + ((4 * half + t) ^ (kk & 7))];
          qop[2 * t] = e4m3x8_to_bf16(x[0], x[1]);
          qop[2 * t + 1] = e4m3x8_to_bf16(x[2], x[3]);
        }
      }

      const int t_end = min(kWaves * s1, n_tiles);
      bool full = true;  // the newest tile's loads are all in flight
      // GEN: every lane looks its four keys' pages up.  Else eight keys of one
      // load share a page: lane 4 k + u holds where load u of tile win + 4 k
      // begins in a kv head's K, for sixteen tiles at a time, and the addresses are scalar.
      int win = 0;
      int64_t at = 0;
      uint64_t whole8 = 0, some8 = 0;  // loads whose eight keys are all cached; whose first is
      auto look_up = [&](int t) {
        const DecodeArgs& a = args_again<TreeArgs>().a;
        win = t;
        const int key = (t + kWaves * (lane >> 2)) * kTile + 8 * (lane & 3);
        int32_t id = -1;
        int pi = 0;
        if (key < L && t + kWaves * (lane >> 2) < t_end) {
          pi = page_index(a, key);
          id = s_pages[pi - p0];
        }
        const int64_t row = key - pi * a.block_size;
        at = int64_t(id) * a.k_blk + row * a.k_row - 1024 * (lane & 3);
        some8 = __ballot(id >= 0);
        whole8 = __ballot(id >= 0 && key + 8 <= L);
      };
      auto issue = [&](int t, uint32_t slot) {
        if constexpr (GEN) {
          int32_t id[4], row[4];
          bool all = true;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int key = t * kTile + 8 * u + lr;
            const int pi = page_index(a, key);
            row[u] = key - pi * a.block_size;
            id[u] = key < L ? s_pages[pi - p0] : -1;
            all = all && id[u] >= 0;
          }
          full = __all(all);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (full || id[u] >= 0) {
              load_lds(slot + 1024 * u, kbase + lchunk + (int64_t(id[u]) * a.k_blk + int64_t(row[u]) * a.k_row));
              load_lds(slot + kHalfSlot + 1024 * u, vbase + lchunk + (int64_t(id[u]) * a.v_blk + int64_t(row[u]) * a.v_row));
            } else {
              *lds_at<u32x4>(slot + 1024 * u + 16 * lane) = u32x4(0);
              *lds_at<u32x4>(slot + kHalfSlot + 1024 * u + 16 * lane) = u32x4(0);
            }
          }
        } else {
          if (t - win >= 16 * kWaves) look_up(t);
          const int k = t - win;  // lane of the tile's first load
          const uint8_t* kp[4];
          const uint8_t* vp[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            kp[u] = kbase + lane_value(at, k + u);
            vp[u] = kp[u] + v_from_k;
          }
          full = ((whole8 >> k) & 15) == 15;
          if (__builtin_expect(full, 1)) {
            load_tile(slot, kp, vp, off);
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              if (((some8 >> (k + u)) & 1) && t * kTile + 8 * u + lr < L) {
                load_lds(slot + 1024 * u, kp[u] + 1024 * u, off);
                load_lds(slot + kHalfSlot + 1024 * u, vp[u] + 1024 * u, off);
              } else {
                *lds_at<u32x4>(slot + 1024 * u + 16 * lane) = u32x4(0);
                *lds_at<u32x4>(slot + kHalfSlot + 1024 * u + 16 * lane) = u32x4(0);
              }
            }
          }
        }
      };

      // NaN values of keys that some row does not see (0 x NaN) must not reach
      // it: they leave the tile, and the (column, row) pairs that do see one are
      // marked, for the end of the piece.
      auto contain_nan = [&](i32x2 (&vraw)[8], uint32_t vis) {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) any |= nan_bytes(uint32_t(vraw[i][0])) | nan_bytes(uint32_t(vraw[i][1]));
        if (__builtin_expect(!__any(any != 0), 1)) return;
        uint32_t rows[4] = {0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll 1
          for (int j = 0; j < 8; ++j) {  // byte j: key 16 u + 8 (j / 4) + 4 half + j % 4
            const uint64_t see = __ballot((vis >> (16 * u + 8 * (j >> 2) + (j & 3))) & 1u);
            const uint32_t mine = half ? uint32_t(see >> 32) : uint32_t(see);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              const int word = j < 4 ? vraw[4 * u + d][0] : vraw[4 * u + d][1];
              rows[d] |= ((uint32_t(word) >> (8 * (j & 3))) & 0x7Fu) == 0x7Fu ? mine : 0u;
            }
          }
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            vraw[4 * u + d][0] &= int(~(nan_bytes(uint32_t(vraw[4 * u + d][0])) * 0xFFu));
            vraw[4 * u + d][1] &= int(~(nan_bytes(uint32_t(vraw[4 * u + d][1])) * 0xFFu));
          }
        }
#pragma unroll
        for (int d = 0; d < 4; ++d)
          if (rows[d]) atomicOr(&s_nan[32 * d + kk], rows[d]);
        s_nans = 1;
      };

      // One tile: its operands leave the slot for registers, the loads of the
      // tile after the next one start into it, and then it is computed.
      auto attend = [&](auto masked_tag, int t, uint32_t slot, const auto& refill) {
        constexpr bool MASKED = decltype(masked_tag)::value;
        u32x4 kraw[4];
        i32x2 vraw[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) kraw[q] = *lds_at<u32x4>(slot + rd_k[q]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          vraw[i] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(lds_at<i32x2>(slot + rd_v[i & 3] + uint32_t(2048 * (i >> 2))));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        refill();
        f32x16 y = {};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          y = __builtin_amdgcn_mfma_f32_32x32x16_bf16(e4m3x8_to_bf16(kraw[q][0], kraw[q][1]), qop[2 * q], y, 0, 0, 0);
          y = __builtin_amdgcn_mfma_f32_32x32x16_bf16(e4m3x8_to_bf16(kraw[q][2], kraw[q][3]), qop[2 * q + 1], y, 0, 0, 0);
        }
        uint32_t vis = 0xFFFFFFFFu;
        if constexpr (MASKED) {
          vis = (live ? visible(mask, ctx, r.n, t * kTile) : 0u) >> (4 * half);
          contain_nan(vraw, vis);
        }
        auto sees = [&](int i) { return !MASKED || ((vis >> (8 * (i >> 2) + (i & 3))) & 1u); };
        float w[16], sum = 0.0f;
        auto weigh = [&] {
          sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float e = __builtin_fmaf(y[i], sl, -m);
            w[i] = __builtin_amdgcn_exp2f(sees(i) ? e : -__builtin_inff());
            sum += w[i];
          }
        };
        weigh();
        if (__builtin_expect(__any(!(sum <= 32768.0f)), 0)) {  // (NaN scores come here too)
          float top = -__builtin_inff();
#pragma unroll
          for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, sees(i) ? y[i] : -__builtin_inff());
          top *= sl;
          top = __builtin_fmaxf(top, __shfl_xor(top, 32)) - kHeadRoom;
          const float mn = live ? __builtin_fmaxf(m, top) : m;
          const float f = __builtin_amdgcn_exp2f(m - mn);
          m = mn;
          l *= f;
#pragma unroll
          for (int d = 0; d < 4; ++d) o[d] *= f;
          weigh();
        }
        l += sum;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          f16x8 pop, rest;
#pragma unroll
          for (int i = 0; i < 8; ++i) pop[i] = _Float16(w[8 * u + i]);
          if constexpr (kPairs) {
#pragma unroll
            for (int i = 0; i < 8; ++i) rest[i] = _Float16(__builtin_fmaf(float(pop[i]), -1.0f, w[8 * u + i]));
          }
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const f16x8 v = e4m3x8_to_f16(uint32_t(vraw[4 * u + d][0]), uint32_t(vraw[4 * u + d][1]));
            if constexpr (kPairs) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, rest, o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pop, o[d], 0, 0, 0);
          }
        }
      };

      int t = kWaves * s0 + wave;
      uint32_t slot = ring;
      bool next_full = false;
      if (t < t_end) {
        if constexpr (!GEN) look_up(t);
        issue(t, slot);
        if (t + kWaves < t_end) {
          issue(t + kWaves, slot + kSlot);
          next_full = full;
        }
      }
      auto step = [&](auto masked_tag) {
        // the tile's own loads: the next one's eight may stay in flight
        if (t + kWaves < t_end && next_full) wait_loads<8>(); else wait_loads<0>();
        attend(masked_tag, t, slot, [&] {
          if (t + 2 * kWaves < t_end) {
            issue(t + 2 * kWaves, slot);
            next_full = full;
          }
        });
        slot = slot == ring ? ring + kSlot : ring;
        t += kWaves;
      };
      while (t < min(t_end, t_mask)) step(std::false_type{});
      while (t < t_end) step(std::true_type{});
    }

    const TreeArgs& rest = args_again<TreeArgs>();
    // the four waves' results, joined in the order of the waves
    const float lt = l + __shfl_xor(l, 32);
    if (lane < 32) {
      s_m[wave][lane] = m;
      s_l[wave][lane] = lt;
    }
    __syncthreads();  // every wave has left its ring, and wrote its maxima
    const bool whole = c.from == 0 && c.to == steps;
    float top = s_m[0][kk];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) top = __builtin_fmaxf(top, s_m[v][kk]);
    const float f = __builtin_amdgcn_exp2f(m - top);
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) sum += s_l[v][kk] * __builtin_amdgcn_exp2f(s_m[v][kk] - top);
    f32x4* s_o = reinterpret_cast<f32x4*>(s_ring);  // [kWaves][16][64]
    static_assert(sizeof(s_ring) >= kWaves * 16 * 64 * sizeof(f32x4), "the accumulators fit the ring");
#pragma unroll
    for (int q = 0; q < 16; ++q)
      s_o[(wave * 16 + q) * 64 + lane] =
          f32x4{o[q >> 2][4 * (q & 3)], o[q >> 2][4 * (q & 3) + 1], o[q >> 2][4 * (q & 3) + 2], o[q >> 2][4 * (q & 3) + 3]} * f;
    __syncthreads();
    float* rec = record(rest, j, block, c.from == 0 ? 1 : 0);
#pragma unroll
    for (int i = 0; i < 16 / kWaves; ++i) {
      const int q = wave + kWaves * i;
      f32x4 v = s_o[q * 64 + lane];
#pragma unroll
      for (int u = 1; u < kWaves; ++u) v += s_o[(u * 16 + q) * 64 + lane];
      if (__builtin_expect(s_nans, 0)) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if ((s_nan[8 * q + 4 * half + k] >> kk) & 1u) v[k] = __builtin_nanf("");
      }
      if (whole) finish<OUT_DT>(rest, r, b, h, row, q, lane, v, top, sum);
      else *reinterpret_cast<f32x4*>(rec + (q * 64 + lane) * 4) = v;
    }
    if (!whole && wave == 0 && lane < 32) {
      rec[4096 + lane] = top;
      rec[4096 + 32 + lane] = sum;
    }
  }
}

// The records of a job joined: a workgroup per 32 rows and 32 columns of a job.  Its
// waves take the records in turn, so that as many as possible are in flight, and
// then a group of 8 columns each, over the four parts in order.
template <int OUT_DT>
__global__ void __launch_bounds__(256) merge_tree_kernel(TreeArgs p) {
  const DecodeArgs& a = p.a;
  __shared__ f32x4 s_o[4][4][64];
  __shared__ float s_m[4][kRows], s_l[4][kRows];
  const int lane = int(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int kk = lane & 31;
  const uint32_t tasks = uint32_t(p.s.num_seqs) * uint32_t(p.s.heads) * uint32_t(p.row_blocks) * 4;  // (host: below 2^26)
  for (uint32_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    // column groups 4 c .. 4 c + 3 of row block `block` of job (b, h)
    const int c = int(task & 3);
    const uint32_t rest = task >> 2, job = rest / uint32_t(p.row_blocks);
    const int block = int(rest - job * uint32_t(p.row_blocks));
    const int b = int(job / uint32_t(p.s.heads)), h = int(job - uint32_t(b) * uint32_t(p.s.heads));
    const SeqRows r = seq_rows(a, p.s.total_q, b);
    const int row = kRows * block + kk;
    if (kRows * block >= r.n * a.heads) continue;
    SeqWindow seqs;
    const StepRuns cost = step_runs(a, p.s, seqs, lane);
    const int64_t before = units_before(a, p.s, b, seqs, lane);
    const int steps = key_steps(p.s, lane_value(seqs.len, b - seqs.b0));
    const int64_t at = before + h * int64_t(p.s.over + steps) + p.s.over;  // the first unit that pays for keys
    const int64_t j0 = uniform_div(at, cost.run), j1 = steps > 0 ? uniform_div(at + steps - 1, cost.run) : j0 - 1;
    if (j0 == j1) continue;  // one run had all the keys and wrote the rows

    float top = kNegBig, sum = 0.0f;
    f32x4 o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int kAhead = 2;  // records of a wave read together
    for (int64_t j = j0 + wave; j <= j1; j += 4 * kAhead) {
      float m[kAhead], l[kAhead];
      f32x4 v[kAhead][4];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int64_t k = min(j + 4 * u, j1);
        const float* rec = record(p, k, block, k == j0 ? 1 : 0);
        m[u] = rec[4096 + kk];
        l[u] = rec[4096 + 32 + kk];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[u][q] = *reinterpret_cast<const f32x4*>(rec + ((4 * c + q) * 64 + lane) * 4);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (j + 4 * u > j1) break;
        const float up = __builtin_fmaxf(top, m[u]);
        const float f0 = __builtin_amdgcn_exp2f(top - up), f1 = __builtin_amdgcn_exp2f(m[u] - up);
        top = up;
        sum = sum * f0 + l[u] * f1;
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = o[q] * f0 + v[u][q] * f1;
      }
    }
    __syncthreads();  // the last task's readers are done
    if (lane < kRows) {
      s_m[wave][lane] = top;
      s_l[wave][lane] = sum;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) s_o[wave][q][lane] = o[q];
    __syncthreads();
    top = s_m[0][kk];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = __builtin_fmaxf(top, s_m[w][kk]);
    sum = 0.0f;
    o[0] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(s_m[w][kk] - top);
      sum += s_l[w][kk] * f;
      o[0] += s_o[w][wave][lane] * f;
    }
    finish<OUT_DT>(p, r, b, h, row, 4 * c + wave, lane, o[0], top, sum);
  }
}

// Workgroups resident at once: two per CU (LDS and registers).
int64_t tree_slots() { return std::min<int64_t>(2 * device_cus(), kMaxSlots); }

struct TreeShape {
  int64_t row_blocks, max_runs;
};
TreeShape tree_shape(int64_t rows, int64_t slots) {
  TreeShape s;
  s.row_blocks = ceil_div(rows, kRows);
  s.max_runs = xcd_rounds(slots / s.row_blocks);
  return s;
}

bool wide_step(int64_t num_seqs, int64_t total_q, int64_t num_q_heads, int64_t num_kv_heads, int64_t max_seq_len) {
  return total_q * (num_q_heads / num_kv_heads) >= kWideRows * num_seqs &&
         double(total_q) * double(num_q_heads) * double(max_seq_len) >= double(kWideWork) && num_seqs <= kOrderMax &&
         num_q_heads / num_kv_heads <= kBlockRows;
}

template <int Q_DT, int OUT_DT>
int launch_tree(const TreeArgs& p, bool general, hipStream_t st) {
  const int64_t jobs = int64_t(p.s.num_seqs) * p.s.heads;
  const dim3 grid{unsigned((p.whole ? ceil_div(jobs, 8) * 8 : p.s.max_runs) * p.row_blocks), 1u, 1u};
  if (general) hipLaunchKernelGGL((tree_attention_kernel<Q_DT, OUT_DT, true>), grid, dim3(kThreads), 0, st, p);
  else hipLaunchKernelGGL((tree_attention_kernel<Q_DT, OUT_DT, false>), grid, dim3(kThreads), 0, st, p);
  if (const int e = check_launch("tree_attention_kernel launch"); e != PSK_OK || p.whole) return e;
  const int64_t groups = std::min<int64_t>(jobs * p.row_blocks * 4, 1 << 20);
  hipLaunchKernelGGL((merge_tree_kernel<OUT_DT>), dim3(unsigned(groups)), dim3(256), 0, st, p);
  return check_launch("merge_tree_kernel launch");
}

// Pages of a multiple of 8 keys whose rows lie within 32-bit offsets (the keys of a
// load share a page), K and V laid out alike.  16 trees of 16 tokens over 8000: pages
// of 16 take 72 us, of 12 with a look-up a lane 85.
bool shares_pages(const DecodeArgs& a) {
  return a.block_size % 8 == 0 && a.k_row >= 0 && 8 * a.k_row < (int64_t(1) << 31) && a.k_row == a.v_row && a.k_blk == a.v_blk;
}

template <int Q_DT>
int launch_tree_q(const TreeArgs& p, int out_dtype, hipStream_t st) {
  const bool general = !shares_pages(p.a);
  return out_dtype == PSK_DTYPE_BF16 ? launch_tree<Q_DT, PSK_DTYPE_BF16>(p, general, st)
                                     : launch_tree<Q_DT, PSK_DTYPE_F32>(p, general, st);
}

}  // namespace

extern "C" {

int64_t psk_paged_tree_workspace_len(int64_t num_seqs, int64_t total_q, int64_t max_seqlen_q, int64_t num_q_heads,
                                     int64_t num_kv_heads, int64_t max_seq_len) {
  if (num_seqs < 0 || total_q < 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads ||
      max_seqlen_q <= 0 || max_seqlen_q > INT32_MAX / (num_q_heads / num_kv_heads) || max_seq_len < 0)
    return PSK_E_ARG;
  const bool wide = wide_step(num_seqs, total_q, num_q_heads, num_kv_heads, max_seq_len);
  if (max_seq_len <= kWholeKeys) return wide ? prefill_runs_words() : 0;
  const TreeShape s = tree_shape(max_seqlen_q * (num_q_heads / num_kv_heads), kMaxSlots);
  const int64_t own = 4 + s.max_runs * s.row_blocks * 2 * kSlab;
  return wide ? std::max(own, prefill_runs_words()) : own;
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
  const int64_t need = psk_paged_tree_workspace_len(num_seqs, total_q, max_seqlen_q, num_q_heads, num_kv_heads, max_seq_len);
  if (workspace_len < need || (need > 0 && !workspace))
    return fail(PSK_E_WORKSPACE, "workspace of %lld floats, need %lld", (long long)workspace_len, (long long)need);
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
  p.scale_log2 = double(softmax_scale) * 1.4426950408889634;
  p.mask = tree_mask;
  p.mask_stride = tree_mask_stride;
  const TreeShape s = tree_shape(max_seqlen_q * a.heads, tree_slots());
  p.s.num_seqs = int32_t(num_seqs);
  p.s.total_q = int32_t(total_q);
  p.s.heads = int32_t(num_kv_heads);
  p.s.step_shift = kStepShift;
  p.s.over = kOver;
  p.s.max_runs = int32_t(s.max_runs);
  p.s.min_run = kMinRun;
  p.s.width = INT32_MAX;
  p.row_blocks = int32_t(s.row_blocks);
  p.whole = max_seq_len <= kWholeKeys;
  if (wide_step(num_seqs, total_q, num_q_heads, num_kv_heads, max_seq_len) && shares_pages(a) &&
      2 * num_kv_heads <= prefill_cus())
    return launch_tree_runs(a, TreeStep{tree_mask, tree_mask_stride, p.scale_log2, int32_t(total_q)}, num_seqs, q_dtype,
                            out_dtype, reinterpret_cast<int32_t*>(workspace), static_cast<hipStream_t>(stream));
  p.records = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~uintptr_t(15));
  constexpr int64_t kMost = (int64_t(1) << 24) - 8;  // workgroups of a launch
  if (std::max(num_seqs * num_kv_heads, s.max_runs) > kMost / s.row_blocks)
    return fail(PSK_E_ARG, "too many rows (%lld sequences of up to %lld drafted tokens)", (long long)num_seqs,
                (long long)max_seqlen_q);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (q_dtype) {
    case PSK_DTYPE_FP8_E4M3FN: return launch_tree_q<PSK_DTYPE_FP8_E4M3FN>(p, out_dtype, st);
    case PSK_DTYPE_BF16: return launch_tree_q<PSK_DTYPE_BF16>(p, out_dtype, st);
    case PSK_DTYPE_F16: return launch_tree_q<PSK_DTYPE_F16>(p, out_dtype, st);
    default: return launch_tree_q<PSK_DTYPE_F32>(p, out_dtype, st);
  }
}

}  // extern "C"
