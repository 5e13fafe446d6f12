// Attention over the paged 4-bit KV cache for MI355X (gfx950): decode, a few drafted
// tokens, and steps of any number of query tokens.
//
// For query token i of the n of sequence b (its last positions), query head hq of kv
// head h, over the keys j that it sees (j < L - n + 1 + i if causal, else j < L):
//   s_j = softmax_scale (q . K_j),  out = sum_j softmax(s)_j V_j,  lse = log sum_j exp s_j
// K and V as their 4-bit rows stand for (mxfp4.h); a row without a page is zeros; a
// query that sees no key gets zeros and -inf.
//
// The values of a 4-bit row are bf16 values, so K goes to the bf16 matrix
// instructions exactly and a bf16 query does too.  An f16 or f32 query is the sum of
// two bf16 (exact for f16, 2^-17 for f32), for twice the products.  The weights are
// the sum of two bf16 as well (2^-17), since V is only bf16 in general (its scales
// reach 2^126, past fp16's range).  Maxima, sums and accumulators are float32.
//
// A wave takes 16 keys (32 for two sets of query rows or a wider query) of one kv head at
// a time (a tile), for 16 kSets query rows (query tokens x heads of the group):
//   * the workgroup's waves load their tiles together, a stage, 16 bytes a lane by
//     global_load_lds in the order of memory, into a ring of three, two stages ahead.  A
//     row of 68 bytes lies on 4-byte boundaries only, where loads of 16 bytes to
//     registers take a cycle a lane: 64 decode sequences took 223 us with those, 199 with
//     dword loads to LDS by each wave for itself, and take 155-160 like this.
//   * lane l reads a group of 32 elements, 16 bytes, of key l % 16's row at group
//     l / 16, and its scale byte, of K and of V.
//   * S^T = K Q^T on v_mfma_f32_16x16x32_bf16: the lane's group is its part of the A
//     operand of four products as it stands (the query operand has the same order of
//     elements), and leaves query row l % 16 with keys 4 (l / 16) + r of each 16.
//   * V becomes bf16 rows in the wave's own LDS, half of the columns at a time, and comes
//     back transposed by ds_read_b64_tr_b16 as the A operand of O^T = V^T P^T, whose P^T
//     operand is the lane's weights as they stand.
// The waves of a workgroup take `hg` kv heads of the same tokens, so that the rows of a
// token, which share cache lines, are read together, and `1 << wph_shift` waves share a
// head's tiles in turn where the heads are fewer than the waves.  Caches that do not allow
// the joint loads (pages that 8 does not divide, heads apart, other alignments) go to
// registers row by row (GEN).
//
// The work is cut into equal runs over sequences and head groups (cached_queries.h); a
// piece that is not all of a job's keys leaves a partial record, and merge_mx4_kernel
// joins a row's records in the order of their keys.  Short contexts are not cut.
//
// Bound by memory: 64 sequences of 500 to 32 thousand keys, 8 kv heads of 4 query heads,
// read 0.67 GB in a step of 155-160 us, its merge included, 4.2-4.3 TB/s (the loads alone take 138;
// a trace has 158 for this kernel and 9 for the merge).  A
// step of two sequences of 150 and 200 thousand keys takes 57 + 9 us, of which about 23 are the
// start of a run, its first loads and its end.
//
// C ABI: include/pipeswift_kv.h.  Nothing here allocates or synchronizes.

#include <algorithm>

#include "mxfp4_attention.h"
#include "prefill_runs.h"

using namespace psk_detail;

namespace {

constexpr int kRowBytes = int(mx_entry_bytes(kHead));
constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kUnit = 8;           // keys that are loaded together
constexpr uint32_t kUnitGap = 16;  // bytes between units in LDS
constexpr int kSlots = 3;          // stages in LDS
constexpr int kPages = 512;        // page ids a piece stages at a time
constexpr int kMaxSlots = 512;     // resident workgroups the workspace is sized for
// The price of a job's start, in stages of keys: 8 ragged sequences take 32 us at 6, 37 at
// 0; 256 of 1500 keys 116 and 112, 122 at 16.
constexpr int kOver = 6;
// Units of a run, at least: one sequence of 8000 keys takes 25 us at 2, 34 at 1, 27 at 8.
constexpr int kMinRun = 2;
// Up to so many keys a workgroup takes all of a job's: no second kernel, but no balance.
// 1, 64 and 256 sequences of 1024 keys take 15, 25 and 78 us so, 19, 38 and 88 cut; one of
// 4096 keys 35 and 21.  Twice the keys where the jobs are few: 8, 64, 128 sequences of 2048
// take 22, 37, 80 us, 29, 52, 82 cut, but 256 of up to 2048 116 and 92; with 32 query rows 16
// and 64 sequences of 8 kv heads 32 and 62, 46 and 83 cut, but 48 of one kv head 40 and 32.
constexpr int kWholeKeys = 1024;
constexpr int kWholeJobs = 128;
// Workgroups that a step of uncut jobs has, if fewer kv heads a workgroup give them: 128
// sequences of 1024 keys take 50 us with 256, 41 with 512, 43 with 1024; 512 of 256 keys
// 43, 43 and 54.
constexpr int kWholeGroups = 512;
// Query rows that are joined by half waves, whatever their records: sixteen waves a row
// take turns on the CUs (24 sequences of 32 rows x 8 heads: 107 us by them, 32 by half waves).
constexpr int64_t kMergeWide = 1024;
static_assert(kRowBytes == 68, "the reads and loads below");

// Keys of a wave's tile: 16, whose registers (128) and LDS let two workgroups share a CU,
// for 16 query rows of bf16 (one sequence of 1000 keys 16.5 us, 22.5 with 32; the loads
// of a long step no faster); else 32, at one workgroup a CU.
constexpr int tile_shift(int q_dtype, int64_t sets) { return q_dtype == PSK_DTYPE_BF16 && sets == 1 ? 4 : 5; }

struct Mx4Args {
  DecodeArgs a;
  JobSpace s;            // heads: groups of kv heads
  double scale_log2;
  int32_t hg;            // kv heads of a group
  int32_t wph_shift;     // log2 of the waves of a head
  int32_t row_blocks;    // workgroups that share a run's keys, 16 kSets query rows each
  int32_t rows;          // query rows of a record
  int32_t max_rows;      // of a sequence and kv head
  int32_t whole_rows;    // the rows of consecutive tokens follow each other
  int32_t whole;         // a workgroup takes all of a job's keys, and nothing is merged
  int32_t out_dtype;
  float* records;        // [max_runs][row_blocks][2][hg][rows][kHead + 4]
};

__device__ __forceinline__ float* record(const Mx4Args& p, int64_t run, int block, int slot, int hl, int row) {
  return p.records + ((((run * p.row_blocks + block) * 2 + slot) * p.hg + hl) * p.rows + row) * kRecord;
}

// 16 bytes a lane to LDS that nothing reads again (nt).
__device__ __forceinline__ void load_lds_once(uint32_t at, const uint8_t* base, uint32_t offset) {
  uint32_t m0;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3 nt\n\ts_mov_b32 m0, %0"
               : "=&s"(m0) : "s"(at), "v"(offset), "s"(base) : "memory");
}

// Until at most n of this wave's loads are in flight.
__device__ __forceinline__ void wait_stage(int n) {
  switch (n) {
    case 0: wait_loads<0>(); break;
    case 1: wait_loads<1>(); break;
    case 2: wait_loads<2>(); break;
    case 3: wait_loads<3>(); break;
    case 4: wait_loads<4>(); break;
    case 5: wait_loads<5>(); break;
    case 6: wait_loads<6>(); break;
    case 7: wait_loads<7>(); break;
    default: wait_loads<8>(); break;
  }
}

// What a lane reads of its tile: 16 bytes and the scale byte of K and V of a key in each
// 16, dword by dword, since rows lie on 4-byte boundaries, off which LDS takes wider reads slowly.
// Lane group g takes its four dwords from the g-th on, round about (k[u][i]: dword (i + g) %
// 4; the queries and the output columns have that order too): a token's rows are 4 hg
// banks apart (17 hg dwords), and so the lanes of a read, with the gap between the units,
// fall on banks of their own.
template <int kHalves>
struct Rows {
  u32x4 k[kHalves], v[kHalves];
  uint32_t ks[kHalves], vs[kHalves];
};

template <int Q_DT, int kSets, bool GEN>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(tile_shift(Q_DT, kSets) == 4 ? 4 : 2)))
mx4_attention_kernel(Mx4Args args) {
  constexpr bool kPairs = Q_DT != PSK_DTYPE_BF16;
  constexpr int kRows = 16 * kSets;
  constexpr int kTileShift = tile_shift(Q_DT, kSets), kTile = 1 << kTileShift, kHalves = kTile / 16;  // keys of a wave's tile
  constexpr int kStageKeys = kWaves * kTile;                                       // of a stage, a tile a wave
  constexpr uint32_t kSlot = 2 * kStageKeys * kRowBytes + 2 * kStageKeys / kUnit * kUnitGap;  // bytes of a stage
  constexpr int kMostChunks = kHalves == 1 ? 3 : 5;         // 16-byte loads of a wave's part of a unit
  // the stages, and half of a tile's V as bf16 a wave; at the end of a piece the waves' accumulators
  __shared__ __attribute__((aligned(1024))) char s_lds[kSlots * kSlot + kStageKeys * kHead];
  static_assert(sizeof(s_lds) >= kWaves * 8 * 64 * sizeof(f32x4), "");
  __shared__ int32_t s_pages[kPages];
  __shared__ float s_m[kWaves][kRows], s_l[kWaves][kRows];
  __shared__ int32_t s_nan[kWaves][4];  // of each head and group of columns the first key whose V is NaN there
  const int tid = int(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l15 = lane & 15, l4 = lane >> 4;
  const int turn = GEN ? 0 : l4;  // (see Rows)
  const int hl = wave >> args.wph_shift, sub = wave & ((1 << args.wph_shift) - 1), wph = 1 << args.wph_shift;
  const bool active = hl < args.hg;

  // the row blocks of a run, which read the same keys, are next to each other on its XCD
  const int w = int(blockIdx.x), idx = (w >> 3) / args.row_blocks, block = (w >> 3) - idx * args.row_blocks;
  int64_t j = 0, x = 0, x_end = 1;  // the run and its units
  int b0 = 0, whole_grp = 0;        // a window of sequences begins with b0
  int64_t window = 0, before = 0, seq_end = 0;  // units before the window, before the sequence and with it
  int b = 0, L = 0;
  SeqRows r{0, 0};
  // the k-th sequence of a window
  auto take = [&](const SeqWindow& seqs, int64_t at, int k) {
    b = b0 + k;
    before = lane_value(at, k);
    seq_end = before + lane_value(seqs.cost, k);
    r = SeqRows{lane_value(seqs.first, k), lane_value(seqs.n, k)};
    L = lane_value(seqs.len, k);
  };
  if (args.whole) {                 // a workgroup a job: x follows with its sequence
    const int jobs = args.s.num_seqs * args.s.heads, per = (jobs + 7) >> 3;
    const int job = (w & 7) * per + idx;
    if (idx >= per || job >= jobs) return;
    b0 = job / args.s.heads;
    whole_grp = job - b0 * args.s.heads;
  } else {
    SeqWindow seqs;
    const StepRuns step_run = step_runs(args.a, args.s, seqs, lane);
    j = xcd_run(step_run, w & 7, idx);
    x = j * step_run.run;
    if (x >= step_run.total) return;
    x_end = min(x + step_run.run, step_run.total);
    if (args.s.num_seqs <= 64) take(seqs, seqs.before, __builtin_ctzll(__ballot(seqs.before <= x && x < seqs.before + seqs.cost)));
  }

  char* const vt = s_lds + kSlots * kSlot + wave * kTile * kHead;
  const uint32_t ring = uint32_t(size_t((lvoid*)s_lds));
  // V goes through LDS half of its columns at a time (16 of each group, see Rows):
  // key t's 32 bytes of group g at 128 t + 32 (g ^ (t / 2 % 4)), their 16-byte halves swapped
  // where t / 8 is odd, which spreads the writes and the reads over the banks
  const uint32_t wr_v = uint32_t(128 * l15 + 32 * (l4 ^ ((l15 >> 1) & 3)) + 16 * (l15 >> 3));
  // V^T reads: lane i of 16 receives column i of keys 4 l4 .. 4 l4 + 3 of a half tile
  const int vkey = 4 * l4 + (l15 >> 2);
  const uint32_t rd_v = uint32_t(128 * vkey + 16 * (((l15 & 3) >> 1) ^ (vkey >> 3)) + 8 * (l15 & 1));
  const uint32_t rd_sw = 32 * ((vkey >> 1) & 3);

  while (x < x_end) {  // over the run's jobs
    const Mx4Args& p = args_again<Mx4Args>();
    const DecodeArgs& a = p.a;
    if (x >= seq_end) {  // the sequence that x falls in
      SeqWindow seqs;
      seqs.load(a, p.s, b0, lane);
      const int64_t at = window + seqs.before;
      const uint64_t here = p.whole ? uint64_t(lane_value(seqs.n, 0) > 0) : __ballot(at <= x && x < at + seqs.cost);
      if (here == 0) {
        if (p.whole) return;
        window += seqs.total;
        b0 += 64;
        continue;
      }
      take(seqs, at, __builtin_ctzll(here));
    }
    const int steps = key_steps(p.s, L);
    const int64_t job_cost = p.s.over + steps;
    if (p.whole) {
      x = whole_grp * job_cost;
      x_end = x + job_cost;
    }
    const int grp = int(uniform_div(x - before, job_cost));
    const int64_t at = before + grp * job_cost;
    const int64_t hi = min(x_end, at + job_cost);
    const Piece c = piece_of(p.s, x - at, hi - at);
    x = hi;
    const int row0 = block * kRows;
    if ((c.from >= c.to && !p.whole) || row0 >= r.n * a.heads) continue;
    const int h = grp * p.hg + (active ? hl : 0);

    // what each row sees; the keys that all rows see, and that any does
    const int base = a.causal ? L - r.n + 1 : L;
    auto limit = [&](int i) { return a.causal ? min(max(base + i, 0), L) : L; };
    const int key_hi = limit(min((row0 + kRows - 1) / a.heads, r.n - 1)), key_open = limit(row0 / a.heads);
    const float sl_signed = float(p.scale_log2);
    int row_lim[kSets];
    bf16x8 qop[kSets][4], qlo[kPairs ? kSets : 1][4];
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      const int row = row0 + 16 * s + l15, i = row / a.heads;
      const bool live = i < r.n;
      row_lim[s] = live ? limit(i) : 0;
      const char* src = live && active ? a.q + (int64_t(r.first) + i) * a.q_tok_stride +
                                             int64_t(h * a.heads + row - i * a.heads) * a.q_head_stride
                                       : nullptr;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        query8<Q_DT>(src ? src + (32 * l4 + 8 * ((q + turn) & 3)) * Elt<Q_DT>::kSize : nullptr, kPairs && sl_signed < 0.0f,
                     qop[s][q], qlo[kPairs ? s : 0][q]);
    }
    float m[kSets], l[kSets];
    // once a row's maximum is_far, the wave's tiles take the masked way, where the scale is applied first
    bool far = false;
    float mul = scale_size(p.scale_log2);  // or 1
    f32x4 o[kSets][8];
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      m[s] = kNoScore;
      l[s] = 0.0f;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[s][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int first_head = GEN ? h : grp * p.hg;  // of what the wave loads
    const uint8_t* kbase = a.k + int64_t(first_head) * a.k_head;
    const uint8_t* vbase = a.v + int64_t(first_head) * a.v_head;
    const int64_t v_from_k = vbase - kbase;
    // this wave's part of a stage: `segs` units of those of K, then of V (or half a unit),
    // `chunks` 16-byte loads of a lane each; off[i] is where load 64 i + lane lies in a unit
    const uint32_t group_bytes = uint32_t(p.hg * kRowBytes), unit_bytes = kUnit * group_bytes + kUnitGap;
    const int units = kTile / kUnit * wph, segs = max(2 * units / kWaves, 1), shared = max(kWaves / (2 * units), 1);
    const int seg0 = wave * segs / shared, chunks = int(kUnit * group_bytes / 16) / shared, chunk0 = (wave & (shared - 1)) * chunks;
    uint32_t off[kMostChunks];
    if constexpr (!GEN) {
#pragma unroll
      for (int i = 0; i < kMostChunks; ++i) {
        const uint32_t in = 16 * uint32_t(chunk0 + 64 * i + lane), row = in / group_bytes;
        off[i] = p.whole_rows ? in : row * uint32_t(a.k_row) + in - row * group_bytes;
      }
    }
    // where a lane's rows of a stage lie
    const uint32_t rd_rows = hl * kRowBytes + (sub * (kTile / kUnit) + (l15 >> 3)) * unit_bytes + (l15 & 7) * group_bytes;
    uint32_t rd_dword[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) rd_dword[i] = rd_rows + 16 * l4 + 4 * ((i + turn) & 3);
    const int wph_shift = p.wph_shift;
    const int step_keys = 1 << p.s.step_shift;
    const int steps_per_window = int(min(int64_t(kPages - 1) * a.block_size / step_keys, int64_t(1) << 24));

    for (int s0 = c.from; s0 < c.to || s0 == c.from; s0 += steps_per_window) {
      const int s1 = min(c.to, s0 + steps_per_window);
      const int p0 = page_index(a, s0 * step_keys);
      __syncthreads();  // the ids, the marks and the results before these are done with
      bool hole = false;
      if (s0 < s1 && L > 0) {
        const int p1 = page_index(a, int(min(int64_t(L), int64_t(s1) * step_keys)) - 1);
        for (int i = tid; i <= p1 - p0; i += kThreads) {
          int32_t id = -1;
          if (p0 + i < a.bt_width) id = a.block_table[int64_t(b) * a.bt_stride + p0 + i];
          const bool gone = id < 0 || id >= a.num_blocks;
          s_pages[i] = gone ? -1 : id;
          hole = hole || gone;
        }
      }
      if (s0 == c.from && tid < kWaves * 4) s_nan[tid >> 2][tid & 3] = INT32_MAX;
      const bool holes = __syncthreads_or(hole) != 0;  // missing pages among them
      if (!kPairs && s0 == c.from && sl_signed < 0.0f) {  // (here, so that nothing waits for the queries before)
#pragma unroll
        for (int s = 0; s < kSets; ++s) {
#pragma unroll
          for (int q = 0; q < 4; ++q) qop[s][q] = -qop[s][q];
        }
      }

      const int t_end = min(s1 << wph_shift, (key_hi + kTile - 1) / kTile);
      const int s_end = (t_end + wph - 1) >> wph_shift;
      int t_mask = far ? 0 : key_open / kTile;  // tiles from here on need masks
      // What is not cached loads from the first page and is dropped by attend().  Unless
      // GEN, a unit's keys share a page: lane units k + u holds where unit u of stage win + k
      // begins, for 64 / units stages at a time.
      int win = 0;
      int64_t at_unit = 0;
      uint64_t some = 0;  // units whose first key is cached
      auto look_up = [&](int st) {
        win = st;
        const int key = (st << p.s.step_shift) + lane * kUnit;
        int id = -1, pi = 0;
        if (key < L && key < t_end * kTile) {
          pi = page_index(a, key);
          id = s_pages[pi - p0];
        }
        at_unit = id >= 0 ? int64_t(id) * a.k_blk + int64_t(key - pi * a.block_size) * a.k_row : 0;
        some = __ballot(id >= 0);
      };
      // Starts a stage's loads and returns which units of the wave's tile are cached.
      auto issue = [&](int st, uint32_t slot) -> uint32_t {
        int k = (st - win) * units;
        if (k + units > 64) {
          look_up(st);
          k = 0;
        }
        for (int i = 0; i < segs; ++i) {
          const int unit = seg0 + i, ku = unit >= units ? unit - units : unit;
          const uint8_t* from = kbase + lane_value(at_unit, k + ku) + (unit >= units ? v_from_k : 0);
          const uint32_t to = slot + ku * unit_bytes + (unit >= units ? kSlot / 2 : 0) + 16 * chunk0;
#pragma unroll
          for (int c0 = 0; c0 < kMostChunks; ++c0) {
            if (64 * c0 < chunks) {
              if (64 * c0 + lane < chunks) load_lds_once(to + 1024 * c0, from, off[c0]);
            }
          }
        }
        return uint32_t(some >> (k + sub * (kTile / kUnit)));
      };
      // One tile.  `there`: which of its units are cached.
      auto read = [&](uint32_t slot, Rows<kHalves>& y) {
#pragma unroll
        for (int u = 0; u < kHalves; ++u) {
          const uint32_t k0 = slot + 2 * u * unit_bytes;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y.k[u][i] = *lds_at<volatile uint32_t>(rd_dword[i] + k0);
            y.v[u][i] = *lds_at<volatile uint32_t>(rd_dword[i] + k0 + kSlot / 2);
          }
          y.ks[u] = *lds_at<volatile uint8_t>(rd_rows + kCodes + l4 + k0);
          y.vs[u] = *lds_at<volatile uint8_t>(rd_rows + kCodes + l4 + k0 + kSlot / 2);
        }
      };
      // GEN: the lane's rows of a tile straight to registers
      auto fetch = [&](int t, Rows<kHalves>& y) {
#pragma unroll
        for (int u = 0; u < kHalves; ++u) {
          const int key = t * kTile + 16 * u + l15;
          const bool in = key < L && t < t_end;
          const int pi = page_index(a, in ? key : 0);
          const int id = in ? s_pages[pi - p0] : -1;
          const int64_t row = id >= 0 ? key - pi * a.block_size : 0, page = id >= 0 ? id : 0;
          const uint8_t* kr = kbase + (page * a.k_blk + row * a.k_row);
          const uint8_t* vr = vbase + (page * a.v_blk + row * a.v_row);
          y.k[u] = *reinterpret_cast<const u32x4_any*>(kr + 16 * l4);
          y.v[u] = *reinterpret_cast<const u32x4_any*>(vr + 16 * l4);
          y.ks[u] = kr[kCodes + l4];
          y.vs[u] = vr[kCodes + l4];
        }
      };
      auto attend = [&](int t, Rows<kHalves>& y, uint32_t there, bool masked) {
        if (__builtin_expect(masked || holes, 0)) {  // (rows behind the last key hold anything)
#pragma unroll
          for (int u = 0; u < kHalves; ++u) {
            const int key = t * kTile + 16 * u + l15;
            bool gone = key >= L;
            if constexpr (GEN) gone = gone || s_pages[page_index(a, key) - p0] < 0;
            else gone = gone || !((there >> (2 * u + (l15 >> 3))) & 1);
            if (gone) {
              y.ks[u] = y.vs[u] = 127;
              y.k[u] = y.v[u] = u32x4(0);
            }
          }
        }
        // Values that are not finite must not reach rows that do not see their key (0 x NaN):
        // they become zeros, and the end of the piece gives NaN to the rows that do
        if (__builtin_expect(__any(max(y.vs[0], y.vs[kHalves - 1]) >= 253u), 0)) {
#pragma unroll
          for (int u = 0; u < kHalves; ++u) {
            if (mx_not_finite(y.v[u], y.vs[u])) {
              atomicMin(&s_nan[hl][l4], t * kTile + 16 * u + l15);
              y.vs[u] = 127;
              y.v[u] = u32x4(0);
            }
          }
        }
        // a lane group's dwords 2 w and 2 w + 1 (of its order) to LDS
        auto put_v = [&](int w) {
#pragma unroll
          for (int u = 0; u < kHalves; ++u) {
            const float s = mx_scale(y.vs[u]);
            *reinterpret_cast<u32x4*>(vt + 2048 * u + wr_v) = mx_bf16x8(y.v[u][2 * w], s);
            *reinterpret_cast<u32x4*>(vt + 2048 * u + (wr_v ^ 16)) = mx_bf16x8(y.v[u][2 * w + 1], s);
          }
        };
        put_v(0);
        const bool was_far = far;
        float sc[kSets][4 * kHalves];
#pragma unroll
        for (int u = 0; u < kHalves; ++u) {
          bf16x8 kop[4];
          const float s = mx_scale(y.ks[u]);
#pragma unroll
          for (int q = 0; q < 4; ++q) kop[q] = __builtin_bit_cast(bf16x8, mx_bf16x8(y.k[u][q], s));
#pragma unroll
          for (int e = 0; e < kSets; ++e) {
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (kPairs) {
#pragma unroll
              for (int q = 0; q < 4; ++q) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop[q], qlo[e][q], acc, 0, 0, 0);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop[q], qop[e][q], acc, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[e][4 * u + i] = acc[i];
          }
        }
        typedef __bf16 Weights __attribute__((ext_vector_type(4 * kHalves)));
        Weights ph[kSets], pl[kSets];
#pragma unroll
        for (int e = 0; e < kSets; ++e) {
          if (masked) {
#pragma unroll
            for (int i = 0; i < 4 * kHalves; ++i)
              sc[e][i] = t * kTile + 16 * (i >> 2) + 4 * l4 + (i & 3) < row_lim[e] ? sc[e][i] : -__builtin_inff();
            if (was_far) {
              const float sl = scale_size(args_again<Mx4Args>().scale_log2);
#pragma unroll
              for (int i = 0; i < 4 * kHalves; ++i) sc[e][i] *= sl;
            }
          }
          float pv[4 * kHalves], sum = 0.0f;
          auto weigh = [&] {
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4 * kHalves; ++i) {
              pv[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e][i], mul, -m[e]));
              sum += pv[i];
            }
          };
          weigh();
          if (__builtin_expect(__any(!(sum <= kShareMost)), 0)) {  // (NaN scores come here too)
            float top = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < 4 * kHalves; ++i) top = __builtin_fmaxf(top, sc[e][i]);
            top *= mul;
            top = __builtin_fmaxf(top, __shfl_xor(top, 16));
            top = __builtin_fmaxf(top, __shfl_xor(top, 32));
            const float mn = __builtin_fmaxf(m[e], top);
            const float f = __builtin_amdgcn_exp2f(m[e] - mn);
            m[e] = mn;
            l[e] *= f;
#pragma unroll
            for (int d = 0; d < 8; ++d) o[e][d] *= f;
            if (!far && __any(is_far(mn))) {  // (this set's scores and those of the sets that follow)
              far = true;
              t_mask = 0;
#pragma unroll
              for (int x = e; x < kSets; ++x) {
#pragma unroll
                for (int i = 0; i < 4 * kHalves; ++i) sc[x][i] *= mul;
              }
              mul = 1.0f;
            }
            weigh();
          }
          l[e] += sum;
#pragma unroll
          for (int i = 0; i < 4 * kHalves; i += 2) {
            const bf16x2 hi = __builtin_convertvector((f32x2{pv[i], pv[i + 1]}), bf16x2);
            const f32x2 left = {pv[i] - float(hi[0]), pv[i + 1] - float(hi[1])};
            const bf16x2 lo = __builtin_convertvector(left, bf16x2);
            ph[e][i] = hi[0];
            ph[e][i + 1] = hi[1];
            pl[e][i] = lo[0];
            pl[e][i + 1] = lo[1];
          }
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (w == 1) put_v(1);  // (behind the reads of the first half: LDS works a wave's accesses in order)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const char* from = vt + (rd_v + (rd_sw ^ (32 * g)));
            auto get = [&](const char* at) {
              return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
            };
            f32x4* const acc = &o[0][2 * g + w];
            if constexpr (kHalves == 2) {
              const s16x4 t0 = get(from), t1 = get(from + 2048);
              const bf16x8 v = __builtin_bit_cast(bf16x8, __builtin_shufflevector(t0, t1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
              for (int e = 0; e < kSets; ++e) {
                acc[8 * e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pl[e], acc[8 * e], 0, 0, 0);
                acc[8 * e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, ph[e], acc[8 * e], 0, 0, 0);
              }
            } else {
              const s16x4 v = get(from);
#pragma unroll
              for (int e = 0; e < kSets; ++e) {
                acc[8 * e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(v, __builtin_bit_cast(s16x4, pl[e]), acc[8 * e], 0, 0, 0);
                acc[8 * e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(v, __builtin_bit_cast(s16x4, ph[e]), acc[8 * e], 0, 0, 0);
              }
            }
          }
        }
      };

      const int stage_loads = segs * ((chunks + 63) >> 6);
      // (the builtin would wait for the loads too, which the compiler does not see)
      auto barrier = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
      // Stage st is computed while st + 1 and st + 2 are on their way.  The barrier says that
      // every wave's loads of st are there, and that none still reads st - 1's slot, which
      // st + 2 takes.
      if constexpr (GEN) {
        int t = (s0 << wph_shift) + sub;
        if (active && t < t_end) {
          Rows<kHalves> y;
          fetch(t, y);
#pragma unroll 1
          for (; t < t_end; t += wph) {
            Rows<kHalves> next;
            fetch(t + wph, next);
            attend(t, y, 0, t >= t_mask);
            y = next;
          }
        }
      } else {
        uint32_t slot = kSlot, there = 0, there1 = 0, there2 = 0;  // (slot 1: that of stage s0 - 2)
        look_up(s0);
#pragma unroll 1
        for (int st = s0 - 2; st < s_end; ++st) {
          if (st >= s0) {
            wait_stage(st + 1 < s_end ? stage_loads : 0);
            barrier();
          }
          there2 = 0;
          if (st + 2 < s_end) there2 = issue(st + 2, ring + (slot == 0 ? 2 * kSlot : slot - kSlot));
          const int t = (st << wph_shift) + sub;
          if (st >= s0 && active && t < t_end) {
            Rows<kHalves> y;
            read(ring + slot, y);
            attend(t, y, there, t >= t_mask);
          }
          slot = slot == 2 * kSlot ? 0 : slot + kSlot;
          there = there1;
          there1 = there2;
        }
      }
    }

    // The waves' results through LDS, a set of rows at a time: joined over the waves of a head
    // in their order, and four columns of a row a thread to the output or the run's record.
    const Mx4Args& rest = args_again<Mx4Args>();
    const bool all = c.from == 0 && c.to == steps;
    f32x4* const s_o = reinterpret_cast<f32x4*>(s_lds);  // [kWaves][8][64]
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      l[s] += __shfl_xor(l[s], 16);
      l[s] += __shfl_xor(l[s], 32);
      if (l4 == 0) {
        s_m[wave][16 * s + l15] = m[s];
        s_l[wave][16 * s + l15] = l[s];
      }
    }
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      __syncthreads();  // every wave has left its tiles (or the last set), and wrote its maxima and marks
      const int first = hl << rest.wph_shift;
      float top = m[s];
      if (wph > 1) {
        top = kNoScore;
#pragma unroll 1
        for (int v = 0; v < wph; ++v) top = __builtin_fmaxf(top, s_m[first + v][16 * s + l15]);
      }
      const float f = __builtin_amdgcn_exp2f(m[s] - top);
#pragma unroll
      for (int d = 0; d < 8; ++d) s_o[512 * wave + 64 * d + lane] = o[s][d] * f;
      __syncthreads();
      const int rows = min(max(r.n * rest.a.heads - row0 - 16 * s, 0), 16), items = rest.hg * rows * 32;
#pragma unroll 1
      for (int i = tid; i < items; i += kThreads) {
        const int hr = i >> 5, head = hr / rows, row16 = hr - head * rows, row = 16 * s + row16;
        const int v0 = head << rest.wph_shift;
        // column 4 (i % 32): dword n of group g, which group g of lanes has as its (n - g) % 4-th
        const int g = (i >> 3) & 3, at = ((i >> 1) - (GEN ? 0 : g)) & 3;
        const int from = 64 * (2 * g + (at >> 1)) + 16 * (2 * (at & 1) + (i & 1)) + row16;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        float high = kNoScore, sum = 0.0f;
#pragma unroll 1
        for (int u = 0; u < wph; ++u) {
          v += s_o[512 * (v0 + u) + from];
          high = __builtin_fmaxf(high, s_m[v0 + u][row]);
        }
#pragma unroll 1
        for (int u = 0; u < wph; ++u) sum += s_l[v0 + u][row] * __builtin_amdgcn_exp2f(s_m[v0 + u][row] - high);
        const int i0 = (row0 + row) / rest.a.heads, lim = rest.a.causal ? min(max(L - r.n + 1 + i0, 0), L) : L;
        if (__builtin_expect(s_nan[head][g] < lim, 0)) v = f32x4(__builtin_nanf(""));
        const int col = 4 * (i & 31);
        if (all) {
          finish(rest.a, rest.out_dtype, r, grp * rest.hg + head, row0 + row, col, v, high, sum, lim > 0);
        } else {
          float* rec = record(rest, j, block, c.from == 0 ? 1 : 0, head, row);
          *reinterpret_cast<f32x4*>(rec + col) = v;
          if (col == 0) {
            rec[kHead] = high;
            rec[kHead + 1] = sum;
          }
        }
      }
    }
  }
}

// The records of a query row joined, in the order of their keys: by half a wave every
// other one (kParts 2, where a row has few), or by sixteen waves every 32nd.

template <int kParts>
constexpr int kMergeThreads = kParts == 2 ? 512 : 32 * kParts;

template <int kRows, int kParts>
__global__ void __launch_bounds__(kMergeThreads<kParts>) merge_mx4_kernel(Mx4Args p, int64_t tasks) {
  const DecodeArgs& a = p.a;
  constexpr int kTasks = kMergeThreads<kParts> / 32 / kParts;  // rows of a workgroup
  __shared__ f32x4 s_o[kParts][32];
  __shared__ float s_m[kParts], s_l[kParts];
  const int tid = int(threadIdx.x), lane = tid & 63, part = (tid >> 5) & (kParts - 1), at4 = tid & 31;
  const int kv_heads = p.s.heads * p.hg;
  const int64_t task = int64_t(blockIdx.x) * kTasks + wave_uniform(tid / (32 * kParts));
  if (task >= tasks) return;
  const int64_t job = uniform_div(task, p.max_rows);
  const int row = int(task - job * p.max_rows);
  const int b = int(uniform_div(job, kv_heads)), h = int(job - int64_t(b) * kv_heads);
  // the step's units, and those before sequence b
  SeqWindow seqs;
  int64_t total = 0, before = 0;
  int L = 0;
  SeqRows r{0, 0};
#pragma unroll 1
  for (int b0 = 0; b0 < p.s.num_seqs; b0 += 64) {
    seqs.load(a, p.s, b0, lane);
    if (seqs.holds(b)) {
      before = total + lane_value(seqs.before, b - b0);
      r = SeqRows{lane_value(seqs.first, b - b0), lane_value(seqs.n, b - b0)};
      L = lane_value(seqs.len, b - b0);
    }
    total += seqs.total;
  }
  if (row >= r.n * a.heads) return;  // (with all the waves of the row)
  const int64_t even = uniform_div(total + p.s.max_runs - 1, p.s.max_runs);
  const int64_t run = even > p.s.min_run ? even : p.s.min_run;
  const int steps = key_steps(p.s, L), grp = h / p.hg;
  const int64_t at = before + grp * int64_t(p.s.over + steps) + p.s.over;  // the first unit that pays for keys
  const int64_t j0 = uniform_div(at, run), j1 = steps > 0 ? uniform_div(at + steps - 1, run) : j0 - 1;
  if (j0 == j1) return;  // one run had all the keys and wrote the row
  const int block = row / kRows, in_block = row - block * kRows;
  const bool sees = (a.causal ? L - r.n + 1 + row / a.heads : L) > 0;

  float top = kNoScore, sum = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int kAhead = kParts == 2 ? 4 : 8;  // records read together
#pragma unroll 1
  for (int64_t j = j0 + part; j <= j1; j += kParts * kAhead) {
    float m[kAhead], l[kAhead];
    f32x4 v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t k = min(j + kParts * u, j1);
      const float* rec = record(p, k, block, k == j0 ? 1 : 0, h - grp * p.hg, in_block);
      m[u] = rec[kHead];
      l[u] = rec[kHead + 1];
      v[u] = *reinterpret_cast<const f32x4*>(rec + 4 * at4);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (j + kParts * u > j1) break;
      const float up = __builtin_fmaxf(top, m[u]);
      const float f0 = __builtin_amdgcn_exp2f(top - up), f1 = __builtin_amdgcn_exp2f(m[u] - up);
      top = up;
      sum = sum * f0 + l[u] * f1;
      o = o * f0 + v[u] * f1;
    }
  }
  if constexpr (kParts == 2) {
    const float m1 = __shfl_xor(top, 32), l1 = __shfl_xor(sum, 32), up = __builtin_fmaxf(top, m1);
    const float f0 = __builtin_amdgcn_exp2f(top - up), f1 = __builtin_amdgcn_exp2f(m1 - up);
    f32x4 other;
#pragma unroll
    for (int i = 0; i < 4; ++i) other[i] = __shfl_xor(o[i], 32);
    if (part == 0) finish(a, p.out_dtype, r, h, row, 4 * at4, o * f0 + other * f1, up, sum * f0 + l1 * f1, sees);
  } else {
    s_o[part][at4] = o;
    if (at4 == 0) {
      s_m[part] = top;
      s_l[part] = sum;
    }
    __syncthreads();
    if (part > 1) return;
    // half a wave every other part: lane i has part i's weight
    static_assert(kParts == 32, "");
    const float m = s_m[at4];
    top = m;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, x));
    const float f = __builtin_amdgcn_exp2f(m - top);
    sum = s_l[at4] * f;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) sum += __shfl_xor(sum, x);
    o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < 16; ++u) o += s_o[2 * u + part][at4] * __shfl(f, 2 * u + part);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], 32);
    if (part > 0) return;
    finish(a, p.out_dtype, r, h, row, 4 * at4, o, top, sum, sees);
  }
}

// How a step is laid out, from the bounds that its caller gives (q_dtype -1: the most runs of any).
struct Mx4Shape {
  int64_t sets, row_blocks, rows, hg, groups, wph_shift, tile_shift, max_runs;
  bool whole;
};
Mx4Shape mx4_shape(int64_t num_seqs, int64_t max_seqlen_q, int64_t num_q_heads, int64_t num_kv_heads, int64_t max_seq_len,
                   int q_dtype) {
  Mx4Shape s;
  const int64_t rows = max_seqlen_q * (num_q_heads / num_kv_heads);
  s.sets = rows <= 16 ? 1 : 2;
  s.row_blocks = ceil_div(rows, 16 * s.sets);
  s.rows = std::min<int64_t>(rows, 16 * s.sets);
  s.hg = 1;
  for (int64_t g = 1; g <= 8; ++g)
    if (num_kv_heads % g == 0) s.hg = g;
  s.whole = max_seq_len <= kWholeKeys || (max_seq_len <= 2 * kWholeKeys && (s.sets == 1 || num_seqs * num_kv_heads >= kWholeJobs) &&
             num_seqs * (num_kv_heads / s.hg) * s.row_blocks <= kWholeJobs);
  // uncut: the fewer the jobs, the more waves to a head
  if (s.whole)
    while (s.hg > 1 && num_seqs * (num_kv_heads / s.hg) * s.row_blocks < kWholeGroups) {
      int64_t g = s.hg - 1;
      while (num_kv_heads % g) --g;
      s.hg = g;
    }
  s.groups = num_kv_heads / s.hg;
  s.wph_shift = 0;
  while ((s.hg << (s.wph_shift + 1)) <= kWaves) ++s.wph_shift;
  s.tile_shift = tile_shift(q_dtype, s.sets);
  s.max_runs = xcd_rounds((q_dtype < 0 ? kMaxSlots : std::min<int64_t>((s.tile_shift == 4 ? 2 : 1) * device_cus(), kMaxSlots)) / s.row_blocks);
  return s;
}

// Which kernels a step takes: sequences of few query rows a kv head go by rows, those of
// more by blocks of 256 (mxfp4_prefill.hip), in one launch each.  The products of 17 to 32
// rows take the larger part of a tile's time, and of a block's less than its loads, so
// that blocks win while they fill no more than the CUs: 32 rows x 8 kv heads of 1, 8, 16,
// 24, 48 sequences of 2000 to 4000 keys take 35, 48, 32, 33, 60 us by rows and 25, 40, 42, 58, 111
// by blocks.  Where the sequences' tokens differ, both kernels would run: 48 sequences of 1 to 4
// tokens x 8 heads take 27 us by rows, 46 by both.
enum Way { kRows, kBlocks, kBoth };
struct Route {
  Way way;
  int64_t row_tokens;  // query tokens of a sequence that goes by rows, at most
};
Route route(int64_t num_seqs, int64_t total_q, int64_t max_seqlen_q, int64_t heads, int64_t num_kv_heads) {
  const bool even = num_seqs == 1 || total_q == num_seqs * max_seqlen_q;
  const int64_t few = even && num_seqs * num_kv_heads < 128 ? 16 : 32;
  if (max_seqlen_q * heads <= few || heads > kBlockRows) return {kRows, max_seqlen_q};
  // (more sequences than are ordered by their lengths: all by blocks)
  if (even || heads > few || num_seqs > kOrderMax) return {kBlocks, 0};
  return {kBoth, few / heads};
}

// Whether a workgroup's waves load their heads' rows together, 16 bytes a lane: units of 8
// keys that share a page, K and V laid out alike, the group's heads side by side, all on
// 16-byte boundaries, and within 32-bit offsets.
bool loads_together(Mx4Args& p) {
  const DecodeArgs& a = p.a;
  const int64_t group = p.hg * kRowBytes;
  if (a.k_row != a.v_row || a.k_blk != a.v_blk || (p.hg > 1 && (a.k_head != kRowBytes || a.v_head != kRowBytes))) return false;
  if (a.block_size % kUnit || a.k_row < group || kUnit * a.k_row >= (int64_t(1) << 31)) return false;
  p.whole_rows = a.k_row == group;
  if (!p.whole_rows && group % 16) return false;
  uint64_t align = uint64_t(uintptr_t(a.k)) | uint64_t(uintptr_t(a.v)) | uint64_t(a.k_blk);
  align |= uint64_t(a.k_row) * (p.whole_rows ? kUnit : 1);
  if (p.s.heads > 1) align |= uint64_t(p.hg * a.k_head) | uint64_t(p.hg * a.v_head);  // of a group
  return (align & 15) == 0;
}

// How a cut step's rows are joined (by the records of a row, about), and by how many workgroups.
bool joins_by_halves(const Mx4Shape& s, int64_t jobs, int64_t tasks) { return s.max_runs <= 8 * jobs || tasks > kMergeWide; }
int64_t merge_groups(bool few, int64_t tasks) { return ceil_div(tasks, few ? kMergeThreads<2> / 64 : 1); }

// Workgroups of the rows' kernel.
int64_t row_groups(const Mx4Shape& s, int64_t jobs) { return (s.whole ? ceil_div(jobs, 8) * 8 : s.max_runs) * s.row_blocks; }

template <int Q_DT>
int launch(Mx4Args p, const Mx4Shape& s, hipStream_t st) {
  const bool general = !loads_together(p);
  const int64_t jobs = int64_t(p.s.num_seqs) * p.s.heads;
  const dim3 grid{unsigned(row_groups(s, jobs)), 1u, 1u};
  const dim3 block(kThreads);
  if (s.sets == 1 && general) hipLaunchKernelGGL((mx4_attention_kernel<Q_DT, 1, true>), grid, block, 0, st, p);
  else if (s.sets == 1) hipLaunchKernelGGL((mx4_attention_kernel<Q_DT, 1, false>), grid, block, 0, st, p);
  else if (general) hipLaunchKernelGGL((mx4_attention_kernel<Q_DT, 2, true>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((mx4_attention_kernel<Q_DT, 2, false>), grid, block, 0, st, p);
  if (const int e = check_launch("mx4_attention_kernel launch"); e != PSK_OK || p.whole) return e;
  const int64_t tasks = int64_t(p.s.num_seqs) * p.s.heads * p.hg * p.max_rows;
  const bool few = joins_by_halves(s, jobs, tasks);
  const dim3 merge{unsigned(merge_groups(few, tasks)), 1u, 1u}, threads{unsigned(few ? kMergeThreads<2> : kMergeThreads<32>)};
  if (s.sets == 1 && few) hipLaunchKernelGGL((merge_mx4_kernel<16, 2>), merge, threads, 0, st, p, tasks);
  else if (s.sets == 1) hipLaunchKernelGGL((merge_mx4_kernel<16, 32>), merge, threads, 0, st, p, tasks);
  else if (few) hipLaunchKernelGGL((merge_mx4_kernel<32, 2>), merge, threads, 0, st, p, tasks);
  else hipLaunchKernelGGL((merge_mx4_kernel<32, 32>), merge, threads, 0, st, p, tasks);
  return check_launch("merge_mx4_kernel launch");
}

}  // namespace

extern "C" {

int64_t psk_paged_mxfp4_workspace_len(int64_t num_seqs, int64_t total_q, int64_t max_seqlen_q, int64_t num_q_heads,
                                      int64_t num_kv_heads, int64_t max_seq_len) {
  if (num_seqs < 0 || total_q < 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads ||
      max_seqlen_q <= 0 || max_seqlen_q > INT32_MAX / (num_q_heads / num_kv_heads) || max_seq_len < 0)
    return PSK_E_ARG;
  const Route r = route(num_seqs, total_q, max_seqlen_q, num_q_heads / num_kv_heads, num_kv_heads);
  int64_t own = 0;
  if (r.way != kBlocks) {
    const Mx4Shape s = mx4_shape(num_seqs, r.row_tokens, num_q_heads, num_kv_heads, max_seq_len, -1);
    if (!s.whole) own = 4 + s.max_runs * s.row_blocks * 2 * s.hg * s.rows * kRecord;
  }
  if (r.way == kRows) return own;
  const int64_t blocks = mx4_prefill_floats(num_seqs, total_q, max_seqlen_q, num_q_heads, num_kv_heads, max_seq_len,
                                            r.way == kBoth ? r.row_tokens : 0);
  return std::max(own, blocks);  // (one after the other)
}

int psk_paged_mxfp4_attention(const void* q, int64_t q_tok_stride, int64_t q_head_stride, int q_dtype,
                              const void* k_cache, const void* v_cache, const int64_t* k_strides,
                              const int64_t* v_strides, const int32_t* block_table, int64_t block_table_stride,
                              int64_t block_table_width, const int32_t* seq_lens, int64_t num_seqs, int64_t num_q_heads,
                              int64_t num_kv_heads, int64_t head_size, int64_t block_size, int64_t num_blocks,
                              int64_t max_seq_len, int64_t total_q, int64_t max_seqlen_q, const int32_t* cu_seqlens_q,
                              int causal, float softmax_scale, void* out, int64_t out_tok_stride,
                              int64_t out_head_stride, int out_dtype, float* lse, int64_t lse_head_stride,
                              float* workspace, int64_t workspace_len, void* stream) {
  begin_device_call();
  const CachedQueries c{q, q_tok_stride, q_head_stride, q_dtype, k_cache, k_strides, block_table, block_table_stride,
                        block_table_width, seq_lens, num_seqs, num_q_heads, num_kv_heads, head_size, block_size,
                        num_blocks, total_q, max_seqlen_q, cu_seqlens_q, softmax_scale, nullptr, nullptr};
  Mx4Args p{};
  DecodeArgs& a = p.a;
  bool empty = false;
  if (out_dtype != PSK_DTYPE_BF16 && out_dtype != PSK_DTYPE_F16 && out_dtype != PSK_DTYPE_F32)
    return fail(PSK_E_DTYPE, "output dtype %d (bf16, f16 or f32)", out_dtype);
  if (max_seq_len < 0) return fail(PSK_E_ARG, "max_seq_len %lld", (long long)max_seq_len);
  if (const int st = check_cached_queries(c, a, &empty, 4); st != PSK_OK) return st;
  if (empty || total_q == 0) return PSK_OK;
  if (!v_cache || !v_strides || !out) return fail(PSK_E_ARG, "NULL pointer");
  const uint64_t v_align[4] = {uint64_t(uintptr_t(v_cache)), uint64_t(v_strides[0]), uint64_t(v_strides[1]),
                               uint64_t(v_strides[2])};
  if (common_align(v_align, 4, 4) < 4) return fail(PSK_E_ARG, "K/V caches need 4-byte aligned bases and strides");
  const int osz = dtype_size(out_dtype);
  const uint64_t o_align[3] = {uint64_t(uintptr_t(out)), uint64_t(out_tok_stride * osz), uint64_t(out_head_stride * osz)};
  if (common_align(o_align, 3, 4 * osz) < 4 * osz)
    return fail(PSK_E_ARG, "output rows need %d-byte alignment", 4 * osz);
  const int64_t need =
      psk_paged_mxfp4_workspace_len(num_seqs, total_q, max_seqlen_q, num_q_heads, num_kv_heads, max_seq_len);
  if (workspace_len < need || (need > 0 && !workspace))
    return fail(PSK_E_WORKSPACE, "workspace of %lld floats, need %lld", (long long)workspace_len, (long long)need);
  a.v = static_cast<const uint8_t*>(v_cache);
  a.v_blk = v_strides[0];
  a.v_row = v_strides[1];
  a.v_head = v_strides[2];
  a.causal = causal ? 1 : 0;
  a.out = static_cast<char*>(out);
  a.out_tok_stride = out_tok_stride * osz;
  a.out_head_stride = out_head_stride * osz;
  a.lse = lse;
  a.lse_head_stride = lse_head_stride;
  p.scale_log2 = double(softmax_scale) * 1.4426950408889634;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Route r = route(num_seqs, total_q, max_seqlen_q, a.heads, num_kv_heads);
  const int64_t row_q = r.row_tokens;
  Mx4Shape s{};
  if (r.way != kBlocks) {  // refused before the first launch, which may be the blocks'
    s = mx4_shape(num_seqs, row_q, num_q_heads, num_kv_heads, max_seq_len, q_dtype);
    const int64_t jobs = num_seqs * s.groups, tasks = num_seqs * num_kv_heads * row_q * a.heads;
    constexpr int64_t kMost = (int64_t(1) << 32) / kThreads - 1;  // a launch has fewer than 2^32 threads
    if (row_groups(s, jobs) > kMost || (!s.whole && merge_groups(joins_by_halves(s, jobs, tasks), tasks) > 1 << 21))
      return fail(PSK_E_ARG, "too many rows (%lld sequences of up to %lld query tokens)", (long long)num_seqs,
                  (long long)row_q);
  }
  if (r.way != kRows) {
    const int32_t most = r.way == kBoth ? int32_t(row_q) : 0;
    const Mx4Prefill step{num_seqs, total_q, max_seqlen_q, max_seq_len, most, p.scale_log2, q_dtype, out_dtype};
    const int e = launch_mx4_prefill(a, step, workspace, st);
    if (e != PSK_OK || r.way == kBlocks) return e;
    p.s.most = most;
  }
  p.s.num_seqs = int32_t(num_seqs);
  p.s.total_q = int32_t(total_q);
  p.s.heads = int32_t(s.groups);
  p.s.step_shift = int32_t(s.tile_shift + s.wph_shift);
  p.s.over = kOver;
  p.s.max_runs = int32_t(s.max_runs);
  p.s.min_run = kMinRun;
  p.s.width = INT32_MAX;
  p.hg = int32_t(s.hg);
  p.wph_shift = int32_t(s.wph_shift);
  p.row_blocks = int32_t(s.row_blocks);
  p.rows = int32_t(s.rows);
  p.max_rows = int32_t(row_q * a.heads);
  p.whole = s.whole;
  p.out_dtype = out_dtype;
  p.records = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~uintptr_t(15));
  switch (q_dtype) {
    case PSK_DTYPE_BF16: return launch<PSK_DTYPE_BF16>(p, s, st);
    case PSK_DTYPE_F16: return launch<PSK_DTYPE_F16>(p, s, st);
    default: return launch<PSK_DTYPE_F32>(p, s, st);
  }
}

}  // extern "C"
