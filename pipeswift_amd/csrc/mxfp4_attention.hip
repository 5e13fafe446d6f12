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
// A wave takes 32 keys of one kv head at a time (a tile), for 16 kSets query rows (query
// tokens x heads of the group):
//   * lane l loads 16 bytes, a whole group of 32 elements, of key l % 16's row at
//     group l / 16, and its scale byte, of K and of V, for both halves of the tile; the
//     next tile's are on their way meanwhile.
//   * S^T = K Q^T on v_mfma_f32_16x16x32_bf16: the lane's group is its part of the A
//     operand of four products as it stands (the query operand has the same order of
//     elements), and leaves query row l % 16 with keys 4 (l / 16) + r of each half.
//   * V becomes bf16 rows in the wave's own 8 KiB of LDS, 16-byte chunk c of key t at
//     c ^ (2 (t & 7)), and comes back transposed by ds_read_b64_tr_b16 as the A operand of
//     O^T = V^T P^T, whose P^T operand is the lane's weights as they stand.
// The waves of a workgroup take `hg` kv heads of the same tokens, so that the rows of a
// token, which share cache lines, are read together, and `1 << wph_shift` waves share a
// head's tiles in turn where the heads are fewer than the waves.  Nothing but the ends of
// a piece of work waits on a barrier.
//
// The work is cut into equal runs over sequences and head groups (cached_queries.h); a
// piece that is not all of a job's keys leaves a partial record, and merge_mx4_kernel
// joins a row's records in the order of their keys.  Short contexts are not cut.
//
// C ABI: include/pipeswift_kv.h.  Nothing here allocates or synchronizes.

#include <algorithm>

#include "mxfp4_attention.h"
#include "prefill_runs.h"

using namespace psk_detail;

namespace {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kTile = 32;          // keys of a wave's tile
constexpr int kTileShift = 5;
constexpr int kPages = 1024;       // page ids a piece stages at a time
constexpr int kMaxSlots = 512;     // resident workgroups the workspace is sized for
constexpr int kOver = 2;
constexpr int kMinRun = 2;
constexpr int kWholeKeys = 1024;

struct Mx4Args {
  DecodeArgs a;
  JobSpace s;            // heads: groups of kv heads
  double scale_log2;
  int32_t hg;            // kv heads of a group
  int32_t wph_shift;     // log2 of the waves of a head
  int32_t row_blocks;    // workgroups that share a run's keys, 16 kSets query rows each
  int32_t rows;          // query rows of a record
  int32_t max_rows;      // of a sequence and kv head
  int32_t whole;         // a workgroup takes all of a job's keys, and nothing is merged
  int32_t out_dtype;
  float* records;        // [max_runs][row_blocks][2][hg][rows][kHead + 4]
};

__device__ __forceinline__ float* record(const Mx4Args& p, int64_t run, int block, int slot, int hl, int row) {
  return p.records + ((((run * p.row_blocks + block) * 2 + slot) * p.hg + hl) * p.rows + row) * kRecord;
}

struct Tile {
  u32x4 k[2], v[2];
  uint32_t ks[2], vs[2];
};

template <int Q_DT, int kSets>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kSets == 1 && Q_DT == PSK_DTYPE_BF16 ? 4 : 2)))
mx4_attention_kernel(Mx4Args args) {
  constexpr bool kPairs = Q_DT != PSK_DTYPE_BF16;
  constexpr int kRows = 16 * kSets;
  __shared__ __attribute__((aligned(1024))) char s_v[kWaves][kTile * 2 * kHead];
  __shared__ int32_t s_pages[kPages];
  __shared__ float s_m[kWaves][kRows], s_l[kWaves][kRows];
  __shared__ int32_t s_nan[kWaves][4];  // of each head and group of columns the first key whose V is NaN there
  const int tid = int(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l15 = lane & 15, l4 = lane >> 4;
  const int hl = wave >> args.wph_shift, sub = wave & ((1 << args.wph_shift) - 1), wph = 1 << args.wph_shift;
  const bool active = hl < args.hg;

  // the row blocks of a run, which read the same keys, are next to each other on its XCD
  const int w = int(blockIdx.x), idx = (w >> 3) / args.row_blocks, block = (w >> 3) - idx * args.row_blocks;
  SeqWindow seqs;
  int64_t j = 0, x, x_end, before = 0;  // the run, its units, the units before the sequence
  int b;
  if (args.whole) {  // a workgroup a job
    const int jobs = args.s.num_seqs * args.s.heads, per = (jobs + 7) >> 3;
    const int job = (w & 7) * per + idx;
    if (idx >= per || job >= jobs) return;
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

  char* const vt = s_v[wave];
  // V^T reads: lane i of 16 receives column 16 c + i of keys 4 l4 .. 4 l4 + 3 of a half
  const int vkey = 4 * l4 + (l15 >> 2);
  const uint32_t vrow = uint32_t(256 * vkey + 8 * (l15 & 1));
  const int vq = (l15 & 3) >> 1, vsw = 2 * (vkey & 7);

  while (x < x_end) {  // over the run's jobs
    const Mx4Args& p = args_again<Mx4Args>();
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
    // a negative scale is applied as -q (exact); a scale of 0 stays above it, for a hidden key's -inf
    const float sl = __builtin_fmaxf(__builtin_fabsf(sl_signed), 0x1p-126f);
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
        query8<Q_DT>(src ? src + (32 * l4 + 8 * q) * Elt<Q_DT>::kSize : nullptr, sl_signed < 0.0f,
                     qop[s][q], qlo[kPairs ? s : 0][q]);
    }
    float m[kSets], l[kSets];
    f32x4 o[kSets][8];
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      m[s] = kNegBig;
      l[s] = 0.0f;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[s][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const uint8_t* kbase = a.k + int64_t(h) * a.k_head;
    const uint8_t* vbase = a.v + int64_t(h) * a.v_head;
    const int step_keys = 1 << p.s.step_shift;
    const int steps_per_window = int(min(int64_t(kPages - 1) * a.block_size / step_keys, int64_t(1) << 24));

    for (int s0 = c.from; s0 < c.to || s0 == c.from; s0 += steps_per_window) {
      const int s1 = min(c.to, s0 + steps_per_window);
      const int p0 = page_index(a, s0 * step_keys);
      __syncthreads();  // the ids, the marks and the results before these are done with
      if (s0 < s1 && L > 0) {
        const int p1 = page_index(a, int(min(int64_t(L), int64_t(s1) * step_keys)) - 1);
        for (int i = tid; i <= p1 - p0; i += kThreads) {
          int32_t id = -1;
          if (p0 + i < a.bt_width) id = a.block_table[int64_t(b) * a.bt_stride + p0 + i];
          s_pages[i] = id < a.num_blocks ? id : -1;
        }
      }
      if (s0 == c.from && tid < kWaves * 4) s_nan[tid >> 2][tid & 3] = INT32_MAX;
      __syncthreads();

      const int t_end = active ? min(s1 << (p.s.step_shift - kTileShift), (key_hi + kTile - 1) / kTile) : 0;
      auto fetch = [&](int t, Tile& y) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int key = t * kTile + 16 * u + l15;
          const int pi = page_index(a, key);
          const int id = key < L ? s_pages[pi - p0] : -1;
          y.k[u] = y.v[u] = u32x4(0);
          y.ks[u] = y.vs[u] = 127;
          if (id >= 0) {
            const int64_t row = key - pi * a.block_size;
            const int64_t ko = int64_t(id) * a.k_blk + row * a.k_row, vo = int64_t(id) * a.v_blk + row * a.v_row;
            y.k[u] = *reinterpret_cast<const u32x4_any*>(kbase + ko + 16 * l4);
            y.ks[u] = kbase[ko + kCodes + l4];
            y.v[u] = *reinterpret_cast<const u32x4_any*>(vbase + vo + 16 * l4);
            y.vs[u] = vbase[vo + kCodes + l4];
          }
        }
      };
      // One tile: V goes to LDS and K to operands, the next tile's loads start into their
      // registers, and then it is computed.
      auto attend = [&](int t, int next, bool masked, Tile& y) {
        // NaN values must not reach rows that do not see their key (0 x NaN): they become
        // zeros, and the end of the piece gives them to the rows that do
        if (__builtin_expect(__any(y.vs[0] == kMxNan || y.vs[1] == kMxNan), 0)) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (y.vs[u] == kMxNan) {
              atomicMin(&s_nan[hl][l4], t * kTile + 16 * u + l15);
              y.vs[u] = 127;
              y.v[u] = u32x4(0);
            }
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int key = 16 * u + l15;
          const float s = mx_scale(y.vs[u]);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<u32x4*>(vt + 256 * key + 16 * ((4 * l4 + q) ^ (2 * (key & 7)))) = mx_bf16x8(y.v[u][q], s);
        }
        float sc[kSets][8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
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
        if (next < t_end) fetch(next, y);
#pragma unroll
        for (int e = 0; e < kSets; ++e) {
          if (masked) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              sc[e][i] = t * kTile + 16 * (i >> 2) + 4 * l4 + (i & 3) < row_lim[e] ? sc[e][i] : -__builtin_inff();
          }
          float pv[8], sum = 0.0f;
          auto weigh = [&] {
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              pv[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e][i], sl, -m[e]));
              sum += pv[i];
            }
          };
          weigh();
          if (__builtin_expect(__any(!(sum <= kShareMost)), 0)) {  // (NaN scores come here too)
            float top = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < 8; ++i) top = __builtin_fmaxf(top, sc[e][i]);
            top *= sl;
            top = __builtin_fmaxf(top, __shfl_xor(top, 16));
            top = __builtin_fmaxf(top, __shfl_xor(top, 32));
            const float mn = __builtin_fmaxf(m[e], top);
            const float f = __builtin_amdgcn_exp2f(m[e] - mn);
            m[e] = mn;
            l[e] *= f;
#pragma unroll
            for (int d = 0; d < 8; ++d) o[e][d] *= f;
            weigh();
          }
          l[e] += sum;
          bf16x8 ph, pl;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            ph[i] = __bf16(pv[i]);
            pl[i] = __bf16(pv[i] - float(ph[i]));
          }
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            const uint32_t off = vrow + uint32_t(16 * ((2 * d + vq) ^ vsw));
            const s16x4 t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vt + off));
            const s16x4 t1 =
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vt + 256 * 16 + off));
            const bf16x8 v = __builtin_bit_cast(bf16x8, __builtin_shufflevector(t0, t1, 0, 1, 2, 3, 4, 5, 6, 7));
            o[e][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pl, o[e][d], 0, 0, 0);
            o[e][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, ph, o[e][d], 0, 0, 0);
          }
        }
      };

      int t = (s0 << (p.s.step_shift - kTileShift)) + sub;
      const int t_mask = key_open / kTile;  // tiles from here on need masks
      Tile y;
      if (t < t_end) fetch(t, y);
      for (; t < t_end; t += wph) attend(t, t + wph, t >= t_mask, y);
    }

    const Mx4Args& rest = args_again<Mx4Args>();
    const bool all = c.from == 0 && c.to == steps;
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      l[s] += __shfl_xor(l[s], 16);
      l[s] += __shfl_xor(l[s], 32);
      if (l4 == 0) {
        s_m[wave][16 * s + l15] = m[s];
        s_l[wave][16 * s + l15] = l[s];
      }
    }
    __syncthreads();  // every wave has left its tiles, and wrote its maxima and marks
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      float top = m[s], sum = l[s];
      if (wph > 1) {
        if (s > 0) __syncthreads();  // the last set's readers are done
        top = kNegBig;
        sum = 0.0f;
        for (int v = 0; v < wph; ++v) top = __builtin_fmaxf(top, s_m[(hl << rest.wph_shift) + v][16 * s + l15]);
        for (int v = 0; v < wph; ++v)
          sum += s_l[(hl << rest.wph_shift) + v][16 * s + l15] *
                 __builtin_amdgcn_exp2f(s_m[(hl << rest.wph_shift) + v][16 * s + l15] - top);
        const float f = __builtin_amdgcn_exp2f(m[s] - top);
#pragma unroll
        for (int d = 0; d < 8; ++d) reinterpret_cast<f32x4*>(vt)[64 * d + lane] = o[s][d] * f;
        __syncthreads();
      }
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        if ((d & (wph - 1)) != sub || !active) continue;
        f32x4 v = o[s][d];
        if (wph > 1) {
          v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          for (int u = 0; u < wph; ++u) v += reinterpret_cast<const f32x4*>(s_v[(hl << rest.wph_shift) + u])[64 * d + lane];
        }
        if (__builtin_expect(s_nan[hl][d >> 1] < row_lim[s], 0))
          v = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
        const int row = row0 + 16 * s + l15, col = 16 * d + 4 * l4;
        if (all) {
          finish(rest.a, rest.out_dtype, r, h, row, col, v, top, sum);
        } else if (row < r.n * rest.a.heads) {
          float* rec = record(rest, j, block, c.from == 0 ? 1 : 0, hl, 16 * s + l15);
          *reinterpret_cast<f32x4*>(rec + col) = v;
          if (col == 0) {
            rec[kHead] = top;
            rec[kHead + 1] = sum;
          }
        }
      }
    }
  }
}

// The records of a query row joined: a workgroup a row at a time.  Each half of a wave takes
// every sixteenth record, and the halves' parts are joined in order.
constexpr int kMergeThreads = 512;
constexpr int kParts = kMergeThreads / 32;

template <int kRows>
__global__ void __launch_bounds__(kMergeThreads) merge_mx4_kernel(Mx4Args p, int64_t tasks) {
  const DecodeArgs& a = p.a;
  __shared__ f32x4 s_o[kParts][32];
  __shared__ float s_m[kParts], s_l[kParts];
  const int tid = int(threadIdx.x), lane = tid & 63, part = tid >> 5, at4 = tid & 31;
  const int max_rows = p.max_rows;
  const int kv_heads = p.s.heads * p.hg;
  for (int64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int64_t job = uniform_div(task, max_rows);
    const int row = int(task - job * max_rows);
    const int b = int(uniform_div(job, kv_heads)), h = int(job - int64_t(b) * kv_heads);
    const SeqRows r = seq_rows(a, p.s.total_q, b);
    if (r.n > p.s.most || row >= r.n * a.heads) continue;
    SeqWindow seqs;
    const StepRuns cost = step_runs(a, p.s, seqs, lane);
    const int64_t before = units_before(a, p.s, b, seqs, lane);
    const int steps = key_steps(p.s, lane_value(seqs.len, b - seqs.b0));
    const int grp = h / p.hg;
    const int64_t at = before + grp * int64_t(p.s.over + steps) + p.s.over;  // the first unit that pays for keys
    const int64_t j0 = uniform_div(at, cost.run), j1 = steps > 0 ? uniform_div(at + steps - 1, cost.run) : j0 - 1;
    if (j0 == j1) continue;  // one run had all the keys and wrote the row
    const int block = row / kRows, in_block = row - block * kRows;

    float top = kNegBig, sum = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int kAhead = 4;  // records read together
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
    __syncthreads();  // the last row's readers are done
    s_o[part][at4] = o;
    if (at4 == 0) {
      s_m[part] = top;
      s_l[part] = sum;
    }
    __syncthreads();
    if (part == 0) {
      for (int u = 1; u < kParts; ++u) top = __builtin_fmaxf(top, s_m[u]);
      sum = 0.0f;
      o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      for (int u = 0; u < kParts; ++u) {
        const float f = __builtin_amdgcn_exp2f(s_m[u] - top);
        sum += s_l[u] * f;
        o += s_o[u][at4] * f;
      }
      finish(a, p.out_dtype, r, h, row, 4 * at4, o, top, sum);
    }
  }
}

// Workgroups resident at once: two per CU (LDS and registers).
int64_t mx4_slots() { return std::min<int64_t>(2 * device_cus(), kMaxSlots); }

// How a step is laid out, from the bounds that its caller gives.
struct Mx4Shape {
  int64_t sets, row_blocks, rows, hg, groups, wph_shift, max_runs;
  bool whole;
};
Mx4Shape mx4_shape(int64_t num_seqs, int64_t max_seqlen_q, int64_t num_q_heads, int64_t num_kv_heads, int64_t max_seq_len,
                   int64_t slots) {
  Mx4Shape s;
  const int64_t rows = max_seqlen_q * (num_q_heads / num_kv_heads);
  s.sets = rows <= 16 ? 1 : 2;
  s.row_blocks = ceil_div(rows, 16 * s.sets);
  s.rows = std::min<int64_t>(rows, 16 * s.sets);
  s.whole = max_seq_len <= kWholeKeys;
  s.hg = 1;
  for (int64_t g = 1; g <= kWaves; ++g)
    if (num_kv_heads % g == 0) s.hg = g;
  // uncut: the fewer the jobs, the more waves to a head
  if (s.whole)
    while (s.hg > 1 && num_seqs * (num_kv_heads / s.hg) * s.row_blocks < 256) {
      int64_t g = s.hg - 1;
      while (num_kv_heads % g) --g;
      s.hg = g;
    }
  s.groups = num_kv_heads / s.hg;
  s.wph_shift = 0;
  while ((s.hg << (s.wph_shift + 1)) <= kWaves) ++s.wph_shift;
  s.max_runs = xcd_rounds(slots / s.row_blocks);
  return s;
}

// Which kernels a step takes: sequences of at most kFewRows query rows a kv head go by
// rows, those of more by blocks of 256 (mxfp4_prefill.hip), in one launch each.
constexpr int kFewRows = 32;
enum Route { kRows, kBlocks, kBoth };
Route route(int64_t num_seqs, int64_t total_q, int64_t max_seqlen_q, int64_t heads) {
  if (max_seqlen_q * heads <= kFewRows || heads > kBlockRows) return kRows;
  // (more sequences than are ordered by their lengths: all by blocks)
  return num_seqs == 1 || heads > kFewRows || total_q == num_seqs * max_seqlen_q || num_seqs > kOrderMax ? kBlocks : kBoth;
}

// Query tokens of a sequence that goes by rows, at most.
int64_t row_tokens(Route r, int64_t max_seqlen_q, int64_t heads) {
  return r == kBoth ? std::max<int64_t>(kFewRows / heads, 1) : max_seqlen_q;
}

template <int Q_DT>
int launch(const Mx4Args& p, const Mx4Shape& s, hipStream_t st) {
  const int64_t jobs = int64_t(p.s.num_seqs) * p.s.heads;
  const dim3 grid{unsigned((p.whole ? ceil_div(jobs, 8) * 8 : s.max_runs) * s.row_blocks), 1u, 1u};
  if (s.sets == 1) hipLaunchKernelGGL((mx4_attention_kernel<Q_DT, 1>), grid, dim3(kThreads), 0, st, p);
  else hipLaunchKernelGGL((mx4_attention_kernel<Q_DT, 2>), grid, dim3(kThreads), 0, st, p);
  if (const int e = check_launch("mx4_attention_kernel launch"); e != PSK_OK || p.whole) return e;
  const int64_t tasks = int64_t(p.s.num_seqs) * p.s.heads * p.hg * p.max_rows;
  const dim3 merge{unsigned(std::min<int64_t>(tasks, 1 << 20)), 1u, 1u};
  if (s.sets == 1) hipLaunchKernelGGL((merge_mx4_kernel<16>), merge, dim3(kMergeThreads), 0, st, p, tasks);
  else hipLaunchKernelGGL((merge_mx4_kernel<32>), merge, dim3(kMergeThreads), 0, st, p, tasks);
  return check_launch("merge_mx4_kernel launch");
}

}  // namespace

extern "C" {

int64_t psk_paged_mxfp4_workspace_len(int64_t num_seqs, int64_t total_q, int64_t max_seqlen_q, int64_t num_q_heads,
                                      int64_t num_kv_heads, int64_t max_seq_len) {
  if (num_seqs < 0 || total_q < 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads ||
      max_seqlen_q <= 0 || max_seqlen_q > INT32_MAX / (num_q_heads / num_kv_heads) || max_seq_len < 0)
    return PSK_E_ARG;
  const Route r = route(num_seqs, total_q, max_seqlen_q, num_q_heads / num_kv_heads);
  const Mx4Shape s = mx4_shape(num_seqs, row_tokens(r, max_seqlen_q, num_q_heads / num_kv_heads), num_q_heads, num_kv_heads,
                               max_seq_len, kMaxSlots);
  const int64_t own = s.whole ? 0 : 4 + s.max_runs * s.row_blocks * 2 * s.hg * s.rows * kRecord;
  if (r == kRows) return own;
  const int64_t blocks = mx4_prefill_floats(num_seqs, total_q, max_seqlen_q, num_q_heads, num_kv_heads, max_seq_len);
  return r == kBlocks ? blocks : std::max(own, blocks);  // (one after the other)
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
  const Route way = route(num_seqs, total_q, max_seqlen_q, a.heads);
  const int64_t row_q = row_tokens(way, max_seqlen_q, a.heads);
  if (way != kRows) {
    const int32_t most = way == kBoth ? int32_t(kFewRows / a.heads) : 0;
    const Mx4Prefill step{num_seqs, total_q, max_seqlen_q, max_seq_len, most, p.scale_log2, q_dtype, out_dtype};
    const int e = launch_mx4_prefill(a, step, workspace, st);
    if (e != PSK_OK || way == kBlocks) return e;
    p.s.most = most;
  }
  const Mx4Shape s = mx4_shape(num_seqs, row_q, num_q_heads, num_kv_heads, max_seq_len, mx4_slots());
  p.s.num_seqs = int32_t(num_seqs);
  p.s.total_q = int32_t(total_q);
  p.s.heads = int32_t(s.groups);
  p.s.step_shift = int32_t(kTileShift + s.wph_shift);
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
  constexpr int64_t kMost = (int64_t(1) << 24) - 8;  // workgroups of a launch
  if (std::max(num_seqs * s.groups, s.max_runs) > kMost / s.row_blocks)
    return fail(PSK_E_ARG, "too many rows (%lld sequences of up to %lld query tokens)", (long long)num_seqs,
                (long long)max_seqlen_q);
  switch (q_dtype) {
    case PSK_DTYPE_BF16: return launch<PSK_DTYPE_BF16>(p, s, st);
    case PSK_DTYPE_F16: return launch<PSK_DTYPE_F16>(p, s, st);
    default: return launch<PSK_DTYPE_F32>(p, s, st);
  }
}

}  // extern "C"
