// The attention weight every cached token received, summed over the queries of
// a step (the scores an eviction goes by), for MI355X (gfx950):
//   A[b, h, j] = decay A[b, h, j] + sum over query tokens i that see j and heads g of
//                exp(s_ij - lse[h G + g, i]),     j < seq_lens[b],
// s as the readers compute it (exactly converted FP8 operands on the bf16 MFMA)
// and lse as they return it.  V is not read, and no sum of a key leaves its
// workgroup, so there are no atomics and the order of every sum is fixed.
//
// Two kernels, by the query rows n G that share a key (one MFMA tile holds 32 of
// them, and K then is all there is to move; 16 sequences of 8000, 32 query heads over
// 8, few / many rows' kernel: 1 query token 30 / 66 us, 8 of them 34 / 61):
//   * few_rows_kernel, at most 32 of them (a decode step): a wave per 32 keys,
//     S = Q K^T on v_mfma_f32_32x32x16_bf16 leaves lane l key l % 32 and rows
//     8 (i / 4) + 4 (l / 32) + i % 4, so a key's sum is one lane's registers and
//     one exchange.  The K rows go to LDS three tiles ahead, the kv heads of a
//     token together; the work is cut into equal runs
//     (cached_queries.h).
//   * many_rows_kernel, more (the last queries of a prompt, a whole prompt): a
//     wave holds 32 keys as MFMA operands and the step's e4m3 queries, quantized
//     once by quantize_queries_kernel, pass by it 32 rows at a time.  S^T = K Q^T
//     leaves lane l query row l % 32, whose lse is one value, and sixteen sums a
//     key tile, which are joined over the lanes at the end.  Where there are
//     too few keys to fill the GPU the waves of a workgroup share its keys and
//     take the rows in turn.
//
// C ABI: include/pipeswift_kv.h.  Nothing here allocates or synchronizes.

#include <algorithm>

#include "cached_queries.h"

using namespace psk_detail;

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kTile = 32;    // keys of an MFMA tile
constexpr int kRows = 32;    // query rows of one
constexpr uint32_t kHalfSlot = kTile * 128;  // bytes of a tile's K
constexpr int kFewRing = 4;  // tiles of K a wave has in LDS (few rows)
constexpr int kPages = 1024; // page ids staged at a time (few rows)
constexpr int kFewRows = 64;   // query rows of a job's heads, each padded to whole groups (few rows)
constexpr int kManyWaves = 8;  // (many rows)
constexpr int kManyRing = 2;   // row tiles a wave has in LDS (many rows)
constexpr int kStepTiles = 4;  // of a step (few rows)
constexpr int kStepKeys = kTile * kStepTiles;

struct WeightArgs {
  DecodeArgs a;
  JobSpace s;
  double scale_log2;  // softmax_scale * log2(e)
  const float* lse;
  int64_t lse_head_stride;
  float* scores;
  int64_t seq_stride, head_stride;  // elements
  float decay;
  const uint8_t* q8;  // many rows: e4m3 queries [total_q][Hq][128]
  int64_t q8_tok, q8_head;
  int32_t hg;         // few rows: kv heads of a job
  int32_t row_tiles;  // many rows: most of any sequence
  int32_t slots;      // many rows: workgroups that fill the GPU
  int32_t cus;
  int32_t near;       // many rows: the rows of a tile lie within 32-bit offsets
};

__device__ __forceinline__ float* score_row(const WeightArgs& p, int b, int h) {
  return p.scores + int64_t(b) * p.seq_stride + int64_t(h) * p.head_stride;
}

// lse log2(e) of a query row, rounded once.
__device__ __forceinline__ float lse_log2(const WeightArgs& p, int hq, int64_t tok) {
  return float(double(p.lse[int64_t(hq) * p.lse_head_stride + tok]) * 1.4426950408889634);
}

__device__ __forceinline__ float decayed(const WeightArgs& p, const float* at) {
  return p.decay == 0.0f ? 0.0f : *at * p.decay;
}

// ---------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------

// A job here is a sequence's keys under `hg` kv heads; `heads` of the JobSpace
// counts its groups of them.  A workgroup's waves take the (tile, head) pairs of
// a run in turn, heads first, so that the rows of a token's heads, which lie next
// to each other, are read together.
// K goes to LDS by global_load_lds, whole rows at a time and past the caches, a
// ring of kFewRing pairs a wave: 107 us for 64 sequences of 128 to 32768 tokens (32
// query heads over 8), 5.0 TB/s, as a large copy; 122 with the caches, and 133 with
// K read straight to registers, where a lane's part of a row makes four requests of
// every line.  Runs of one kv head instead of all of a token's: 164.
template <int Q_DT, bool OLD, bool GEN>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2)))
few_rows_kernel(WeightArgs args) {
  __shared__ __attribute__((aligned(1024))) char s_ring[kWaves * kFewRing * kHalfSlot];
  __shared__ float s_old[kWaves * kFewRing * kTile];
  __shared__ int32_t s_pages[kPages];
  __shared__ u32x4 s_q[kFewRows * 8];  // e4m3 queries, [head][padded row], chunk c of row r at c ^ (r & 7)
  __shared__ f32x4 s_lse[kFewRows / 4];  // of each row; +inf for rows without a token
  __shared__ float s_sl[kFewRows / 8];   // of each head
  const int tid = int(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, kk = lane & 31;
  const uint32_t ring = (uint32_t)(size_t)(lvoid*)s_ring + uint32_t(wave * kFewRing) * kHalfSlot;
  const uint32_t old_at = (uint32_t)(size_t)(lvoid*)s_old + uint32_t(wave * kFewRing * kTile * 4);
  // loads: lane l takes chunk position l % 8 of keys 8 u + l / 8, chunk c of key t lies at c ^ (t & 7)
  const int lr = lane >> 3, lchunk = 16 * ((lane & 7) ^ lr);
  const uint32_t off_k = uint32_t(lr * args.a.k_row) + lchunk;
  SeqWindow seqs;
  const StepRuns step_run = step_runs(args.a, args.s, seqs, lane);
  int64_t x = xcd_run(step_run, int(blockIdx.x) & 7, int(blockIdx.x) >> 3) * step_run.run;
  if (x >= step_run.total) return;
  const int64_t x_end = min(x + step_run.run, step_run.total);
  int64_t before;
  int b = seq_of_unit(args.a, args.s, x, seqs, lane, before);
  while (x < x_end) {  // over the run's jobs
    const WeightArgs& p = args_again<WeightArgs>();
    const DecodeArgs& a = p.a;
    if (!seqs.holds(b)) seqs.load(a, p.s, b, lane);
    const SeqRows r{lane_value(seqs.first, b - seqs.b0), lane_value(seqs.n, b - seqs.b0)};
    const int full = lane_value(seqs.len, b - seqs.b0), L = min(full, p.s.width);
    const int64_t seq_cost = lane_value(seqs.cost, b - seqs.b0);
    if (x >= before + seq_cost) {
      before += seq_cost;
      ++b;
      continue;
    }
    const int64_t job_cost = p.s.over + key_steps(p.s, L);
    const int job = int(uniform_div(x - before, job_cost));
    const int64_t at = before + job * job_cost;
    const int64_t hi = min(x_end, at + job_cost);
    const Piece c = piece_of(p.s, x - at, hi - at);
    x = hi;
    if (c.from >= c.to) continue;
    const int h0 = job * p.hg, heads = min(p.hg, a.num_kv_heads - h0);

    if (r.n <= 0) {  // the old sums decay all the same
      for (int h = h0; h < h0 + heads; ++h) {
        float* scores = score_row(p, b, h);
        for (int key = c.from * kStepKeys + tid; key < min(L, c.to * kStepKeys); key += kThreads)
          scores[key] = decayed(p, scores + key);
      }
      continue;
    }
    const int R = r.n * a.heads, ctx = full - r.n;
    const int groups = (R + 7) >> 3, padded = 8 * groups;  // register groups of four (of each half) that hold rows
    __syncthreads();  // readers of the last piece's queries are done
    for (int i = tid; i < heads * padded * 8; i += kThreads) {
      const int row = i >> 3, hh = row / padded, rr = row - hh * padded;
      const int qi = rr / a.heads, h = h0 + hh, hq = h * a.heads + rr - qi * a.heads;
      const float qd = descale(a.qd, a.qd_b, a.qd_h, b, h);
      QueryBytes<Q_DT> qb;
      qb.load(rr < R ? a.q + (int64_t(r.first) + qi) * a.q_tok_stride + int64_t(hq) * a.q_head_stride : nullptr, 16 * (i & 7));
      s_q[row * 8 + ((i & 7) ^ (row & 7))] = qb.quantized(qd, 0u);
      if ((i & 7) == 0) {
        reinterpret_cast<float*>(s_lse)[row] = rr < R ? lse_log2(p, hq, int64_t(r.first) + qi) : __builtin_inff();
        if (rr == 0) s_sl[hh] = score_scale(p.scale_log2, qd, descale(a.kd, a.kd_b, a.kd_h, b, h));
      }
    }
    // row of this lane in the query operand (rows past the padded ones: any, their results are not used)
    const int row_k = min(kk, padded - 1);
    const int n_tiles = (L + kTile - 1) / kTile;
    const int t_mask = a.causal ? max(ctx, 0) / kTile : n_tiles;  // tiles below are seen by every row
    const int steps_per_window = int(min(int64_t(kPages - 1) * a.block_size / kStepKeys, int64_t(1) << 24));
    for (int s0 = c.from; s0 < c.to; s0 += steps_per_window) {
      const int s1 = min(c.to, s0 + steps_per_window);
      const int p0 = page_index(a, s0 * kStepKeys);
      const int p1 = page_index(a, int(min(int64_t(L), int64_t(s1) * kStepKeys)) - 1);
      if (s0 > c.from) __syncthreads();  // the ids before these are done with
      for (int i = tid; i <= p1 - p0; i += kThreads) {
        int32_t id = -1;
        if (p0 + i < a.bt_width) id = a.block_table[int64_t(b) * a.bt_stride + p0 + i];
        s_pages[i] = id < a.num_blocks ? id : -1;
      }
      __syncthreads();

      const int t_end = min(kStepTiles * s1, n_tiles);
      struct Place {
        int t, hh;  // tile and head of the group
      };
      auto next = [&](Place& w, int by) {
        w.hh += by;
        while (w.hh >= heads) {
          w.hh -= heads;
          ++w.t;
        }
      };
      // Where the eight keys of a load lie: lane 4 k + u those of load u of tile
      // win + k, sixteen tiles at a time (GEN: every lane its own key's place).
      int win = kStepTiles * s0;
      int64_t at_k = 0;
      uint64_t whole8 = 0, some8 = 0;  // loads whose eight keys are all cached; whose first is
      auto look_up = [&](int t) {
        win = t;
        const int key = (t + (lane >> 2)) * kTile + 8 * (lane & 3);
        int32_t id = -1;
        int pi = 0;
        if (t + (lane >> 2) < t_end && key < L) {
          pi = page_index(a, key);
          id = s_pages[pi - p0];
        }
        at_k = int64_t(id) * a.k_blk + int64_t(key - pi * a.block_size) * a.k_row - 1024 * (lane & 3);
        some8 = __ballot(id >= 0);
        whole8 = __ballot(id >= 0 && key + 8 <= L);
      };
      // The loads of a pair into a slot: K rows (four), old sums (one).  Pairs whose
      // loads were not all started are counted out of `sure`, the newest run of
      // pairs that were.
      int sure = 0;
      auto start = [&](const Place& w, int slot_no) {
        const uint32_t slot = ring + uint32_t(slot_no) * kHalfSlot;
        const uint8_t* base = a.k + int64_t(h0 + w.hh) * a.k_head;
        if constexpr (OLD) {
          const float* sums = reinterpret_cast<const float*>(
              wave_uniform(int64_t(reinterpret_cast<uintptr_t>(score_row(p, b, h0 + w.hh) + w.t * kTile))));
          if (half == 0 && w.t * kTile + kk < L) load_lds_dword(old_at + 128 * slot_no, sums, 4 * kk);
        }
        bool full;
        if constexpr (GEN) {
          const uint8_t* from[4];
          full = true;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int key = w.t * kTile + 8 * u + lr;
            const int pi = page_index(a, key);
            const int32_t id = key < L ? s_pages[pi - p0] : -1;
            from[u] = id >= 0 ? base + lchunk + (int64_t(id) * a.k_blk + int64_t(key - pi * a.block_size) * a.k_row) : nullptr;
            full = full && __all(id >= 0);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (from[u]) load_lds(slot + 1024 * u, from[u]);
            else *lds_at<u32x4>(slot + 1024 * u + 16 * lane) = u32x4(0);
          }
        } else {
          if (w.t - win >= 16) look_up(w.t);
          const int k = 4 * (w.t - win);
          full = ((whole8 >> k) & 15) == 15;
          if (__builtin_expect(full, 1)) {
            const uint8_t* from[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) from[u] = base + lane_value(at_k, k + u);
            load_lds_4k_once(slot, from, off_k);
          } else {
#pragma unroll 1
            for (int u = 0; u < 4; ++u) {
              if (((some8 >> (k + u)) & 1) && w.t * kTile + 8 * u + lr < L)
                load_lds(slot + 1024 * u, base + lane_value(at_k, k + u) + 1024 * u, off_k);
              else
                *lds_at<u32x4>(slot + 1024 * u + 16 * lane) = u32x4(0);
            }
          }
        }
        sure = full ? sure + 1 : 0;
      };
      auto add_up = [&](const Place& w, int slot_no) {
        const uint32_t slot = ring + uint32_t(slot_no) * kHalfSlot;
        f32x16 y = {};
        const int row = w.hh * padded + row_k;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const u32x4 k = *lds_at<u32x4>(slot + uint32_t(128 * kk + 16 * ((4 * half + q) ^ (kk & 7))));
          const u32x4 v = s_q[row * 8 + ((4 * half + q) ^ (row & 7))];
          y = __builtin_amdgcn_mfma_f32_32x32x16_bf16(e4m3x8_to_bf16(v[0], v[1]), e4m3x8_to_bf16(k[0], k[1]), y, 0, 0, 0);
          y = __builtin_amdgcn_mfma_f32_32x32x16_bf16(e4m3x8_to_bf16(v[2], v[3]), e4m3x8_to_bf16(k[2], k[3]), y, 0, 0, 0);
        }
        const int key = w.t * kTile + kk;
        const float sl = s_sl[w.hh];
        float sum = 0.0f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          if (g < groups) {
            const f32x4 lse = s_lse[(w.hh * padded + 8 * g + 4 * half) >> 2];
            f32x4 e;
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(y[4 * g + i], sl, -lse[i]));
            if (w.t >= t_mask) {
#pragma unroll
              for (int i = 0; i < 4; ++i) e[i] = key <= ctx + (8 * g + 4 * half + i) / a.heads ? e[i] : 0.0f;
            }
            sum += (e[0] + e[1]) + (e[2] + e[3]);
          }
        }
        sum += __shfl_xor(sum, 32);
        float o = 0.0f;
        if constexpr (OLD) o = *lds_at<float>(old_at + 128 * slot_no + 4 * kk) * p.decay;
        if (half == 0 && key < L) score_row(p, b, h0 + w.hh)[key] = o + sum;
        // every read of the slot is done before its next loads start
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      };
      Place now{kStepTiles * s0, 0};
      next(now, wave);
      Place then = now;  // the pair whose loads are started next
      int flying = 0;    // pairs whose loads are in flight
      if constexpr (!GEN) look_up(win);
#pragma unroll 1
      for (int u = 0; u < kFewRing - 1 && then.t < t_end; ++u, ++flying) {
        start(then, u);
        next(then, kWaves);
      }
      int slot_no = 0, to = kFewRing - 1;
      while (now.t < t_end) {
        if (then.t < t_end) {
          start(then, to);
          next(then, kWaves);
          ++flying;
        }
        // the pair's own loads: those of the pairs after it may stay in flight
        // (stores in between count too, and make this wait longer, not shorter)
        constexpr int kLoads = OLD ? 5 : 4;
        --flying;
        if (sure >= flying && flying == 3) wait_loads<3 * kLoads>();
        else if (sure >= flying && flying == 2) wait_loads<2 * kLoads>();
        else if (sure >= flying && flying == 1) wait_loads<kLoads>();
        else wait_loads<0>();
        add_up(now, slot_no);
        next(now, kWaves);
        slot_no = slot_no == kFewRing - 1 ? 0 : slot_no + 1;
        to = to == kFewRing - 1 ? 0 : to + 1;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------

// e4m3 queries of all rows, [total_q][Hq][128], sixteen elements a thread.
template <int Q_DT>
__global__ void __launch_bounds__(kThreads) quantize_queries_kernel(WeightArgs p, int num_q_heads, uint8_t* q8) {
  const DecodeArgs& a = p.a;
  const uint32_t x = blockIdx.x * kThreads + threadIdx.x;  // (host: below 2^32)
  const uint32_t row = x >> 3, token = row / uint32_t(num_q_heads);
  const int tok = int(token), hq = int(row - token * uint32_t(num_q_heads));
  if (tok >= p.s.total_q) return;
  float qd = 1.0f;
  if (a.qd) {  // the descale of the row's sequence and kv head
    const int b = a.cu_q ? int(sequence_from(a.cu_q, p.s.num_seqs, 0, tok)) : tok / a.q_len;
    qd = b < p.s.num_seqs ? descale(a.qd, a.qd_b, a.qd_h, b, hq / a.heads) : 1.0f;
  }
  QueryBytes<Q_DT> qb;
  qb.load(a.q + int64_t(tok) * a.q_tok_stride + int64_t(hq) * a.q_head_stride, 16 * int(x & 7));
  *reinterpret_cast<u32x4*>(q8 + 16 * int64_t(x)) = qb.quantized(qd, 0u);
}

// Sixteen values of a lane summed over the 32 lanes of its half, in a fixed
// order: lane l returns value (l >> 1) & 15.
__device__ __forceinline__ float sum_lanes(float (&v)[16], int lane) {
#pragma unroll
  for (int n = 8; n >= 1; n >>= 1) {
    const bool up = lane & (2 * n);
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = up ? v[i + n] : v[i], give = up ? v[i] : v[i + n];
      v[i] = keep + __shfl_xor(give, 2 * n);
    }
  }
  return v[0] + __shfl_xor(v[0], 1);
}

// The rows go to LDS two tiles ahead, whole 128-byte rows by global_load_lds, so
// that the loop's registers let four waves share a SIMD (128 of them, with two spilled
// outside the loop): 38 us for the last 64 queries of 4 contexts of 8000 to 32000
// tokens (32 query heads over 4), 77 % of it vector time.  Of the 27 us of that, 14
// are the scores' (an fma, a quarter-rate exp2 and an addition each), 5 the queries'
// conversion and 8 a unit's start and end: of 143 vector instructions a tile of 32 x
// 32, the loop has about 90.  Rows read
// straight to registers, 64 keys a wave and two waves a SIMD: 48; 64 keys from LDS:
// 49.  Units go keys first and the CUs take them forwards and backwards in turn, so
// that under a causal mask a CU's long and short ones add up alike: 28 us for a
// prompt of 2000 tokens (32 over 8).
//
// The unit of workgroup w, which runs on XCD w % 8: forwards over the CUs in even
// rounds, backwards in odd ones.
__device__ __forceinline__ int64_t unit_of(int64_t w, int cus) {
  const int64_t round = uniform_div(w, cus);
  if ((round & 1) == 0) return w;
  const int64_t q = (w >> 3) - round * (cus >> 3);
  return 8 * (round * (cus >> 3) + (cus >> 3) - 1 - q) + (w & 7);
}

__global__ void __launch_bounds__(64 * kManyWaves) __attribute__((amdgpu_waves_per_eu(4))) many_rows_kernel(WeightArgs args) {
  __shared__ __attribute__((aligned(1024))) char s_ring[kManyWaves * kManyRing * kHalfSlot];
  __shared__ float s_lse[kManyWaves * kManyRing * kRows];
  __shared__ float s_sum[kManyWaves][kTile];
  const int tid = int(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, kk = lane & 31;
  const uint32_t ring = (uint32_t)(size_t)(lvoid*)s_ring + uint32_t(wave * kManyRing) * kHalfSlot;
  const uint32_t lse_ring = (uint32_t)(size_t)(lvoid*)s_lse + uint32_t(wave * kManyRing * kRows * 4);
  // As many keys to a workgroup as leave `slots` of them; the fewer keys the step
  // has, the more waves share them (as far as there are row tiles for each).  From
  // the lengths and max_seqlen_q, so that the order of the sums does not depend on
  // max_seq_len.
  SeqWindow seqs;
  JobSpace s = args.s;  // (a step of kTile keys)
  StepRuns step = step_runs(args.a, s, seqs, lane);
  int split = 1;
  while (split < kManyWaves && split < args.row_tiles && step.total * split < int64_t(args.slots) * kManyWaves) split *= 2;
  for (int w = split; w < kManyWaves; w *= 2) ++s.step_shift;
  if (s.num_seqs <= 64) {
    seqs.price(s, lane);
    step.total = seqs.total;
  } else {
    step = step_runs(args.a, s, seqs, lane);
    seqs.b0 = -64;  // (the last window is there, not the first)
  }
  // waves w, w + 1 .. of a group of `split` hold the same keys and take the row tiles in turn
  const int group = wave / split, turn = wave - group * split;
  const int64_t places = uniform_div(step.total + args.cus - 1, args.cus) * args.cus;
  for (int64_t w = blockIdx.x; w < places; w += gridDim.x) {  // a unit: a workgroup's keys of a kv head
    const WeightArgs& p = args_again<WeightArgs>();
    const DecodeArgs& a = p.a;
    const int G = a.heads;
    const int64_t x = unit_of(w, p.cus);
    if (x >= step.total) continue;
    int64_t before;
    const int b = seq_of_unit(a, s, x, seqs, lane, before);
    const SeqRows r{lane_value(seqs.first, b - seqs.b0), lane_value(seqs.n, b - seqs.b0)};
    const int full = lane_value(seqs.len, b - seqs.b0), L = min(full, p.s.width);
    const int unit = int(uniform_div(x - before, s.heads)), h = int(x - before) - unit * s.heads;
    const int k0 = unit * (1 << s.step_shift) + group * kTile;  // the wave's keys
    const int ctx = full - r.n;

    // lane l: of keys l % 32 the 16-byte chunks 2 q + l / 32 (the queries' the same);
    // missing rows and keys past the end as zeros
    bf16x8 kop[8];
    {
      const int key = k0 + kk;
      int32_t id = -1;
      int pi = 0;
      if (key < L) {
        pi = page_index(a, key);
        if (pi < a.bt_width) id = a.block_table[int64_t(b) * a.bt_stride + pi];
        if (id >= a.num_blocks) id = -1;
      }
      const uint8_t* row = a.k + int64_t(h) * a.k_head + 16 * half + int64_t(id) * a.k_blk +
                           int64_t(key - pi * a.block_size) * a.k_row;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const u32x4 v = id >= 0 ? *reinterpret_cast<const u32x4*>(row + 32 * q) : u32x4(0);
        kop[2 * q] = e4m3x8_to_bf16(v[0], v[1]);
        kop[2 * q + 1] = e4m3x8_to_bf16(v[2], v[3]);
      }
    }
    const float sl = score_scale(p.scale_log2, descale(a.qd, a.qd_b, a.qd_h, b, h), descale(a.kd, a.kd_b, a.kd_h, b, h));

    float acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
    // A row tile is 2^hs heads of 32 >> hs consecutive tokens, the shape that needs
    // the fewest of them; row r is token r >> hs, head r & (2^hs - 1).
    int hs = 0, fewest = INT32_MAX;
    for (int e = 0; e <= 5 && (1 << e) < 2 * G; ++e) {
      const int n = ((r.n + (kRows >> e) - 1) >> (5 - e)) * ((G + (1 << e) - 1) >> e);
      if (n < fewest) {
        fewest = n;
        hs = e;
      }
    }
    const int toks = kRows >> hs, mask = (1 << hs) - 1;
    const int hgroups = (G + mask) >> hs, hend = hgroups << hs, tiles = ((r.n + toks - 1) >> (5 - hs)) * hgroups;
    // tiles from the first that holds a token that sees the first key
    const bool causal = a.causal;
    const int skip = causal ? min(max(k0 - ctx, 0), r.n) >> (5 - hs) : 0;
    int tile = skip * hgroups + turn;
    // tokens and heads that `t` < 9 tiles are (a wrap of the heads is the next tokens)
    auto apart = [&](int t, int& tok, int& hd) {
      tok = 0;
      for (; t >= hgroups; t -= hgroups) tok += toks;
      hd = t << hs;
    };
    int tok, hd, dt, dh;
    apart(turn, tok, hd);
    apart(split, dt, dh);
    tok += skip * toks;          // tok, hd: the tile computed next
    int tok_a = tok, hd_a = hd;  // the tile loaded next
    const uint8_t* q0 = p.q8 + int64_t(r.first) * p.q8_tok + int64_t(h) * G * p.q8_head;
    const float* lse0 = p.lse + int64_t(h) * G * p.lse_head_stride + r.first;
    const uint8_t* q_at = q0 + tok * p.q8_tok + hd * p.q8_head;
    const float* lse_at = lse0 + tok + hd * p.lse_head_stride;
    const int64_t q_step = dt * p.q8_tok + dh * p.q8_head, q_wrap = toks * p.q8_tok - hend * p.q8_head;
    const int64_t lse_step = dt + dh * p.lse_head_stride, lse_wrap = toks - hend * p.lse_head_stride;
    // loads: lane l takes chunk position l % 8 of rows 8 u + l / 8, chunk c of row t lies at c ^ (t & 7)
    const int lr = lane >> 3, lchunk = 16 * ((lane & 7) ^ lr);
    // (rows no closer than 128 bytes: offsets less their 1024 u, see load_lds_4k, stay positive)
    const bool near = p.near && p.q8_tok >= int64_t(kHead) << hs;
    uint32_t off_q[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int row = 8 * u + lr;
      off_q[u] = uint32_t((row >> hs) * p.q8_tok + (row & mask) * p.q8_head) + lchunk - 1024 * u;
    }
    const uint32_t off_lse = 4 * uint32_t((kk >> hs) + (kk & mask) * p.lse_head_stride);
    auto start = [&](int slot_no) {  // five loads: the rows, their lse
      const uint32_t slot = ring + uint32_t(slot_no) * kHalfSlot, lse_slot = lse_ring + uint32_t(slot_no * kRows * 4);
      if (__builtin_expect(near && tok_a + toks <= r.n && hd_a + mask < G, 1)) {
        load_lds_4k(slot, q_at, off_q);
        if (half == 0) load_lds_dword(lse_slot, lse_at, off_lse);
      } else {  // rows that are not there: any that is, they count for nothing
#pragma unroll 1
        for (int u = 0; u < 4; ++u) {
          const int row = 8 * u + lr;
          load_lds(slot + 1024 * u, q0 + min(tok_a + (row >> hs), r.n - 1) * p.q8_tok +
                                        min(hd_a + (row & mask), G - 1) * p.q8_head + lchunk);
        }
        if (half == 0)
          load_lds_dword(lse_slot, lse0 + min(hd_a + (kk & mask), G - 1) * p.lse_head_stride + min(tok_a + (kk >> hs), r.n - 1));
      }
      tok_a += dt;
      hd_a += dh;
      q_at += q_step;
      lse_at += lse_step;
      if (hd_a >= hend) {
        hd_a -= hend;
        tok_a += toks;
        q_at += q_wrap;
        lse_at += lse_wrap;
      }
    };
    auto pass = [&](int slot_no) {
      const uint32_t slot = ring + uint32_t(slot_no) * kHalfSlot;
      f32x16 y = {};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const u32x4 v = *lds_at<u32x4>(slot + uint32_t(128 * kk + 16 * ((2 * q + half) ^ (kk & 7))));
        const bf16x8 v0 = e4m3x8_to_bf16(v[0], v[1]), v1 = e4m3x8_to_bf16(v[2], v[3]);
        y = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kop[2 * q], v0, y, 0, 0, 0);
        y = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kop[2 * q + 1], v1, y, 0, 0, 0);
      }
      // lse log2(e), in two parts so that it is rounded once
      const float lse = *lds_at<float>(lse_ring + uint32_t(slot_no * kRows * 4) + 4 * kk);
      const float lse2 = __builtin_fmaf(lse, 0x1.715476p+0f, lse * 0x1.4ae0cp-26f);
#pragma unroll
      for (int n = 0; n < 16; ++n) y[n] = __builtin_fmaf(y[n], sl, -lse2);
      if (!(tok + toks <= r.n && hd + mask < G && (!causal || ctx + tok >= k0 + kTile - 1))) {
        // the last key the row sees, -1 for none
        const int i = tok + (kk >> hs), last = i < r.n && hd + (kk & mask) < G ? (causal ? ctx + i : full - 1) : -1;
        const int limit = last - k0 - 4 * half;
#pragma unroll
        for (int n = 0; n < 16; ++n) y[n] = 8 * (n >> 2) + (n & 3) <= limit ? y[n] : -__builtin_inff();
      }
#pragma unroll
      for (int n = 0; n < 16; ++n) acc[n] += __builtin_amdgcn_exp2f(y[n]);
      tok += dt;
      hd += dh;
      if (hd >= hend) {
        hd -= hend;
        tok += toks;
      }
      // every read of the slot is done before its next loads start
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    int ahead = tile, slot_no = 0, to = 0;
#pragma unroll 1
    for (; ahead < tiles && to < kManyRing - 1; ahead += split, ++to) {
      start(to);
    }
    to = kManyRing - 1;
#pragma unroll 1
    for (; tile < tiles; tile += split) {
      if (ahead < tiles) {
        start(to);
        ahead += split;
        wait_loads<5 * (kManyRing - 1)>();
      } else {
        wait_loads<0>();
      }
      pass(slot_no);
      slot_no = slot_no == kManyRing - 1 ? 0 : slot_no + 1;
      to = to == kManyRing - 1 ? 0 : to + 1;
    }

    const WeightArgs& o = args_again<WeightArgs>();
    float* scores = score_row(o, b, h);
    // the key of the lane's sum, two lanes a key
    const int idx = (lane >> 1) & 15, key_of = 8 * (idx >> 2) + 4 * half + (idx & 3);
    const float total = sum_lanes(acc, lane);
    if (split > 1) {
      if ((lane & 1) == 0) s_sum[wave][key_of] = total;
    } else if ((lane & 1) == 0 && k0 + key_of < L) {
      scores[k0 + key_of] = decayed(o, scores + k0 + key_of) + total;
    }
    if (split > 1) {
      __syncthreads();
      if (turn == 0) {  // the group's first wave joins its waves' sums
        const int key = k0 + lane;
        if (lane < kTile && key < L) {
          float sum = s_sum[wave][lane];
          for (int i = 1; i < split; ++i) sum += s_sum[wave + i][lane];
          scores[key] = decayed(o, scores + key) + sum;
        }
      }
      __syncthreads();
    }
  }
}

template <int Q_DT>
int quantize_queries(const WeightArgs& p, int64_t total_q, int64_t num_q_heads, uint8_t* q8, hipStream_t st) {
  hipLaunchKernelGGL((quantize_queries_kernel<Q_DT>), dim3(unsigned(ceil_div(total_q * num_q_heads * 8, kThreads))),
                     dim3(kThreads), 0, st, p, int(num_q_heads), q8);
  return check_launch("quantize_queries_kernel launch");
}

template <int Q_DT, bool OLD>
int launch_few_rows_old(const WeightArgs& p, hipStream_t st) {
  const DecodeArgs& a = p.a;
  // pages of a multiple of 8 keys whose rows lie within 32-bit offsets: the keys of a load share a page
  // (16 sequences of 8000: pages of 16 take 28 us, of 12 with a look-up a lane 40)
  const bool general = a.block_size % 8 != 0 || a.k_row < 0 || 8 * a.k_row >= (int64_t(1) << 31);
  const dim3 grid{unsigned(p.s.max_runs), 1u, 1u};
  if (general) hipLaunchKernelGGL((few_rows_kernel<Q_DT, OLD, true>), grid, dim3(kThreads), 0, st, p);
  else hipLaunchKernelGGL((few_rows_kernel<Q_DT, OLD, false>), grid, dim3(kThreads), 0, st, p);
  return check_launch("few_rows_kernel launch");
}

template <int Q_DT>
int launch_few_rows(const WeightArgs& p, hipStream_t st) {
  return p.decay != 0.0f ? launch_few_rows_old<Q_DT, true>(p, st) : launch_few_rows_old<Q_DT, false>(p, st);
}

}  // namespace

extern "C" {

int64_t psk_attention_weights_workspace_bytes(int64_t total_q, int64_t max_seqlen_q, int64_t num_q_heads,
                                              int64_t num_kv_heads, int q_dtype) {
  if (total_q < 0 || max_seqlen_q <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads ||
      max_seqlen_q > INT32_MAX / (num_q_heads / num_kv_heads) || total_q > INT32_MAX / num_q_heads)
    return PSK_E_ARG;
  const bool few = max_seqlen_q * (num_q_heads / num_kv_heads) <= kRows;
  return few || q_dtype == PSK_DTYPE_FP8_E4M3FN ? 0 : 16 + total_q * num_q_heads * kHead;
}

int psk_accumulate_attention_weights(float* scores, int64_t scores_seq_stride, int64_t scores_head_stride,
                                     int64_t scores_width, const void* q, int64_t q_tok_stride, int64_t q_head_stride,
                                     int q_dtype, const void* k_cache, const int64_t* k_strides, const float* lse,
                                     int64_t lse_head_stride, const int32_t* block_table, int64_t block_table_stride,
                                     int64_t block_table_width, const int32_t* seq_lens, int64_t num_seqs,
                                     int64_t num_q_heads, int64_t num_kv_heads, int64_t head_size, int64_t block_size,
                                     int64_t num_blocks, int64_t max_seq_len, int64_t total_q, int64_t max_seqlen_q,
                                     const int32_t* cu_seqlens_q, int causal, float softmax_scale, float decay,
                                     const float* q_descale, const float* k_descale, const int64_t* descale_strides,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
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
  p.s.num_seqs = int32_t(num_seqs);
  p.s.total_q = int32_t(total_q);
  p.s.heads = int32_t(num_kv_heads);
  p.s.idle = decay != 1.0f;
  p.s.width = int32_t(std::min<int64_t>(scores_width, INT32_MAX - 1024));
  p.scale_log2 = double(softmax_scale) * 1.4426950408889634;
  p.lse = lse;
  p.lse_head_stride = lse_head_stride;
  p.scores = scores;
  p.seq_stride = scores_seq_stride;
  p.head_stride = scores_head_stride;
  p.decay = decay;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t cus = device_cus();
  const int64_t rows = max_seqlen_q * a.heads;
  if (rows <= kRows) {
    p.s.step_shift = log2_exact(kStepKeys);
    // (64 / 16 sequences of 500 / 2000, us: runs of at least one unit 17 / 16, two 22 / 21;
    // 256 of 300, a job's start priced as one 27, two 33)
    p.s.over = 1;
    p.s.min_run = 1;
    p.s.max_runs = int32_t(xcd_rounds(2 * cus));  // resident at once
    p.hg = int32_t(std::min<int64_t>(num_kv_heads, kFewRows / (8 * ceil_div(rows, 8))));
    p.s.heads = int32_t(ceil_div(num_kv_heads, p.hg));
    switch (q_dtype) {
      case PSK_DTYPE_FP8_E4M3FN: return launch_few_rows<PSK_DTYPE_FP8_E4M3FN>(p, st);
      case PSK_DTYPE_BF16: return launch_few_rows<PSK_DTYPE_BF16>(p, st);
      case PSK_DTYPE_F16: return launch_few_rows<PSK_DTYPE_F16>(p, st);
      default: return launch_few_rows<PSK_DTYPE_F32>(p, st);
    }
  }
  const int64_t need = psk_attention_weights_workspace_bytes(total_q, max_seqlen_q, num_q_heads, num_kv_heads, q_dtype);
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(PSK_E_WORKSPACE, "workspace of %lld bytes, need %lld", (long long)workspace_bytes, (long long)need);
  if (need > 0) {
    if (total_q * num_q_heads >= int64_t(1) << 29) return fail(PSK_E_ARG, "%lld query rows", (long long)(total_q * num_q_heads));
    uint8_t* q8 = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~uintptr_t(15));
    p.q8 = q8;
    p.q8_tok = num_q_heads * kHead;
    p.q8_head = kHead;
    int e = PSK_OK;
    if (total_q > 0) {
      switch (q_dtype) {
        case PSK_DTYPE_BF16: e = quantize_queries<PSK_DTYPE_BF16>(p, total_q, num_q_heads, q8, st); break;
        case PSK_DTYPE_F16: e = quantize_queries<PSK_DTYPE_F16>(p, total_q, num_q_heads, q8, st); break;
        default: e = quantize_queries<PSK_DTYPE_F32>(p, total_q, num_q_heads, q8, st); break;
      }
    }
    if (e != PSK_OK) return e;
  } else {
    p.q8 = reinterpret_cast<const uint8_t*>(a.q);
    p.q8_tok = a.q_tok_stride;
    p.q8_head = a.q_head_stride;
  }
  const int64_t reach = INT32_MAX / (2 * kRows);
  p.near = p.q8_tok >= kHead && p.q8_tok <= reach && p.q8_head >= kHead && p.q8_head <= reach && lse_head_stride >= 0 &&
           lse_head_stride <= reach / 4;
  const int64_t keys = std::max<int64_t>(1, std::min(max_seq_len, scores_width));
  p.row_tiles = int32_t(ceil_div(rows, kRows));
  p.slots = int32_t(2 * cus);  // resident at once
  p.cus = int32_t(std::max<int64_t>(cus & ~7, 8));
  p.s.step_shift = log2_exact(kTile);
  p.s.over = 0;
  p.s.min_run = 1;
  p.s.max_runs = 1;
  const int64_t most = ceil_div(num_seqs * num_kv_heads * ceil_div(keys, kTile), p.cus) * p.cus;
  hipLaunchKernelGGL(many_rows_kernel, dim3(unsigned(std::min<int64_t>(most, 4 * p.slots))),
                     dim3(64 * kManyWaves), 0, st, p);
  return check_launch("many_rows_kernel launch");
}

}  // extern "C"
