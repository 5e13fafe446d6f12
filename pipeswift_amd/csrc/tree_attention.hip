// Attention of a tree of drafted tokens over the paged FP8 E4M3FN cache for
// MI355X (gfx950).
//
// Sequence b of L cached tokens has n drafted tokens, its last n; drafted token
// i sees every key before them and the drafted keys t whose bit of its mask is
// set.  Otherwise as the readers of paged_attention.hip and prefill_runs.hip:
// q~ = e4m3(q / qd), s = softmax_scale qd kd (q~ . K), out = vd softmax(s) V,
// lse = log sum exp s, Q K^T on the bf16 MFMA over exactly converted FP8
// operands, P V on the fp16 MFMA with V exact and P rounded once, float32 sums.
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
// that every weight is a finite fp16 value and the common path has no rescale.
//
// The work is cut into equal runs over sequences and kv heads (cached_queries.h).
// A run's piece that is not all of a job's keys leaves a partial record (maxima,
// sums, float32 accumulators); merge_tree_kernel joins a job's records in the
// order of its keys.
//
// C ABI: include/pipeswift_kv.h.  Nothing here allocates or synchronizes.

#include <algorithm>
#include <map>
#include <mutex>

#include "cached_queries.h"

using namespace psk_detail;

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows = 32;                  // query rows of a workgroup
constexpr int kTile = 32;                  // keys of a tile
constexpr uint32_t kHalfSlot = kTile * 128;  // bytes of a tile's K (its V follows)
constexpr uint32_t kSlot = 2 * kHalfSlot;
constexpr int kRing = 2;
constexpr int kPages = 1024;               // page ids a piece stages at a time
constexpr int kSlab = 4096 + 64;           // floats of 32 rows' partial result: accumulators, maxima, sums
constexpr int kMaxSlots = 512;             // resident workgroups the workspace is sized for
static_assert(kStepKeys == kTile * kWaves, "a step is a tile a wave");
static_assert(kPages >= kStepKeys + 1, "a step's pages fit, whatever the page size");

struct TreeArgs {
  DecodeArgs a;
  JobSpace s;
  double scale_log2;     // softmax_scale * log2(e)
  const int64_t* mask;
  int64_t mask_stride;   // words from a query token's mask to the next one's
  int32_t row_blocks;    // workgroups that share a run's keys
  float* records;        // [max_runs][row_blocks][2][kSlab]
};

__device__ __forceinline__ float* record(const TreeArgs& p, int64_t run, int block, int slot) {
  return p.records + ((run * p.row_blocks + block) * 2 + slot) * kSlab;
}

// Steps [from, to) of a job of `steps` that the units [lo, hi) of it pay for.
struct Piece {
  int32_t from, to;
};
__device__ __forceinline__ Piece piece_of(const JobSpace& s, int64_t lo, int64_t hi) {
  return Piece{int32_t(max(lo - s.over, int64_t(0))), int32_t(max(hi - s.over, int64_t(0)))};
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

template <int Q_DT, int OUT_DT>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2)))
tree_attention_kernel(TreeArgs p) {
  const DecodeArgs& a = p.a;
  __shared__ __attribute__((aligned(1024))) char s_ring[kWaves * kRing * kSlot];
  __shared__ int32_t s_pages[kPages];
  __shared__ float s_m[kWaves][kRows], s_l[kWaves][kRows];
  const int tid = int(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, kk = lane & 31;

  // workgroup w runs on XCD w % 8: the row blocks of a run on one, next to each other
  const int w = int(blockIdx.x);
  const int64_t j = int64_t(w / (8 * p.row_blocks)) * 8 + (w & 7);
  const int block = (w >> 3) % p.row_blocks;
  const StepCost cost = step_cost(a, p.s, lane);
  int64_t x = j * cost.run;
  if (j >= p.s.max_runs || x >= cost.total) return;
  const int64_t x_end = min(x + cost.run, cost.total);

  const uint32_t ring = (uint32_t)(size_t)(lvoid*)s_ring + uint32_t(wave * kRing) * kSlot;
  // loads: lane l takes chunk position l % 8 of keys 8 u + l / 8
  const int lr = lane >> 3, lchunk = 16 * ((lane & 7) ^ lr);
  // reads (see above)
  const uint32_t rd_k = uint32_t(128 * kk);
  const int ksw = kk & 7;
  const int vr = lane & 15, vg = (lane >> 4) & 1;
  const int vkey = 8 * (vr >> 3) + 4 * half + ((vr >> 1) & 3);  // of each 16
  const uint32_t rd_v = kHalfSlot + uint32_t(128 * vkey + 8 * (vr & 1));
  const int vsw = vkey & 7;

  int64_t before;
  int b = seq_of_unit(a, p.s, x, lane, before);
  while (x < x_end) {  // over the run's jobs
    const SeqRows r = seq_rows(a, p.s.total_q, b);
    const int L = cached_len(a, b);
    const int64_t job_cost = p.s.over + seq_steps(L);
    if (r.n <= 0 || x >= before + job_cost * p.s.heads) {
      if (r.n > 0) before += job_cost * p.s.heads;
      ++b;
      continue;
    }
    const int h = int((x - before) / job_cost);
    const int64_t at = before + h * job_cost;
    const int64_t hi = min(x_end, at + job_cost);
    const Piece c = piece_of(p.s, x - at, hi - at);
    x = hi;
    const int row0 = block * kRows;
    if (c.from >= c.to || row0 >= r.n * a.heads) continue;

    // the rows' queries
    const int ctx = L - r.n;
    const float qd = descale(a.qd, a.qd_b, a.qd_h, b, h);
    const float sl_signed = score_scale(p.scale_log2, qd, descale(a.kd, a.kd_b, a.kd_h, b, h));
    const float sl = __builtin_fabsf(sl_signed);  // a negative scale is applied as -q~ (exact)
    const int row = row0 + kk, i0 = row / a.heads;
    const bool live = i0 < r.n;
    const int64_t tok = int64_t(r.first) + (live ? i0 : 0);
    const int64_t* mask = p.mask + tok * p.mask_stride;
    bf16x8 qop[8];
    {
      const char* src = a.q + tok * a.q_tok_stride + int64_t(h * a.heads + (live ? row - i0 * a.heads : 0)) * a.q_head_stride;
      uint32_t q0[8], q1[8];
      load_query_as<Q_DT>(src, qd, 64 * half, q0);
      load_query_as<Q_DT>(src, qd, 64 * half + 32, q1);
      const uint32_t sign = sl_signed < 0.0f ? 0x80808080u : 0u;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        qop[t] = live ? e4m3x8_to_bf16(q0[2 * t] ^ sign, q0[2 * t + 1] ^ sign) : bf16x8{};
        qop[4 + t] = live ? e4m3x8_to_bf16(q1[2 * t] ^ sign, q1[2 * t + 1] ^ sign) : bf16x8{};
      }
    }
    float m = live ? kNegBig : -kNegBig, l = 0.0f;  // rows without a token keep every weight at 0
    f32x16 o[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) o[d] = f32x16{};

    const uint8_t* kbase = a.k + int64_t(h) * a.k_head + lchunk;
    const uint8_t* vbase = a.v + int64_t(h) * a.v_head + lchunk;
    const int n_tiles = (L + kTile - 1) / kTile;
    const int t_mask = max(ctx, 0) / kTile;  // tiles from here on need masks
    const int steps_per_window = int(min(int64_t(kPages - 1) * a.block_size / kStepKeys, int64_t(1) << 24));

    for (int s0 = c.from; s0 < c.to; s0 += steps_per_window) {
      const int s1 = min(c.to, s0 + steps_per_window);
      // the pages of the window's keys, missing ones as -1
      const int p0 = page_index(a, s0 * kStepKeys);
      const int p1 = page_index(a, int(min(int64_t(L), int64_t(s1) * kStepKeys)) - 1);
      __syncthreads();  // readers of the ring (the last piece's merge) and of the ids are done
      for (int i = tid; i <= p1 - p0; i += kThreads) {
        int32_t id = -1;
        if (p0 + i < a.bt_width) id = a.block_table[int64_t(b) * a.bt_stride + p0 + i];
        s_pages[i] = id < a.num_blocks ? id : -1;
      }
      __syncthreads();

      const int t_end = min(4 * s1, n_tiles);
      bool full = true;  // the newest tile's loads are all in flight
      auto issue = [&](int t, uint32_t slot) {
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
            load_lds(slot + 1024 * u, kbase + (int64_t(id[u]) * a.k_blk + int64_t(row[u]) * a.k_row));
            load_lds(slot + kHalfSlot + 1024 * u, vbase + (int64_t(id[u]) * a.v_blk + int64_t(row[u]) * a.v_row));
          } else {
            *lds_at<u32x4>(slot + 1024 * u + 16 * lane) = u32x4(0);
            *lds_at<u32x4>(slot + kHalfSlot + 1024 * u + 16 * lane) = u32x4(0);
          }
        }
      };

      auto read_v = [&](uint32_t slot, int u, int d) {
        return __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            lds_at<i32x2>(slot + rd_v + uint32_t(2048 * u + 16 * ((2 * d + vg) ^ vsw))));
      };
      // NaN values of keys that some row does not see (0 x NaN) must not reach
      // it: they leave the tile, and the rows that do see one become NaN in its
      // column, by the count of those they see.
      auto contain_nan = [&](uint32_t slot, uint32_t vis) {
        auto nan_bytes = [](uint32_t x) { return (((x & 0x7F7F7F7Fu) + 0x01010101u) >> 7) & 0x01010101u; };
        const uint32_t own = slot + kHalfSlot + uint32_t(16 * lane);
        uint32_t any = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const u32x4 v = *lds_at<u32x4>(own + 1024 * u);
          any |= nan_bytes(v[0]) | nan_bytes(v[1]) | nan_bytes(v[2]) | nan_bytes(v[3]);
        }
        if (__builtin_expect(!__any(any != 0), 1)) return;
#pragma unroll 1
        for (int u = 0; u < 2; ++u) {
          f16x8 seen;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            seen[i] = ((vis >> (16 * u + 8 * (i >> 2) + (i & 3))) & 1u) ? _Float16(1.0f) : _Float16(0.0f);
          }
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const i32x2 raw = read_v(slot, u, d);
            const f16x8 bad = e4m3x8_to_f16(nan_bytes(uint32_t(raw[0])) * 0x38u, nan_bytes(uint32_t(raw[1])) * 0x38u);  // 1.0
            const f32x16 count = __builtin_amdgcn_mfma_f32_32x32x16_f16(bad, seen, f32x16{}, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = count[i] > 0.0f ? __builtin_nanf("") : o[d][i];
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          u32x4 v = *lds_at<u32x4>(own + 1024 * u);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] &= ~(nan_bytes(v[i]) * 0xFFu);
          *lds_at<u32x4>(own + 1024 * u) = v;
        }
      };

      auto attend = [&](auto masked_tag, int t, uint32_t slot) {
        constexpr bool MASKED = decltype(masked_tag)::value;
        f32x16 y = {};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const u32x4 kw = *lds_at<u32x4>(slot + rd_k + uint32_t(16 * ((4 * half + q) ^ ksw)));
          y = __builtin_amdgcn_mfma_f32_32x32x16_bf16(e4m3x8_to_bf16(kw[0], kw[1]), qop[2 * q], y, 0, 0, 0);
          y = __builtin_amdgcn_mfma_f32_32x32x16_bf16(e4m3x8_to_bf16(kw[2], kw[3]), qop[2 * q + 1], y, 0, 0, 0);
        }
        uint32_t vis = 0xFFFFFFFFu;
        if constexpr (MASKED) {
          vis = (live ? visible(mask, ctx, r.n, t * kTile) : 0u) >> (4 * half);
          contain_nan(slot, vis);
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
          top = __builtin_fmaxf(top, __shfl_xor(top, 32));
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
          uint32_t pw[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            pw[i] = __builtin_bit_cast(uint32_t,
                                       __builtin_convertvector((f32x2{w[8 * u + 2 * i], w[8 * u + 2 * i + 1]}), f16x2));
          const f16x8 pop = __builtin_bit_cast(f16x8, u32x4{pw[0], pw[1], pw[2], pw[3]});
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const i32x2 raw = read_v(slot, u, d);
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(e4m3x8_to_f16(uint32_t(raw[0]), uint32_t(raw[1])), pop, o[d], 0, 0,
                                                          0);
          }
        }
      };

      int t = kWaves * s0 + wave;
      uint32_t slot = ring;
      if (t < t_end) issue(t, slot);
      bool next_full = false;
      if (t + kWaves < t_end) {
        issue(t + kWaves, slot + kSlot);
        next_full = full;
      }
      auto step = [&](auto masked_tag) {
        // the tile's own loads: the next one's eight may stay in flight
        if (t + kWaves < t_end && next_full) wait_loads<8>(); else wait_loads<0>();
        attend(masked_tag, t, slot);
        if (t + 2 * kWaves < t_end) {
          issue(t + 2 * kWaves, slot);
          next_full = full;
        }
        slot = slot == ring ? ring + kSlot : ring;
        t += kWaves;
      };
      while (t < min(t_end, t_mask)) step(std::false_type{});
      while (t < t_end) step(std::true_type{});
    }

    // the four waves' results, joined in the order of the waves
    const float lt = l + __shfl_xor(l, 32);
    if (lane < 32) {
      s_m[wave][lane] = m;
      s_l[wave][lane] = lt;
    }
    __syncthreads();  // every wave has left its ring, and wrote its maxima
    const bool whole = c.from == 0 && c.to == int(job_cost) - p.s.over;
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
    float* rec = record(p, j, block, c.from == 0 ? 1 : 0);
#pragma unroll
    for (int i = 0; i < 16 / kWaves; ++i) {
      const int q = wave + kWaves * i;
      f32x4 v = s_o[q * 64 + lane];
#pragma unroll
      for (int u = 1; u < kWaves; ++u) v += s_o[(u * 16 + q) * 64 + lane];
      if (whole) finish<OUT_DT>(p, r, b, h, row, q, lane, v, top, sum);
      else *reinterpret_cast<f32x4*>(rec + (q * 64 + lane) * 4) = v;
    }
    if (!whole && wave == 0 && lane < 32) {
      rec[4096 + lane] = top;
      rec[4096 + 32 + lane] = sum;
    }
  }
}

// The records of a job joined: a wave per (job, 32 rows, 8 columns).
template <int OUT_DT>
__global__ void __launch_bounds__(256) merge_tree_kernel(TreeArgs p) {
  const DecodeArgs& a = p.a;
  const int lane = int(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int kk = lane & 31;
  // the wave's task: column group q of row block `block` of job (b, h)
  const int64_t task = int64_t(blockIdx.x) * 4 + wave;
  const int q = int(task & 15);
  const int64_t rest = task >> 4;
  const int block = int(rest % p.row_blocks);
  const int64_t job = rest / p.row_blocks;
  const int h = int(job % p.s.heads), b = int(job / p.s.heads);
  if (b >= p.s.num_seqs) return;
  const SeqRows r = seq_rows(a, p.s.total_q, b);
  const int row = kRows * block + kk;
  if (kRows * block >= r.n * a.heads) return;
  const StepCost cost = step_cost(a, p.s, lane);
  const int64_t job_cost = p.s.over + seq_steps(cached_len(a, b));
  const int64_t at = units_before(a, p.s, b, lane) + h * job_cost;
  const int64_t j0 = at / cost.run, j1 = (at + job_cost - 1) / cost.run;
  const int32_t steps = int32_t(job_cost) - p.s.over;

  float top = kNegBig, sum = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t j = j0; j <= j1; ++j) {
    const Piece c = piece_of(p.s, max(j * cost.run - at, int64_t(0)), min((j + 1) * cost.run - at, job_cost));
    if (c.from >= c.to) continue;
    if (c.from == 0 && c.to == steps) return;  // one run had it all and wrote the rows
    const float* rec = record(p, j, block, c.from == 0 ? 1 : 0);
    const float m = rec[4096 + kk], l = rec[4096 + 32 + kk];
    const f32x4 v = *reinterpret_cast<const f32x4*>(rec + (q * 64 + lane) * 4);
    const float up = __builtin_fmaxf(top, m);
    const float f0 = __builtin_amdgcn_exp2f(top - up), f1 = __builtin_amdgcn_exp2f(m - up);
    top = up;
    sum = sum * f0 + l * f1;
    o = o * f0 + v * f1;
  }
  finish<OUT_DT>(p, r, b, h, row, q, lane, o, top, sum);
}

// Workgroups resident at once: two per CU (LDS and registers).
int64_t tree_slots() {
  static std::mutex mu;
  static std::map<int, int64_t> cache;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return kMaxSlots;
  std::lock_guard<std::mutex> lock(mu);
  auto it = cache.find(dev);
  if (it != cache.end()) return it->second;
  int cus = 0;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) return kMaxSlots;
  return cache[dev] = std::min<int64_t>(2 * cus, kMaxSlots);
}

struct TreeShape {
  int64_t row_blocks, max_runs;
};
TreeShape tree_shape(int64_t rows, int64_t slots) {
  TreeShape s;
  s.row_blocks = ceil_div(rows, kRows);
  // runs in whole rounds of the eight XCDs
  s.max_runs = std::max<int64_t>(8, slots / s.row_blocks / 8 * 8);
  return s;
}

template <int Q_DT, int OUT_DT>
int launch_tree(const TreeArgs& p, hipStream_t st) {
  hipLaunchKernelGGL((tree_attention_kernel<Q_DT, OUT_DT>), dim3(unsigned(p.s.max_runs * p.row_blocks)), dim3(kThreads), 0,
                     st, p);
  if (const int e = check_launch("tree_attention_kernel launch"); e != PSK_OK) return e;
  const int64_t tasks = int64_t(p.s.num_seqs) * p.s.heads * p.row_blocks * 16;
  hipLaunchKernelGGL((merge_tree_kernel<OUT_DT>), dim3(unsigned(tasks / 4)), dim3(256), 0, st, p);
  return check_launch("merge_tree_kernel launch");
}

template <int Q_DT>
int launch_tree_q(const TreeArgs& p, int out_dtype, hipStream_t st) {
  return out_dtype == PSK_DTYPE_BF16 ? launch_tree<Q_DT, PSK_DTYPE_BF16>(p, st) : launch_tree<Q_DT, PSK_DTYPE_F32>(p, st);
}

}  // namespace

extern "C" {

int64_t psk_paged_tree_workspace_len(int64_t num_seqs, int64_t total_q, int64_t max_seqlen_q, int64_t num_q_heads,
                                     int64_t num_kv_heads, int64_t max_seq_len) {
  if (num_seqs < 0 || total_q < 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads ||
      max_seqlen_q <= 0 || max_seqlen_q > INT32_MAX / (num_q_heads / num_kv_heads) || max_seq_len < 0)
    return PSK_E_ARG;
  const TreeShape s = tree_shape(max_seqlen_q * (num_q_heads / num_kv_heads), kMaxSlots);
  return 4 + s.max_runs * s.row_blocks * 2 * kSlab;
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
  if (!v_cache || !v_strides || !tree_mask || !out || !workspace) return fail(PSK_E_ARG, "NULL pointer");
  const uint64_t v_align[4] = {uint64_t(uintptr_t(v_cache)), uint64_t(v_strides[0]), uint64_t(v_strides[1]),
                               uint64_t(v_strides[2])};
  if (common_align(v_align, 4, 16) < 16) return fail(PSK_E_ARG, "K/V caches need 16-byte aligned bases and strides");
  const int osz = dtype_size(out_dtype);
  const uint64_t o_align[3] = {uint64_t(uintptr_t(out)), uint64_t(out_tok_stride * osz),
                               uint64_t(out_head_stride * osz)};
  if (common_align(o_align, 3, 4 * osz) < 4 * osz)
    return fail(PSK_E_ARG, "output rows need %d-byte alignment", 4 * osz);
  const int64_t need = psk_paged_tree_workspace_len(num_seqs, total_q, max_seqlen_q, num_q_heads, num_kv_heads, max_seq_len);
  if (workspace_len < need)
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
  p.s.over = 2;
  p.s.max_runs = int32_t(s.max_runs);
  p.s.min_run = 3;
  p.row_blocks = int32_t(s.row_blocks);
  p.records = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~uintptr_t(15));
  if (num_seqs * num_kv_heads * s.row_blocks > INT32_MAX / 16 || s.max_runs * s.row_blocks > INT32_MAX)
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
