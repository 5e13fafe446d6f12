// RMS norms of the query and key heads with the rotation of their positions, and
// the append of K and V, in one pass for MI355X (gfx950).
//
// For a token's head x of D elements, with a weight w (or none: no norm):
//   y = x rsqrt(mean x^2 + eps) w
// and for pair i of the first R elements, (a, b) = (y_i, y_(i + R/2)) or, interleaved,
// (y_2i, y_(2i + 1)):  (a c - b s, b c + a s),  c = T[p, i], s = T[p, R/2 + i],
// T the caller's table of cosines and sines and p the token's position on the pair's
// axis.  The result is rounded once to the input's type; K then goes to the cache as
// psk_reshape_and_cache (or its 4-bit form) would write that, V as it is.
//
// A token is a wave's, or a workgroup's where the tokens are few.  A lane holds eight
// elements of a head (so a head is a power of two of lanes, LPR, and its sum of
// squares a few DPP steps), and the same eight of every head it takes: the factors of
// its elements, w c and w s, are made once for the queries and once for the keys.  An
// element's partner comes from its lane by ds_bpermute as it was loaded; its norm is the
// row's own.  The lanes of a head past its size (sizes that are no power of two) idle.
//
// Bound by memory where the tokens are many: 8192 tokens of 32 + 8 + 8 bf16 heads of 128
// with the append take 49 us, 4.15 TB/s read and written, where a plain elementwise pass over a
// large tensor reaches 6.2; 20011 of 8 + 2 heads on three axes 28 us, 4.1 TB/s.  64 tokens take 5 us, the time of a launch and of
// the chain from the position over the table to the store.  A wave a head, with the
// factors made anew for each, took 114 us for the prompt.
//
// C ABI: include/pipeswift_kv.h.  Nothing here allocates or synchronizes.

#include <cmath>
#include <type_traits>

#include "mxfp4.h"

using namespace psk_detail;

namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 4;  // heads of a lane loaded before the first is computed
constexpr int kAxes = 4;
// Tokens from which on a wave takes a whole token, so that the factors are made once: 2048 of 48
// heads take 15.0 us so and 15.5 by four waves each, 8192 37 and 47, 64 9.7 and 5.3 (the same
// inputs pass after pass, which the caches hold in part: with others each time 8192 take 49).
constexpr int64_t kManyTokens = 2048;

enum CacheKind { kNoCache = 0, kCopy = 1, kFp8 = 2, kMx4 = 3 };

struct NormRopeArgs {
  const char* in[3];                // q, k, v
  int64_t in_tok[3], in_head[3];    // bytes
  char* out[2];                     // q, k; NULL: not written
  int64_t out_tok[2], out_head[2];
  const char* weight[2];            // NULL: no norm
  int32_t weight_f32, weight_wide;  // on 16-byte boundaries
  int32_t tokens_shift;             // log2 of the tokens of a workgroup (of four waves)
  int64_t num_tokens;
  float eps;
  int32_t num_q, num_kv, head_size, chunks;
  const char* pos;
  int64_t pos_axis;                 // elements
  int32_t pos64, axes;
  int32_t axis_end[kAxes];          // pairs before the end of each axis
  int32_t whole_axes;               // a lane's pairs share an axis and its factors lie on 16-byte boundaries
  const float* table;
  int64_t table_stride, num_positions;
  int32_t half, interleaved;        // pairs
  char* cache[2];
  int64_t blk[2], row[2], head[2];  // bytes
  const int64_t* slots;
  int64_t num_slots, block_size;
  int32_t bs_shift;
  const float* scale[2];
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, false));
}

// The sum over LPR consecutive lanes, in each of them.
template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
  x = dpp_add<0xB1>(x);                       // quad_perm [1,0,3,2]
  x = dpp_add<0x4E>(x);                       // quad_perm [2,3,0,1]
  if constexpr (LPR >= 8) x = dpp_add<0x141>(x);   // row_half_mirror
  if constexpr (LPR >= 16) x = dpp_add<0x140>(x);  // row_mirror
  if constexpr (LPR >= 32) x += __shfl_xor(x, 16);
  if constexpr (LPR >= 64) x += __shfl_xor(x, 32);
  return x;
}

// 1 / sqrt(x); v_rsq_f32 takes a subnormal x (a small row without an eps) for zero.
__device__ __forceinline__ float rsqrt_any(float x) {
  const bool small = x < 0x1p-100f;
  return __builtin_amdgcn_rsqf(small ? x * 0x1p64f : x) * (small ? 0x1p32f : 1.0f);
}

// Eight elements as they were loaded.
template <int DT>
struct Eight {
  static constexpr int kWords = 2 * Elt<DT>::kSize;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const char* p) {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const u32x4 x = vload<16>(p + 16 * i);
      __builtin_memcpy(w + 4 * i, &x, 16);
    }
  }
  __device__ __forceinline__ void store(char* p) const {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      u32x4 x;
      __builtin_memcpy(&x, w + 4 * i, 16);
      vstore<16>(p + 16 * i, x);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
    typename Elt<DT>::Bits e[8];
    __builtin_memcpy(e, w, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elt<DT>::to_f32(e[i]);
  }
  __device__ __forceinline__ void pack(const float (&x)[8]) {
    if constexpr (DT == PSK_DTYPE_BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x[2 * i], x[2 * i + 1]}), mx_bf16x2));
    } else {
      typename Elt<DT>::Bits e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = Elt<DT>::from_f32(x[i]);
      __builtin_memcpy(w, e, sizeof(e));
    }
  }
  __device__ __forceinline__ Eight from_lane(int lane) const {
    Eight y;
#pragma unroll
    for (int i = 0; i < kWords; ++i) y.w[i] = uint32_t(__builtin_amdgcn_ds_bpermute(lane << 2, int(w[i])));
    return y;
  }
};

// Eight elements of a head into its cache row, as the append writes them.
template <int DT, int KIND>
__device__ __forceinline__ void put(const Eight<DT>& x, char* row, int chunk, int head_size, const QScale& qs, bool live) {
  if constexpr (KIND == kCopy) {
    if (live) x.store(row + chunk * 8 * Elt<DT>::kSize);
  } else if constexpr (KIND == kFp8) {
    constexpr int E = 16 / Elt<DT>::kSize;
    using QC = QuantConv<DT, E>;
    uint8_t bytes[8];
#pragma unroll
    for (int i = 0; i < 8 / E; ++i) {
      typename QC::In v;
      __builtin_memcpy(&v, x.w + 4 * i, 16);
      const typename QC::Out y = QC::apply(v, qs);
      __builtin_memcpy(bytes + E * i, &y, E);
    }
    u32x2 y;
    __builtin_memcpy(&y, bytes, 8);
    if (live) vstore<8>(row + 8 * chunk, y);
  } else if constexpr (KIND == kMx4) {
    typename Elt<DT>::Bits e[8];
    __builtin_memcpy(e, x.w, sizeof(e));
    uint32_t byte;
    const uint32_t codes = mx_quantize8<DT>(e, byte);
    if (live) mx_store8(row, chunk, head_size, codes, byte);
  }
}

template <int DT, int LPR, int KIND>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(NormRopeArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = int(threadIdx.x) & 63;
  const int64_t t = (int64_t(blockIdx.x) << a.tokens_shift) + (wave >> (2 - a.tokens_shift));
  if (t >= a.num_tokens) return;
  const int c = lane & (LPR - 1);          // this lane's eight elements of a head
  const bool in_row = c < a.chunks;
  constexpr int kRows = 64 / LPR;          // heads of a unit
  // units of queries, keys and values: a wave takes every `stride`-th
  const int stride = 4 >> a.tokens_shift, first_unit = wave & (stride - 1);
  const int q_units = (a.num_q + kRows - 1) / kRows, kv_units = (a.num_kv + kRows - 1) / kRows;
  const int units = q_units + kv_units * (KIND == kNoCache ? 1 : 2);
  const int d0 = 8 * c;
  const bool turns = d0 < 2 * a.half;

  struct Unit {
    int which, h;  // uniform; this lane's head
    bool live;     // the head is there
  };
  auto unit_of = [&](int u) {
    Unit x;
    x.which = u < q_units ? 0 : u < q_units + kv_units ? 1 : 2;
    x.h = (u - (x.which == 0 ? 0 : x.which == 1 ? q_units : q_units + kv_units)) * kRows + lane / LPR;
    x.live = u < units && x.h < (x.which == 0 ? a.num_q : a.num_kv);
    return x;
  };
  // the first heads are on their way while the factors are made
  Eight<DT> x[kBatch];
  auto load = [&](int u0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const Unit y = unit_of(u0 + i * stride);
      x[i].zero();
      if (y.live && in_row) x[i].load(a.in[y.which] + t * a.in_tok[y.which] + y.h * a.in_head[y.which] + d0 * Elt<DT>::kSize);
    }
  };
  load(first_unit);

  int64_t slot = -1;
  if constexpr (KIND != kNoCache) slot = a.slots[t];

  // cosine and signed sine of each element's pair; a position outside the table gives NaN
  float cs[8], sn[8];
  const bool first = d0 < a.half;
  // the chunk that holds the other halves of its pairs
  const int partner = a.interleaved || !turns ? c : first ? c + a.half / 8 : c - a.half / 8;
  {
    const int i0 = a.interleaved ? d0 / 2 : first ? d0 : d0 - a.half;
    auto position = [&](int axis) {
      const int64_t at = axis * a.pos_axis + t;
      return a.pos64 ? reinterpret_cast<const int64_t*>(a.pos)[at] : int64_t(reinterpret_cast<const int32_t*>(a.pos)[at]);
    };
    auto axis_of = [&](int i) {
      int axis = 0;
#pragma unroll
      for (int k = 0; k < kAxes - 1; ++k) axis += k < a.axes - 1 && i >= a.axis_end[k];
      return axis;
    };
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      cs[j] = 1.0f;
      sn[j] = 0.0f;
    }
    if (turns) {
      const int n = a.interleaved ? 4 : 8;
      float cj[8], sj[8];
      if (a.whole_axes) {
        const int64_t p = position(axis_of(i0));
        const bool known = p >= 0 && p < a.num_positions;
        const char* row = reinterpret_cast<const char*>(a.table + (known ? p : 0) * a.table_stride + i0);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          if (4 * q < n) {
            const u32x4 cv = vload<16>(row + 16 * q), sv = vload<16>(row + 16 * q + 4 * a.half);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              cj[4 * q + j] = known ? __uint_as_float(cv[j]) : __builtin_nanf("");
              sj[4 * q + j] = known ? __uint_as_float(sv[j]) : __builtin_nanf("");
            }
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j < n) {
            const int64_t p = position(axis_of(i0 + j));
            const bool known = p >= 0 && p < a.num_positions;
            const float* row = a.table + (known ? p : 0) * a.table_stride + i0 + j;
            cj[j] = known ? row[0] : __builtin_nanf("");
            sj[j] = known ? row[a.half] : __builtin_nanf("");
          }
        }
      }
      if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          cs[j] = cj[j / 2];
          sn[j] = (j & 1) ? sj[j / 2] : -sj[j / 2];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          cs[j] = cj[j];
          sn[j] = first ? -sj[j] : sj[j];
        }
      }
    }
  }
  // w c of each element and w s of its partner, for queries and keys
  float wc[2][8], ws[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float w[8], wp[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = wp[j] = 1.0f;
    if (a.weight[k] && in_row) {
      auto get = [&](int at, float (&y)[8]) {
        if (a.weight_f32) {
          typename Elt<PSK_DTYPE_F32>::Bits e[8];
          load8<PSK_DTYPE_F32>(a.weight[k] + 4 * at, a.weight_wide, e);
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = Elt<PSK_DTYPE_F32>::to_f32(e[j]);
        } else {
          typename Elt<DT>::Bits e[8];
          load8<DT>(a.weight[k] + Elt<DT>::kSize * at, a.weight_wide, e);
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = Elt<DT>::to_f32(e[j]);
        }
      };
      get(d0, w);
      if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < 8; ++j) wp[j] = w[j ^ 1];
      } else {
        get(8 * partner, wp);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      wc[k][j] = w[j] * cs[j];
      ws[k][j] = wp[j] * sn[j];
    }
  }
  int64_t page = 0, off = 0;
  const bool cached = KIND != kNoCache && slot >= 0 && slot < a.num_slots;
  if (cached) {
    page = a.bs_shift >= 0 ? slot >> a.bs_shift : slot / a.block_size;
    off = slot - page * a.block_size;
  }
  const int from = lane - c + partner;  // the partner's lane
  QScale qs[2] = {};
  if constexpr (KIND == kFp8) {
#pragma unroll
    for (int k = 0; k < 2; ++k) qs[k] = make_qscale_uniform(a.scale[k] ? *a.scale[k] : 1.0f);
  }

  // a unit of queries (0) or keys (1)
  auto turn = [&](auto kind, const Eight<DT>& raw, const Unit& y) {
    constexpr int K = decltype(kind)::value;
    float v[8], vp[8];
    raw.unpack(v);
    if (a.interleaved) {
#pragma unroll
      for (int j = 0; j < 8; ++j) vp[j] = v[j ^ 1];
    } else {
      raw.from_lane(from).unpack(vp);
    }
    float rstd = 1.0f;
    if (a.weight[K]) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(v[j], v[j], sum);
      rstd = rsqrt_any(row_sum<LPR>(sum) / float(a.head_size) + a.eps);
    }
    float z[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float own = v[j] * rstd * wc[K][j];
      z[j] = turns ? __builtin_fmaf(vp[j] * rstd, ws[K][j], own) : own;
    }
    Eight<DT> packed;
    packed.pack(z);
    if (a.out[K] && y.live && in_row)
      packed.store(a.out[K] + t * a.out_tok[K] + y.h * a.out_head[K] + d0 * Elt<DT>::kSize);
    if constexpr (K == 1 && KIND != kNoCache)
      put<DT, KIND>(packed, a.cache[0] + page * a.blk[0] + off * a.row[0] + y.h * a.head[0], c, a.head_size, qs[0],
                    cached && y.live && in_row);
  };
  for (int u0 = first_unit; u0 < units; u0 += kBatch * stride) {
    if (u0 > first_unit) load(u0);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (u0 + i * stride >= units) break;
      const Unit y = unit_of(u0 + i * stride);
      if (y.which == 0) {
        turn(std::integral_constant<int, 0>{}, x[i], y);
      } else if (y.which == 1) {
        turn(std::integral_constant<int, 1>{}, x[i], y);
      } else if constexpr (KIND != kNoCache) {
        put<DT, KIND>(x[i], a.cache[1] + page * a.blk[1] + off * a.row[1] + y.h * a.head[1], c, a.head_size, qs[1],
                      cached && y.live && in_row);
      }
    }
  }
}

template <int DT, int LPR>
void launch_kind(const NormRopeArgs& a, int kind, int64_t tokens, hipStream_t st) {
  const dim3 grid{unsigned(ceil_div(tokens, int64_t(1) << a.tokens_shift)), 1u, 1u};
  switch (kind) {
    case kNoCache: hipLaunchKernelGGL((norm_rope_kernel<DT, LPR, kNoCache>), grid, dim3(kThreads), 0, st, a); break;
    case kCopy: hipLaunchKernelGGL((norm_rope_kernel<DT, LPR, kCopy>), grid, dim3(kThreads), 0, st, a); break;
    case kFp8: hipLaunchKernelGGL((norm_rope_kernel<DT, LPR, kFp8>), grid, dim3(kThreads), 0, st, a); break;
    default: hipLaunchKernelGGL((norm_rope_kernel<DT, LPR, kMx4>), grid, dim3(kThreads), 0, st, a); break;
  }
}

template <int DT>
void launch_rows(const NormRopeArgs& a, int kind, int64_t tokens, hipStream_t st) {
  if (a.chunks <= 4) launch_kind<DT, 4>(a, kind, tokens, st);
  else if (a.chunks <= 8) launch_kind<DT, 8>(a, kind, tokens, st);
  else if (a.chunks <= 16) launch_kind<DT, 16>(a, kind, tokens, st);
  else if (a.chunks <= 32) launch_kind<DT, 32>(a, kind, tokens, st);
  else launch_kind<DT, 64>(a, kind, tokens, st);
}

}  // namespace

extern "C" {

int psk_norm_rope(const void* q, const void* k, const void* v, void* q_out, void* k_out, void* key_cache, void* value_cache,
                  const int64_t* strides, int dtype, int64_t num_tokens, int64_t num_q_heads, int64_t num_kv_heads,
                  int64_t head_size, const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                  const void* positions, int position_bytes, int64_t position_axis_stride, int64_t num_axes,
                  const int64_t* sections, const float* cos_sin, int64_t cos_sin_stride, int64_t num_positions,
                  int64_t rot_dim, int interleaved, int cache_dtype, const int64_t* slot_mapping, int64_t block_size,
                  int64_t num_blocks, const float* k_scale, const float* v_scale, void* stream) {
  begin_device_call();
  if (num_tokens < 0 || num_tokens > INT32_MAX || num_q_heads < 0 || num_kv_heads < 0 || num_q_heads + num_kv_heads <= 0 ||
      num_q_heads > 65536 || num_kv_heads > 65536)
    return fail(PSK_E_ARG, "bad sizes: num_tokens=%lld q heads %lld kv heads %lld", (long long)num_tokens,
                (long long)num_q_heads, (long long)num_kv_heads);
  if (head_size <= 0 || head_size % 8 || head_size > 512)
    return fail(PSK_E_ARG, "head_size %lld must be a multiple of 8, at most 512", (long long)head_size);
  const int step = interleaved ? 8 : 16;
  if (rot_dim <= 0 || rot_dim > head_size || rot_dim % step)
    return fail(PSK_E_ARG, "rot_dim %lld must be a multiple of %d, at most the head's %lld", (long long)rot_dim, step,
                (long long)head_size);
  if (dtype != PSK_DTYPE_F32 && dtype != PSK_DTYPE_F16 && dtype != PSK_DTYPE_BF16)
    return fail(PSK_E_DTYPE, "queries and keys are bf16, f16 or f32 (got %d)", dtype);
  if (weight_dtype != dtype && weight_dtype != PSK_DTYPE_F32)
    return fail(PSK_E_DTYPE, "weights have the queries' type or f32 (got %d)", weight_dtype);
  if (num_axes < 1 || num_axes > kAxes) return fail(PSK_E_ARG, "%lld position axes (1 to %d)", (long long)num_axes, kAxes);
  if (position_bytes != 4 && position_bytes != 8) return fail(PSK_E_DTYPE, "positions are int32 or int64");
  if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail(PSK_E_ARG, "eps is negative or not finite");
  if (num_positions <= 0 || cos_sin_stride < rot_dim)
    return fail(PSK_E_ARG, "a table of %lld positions with rows of %lld", (long long)num_positions,
                (long long)cos_sin_stride);
  const bool cache = key_cache != nullptr || value_cache != nullptr;
  int kind = kNoCache;
  if (cache) {
    if (cache_dtype == dtype) kind = kCopy;
    else if (cache_dtype == PSK_DTYPE_FP8_E4M3FN) kind = kFp8;
    else if (cache_dtype == PSK_DTYPE_MXFP4) kind = kMx4;
    else return fail(PSK_E_DTYPE, "cache dtype %d for rows of %d", cache_dtype, dtype);
    if (kind == kMx4 && head_size % kMxGroup)
      return fail(PSK_E_ARG, "a 4-bit cache takes heads of a multiple of %d (got %lld)", kMxGroup, (long long)head_size);
    if (block_size <= 0 || num_blocks < 0) return fail(PSK_E_ARG, "bad cache geometry");
  }
  if (num_tokens == 0) return PSK_OK;
  if (!strides || (num_q_heads && (!q || !q_out)) || (num_kv_heads && !k) || !positions || !cos_sin ||
      (num_axes > 1 && !sections))
    return fail(PSK_E_ARG, "NULL pointer");
  if (cache && (!key_cache || !value_cache || !v || !slot_mapping)) return fail(PSK_E_ARG, "NULL pointer");
  if (!cache && num_kv_heads && !k_out) return fail(PSK_E_ARG, "NULL pointer");

  NormRopeArgs a{};
  const int esz = dtype_size(dtype);
  uint64_t align = 0;
  const void* in[3] = {q, k, v};
  for (int i = 0; i < (cache ? 3 : 2); ++i) {
    if (i == 0 ? num_q_heads == 0 : num_kv_heads == 0) continue;
    a.in[i] = static_cast<const char*>(in[i]);
    a.in_tok[i] = strides[2 * i] * esz;
    a.in_head[i] = strides[2 * i + 1] * esz;
    align |= uint64_t(uintptr_t(in[i])) | uint64_t(a.in_tok[i]) | uint64_t(a.in_head[i]);
  }
  void* out[2] = {q_out, k_out};
  for (int i = 0; i < 2; ++i) {
    if (!out[i] || (i == 0 ? num_q_heads == 0 : num_kv_heads == 0)) continue;
    a.out[i] = static_cast<char*>(out[i]);
    a.out_tok[i] = strides[6 + 2 * i] * esz;
    a.out_head[i] = strides[7 + 2 * i] * esz;
    align |= uint64_t(uintptr_t(out[i])) | uint64_t(a.out_tok[i]) | uint64_t(a.out_head[i]);
  }
  if (align & 15) return fail(PSK_E_ARG, "heads must start on 16-byte boundaries");
  if (cache) {
    void* ca[2] = {key_cache, value_cache};
    const int csz = kind == kMx4 ? 1 : dtype_size(cache_dtype);
    uint64_t calign = 0;
    for (int i = 0; i < 2; ++i) {
      a.cache[i] = static_cast<char*>(ca[i]);
      a.blk[i] = strides[10 + 3 * i] * csz;
      a.row[i] = strides[11 + 3 * i] * csz;
      a.head[i] = strides[12 + 3 * i] * csz;
      calign |= uint64_t(uintptr_t(ca[i])) | uint64_t(a.blk[i]) | uint64_t(a.row[i]) | uint64_t(a.head[i]);
    }
    const uint64_t need = kind == kMx4 ? 4 : kind == kFp8 ? 8 : 16;
    if (calign & (need - 1)) return fail(PSK_E_ARG, "cache rows must start on %d-byte boundaries", int(need));
    const int64_t row_bytes = kind == kMx4 ? mx_entry_bytes(head_size) : head_size * csz;
    for (int i = 0; i < 2; ++i)
      if ((num_kv_heads > 1 && a.head[i] < row_bytes) || (block_size > 1 && a.row[i] < row_bytes))
        return fail(PSK_E_ARG, "cache strides are shorter than the %lld-byte row", (long long)row_bytes);
    if (kind != kFp8 && (k_scale || v_scale)) return fail(PSK_E_ARG, "scales only apply to an fp8 cache");
    a.slots = slot_mapping;
    a.block_size = block_size;
    a.num_slots = num_blocks * block_size;
    a.bs_shift = log2_exact(block_size);
    a.scale[0] = k_scale;
    a.scale[1] = v_scale;
  }
  a.weight[0] = static_cast<const char*>(q_weight);
  a.weight[1] = static_cast<const char*>(k_weight);
  a.weight_f32 = weight_dtype == PSK_DTYPE_F32;
  a.weight_wide = ((uint64_t(uintptr_t(q_weight)) | uint64_t(uintptr_t(k_weight))) & 15) == 0;
  a.num_tokens = num_tokens;
  a.tokens_shift = num_tokens >= kManyTokens ? 2 : 0;
  a.eps = eps;
  a.num_q = int32_t(num_q_heads);
  a.num_kv = int32_t(num_kv_heads);
  a.head_size = int32_t(head_size);
  a.chunks = int32_t(head_size / 8);
  a.pos = static_cast<const char*>(positions);
  a.pos_axis = position_axis_stride;
  a.pos64 = position_bytes == 8;
  a.axes = int32_t(num_axes);
  a.half = int32_t(rot_dim / 2);
  a.interleaved = interleaved ? 1 : 0;
  const int per_lane = interleaved ? 4 : 8;
  a.whole_axes = ((uint64_t(uintptr_t(cos_sin)) | uint64_t(cos_sin_stride * 4) | uint64_t(a.half * 4)) & 15) == 0;
  int64_t end = 0;
  for (int i = 0; i < int(num_axes); ++i) {
    const int64_t n = num_axes == 1 ? a.half : sections[i];
    if (n < 0 || n > a.half) return fail(PSK_E_ARG, "section %d of %lld pairs", i, (long long)n);
    end += n;
    a.axis_end[i] = int32_t(end);
    if (end % per_lane) a.whole_axes = 0;
  }
  if (end != a.half)
    return fail(PSK_E_ARG, "sections of %lld pairs in all for a rotation of %d", (long long)end, a.half);
  a.table = cos_sin;
  a.table_stride = cos_sin_stride;
  a.num_positions = num_positions;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case PSK_DTYPE_BF16: launch_rows<PSK_DTYPE_BF16>(a, kind, num_tokens, st); break;
    case PSK_DTYPE_F16: launch_rows<PSK_DTYPE_F16>(a, kind, num_tokens, st); break;
    default: launch_rows<PSK_DTYPE_F32>(a, kind, num_tokens, st); break;
  }
  return check_launch("norm_rope_kernel launch");
}

}  // extern "C"
