// The 4-bit KV cache written and read back (mxfp4.h has the row).
//
// C ABI: include/pipeswift_kv.h.  Nothing here allocates or synchronizes.

#include <algorithm>

#include "mxfp4.h"

using namespace psk_detail;

namespace {

constexpr int kThreads = 256;

struct Mx4AppendArgs {
  const char* in[2];
  char* cache[2];
  const int64_t* slots;
  int64_t num_tokens, num_slots;
  int64_t in_tok[2], in_head[2];               // bytes
  int64_t blk[2], row[2], head[2];             // bytes
  int64_t block_size;
  int32_t bs_shift;
  int32_t num_heads, head_size;
  int32_t chunks;                              // lanes of a row: head_size / 8
  int32_t wide;                                // rows on 16-byte boundaries
};

// A lane takes eight elements, a quad of lanes a group: its maximum is two DPP steps
// away and nothing goes through LDS.  The lanes run over (token, K or V, head, group).
// Bound by memory: 4096 tokens of 8 heads of 128 in bf16 (16.8 MB in, 4.5 out) take 7.9 us
// with their launch, 2.7 TB/s, most of it the launch and one round of loads; 17 tokens 3.4.
template <int DT>
__global__ void __launch_bounds__(kThreads) mx4_append_kernel(Mx4AppendArgs a) {
  const int per = 2 * a.num_heads * a.chunks;  // lanes of a token (host: below 2^31)
  const int64_t at = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t t = at / per;
  if (t >= a.num_tokens) return;  // (whole quads: per is a multiple of 4)
  int r = int(at - t * per);
  const int which = r >= per / 2;
  r -= which ? per / 2 : 0;
  const int h = r / a.chunks, c = r - h * a.chunks;
  const int64_t slot = a.slots[t];
  typename Elt<DT>::Bits e[8];
  load8<DT>(a.in[which] + t * a.in_tok[which] + h * a.in_head[which] + c * 8 * Elt<DT>::kSize, a.wide, e);
  uint32_t byte;
  const uint32_t codes = mx_quantize8<DT>(e, byte);
  if (slot < 0 || slot >= a.num_slots) return;
  const int64_t page = a.bs_shift >= 0 ? slot >> a.bs_shift : slot / a.block_size;
  const int64_t off = slot - page * a.block_size;
  mx_store8(a.cache[which] + page * a.blk[which] + off * a.row[which] + h * a.head[which], c, a.head_size, codes, byte);
}

struct Mx4GatherArgs {
  const char* cache[2];
  char* dst[2];
  const int32_t* block_table;
  const int32_t* cu;
  const int32_t* starts;
  int64_t batch, bt_stride, bt_width, num_tokens, block_size, num_blocks;
  int64_t blk, row, head;  // bytes, both caches
  int64_t dst_tok;         // bytes
  int32_t bs_shift;
  int32_t num_heads, head_size, chunks;
  int32_t two;
  int32_t wide;
};

template <int DT>
__device__ __forceinline__ void store8(char* p, bool wide, uint32_t codes, float s) {
  u32x4 x[2];
  if constexpr (DT == PSK_DTYPE_F32) mx_f32x8(codes, s, x[0], x[1]);
  else x[0] = DT == PSK_DTYPE_BF16 ? mx_bf16x8(codes, s) : mx_f16x8(codes, s);
  if (wide) {
#pragma unroll
    for (int i = 0; i < Elt<DT>::kSize / 2; ++i) vstore_nt<16>(p + 16 * i, x[i]);
  } else {
    typename Elt<DT>::Bits e[8];
    __builtin_memcpy(e, x, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<typename Elt<DT>::Bits*>(p)[i] = e[i];
  }
}

// A wave takes a token's rows of K and V, eight elements a lane, with a dword of codes a
// lane: the rows lie on 4-byte boundaries, and a wave's loads side by side all the same.
// The results are not read again soon and go past the caches.  Bound by memory: 38
// thousand tokens of 8 heads of 128 (41 MB of K and V into 156 MB of bf16) take 31 us,
// 6.4 TB/s; 617 tokens 4.8, the chain of a token's sequence, its page id and its rows.
template <int DT>
__global__ void __launch_bounds__(kThreads) mx4_gather_kernel(Mx4GatherArgs g) {
  const int lane = int(threadIdx.x) & 63;
  const int64_t t = int64_t(blockIdx.x) * (kThreads / 64) + __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  if (t >= g.num_tokens) return;
  int64_t seq[1], pos[1], cu0;
  find_rows<1>(g.cu, g.starts, g.batch, t, lane, seq, pos, cu0);
  const int64_t b = seq[0], p = pos[0];
  if (b >= g.batch || t < cu0) return;  // no sequence's row: untouched
  const int64_t page = g.bs_shift >= 0 ? p >> g.bs_shift : p / g.block_size;
  int64_t id = -1;
  if (p >= 0 && page < g.bt_width) id = g.block_table[b * g.bt_stride + page];
  const bool there = id >= 0 && id < g.num_blocks;
  const int64_t from = there ? id * g.blk + (p - page * g.block_size) * g.row : 0;
  const int n = g.num_heads * g.chunks;
  for (int which = 0; which <= g.two; ++which) {
    const char* rows = g.cache[which] + from;
    char* out = g.dst[which] + t * g.dst_tok;
    for (int i = lane; i < n; i += 64) {
      const int h = i / g.chunks, c = i - h * g.chunks;
      uint32_t codes = 0, byte = 127;
      if (there) {
        const char* row = rows + h * g.head;
        codes = vload<4>(row + 4 * c);
        byte = uint8_t(row[g.head_size / 2 + (c >> 2)]);
      }
      store8<DT>(out + int64_t(i) * 8 * Elt<DT>::kSize, g.wide, codes, mx_scale(byte));
    }
  }
}

bool bad_head(int64_t num_heads, int64_t head_size) {
  return num_heads <= 0 || head_size <= 0 || head_size % kMxGroup || head_size > 4096 || num_heads > (1 << 24) / head_size;
}

}  // namespace

extern "C" {

int64_t psk_mxfp4_entry_bytes(int64_t head_size) {
  g_err[0] = 0;
  if (head_size <= 0 || head_size % kMxGroup || head_size > 4096)
    return fail(PSK_E_ARG, "head_size %lld must be a positive multiple of %d, at most 4096", (long long)head_size, kMxGroup);
  return mx_entry_bytes(head_size);
}

int psk_reshape_and_cache_mxfp4(const void* key, const void* value, void* key_cache, void* value_cache,
                                const int64_t* slot_mapping, int64_t num_tokens, int64_t num_heads, int64_t head_size,
                                int64_t block_size, int64_t num_blocks, const int64_t* strides, int in_dtype,
                                void* stream) {
  begin_device_call();
  if (bad_head(num_heads, head_size) || num_tokens < 0 || block_size <= 0 || num_blocks < 0)
    return fail(PSK_E_ARG, "bad sizes: num_tokens=%lld num_heads=%lld head_size=%lld block_size=%lld",
                (long long)num_tokens, (long long)num_heads, (long long)head_size, (long long)block_size);
  if (in_dtype != PSK_DTYPE_F32 && in_dtype != PSK_DTYPE_F16 && in_dtype != PSK_DTYPE_BF16)
    return fail(PSK_E_DTYPE, "a 4-bit cache takes bf16, f16 or f32 rows (got %d)", in_dtype);
  if (num_tokens == 0 || num_blocks == 0) return PSK_OK;
  if (!key || !value || !key_cache || !value_cache || !slot_mapping || !strides) return fail(PSK_E_ARG, "NULL pointer");
  const int64_t *k_strides = strides + 4, *v_strides = strides + 7;
  const int64_t entry = mx_entry_bytes(head_size);
  const int esz = dtype_size(in_dtype);
  uint64_t align = uint64_t(uintptr_t(key_cache)) | uint64_t(uintptr_t(value_cache));
  for (int i = 0; i < 3; ++i) align |= uint64_t(k_strides[i]) | uint64_t(v_strides[i]);
  if (align & 3) return fail(PSK_E_ARG, "cache rows must start on 4-byte boundaries");
  if ((num_heads > 1 && (k_strides[2] < entry || v_strides[2] < entry)) ||
      (block_size > 1 && (k_strides[1] < entry || v_strides[1] < entry)))
    return fail(PSK_E_ARG, "cache strides are shorter than the %lld-byte row", (long long)entry);
  Mx4AppendArgs a{};
  a.in[0] = static_cast<const char*>(key);
  a.in[1] = static_cast<const char*>(value);
  a.cache[0] = static_cast<char*>(key_cache);
  a.cache[1] = static_cast<char*>(value_cache);
  a.slots = slot_mapping;
  a.num_tokens = num_tokens;
  a.num_slots = num_blocks * block_size;
  const int64_t* in[2] = {strides, strides + 2};
  const int64_t* ca[2] = {k_strides, v_strides};
  uint64_t in_align = uint64_t(uintptr_t(key)) | uint64_t(uintptr_t(value));
  for (int i = 0; i < 2; ++i) {
    a.in_tok[i] = in[i][0] * esz;
    a.in_head[i] = in[i][1] * esz;
    in_align |= uint64_t(a.in_tok[i]) | uint64_t(a.in_head[i]);
    a.blk[i] = ca[i][0];
    a.row[i] = ca[i][1];
    a.head[i] = ca[i][2];
  }
  a.wide = (in_align & 15) == 0;
  a.block_size = block_size;
  a.bs_shift = log2_exact(block_size);
  a.num_heads = int32_t(num_heads);
  a.head_size = int32_t(head_size);
  a.chunks = int32_t(head_size / 8);
  const int64_t lanes = num_tokens * 2 * num_heads * a.chunks;
  if (num_tokens > INT32_MAX || ceil_div(lanes, kThreads) > INT32_MAX)
    return fail(PSK_E_ARG, "num_tokens %lld", (long long)num_tokens);
  const dim3 grid{unsigned(ceil_div(lanes, kThreads)), 1u, 1u};
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (in_dtype) {
    case PSK_DTYPE_BF16: hipLaunchKernelGGL((mx4_append_kernel<PSK_DTYPE_BF16>), grid, dim3(kThreads), 0, st, a); break;
    case PSK_DTYPE_F16: hipLaunchKernelGGL((mx4_append_kernel<PSK_DTYPE_F16>), grid, dim3(kThreads), 0, st, a); break;
    default: hipLaunchKernelGGL((mx4_append_kernel<PSK_DTYPE_F32>), grid, dim3(kThreads), 0, st, a); break;
  }
  return check_launch("mx4_append_kernel launch");
}

int psk_gather_mxfp4(const void* cache, const void* cache_v, void* dst, void* dst_v, const int32_t* block_table,
                     const int32_t* cu_seq_lens, const int32_t* seq_starts, int64_t batch_size,
                     int64_t block_table_stride, int64_t block_table_width, int64_t num_tokens, int64_t num_heads,
                     int64_t head_size, int64_t block_size, int64_t num_blocks, const int64_t* cache_strides,
                     int64_t dst_row_stride, int out_dtype, void* stream) {
  begin_device_call();
  if (bad_head(num_heads, head_size) || batch_size < 0 || num_tokens < 0 || block_size <= 0 || num_blocks < 0 ||
      batch_size > INT32_MAX || num_tokens > INT32_MAX || block_table_width < 0)
    return fail(PSK_E_ARG, "bad sizes: batch=%lld num_tokens=%lld num_heads=%lld head_size=%lld block_size=%lld",
                (long long)batch_size, (long long)num_tokens, (long long)num_heads, (long long)head_size,
                (long long)block_size);
  if (out_dtype != PSK_DTYPE_F32 && out_dtype != PSK_DTYPE_F16 && out_dtype != PSK_DTYPE_BF16)
    return fail(PSK_E_DTYPE, "a 4-bit cache is read as bf16, f16 or f32 (got %d)", out_dtype);
  if (num_tokens == 0 || batch_size == 0) return PSK_OK;
  if (!cache || !dst || !block_table || !cu_seq_lens || !cache_strides || !cache_v != !dst_v)
    return fail(PSK_E_ARG, "NULL pointer");
  const int osz = dtype_size(out_dtype);
  uint64_t align = uint64_t(uintptr_t(cache)) | uint64_t(uintptr_t(cache_v));
  for (int i = 0; i < 3; ++i) align |= uint64_t(cache_strides[i]);
  if (align & 3) return fail(PSK_E_ARG, "cache rows must start on 4-byte boundaries");
  if (num_tokens > 1 && dst_row_stride < num_heads * head_size)
    return fail(PSK_E_ARG, "dst row stride %lld is shorter than a row", (long long)dst_row_stride);
  Mx4GatherArgs g{};
  g.cache[0] = static_cast<const char*>(cache);
  g.cache[1] = static_cast<const char*>(cache_v);
  g.dst[0] = static_cast<char*>(dst);
  g.dst[1] = static_cast<char*>(dst_v);
  g.two = cache_v ? 1 : 0;
  g.block_table = block_table;
  g.cu = cu_seq_lens;
  g.starts = seq_starts;
  g.batch = batch_size;
  g.bt_stride = block_table_stride;
  g.bt_width = block_table_width;
  g.num_tokens = num_tokens;
  g.block_size = block_size;
  g.num_blocks = num_blocks;
  g.blk = cache_strides[0];
  g.row = cache_strides[1];
  g.head = cache_strides[2];
  g.dst_tok = dst_row_stride * osz;
  g.bs_shift = log2_exact(block_size);
  g.num_heads = int32_t(num_heads);
  g.head_size = int32_t(head_size);
  g.chunks = int32_t(head_size / 8);
  g.wide = ((uint64_t(uintptr_t(dst)) | uint64_t(uintptr_t(dst_v)) | uint64_t(g.dst_tok)) & 15) == 0;
  const dim3 grid{unsigned(ceil_div(num_tokens, kThreads / 64)), 1u, 1u};
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (out_dtype) {
    case PSK_DTYPE_BF16: hipLaunchKernelGGL((mx4_gather_kernel<PSK_DTYPE_BF16>), grid, dim3(kThreads), 0, st, g); break;
    case PSK_DTYPE_F16: hipLaunchKernelGGL((mx4_gather_kernel<PSK_DTYPE_F16>), grid, dim3(kThreads), 0, st, g); break;
    default: hipLaunchKernelGGL((mx4_gather_kernel<PSK_DTYPE_F32>), grid, dim3(kThreads), 0, st, g); break;
  }
  return check_launch("mx4_gather_kernel launch");
}

}  // extern "C"
