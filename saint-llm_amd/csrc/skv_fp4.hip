// Writing tokens into the 4-bit pages and reading them back as bf16
// (skv_fp4.h has the format).
//
//   append: per 32 dims e = the smallest integer with max|x| <= 6 * 2^e, code =
//           RNE_e2m1(x / 2^e)
//   gather: value = code * 2^e (exact in bf16)
//
// Both move a token's K and V of all heads in items of 8 dims: 16 bytes of bf16
// (32 of fp32) on one side, a word of codes on the other; the four lanes of a
// 32-dim block find its largest magnitude by two quad permutes.  A thread has the
// same item of four tokens, whose loads it sends together: where an item lies in
// a token is worked out once for the four.
//
// HBM bounds both: 8 prompts of 8192 tokens, 8 heads of 128 dims (339 MB) are written
// in 65 us (5.2 TB/s) and read back in 51 us (6.6 TB/s, part of the codes from the
// last-level cache); with one token's item at a time and its place worked out anew
// 97 and 87 us.  A step of 64 single tokens takes 3.8 and 3.1 us, its launch's latency.
#include <algorithm>

#include "skv_fp4.h"

namespace skv {

constexpr int kFp4Threads = 256;
typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct Fp4RowsArgs {
  uint8_t* pool;
  int64_t n_pages;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* lens;
  const int32_t* n_new;
  int n_uni;
  uint8_t* x[2];  // K and V rows outside the pages
  int64_t seq_stride[2], tok_stride[2], head_stride[2];  // bytes
  int64_t rows;   // tokens per sequence that x holds
  int bs, heads, dim;
  int items;      // of a token: 2 * heads * dim / 8
  int together;   // tokens whose items a workgroup's threads take at once
};
constexpr int kFp4Tokens = 4;  // of a thread, a.together apart

// Where the tokens of a thread lie: page 0 where the page is not mapped or there is no token.
struct Fp4Places {
  int64_t page[kFp4Tokens];  // in bytes
  int slot[kFp4Tokens];
  int i[kFp4Tokens];  // token of its sequence's new ones
  bool in[kFp4Tokens], mapped[kFp4Tokens];
};

__device__ __forceinline__ Fp4Places fp4_places(const Fp4RowsArgs& a, const Fp4Page& pg, int b, int64_t first, int i0, int n) {
  Fp4Places at;
#pragma unroll
  for (int k = 0; k < kFp4Tokens; ++k) {
    const int i = i0 + k * a.together;
    at.in[k] = i < n;
    at.i[k] = at.in[k] ? i : 0;
    const int pos = static_cast<int>(first) + at.i[k];  // <= 2^24
    const int p = static_cast<int>(udiv24(pos, a.bs));
    at.slot[k] = pos - p * a.bs;
    const int32_t page = at.in[k] && p < a.bt_stride ? a.bt[b * a.bt_stride + p] : -1;
    at.mapped[k] = page >= 0 && page < a.n_pages;
    at.page[k] = at.mapped[k] ? page * pg.page : 0;
  }
  return at;
}

// An item of a token: K or V, head, 8-dim group; its codes, its block's scale byte
// in slot 0 of page 0, and its values' row of token 0.
struct Fp4Item {
  uint8_t* codes;
  uint8_t* scale;
  uint8_t* x;
  int64_t tok_stride;
  int d0;
};

__device__ __forceinline__ Fp4Item fp4_item(const Fp4RowsArgs& a, const Fp4Page& pg, int b, int r) {
  Fp4Item it;
  const int kv = r >= a.items >> 1 ? 1 : 0;
  r -= kv * (a.items >> 1);
  const int groups = a.dim >> 3;
  const int head = static_cast<int>(udiv24(r, groups));
  it.d0 = (r - head * groups) * 8;
  uint8_t* block = a.pool + head * pg.head;
  it.codes = block + (kv ? pg.v_codes : 0) + (it.d0 >> 1);
  it.scale = block + pg.scales + kv * (a.dim >> 5) + (it.d0 >> 5);
  it.x = a.x[kv] + b * a.seq_stride[kv] + head * a.head_stride[kv];
  it.tok_stride = a.tok_stride[kv];
  return it;
}

// Tokens [lens - n, lens) of sequence b, n its new ones; none where the counts
// are not those of an append, or the length is past what a table holds.
__device__ __forceinline__ int fp4_new(const Fp4RowsArgs& a, int b, int64_t* first) {
  const int64_t L = a.lens[b];
  const int64_t n = a.n_new ? a.n_new[b] : a.n_uni;
  *first = L - n;
  return n > L || n < 0 || L > (1 << 24) ? 0 : static_cast<int>(min(n, a.rows));
}

// A thread's first item and token: of the a.together tokens that the threads take
// at once (past them: no token).
__device__ __forceinline__ int fp4_first(const Fp4RowsArgs& a, int* r) {
  const int tid = threadIdx.x;
  if (a.items >= kFp4Threads) {
    *r = tid;
    return 0;
  }
  const int t = static_cast<int>(udiv24(tid, a.items));
  *r = tid - t * a.items;
  return t;
}

// grid: (workgroups over a sequence's tokens, batch)
template <bool kF32>
__global__ __launch_bounds__(kFp4Threads) void k_fp4_quant_append(Fp4RowsArgs a) {
  const int b = blockIdx.y;
  int64_t first;
  const int n = fp4_new(a, b, &first);
  const int i0 = blockIdx.x * kFp4Tokens * a.together;
  if (i0 >= n) return;  // uniform
  int r;
  const int t = fp4_first(a, &r);
  if (t >= a.together) return;  // whole blocks of lanes: an item count is a multiple of 8
  const Fp4Page pg = fp4_page(a.bs, a.heads, a.dim);
  const Fp4Places at = fp4_places(a, pg, b, first, i0 + t, n);
  for (; r < a.items; r += kFp4Threads) {
    const Fp4Item it = fp4_item(a, pg, b, r);
    u32x4 raw[kFp4Tokens][kF32 ? 2 : 1];
#pragma unroll
    for (int k = 0; k < kFp4Tokens; ++k) {
      const uint8_t* x = it.x + at.i[k] * it.tok_stride + it.d0 * (kF32 ? 4 : 2);
      raw[k][0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(x));
      if constexpr (kF32) raw[k][1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(x + 16));
    }
#pragma unroll
    for (int k = 0; k < kFp4Tokens; ++k) {
      float v[8];
      if constexpr (kF32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(raw[k][j / 4][j % 4]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[2 * j] = __uint_as_float(raw[k][0][j] << 16);
          v[2 * j + 1] = __uint_as_float(raw[k][0][j] & 0xffff0000u);
        }
      }
      uint32_t amax = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
      amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 1, 4)));
      amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 2, 4)));
      const uint32_t byte = fp4_scale_byte(amax), codes = fp4_encode8(v, byte);
      if (at.mapped[k]) {
        *reinterpret_cast<uint32_t*>(it.codes + at.page[k] + at.slot[k] * (a.dim >> 1)) = codes;
        if ((it.d0 & 31) == 0) it.scale[at.page[k] + at.slot[k] * (a.dim >> 4)] = static_cast<uint8_t>(byte);
      }
    }
  }
}

__global__ __launch_bounds__(kFp4Threads) void k_fp4_gather(Fp4RowsArgs a) {
  const int b = blockIdx.y;
  int64_t first;
  const int n = fp4_new(a, b, &first);
  const int i0 = blockIdx.x * kFp4Tokens * a.together;
  if (i0 >= n) return;  // uniform
  int r;
  const int t = fp4_first(a, &r);
  if (t >= a.together) return;
  const Fp4Page pg = fp4_page(a.bs, a.heads, a.dim);
  const Fp4Places at = fp4_places(a, pg, b, first, i0 + t, n);
  for (; r < a.items; r += kFp4Threads) {
    const Fp4Item it = fp4_item(a, pg, b, r);
    uint32_t codes[kFp4Tokens], byte[kFp4Tokens];
#pragma unroll
    for (int k = 0; k < kFp4Tokens; ++k) {
      codes[k] = *reinterpret_cast<const uint32_t*>(it.codes + at.page[k] + at.slot[k] * (a.dim >> 1));
      byte[k] = it.scale[at.page[k] + at.slot[k] * (a.dim >> 4)];
    }
#pragma unroll
    for (int k = 0; k < kFp4Tokens; ++k) {
      const u32x4 v = fp4_decode8(codes[k], fp4_scale(byte[k]));
      if (at.in[k]) {
        u32x4* x = reinterpret_cast<u32x4*>(it.x + at.i[k] * it.tok_stride + it.d0 * 2);
        __builtin_nontemporal_store(at.mapped[k] ? v : u32x4{0u, 0u, 0u, 0u}, x);
      }
    }
  }
}

// The checks of both directions; fills a.
int fp4_rows_args(Fp4RowsArgs& a, const char* what, const skv_fp4_cache* c, const int32_t* seq_lens, const int32_t* n_new,
                  int32_t n_uni, const skv_fp4_rows* k, const skv_fp4_rows* v, int64_t rows) {
  if (const int rc = fp4_check_cache(c, what)) return rc;
  if (!k || !v || !seq_lens) return set_error(SKV_EINVAL, "%s: NULL pointer", what);
  if (rows < 0 || rows > INT32_MAX) return set_error(SKV_EINVAL, "%s: bad number of rows", what);
  if (!n_new && n_uni < 0) return set_error(SKV_EINVAL, "%s: n_new_uniform must be >= 0", what);
  const skv_fp4_rows* kv[2] = {k, v};
  for (int i = 0; i < 2; ++i) {
    if (!kv[i]->data && rows > 0 && c->batch > 0) return set_error(SKV_EINVAL, "%s: NULL pointer", what);
    if ((reinterpret_cast<uintptr_t>(kv[i]->data) | static_cast<uintptr_t>(kv[i]->seq_stride) |
         static_cast<uintptr_t>(kv[i]->tok_stride) | static_cast<uintptr_t>(kv[i]->head_stride)) & 15) {
      return set_error(SKV_EINVAL, "%s: rows and their strides must be 16-byte aligned", what);
    }
    a.x[i] = static_cast<uint8_t*>(kv[i]->data);
    a.seq_stride[i] = kv[i]->seq_stride;
    a.tok_stride[i] = kv[i]->tok_stride;
    a.head_stride[i] = kv[i]->head_stride;
  }
  a.pool = static_cast<uint8_t*>(c->pool);
  a.n_pages = c->n_pages;
  a.bt = c->block_table;
  a.bt_stride = c->bt_stride;
  a.lens = seq_lens;
  a.n_new = n_new;
  a.n_uni = n_uni;
  a.rows = std::min<int64_t>(rows, 1 << 24);  // a sequence has no more tokens
  a.bs = static_cast<int>(c->block_size);
  a.heads = static_cast<int>(c->n_kv_heads);
  a.dim = static_cast<int>(c->head_dim);
  a.items = 2 * a.heads * (a.dim / 8);
  a.together = std::max(1, kFp4Threads / a.items);
  return SKV_OK;
}

}  // namespace skv

using namespace skv;

extern "C" int64_t skv_fp4_page_bytes(int64_t block_size, int64_t n_kv_heads, int64_t head_dim) {
  skv_fp4_cache c{};
  c.block_size = block_size;
  c.n_kv_heads = n_kv_heads;
  c.head_dim = head_dim;
  if (fp4_check_shape(&c, "skv_fp4_page_bytes") != SKV_OK) return -1;
  return fp4_page(static_cast<int>(block_size), static_cast<int>(n_kv_heads), static_cast<int>(head_dim)).page;
}

extern "C" int skv_fp4_quant_append(const skv_fp4_cache* cache, const int32_t* seq_lens, const int32_t* n_new,
                                    int32_t n_new_uniform, const skv_fp4_rows* k, const skv_fp4_rows* v, int64_t src_len,
                                    int32_t src_f32, void* stream) {
  const char* what = "skv_fp4_quant_append";
  Fp4RowsArgs a{};
  if (const int rc = fp4_rows_args(a, what, cache, seq_lens, n_new, n_new_uniform, k, v, src_len)) return rc;
  if (cache->batch == 0 || src_len == 0) return SKV_OK;
  const dim3 grid(static_cast<unsigned>(ceil_div(a.rows, kFp4Tokens * a.together)), static_cast<unsigned>(cache->batch));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (src_f32) {
    hipLaunchKernelGGL((k_fp4_quant_append<true>), grid, dim3(kFp4Threads), 0, s, a);
  } else {
    hipLaunchKernelGGL((k_fp4_quant_append<false>), grid, dim3(kFp4Threads), 0, s, a);
  }
  return check_launch(what);
}

extern "C" int skv_fp4_gather(const skv_fp4_cache* cache, const int32_t* seq_lens, const int32_t* n_rows,
                              int32_t n_rows_uniform, const skv_fp4_rows* k, const skv_fp4_rows* v, int64_t dst_len,
                              void* stream) {
  const char* what = "skv_fp4_gather";
  Fp4RowsArgs a{};
  if (const int rc = fp4_rows_args(a, what, cache, seq_lens, n_rows, n_rows_uniform, k, v, dst_len)) return rc;
  if (cache->batch == 0 || dst_len == 0) return SKV_OK;
  const dim3 grid(static_cast<unsigned>(ceil_div(a.rows, kFp4Tokens * a.together)), static_cast<unsigned>(cache->batch));
  hipLaunchKernelGGL(k_fp4_gather, grid, dim3(kFp4Threads), 0, static_cast<hipStream_t>(stream), a);
  return check_launch(what);
}
