// Writing tokens into the 4-bit pages and reading them back as bf16
// (skv_fp4.h has the format).
//
//   append: per 32 dims e = the smallest integer with max|x| <= 6 * 2^e, code =
//           RNE_e2m1(x / 2^e)
//   gather: value = code * 2^e (exact in bf16)
//
// Both move a token's K and V of all heads in items of 8 dims: 16 bytes of bf16
// (32 of fp32) on one side, a word of codes on the other; the four lanes of a
// 32-dim block find its largest magnitude by two quad permutes.
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
};

// An item: token i of sequence b's n, K or V, head, 8-dim group.
struct Fp4Item {
  uint8_t* x;      // its values outside the pages (of token 0 past the last token)
  uint8_t* codes;  // its word of codes
  uint8_t* scale;  // its block's scale byte
  int i, d0;
  bool mapped;     // a token whose page is mapped
};

__device__ __forceinline__ Fp4Item fp4_item(const Fp4RowsArgs& a, const Fp4Page& pg, int b, int64_t first, int i0, int n,
                                            int q) {
  Fp4Item it;
  const int t = static_cast<int>(udiv24(q, a.items));
  int r = q - t * a.items;
  const int kv = r >= a.items >> 1 ? 1 : 0;
  r -= kv * (a.items >> 1);
  const int groups = a.dim >> 3;
  const int head = static_cast<int>(udiv24(r, groups));
  it.d0 = (r - head * groups) * 8;
  it.i = i0 + t;
  const bool in = it.i < n;
  const int pos = static_cast<int>(first) + (in ? it.i : 0);  // <= 2^24
  const int p = static_cast<int>(udiv24(pos, a.bs));
  const int slot = pos - p * a.bs;
  const int32_t page = in && p < a.bt_stride ? a.bt[b * a.bt_stride + p] : -1;
  it.mapped = page >= 0 && page < a.n_pages;
  uint8_t* block = a.pool + (it.mapped ? page : 0) * pg.page + head * pg.head;
  it.codes = block + (kv ? pg.v_codes : 0) + slot * (a.dim >> 1) + (it.d0 >> 1);
  it.scale = block + pg.scales + (2 * slot + kv) * (a.dim >> 5) + (it.d0 >> 5);
  it.x = a.x[kv] + b * a.seq_stride[kv] + (in ? it.i : 0) * a.tok_stride[kv] + head * a.head_stride[kv];
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

// grid: (workgroups over a sequence's tokens, batch)
template <bool kF32>
__global__ __launch_bounds__(kFp4Threads) void k_fp4_quant_append(Fp4RowsArgs a, int tokens) {
  const int b = blockIdx.y;
  int64_t first;
  const int n = fp4_new(a, b, &first);
  const int i0 = blockIdx.x * tokens;
  if (i0 >= n) return;  // uniform
  const Fp4Page pg = fp4_page(a.bs, a.heads, a.dim);
  const int end = min(tokens, n - i0) * a.items;
  for (int q = threadIdx.x; q < end; q += kFp4Threads) {  // the four lanes of a block take the same turns
    const Fp4Item it = fp4_item(a, pg, b, first, i0, n, q);
    if (!it.mapped) continue;
    float v[8];
    if constexpr (kF32) {
      const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(it.x + it.d0 * 4);
      const f32x4_t hi = *reinterpret_cast<const f32x4_t*>(it.x + it.d0 * 4 + 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = lo[j];
        v[j + 4] = hi[j];
      }
    } else {
      const u32x4 w = *reinterpret_cast<const u32x4*>(it.x + it.d0 * 2);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    }
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
    amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 1, 4)));
    amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 2, 4)));
    const uint32_t byte = fp4_scale_byte(amax);
    *reinterpret_cast<uint32_t*>(it.codes) = fp4_encode8(v, byte);
    if ((it.d0 & 31) == 0) *it.scale = static_cast<uint8_t>(byte);
  }
}

__global__ __launch_bounds__(kFp4Threads) void k_fp4_gather(Fp4RowsArgs a, int tokens) {
  const int b = blockIdx.y;
  int64_t first;
  const int n = fp4_new(a, b, &first);
  const int i0 = blockIdx.x * tokens;
  if (i0 >= n) return;  // uniform
  const Fp4Page pg = fp4_page(a.bs, a.heads, a.dim);
  const int end = min(tokens, n - i0) * a.items;
  for (int q = threadIdx.x; q < end; q += kFp4Threads) {
    const Fp4Item it = fp4_item(a, pg, b, first, i0, n, q);
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(it.codes);
    const u32x4 v = fp4_decode8(codes, fp4_scale(*it.scale));
    *reinterpret_cast<u32x4*>(it.x + it.d0 * 2) = it.mapped ? v : u32x4{0u, 0u, 0u, 0u};
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
  a.rows = rows;
  a.bs = static_cast<int>(c->block_size);
  a.heads = static_cast<int>(c->n_kv_heads);
  a.dim = static_cast<int>(c->head_dim);
  a.items = 2 * a.heads * (a.dim / 8);
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
  const int tokens = static_cast<int>(std::max(1, 1024 / a.items));
  const dim3 grid(static_cast<unsigned>(ceil_div(src_len, tokens)), static_cast<unsigned>(cache->batch));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (src_f32) {
    hipLaunchKernelGGL((k_fp4_quant_append<true>), grid, dim3(kFp4Threads), 0, s, a, tokens);
  } else {
    hipLaunchKernelGGL((k_fp4_quant_append<false>), grid, dim3(kFp4Threads), 0, s, a, tokens);
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
  const int tokens = static_cast<int>(std::max(1, 1024 / a.items));
  const dim3 grid(static_cast<unsigned>(ceil_div(dst_len, tokens)), static_cast<unsigned>(cache->batch));
  hipLaunchKernelGGL(k_fp4_gather, grid, dim3(kFp4Threads), 0, static_cast<hipStream_t>(stream), a, tokens);
  return check_launch(what);
}
