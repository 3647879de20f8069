// The 4-bit token cache: pages of K and V codes and their scales.
//
// A code is e2m1 (sign, 2 exponent bits, 1 mantissa bit: 0, .5, 1, 1.5, 2, 3, 4,
// 6); 32 consecutive dims share a scale byte s, the power of two 2^(s - 127).
// A value is code * 2^(s - 127), exact in bf16 for s <= 252: gfx950's
// conversions from and to this format (v_cvt_scalef32_pk_*) are used as they
// are.  They were compared with the definition on the GPU: decoding for all 256
// code bytes under every scale byte up to 252 (255 gives NaN), encoding for
// every fp32 value of [-6, 6] times nine scales of 2^-120 .. 2^123.
//
// Page layout, for block_size tokens, H K/V heads of D dims: per head
//   [block_size][D / 2]  the keys' codes, dims 2i and 2i + 1 in byte i (2i low),
//   [block_size][D / 2]  the values' codes,
//   [block_size][2][D / 32]  scale bytes: the token's key, then its value,
// so that a head's 16 tokens are one run of each plane (a head's block in a page:
// 17/16 * block_size * D bytes).  block_size is a multiple of 16: every plane
// starts at a multiple of 16 bytes.
#pragma once

#include "skv_common.h"

namespace skv {

constexpr int kFp4Block = 32;         // dims per scale
constexpr int kFp4MaxDim = 512;
constexpr int kFp4NaN = 255;          // scale byte of a block that held a NaN or an infinity
constexpr int kFp4MinScale = 7;       // 2^-120: values and scores stay clear of bf16's subnormals
constexpr int kFp4MaxScale = 252;     // 2^125: 6 * 2^125 is finite in bf16

// Bytes of one head's block of a page, and where its planes start.
struct Fp4Page {
  int64_t head, page;
  int v_codes, scales;  // of the head's block
};

__host__ __device__ __forceinline__ Fp4Page fp4_page(int block_size, int heads, int dim) {
  Fp4Page p;
  p.v_codes = block_size * (dim / 2);
  p.scales = 2 * p.v_codes;
  p.head = static_cast<int64_t>(p.scales) + static_cast<int64_t>(block_size) * (dim / 16);
  p.page = p.head * heads;
  return p;
}

__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// The scale byte of a block whose largest magnitude has the fp32 bits `amax`:
// the smallest power of two under which no value passes 6 (6 * 2^e = 1.5 *
// 2^(e + 2)).  The bits of a NaN are above infinity's, infinity's above the
// finite ones', so an integer maximum finds all three.
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t amax) {
  if (amax >= 0x7f800000u) return kFp4NaN;
  const int e = static_cast<int>(amax >> 23) - 2 + ((amax & 0x7fffffu) > 0x400000u ? 1 : 0);
  return static_cast<uint32_t>(min(max(e, kFp4MinScale), kFp4MaxScale));
}

// Eight values' codes under a scale byte (round to nearest even; past 6, where
// the scale is at its largest, 6; zeros in a NaN block).
__device__ __forceinline__ uint32_t fp4_encode8(const float* x, uint32_t byte) {
  if (byte == kFp4NaN) return 0u;
  const float scale = fp4_scale(byte), top = 6.f * scale;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = __builtin_amdgcn_fmed3f(x[j], -top, top);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
  return r;
}

// Shape and page geometry of a cache, as the entry points take it.
inline int fp4_check_shape(const skv_fp4_cache* c, const char* what) {
  if (c->block_size < 16 || c->block_size % 16 || c->block_size > 65536) {
    return set_error(SKV_EINVAL, "%s: block_size must be a multiple of 16 in [16, 65536]; got %lld", what,
                     (long long)c->block_size);
  }
  if (c->n_kv_heads < 1 || c->n_kv_heads > 256) {
    return set_error(SKV_EINVAL, "%s: n_kv_heads must be in [1, 256]; got %lld", what, (long long)c->n_kv_heads);
  }
  if (c->head_dim < kFp4Block || c->head_dim > kFp4MaxDim || c->head_dim % kFp4Block) {
    return set_error(SKV_EINVAL, "%s: head_dim must be a multiple of %d in [%d, %d]; got %lld", what, kFp4Block,
                     kFp4Block, kFp4MaxDim, (long long)c->head_dim);
  }
  return SKV_OK;
}

inline int fp4_check_cache(const skv_fp4_cache* c, const char* what) {
  if (!c) return set_error(SKV_EINVAL, "%s: NULL cache", what);
  if (const int rc = fp4_check_shape(c, what)) return rc;
  if (c->batch < 0 || c->batch > 65535) {
    return set_error(SKV_EINVAL, "%s: batch must be in [0, 65535]; got %lld", what, (long long)c->batch);
  }
  if (c->n_pages < 1 || c->n_pages > INT32_MAX || c->bt_stride < 1 || c->bt_stride > (1 << 24) ||
      c->bt_stride * c->block_size > (1 << 24)) {
    return set_error(SKV_EINVAL, "%s: bad page geometry (n_pages >= 1, bt_stride * block_size <= 2^24)", what);
  }
  if (c->batch == 0) return SKV_OK;
  if (!c->pool || !c->block_table) return set_error(SKV_EINVAL, "%s: NULL pointer", what);
  if (reinterpret_cast<uintptr_t>(c->pool) & 15) return set_error(SKV_EINVAL, "%s: pool must be 16-byte aligned", what);
  return SKV_OK;
}

// The eight codes of a word as bf16, dims in order.
__device__ __forceinline__ u32x4 fp4_decode8(uint32_t codes, float scale) {
  u32x4 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  return r;
}

}  // namespace skv
