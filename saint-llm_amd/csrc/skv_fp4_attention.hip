// Attention over the pages of the 4-bit token cache (skv_fp4.h has the format).
//
//   s_j = scale * q . k_j, softcap * tanh(s_j / softcap) where asked for
//   out = sum_j exp(s_j) v_j / (sum_j exp(s_j) + exp(sink))
//
// over the positions j that the query token sees: one pass over them with the
// running maximum m and sum l of the softmax (log2 domain), the output rescaled
// by exp2(m_old - m_new) where the maximum moves.
#include <algorithm>

#include "skv_fp4.h"

namespace skv {

constexpr int kF4Threads = 256;
constexpr int kF4Waves = kF4Threads / kWave;
constexpr float kF4Log2e = 1.4426950408889634f;

struct Fp4AttnArgs {
  const uint8_t* q;
  int64_t q_seq, q_tok, q_head;
  uint16_t* out;  // [B, T, H, D] bf16
  const int32_t* lens;
  const uint8_t* pool;
  const int32_t* bt;
  const float* sink;
  int32_t n_pages, bt_stride, bs;
  int32_t T, H, Hkv, G, D;
  int32_t window;  // 0: none
  float scale, softcap;
};

// One workgroup per (query head, query token, sequence): each wave takes every
// fourth run of 64 positions, one position a lane for the scores, dims spread
// over the lanes for the values.
__global__ __launch_bounds__(kF4Threads) void k_fp4_attn_row(Fp4AttnArgs a) {
  __shared__ float qs[kFp4MaxDim];
  __shared__ float ps[kF4Waves][kWave];
  __shared__ float ml[kF4Waves][2];
  __shared__ float os[kF4Waves][kFp4MaxDim];
  const int h = blockIdx.x, t = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const int hk = h / a.G;
  const int64_t L = min(a.lens[b], a.bt_stride * a.bs);
  const int end = static_cast<int>(max<int64_t>(0, L - a.T + t + 1));  // positions before it are seen
  const int begin = a.window > 0 ? max(0, end - a.window) : 0;
  const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q + b * a.q_seq + t * a.q_tok + h * a.q_head);
  for (int d = tid; d < a.D; d += kF4Threads) qs[d] = bf16_to_f32(q[d]);
  __syncthreads();
  const Fp4Page pg = fp4_page(a.bs, a.Hkv, a.D);
  const int nb = a.D / kFp4Block, row = a.D / 2;
  const float ninf = -__builtin_huge_valf();
  float m = ninf, l = 0.f;
  float o[kFp4MaxDim / kWave];  // dims 2 * (lane + 64 c), and the next
#pragma unroll
  for (int c = 0; c < kFp4MaxDim / kWave; ++c) o[c] = 0.f;
  for (int j0 = begin + wave * kWave; j0 < end; j0 += kF4Threads) {
    const int j = j0 + lane;
    const int p = j / a.bs, slot = j % a.bs;
    const int32_t page = j < end ? a.bt[static_cast<int64_t>(b) * a.bt_stride + p] : -1;
    const bool live = page >= 0 && page < a.n_pages;
    const uint8_t* block = a.pool + (live ? page : 0) * pg.page + hk * pg.head;
    float s = 0.f;
    bool bad = false;  // a NaN block among the values
    if (live) {
      for (int i = 0; i < nb; ++i) {
        const float sc = fp4_scale(block[pg.scales + (2 * slot) * nb + i]);
        bad |= block[pg.scales + (2 * slot + 1) * nb + i] == kFp4NaN;
        for (int w = 0; w < 4; ++w) {
          const u32x4 k = fp4_decode8(*reinterpret_cast<const uint32_t*>(block + slot * row + i * 16 + w * 4), sc);
          for (int e = 0; e < 4; ++e) {
            s = fmaf(__uint_as_float(k[e] << 16), qs[i * 32 + w * 8 + 2 * e], s);
            s = fmaf(__uint_as_float(k[e] & 0xffff0000u), qs[i * 32 + w * 8 + 2 * e + 1], s);
          }
        }
      }
    }
    s *= a.scale;
    if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
    if (bad) s = __builtin_nanf("");
    s = live ? s * kF4Log2e : ninf;
    float mx = s;
    for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
    const float mn = fmaxf(m, mx);
    const float alpha = m == ninf ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    float pr = live ? __builtin_amdgcn_exp2f(s - (mn == ninf ? 0.f : mn)) : 0.f;
    m = mn;
    float sum = pr;
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    l = l * alpha + sum;
#pragma unroll
    for (int c = 0; c < kFp4MaxDim / kWave; ++c) o[c] *= alpha;
    ps[wave][lane] = pr;
    uint64_t todo = __ballot(live);
    while (todo) {
      const int i = __builtin_ctzll(todo);
      todo &= todo - 1;
      const int jj = j0 + i, pp = jj / a.bs, sl = jj % a.bs;
      const uint8_t* blk = a.pool + a.bt[static_cast<int64_t>(b) * a.bt_stride + pp] * pg.page + hk * pg.head;
      const float w = __shfl(pr, i);
#pragma unroll
      for (int c = 0; c < kFp4MaxDim / (2 * kWave); ++c) {
        const int byte = lane + c * kWave;
        if (byte < row) {
          const float sc = fp4_scale(blk[pg.scales + (2 * sl + 1) * nb + byte / 16]);
          const uint32_t v = fp4_decode8(blk[pg.v_codes + sl * row + byte], sc)[0];
          o[2 * c] = fmaf(w, __uint_as_float(v << 16), o[2 * c]);
          o[2 * c + 1] = fmaf(w, __uint_as_float(v & 0xffff0000u), o[2 * c + 1]);
        }
      }
    }
  }
  if (lane == 0) {
    ml[wave][0] = m;
    ml[wave][1] = l;
  }
#pragma unroll
  for (int c = 0; c < kFp4MaxDim / (2 * kWave); ++c) {
    const int byte = lane + c * kWave;
    if (byte < row) {
      os[wave][2 * byte] = o[2 * c];
      os[wave][2 * byte + 1] = o[2 * c + 1];
    }
  }
  __syncthreads();
  float mx = ninf;
  for (int w = 0; w < kF4Waves; ++w) mx = fmaxf(mx, ml[w][0]);
  const bool none = mx == ninf && !(ml[0][1] != ml[0][1]) && !(ml[1][1] != ml[1][1]) && !(ml[2][1] != ml[2][1]) &&
                    !(ml[3][1] != ml[3][1]);
  const float sink = a.sink ? a.sink[h] * kF4Log2e : ninf;
  const float top = fmaxf(mx, sink) == ninf ? 0.f : fmaxf(mx, sink);
  float f[kF4Waves], den = a.sink ? __builtin_amdgcn_exp2f(sink - top) : 0.f;
  for (int w = 0; w < kF4Waves; ++w) {
    f[w] = __builtin_amdgcn_exp2f(ml[w][0] - top);
    den += f[w] == 0.f && ml[w][1] == 0.f ? 0.f : ml[w][1] * f[w];
  }
  uint16_t* out = a.out + ((static_cast<int64_t>(b) * a.T + t) * a.H + h) * a.D;
  for (int d = tid; d < a.D; d += kF4Threads) {
    float v = 0.f;
    for (int w = 0; w < kF4Waves; ++w) v += os[w][d] * f[w];
    out[d] = none ? 0 : f32_to_bf16(v / den);
  }
}

struct Fp4AttnPlan {
  int64_t ws_bytes;
};

int fp4_attn_plan(const skv_fp4_attention_desc* d, Fp4AttnPlan& p) {
  const char* what = "skv_fp4_attention";
  if (!d) return set_error(SKV_EINVAL, "%s: NULL descriptor", what);
  if (const int rc = fp4_check_cache(&d->cache, what)) return rc;
  const int64_t hkv = d->cache.n_kv_heads;
  if (d->n_heads < 1 || d->n_heads > 1024 || d->n_heads % hkv) {
    return set_error(SKV_EINVAL, "%s: n_heads must be a multiple of n_kv_heads in [1, 1024]; got %lld over %lld", what,
                     (long long)d->n_heads, (long long)hkv);
  }
  if (d->n_queries < 1 || d->n_queries > 65535) {
    return set_error(SKV_EINVAL, "%s: n_queries must be in [1, 65535]; got %lld", what, (long long)d->n_queries);
  }
  if (d->window < 0 || d->window > (1 << 24)) return set_error(SKV_EINVAL, "%s: window must be in [0, 2^24]", what);
  if (d->max_len < 0 || d->splits < 0) return set_error(SKV_EINVAL, "%s: max_len and splits must be >= 0", what);
  if (!(d->scale >= 0.f) || d->scale > 3e38f || !(d->softcap >= 0.f) || d->softcap > 3e38f) {
    return set_error(SKV_EINVAL, "%s: scale and softcap must be finite and >= 0", what);
  }
  p.ws_bytes = 0;
  return SKV_OK;
}

}  // namespace skv

using namespace skv;

extern "C" int64_t skv_fp4_attention_desc_size(void) { return static_cast<int64_t>(sizeof(skv_fp4_attention_desc)); }

extern "C" int64_t skv_fp4_attention_workspace(const skv_fp4_attention_desc* d) {
  Fp4AttnPlan p;
  return fp4_attn_plan(d, p) == SKV_OK ? p.ws_bytes : -1;
}

extern "C" int skv_fp4_attention(const skv_fp4_attention_desc* d, void* workspace, int64_t ws_bytes, void* stream) {
  const char* what = "skv_fp4_attention";
  Fp4AttnPlan p;
  if (const int rc = fp4_attn_plan(d, p)) return rc;
  if (d->cache.batch == 0) return SKV_OK;
  if (!d->q || !d->out || !d->seq_lens) return set_error(SKV_EINVAL, "%s: NULL pointer", what);
  if ((reinterpret_cast<uintptr_t>(d->q) | reinterpret_cast<uintptr_t>(d->out) | static_cast<uintptr_t>(d->q_seq_stride) |
       static_cast<uintptr_t>(d->q_tok_stride) | static_cast<uintptr_t>(d->q_head_stride)) & 15) {
    return set_error(SKV_EINVAL, "%s: q, its strides and out must be 16-byte aligned", what);
  }
  if (p.ws_bytes > 0 && (!workspace || ws_bytes < p.ws_bytes || (reinterpret_cast<uintptr_t>(workspace) & 15))) {
    return set_error(SKV_EINVAL, "%s: a 16-byte aligned workspace of %lld bytes is needed", what, (long long)p.ws_bytes);
  }
  Fp4AttnArgs a{};
  a.q = static_cast<const uint8_t*>(d->q);
  a.q_seq = d->q_seq_stride;
  a.q_tok = d->q_tok_stride;
  a.q_head = d->q_head_stride;
  a.out = static_cast<uint16_t*>(d->out);
  a.lens = d->seq_lens;
  a.pool = static_cast<const uint8_t*>(d->cache.pool);
  a.bt = d->cache.block_table;
  a.sink = d->sink;
  a.n_pages = static_cast<int32_t>(d->cache.n_pages);
  a.bt_stride = static_cast<int32_t>(d->cache.bt_stride);
  a.bs = static_cast<int32_t>(d->cache.block_size);
  a.T = static_cast<int32_t>(d->n_queries);
  a.H = static_cast<int32_t>(d->n_heads);
  a.Hkv = static_cast<int32_t>(d->cache.n_kv_heads);
  a.G = a.H / a.Hkv;
  a.D = static_cast<int32_t>(d->cache.head_dim);
  a.window = static_cast<int32_t>(d->window);
  a.scale = d->scale > 0.f ? d->scale : 1.f / sqrtf(static_cast<float>(a.D));
  a.softcap = d->softcap;
  hipLaunchKernelGGL(k_fp4_attn_row, dim3(static_cast<unsigned>(a.H), static_cast<unsigned>(a.T), static_cast<unsigned>(d->cache.batch)),
                     dim3(kF4Threads), 0, static_cast<hipStream_t>(stream), a);
  return check_launch(what);
}
