// Log probabilities of given tokens, the entropy and the most likely tokens of rows of logits.
//
//   m = max x, l = sum exp(x - m), s = sum exp(x - m) (x - m)
//   logprob = x_token - m - ln l,  entropy = ln l - s / l
//
// One pass over a row: a lane keeps a running m, l and s of the logits that it sees; lanes, waves and (of rows
// that several workgroups share) segments are joined by exp(m_i - m), under which s_i becomes s_i + l_i (m_i - m).
// HBM bounds it with many rows (each logit is read once), the vector work close behind: about eight instructions
// and an exponential a logit.
//
// The `top` largest cost next to nothing on the way: a lane notes the maximum of every 64 bytes (4 loads of 16)
// that it sees, in LDS.  The top-th largest of the lanes' own maxima is a bound that at least `top` logits
// reach, and little more do (of 256 lanes and 20 wanted about 21); only the noted 64 bytes that reach it are
// read again and what reaches it in them is sorted, by value and then id, as one 64-bit key.  Where too much
// does (equal logits throughout, or most of a row -inf), the waves go through the row once more with a list
// of the best so far each.
#include <algorithm>

#include "skv_common.h"

namespace skv {

constexpr int kLpThreads = 256;
constexpr int kLpWaves = kLpThreads / kWave;
constexpr int kLpVecs = 4;        // 16-byte loads of a lane's chunk
constexpr int kLpMaxTop = 64;     // a wave's list
constexpr int kLpMaxChunks = 32;  // of a segment: LDS holds their maxima
constexpr int kLpList = 256;      // chunks read again
constexpr int kLpPend = 512;      // logits that reach the bound
constexpr float kLpLog2e = 1.4426950408889634f;
constexpr float kLpLowest = -3.4028234663852886e38f;
constexpr float kLpGone = -1e4f;  // exp of it is 0; times 0 it is 0, as -inf would not be

struct LpArgs {
  const uint8_t* x;
  int64_t row_bytes;  // between rows
  int64_t vocab;
  int32_t rows, top;
  int32_t chunks, segments;  // of a segment; of a row
  const void* tokens;
  int64_t tok_stride;
  int32_t wide;
  float* logprobs;
  float* entropy;
  int32_t* top_ids;
  float* top_logprobs;
  uint8_t* parts;  // [rows, segments]: LpPart, then `top` keys
};

struct LpPart {
  float top, m, l, s;
};

// The logits' types: values of a 16-byte vector, and the low bits of their keys that say nothing.
template <int kFormat>
struct LpType;
template <>
struct LpType<SKV_LOGITS_BF16> {
  using elem = uint16_t;
  static constexpr int kVec = 8, kLowBit = 16;
  static constexpr uint32_t kNone = 0xff80u;
  __device__ __forceinline__ static float value(elem v) { return bf16_to_f32(v); }
  __device__ __forceinline__ static void unpack(u32x4 r, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(r[i] << 16);
      x[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  }
};
template <>
struct LpType<SKV_LOGITS_F16> {
  using elem = uint16_t;
  static constexpr int kVec = 8, kLowBit = 13;
  static constexpr uint32_t kNone = 0xfc00u;
  __device__ __forceinline__ static float value(elem v) { return static_cast<float>(__builtin_bit_cast(_Float16, v)); }
  __device__ __forceinline__ static void unpack(u32x4 r, float* x) {
    typedef _Float16 half2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = r[i];  // (a bit cast of the vector's element itself takes its first)
      const half2 h = __builtin_bit_cast(half2, w);
      x[2 * i] = static_cast<float>(h[0]);
      x[2 * i + 1] = static_cast<float>(h[1]);
    }
  }
};
template <>
struct LpType<SKV_LOGITS_F32> {
  using elem = uint32_t;
  static constexpr int kVec = 4, kLowBit = 0;
  static constexpr uint32_t kNone = 0xff800000u;
  __device__ __forceinline__ static float value(elem v) { return __uint_as_float(v); }
  __device__ __forceinline__ static void unpack(u32x4 r, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(r[i]);
  }
};

// A value as an integer of the same order (equal zeros equal, a NaN above all); 0 stands for none.
__device__ __forceinline__ uint32_t lp_order(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  if (x != x) return 0xffc00000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// Larger values first, of equal ones the lower id.
__device__ __forceinline__ uint64_t lp_key(uint32_t order, uint32_t id) { return static_cast<uint64_t>(order) << 32 | ~id; }

__device__ __forceinline__ uint64_t lp_shfl_xor(uint64_t v, int by) {
  const uint32_t lo = __shfl_xor(static_cast<int>(v), by), hi = __shfl_xor(static_cast<int>(v >> 32), by);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t lp_shfl(uint64_t v, int from) {
  const uint32_t lo = __shfl(static_cast<int>(v), from), hi = __shfl(static_cast<int>(v >> 32), from);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// A wave's 64 keys, one a lane, in descending order.
__device__ __forceinline__ uint64_t lp_sort(uint64_t v) {
  const int lane = threadIdx.x % kWave;
#pragma unroll
  for (int size = 2; size <= kWave; size *= 2) {
#pragma unroll
    for (int by = size / 2; by > 0; by /= 2) {
      const uint64_t o = lp_shfl_xor(v, by);
      const bool larger = ((lane & size) == 0) == ((lane & by) == 0);
      v = (o > v) == larger ? o : v;
    }
  }
  return v;
}
// The 64 largest of two lists in descending order, in that order.
__device__ __forceinline__ uint64_t lp_merge(uint64_t a, uint64_t b) {
  const int lane = threadIdx.x % kWave;
  const uint64_t o = lp_shfl(b, kWave - 1 - lane);
  uint64_t v = o > a ? o : a;
#pragma unroll
  for (int by = kWave / 2; by > 0; by /= 2) {
    const uint64_t p = lp_shfl_xor(v, by);
    v = (p > v) == ((lane & by) == 0) ? p : v;
  }
  return v;
}

__device__ __forceinline__ float lp_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }  // a NaN stays

// (m, l, s) under the maximum `to`.
__device__ __forceinline__ void lp_rebase(float& m, float& l, float& s, float to) {
  const float d = fmaxf(m - to, kLpGone), f = __builtin_amdgcn_exp2f(d * kLpLog2e);
  s = f * __builtin_fmaf(l, d, s);
  l *= f;
  m = to;
}

// A row's numbers, from the joined state and the token's logit; of wave 0.
__device__ __forceinline__ void lp_finish(const LpArgs& a, int64_t row, float top, float m, float l, float s, uint64_t key, int64_t token,
                                          float logit) {
  const int lane = threadIdx.x % kWave;
  const bool bad = !(__builtin_fabsf(top) < __builtin_huge_valf());
  const float nan = __builtin_nanf(""), norm = bad ? nan : logf(l);
  if (lane == 0) {
    if (a.logprobs) a.logprobs[row] = token < 0 ? 0.f : token >= a.vocab ? nan : (logit - m) - norm;
    a.entropy[row] = norm - s / l;
  }
  if (lane < a.top) {
    a.top_ids[row * a.top + lane] = static_cast<int32_t>(~static_cast<uint32_t>(key));
    a.top_logprobs[row * a.top + lane] = (lp_value(static_cast<uint32_t>(key >> 32)) - m) - norm;
  }
}

template <int kFormat>
__device__ __forceinline__ void lp_token(const LpArgs& a, int64_t row, int64_t& token, float& logit) {
  using Type = LpType<kFormat>;
  token = -1;
  logit = 0.f;
  if (!a.tokens) return;
  token = a.wide ? static_cast<const int64_t*>(a.tokens)[row * a.tok_stride]
                 : static_cast<const int32_t*>(a.tokens)[row * a.tok_stride];
  const bool in = token >= 0 && token < a.vocab;
  const auto* x = reinterpret_cast<const typename Type::elem*>(a.x + row * a.row_bytes);
  logit = Type::value(x[in ? token : 0]);
}

template <bool kTop>
struct LpSmem {
  float part[kLpWaves][4];
  uint32_t bins[kTop ? kLpThreads : 1];
  uint32_t bound;
  int n_list, n_pend;
  int32_t list[kTop ? kLpList : 1];
  uint64_t pend[kTop ? kLpPend : 1];
};

// grid: rows x segments.  A segment is `chunks` times kLpThreads * kLpVecs vectors of the row, which are
// counted from the 16-byte boundary at or before its first logit.
template <int kFormat, bool kTop>
__global__ __launch_bounds__(kLpThreads) void k_logprobs(LpArgs a) {
  using Type = LpType<kFormat>;
  using Elem = typename Type::elem;
  constexpr int kVec = Type::kVec, kElems = kVec * kLpVecs;
  __shared__ LpSmem<kTop> sm;
  extern __shared__ float noted[];  // [chunks][kLpThreads]
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int64_t row = blockIdx.x / a.segments;
  const int seg = blockIdx.x - static_cast<int>(row) * a.segments;
  const uint8_t* base = a.x + row * a.row_bytes;
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(base) & 15) / sizeof(Elem));
  const uint8_t* x0 = base - off * sizeof(Elem);
  const int V = static_cast<int>(a.vocab), end = off + V;
  int64_t token = -1;
  float logit = 0.f;
  if (a.segments == 1 && tid == 0) lp_token<kFormat>(a, row, token, logit);
  if (kTop && tid == 0) sm.n_list = sm.n_pend = 0;
  const int first = seg * a.chunks * kLpVecs * kLpThreads;  // vector
  const auto vector_of = [&](int c, int i) { return first + (c * kLpVecs + i) * kLpThreads + tid; };
  const auto load = [&](u32x4* r, int c) {
    const int v0 = first + c * kLpVecs * kLpThreads;
    if (v0 * kVec >= off && (v0 + kLpVecs * kLpThreads) * kVec <= end) {  // uniform: inside the row
#pragma unroll
      for (int i = 0; i < kLpVecs; ++i) r[i] = ld_stream(reinterpret_cast<const u32x4*>(x0) + vector_of(c, i));
    } else {
#pragma unroll
      for (int i = 0; i < kLpVecs; ++i) {
        const int u = vector_of(c, i) * kVec;
        if (u >= off && u + kVec <= end) {
          r[i] = ld_stream(reinterpret_cast<const u32x4*>(x0 + u * static_cast<int64_t>(sizeof(Elem))));
        } else {  // logits past the ends: none
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            w[k] = 0;
#pragma unroll
            for (int j = 0; j < kVec / 4; ++j) {
              const int at = u + k * (kVec / 4) + j - off;
              const uint32_t e = at >= 0 && at < V ? reinterpret_cast<const Elem*>(base)[at] : Type::kNone;
              w[k] |= e << (16 * j);
            }
          }
          r[i] = u32x4{w[0], w[1], w[2], w[3]};
        }
      }
    }
  };
  float m = kLpLowest, l = 0.f, s = 0.f, top = -__builtin_huge_valf();
  const auto fold = [&](const u32x4* r, int c) {
    float x[kElems];
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) Type::unpack(r[i], x + i * kVec);
    float cm = x[0];
#pragma unroll
    for (int i = 1; i < kElems; ++i) cm = lp_max(cm, x[i]);
    if (kTop) noted[c * kLpThreads + tid] = cm;
    top = lp_max(top, cm);
    lp_rebase(m, l, s, lp_max(m, cm));
    float lk[4] = {0.f, 0.f, 0.f, 0.f}, sk[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kElems; ++i) {
      const float d = fmaxf(x[i] - m, kLpGone), e = __builtin_amdgcn_exp2f(d * kLpLog2e);
      lk[i & 3] += e;
      sk[i & 3] = __builtin_fmaf(e, d, sk[i & 3]);
    }
    l += (lk[0] + lk[1]) + (lk[2] + lk[3]);
    s += (sk[0] + sk[1]) + (sk[2] + sk[3]);
  };
  u32x4 r0[kLpVecs], r1[kLpVecs];
  load(r0, 0);
  int c = 0;
  for (; c + 1 < a.chunks; c += 2) {
    load(r1, c + 1);
    fold(r0, c);
    if (c + 2 < a.chunks) load(r0, c + 2);
    fold(r1, c + 1);
  }
  if (c < a.chunks) fold(r0, c);
  // join the lanes, then the waves
  float wm = m, wtop = top;
#pragma unroll
  for (int by = 1; by < kWave; by *= 2) {
    wm = lp_max(wm, __shfl_xor(wm, by));
    wtop = lp_max(wtop, __shfl_xor(wtop, by));
  }
  lp_rebase(m, l, s, wm);
#pragma unroll
  for (int by = 1; by < kWave; by *= 2) {
    l += __shfl_xor(l, by);
    s += __shfl_xor(s, by);
  }
  if (lane == 0) {
    sm.part[wave][0] = wtop;
    sm.part[wave][1] = wm;
    sm.part[wave][2] = l;
    sm.part[wave][3] = s;
  }
  if (kTop) sm.bins[tid] = lp_order(top);
  __syncthreads();
  uint64_t best = 0;
  if constexpr (kTop) {
    // the bound: the largest that `top` bins reach
    if (wave == 0) {
      uint32_t b[kLpWaves], t = 0;
#pragma unroll
      for (int i = 0; i < kLpWaves; ++i) b[i] = sm.bins[i * kWave + lane];
#pragma unroll
      for (int bit = 31; bit >= Type::kLowBit; --bit) {
        const uint32_t up = t | 1u << bit;
        int n = 0;
#pragma unroll
        for (int i = 0; i < kLpWaves; ++i) n += __popcll(__ballot(b[i] >= up));
        if (n >= a.top) t = up;
      }
      if (lane == 0) sm.bound = t;
    }
    __syncthreads();
    const uint32_t bound = sm.bound;
    if (lp_order(top) >= bound) {
      for (int k = 0; k < a.chunks; ++k) {
        if (lp_order(noted[k * kLpThreads + tid]) >= bound) {
          const int at = atomicAdd(&sm.n_list, 1);
          if (at < kLpList) sm.list[at] = k * kLpThreads + tid;
        }
      }
    }
    __syncthreads();
    const int listed = sm.n_list;
    if (listed <= kLpList) {  // uniform
      for (int i = tid / kElems; i < listed; i += kLpThreads / kElems) {
        const int at = sm.list[i], k = at / kLpThreads, t = at % kLpThreads, e = tid % kElems;
        const int id = (first + (k * kLpVecs + e / kVec) * kLpThreads + t) * kVec + e % kVec - off;
        if (id < 0 || id >= V) continue;
        const uint32_t order = lp_order(Type::value(reinterpret_cast<const Elem*>(base)[id]));
        if (order >= bound) {
          const int p = atomicAdd(&sm.n_pend, 1);
          if (p < kLpPend) sm.pend[p] = lp_key(order, id);
        }
      }
    }
    __syncthreads();
    const int pending = sm.n_pend;
    if (listed <= kLpList && pending <= kLpPend) {  // uniform
      if (wave == 0) {
        best = lp_sort(lane < pending ? sm.pend[lane] : 0);
        for (int p = kWave; p < pending; p += kWave) best = lp_merge(best, lp_sort(p + lane < pending ? sm.pend[p + lane] : 0));
      }
    } else {
      // a quarter of the segment to a wave, in the order of the ids, and a list of the best so far
      __syncthreads();  // pend has been counted
      constexpr int kAhead = 16;
      uint64_t* mine = sm.pend + wave * (kLpPend / kLpWaves);
      static_assert(kLpPend / kLpWaves >= 2 * kWave, "a wave's pending keys: 63 and a load's 64");
      const int span = a.chunks * kLpVecs * kLpThreads * kVec / kLpWaves;
      const int lo = max(first * kVec + wave * span - off, 0), hi = min(first * kVec + (wave + 1) * span - off, V);
      uint64_t least = 0;  // the top-th of the list
      int n = 0;
      const auto flush = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        best = lp_merge(best, lp_sort(lane < n ? mine[lane] : 0));
        least = lp_shfl(best, a.top - 1);
        const uint64_t rest = kWave + lane < n ? mine[kWave + lane] : 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (kWave + lane < n) mine[lane] = rest;
        n = max(n - kWave, 0);
      };
      for (int i0 = lo; i0 < hi; i0 += kAhead * kWave) {  // uniform in the wave
        Elem v[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) v[i] = reinterpret_cast<const Elem*>(base)[min(i0 + i * kWave + lane, hi - 1)];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int id = i0 + i * kWave + lane;
          const uint64_t key = id < hi ? lp_key(lp_order(Type::value(v[i])), id) : 0;
          const uint64_t in = __ballot(key > least);
          if (in == 0) continue;
          if (key > least) mine[n + __popcll(in & ((1ull << lane) - 1))] = key;
          n += __popcll(in);
          if (n >= kWave) flush();
        }
      }
      while (n > 0) flush();
      __syncthreads();  // all pending keys are done with
      sm.pend[wave * kWave + lane] = best;
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int w = 1; w < kLpWaves; ++w) best = lp_merge(best, sm.pend[w * kWave + lane]);
      }
    }
  }
  if (wave != 0) return;
  top = -__builtin_huge_valf();
  m = kLpLowest;
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) {
    top = lp_max(top, sm.part[w][0]);
    m = lp_max(m, sm.part[w][1]);
  }
  l = s = 0.f;
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) {
    float pm = sm.part[w][1], pl = sm.part[w][2], ps = sm.part[w][3];
    lp_rebase(pm, pl, ps, m);
    l += pl;
    s += ps;
  }
  if (a.segments == 1) return lp_finish(a, row, top, m, l, s, best, token, logit);
  uint8_t* part = a.parts + blockIdx.x * (sizeof(LpPart) + 8 * static_cast<int64_t>(a.top));
  if (lane == 0) *reinterpret_cast<LpPart*>(part) = LpPart{top, m, l, s};
  if (lane < a.top) reinterpret_cast<uint64_t*>(part + sizeof(LpPart))[lane] = best;
}

// grid: rows.  Segments' states and lists, a wave every fourth of them.
template <int kFormat>
__global__ __launch_bounds__(kLpThreads) void k_logprobs_join(LpArgs a) {
  __shared__ float parts[kLpWaves][4];
  __shared__ uint64_t lists[kLpWaves][kWave];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int64_t row = blockIdx.x;
  int64_t token = -1;
  float logit = 0.f;
  if (tid == 0) lp_token<kFormat>(a, row, token, logit);
  const int64_t size = sizeof(LpPart) + 8 * static_cast<int64_t>(a.top);
  const uint8_t* part = a.parts + row * a.segments * size;
  // a lane's segments
  float top = -__builtin_huge_valf(), m = kLpLowest, l = 0.f, s = 0.f;
  for (int i = tid; i < a.segments; i += kLpThreads) {
    LpPart p = *reinterpret_cast<const LpPart*>(part + i * size);
    top = lp_max(top, p.top);
    const float to = lp_max(m, p.m);
    lp_rebase(m, l, s, to);
    lp_rebase(p.m, p.l, p.s, to);
    l += p.l;
    s += p.s;
  }
  float wm = m, wtop = top;
#pragma unroll
  for (int by = 1; by < kWave; by *= 2) {
    wm = lp_max(wm, __shfl_xor(wm, by));
    wtop = lp_max(wtop, __shfl_xor(wtop, by));
  }
  lp_rebase(m, l, s, wm);
#pragma unroll
  for (int by = 1; by < kWave; by *= 2) {
    l += __shfl_xor(l, by);
    s += __shfl_xor(s, by);
  }
  if (lane == 0) {
    parts[wave][0] = wtop;
    parts[wave][1] = wm;
    parts[wave][2] = l;
    parts[wave][3] = s;
  }
  uint64_t best = 0;
  if (a.top > 0) {
    for (int i = wave; i < a.segments; i += kLpWaves) {
      const uint64_t key = lane < a.top ? reinterpret_cast<const uint64_t*>(part + i * size + sizeof(LpPart))[lane] : 0;
      best = lp_merge(best, key);
    }
    lists[wave][lane] = best;
  }
  __syncthreads();
  if (wave != 0) return;
  if (a.top > 0) {
#pragma unroll
    for (int w = 1; w < kLpWaves; ++w) best = lp_merge(best, lists[w][lane]);
  }
  top = -__builtin_huge_valf();
  m = kLpLowest;
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) {
    top = lp_max(top, parts[w][0]);
    m = lp_max(m, parts[w][1]);
  }
  l = s = 0.f;
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) {
    float pm = parts[w][1], pl = parts[w][2], ps = parts[w][3];
    lp_rebase(pm, pl, ps, m);
    l += pl;
    s += ps;
  }
  lp_finish(a, row, top, m, l, s, best, token, logit);
}

struct LpPlan {
  int elem, vec;
  int64_t chunks, segments;  // of a segment; of a row
  int64_t ws_bytes;
};

int lp_plan(int64_t rows, int64_t vocab, int32_t format, int64_t top, LpPlan& p) {
  const char* what = "skv_token_logprobs";
  if (format < SKV_LOGITS_BF16 || format > SKV_LOGITS_F32) return set_error(SKV_EINVAL, "%s: unknown format %d", what, format);
  if (vocab < 1 || vocab > (1 << 24)) return set_error(SKV_EINVAL, "%s: vocab must be in [1, 2^24]; got %lld", what, (long long)vocab);
  if (rows < 0 || rows > (1 << 24)) return set_error(SKV_EINVAL, "%s: rows must be in [0, 2^24]; got %lld", what, (long long)rows);
  if (top < 0 || top > kLpMaxTop || top > vocab) {
    return set_error(SKV_EINVAL, "%s: top must be in [0, %d] and at most vocab; got %lld", what, kLpMaxTop, (long long)top);
  }
  p.elem = format == SKV_LOGITS_F32 ? 4 : 2;
  p.vec = 16 / p.elem;
  // chunks of a row that begins anywhere between 16-byte boundaries
  const int64_t chunks = ceil_div(ceil_div(vocab + p.vec - 1, p.vec), kLpVecs * kLpThreads);
  const int64_t wanted = std::min<int64_t>(chunks, ceil_div(4 * device_cus(), std::max<int64_t>(rows, 1)));
  p.chunks = std::min<int64_t>(kLpMaxChunks, ceil_div(chunks, wanted));
  p.segments = ceil_div(chunks, p.chunks);
  if (rows * p.segments >= (int64_t{1} << 31)) return set_error(SKV_EINVAL, "%s: too many rows of so many logits", what);
  p.ws_bytes = p.segments > 1 ? rows * p.segments * (static_cast<int64_t>(sizeof(LpPart)) + 8 * top) : 0;
  return SKV_OK;
}

template <int kFormat>
int lp_launch(const LpArgs& a, hipStream_t s, const char* what) {
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.rows) * a.segments));
  if (a.top > 0) {
    hipLaunchKernelGGL((k_logprobs<kFormat, true>), grid, dim3(kLpThreads), a.chunks * kLpThreads * 4, s, a);
  } else {
    hipLaunchKernelGGL((k_logprobs<kFormat, false>), grid, dim3(kLpThreads), 0, s, a);
  }
  if (const int rc = check_launch(what)) return rc;
  if (a.segments == 1) return SKV_OK;
  hipLaunchKernelGGL((k_logprobs_join<kFormat>), dim3(static_cast<unsigned>(a.rows)), dim3(kLpThreads), 0, s, a);
  return check_launch(what);
}

}  // namespace skv

using namespace skv;

extern "C" int64_t skv_token_logprobs_workspace(int64_t rows, int64_t vocab, int32_t format, int64_t top) {
  LpPlan p;
  return lp_plan(rows, vocab, format, top, p) == SKV_OK ? p.ws_bytes : -1;
}

extern "C" int skv_token_logprobs(const void* logits, int64_t rows, int64_t vocab, int64_t row_stride, int32_t format,
                                  const skv_token_ids* tokens, int64_t top, float* logprobs, float* entropy, int32_t* top_ids,
                                  float* top_logprobs, void* workspace, int64_t ws_bytes, void* stream) {
  const char* what = "skv_token_logprobs";
  LpPlan p;
  if (const int rc = lp_plan(rows, vocab, format, top, p)) return rc;
  if (rows == 0) return SKV_OK;
  if (!logits || !entropy || (tokens && (!tokens->data || !logprobs)) || (top > 0 && (!top_ids || !top_logprobs))) {
    return set_error(SKV_EINVAL, "%s: NULL pointer", what);
  }
  if (row_stride < 0) return set_error(SKV_EINVAL, "%s: row_stride must be >= 0", what);
  if (reinterpret_cast<uintptr_t>(logits) % p.elem) return set_error(SKV_EINVAL, "%s: logits must be aligned to their size", what);
  if (p.ws_bytes > 0 && (!workspace || ws_bytes < p.ws_bytes || (reinterpret_cast<uintptr_t>(workspace) & 15))) {
    return set_error(SKV_EINVAL, "%s: a 16-byte aligned workspace of %lld bytes is needed", what, (long long)p.ws_bytes);
  }
  LpArgs a{};
  a.x = static_cast<const uint8_t*>(logits);
  a.row_bytes = row_stride * p.elem;
  a.vocab = vocab;
  a.rows = static_cast<int32_t>(rows);
  a.top = static_cast<int32_t>(top);
  a.chunks = static_cast<int32_t>(p.chunks);
  a.segments = static_cast<int32_t>(p.segments);
  if (tokens) {
    a.tokens = tokens->data;
    a.tok_stride = tokens->tok_stride;
    a.wide = tokens->wide;
    a.logprobs = logprobs;
  }
  a.entropy = entropy;
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  a.parts = static_cast<uint8_t*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (format == SKV_LOGITS_BF16) return lp_launch<SKV_LOGITS_BF16>(a, s, what);
  if (format == SKV_LOGITS_F16) return lp_launch<SKV_LOGITS_F16>(a, s, what);
  return lp_launch<SKV_LOGITS_F32>(a, s, what);
}
