// Log probabilities of given tokens, the entropy and the most likely tokens of rows of logits.
//
//   m = max x, l = sum exp(x - m), s = sum exp(x - m) (x - m)
//   logprob = x_token - m - ln l,  entropy = ln l - s / l
//
// One pass over a row: a lane keeps a running m, l and s of the logits that it sees; lanes, waves and (of rows
// that several workgroups share) segments are joined by exp(m_i - m), under which s_i becomes s_i + l_i (m_i - m).
// HBM bounds it with many rows (each logit is read once), the vector work close behind: about five instructions
// and an exponential a logit.  A launch over 3001 rows of 100,003 logits, 8 alternatives: 113 us of fp16 (5.3 TB/s, some
// rows half -inf), 191 of fp32 (6.3 TB/s); over 256 of 131,072 bf16, 20 alternatives: 17 - 19 us (3.5 - 4 TB/s, the last steps
// of rows that all end at once); one of 32,000 fp32 in a graph of several: 8.5 us.
//
// The `top` largest cost next to nothing on the way: a lane notes the maximum of every 64 bytes (4 loads of 16)
// that it sees, in LDS.  The top-th largest of the lanes' own maxima is a bound that at least `top` logits
// reach, and little more do (of 256 lanes and 20 wanted about 21); only the noted 64 bytes that reach it are
// read again and what reaches it in them is sorted, by value and then id, as one 64-bit key.  Where too much
// does (equal logits throughout, or most of a row -inf), the waves go through the row once more with a list
// of the best so far each (256 rows of 131,072 zeros: 46 us).
#include <algorithm>
#include <type_traits>

#include "skv_common.h"

// A rounded product and its rest are told apart below: fused operations are those written as such.
#pragma clang fp contract(off)

namespace skv {

constexpr int kLpSmall = 256, kLpLarge = 1024;  // threads of a workgroup
constexpr int kLpVecs = 4;     // 16-byte loads of a lane's chunk
constexpr int kLpMaxTop = 64;  // a wave's list
constexpr int kLpBins = 256;   // lanes' maxima, or those of four lanes
constexpr int kLpMine = 2 * kWave;  // a wave's pending keys: 63 and a load's 64
// Chunks of a segment whose maxima LDS holds.
constexpr int lp_max_chunks(int threads) { return threads == kLpSmall ? 32 : 8; }
constexpr float kLpLog2e = 1.4426950408889634f;
constexpr float kLpLowest = -3.4028234663852886e38f;
constexpr float kLpLn2 = 0.6931471805599453f;
constexpr float kLpGone = -1e4f;   // exp of it is 0; times 0 it is 0, as -inf would not be
constexpr float kLpFar = 1e37f;       // logits up to it stay finite in the log2 domain
// Of maxima up to it the product with log2(e) is rounded by at most 4 (a step is 8 there): weights up to 2^4.
constexpr float kLpHuge = 67108864.f;

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

// The value of lane ^ kBy, without LDS: within a row of 16 lanes by its permutes (xor 4 is the mirror of 8 lanes,
// xor 7, and that of 4, xor 3), across rows by swaps.
template <int kBy>
__device__ __forceinline__ uint32_t lp_xor(uint32_t v) {
  const auto dpp = [](auto ctrl, uint32_t x) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  if constexpr (kBy == 1) return dpp(std::integral_constant<int, 0xb1>{}, v);   // quad_perm 1 0 3 2
  if constexpr (kBy == 2) return dpp(std::integral_constant<int, 0x4e>{}, v);   // quad_perm 2 3 0 1
  if constexpr (kBy == 4) return dpp(std::integral_constant<int, 0x1b>{}, dpp(std::integral_constant<int, 0x141>{}, v));
  if constexpr (kBy == 8) return dpp(std::integral_constant<int, 0x128>{}, v);  // row_ror 8
  if constexpr (kBy == 16) {  // rows 0 1 2 3 of the first with those of the second: 0 0 2 2 and 1 1 3 3
    const auto x = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? x[0] : x[1];
  }
  if constexpr (kBy == 32) {
    const auto x = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? x[0] : x[1];
  }
}
template <int kBy>
__device__ __forceinline__ uint64_t lp_xor64(uint64_t v) {
  return static_cast<uint64_t>(lp_xor<kBy>(static_cast<uint32_t>(v >> 32))) << 32 | lp_xor<kBy>(static_cast<uint32_t>(v));
}
// f(x of lane ^ 1), then ^ 2, ^ 4 .. ^ 32.
template <class F>
__device__ __forceinline__ void lp_lanes(const F& f) {
  f(std::integral_constant<int, 1>{});
  f(std::integral_constant<int, 2>{});
  f(std::integral_constant<int, 4>{});
  f(std::integral_constant<int, 8>{});
  f(std::integral_constant<int, 16>{});
  f(std::integral_constant<int, 32>{});
}
template <int kBy>
__device__ __forceinline__ float lp_xorf(float v) { return __uint_as_float(lp_xor<kBy>(__float_as_uint(v))); }
__device__ __forceinline__ uint64_t lp_shfl(uint64_t v, int from) {
  const uint32_t lo = __shfl(static_cast<int>(v), from), hi = __shfl(static_cast<int>(v >> 32), from);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// One step of a bitonic sort: of lanes kBy apart the lower one keeps the larger key where `down`.
template <int kBy>
__device__ __forceinline__ uint64_t lp_step(uint64_t v, bool down) {
  const uint64_t o = lp_xor64<kBy>(v);
  return (o > v) == (down == ((threadIdx.x & kBy) == 0)) ? o : v;
}
// Of blocks of kSize keys that rise and then fall (or the other way round) the order asked for.
template <int kSize>
__device__ __forceinline__ uint64_t lp_bitonic(uint64_t v, bool down) {
  if constexpr (kSize >= 64) v = lp_step<32>(v, down);
  if constexpr (kSize >= 32) v = lp_step<16>(v, down);
  if constexpr (kSize >= 16) v = lp_step<8>(v, down);
  if constexpr (kSize >= 8) v = lp_step<4>(v, down);
  if constexpr (kSize >= 4) v = lp_step<2>(v, down);
  return lp_step<1>(v, down);
}
// A wave's 64 keys, one a lane, in descending order.
__device__ __forceinline__ uint64_t lp_sort(uint64_t v) {
  const int lane = threadIdx.x;
  v = lp_bitonic<2>(v, (lane & 2) == 0);
  v = lp_bitonic<4>(v, (lane & 4) == 0);
  v = lp_bitonic<8>(v, (lane & 8) == 0);
  v = lp_bitonic<16>(v, (lane & 16) == 0);
  v = lp_bitonic<32>(v, (lane & 32) == 0);
  return lp_bitonic<64>(v, true);
}
// The 64 largest of two lists in descending order, in that order.
__device__ __forceinline__ uint64_t lp_merge(uint64_t a, uint64_t b) {
  const uint64_t o = lp_shfl(b, kWave - 1 - threadIdx.x % kWave);
  return lp_bitonic<64>(o > a ? o : a, true);
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

template <bool kTop, int kThreads>
struct LpSmem {
  static constexpr int kWaves = kThreads / kWave;
  static constexpr int kList = 256;               // chunks read again
  static constexpr int kPend = kWaves * kLpMine;  // logits that reach the bound
  float part[kWaves][4];
  uint32_t bins[kTop ? kLpBins : 1];
  uint32_t bound;
  int n_list, n_pend;
  int32_t list[kTop ? kList : 1];
  uint64_t pend[kTop ? kPend : 1];
};

// grid: rows x segments.  A segment is `chunks` times kThreads * kLpVecs vectors of the row, which are
// counted from the 16-byte boundary at or before its first logit.
template <int kFormat, bool kTop, int kThreads>
__global__ __launch_bounds__(kThreads) void k_logprobs(LpArgs a) {
  using Smem = LpSmem<kTop, kThreads>;
  constexpr int kWaves = Smem::kWaves;
  using Type = LpType<kFormat>;
  using Elem = typename Type::elem;
  constexpr int kVec = Type::kVec, kElems = kVec * kLpVecs;
  __shared__ Smem sm;
  extern __shared__ float noted[];  // [chunks][kThreads]
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
  const int first = seg * a.chunks * kLpVecs * kThreads;  // vector
  // chunks that hold logits: the last may be there for rows that begin off a boundary alone
  const int chunks = min(a.chunks, ((end + kVec - 1) / kVec - first + kLpVecs * kThreads - 1) / (kLpVecs * kThreads));
  const auto vector_of = [&](int c, int i) { return first + (c * kLpVecs + i) * kThreads + tid; };
  const auto load = [&](u32x4* r, int c) {
    const int v0 = first + c * kLpVecs * kThreads;
    if (v0 * kVec >= off && (v0 + kLpVecs * kThreads) * kVec <= end) {  // uniform: inside the row
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
  // In the log2 domain: l = sum 2^(x log2(e) - c), s = sum of the same times its exponent, c = m log2(e) rounded; of a
  // product and c the difference is one rounding.  m stays within kLpHuge: a lane that sees less has weights near 0, and
  // waves whose maximum is past it (c's rounding would be) go through their logits again below.
  float m = -kLpHuge, c = -kLpHuge * kLpLog2e, l = 0.f, s = 0.f, top = -__builtin_huge_valf();
  const auto fold = [&](const u32x4* r, int k) {
    float x[kElems];
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) Type::unpack(r[i], x + i * kVec);
    float most = x[0], least = x[0];
#pragma unroll
    for (int i = 1; i < kElems; ++i) {
      most = lp_max(most, x[i]);
      least = fminf(least, x[i]);
    }
    if (kTop) noted[k * kThreads + tid] = most;
    top = lp_max(top, most);
    m = fminf(fmaxf(m, most), kLpHuge);
    const float up = m * kLpLog2e, by = fmaxf(c - up, kLpGone), f = __builtin_amdgcn_exp2f(by);
    s = f * __builtin_fmaf(l, by, s);  // finite before it meets a weight of 0
    l *= f;
    c = up;
    float lk[4] = {0.f, 0.f, 0.f, 0.f}, sk[4] = {0.f, 0.f, 0.f, 0.f};
    const auto sum = [&](auto clamped) {
#pragma unroll
      for (int i = 0; i < kElems; ++i) {
        float d = __builtin_fmaf(x[i], kLpLog2e, -c);
        if constexpr (decltype(clamped)::value) d = fmaxf(d, kLpGone);
        const float e = __builtin_amdgcn_exp2f(d);
        lk[i & 3] += e;
        sk[i & 3] = __builtin_fmaf(e, d, sk[i & 3]);
      }
    };
    // an exponent of -inf has to go before it meets its weight of 0: where a lane of the wave has one
    if (__ballot(!(least >= -kLpFar))) sum(std::true_type{}); else sum(std::false_type{});
    l += (lk[0] + lk[1]) + (lk[2] + lk[3]);
    s += (sk[0] + sk[1]) + (sk[2] + sk[3]);
  };
  u32x4 r0[kLpVecs], r1[kLpVecs];
  if (chunks > 0) load(r0, 0);
  int at = 0;
  for (; at + 1 < chunks; at += 2) {
    load(r1, at + 1);
    fold(r0, at);
    if (at + 2 < chunks) load(r0, at + 2);
    fold(r1, at + 1);
  }
  if (at < chunks) fold(r0, at);
  // join the lanes, then the waves; and back to m itself: c = m log2(e) - r
  float wm = m, wtop = top;
  lp_lanes([&](auto by) {
    wm = fmaxf(wm, lp_xorf<decltype(by)::value>(wm));
    wtop = lp_max(wtop, lp_xorf<decltype(by)::value>(wtop));
  });
  {
    const float up = wm * kLpLog2e, r = __builtin_fmaf(wm, kLpLog2e, -up);
    const float by = fmaxf((c - up) - r, kLpGone), f = __builtin_amdgcn_exp2f(by);
    s = f * __builtin_fmaf(l, by, s) * kLpLn2;
    l *= f;
    m = wm;
  }
  lp_lanes([&](auto by) {
    l += lp_xorf<decltype(by)::value>(l);
    s += lp_xorf<decltype(by)::value>(s);
  });
  if (__builtin_fabsf(wtop) > kLpHuge && __builtin_fabsf(wtop) < __builtin_huge_valf()) {  // uniform in the wave
    // too large for that: once more by differences
    m = kLpLowest;
    l = s = 0.f;
    for (int k = 0; k < chunks; ++k) {
      load(r0, k);
      float x[kElems];
#pragma unroll
      for (int i = 0; i < kLpVecs; ++i) Type::unpack(r0[i], x + i * kVec);
#pragma unroll
      for (int i = 0; i < kElems; ++i) {
        const float d = fmaxf(x[i] - wtop, kLpGone), e = __builtin_amdgcn_exp2f(d * kLpLog2e);
        l += e;
        s = __builtin_fmaf(e, d, s);
      }
    }
    wm = wtop;
    lp_lanes([&](auto by) {
      l += lp_xorf<decltype(by)::value>(l);
      s += lp_xorf<decltype(by)::value>(s);
    });
  }
  if (lane == 0) {
    sm.part[wave][0] = wtop;
    sm.part[wave][1] = wtop == -__builtin_huge_valf() ? kLpLowest : wm;  // (nothing but -inf: below all others)
    sm.part[wave][2] = l;
    sm.part[wave][3] = s;
  }
  if constexpr (kTop) {
    uint32_t bin = lp_order(top);
    if constexpr (kThreads > kLpBins) {  // of four lanes
      static_assert(kThreads == 4 * kLpBins, "a bin is a lane's or four lanes'");
      bin = max(bin, lp_xor<1>(bin));
      bin = max(bin, lp_xor<2>(bin));
      if ((tid & 3) == 0) sm.bins[tid >> 2] = bin;
    } else {
      sm.bins[tid] = bin;
    }
  }
  __syncthreads();
  uint64_t best = 0;
  if constexpr (kTop) {
    // the bound: the largest that `top` bins reach
    if (wave == 0) {
      constexpr int kOf = kLpBins / kWave;
      uint32_t b[kOf], t = 0;
#pragma unroll
      for (int i = 0; i < kOf; ++i) b[i] = sm.bins[i * kWave + lane];
#pragma unroll
      for (int bit = 31; bit >= Type::kLowBit; --bit) {
        const uint32_t up = t | 1u << bit;
        int n = 0;
#pragma unroll
        for (int i = 0; i < kOf; ++i) n += __popcll(__ballot(b[i] >= up));
        if (n >= a.top) t = up;
      }
      if (lane == 0) sm.bound = t;
    }
    __syncthreads();
    const uint32_t bound = sm.bound;
    if (lp_order(top) >= bound) {
      for (int k = 0; k < chunks; ++k) {
        if (lp_order(noted[k * kThreads + tid]) >= bound) {
          const int at = atomicAdd(&sm.n_list, 1);
          if (at < Smem::kList) sm.list[at] = k * kThreads + tid;
        }
      }
    }
    __syncthreads();
    const int listed = sm.n_list;
    if (listed <= Smem::kList) {  // uniform
      for (int i = tid / kElems; i < listed; i += kThreads / kElems) {
        const int at = sm.list[i], k = at / kThreads, t = at % kThreads, e = tid % kElems;
        const int id = (first + (k * kLpVecs + e / kVec) * kThreads + t) * kVec + e % kVec - off;
        if (id < 0 || id >= V) continue;
        const uint32_t order = lp_order(Type::value(reinterpret_cast<const Elem*>(base)[id]));
        if (order >= bound) {
          const int p = atomicAdd(&sm.n_pend, 1);
          if (p < Smem::kPend) sm.pend[p] = lp_key(order, id);
        }
      }
    }
    __syncthreads();
    const int pending = sm.n_pend;
    if (listed <= Smem::kList && pending <= Smem::kPend) {  // uniform
      if (wave == 0) {
        best = lp_sort(lane < pending ? sm.pend[lane] : 0);
        for (int p = kWave; p < pending; p += kWave) best = lp_merge(best, lp_sort(p + lane < pending ? sm.pend[p + lane] : 0));
      }
    } else {
      // a part of the segment to each wave, in the order of the ids, and a list of the best so far
      __syncthreads();  // pend has been counted
      constexpr int kAhead = 8;
      uint64_t* mine = sm.pend + wave * kLpMine;
      const int span = max(chunks, 0) * kLpVecs * kThreads * kVec / kWaves;
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
        for (int w = 1; w < kWaves; ++w) best = lp_merge(best, sm.pend[w * kWave + lane]);
      }
    }
  }
  if (wave != 0) return;
  top = -__builtin_huge_valf();
  m = kLpLowest;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    top = lp_max(top, sm.part[w][0]);
    m = lp_max(m, sm.part[w][1]);
  }
  l = s = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
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
__global__ __launch_bounds__(kLpSmall) void k_logprobs_join(LpArgs a) {
  __shared__ float parts[(kLpSmall / kWave)][4];
  __shared__ uint64_t lists[(kLpSmall / kWave)][kWave];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int64_t row = blockIdx.x;
  int64_t token = -1;
  float logit = 0.f;
  if (tid == 0) lp_token<kFormat>(a, row, token, logit);
  const int64_t size = sizeof(LpPart) + 8 * static_cast<int64_t>(a.top);
  const uint8_t* part = a.parts + row * a.segments * size;
  // a lane's segments
  float top = -__builtin_huge_valf(), m = kLpLowest, l = 0.f, s = 0.f;
  for (int i = tid; i < a.segments; i += kLpSmall) {
    LpPart p = *reinterpret_cast<const LpPart*>(part + i * size);
    top = lp_max(top, p.top);
    const float to = lp_max(m, p.m);
    lp_rebase(m, l, s, to);
    lp_rebase(p.m, p.l, p.s, to);
    l += p.l;
    s += p.s;
  }
  float wm = m, wtop = top;
  lp_lanes([&](auto by) {
    wm = lp_max(wm, lp_xorf<decltype(by)::value>(wm));
    wtop = lp_max(wtop, lp_xorf<decltype(by)::value>(wtop));
  });
  lp_rebase(m, l, s, wm);
  lp_lanes([&](auto by) {
    l += lp_xorf<decltype(by)::value>(l);
    s += lp_xorf<decltype(by)::value>(s);
  });
  if (lane == 0) {
    parts[wave][0] = wtop;
    parts[wave][1] = wm;
    parts[wave][2] = l;
    parts[wave][3] = s;
  }
  uint64_t best = 0;
  if (a.top > 0) {
    for (int i = wave; i < a.segments; i += (kLpSmall / kWave)) {
      const uint64_t key = lane < a.top ? reinterpret_cast<const uint64_t*>(part + i * size + sizeof(LpPart))[lane] : 0;
      best = lp_merge(best, key);
    }
    lists[wave][lane] = best;
  }
  __syncthreads();
  if (wave != 0) return;
  if (a.top > 0) {
#pragma unroll
    for (int w = 1; w < (kLpSmall / kWave); ++w) best = lp_merge(best, lists[w][lane]);
  }
  top = -__builtin_huge_valf();
  m = kLpLowest;
#pragma unroll
  for (int w = 0; w < (kLpSmall / kWave); ++w) {
    top = lp_max(top, parts[w][0]);
    m = lp_max(m, parts[w][1]);
  }
  l = s = 0.f;
#pragma unroll
  for (int w = 0; w < (kLpSmall / kWave); ++w) {
    float pm = parts[w][1], pl = parts[w][2], ps = parts[w][3];
    lp_rebase(pm, pl, ps, m);
    l += pl;
    s += ps;
  }
  lp_finish(a, row, top, m, l, s, best, token, logit);
}

struct LpPlan {
  int elem, vec, threads;
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
  const int64_t cus = device_cus();
  // chunks of a row that begins anywhere between 16-byte boundaries
  const auto chunks_of = [&](int threads) { return ceil_div(ceil_div(vocab + p.vec - 1, p.vec), kLpVecs * threads); };
  // Rows for every compute unit four times over: a workgroup of 256 threads each.  Fewer are cut into segments for as
  // many workgroups, which a second launch joins; but for no more rows than compute units one workgroup of 1024 threads,
  // which has as much in flight as four, does with one launch what is not too long for it (us, bf16, 20 alternatives):
  //   1, 64, 256 rows of 32,000    7.6, 8.3, 9.0 for 9.9, 10.5, 14.1      384 rows  15.6 for 16.0, 768  24.5 for 26.7, 1024  32.4 for 21.2
  //   1, 64, 256 rows of 131,072   13.6, 13.6, 19.1 for 11.2, 15.0, 24.8
  //   1, 64, 256 rows of 262,144   24.3, 26.3, 51.4 for 12.9, 17.8, 38.3
  // and rows that 256 threads see at once need no more (64 rows of 5,000: 9.2 for 7.3).
  const bool wide = rows <= cus && chunks_of(kLpSmall) > 1 &&
                    (chunks_of(kLpLarge) <= 3 || (chunks_of(kLpLarge) <= 5 && 4 * rows >= cus));
  p.threads = wide ? kLpLarge : kLpSmall;
  const int64_t chunks = chunks_of(p.threads);
  const int64_t wanted = wide ? 1 : std::min<int64_t>(chunks, ceil_div(4 * cus, std::max<int64_t>(rows, 1)));
  p.chunks = std::min<int64_t>(lp_max_chunks(p.threads), ceil_div(chunks, wanted));
  p.segments = ceil_div(chunks, p.chunks);
  if (rows * p.segments * p.threads >= (int64_t{1} << 32)) return set_error(SKV_EINVAL, "%s: too many rows of so many logits", what);
  p.ws_bytes = p.segments > 1 ? rows * p.segments * (static_cast<int64_t>(sizeof(LpPart)) + 8 * top) : 0;
  return SKV_OK;
}

template <int kFormat, int kThreads>
void lp_launch_rows(const LpArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.rows) * a.segments));
  if (a.top > 0) {
    hipLaunchKernelGGL((k_logprobs<kFormat, true, kThreads>), grid, dim3(kThreads), a.chunks * kThreads * 4, s, a);
  } else {
    hipLaunchKernelGGL((k_logprobs<kFormat, false, kThreads>), grid, dim3(kThreads), 0, s, a);
  }
}

template <int kFormat>
int lp_launch(const LpArgs& a, int threads, hipStream_t s, const char* what) {
  if (threads == kLpSmall) lp_launch_rows<kFormat, kLpSmall>(a, s); else lp_launch_rows<kFormat, kLpLarge>(a, s);
  if (const int rc = check_launch(what)) return rc;
  if (a.segments == 1) return SKV_OK;
  hipLaunchKernelGGL((k_logprobs_join<kFormat>), dim3(static_cast<unsigned>(a.rows)), dim3(kLpSmall), 0, s, a);
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
  if (format == SKV_LOGITS_BF16) return lp_launch<SKV_LOGITS_BF16>(a, p.threads, s, what);
  if (format == SKV_LOGITS_F16) return lp_launch<SKV_LOGITS_F16>(a, p.threads, s, what);
  return lp_launch<SKV_LOGITS_F32>(a, p.threads, s, what);
}
