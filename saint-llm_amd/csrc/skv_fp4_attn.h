// The attention over the 4-bit cache's pages: its waves, segments and launches, of the plain entry point
// (skv_fp4_attention.hip, which describes them) and of the one with a view (skv_fp4_view.hip).
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "skv_fp4.h"

namespace skv {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kF4Threads = 256;
constexpr int kF4Waves = kF4Threads / kWave;
constexpr int kF4Tile = 32;        // positions per tile
constexpr float kF4Log2e = 1.4426950408889634f;
constexpr float kF4Move = 8.f;     // log2: the reference maximum moves when a tile's passes it by more
constexpr float kF4None = -3e38f;  // the reference maximum before the first key: exp2(-inf - kF4None) is 0, not NaN

// Workgroups that a CU holds at once: their four waves share its 4 x 512 registers
// a lane.
constexpr int fp4_resident(int dims, int mt) {
  return dims == 64 ? (mt == 1 ? 4 : 3) : dims == 128 ? (mt == 1 ? 3 : 2) : dims == 256 && mt == 1 ? 2 : 1;
}

// Row tiles of a wave that shares its tiles.
constexpr int fp4_shared_mt(int dims) { return dims <= 128 ? 2 : 1; }

struct Fp4AttnArgs {
  const uint8_t* q;
  int64_t q_seq, q_tok, q_head;
  uint16_t* out;  // [B, T, H, D] bf16
  float* part;    // of chunk parts: (m, l) of every row, then the rows' outputs
  const int32_t* lens;
  const int32_t* n_new;  // each sequence's tokens of the T in q, or null: all
  const uint8_t* pool;
  const int32_t* bt;
  const float* sink;
  int32_t n_pages, bt_stride, bs;
  int32_t B, T, H, Hkv, G, D;
  int32_t window;  // 0: none
  float scale;             // to the log2 domain
  float cap, cap_k;        // the softcap in the log2 domain (0: none); 2 log2(e) scale / softcap
  int32_t row_blocks;
  int32_t* sched;   // for the join: [items + 1] tiles before every (sequence, row block), and `small`
  int32_t lead;     // kF4Lead, or 0
  int32_t max_groups, small;  // see fp4_groups; items of at most `small` tiles are not cut
};

// With a view: of the newest tokens those that a token's mask names, and of a window's
// history the first tokens, too (skv_fp4_view).
struct Fp4ViewArgs : Fp4AttnArgs {
  const uint64_t* tree;  // [B, T, words], or null: every token up to itself
  int32_t words;
  int32_t keep;          // first tokens of a history that stay visible
};
template <bool kView>
using Fp4Args = std::conditional_t<kView, Fp4ViewArgs, Fp4AttnArgs>;

// The positions that the rows [r0, r0 + n) of a K/V head see.
struct Fp4Span {
  int L, T, r_end;       // tokens of the sequence, and new ones among them; rows of the head
  int first, last;       // [first, last): some row sees them
  int all_lo, all_hi;    // [all_lo, all_hi): every row sees them
  int tile0, tiles;
  int head;              // with a view: so many of the tiles are the sequence's first ones, the others follow from tile0 on
  __device__ __forceinline__ int units() const { return max(tiles, 1); }  // an item that sees nothing is one, too
};

__device__ __forceinline__ Fp4Span fp4_span(const Fp4AttnArgs& a, int b, int r0, int n) {
  Fp4Span s;
  s.L = min(max(a.lens[b], 0), a.bt_stride * a.bs);
  s.T = a.n_new ? min(max(a.n_new[b], 0), a.T) : a.T;
  s.r_end = a.T * a.G;
  const int t0 = r0 / a.G, t1 = (min(r0 + n, s.r_end) - 1) / a.G;
  // one past the last position seen
  const int end0 = s.L - s.T + t0 + 1, end1 = s.L - s.T + min(t1, s.T - 1) + 1;
  s.last = t0 < s.T ? max(end1, 0) : 0;
  s.all_hi = t1 < s.T ? end0 : 0;  // a row past the new tokens sees none
  s.first = a.window > 0 ? max(end0 - a.window, 0) : 0;
  s.all_lo = a.window > 0 ? end1 - a.window : 0;
  s.tile0 = s.first / kF4Tile;
  s.tiles = s.last > s.first ? (s.last + kF4Tile - 1) / kF4Tile - s.tile0 : 0;
  return s;
}

__device__ __forceinline__ Fp4Span fp4_span(const Fp4ViewArgs& a, int b, int r0, int n) {
  Fp4Span s = fp4_span(static_cast<const Fp4AttnArgs&>(a), b, r0, n);
  const int t0 = r0 / a.G, base = s.L - s.T;
  if (a.tree) {
    // a token of depth d (at most its own number) is d past the first new one: its window begins at most so far behind
    const bool some = t0 < s.T && base >= 0;
    const int t1 = min((min(r0 + n, s.r_end) - 1) / a.G, s.T - 1);
    s.last = some ? base + t1 + 1 : 0;
    s.all_hi = some ? base : 0;  // (rows that see nothing are cleared at the end)
    s.first = a.window > 0 ? max(base + 1 - a.window, 0) : 0;
    s.all_lo = a.window > 0 ? base + t1 + 1 - a.window : 0;
    s.tile0 = s.first / kF4Tile;
    s.tiles = s.last > s.first ? (s.last + kF4Tile - 1) / kF4Tile - s.tile0 : 0;
  }
  s.head = a.window > 0 && s.tiles > 0 ? min((a.keep + kF4Tile - 1) / kF4Tile, s.tile0) : 0;
  s.tiles += s.head;
  return s;
}

// The tile of the sequence that is number i of a span's (of a span without a view i counts from the
// sequence's first tile on).
template <bool kView>
__device__ __forceinline__ int fp4_tile(const Fp4Span& s, int i) {
  if constexpr (kView) {
    return i < s.head ? i : s.tile0 - s.head + i;
  } else {
    return i;
  }
}
template <bool kView>
__device__ __forceinline__ int fp4_tile_base(const Fp4Span& s) { return kView ? 0 : s.tile0; }

// Workgroups that share the units: a run of fewer than 8 tiles, 2 a wave, is not
// worth a workgroup, but an item is.  Workgroup i of n takes total / n tiles,
// the first total mod n one more.
constexpr int kF4RunTiles = 8;
constexpr int kF4SmallTiles = 16;
// What a segment costs beside its tiles, in tiles: the first loads' latencies and the
// waves' join.  A step of 64 sequences of 1k - 32k, 8 K/V heads: 156 us without it, with 12 tiles
// 135 and with 20 131 us; the other cases of skv_fp4_attention.hip stay within 1%.  Counted where
// there are about as many items as workgroups or more; a run that would begin in this
// lead or just past it begins with the item.
constexpr int kF4Lead = 20;
// No (sequence, row block, head) is cut where a workgroup for each leaves less than an
// eighth of the chip's time unused: there is nothing to join then.
constexpr int kF4Idle = 8;
constexpr int kF4MaxItems = 2048;  // (sequence, row block)s whose prefix sum LDS holds

__device__ __forceinline__ int fp4_groups(const Fp4AttnArgs& a, int total) {
  const int units = a.B * a.row_blocks * a.Hkv;
  return min(a.max_groups, max((total - units * a.lead + kF4RunTiles - 1) / kF4RunTiles, units));
}
// A run that begins at most so far into an item begins with it.
__device__ __forceinline__ int fp4_early(const Fp4AttnArgs& a) { return a.lead ? a.lead + kF4Waves : 0; }
__device__ __forceinline__ int fp4_run_start(int i, int total, int n) {
  const uint32_t each = static_cast<uint32_t>(total) / static_cast<uint32_t>(n);
  return static_cast<int>(i * each) + min(i, static_cast<int>(total - n * each));
}
// The workgroup whose run holds unit x.
__device__ __forceinline__ int fp4_owner(int x, int total, int n) {
  const uint32_t each = static_cast<uint32_t>(total) / static_cast<uint32_t>(n), more = total - n * each, longer = more * (each + 1);
  const uint32_t u = x;
  return static_cast<int>(u < longer ? u / (each + 1) : more + (u - longer) / each);
}

// cap tanh(x) of a score s in the log2 domain: lin s is the score without the cap, k s = u is
// 2x log2(e).  tanh(x) = 1 - 2 / (exp(2x) + 1) has an error of 2^-23 whatever x is, which a cap far above
// the scores would make as large as they are; for |x| < 1/4 the series stands instead, as a factor of
// the score itself (its first term left out is 2^-26 there).  On either side 2^-20 of the result.
struct Fp4Cap {
  float lin, k, cap;
  float c[4], sq;  // the series' coefficients; x^2 = sq u^2
  __device__ __forceinline__ Fp4Cap(float lin_, float k_, float cap_) : lin(lin_), k(k_), cap(cap_) {
    c[0] = -1.f / 3.f;
    c[1] = 2.f / 15.f;
    c[2] = -17.f / 315.f;
    c[3] = 62.f / 2835.f;
    sq = 0.25f / (kF4Log2e * kF4Log2e);
    // made here, in scalar registers: as vector registers held through the tiles they cost calls without a
    // cap 1-2% (64 sequences of 1k - 32k 137.6 us for 136.0, 4 of 256k - 1M 93.7 for 92.1)
    asm volatile("" : "+s"(c[0]), "+s"(c[1]), "+s"(c[2]), "+s"(c[3]), "+s"(sq));
  }
  __device__ __forceinline__ float operator()(float s) const {
    const float u = s * k, x2 = u * u * sq;
    float f = __builtin_fmaf(x2, c[3], c[2]);
    f = __builtin_fmaf(x2, f, c[1]);
    f = __builtin_fmaf(x2, f, c[0]);
    f = __builtin_fmaf(x2, f, 1.f);
    const float far = cap * (1.f - 2.f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(u) + 1.f));
    return __builtin_fabsf(u) < 0.5f * kF4Log2e ? s * lin * f : far;
  }
};

__device__ __forceinline__ bf16x8 fp4_bf16x8(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }

// The larger of x over the lanes 16, 32 and 48 away, and their sum.
__device__ __forceinline__ float fp4_max_groups(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float fp4_sum_groups(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Chunk c (8 dims) of LDS row r sits at chunk c ^ f(r): the 8 lanes of a cycle
// of a 16-byte write (8 rows, one chunk) and the 16 lanes of a cycle of a
// transposing read (4 rows, an aligned pair of chunks each) touch every bank once.
__device__ __forceinline__ int fp4_chunk(int r, int c) { return c ^ (((r & 3) << 1) | ((r >> 2) & 1)); }

// Four rows of one dim, transposed: lane i of a group of 16 gets dim c + i of
// the rows that the group's lanes point at (lane s: row s / 4, dims c + 4 (s % 4)..).
__device__ __forceinline__ u32x2 fp4_read_tr(const uint16_t* p) {
  const short4v v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(p));
  return __builtin_bit_cast(u32x2, v);
}

// A tile's codes and scale bytes in flight: [16-key half][word of 8 dims].
template <int DP>
struct Fp4Raw {
  static constexpr int kWords = DP / 32;                    // of a lane's quarter of a row
  static constexpr int kScales = DP >= 128 ? DP / 128 : 1;  // 32-dim blocks it reaches into
  static constexpr int kKeyWords = DP >= 128 ? kWords : 4;  // of 64 dims a whole block, each in two lanes
  uint32_t k[2][kKeyWords], v[2][kWords];
  uint32_t ks[2][kScales], vs[2][kScales];
  uint32_t packed[2];  // scale bytes as loaded, of heads of 64 and 128 dims
  int slot[2];  // uniform; -1: not mapped
};

// A tile's scores, and what their masks need (uniform): every row sees every
// key; the halves that are mapped; keys with a NaN block among their values.
template <int MT>
struct Fp4Tile {
  f32x4 st[MT][2];  // row 16 mt + col, keys 16 h + 4 grp + i
  int slot[2];
  bool masked;
  uint32_t nan_keys;
};

template <int kBytes>
struct Fp4Run { using type = uint32_t; };
template <>
struct Fp4Run<2> { using type = uint16_t; };
template <>
struct Fp4Run<8> { using type = u32x2; };

template <int DP, bool kShared>
struct Fp4Smem {
  // per wave: 32 value rows of DP bf16; at the end 16 output rows of DP fp32 (private tiles)
  alignas(16) uint8_t tile[kF4Waves][64 * DP];
  float m[kF4Waves][32], l[kF4Waves][32];
  uint32_t nan_keys[kF4Waves];  // of shared tiles
  int pre[kF4MaxItems + 1];
  int scan[17];
  int longest;
  // of shared tiles the keys' codes and scale bytes, as the lanes hold them: of four tiles and of the next four
  static constexpr bool kKeys = kShared && DP <= 128;
  alignas(16) uint32_t keys[2][kKeys ? kF4Waves : 1][2][kKeys ? (Fp4Raw<DP>::kKeyWords + Fp4Raw<DP>::kScales) * kWave : 4];
};

// Four words of an operand register's eight.
__device__ __forceinline__ u32x4 fp4_quarter(i32x8 v, int half) {
  return half ? u32x4{static_cast<uint32_t>(v[4]), static_cast<uint32_t>(v[5]), static_cast<uint32_t>(v[6]), static_cast<uint32_t>(v[7])}
              : u32x4{static_cast<uint32_t>(v[0]), static_cast<uint32_t>(v[1]), static_cast<uint32_t>(v[2]), static_cast<uint32_t>(v[3])};
}

// DP: the head's dims padded to 64, 128, 256 or 512 (kExact: D == DP).
template <int DP, int MT, bool kExact, bool kShared, bool kView>
struct Fp4Wave {
  using Raw = Fp4Raw<DP>;
  static constexpr int kWords = Raw::kWords, kScales = Raw::kScales;
  static constexpr int kSteps = DP >= 128 ? DP / 128 : 1;  // products of 128 dims, or of the two parts of 64
  static constexpr int kBlocks = DP / 16;  // 16-dim blocks of the output
  static constexpr bool kPacked = kExact && DP <= 128;
  // A weight's bf16 rounding, 2^-9 of it on average over few keys as over many, is as
  // large an error as the output's own.  Waves with tiles of their own carry its rest
  // into a second product, 131 us for a step of 64 sequences and 129 without (64 rows on one
  // head 78 and 66, trees of 7 nodes over 256k - 1M 154 and 128); where the products bound the time (a
  // prompt's chunk 510, with rests 709 us) the rounded weight stands.  Heads of more than 256 dims keep the rests where
  // a view's tiles are shared, too, as the plain call, which shares none, keeps them (6 trees of 99 nodes, 16 heads on 1
  // of 512, in windows of 128: 46 us, 44 without; over 8k 420 and 386).
  static constexpr bool kRest = !kShared || DP > 256;
  // Waves of the same rows split a wide query's steps among them (a step is about 1,100 instructions;
  // 32 windows of 128, 64 rows of 512 dims: 20 us a call, 23 with every wave splitting all four steps).
  static constexpr bool kSplit = !kShared && kSteps > 1;
  static constexpr int kSplitWords = 17 * kWave;
  static constexpr bool kTwo = DP * MT <= 256;  // two tiles in flight; wider ones have registers for one
  // A page is read by one workgroup, or by two: nontemporal loads (a step of 64 sequences 131 us,
  // 151 with plain ones; 4 of 256k - 1M 94 and 103; 64 rows on one head, read twice, 78 either way).
  static constexpr bool kOnce = !kShared && DP * MT <= 256;

  const Fp4Args<kView>& a;
  const Fp4Span& sp;
  const Fp4Page pg;
  int col, grp;
  const uint8_t* head;  // the K/V head's block in page 0
  uint32_t code_at, scale_at;  // the lane's place in 16 keys' codes and scale bytes
  i32x8 q[MT][kSteps][DP >= 128 ? 2 : 1];  // the two parts of the query (64 dims: both in one)
  int q_scale[MT][kSteps];                 // scale byte of k-block g: byte 0 of the first part, byte 1 of the second
  int hi[MT], lo[MT];   // the positions that row 16 mt + col sees
  int keep[kView ? MT : 1];             // with a view: those below keep, too; of a tree hi is the first new token's
  const uint64_t* mask[kView ? MT : 1]; // and those of a row's mask past it see a bit, up to token own
  int own[kView ? MT : 1];
  float m[MT], l[MT];
  f32x4 acc[MT][kBlocks];

  // `split`: LDS where waves of the same rows share the query's split (kSplit), else unused.
  __device__ __forceinline__ Fp4Wave(const Fp4Args<kView>& a_, const Fp4Span& sp_, int b, int hk, int r0, int lane, uint32_t* split = nullptr)
      : a(a_), sp(sp_), pg(fp4_page(a_.bs, a_.Hkv, kExact ? DP : a_.D)) {
    col = lane & 15;
    grp = lane >> 4;
    head = a.pool + hk * pg.head;
    const int nb = dims() / kFp4Block;
    code_at = col * (dims() / 2) + grp * (DP / 8);
    scale_at = col * 2 * nb + grp * kScales;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = r0 + 16 * mt + col;
      const bool in = r < sp.r_end;
      const int t = in ? r / a.G : 0, g = in ? r - t * a.G : 0;
      hi[mt] = in && t < sp.T ? sp.L - sp.T + t + 1 : 0;
      lo[mt] = a.window > 0 ? hi[mt] - a.window : 0;
      if constexpr (kView) look(mt, b, in ? t : a.T);
      const uint8_t* row = a.q + b * a.q_seq + t * a.q_tok + (hk * a.G + g) * a.q_head;
      if constexpr (!kSplit) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) q_scale[mt][s] = load_query(s, row, in, q[mt][s]);
      } else {
        const int s = __builtin_amdgcn_readfirstlane(threadIdx.x) / kWave - mt * kSteps % kF4Waves;  // of these rows this wave's step
        if (s >= 0 && s < kSteps) {
          i32x8 part[2];
          const int scale = load_query(s, row, in, part);
          uint32_t* to = split + (mt * kSteps + s) * kSplitWords;
#pragma unroll
          for (int i = 0; i < 4; ++i) reinterpret_cast<u32x4*>(to)[i * kWave + lane] = fp4_quarter(part[i >> 1], i & 1);
          to[16 * kWave + lane] = scale;
        }
      }
      m[mt] = kF4None;
      l[mt] = 0.f;
#pragma unroll
      for (int x = 0; x < kBlocks; ++x) acc[mt][x] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if constexpr (kSplit) {
      lds_barrier();  // the steps are there
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const uint32_t* from = split + (mt * kSteps + s) * kSplitWords;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const u32x4 x = reinterpret_cast<const u32x4*>(from)[i * kWave + lane];
#pragma unroll
            for (int k = 0; k < 4; ++k) q[mt][s][i >> 1][4 * (i & 1) + k] = static_cast<int>(x[k]);
          }
          q_scale[mt][s] = static_cast<int>(from[16 * kWave + lane]);
        }
      }
      lds_barrier();  // and have been read
    }
  }

  // What row 16 mt + col, of token t, sees with a view.
  __device__ __forceinline__ void look(int mt, int b, int t) {
    keep[mt] = a.window > 0 ? a.keep : 0;
    mask[mt] = nullptr;
    own[mt] = -1;
    if (!a.tree) return;
    const int base = sp.L - sp.T;
    const bool live = t < sp.T && base >= 0;
    const uint64_t* m = a.tree + (static_cast<int64_t>(b) * a.T + (live ? t : 0)) * a.words;
    int seen = 0;
    for (int w = 0; w < a.words; ++w) seen += __popcll(upto(m[w], t - 64 * w));
    if (!live) seen = 0;
    hi[mt] = seen > 0 ? base : 0;
    lo[mt] = 0;
    if (seen == 0) return;
    mask[mt] = m;
    own[mt] = t;
    if (a.window > 0) {
      // of the history, base tokens and those of the mask: the last `window` and the first `keep`
      const int skip = seen - a.window;
      lo[mt] = skip > 0 ? base + nth(m, skip) : base + skip;
      const int more = a.keep - base;
      if (more > 0) keep[mt] = more < seen ? base + nth(m, more) : INT32_MAX;
    }
  }
  // Bits 0 .. n of a word (none where n < 0).
  __device__ __forceinline__ static uint64_t upto(uint64_t w, int n) {
    return n >= 63 ? w : n < 0 ? 0 : w & ((2ull << n) - 1);
  }
  // The place of the set bit that n others come before; there are more than n.
  __device__ __forceinline__ int nth(const uint64_t* m, int n) const {
    int w = 0;
    uint64_t x = m[0];
    while (w + 1 < a.words && __popcll(x) <= n) {
      n -= __popcll(x);
      x = m[++w];
    }
    for (; n > 0; --n) x &= x - 1;
    return 64 * w + __ffsll(static_cast<unsigned long long>(x)) - 1;
  }
  // Bit i: row 16 mt + col's mask has position pos + i, i < 32.
  __device__ __forceinline__ uint32_t bits(int mt, int pos) const {
    const int o = pos - hi[mt];
    if (own[mt] < 0 || o <= -kF4Tile || o > own[mt]) return 0;
    const int w = max(o, 0) >> 6, s = o & 63;
    const uint64_t x = upto(mask[mt][w], own[mt] - 64 * w);
    if (o < 0) return static_cast<uint32_t>(x << -o);
    uint64_t y = x >> s;
    if (s > 32 && w + 1 < a.words) y |= upto(mask[mt][w + 1], own[mt] - 64 * (w + 1)) << (64 - s);
    return static_cast<uint32_t>(y);
  }
  // Rows that see nothing, as all of a tile where the others see it all.
  __device__ __forceinline__ void drop_blind() {
    if constexpr (kView) {
      if (!a.tree) return;  // uniform
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if (own[mt] >= 0) continue;
        m[mt] = kF4None;
        l[mt] = 0.f;
#pragma unroll
        for (int x = 0; x < kBlocks; ++x) acc[mt][x] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  }

  // 16 dims of a query row from `d` on as e4m3 parts: words of the first and the
  // second part, and the scale byte of the 32 dims that this lane and the one 16 away
  // hold the halves of.
  __device__ __forceinline__ uint32_t split16(const uint8_t* row, int d, bool in, uint32_t* hi, uint32_t* lo) const {
    uint32_t x[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool live = in && (kExact || d + 8 * i < a.D);
      const u32x4 v = *reinterpret_cast<const u32x4*>(live ? row + 2 * (d + 8 * i) : a.q);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * i + j] = live ? v[j] : 0u;
    }
    uint32_t big = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) big = max(big, max((x[j] << 16) & 0x7fffffffu, x[j] & 0x7fff0000u));
    big = max(big, static_cast<uint32_t>(__shfl_xor(static_cast<int>(big), 16)));
    const int byte = max(static_cast<int>(big >> 23) - 7, 6);  // the largest lands in [2^7, 2^8)
    const float f = __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float v[4] = {__uint_as_float(x[2 * j] << 16) * f, __uint_as_float(x[2 * j] & 0xffff0000u) * f,
                          __uint_as_float(x[2 * j + 1] << 16) * f, __uint_as_float(x[2 * j + 1] & 0xffff0000u) * f};
      hi[j] = e4m3fn_pack2<true>(v[2], v[3], e4m3fn_pack2<false>(v[0], v[1], 0u));
      float h[4];
      e4m3fn_x4_to_f32(hi[j], h);
      lo[j] = e4m3fn_pack2<true>((v[2] - h[2]) * 32.f, (v[3] - h[3]) * 32.f,
                                 e4m3fn_pack2<false>((v[0] - h[0]) * 32.f, (v[1] - h[1]) * 32.f, 0u));
      if (big >= 0x7f800000u) hi[j] = 0x7f7f7f7fu;  // an infinity or a NaN: NaN scores
    }
    return static_cast<uint32_t>(byte);
  }

  // The query of row 16 mt + col for step s.  The second operand's lane g holds
  // k = 16 g .. + 15 and 64 + 16 g .. + 15 of the 128, and the scale of k-block g (k = 32 g ..);
  // k-block j is dims 32 (j kScales + s) .. as the keys' lanes have them.
  __device__ __forceinline__ int load_query(int s, const uint8_t* row, bool in, i32x8* parts) const {
    const int half = 16 * (grp & 1);
    uint32_t hi[8], lo[8];
    if constexpr (DP >= 128) {
      const uint32_t b0 = split16(row, 32 * ((grp >> 1) * kScales + s) + half, in, hi, lo);
      const uint32_t b1 = split16(row, 32 * ((2 + (grp >> 1)) * kScales + s) + half, in, hi + 4, lo + 4);
      const int from = col + 32 * (grp & 1);  // k-blocks 0, 1 (2, 3) are the first (second) 16 of lanes 0 and 32
      const int a0 = __shfl(static_cast<int>(b0), from), a1 = __shfl(static_cast<int>(b1), from);
      const int own = grp < 2 ? a0 : a1;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        parts[0][i] = static_cast<int>(hi[i]);
        parts[DP >= 128 ? 1 : 0][i] = static_cast<int>(lo[i]);
      }
      return own | (own - 5) << 8;
    } else {
      // k-blocks 0, 1: the first part of dims 0 .. 63; 2, 3: the second part of the same
      const uint32_t b = split16(row, 16 * grp, in, hi, lo);
      const int own = __shfl(static_cast<int>(b), col + 32 * (grp & 1));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        parts[0][i] = static_cast<int>(hi[i]);
        parts[0][i + 4] = static_cast<int>(lo[i]);
      }
      return grp < 2 ? own : own - 5;
    }
  }

  __device__ __forceinline__ int dims() const { return kExact ? DP : a.D; }

  // Where the codes of the 16 positions from `pos` on begin, as an offset from the
  // pool, and their first slot (-1 and page 0: not mapped).
  __device__ __forceinline__ void lookup(int b, int pos, uint64_t& at, int& slot) const {
    const int p = static_cast<int>(udiv24(pos, a.bs));
    int page = pos < sp.last ? a.bt[static_cast<int64_t>(b) * a.bt_stride + p] : -1;
    if (page >= a.n_pages) page = -1;
    slot = page < 0 ? -1 : pos - p * a.bs;
    at = static_cast<uint64_t>(max(page, 0)) * static_cast<uint64_t>(pg.page) + static_cast<uint64_t>(max(slot, 0) * (dims() / 2));
  }

  // The codes of half h of a tile, 16 keys from `kc` on (uniform).
  template <bool kKeys, bool kValues>
  __device__ __forceinline__ void load_codes(Raw& r, int h, const uint8_t* kc) const {
    const uint8_t* vc = kc + pg.v_codes;
    uint32_t lane_at = code_at;
    asm("" : "+v"(lane_at));
    constexpr int kRun = DP >= 128 ? 4 : 2;  // words of one load
    typedef uint32_t run_t __attribute__((ext_vector_type(kRun)));
    const auto get = [&](auto* p) {
      if constexpr (kOnce) {
        return __builtin_nontemporal_load(p);
      } else {
        return *p;
      }
    };
    if constexpr (DP == 64 && kKeys) {  // lanes g and g + 2: block g of the key
      const bool in = kExact || 32 * (grp & 1) < a.D;
      uint32_t key_at = col * (dims() / 2) + 16 * (grp & 1);
      asm("" : "+v"(key_at));
      const u32x4 x = get(reinterpret_cast<const u32x4*>(kc + (in ? key_at : 0u)));
#pragma unroll
      for (int i = 0; i < 4; ++i) r.k[h][i] = in ? x[i] : 0u;
    }
#pragma unroll
    for (int w = 0; w < kWords; w += kRun) {
      const bool in = kExact || grp * (DP / 4) + 8 * w < a.D;
      const uint32_t at = in ? lane_at + 4 * w : 0u;
      if constexpr (DP >= 128 && kKeys) {
        const run_t x = get(reinterpret_cast<const run_t*>(kc + at));
#pragma unroll
        for (int i = 0; i < kRun; ++i) r.k[h][w + i] = in ? x[i] : 0u;
      }
      if constexpr (kValues) {
        const run_t y = get(reinterpret_cast<const run_t*>(vc + at));
#pragma unroll
        for (int i = 0; i < kRun; ++i) r.v[h][w + i] = in ? y[i] : 0u;
      }
    }
  }

  // Both halves' scale bytes.  Heads of 64 and 128 dims: a token's (4 or 8, its
  // key's and its value's) in one load, half h's by the lanes of odd or even g = h, which
  // then hand them to the rest; others a lane's own.
  __device__ __forceinline__ const uint8_t* scales_of(const uint8_t* kc, int slot) const {
    return kc + static_cast<uint32_t>(pg.scales - max(slot, 0) * (dims() / 2 - 2 * (dims() / kFp4Block)));
  }
  template <bool kKeys, bool kValues>
  __device__ __forceinline__ void load_scales(Raw& r, const uint8_t* kc0, int slot0, const uint8_t* kc1, int slot1) const {
    const int nb = dims() / kFp4Block;
    if constexpr (kPacked) {
      using run_t = typename Fp4Run<(kKeys && kValues ? DP / 16 : DP / 32)>::type;
      uintptr_t sc0 = reinterpret_cast<uintptr_t>(scales_of(kc0, slot0)), sc1 = reinterpret_cast<uintptr_t>(scales_of(kc1, slot1));
      asm("" : "+s"(sc0), "+s"(sc1));  // made in scalar registers, then chosen
      const run_t x = *global_from_bits<const run_t>(((grp & 1) ? sc1 : sc0) + col * (DP / 16) + (kKeys ? 0 : DP / 32));
      if constexpr (sizeof(run_t) == 8) {
        r.packed[0] = x[0];
        r.packed[1] = x[1];
      } else {
        r.packed[0] = x;
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* sc = scales_of(h ? kc1 : kc0, h ? slot1 : slot0);
        if constexpr (kExact && kScales > 1) {
          typedef uint8_t run_t __attribute__((ext_vector_type(kScales)));
          if constexpr (kKeys) {
            const run_t x = *reinterpret_cast<const run_t*>(sc + scale_at);
#pragma unroll
            for (int i = 0; i < kScales; ++i) r.ks[h][i] = x[i];
          }
          if constexpr (kValues) {
            const run_t y = *reinterpret_cast<const run_t*>(sc + nb + scale_at);
#pragma unroll
            for (int i = 0; i < kScales; ++i) r.vs[h][i] = y[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < kScales; ++i) {
            const int kb = DP >= 128 ? grp * kScales + i : grp & 1, vb = DP >= 128 ? kb : grp >> 1;
            if constexpr (kKeys) {
              const uint32_t ks = sc[col * 2 * nb + (kb < nb ? kb : 0)];
              r.ks[h][i] = kb < nb ? ks : 127u;
            }
            if constexpr (kValues) {
              const uint32_t vs = sc[col * 2 * nb + nb + (vb < nb ? vb : 0)];
              r.vs[h][i] = vb < nb ? vs : 127u;
            }
          }
        }
      }
    }
  }
  template <bool kKeys, bool kValues>
  __device__ __forceinline__ void unpack_scales(Raw& r) const {
    if constexpr (kPacked) {
      // 64 dims: K0 K1 V0 V1; 128: a word of K's, one of V's, g's block g
      constexpr int kWordsIn = kKeys && kValues ? DP / 64 : 1;
#pragma unroll
      for (int i = 0; i < kWordsIn; ++i) {
        const auto x = __builtin_amdgcn_permlane16_swap(r.packed[i], r.packed[i], false, false);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (DP == 64) {  // g's key block is g % 2, its values' block g / 2
            if constexpr (kKeys) r.ks[h][0] = x[h] >> (8 * (grp & 1));
            if constexpr (kValues) r.vs[h][0] = (x[h] >> ((kKeys ? 16 : 0) + 8 * (grp >> 1))) & 0xff;
          } else if (kKeys && i == 0) {
            r.ks[h][0] = x[h] >> (8 * grp);  // the products take byte 0
          } else {
            r.vs[h][0] = (x[h] >> (8 * grp)) & 0xff;
          }
        }
      }
    }
  }

  // A tile's loads, or those of its keys or its values alone.
  template <bool kKeys, bool kValues>
  __device__ __forceinline__ void fetch(Raw& r, uint64_t at, int slot, int from) const {
    const uint8_t* kc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(at), from + h);
      const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(at >> 32), from + h);
      kc[h] = head + (static_cast<uint64_t>(hi) << 32 | lo);
      r.slot[h] = __builtin_amdgcn_readlane(slot, from + h);
    }
    load_scales<kKeys, kValues>(r, kc[0], r.slot[0], kc[1], r.slot[1]);
    load_codes<kKeys, kValues>(r, 0, kc[0]);
    load_codes<kKeys, kValues>(r, 1, kc[1]);
  }

  // Where not every row sees every key, or a value's block is NaN: the values of
  // keys that no row sees (stale bytes, whose weights are zero) and of NaN blocks
  // become zeros.  Returns the keys with a NaN block, whose scores will be NaN.
  __device__ __forceinline__ uint32_t clean(Raw& r, int pos) const {
    uint32_t nan_keys = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bool nan = false;
#pragma unroll
      for (int i = 0; i < kScales; ++i) nan |= r.vs[h][i] == kFp4NaN;
      const int at = pos + 16 * h + col;
      if (nan || at >= sp.last || (!kView && at < sp.first) || r.slot[h] < 0) {
#pragma unroll
        for (int w = 0; w < kWords; ++w) r.v[h][w] = 0u;
#pragma unroll
        for (int i = 0; i < kScales; ++i) r.vs[h][i] = 127u;
      }
      const uint64_t n = __ballot(nan);
      nan_keys |= static_cast<uint32_t>((n | n >> 16 | n >> 32 | n >> 48) & 0xffff) << (16 * h);
    }
    return nan_keys;
  }

  // Whether a row may not see a key of the tile at `pos`, or a key's values are NaN somewhere.
  __device__ __forceinline__ bool uneven(const int (&slot)[2], int pos) const {
    return pos < sp.all_lo || pos + kF4Tile > sp.all_hi || (slot[0] | slot[1]) < 0;
  }
  __device__ __forceinline__ bool any_nan(const Raw& r) const {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kScales; ++i) nan |= r.vs[0][i] == kFp4NaN || r.vs[1][i] == kFp4NaN;
    return __ballot(nan) != 0;
  }

  // A tile's keys to LDS and from there: words of 16 bytes by lane, then the scales'.
  __device__ __forceinline__ void keep_keys(const Raw& r, uint32_t (*to)[(Raw::kKeyWords + kScales) * kWave], int lane) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int w = 0; w < Raw::kKeyWords; w += 4) {
        reinterpret_cast<u32x4*>(to[h])[(w / 4) * kWave + lane] = u32x4{r.k[h][w], r.k[h][w + 1], r.k[h][w + 2], r.k[h][w + 3]};
      }
#pragma unroll
      for (int s = 0; s < kScales; ++s) to[h][(Raw::kKeyWords + s) * kWave + lane] = r.ks[h][s];
    }
  }
  __device__ __forceinline__ void take_keys(Raw& r, const uint32_t (*from)[(Raw::kKeyWords + kScales) * kWave], int lane) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int w = 0; w < Raw::kKeyWords; w += 4) {
        const u32x4 x = reinterpret_cast<const u32x4*>(from[h])[(w / 4) * kWave + lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) r.k[h][w + i] = x[i];
      }
#pragma unroll
      for (int s = 0; s < kScales; ++s) r.ks[h][s] = from[h][(Raw::kKeyWords + s) * kWave + lane];
    }
  }

  // The scores of 32 keys.
  __device__ __forceinline__ void scores(const Raw& r, Fp4Tile<MT>& tl) const {
    auto& st = tl.st;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) st[mt][0] = st[mt][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        i32x8 k = {0, 0, 0, 0, 0, 0, 0, 0};  // of e2m1 operands the first half counts
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = static_cast<int>(r.k[h][4 * s + i]);
        const int ks = static_cast<int>(r.ks[h][s]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          st[mt][h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q[mt][s][0], st[mt][h], 4, 0, 0, ks, 0, q_scale[mt][s]);
          if constexpr (DP >= 128) {
            st[mt][h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q[mt][s][1], st[mt][h], 4, 0, 0, ks, 1, q_scale[mt][s]);
          }
        }
      }
    }
  }

  // Chunk far + near + i of row r (near + i % 8 < 8).  A swizzle is within eight chunks, so that those eight apart have one
  // address; waves with tiles of their own, which are short of registers, take it so (64 windows of 4k, 64 heads on 8
  // of 128: 55 us, 60 with an address for each; heads of 512 dims 54 and 56; the shared tiles' 205 and 200).
  __device__ __forceinline__ static int chunk(int r, int far, int near, int i) {
    if constexpr (kShared && DP <= 256) return fp4_chunk(r, far + near + i);
    return far + (i & ~7) + fp4_chunk(r, near + (i & 7));
  }

  // 32 keys' values to LDS.
  __device__ __forceinline__ void values(const Raw& r, uint16_t* vt) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint16_t* dst = vt + (16 * h + col) * DP;
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        *reinterpret_cast<u32x4*>(dst + 8 * chunk(col, grp * kWords & ~7, grp * kWords & 7, w)) =
            fp4_decode8(r.v[h][w], fp4_scale(r.vs[h][w / 4 < kScales ? w / 4 : 0]));
      }
    }
  }

  // The tile's scores under their cap and masks, and the rows' maxima with them.  Returns what the
  // scores are multiplied by on the way to the log2 domain.
  __device__ __forceinline__ float settle(Fp4Tile<MT>& tl, int pos) {
    auto& st = tl.st;
    const bool capped = a.cap > 0.f;
    float mult = a.scale;
    if (capped) {  // uniform
      mult = 1.f;
      const Fp4Cap capped_score(a.scale, a.cap_k, a.cap);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int i = 0; i < 4; ++i) st[mt][h][i] = capped_score(st[mt][h][i]);
        }
      }
    }
    if (tl.masked) {  // uniform
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if constexpr (kView) {
          // of the 32 keys: those ahead of hi and those of the mask, less those that are neither in the window nor first
          const auto below = [pos](int end) { return end - pos >= kF4Tile ? ~0u : end > pos ? (1u << (end - pos)) - 1 : 0u; };
          const uint32_t seen = (below(hi[mt]) | bits(mt, pos)) & (~below(lo[mt]) | below(keep[mt]));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t in = tl.slot[h] < 0 ? 0u : seen >> (16 * h + 4 * grp), nan = tl.nan_keys >> (16 * h + 4 * grp);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float v = (nan >> i) & 1 ? __builtin_nanf("") : st[mt][h][i];
              st[mt][h][i] = (in >> i) & 1 ? v : -__builtin_huge_valf();
            }
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // keys 4 grp + i of the half: the first that the row may see, and how many
            const int from = lo[mt] - pos - 16 * h - 4 * grp, to = tl.slot[h] < 0 ? INT32_MIN : hi[mt] - pos - 16 * h - 4 * grp;
            const uint32_t nan = tl.nan_keys >> (16 * h + 4 * grp);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float v = (nan >> i) & 1 ? __builtin_nanf("") : st[mt][h][i];
              st[mt][h][i] = i >= from && i < to ? v : -__builtin_huge_valf();
            }
          }
        }
      }
    }
    // the reference maximum is one for the four lanes of a row, and so is "no score of
    // mine passes it by kF4Move": the row's own maximum is needed where one does
    float mx[MT];
    bool any = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const f32x4 x = st[mt][0], y = st[mt][1];
      // (a NaN score makes its row NaN, whatever the maximum)
      const auto top3 = [](float u, float v, float w) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(u, v), w); };
      mx[mt] = __builtin_elementwise_maximum(top3(top3(top3(x[0], x[1], x[2]), x[3], y[0]), y[1], y[2]), y[3]) * mult;
      any |= mx[mt] > m[mt] + kF4Move;
    }
    if (__ballot(any)) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const float top = fp4_max_groups(mx[mt]);
        const bool move = top > m[mt] + kF4Move;
        const float alpha = move ? __builtin_amdgcn_exp2f(m[mt] - top) : 1.f;
        if (move) m[mt] = top;
        l[mt] *= alpha;
#pragma unroll
        for (int x = 0; x < kBlocks; ++x) acc[mt][x] *= alpha;
      }
    }
    return mult;
  }

  struct Weights {
    u32x4 p[MT], rest[kRest ? MT : 1];
  };

  // The tile's weights as bf16 pairs.
  __device__ __forceinline__ void weigh(const Fp4Tile<MT>& tl, float mult, Weights& w) {
    const auto& st = tl.st;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float e[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[4 * h + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[mt][h][i], mult, -m[mt]));
      }
      l[mt] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t p = bf16_pack2(e[2 * i], e[2 * i + 1]);
        w.p[mt][i] = p;
        if constexpr (kRest) {
          w.rest[mt][i] = bf16_pack2(e[2 * i] - __uint_as_float(p << 16), e[2 * i + 1] - __uint_as_float(p & 0xffff0000u));
        }
      }
    }
  }

  // O^T += V^T P^T: dims 16 x + 4 grp + i of the output, row 16 mt + col.
  __device__ __forceinline__ void product(const Weights& w, const uint16_t* vt) {
    const int vr = 4 * grp + (col >> 2);
    const uint16_t* v0 = vt + vr * DP + 4 * (col & 1);
#pragma unroll
    for (int x = 0; x < kBlocks; ++x) {
      const uint16_t* src = v0 + 8 * chunk(vr, 0, (col & 3) >> 1, 2 * x);
      const u32x2 lo2 = fp4_read_tr(src), hi2 = fp4_read_tr(src + 16 * DP);
      const u32x4 v = u32x4{lo2[0], lo2[1], hi2[0], hi2[1]};
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        acc[mt][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp4_bf16x8(v), fp4_bf16x8(w.p[mt]), acc[mt][x], 0, 0, 0);
        if constexpr (kRest) {
          acc[mt][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp4_bf16x8(v), fp4_bf16x8(w.rest[mt]), acc[mt][x], 0, 0, 0);
        }
      }
    }
  }

  __device__ __forceinline__ void output(Fp4Tile<MT>& tl, int pos, const uint16_t* vt) {
    const float mult = settle(tl, pos);
    Weights w;
    weigh(tl, mult, w);
    product(w, vt);
  }
};

// The thread's index, worked out where it is asked for: what is derived from it for
// the end of a segment would otherwise be made ahead of the tiles and held through them.
__device__ __forceinline__ int fp4_fresh_tid() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// Of the workgroups that share a CU the oldest is served first, so that of equal runs
// its ends long before the youngest's (at 52, 58, 66 and 75 us where four share it),
// and few are left to keep the memory busy.  A workgroup's priority therefore falls at a
// half, three quarters and seven eighths of its run: those behind are served first (66,
// 69, 71 and 73 us).
struct Fp4Pace {
  int next, rest, left;  // tiles of the run up to the next fall, and from there on; falls to come
  __device__ __forceinline__ void start(int tiles) {
    rest = tiles / 2;
    next = rest;
    left = 3;
    __builtin_amdgcn_s_setprio(3);
  }
  __device__ __forceinline__ void at(int tile) {
    if (tile < next || left == 0) return;  // uniform
    if (left == 3) __builtin_amdgcn_s_setprio(2);
    if (left == 2) __builtin_amdgcn_s_setprio(1);
    if (left == 1) __builtin_amdgcn_s_setprio(0);
    --left;
    rest /= 2;
    next += rest;
  }
};

// A segment: tiles [t_from, t_to) of an item; its rows' outputs, or where the
// segment is a piece of the item, slot `slot_of_part` of the partial ones.  Every wave
// takes tiles of its own for all of the item's rows.
template <int DP, int MT, bool kExact, bool kView>
__device__ __forceinline__ void fp4_segment(Fp4Smem<DP, false>& sm, const Fp4Args<kView>& a, int b, int rb, int hk, const Fp4Span& sp,
                                            int t_from, int t_to, int slot_of_part, Fp4Pace& pace, int done) {
  using Wave = Fp4Wave<DP, MT, kExact, false, kView>;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x) / kWave, lane = fp4_fresh_tid() % kWave;
  const int r0 = rb * 16 * MT;
  const int t_lo = fp4_tile_base<kView>(sp) + t_from, t_hi = fp4_tile_base<kView>(sp) + min(t_to, sp.tiles);
  Wave w(a, sp, b, hk, r0, lane, reinterpret_cast<uint32_t*>(sm.tile));
  uint16_t* vt = reinterpret_cast<uint16_t*>(sm.tile[wave]);
  // this wave's tiles t_lo + wave, + 4, ...; the places of 32 of them at a time
  uint64_t at = 0;
  int slot = -1;
  const int n = t_hi > t_lo + wave ? (t_hi - t_lo - wave + kF4Waves - 1) / kF4Waves : 0;
  const auto fetch = [&](typename Wave::Raw& raw, int i) {
    // past the last tile something mapped is read, so that the loads in flight are the
    // same number whatever the path: a wait for a tile's then leaves the next one's alone
    if ((i & 31) == 0 && i < n) {  // lane 2 j + h: half h of tile i + j
      const int t = t_lo + wave + (i + (lane >> 1)) * kF4Waves;
      w.lookup(b, fp4_tile<kView>(sp, min(t, t_hi)) * kF4Tile + 16 * (lane & 1), at, slot);
    }
    w.template fetch<true, true>(raw, at, slot, 2 * (i & 31));
  };
  // the tile's registers take the next tile (of two in flight, the one after) as soon
  // as its scores are made
  constexpr int kAhead = Wave::kTwo ? 2 : 1;
  const auto step = [&](typename Wave::Raw& raw, int i) {
    const int pos = fp4_tile<kView>(sp, t_lo + wave + i * kF4Waves) * kF4Tile;
    w.template unpack_scales<true, true>(raw);
    Fp4Tile<MT> tl;
    tl.slot[0] = raw.slot[0];
    tl.slot[1] = raw.slot[1];
    tl.masked = w.uneven(raw.slot, pos) || w.any_nan(raw);
    tl.nan_keys = 0;
    if (tl.masked) tl.nan_keys = w.clean(raw, pos);  // uniform
    w.scores(raw, tl);
    w.values(raw, vt);
    fetch(raw, i + kAhead);
    w.output(tl, pos, vt);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  };
  typename Wave::Raw raw0;
  fetch(raw0, 0);
  if constexpr (Wave::kTwo) {
    typename Wave::Raw raw1;
    fetch(raw1, 1);
    int i = 0;
    for (; i + 1 < n; i += 2) {
      pace.at(done + i * kF4Waves);
      step(raw0, i);
      step(raw1, i + 1);
    }
    if (i < n) step(raw0, i);
  } else {
    for (int i = 0; i < n; ++i) {
      pace.at(done + i * kF4Waves);
      step(raw0, i);
    }
  }
  w.drop_blind();
  // join the waves: maxima and sums of every row, then the outputs, a row tile at a time
  const int tid = fp4_fresh_tid(), col = tid & 15, grp = (tid >> 4) & 3;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const float l = fp4_sum_groups(w.l[mt]);
    if (grp == 0) {
      sm.m[wave][16 * mt + col] = w.m[mt];
      sm.l[wave][16 * mt + col] = l;
    }
  }
  const float ninf = -__builtin_huge_valf();
  const bool whole = slot_of_part < 0;
  const int D = kExact ? DP : a.D;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    __syncthreads();  // the tiles (or the last row tile's outputs) have been read, the maxima are written
    f32x4* o = reinterpret_cast<f32x4*>(sm.tile[wave]);
#pragma unroll
    for (int x = 0; x < Wave::kBlocks; ++x) o[col * (DP / 4) + ((4 * x + grp) ^ (col & 7))] = w.acc[mt][x];
    __syncthreads();
    for (int i = tid; i < 16 * (DP / 4); i += kF4Threads) {
      const int row = i / (DP / 4), c = i % (DP / 4), r = r0 + 16 * mt + row;
      const int d = 4 * c;
      if (r >= sp.r_end || (!kExact && d >= D)) continue;
      const int t = r / a.G, h = hk * a.G + r - t * a.G;
      float top = kF4None;
#pragma unroll
      for (int k = 0; k < kF4Waves; ++k) top = fmaxf(top, sm.m[k][16 * mt + row]);
      const float sink = whole && a.sink ? a.sink[h] * kF4Log2e : ninf;
      const float ref = fmaxf(top, sink) == kF4None ? 0.f : fmaxf(top, sink);
      float den = 0.f;
      f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kF4Waves; ++k) {
        const float f = __builtin_amdgcn_exp2f(sm.m[k][16 * mt + row] - ref);
        const float lk = sm.l[k][16 * mt + row];
        den += lk != lk ? lk : f == 0.f ? 0.f : f * lk;  // NaN keys alone leave no maximum
        v += reinterpret_cast<const f32x4*>(sm.tile[k])[row * (DP / 4) + (c ^ (row & 7))] * f;
      }
      if (whole) {
        if (sink != ninf) den += __builtin_amdgcn_exp2f(sink - ref);
        const float inv = den == 0.f ? 0.f : 1.f / den;
        u32x2 y;
        y[0] = bf16_pack2(v[0] * inv, v[1] * inv);
        y[1] = bf16_pack2(v[2] * inv, v[3] * inv);
        *reinterpret_cast<u32x2*>(a.out + ((static_cast<int64_t>(b) * a.T + t) * a.H + h) * D + d) = y;
      } else {
        const int64_t pr = static_cast<int64_t>(slot_of_part) * (16 * MT) + 16 * mt + row;
        float* part = a.part + pr * (D + 4);
        if (c == 0) {
          part[0] = top;
          part[1] = den;
        }
        reinterpret_cast<f32x4*>(part + 4)[c] = v;
      }
    }
  }
}

// A wave's part of a cut item of shared tiles: its rows' maxima and sums, then 16 dims of 16 rows at a time, so
// that a store of the wave is one run of 1 KB.
struct Fp4Part {
  float* base;
  int rows, blocks;
  __device__ __forceinline__ float* m(int row) const { return base + row; }
  __device__ __forceinline__ float* l(int row) const { return base + rows + row; }
  __device__ __forceinline__ f32x4* quad(int row, int d) const {
    return reinterpret_cast<f32x4*>(base + 2 * rows) + (((row >> 4) * blocks + (d >> 2)) * 16 + (row & 15)) * 4 + (d & 3);
  }
};

// The tiles [t_lo, t_hi) that the waves share, in rounds of four: a wave brings one of them to LDS, its
// values decoded, its keys as they are, these a round earlier, so that a tile's scores are made beside the weights
// of the one before, over a round's end too.  (2 prompts' 1000 tokens over 16k, 32 heads on 8 of 128: 512 us, 556 with
// every wave loading all keys itself and a tile's scores ahead of its own weights.)
template <int DP, int MT, bool kExact, bool kView>
__device__ __forceinline__ void fp4_rounds_ahead(Fp4Smem<DP, true>& sm, Fp4Wave<DP, MT, kExact, true, kView>& w, const Fp4Span& sp, int b,
                                           int wave, int lane, int t_lo, int t_hi, Fp4Pace& pace, int done) {
  using Wave = Fp4Wave<DP, MT, kExact, true, kView>;
  const int n = t_hi - t_lo;
  // lane 2 j + h, j < 4: half h of tile i + j (past the last something mapped)
  const auto places = [&](int i, uint64_t& at, int& slot) {
    w.lookup(b, fp4_tile<kView>(sp, min(t_lo + i + ((lane >> 1) & 3), t_hi)) * kF4Tile + 16 * (lane & 1), at, slot);
  };
  // A round is four tiles: a wave brings one of them to LDS, its values decoded, its keys a round earlier, so that
  // the first scores of a round are made in the one before.
  typename Wave::Raw keys, vals, now;
  uint64_t at[2];  // of the next round and the one after
  int slot, slot_next[2];
  places(0, at[0], slot);
  w.template fetch<true, false>(keys, at[0], slot, 2 * wave);
  w.template fetch<false, true>(vals, at[0], slot, 2 * wave);
  places(kF4Waves, at[0], slot_next[0]);
  places(2 * kF4Waves, at[1], slot_next[1]);
  w.template unpack_scales<true, false>(keys);
  w.keep_keys(keys, sm.keys[0][wave], lane);
  w.template fetch<true, false>(keys, at[0], slot_next[0], 2 * wave);
  lds_barrier();
  Fp4Tile<MT> tl;
  w.take_keys(now, sm.keys[0][0], lane);
  w.scores(now, tl);
  float mult = 0.f;
  // a tile's masks, and its scores under them
  const auto settle = [&](int i, int j) {
    const int pos = fp4_tile<kView>(sp, t_lo + i + j) * kF4Tile;
    tl.slot[0] = __builtin_amdgcn_readlane(slot, 2 * j);
    tl.slot[1] = __builtin_amdgcn_readlane(slot, 2 * j + 1);
    tl.nan_keys = __builtin_amdgcn_readfirstlane(sm.nan_keys[j]);
    tl.masked = w.uneven(tl.slot, pos) || tl.nan_keys != 0;
    mult = w.settle(tl, pos);
  };
  for (int i = 0; i < n; i += kF4Waves) {
    pace.at(done + i);
    const int buf = (i / kF4Waves) & 1;
    {
      const int pos = fp4_tile<kView>(sp, t_lo + i + wave) * kF4Tile;
      w.template unpack_scales<false, true>(vals);
      uint32_t nan_keys = 0;
      if (w.uneven(vals.slot, pos) || w.any_nan(vals)) nan_keys = w.clean(vals, pos);  // uniform
      w.values(vals, reinterpret_cast<uint16_t*>(sm.tile[wave]));
      if (lane == 0) sm.nan_keys[wave] = nan_keys;
      w.template unpack_scales<true, false>(keys);
      w.keep_keys(keys, sm.keys[buf ^ 1][wave], lane);
    }
    w.template fetch<false, true>(vals, at[0], slot_next[0], 2 * wave);
    w.template fetch<true, false>(keys, at[1], slot_next[1], 2 * wave);
    lds_barrier();  // the tiles are there
    settle(i, 0);
#pragma unroll
    for (int j = 0; j < kF4Waves; ++j) {
      if (i + j < n) {  // uniform
        // the next tile's scores beside this one's weights
        typename Wave::Weights p;
        Fp4Tile<MT> next;
        w.take_keys(now, j < kF4Waves - 1 ? sm.keys[buf][j + 1] : sm.keys[buf ^ 1][0], lane);
        w.scores(now, next);
        w.weigh(tl, mult, p);
        w.product(p, reinterpret_cast<const uint16_t*>(sm.tile[j]));
        tl = next;
        if (j < kF4Waves - 1 && i + j + 1 < n) settle(i, j + 1);
      }
    }
    slot = slot_next[0];
    at[0] = at[1];
    slot_next[0] = slot_next[1];
    places(i + 3 * kF4Waves, at[1], slot_next[1]);
    lds_barrier();  // the tiles have been read
  }
}

// The same where LDS has no room for keys beside two workgroups' values (heads of 256 dims; one workgroup with it: 764 us
// become 1060 for 2 prompts of 16 heads on 4).
template <int DP, int MT, bool kExact, bool kView>
__device__ __forceinline__ void fp4_rounds(Fp4Smem<DP, true>& sm, Fp4Wave<DP, MT, kExact, true, kView>& w, const Fp4Span& sp, int b,
                                           int wave, int lane, int t_lo, int t_hi, Fp4Pace& pace, int done) {
  using Wave = Fp4Wave<DP, MT, kExact, true, kView>;
  const int n = t_hi - t_lo;
  // lane 2 j + h, j < 4: half h of tile i + j (past the last something mapped)
  const auto places = [&](int i, uint64_t& at, int& slot) {
    w.lookup(b, fp4_tile<kView>(sp, min(t_lo + i + ((lane >> 1) & 3), t_hi)) * kF4Tile + 16 * (lane & 1), at, slot);
  };
  typename Wave::Raw keys[2], vals;
  uint64_t at, at_next;
  int slot, slot_next;
  places(0, at, slot);
  w.template fetch<false, true>(vals, at, slot, 2 * wave);
  w.template fetch<true, false>(keys[0], at, slot, 0);
  for (int i = 0; i < n; i += kF4Waves) {
    pace.at(done + i);
    {
      const int pos = fp4_tile<kView>(sp, t_lo + i + wave) * kF4Tile;
      w.template unpack_scales<false, true>(vals);
      uint32_t nan_keys = 0;
      if (w.uneven(vals.slot, pos) || w.any_nan(vals)) nan_keys = w.clean(vals, pos);  // uniform
      w.values(vals, reinterpret_cast<uint16_t*>(sm.tile[wave]));
      if (lane == 0) sm.nan_keys[wave] = nan_keys;
    }
    places(i + kF4Waves, at_next, slot_next);
    lds_barrier();  // the tiles are there
#pragma unroll
    for (int j = 0; j < kF4Waves; ++j) {
      typename Wave::Raw &kr = keys[j & 1], &next = keys[(j + 1) & 1];
      if (j < kF4Waves - 1) {
        w.template fetch<true, false>(next, at, slot, 2 * (j + 1));
      } else {
        w.template fetch<true, false>(next, at_next, slot_next, 0);
      }
      if (j == 1) w.template fetch<false, true>(vals, at_next, slot_next, 2 * wave);
      const int pos = fp4_tile<kView>(sp, t_lo + i + j) * kF4Tile;
      Fp4Tile<MT> tl;
      tl.slot[0] = kr.slot[0];
      tl.slot[1] = kr.slot[1];
      tl.nan_keys = __builtin_amdgcn_readfirstlane(sm.nan_keys[j]);
      tl.masked = w.uneven(kr.slot, pos) || tl.nan_keys != 0;
      w.template unpack_scales<true, false>(kr);
      w.scores(kr, tl);
      if (i + j < n) w.output(tl, pos, reinterpret_cast<const uint16_t*>(sm.tile[j]));  // uniform
    }
    at = at_next;
    slot = slot_next;
    lds_barrier();  // the tiles have been read
  }
}

// The same with every wave loading all keys itself (heads of 512 dims: one workgroup on a compute unit, whose LDS the
// values fill).  A tile's keys take their registers from the ones before once these have been multiplied.  (6 trees of 99 nodes,
// 16 heads on one, in windows of 128: 46 us a call, 53 with tiles of each wave's own; 9 trees of 401 nodes, 8 heads on one,
// over 4k: 632 and 799.  A tile's scores ahead of its own weights, both without the weights' rests: 54 us for 43, 661 for 585.
// Two waves on a SIMD hide more of each other's waits without it: 2 prompts of 16 heads on 4 of 256 dims 835 us with it and 754.)
template <int DP, int MT, bool kExact, bool kView>
__device__ __forceinline__ void fp4_rounds_wide(Fp4Smem<DP, true>& sm, Fp4Wave<DP, MT, kExact, true, kView>& w, const Fp4Span& sp, int b,
                                           int wave, int lane, int t_lo, int t_hi, Fp4Pace& pace, int done) {
  using Wave = Fp4Wave<DP, MT, kExact, true, kView>;
  const int n = t_hi - t_lo;
  // lane 2 j + h, j < 4: half h of tile i + j (past the last something mapped)
  const auto places = [&](int i, uint64_t& at, int& slot) {
    w.lookup(b, fp4_tile<kView>(sp, min(t_lo + i + ((lane >> 1) & 3), t_hi)) * kF4Tile + 16 * (lane & 1), at, slot);
  };
  typename Wave::Raw keys, vals;
  uint64_t at, at_next;
  int slot, slot_next;
  places(0, at, slot);
  w.template fetch<true, false>(keys, at, slot, 0);
  w.template fetch<false, true>(vals, at, slot, 2 * wave);
  places(kF4Waves, at_next, slot_next);
  Fp4Tile<MT> tl;
  w.scores(keys, tl);
  w.template fetch<true, false>(keys, at, slot, 2);
  float mult = 0.f;
  // a tile's masks, and its scores under them
  const auto settle = [&](int i, int j) {
    const int pos = fp4_tile<kView>(sp, t_lo + i + j) * kF4Tile;
    tl.slot[0] = __builtin_amdgcn_readlane(slot, 2 * j);
    tl.slot[1] = __builtin_amdgcn_readlane(slot, 2 * j + 1);
    tl.nan_keys = __builtin_amdgcn_readfirstlane(sm.nan_keys[j]);
    tl.masked = w.uneven(tl.slot, pos) || tl.nan_keys != 0;
    mult = w.settle(tl, pos);
  };
  for (int i = 0; i < n; i += kF4Waves) {
    pace.at(done + i);
    {
      const int pos = fp4_tile<kView>(sp, t_lo + i + wave) * kF4Tile;
      w.template unpack_scales<false, true>(vals);
      uint32_t nan_keys = 0;
      if (w.uneven(vals.slot, pos) || w.any_nan(vals)) nan_keys = w.clean(vals, pos);  // uniform
      w.values(vals, reinterpret_cast<uint16_t*>(sm.tile[wave]));
      if (lane == 0) sm.nan_keys[wave] = nan_keys;
    }
    lds_barrier();  // the tiles are there
    settle(i, 0);
#pragma unroll
    for (int j = 0; j < kF4Waves; ++j) {
      if (i + j < n) {  // uniform
        // the next tile's scores beside this one's weights, the keys of the one after on their way
        typename Wave::Weights p;
        Fp4Tile<MT> next;
        w.scores(keys, next);
        if (j < kF4Waves - 2) {
          w.template fetch<true, false>(keys, at, slot, 2 * (j + 2));
        } else {
          w.template fetch<true, false>(keys, at_next, slot_next, 2 * (j + 2 - kF4Waves));
        }
        if (j == 1) w.template fetch<false, true>(vals, at_next, slot_next, 2 * wave);
        w.weigh(tl, mult, p);
        w.product(p, reinterpret_cast<const uint16_t*>(sm.tile[j]));
        tl = next;
        if (j < kF4Waves - 1 && i + j + 1 < n) settle(i, j + 1);
      }
    }
    at = at_next;
    slot = slot_next;
    places(i + 2 * kF4Waves, at_next, slot_next);
    lds_barrier();  // the tiles have been read
  }
}

// The same with tiles that the waves share: each has 16 MT of the item's rows and
// decodes one in four tiles' values for all of them.
template <int DP, int MT, bool kExact, bool kView>
__device__ __forceinline__ void fp4_segment_shared(Fp4Smem<DP, true>& sm, const Fp4Args<kView>& a, int b, int rb, int hk, const Fp4Span& sp,
                                                   int t_from, int t_to, int slot_of_part, Fp4Pace& pace, int done) {
  using Wave = Fp4Wave<DP, MT, kExact, true, kView>;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x) / kWave, lane = fp4_fresh_tid() % kWave;
  const int r0 = (rb * kF4Waves + wave) * 16 * MT;
  const int t_lo = fp4_tile_base<kView>(sp) + t_from, t_hi = fp4_tile_base<kView>(sp) + min(t_to, sp.tiles);
  Wave w(a, sp, b, hk, r0, lane);
  if constexpr (Fp4Smem<DP, true>::kKeys) {
    fp4_rounds_ahead(sm, w, sp, b, wave, lane, t_lo, t_hi, pace, done);
  } else if constexpr (DP > 256) {
    fp4_rounds_wide(sm, w, sp, b, wave, lane, t_lo, t_hi, pace, done);
  } else {
    fp4_rounds(sm, w, sp, b, wave, lane, t_lo, t_hi, pace, done);
  }
  w.drop_blind();
  const int tid = fp4_fresh_tid(), col = tid & 15, grp = (tid >> 4) & 3;
  const float ninf = -__builtin_huge_valf();
  const bool whole = slot_of_part < 0;
  const int D = kExact ? DP : a.D;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const float l = fp4_sum_groups(w.l[mt]);
    const int r = r0 + 16 * mt + col;
    if (r >= sp.r_end) continue;
    const int t = r / a.G, h = hk * a.G + r - t * a.G;
    if (whole) {
      const float sink = a.sink ? a.sink[h] * kF4Log2e : ninf;
      const float ref = fmaxf(w.m[mt], sink) == kF4None ? 0.f : fmaxf(w.m[mt], sink);
      const float f = __builtin_amdgcn_exp2f(w.m[mt] - ref);
      float den = l != l ? l : f == 0.f ? 0.f : f * l;
      if (sink != ninf) den += __builtin_amdgcn_exp2f(sink - ref);
      const float inv = den == 0.f ? 0.f : f / den;
      uint16_t* out = a.out + ((static_cast<int64_t>(b) * a.T + t) * a.H + h) * D;
#pragma unroll
      for (int x = 0; x < Wave::kBlocks; ++x) {
        const int d = 16 * x + 4 * grp;
        if (!kExact && d >= D) continue;
        const f32x4 v = w.acc[mt][x] * inv;
        *reinterpret_cast<u32x2*>(out + d) = u32x2{bf16_pack2(v[0], v[1]), bf16_pack2(v[2], v[3])};
      }
    } else {
      const Fp4Part part{a.part + (static_cast<int64_t>(slot_of_part) * kF4Waves + wave) * (16 * MT) * (D + 4), 16 * MT, D / 16};
      if (grp == 0) {
        *part.m(16 * mt + col) = w.m[mt];
        *part.l(16 * mt + col) = l;
      }
#pragma unroll
      for (int x = 0; x < Wave::kBlocks; ++x) {
        if (kExact || 16 * x < D) *part.quad(16 * mt + col, 4 * x + grp) = w.acc[mt][x];
      }
    }
  }
}

template <int DP, int MT, bool kExact, bool kShared, bool kView>
__global__ __launch_bounds__(kF4Threads, fp4_resident(DP, MT)) void k_fp4_attn(Fp4Args<kView> a) {
  constexpr int kRows = 16 * MT * (kShared ? kF4Waves : 1);
  __shared__ Fp4Smem<DP, kShared> sm;
  const int tid = threadIdx.x;
  const int items = a.B * a.row_blocks;
  const auto span_of = [&](int item, int& b, int& rb) {
    b = item / a.row_blocks;
    rb = item - b * a.row_blocks;
    return fp4_span(a, b, rb * kRows, kRows);
  };
  // values worked out in LDS are the same in every lane: scalar registers hold them
  const auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  const bool each = a.max_groups == 0;  // none is cut, a workgroup each
  const int g = blockIdx.x;
  int x = g, end = g + 1, total = 0, b, rb;
  // with a view: the piece of an item that a workgroup has where it has one alone
  bool alone = false;
  int own_item = 0, own_head = 0, own_piece = 0, own_pieces = 1;
  const auto item_of = [&](int u) {  // u < total: pre[item] <= u < pre[item + 1]; the wave looks in 64 places at a time
    const int lane = tid % kWave, step = (items + kWave - 1) / kWave;
    const auto last_of = [&](int first, int by, int n) {  // of pre[first + by i] <= u, i < n
      const int at = first + by * lane;
      return first + by * (__popcll(__ballot(lane < n && at < items && sm.pre[at] <= u)) - 1);
    };
    const int from = last_of(0, step, kWave);
    return step == 1 ? from : last_of(from, 1, step);
  };
  if (!each) {
    if (tid == 0) sm.longest = 0;
    __syncthreads();
    int longest = 0;
    for (int base = 0; base < items; base += kF4Threads) {
      const int item = base + tid;
      const int own = item < items ? span_of(item, b, rb).units() + a.lead : 0, n = own * a.Hkv;
      longest = max(longest, own);
      int tot;
      const int ex = block_exclusive_scan(n, sm.scan, &tot);
      if (item < items) sm.pre[item] = total + ex;
      total += tot;
    }
    if (tid == 0) sm.pre[items] = total;
    if (longest > 0) atomicMax(&sm.longest, longest);
    __syncthreads();
    total = uniform(total);
    int groups = fp4_groups(a, total);
    const int units = items * a.Hkv;
    // The workgroups that the chip's time is counted in: as many as run; with a view, whose items are often of one
    // length, and two or more for each compute unit, which keep the memory busy, as many as the items put there (64
    // windows of 4k, 64 heads on 8 of 128: 59 us uncut with 512 of the 768 workgroups that fit, 69 cut for all; of 64 dims 42
    // and 48, before the plan itself left such windows whole).
    int slots = groups;
    if constexpr (kView) {
      const int cus = a.max_groups / fp4_resident(DP, MT);
      if (units >= 2 * cus) slots = (units + cus - 1) / cus * cus;
    }
    const bool whole = a.small == kF4SmallTiles && units <= groups &&
                       static_cast<int64_t>(uniform(sm.longest)) * slots * (kF4Idle - 1) <= static_cast<int64_t>(total) * kF4Idle;
    // With a view and fewer items than half of the workgroups, an item is cut into pieces of its own instead, one to a
    // workgroup: a run over an item's end would pay for a segment's start and end twice (5 trees of 25 nodes, 8 heads on 1 of
    // 512, over 1.2k tokens: 35 us for 85; 20 of 8 nodes, 16 on 4 of 32, over 2.2k: 31 for 44).
    if constexpr (kView) alone = a.lead == 0 && a.small == kF4SmallTiles && !whole;  // uniform
    if (alone) {
      // of about run tiles, no more pieces than workgroups: sum ceil(n / run) <= total / run + units
      const int room = max(a.max_groups - units, 1), run = max((total + room - 1) / room, kF4RunTiles);
      total = 0;
      for (int base = 0; base < items; base += kF4Threads) {
        const int item = base + tid;
        const int n = item < items ? (sm.pre[item + 1] - sm.pre[item]) / a.Hkv : 0;
        __syncthreads();  // before they are written over
        int tot;
        const int ex = block_exclusive_scan((n + run - 1) / run * a.Hkv, sm.scan, &tot);
        if (item < items) sm.pre[item] = total + ex;
        total += tot;
      }
      if (tid == 0) sm.pre[items] = total;
      __syncthreads();
      total = uniform(total);
      groups = total;
    }
    if (g == 0) {
      for (int i = tid; i <= items; i += kF4Threads) a.sched[i] = sm.pre[i];
      if (tid == 0) a.sched[items + 1] = whole ? INT32_MAX : alone ? -1 : a.small;
    }
    if (whole) groups = units;
    if (g >= groups) return;  // uniform
    if (alone) {
      own_item = uniform(item_of(g));
      own_pieces = uniform((sm.pre[own_item + 1] - sm.pre[own_item]) / a.Hkv);
      const int in = g - uniform(sm.pre[own_item]);
      own_head = in / own_pieces;
      own_piece = in - own_head * own_pieces;
    }
    // a run's end inside a small item moves to one of the item's
    const auto run_start = [&](int i) {
      if (whole) return i == units ? total : sm.pre[i / a.Hkv] + i % a.Hkv * ((sm.pre[i / a.Hkv + 1] - sm.pre[i / a.Hkv]) / a.Hkv);
      const int u = fp4_run_start(i, total, groups);
      if (u <= 0 || u >= total) return u;
      const int item = item_of(u), n = (sm.pre[item + 1] - sm.pre[item]) / a.Hkv;
      const int over = (u - sm.pre[item]) % n;
      if (n - a.lead <= a.small) return 2 * over < n ? u - over : u - over + n;
      return over <= fp4_early(a) ? u - over : u;
    };
    if (alone) {
      const int n = span_of(own_item, b, rb).units();
      x = n * own_piece / own_pieces;
      end = n * (own_piece + 1) / own_pieces;
    } else {
      x = uniform(run_start(g));
      end = uniform(run_start(g + 1));
    }
  }
  Fp4Pace pace{0, 0, 0};
  if (!each) pace.start(end - x);  // in a grid of more than the device holds the oldest may go first
  const int x0 = x;
  while (x < end) {
    const int item = each ? x / a.Hkv : alone ? own_item : uniform(item_of(x));
    const Fp4Span sp = span_of(item, b, rb);
    const int lead = each ? 0 : a.lead, n = sp.units() + lead;
    const int in = each || alone ? 0 : x - uniform(sm.pre[item]);
    const int hk = each ? x - item * a.Hkv : alone ? own_head : in / n;
    const int x1 = each ? 0 : alone ? x : in - hk * n, x2 = each ? n : min(n, x1 + end - x);
    const int from = max(x1 - lead, 0), to = x2 - lead;
    const int part = x1 == 0 && x2 == n ? -1 : x1 == 0 ? 2 * g + 1 : 2 * g;
    if constexpr (kShared) {
      fp4_segment_shared<DP, MT, kExact, kView>(sm, a, b, rb, hk, sp, from, to, part, pace, x - x0);
    } else {
      fp4_segment<DP, MT, kExact, kView>(sm, a, b, rb, hk, sp, from, to, part, pace, x - x0);
    }
    x += each ? 1 : x2 - x1;
    __syncthreads();  // the segment's LDS has been read
  }
}

constexpr int kF4MaxNodes = 1024;
// What cutting and joining costs in the tiles of a workgroup's own time, of heads up to 128 dims on tiles of each wave's
// own and of others; and the longest items (in tiles) that a window leaves whole for it (see fp4_attn_plan).
constexpr int kF4JoinTiles = 48, kF4JoinTilesWide = 24, kF4UncutTiles = 160;

struct Fp4AttnPlan {
  int dims, mt;  // padded dims, row tiles of a wave
  bool shared;   // the waves share the tiles, each with rows of its own
  int rows;      // of a workgroup
  int64_t row_blocks, items;
  bool cut;        // items may be cut
  int64_t groups;  // then: the most workgroups
  int64_t sched_bytes, ws_bytes;
};

inline int fp4_check_view(const skv_fp4_attention_desc* d, const skv_fp4_view* v) {
  const char* what = "skv_fp4_attention";
  if (v->first < 0 || v->first > (1 << 24)) return set_error(SKV_EINVAL, "%s: first must be in [0, 2^24]", what);
  if (v->tree && (d->n_queries > kF4MaxNodes || v->tree_words != ceil_div(d->n_queries, 64))) {
    return set_error(SKV_EINVAL, "%s: a tree has at most %d nodes and a word for every 64; got %lld nodes and %lld words", what,
                     kF4MaxNodes, (long long)d->n_queries, (long long)v->tree_words);
  }
  if (reinterpret_cast<uintptr_t>(v->tree) & 7) return set_error(SKV_EINVAL, "%s: tree must be 8-byte aligned", what);
  return SKV_OK;
}

inline int fp4_attn_plan(const skv_fp4_attention_desc* d, const skv_fp4_view* v, Fp4AttnPlan& p) {
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
  const float scale = d->scale > 0.f ? d->scale : 1.f / sqrtf(static_cast<float>(d->cache.head_dim));
  if (!std::isfinite(scale * kF4Log2e) || !std::isfinite(d->softcap * kF4Log2e) ||
      (d->softcap > 0.f && !std::isfinite(2.f * kF4Log2e * scale / d->softcap))) {
    return set_error(SKV_EINVAL, "%s: scale, softcap and scale / softcap must leave fp32 room for a factor of 3", what);
  }
  const int64_t D = d->cache.head_dim, rows = d->n_queries * (d->n_heads / hkv);
  p.dims = D <= 64 ? 64 : D <= 128 ? 128 : D <= 256 ? 256 : 512;
  // A wave's tiles are its own, or all four waves' with rows of their own for each, once
  // more than half of the rows of such a workgroup are there: 16 sequences of 32k on one
  // head of 128 dims take 56 us shared and 48 apart with 64 rows, 56 and 71 with 65 (another row
  // block), 53 and 36 with 32; of 64 dims 44 and 42 with 64 rows, 45 either way with 65, 49 and 60 with
  // 128; of 256 dims 68 and 65 with 32 rows, 68 and 101 with 33.  Heads of up to 512 dims stay apart, but with a view
  // those of 512 where a sixteenth of the compute units get such a workgroup, as a cut into more pieces is more to join (us
  // shared and apart: 300 windows of 128, 33 rows 58 and 70, 64 rows 64 and 91; 16 of 4k 50 and 46, 53 and 59; 8 windows of 9k, 64
  // rows 55 and 57; one of 100k 94 and 68).  The sizes between spill registers (40 trees of 9 nodes, 32 heads on 2 of 288 dims,
  // over 8k: 720, without the weights' rests, and 650).
  const int mt = fp4_shared_mt(p.dims);
  p.shared = rows > 16 * mt * kF4Waves / 2 &&
             (p.dims <= 256 || (v && D == 512 && 16 * d->cache.batch * hkv * ceil_div(rows, 16 * mt * kF4Waves) >= device_cus()));
  if (v) {
    if (const int rc = fp4_check_view(d, v)) return rc;
  }
  p.mt = p.shared ? mt : rows <= 16 || p.dims > 256 ? 1 : 2;
  // the most tiles that a block of so many rows may see
  const int64_t capacity = d->cache.bt_stride * d->cache.block_size;
  const auto tiles_of = [&](int64_t block_rows) {
    int64_t len = d->max_len > 0 ? std::min(d->max_len, capacity) : capacity;
    if (d->window > 0) {
      // the rows' tokens see a window and as many more as they are (in a tree: as there are nodes), and the first ones
      const int64_t tokens = v && v->tree ? d->n_queries : ceil_div(block_rows, d->n_heads / hkv);
      len = std::min(len, d->window + tokens + (v && v->first > 0 ? v->first + kF4Tile : 0));
    }
    return ceil_div(len, kF4Tile) + 1;
  };
  // With a view, few tiles and few rows: a workgroup's latency is the call's, and blocks of 16 rows have the shortest, as
  // long as the device holds them all at once (trees of 8 nodes, 16 heads on 2 of 128, over 400 tokens: 11.0 us for 14.6 with
  // 1 sequence, 14.8 for 15.9 with 64; 32 nodes, 64 heads on 8: 11.2 for 22.1 with 1, 13.8 for 22.5 with 4, but 38.3 for
  // 24.8 with 16, which are 2,048 blocks).
  if (v && d->splits == 0 && tiles_of(16) <= kF4SmallTiles &&
      d->cache.batch * ceil_div(rows, 16) * hkv <= static_cast<int64_t>(fp4_resident(p.dims, 1)) * device_cus()) {
    p.shared = false;
    p.mt = 1;
  }
  p.rows = 16 * p.mt * (p.shared ? kF4Waves : 1);
  p.row_blocks = ceil_div(rows, p.rows);
  p.items = d->cache.batch * p.row_blocks;
  const int64_t tiles = tiles_of(p.rows), units = std::max<int64_t>(p.items * hkv, 1);
  p.cut = tiles > kF4SmallTiles || d->splits > 0;
  if (p.items > kF4MaxItems || units > INT32_MAX / (ceil_div(capacity, kF4Tile) + 1 + kF4Lead)) p.cut = false;
  // With a view, the items of a window are at most a few tiles long.  They stay whole, a workgroup each, dealt out as others
  // end, where the workgroups that the last round leaves idle lose less than runs, parts and the join cost (us whole and
  // cut, sequences far longer than the window and, second, of anything from 64 tokens to two windows; 64 heads on 8 of 128,
  // windows of 1k, one token: 64 of them 20 and 25, 20 and 34; 16 of them 14.5 and 22, 15 and 20; chunks of 1000 tokens, 32 heads:
  // one 42 and 57, three 86 and 110, of windows of 2k two 90 and 93; 90 windows of 4k 74 and 79, 63 and 74).  Past these numbers
  // they lose (a chunk of 500 tokens in windows of 2k: 66 and 51; 64 tokens of 16 heads on 1 of 512, windows of 1k: 40 and 34;
  // windows of 8k, 220 of 4 tokens, 16 heads on 4 of 64: 110 and 120, but 102 and 98).
  if (v && p.cut && d->window > 0 && d->splits == 0 && tiles <= kF4UncutTiles) {
    const int64_t slots = static_cast<int64_t>(fp4_resident(p.dims, p.mt)) * device_cus();
    const int64_t idle = ceil_div(units, slots) * slots - units;
    if (idle * tiles <= (p.shared || p.dims > 128 ? kF4JoinTilesWide : kF4JoinTiles) * slots) p.cut = false;
  }
  if (units >= (1 << 24)) return set_error(SKV_EINVAL, "%s: too many workgroups", what);
  if (p.cut && d->splits > ((1 << 24) - 1) / units) {  // before it is multiplied: the product could wrap
    return set_error(SKV_EINVAL, "%s: splits must leave fewer than 2^24 runs; got %lld of %lld rows and heads", what,
                     (long long)d->splits, (long long)units);
  }
  p.groups = !p.cut ? 0 : d->splits > 0 ? d->splits * units : static_cast<int64_t>(fp4_resident(p.dims, p.mt)) * device_cus();
  p.sched_bytes = p.cut ? ceil_div((p.items + 2) * 4, 16) * 16 : 0;
  p.ws_bytes = p.cut ? p.sched_bytes + 2 * p.groups * p.rows * (D + 4) * 4 : 0;
  return SKV_OK;
}

// The part launch for padded dims DP.
template <int DP, bool kExact, bool kView>
void launch_rows(const Fp4Args<kView>& a, const Fp4AttnPlan& p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.max_groups > 0 ? a.max_groups : static_cast<int64_t>(a.B) * a.row_blocks * a.Hkv));
  const auto go = [&](auto* kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kF4Threads), 0, s, a); };
  if constexpr (DP <= 256 || (kExact && kView)) {
    if (p.shared) return go(&k_fp4_attn<DP, fp4_shared_mt(DP), kExact, true, kView>);
  }
  if constexpr (DP <= 256) {
    if (p.mt == 2) return go(&k_fp4_attn<DP, 2, kExact, false, kView>);
  }
  go(&k_fp4_attn<DP, 1, kExact, false, kView>);
}
template <bool kExact, bool kView>
void launch_dims(const Fp4Args<kView>& a, const Fp4AttnPlan& p, hipStream_t s) {
  if (p.dims == 64) launch_rows<64, kExact, kView>(a, p, s);
  if (p.dims == 128) launch_rows<128, kExact, kView>(a, p, s);
  if (p.dims == 256) launch_rows<256, kExact, kView>(a, p, s);
  if (p.dims == 512) launch_rows<512, kExact, kView>(a, p, s);
}

void fp4_attn_join(const Fp4AttnArgs& a, const Fp4AttnPlan& p, hipStream_t s);  // skv_fp4_attention.hip

template <bool kView>
int fp4_attn_call(const skv_fp4_attention_desc* d, const skv_fp4_view* v, void* workspace, int64_t ws_bytes, void* stream) {
  const char* what = "skv_fp4_attention";
  Fp4AttnPlan p;
  if (const int rc = fp4_attn_plan(d, v, p)) return rc;
  if (d->cache.batch == 0) return SKV_OK;
  if (!d->q || !d->out || !d->seq_lens) return set_error(SKV_EINVAL, "%s: NULL pointer", what);
  if ((reinterpret_cast<uintptr_t>(d->q) | reinterpret_cast<uintptr_t>(d->out) | static_cast<uintptr_t>(d->q_seq_stride) |
       static_cast<uintptr_t>(d->q_tok_stride) | static_cast<uintptr_t>(d->q_head_stride)) & 15) {
    return set_error(SKV_EINVAL, "%s: q, its strides and out must be 16-byte aligned", what);
  }
  if (p.ws_bytes > 0 && (!workspace || ws_bytes < p.ws_bytes || (reinterpret_cast<uintptr_t>(workspace) & 15))) {
    return set_error(SKV_EINVAL, "%s: a 16-byte aligned workspace of %lld bytes is needed", what, (long long)p.ws_bytes);
  }
  Fp4Args<kView> a{};
  a.q = static_cast<const uint8_t*>(d->q);
  a.q_seq = d->q_seq_stride;
  a.q_tok = d->q_tok_stride;
  a.q_head = d->q_head_stride;
  a.out = static_cast<uint16_t*>(d->out);
  a.lens = d->seq_lens;
  a.n_new = d->n_new;
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
  const float scale = d->scale > 0.f ? d->scale : 1.f / sqrtf(static_cast<float>(a.D));
  a.scale = scale * kF4Log2e;
  a.cap = d->softcap * kF4Log2e;
  a.cap_k = d->softcap > 0.f ? 2.f * kF4Log2e * scale / d->softcap : 0.f;
  a.B = static_cast<int32_t>(d->cache.batch);
  a.sched = p.cut ? static_cast<int32_t*>(workspace) : nullptr;
  a.part = p.cut ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + p.sched_bytes) : nullptr;
  a.row_blocks = static_cast<int32_t>(p.row_blocks);
  a.max_groups = static_cast<int32_t>(p.groups);
  a.small = d->splits > 0 ? 0 : kF4SmallTiles;
  a.lead = d->splits == 0 && 2 * p.items * a.Hkv >= p.groups ? kF4Lead : 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if constexpr (kView) {
    a.tree = v->tree;
    a.words = static_cast<int32_t>(v->tree_words);
    a.keep = static_cast<int32_t>(v->first);
  }
  if (a.D == p.dims) launch_dims<true, kView>(a, p, s); else launch_dims<false, kView>(a, p, s);
  if (const int rc = check_launch(what)) return rc;
  if (!p.cut) return SKV_OK;
  fp4_attn_join(a, p, s);
  return check_launch(what);
}

}  // namespace skv
