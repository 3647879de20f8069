// Attention over the pages of the 4-bit token cache (skv_fp4.h has the format).
//
//   s_j = scale * q . k_j, softcap * tanh(s_j / softcap) where asked for
//   out = sum_j exp(s_j) v_j / (sum_j exp(s_j) + exp(sink))
//
// over the positions j that the query token sees: one pass over them with the
// running maximum m and sum l of the softmax (log2 domain), the output rescaled
// by exp2(m_old - m_new) where the maximum moves.
//
// A K/V head's query rows (its query heads times the query tokens) are cut into
// blocks of 16 MT rows a wave, over tiles of 32 positions:
//   * S^T = K Q^T by the scaled products of gfx950 (v_mfma_scale_f32_16x16x128_f8f6f4),
//     which take e2m1 codes and their scale bytes as they lie in the page: lane
//     (key, g) of 16 keys reads g's quarter of its key's codes straight into the operand
//     registers, 16 bytes of 128 dims a step.  The query goes in as two e4m3 parts,
//     q = hi 2^a + lo 2^(a - 5) with 2^a by 32 dims: a bf16 value's 8 bits are 4 and 4, so
//     the parts are exact (but for values below 2^-13 of their 32's largest, which are
//     exact to 2^-23 of it).
//   * the values go through LDS as bf16, rows of D in swizzled chunks, and come back
//     transposed (ds_read_b64_tr_b16) as the A operand of O^T = V^T P^T, whose B
//     operand is P^T as the scores' accumulators hold it.  O^T keeps a row's output in
//     the lanes that hold its m and l.  The values are exact in bf16; a weight goes in as
//     a bf16 and, with few rows, its rounding's rest (see kRest).  Scores, m, l and O are
//     fp32.
// Few rows (fp4_segment): all of a workgroup's rows are every wave's, and each wave takes
// tiles of its own, with a softmax of its own, joined at the end; no wave waits for
// another on the way, and the codes of the next two tiles are in flight while one is
// multiplied.  Memory bounds it.  Many (fp4_segment_shared): the waves have rows of their
// own and share the tiles, each decoding the values of one in four; a tile is read and
// decoded once for 128 rows (64 of 256 dims).  The softmax's vector work and the matrix
// products bound it.
//
// Work: the tiles of all (sequence, row block, head) items, one after another, are
// dealt to as many workgroups as the device holds at once, in equal runs that may
// cut a long item; the lengths are on the device, so every workgroup works the
// runs out for itself from their prefix sum.  A cut item's pieces are joined by a
// second launch.  (Twice as many workgroups of half the run, for the hardware to deal out
// as others end, took 1.3 times as long for the step below.)
//
// Measured, us a call (both launches) in a graph of several, with the time of the bytes
// at 6.1 TB/s (or of the products at 1.4 PFLOP/s, an 8192^3 library product's rate):
//   64 sequences of 1k - 32k, 64 heads on 8 of 128 dims                    139 (117)
//   4 of 256k - 1M, 4 tokens, 16 heads on 4 of 64                          91 (74)
//   16 of 64k, 64 heads on 1 of 128                                        79 (25, products)
//   2 prompts' 1000 tokens over 16k, 32 heads on 8 of 128                  557 (367, products)
//   1 prompt's 512 tokens over 200k, the same heads                        1690 (1200, products)
//   32 windows of 128, 64 heads on 1 of 512                                23 (1)
// and dropped: two row groups of two waves with half the tiles each for 33 - 64 rows (68 ->
// 74 us for the 64k sequences, before their weights had rests: a tile's latency is then seen by
// all four waves); the next tile's scores ahead of a tile's weights (1%); a prologue that loads
// the queries last.
#include <algorithm>
#include <cmath>

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

// The positions that the rows [r0, r0 + n) of a K/V head see.
struct Fp4Span {
  int L, T, r_end;       // tokens of the sequence, and new ones among them; rows of the head
  int first, last;       // [first, last): some row sees them
  int all_lo, all_hi;    // [all_lo, all_hi): every row sees them
  int tile0, tiles;
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

// Workgroups that share the units: a run of fewer than 8 tiles, 2 a wave, is not
// worth a workgroup, but an item is.  Workgroup i of n takes total / n tiles,
// the first total mod n one more.
constexpr int kF4RunTiles = 8;
constexpr int kF4SmallTiles = 16;
// What a segment costs beside its tiles, in tiles: the first loads' latencies and the
// waves' join.  A step of 64 sequences of 1k - 32k, 8 K/V heads: 165 us without it, with 12 tiles
// 144 and with 20 139 us; the other cases above stay within 1%.  Counted where
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

template <int DP>
struct Fp4Smem {
  // per wave: 32 value rows of DP bf16; at the end 16 output rows of DP fp32 (private tiles)
  alignas(16) uint8_t tile[kF4Waves][64 * DP];
  float m[kF4Waves][32], l[kF4Waves][32];
  uint32_t nan_keys[kF4Waves];  // of shared tiles
  int pre[kF4MaxItems + 1];
  int scan[17];
  int longest;
};

// DP: the head's dims padded to 64, 128, 256 or 512 (kExact: D == DP).
template <int DP, int MT, bool kExact, bool kShared>
struct Fp4Wave {
  using Raw = Fp4Raw<DP>;
  static constexpr int kWords = Raw::kWords, kScales = Raw::kScales;
  static constexpr int kSteps = DP >= 128 ? DP / 128 : 1;  // products of 128 dims, or of the two parts of 64
  static constexpr int kBlocks = DP / 16;  // 16-dim blocks of the output
  static constexpr bool kPacked = kExact && DP <= 128;
  // A weight's bf16 rounding, 2^-9 of it on average over few keys as over many, is as
  // large an error as the output's own.  Waves with tiles of their own carry its rest
  // into a second product, 139 us for a step of 64 sequences and 138 without (64 rows on one
  // head 79 and 67); where the products bound the time (a prompt's chunk 557, with rests 705 us)
  // the rounded weight stands.
  static constexpr bool kRest = !kShared;
  static constexpr bool kTwo = DP * MT <= 256;  // two tiles in flight; wider ones have registers for one
  // A page is read by one workgroup, or by two: nontemporal loads (a step of 64 sequences 139 us,
  // 156 with plain ones; 4 of 256k - 1M 91 and 103; 64 rows on one head, read twice, 79 either way).
  static constexpr bool kOnce = !kShared && DP * MT <= 256;

  const Fp4AttnArgs& a;
  const Fp4Span& sp;
  const Fp4Page pg;
  int col, grp;
  const uint8_t* head;  // the K/V head's block in page 0
  uint32_t code_at, scale_at;  // the lane's place in 16 keys' codes and scale bytes
  i32x8 q[MT][kSteps][DP >= 128 ? 2 : 1];  // the two parts of the query (64 dims: both in one)
  int q_scale[MT][kSteps];                 // scale byte of k-block g: byte 0 of the first part, byte 1 of the second
  int hi[MT], lo[MT];   // the positions that row 16 mt + col sees
  float m[MT], l[MT];
  f32x4 acc[MT][kBlocks];

  __device__ __forceinline__ Fp4Wave(const Fp4AttnArgs& a_, const Fp4Span& sp_, int b, int hk, int r0, int lane)
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
      const uint8_t* row = a.q + b * a.q_seq + t * a.q_tok + (hk * a.G + g) * a.q_head;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) load_query(mt, s, row, in);
      m[mt] = kF4None;
      l[mt] = 0.f;
#pragma unroll
      for (int x = 0; x < kBlocks; ++x) acc[mt][x] = f32x4{0.f, 0.f, 0.f, 0.f};
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
  __device__ __forceinline__ void load_query(int mt, int s, const uint8_t* row, bool in) {
    const int half = 16 * (grp & 1);
    uint32_t hi[8], lo[8];
    if constexpr (DP >= 128) {
      const uint32_t b0 = split16(row, 32 * ((grp >> 1) * kScales + s) + half, in, hi, lo);
      const uint32_t b1 = split16(row, 32 * ((2 + (grp >> 1)) * kScales + s) + half, in, hi + 4, lo + 4);
      const int from = col + 32 * (grp & 1);  // k-blocks 0, 1 (2, 3) are the first (second) 16 of lanes 0 and 32
      const int a0 = __shfl(static_cast<int>(b0), from), a1 = __shfl(static_cast<int>(b1), from);
      const int own = grp < 2 ? a0 : a1;
      q_scale[mt][s] = own | (own - 5) << 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        q[mt][s][0][i] = static_cast<int>(hi[i]);
        q[mt][s][DP >= 128 ? 1 : 0][i] = static_cast<int>(lo[i]);
      }
    } else {
      // k-blocks 0, 1: the first part of dims 0 .. 63; 2, 3: the second part of the same
      const uint32_t b = split16(row, 16 * grp, in, hi, lo);
      const int own = __shfl(static_cast<int>(b), col + 32 * (grp & 1));
      q_scale[mt][s] = grp < 2 ? own : own - 5;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        q[mt][s][0][i] = static_cast<int>(hi[i]);
        q[mt][s][0][i + 4] = static_cast<int>(lo[i]);
      }
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
      if (nan || at >= sp.last || at < sp.first || r.slot[h] < 0) {
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
  __device__ __forceinline__ bool uneven(const Raw& r, int pos) const {
    return pos < sp.all_lo || pos + kF4Tile > sp.all_hi || (r.slot[0] | r.slot[1]) < 0;
  }
  __device__ __forceinline__ bool any_nan(const Raw& r) const {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kScales; ++i) nan |= r.vs[0][i] == kFp4NaN || r.vs[1][i] == kFp4NaN;
    return __ballot(nan) != 0;
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

  // 32 keys' values to LDS.
  __device__ __forceinline__ void values(const Raw& r, uint16_t* vt) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint16_t* dst = vt + (16 * h + col) * DP;
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        *reinterpret_cast<u32x4*>(dst + 8 * fp4_chunk(col, grp * kWords + w)) =
            fp4_decode8(r.v[h][w], fp4_scale(r.vs[h][w / 4 < kScales ? w / 4 : 0]));
      }
    }
  }

  // The tile's weights, and its values times them onto the output.
  __device__ __forceinline__ void output(Fp4Tile<MT>& tl, int pos, const uint16_t* vt) {
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
    u32x4 p[MT], rest[kRest ? MT : 1];
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
        p[mt][i] = bf16_pack2(e[2 * i], e[2 * i + 1]);
        if constexpr (kRest) {
          rest[mt][i] = bf16_pack2(e[2 * i] - __uint_as_float(p[mt][i] << 16), e[2 * i + 1] - __uint_as_float(p[mt][i] & 0xffff0000u));
        }
      }
    }
    // O^T += V^T P^T: dims 16 x + 4 grp + i of the output, row 16 mt + col
    const int vr = 4 * grp + (col >> 2);
    const uint16_t* v0 = vt + vr * DP + 4 * (col & 1);
#pragma unroll
    for (int x = 0; x < kBlocks; ++x) {
      const uint16_t* src = v0 + 8 * fp4_chunk(vr, 2 * x + ((col & 3) >> 1));
      const u32x2 lo2 = fp4_read_tr(src), hi2 = fp4_read_tr(src + 16 * DP);
      const u32x4 v = u32x4{lo2[0], lo2[1], hi2[0], hi2[1]};
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        acc[mt][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp4_bf16x8(v), fp4_bf16x8(p[mt]), acc[mt][x], 0, 0, 0);
        if constexpr (kRest) {
          acc[mt][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp4_bf16x8(v), fp4_bf16x8(rest[mt]), acc[mt][x], 0, 0, 0);
        }
      }
    }
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
template <int DP, int MT, bool kExact>
__device__ __forceinline__ void fp4_segment(Fp4Smem<DP>& sm, const Fp4AttnArgs& a, int b, int rb, int hk, const Fp4Span& sp,
                                            int t_from, int t_to, int slot_of_part, Fp4Pace& pace, int done) {
  using Wave = Fp4Wave<DP, MT, kExact, false>;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x) / kWave, lane = fp4_fresh_tid() % kWave;
  const int r0 = rb * 16 * MT;
  const int t_lo = sp.tile0 + t_from, t_hi = sp.tile0 + min(t_to, sp.tiles);
  Wave w(a, sp, b, hk, r0, lane);
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
      w.lookup(b, min(t, t_hi) * kF4Tile + 16 * (lane & 1), at, slot);
    }
    w.template fetch<true, true>(raw, at, slot, 2 * (i & 31));
  };
  // the tile's registers take the next tile (of two in flight, the one after) as soon
  // as its scores are made
  constexpr int kAhead = Wave::kTwo ? 2 : 1;
  const auto step = [&](typename Wave::Raw& raw, int i) {
    const int pos = (t_lo + wave + i * kF4Waves) * kF4Tile;
    w.template unpack_scales<true, true>(raw);
    Fp4Tile<MT> tl;
    tl.slot[0] = raw.slot[0];
    tl.slot[1] = raw.slot[1];
    tl.masked = w.uneven(raw, pos) || w.any_nan(raw);
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

// The same with tiles that the waves share: each has 16 MT of the item's rows and
// decodes one in four tiles' values for all of them.
template <int DP, int MT, bool kExact>
__device__ __forceinline__ void fp4_segment_shared(Fp4Smem<DP>& sm, const Fp4AttnArgs& a, int b, int rb, int hk, const Fp4Span& sp,
                                                   int t_from, int t_to, int slot_of_part, Fp4Pace& pace, int done) {
  using Wave = Fp4Wave<DP, MT, kExact, true>;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x) / kWave, lane = fp4_fresh_tid() % kWave;
  const int r0 = (rb * kF4Waves + wave) * 16 * MT;
  const int t_lo = sp.tile0 + t_from, t_hi = sp.tile0 + min(t_to, sp.tiles);
  Wave w(a, sp, b, hk, r0, lane);
  const int n = t_hi - t_lo;
  // lane 2 j + h, j < 4: half h of tile i + j (past the last something mapped)
  const auto places = [&](int i, uint64_t& at, int& slot) {
    w.lookup(b, min(t_lo + i + ((lane >> 1) & 3), t_hi) * kF4Tile + 16 * (lane & 1), at, slot);
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
      const int pos = (t_lo + i + wave) * kF4Tile;
      w.template unpack_scales<false, true>(vals);
      uint32_t nan_keys = 0;
      if (w.uneven(vals, pos) || w.any_nan(vals)) nan_keys = w.clean(vals, pos);  // uniform
      w.values(vals, reinterpret_cast<uint16_t*>(sm.tile[wave]));
      if (lane == 0) sm.nan_keys[wave] = nan_keys;
    }
    places(i + kF4Waves, at_next, slot_next);
    __syncthreads();  // the tiles are there
#pragma unroll
    for (int j = 0; j < kF4Waves; ++j) {
      typename Wave::Raw &kr = keys[j & 1], &next = keys[(j + 1) & 1];
      if (j < kF4Waves - 1) {
        w.template fetch<true, false>(next, at, slot, 2 * (j + 1));
      } else {
        w.template fetch<true, false>(next, at_next, slot_next, 0);
      }
      if (j == 1) w.template fetch<false, true>(vals, at_next, slot_next, 2 * wave);
      const int pos = (t_lo + i + j) * kF4Tile;
      Fp4Tile<MT> tl;
      tl.slot[0] = kr.slot[0];
      tl.slot[1] = kr.slot[1];
      tl.nan_keys = __builtin_amdgcn_readfirstlane(sm.nan_keys[j]);
      tl.masked = w.uneven(kr, pos) || tl.nan_keys != 0;
      w.template unpack_scales<true, false>(kr);
      w.scores(kr, tl);
      if (i + j < n) w.output(tl, pos, reinterpret_cast<const uint16_t*>(sm.tile[j]));  // uniform
    }
    at = at_next;
    slot = slot_next;
    __syncthreads();  // the tiles have been read
  }
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
      float* part = a.part + (static_cast<int64_t>(slot_of_part) * kF4Waves + wave) * (16 * MT) * (D + 4) + (16 * mt + col) * (D + 4);
      if (grp == 0) {
        part[0] = w.m[mt];
        part[1] = l;
      }
#pragma unroll
      for (int x = 0; x < Wave::kBlocks; ++x) {
        const int d = 16 * x + 4 * grp;
        if (kExact || d < D) *reinterpret_cast<f32x4*>(part + 4 + d) = w.acc[mt][x];
      }
    }
  }
}

template <int DP, int MT, bool kExact, bool kShared>
__global__ __launch_bounds__(kF4Threads, fp4_resident(DP, MT)) void k_fp4_attn(Fp4AttnArgs a) {
  constexpr int kRows = 16 * MT * (kShared ? kF4Waves : 1);
  __shared__ Fp4Smem<DP> sm;
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
    const bool whole = a.small == kF4SmallTiles && units <= groups &&
                       static_cast<int64_t>(uniform(sm.longest)) * groups * (kF4Idle - 1) <= static_cast<int64_t>(total) * kF4Idle;
    if (g == 0) {
      for (int i = tid; i <= items; i += kF4Threads) a.sched[i] = sm.pre[i];
      if (tid == 0) a.sched[items + 1] = whole ? INT32_MAX : a.small;
    }
    if (whole) groups = units;
    if (g >= groups) return;  // uniform
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
    x = uniform(run_start(g));
    end = uniform(run_start(g + 1));
  }
  Fp4Pace pace{0, 0, 0};
  if (!each) pace.start(end - x);  // in a grid of more than the device holds the oldest may go first
  const int x0 = x;
  while (x < end) {
    const int item = each ? x / a.Hkv : uniform(item_of(x));
    const Fp4Span sp = span_of(item, b, rb);
    const int lead = each ? 0 : a.lead, n = sp.units() + lead;
    const int in = each ? 0 : x - uniform(sm.pre[item]);
    const int hk = each ? x - item * a.Hkv : in / n;
    const int x1 = each ? 0 : in - hk * n, x2 = each ? n : min(n, x1 + end - x);
    const int from = max(x1 - lead, 0), to = x2 - lead;
    const int part = x1 == 0 && x2 == n ? -1 : x1 == 0 ? 2 * g + 1 : 2 * g;
    if constexpr (kShared) {
      fp4_segment_shared<DP, MT, kExact>(sm, a, b, rb, hk, sp, from, to, part, pace, x - x0);
    } else {
      fp4_segment<DP, MT, kExact>(sm, a, b, rb, hk, sp, from, to, part, pace, x - x0);
    }
    x += each ? 1 : x2 - x1;
    __syncthreads();  // the segment's LDS has been read
  }
}

// Joins the pieces of a cut item's row: the pieces' weights, then the weighted sum
// of their outputs with D / 4 threads to a piece, as many pieces at a time as the
// row's kThreads threads have room for.  (256 threads a row where there are few rows,
// a wave where there are many.)
template <int kThreads>
__global__ __launch_bounds__(kF4Threads) void k_fp4_attn_join(Fp4AttnArgs a, int rows_per_block, int rows_per_group) {
  constexpr int kRows = kF4Threads / kThreads;
  __shared__ alignas(16) f32x4 sum[kF4Threads];
  const int items = a.B * a.row_blocks;
  const int item = blockIdx.x / a.Hkv, hk = blockIdx.x - item * a.Hkv;
  const int b = item / a.row_blocks, rb = item - b * a.row_blocks;
  const int total = a.sched[items], p0 = a.sched[item], n = (a.sched[item + 1] - p0) / a.Hkv;
  if (n - a.lead <= a.sched[items + 1]) return;  // uniform
  const int groups = fp4_groups(a, total);
  const int x0 = p0 + hk * n;
  const int w0 = fp4_owner(x0 + min(fp4_early(a), n - 1), total, groups), pieces = fp4_owner(x0 + n - 1, total, groups) - w0 + 1;
  if (pieces == 1) return;  // uniform
  const int tid = threadIdx.x % kThreads, mine = threadIdx.x / kThreads, lane = threadIdx.x % kWave;
  const int64_t pitch = a.D + 4;
  const int quads = a.D / 4;
  const int lanes = min(quads, kThreads), sets = kThreads / lanes;
  const int set = tid / lanes, d0 = tid - set * lanes;
  const float ninf = -__builtin_huge_valf();
  for (int r1 = 0; r1 < rows_per_group; r1 += kRows) {  // uniform
    const int at = blockIdx.y * rows_per_group + r1 + mine, r = rb * rows_per_block + at;
    const bool live = r1 + mine < rows_per_group && at < rows_per_block && r < a.T * a.G;
    const int t = live ? r / a.G : 0, h = live ? hk * a.G + r - t * a.G : 0;
    const auto piece = [&](int k) {
      return a.part + ((k == 0 ? 2 * static_cast<int64_t>(w0) + 1 : 2 * static_cast<int64_t>(w0 + k)) * rows_per_block + (live ? at : 0)) * pitch;
    };
    // every wave of the row works the weights' sum out for itself
    float top = kF4None;
    for (int k = lane; k < pieces; k += kWave) top = fmaxf(top, piece(k)[0]);
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    const float sink = a.sink ? a.sink[h] * kF4Log2e : ninf;
    const float ref = fmaxf(top, sink) == kF4None ? 0.f : fmaxf(top, sink);
    float den = 0.f;
    for (int k = lane; k < pieces; k += kWave) {
      const float f = __builtin_amdgcn_exp2f(piece(k)[0] - ref), l = piece(k)[1];
      den += l != l ? l : f == 0.f ? 0.f : f * l;
    }
    for (int off = 32; off > 0; off >>= 1) den += __shfl_xor(den, off);
    if (sink != ninf) den += __builtin_amdgcn_exp2f(sink - ref);
    const float inv = den == 0.f ? 0.f : 1.f / den;
    for (int d1 = 0; d1 < quads; d1 += lanes) {  // once, but for wide heads on a wave
      const int d = d1 + d0;
      f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
      if (set < sets && d < quads) {
        constexpr int kAhead = 4;
        for (int k0 = set; k0 < pieces; k0 += kAhead * sets) {
          f32x4 x[kAhead];
          float m[kAhead];
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            const float* p = piece(min(k0 + k * sets, pieces - 1));
            m[k] = p[0];
            x[k] = reinterpret_cast<const f32x4*>(p + 4)[d];
          }
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            if (k0 + k * sets < pieces) v += x[k] * __builtin_amdgcn_exp2f(m[k] - ref);
          }
        }
      }
      __syncthreads();
      sum[threadIdx.x] = v;
      __syncthreads();
      if (live && set == 0 && d < quads) {
        for (int k = 1; k < min(sets, pieces); ++k) v += sum[mine * kThreads + k * lanes + d0];
        u32x2 y;
        y[0] = bf16_pack2(v[0] * inv, v[1] * inv);
        y[1] = bf16_pack2(v[2] * inv, v[3] * inv);
        *reinterpret_cast<u32x2*>(a.out + ((static_cast<int64_t>(b) * a.T + t) * a.H + h) * a.D + 4 * d) = y;
      }
    }
  }
}

struct Fp4AttnPlan {
  int dims, mt;  // padded dims, row tiles of a wave
  bool shared;   // the waves share the tiles, each with rows of its own
  int rows;      // of a workgroup
  int64_t row_blocks, items;
  bool cut;        // items may be cut
  int64_t groups;  // then: the most workgroups
  int64_t sched_bytes, ws_bytes;
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
  // 128; of 256 dims 68 and 65 with 32 rows, 68 and 101 with 33.  Heads of 512 dims stay apart (16
  // sequences of 4k: 57 us with 33 rows and 53 with 64, shared 61 and 64; their registers spill).
  const int mt = fp4_shared_mt(p.dims);
  p.shared = p.dims <= 256 && rows > 16 * mt * kF4Waves / 2;
  p.mt = p.shared ? mt : rows <= 16 || p.dims > 256 ? 1 : 2;
  p.rows = 16 * p.mt * (p.shared ? kF4Waves : 1);
  p.row_blocks = ceil_div(rows, p.rows);
  p.items = d->cache.batch * p.row_blocks;
  // the most tiles that a row block may see
  const int64_t capacity = d->cache.bt_stride * d->cache.block_size;
  int64_t len = d->max_len > 0 ? std::min(d->max_len, capacity) : capacity;
  if (d->window > 0) len = std::min(len, d->window + ceil_div(p.rows, d->n_heads / hkv));
  const int64_t tiles = ceil_div(len, kF4Tile) + 1, units = std::max<int64_t>(p.items * hkv, 1);
  p.cut = tiles > kF4SmallTiles || d->splits > 0;
  if (p.items > kF4MaxItems || units > INT32_MAX / (ceil_div(capacity, kF4Tile) + 1 + kF4Lead)) p.cut = false;
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
template <int DP, bool kExact>
void launch_rows(const Fp4AttnArgs& a, const Fp4AttnPlan& p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.max_groups > 0 ? a.max_groups : static_cast<int64_t>(a.B) * a.row_blocks * a.Hkv));
  const auto go = [&](auto* kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kF4Threads), 0, s, a); };
  if constexpr (DP <= 256) {
    if (p.shared) return go(&k_fp4_attn<DP, fp4_shared_mt(DP), kExact, true>);
    if (p.mt == 2) return go(&k_fp4_attn<DP, 2, kExact, false>);
  }
  go(&k_fp4_attn<DP, 1, kExact, false>);
}
template <bool kExact>
void launch_dims(const Fp4AttnArgs& a, const Fp4AttnPlan& p, hipStream_t s) {
  if (p.dims == 64) launch_rows<64, kExact>(a, p, s);
  if (p.dims == 128) launch_rows<128, kExact>(a, p, s);
  if (p.dims == 256) launch_rows<256, kExact>(a, p, s);
  if (p.dims == 512) launch_rows<512, kExact>(a, p, s);
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
  if (a.D == p.dims) launch_dims<true>(a, p, s); else launch_dims<false>(a, p, s);
  if (const int rc = check_launch(what)) return rc;
  if (!p.cut) return SKV_OK;
  // a row to a workgroup where that makes few of them, else to a wave, up to about 8,192 workgroups
  const int64_t units = p.items * a.Hkv, block_rows = std::min<int64_t>(p.rows, static_cast<int64_t>(a.T) * a.G);
  const bool few = units * block_rows <= 2048;
  const int64_t per = few ? 1 : std::min(block_rows, std::max<int64_t>(kF4Waves, ceil_div(units * block_rows, 8192)));
  const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>(ceil_div(block_rows, per)));
  if (few) {
    hipLaunchKernelGGL((k_fp4_attn_join<kF4Threads>), grid, dim3(kF4Threads), 0, s, a, p.rows, static_cast<int>(per));
  } else {
    hipLaunchKernelGGL((k_fp4_attn_join<kWave>), grid, dim3(kF4Threads), 0, s, a, p.rows, static_cast<int>(per));
  }
  return check_launch(what);
}
