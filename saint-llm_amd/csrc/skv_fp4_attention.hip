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
// blocks of 16 MT rows, the positions into chunks; a workgroup takes a row block over a
// chunk, its four waves tiles of 32 positions in turn, each with a softmax of
// its own, joined at the end.  No wave waits for another on the way:
//   * S^T = K Q^T: lane (key, g) of a 16-key tile reads D / 4 consecutive dims of
//     its key, g's quarter, from the page straight into the registers of the
//     products' A operand (the order of the dims within a product is free as
//     long as the query's is the same: step s takes dims g D / 4 + 8 s ..+7);
//     for 128 dims that is 16 bytes and one scale byte a lane, a tile 1 KB in one run.
//   * the values go through the wave's own part of LDS as bf16, rows of D in
//     swizzled chunks, and come back transposed (ds_read_b64_tr_b16) as the A
//     operand of O^T = V^T P^T, whose B operand is P^T as the scores' accumulators
//     hold it.  O^T keeps a row's output in the lanes that hold its m and l.
// The codes of the next tile are in flight while one is multiplied, the page
// ids of 32 tiles sit in the lanes of a register.  Chunks of long sequences are
// joined by a second launch.
#include <algorithm>

#include "skv_fp4.h"

namespace skv {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));

constexpr int kF4Threads = 256;
constexpr int kF4Waves = kF4Threads / kWave;
constexpr int kF4Tile = 32;        // positions per tile
constexpr float kF4Log2e = 1.4426950408889634f;
constexpr float kF4Move = 8.f;     // log2: the reference maximum moves when a tile's passes it by more

struct Fp4AttnArgs {
  const uint8_t* q;
  int64_t q_seq, q_tok, q_head;
  uint16_t* out;  // [B, T, H, D] bf16
  float* part;    // of chunk parts: (m, l) of every row, then the rows' outputs
  const int32_t* lens;
  const uint8_t* pool;
  const int32_t* bt;
  const float* sink;
  int32_t n_pages, bt_stride, bs;
  int32_t B, T, H, Hkv, G, D;
  int32_t window;  // 0: none
  float scale, softcap;
  int32_t row_blocks, chunks, chunk_tiles;
};

// The positions that the rows [r0, r0 + n) of a K/V head see.
struct Fp4Span {
  int L, r_end;          // tokens of the sequence; rows of the head
  int first, last;       // [first, last): some row sees them
  int all_lo, all_hi;    // [all_lo, all_hi): every row sees them
  int tile0, tiles;
};

__device__ __forceinline__ Fp4Span fp4_span(const Fp4AttnArgs& a, int b, int r0, int n) {
  Fp4Span s;
  s.L = min(max(a.lens[b], 0), a.bt_stride * a.bs);
  s.r_end = a.T * a.G;
  const int r1 = min(r0 + n, s.r_end) - 1;
  const int end0 = s.L - a.T + r0 / a.G + 1, end1 = s.L - a.T + r1 / a.G + 1;  // one past the last position seen
  s.last = max(end1, 0);
  s.all_hi = end0;
  s.first = a.window > 0 ? max(end0 - a.window, 0) : 0;
  s.all_lo = a.window > 0 ? end1 - a.window : 0;
  s.tile0 = s.first / kF4Tile;
  s.tiles = s.last > s.first ? (s.last + kF4Tile - 1) / kF4Tile - s.tile0 : 0;
  return s;
}

// Chunks that hold positions of a span: the last takes what is past the bound
// that the chunks were made for.
__device__ __forceinline__ int fp4_chunks(const Fp4AttnArgs& a, const Fp4Span& s) {
  return min((s.tiles + a.chunk_tiles - 1) / a.chunk_tiles, a.chunks);
}

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
  uint32_t k[2][kWords], v[2][kWords];
  uint8_t ks[2][kScales], vs[2][kScales];
  bool mapped[2];  // uniform
};

template <int DP>
struct Fp4Smem {
  // per wave: 32 value rows of DP bf16; at the end 16 output rows of DP fp32
  alignas(16) uint8_t tile[kF4Waves][64 * DP];
  float m[kF4Waves][64], l[kF4Waves][64];
};

// DP: the head's dims padded to 64, 128, 256 or 512 (kExact: D == DP).
template <int DP, int MT, bool kExact>
struct Fp4Wave {
  using Raw = Fp4Raw<DP>;
  static constexpr int kWords = Raw::kWords, kScales = Raw::kScales;
  static constexpr int kBlocks = DP / 16;  // 16-dim blocks of the output

  const Fp4AttnArgs& a;
  const Fp4Span& sp;
  const Fp4Page pg;
  int lane, col, grp;
  const uint8_t* head;  // the K/V head's block in page 0
  u32x4 q[MT][kWords];
  int hi[MT], lo[MT];   // the positions that row 16 mt + col sees
  float m[MT], l[MT];
  f32x4 acc[MT][kBlocks];

  __device__ __forceinline__ Fp4Wave(const Fp4AttnArgs& a_, const Fp4Span& sp_, int b, int hk, int r0)
      : a(a_), sp(sp_), pg(fp4_page(a_.bs, a_.Hkv, kExact ? DP : a_.D)) {
    lane = threadIdx.x % kWave;
    col = lane & 15;
    grp = lane >> 4;
    head = a.pool + hk * pg.head;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = r0 + 16 * mt + col;
      const bool in = r < sp.r_end;
      const int t = in ? r / a.G : 0, g = in ? r - t * a.G : 0;
      hi[mt] = in ? sp.L - a.T + t + 1 : 0;
      lo[mt] = a.window > 0 ? hi[mt] - a.window : 0;
      const uint8_t* row = a.q + b * a.q_seq + t * a.q_tok + (hk * a.G + g) * a.q_head;
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        const int d = grp * (DP / 4) + 8 * w;
        q[mt][w] = u32x4{0u, 0u, 0u, 0u};
        if (in && (kExact || d < a.D)) q[mt][w] = *reinterpret_cast<const u32x4*>(row + 2 * d);
      }
      m[mt] = -__builtin_huge_valf();
      l[mt] = 0.f;
#pragma unroll
      for (int x = 0; x < kBlocks; ++x) acc[mt][x] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // page id (-1: not mapped) and first slot of the 16 positions from `pos` on
  __device__ __forceinline__ void lookup(int b, int pos, int& page, int& slot) const {
    const int p = static_cast<int>(udiv24(pos, a.bs));
    slot = pos - p * a.bs;
    page = pos < sp.last ? a.bt[static_cast<int64_t>(b) * a.bt_stride + p] : -1;
    if (page >= a.n_pages) page = -1;
  }

  __device__ __forceinline__ void load(Raw& r, int half, int page, int slot) const {
    r.mapped[half] = page >= 0;
    const uint8_t* base = head + (page >= 0 ? page : 0) * pg.page;  // uniform
    const int D = kExact ? DP : a.D;
    const int nb = D / kFp4Block;
    const int row = (slot + col) * (D / 2) + grp * (DP / 8);
    const int sc = pg.scales + 2 * (slot + col) * nb;
    if constexpr (kExact && DP >= 128) {
#pragma unroll
      for (int w = 0; w < kWords; w += 4) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(base + row + 4 * w);
        const u32x4 y = *reinterpret_cast<const u32x4*>(base + pg.v_codes + row + 4 * w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          r.k[half][w + i] = x[i];
          r.v[half][w + i] = y[i];
        }
      }
    } else {
#pragma unroll
      for (int w = 0; w < kWords; w += 2) {
        const bool in = kExact || grp * (DP / 4) + 8 * w < D;
        const int o = in ? row + 4 * w : 0;
        const u32x2 x = *reinterpret_cast<const u32x2*>(base + o);
        const u32x2 y = *reinterpret_cast<const u32x2*>(base + pg.v_codes + o);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          r.k[half][w + i] = in ? x[i] : 0u;
          r.v[half][w + i] = in ? y[i] : 0u;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kScales; ++i) {
      const int blk = DP >= 128 ? grp * kScales + i : grp >> 1;
      const int o = kExact || blk < nb ? blk : 0;
      r.ks[half][i] = base[sc + o];
      r.vs[half][i] = base[sc + nb + o];
    }
  }

  // One tile: positions pos .. pos + 31.
  __device__ __forceinline__ void tile(Raw& r, int pos, uint16_t* vt) {
    // keys that no row sees hold stale bytes: their values become zeros (their
    // weights are); a NaN block among the values too, and its key's scores NaN
    const bool whole = pos >= sp.all_lo && pos + kF4Tile <= sp.all_hi && r.mapped[0] && r.mapped[1];  // uniform
    uint32_t nan_keys = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bool nan = false;
#pragma unroll
      for (int i = 0; i < kScales; ++i) nan |= r.vs[h][i] == kFp4NaN;
      if constexpr (!kExact) nan &= grp * (DP / 4) < a.D;
      bool dead = nan;
      if (!whole) dead |= pos + 16 * h + col >= sp.last || pos + 16 * h + col < sp.first || !r.mapped[h];
      if (__ballot(dead)) {
        const uint64_t n = __ballot(nan);
        nan_keys |= static_cast<uint32_t>((n | n >> 16 | n >> 32 | n >> 48) & 0xffff) << (16 * h);
        if (dead) {
#pragma unroll
          for (int w = 0; w < kWords; ++w) r.v[h][w] = 0u;
#pragma unroll
          for (int i = 0; i < kScales; ++i) r.vs[h][i] = 127;
        }
      }
      uint16_t* dst = vt + (16 * h + col) * DP;
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        *reinterpret_cast<u32x4*>(dst + 8 * fp4_chunk(col, grp * kWords + w)) =
            fp4_decode8(r.v[h][w], fp4_scale(r.vs[h][w / 4 < kScales ? w / 4 : 0]));
      }
    }
    f32x4 st[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) st[mt][0] = st[mt][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 k = fp4_decode8(r.k[h][w], fp4_scale(r.ks[h][w / 4 < kScales ? w / 4 : 0]));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          st[mt][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp4_bf16x8(k), fp4_bf16x8(q[mt][w]), st[mt][h], 0, 0, 0);
        }
      }
    }
    const bool capped = a.softcap > 0.f;
    const float mult = capped ? 1.f : a.scale * kF4Log2e;
    u32x4 p[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      // scores of positions pos + 16 h + 4 grp + i for row 16 mt + col
      if (capped) {
        const float to = 2.f * kF4Log2e * a.scale / a.softcap, cap = a.softcap * kF4Log2e;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // tanh(x) = 1 - 2 / (exp(2x) + 1)
            st[mt][h][i] = cap * (1.f - 2.f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(st[mt][h][i] * to) + 1.f));
          }
        }
      }
      if (!whole || nan_keys) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = 16 * h + 4 * grp + i;
            float v = (nan_keys >> key) & 1 ? __builtin_nanf("") : st[mt][h][i];
            const bool seen = pos + key < hi[mt] && pos + key >= lo[mt] && r.mapped[h];
            st[mt][h][i] = seen ? v : -__builtin_huge_valf();
          }
        }
      }
      float mx = fmaxf(fmaxf(fmaxf(st[mt][0][0], st[mt][0][1]), fmaxf(st[mt][0][2], st[mt][0][3])),
                       fmaxf(fmaxf(st[mt][1][0], st[mt][1][1]), fmaxf(st[mt][1][2], st[mt][1][3])));
      mx = fp4_max_groups(mx) * mult;
      const bool move = mx > m[mt] + kF4Move;
      if (__ballot(move)) {
        const float alpha = move ? __builtin_amdgcn_exp2f(m[mt] - mx) : 1.f;
        if (move) m[mt] = mx;
        l[mt] *= alpha;
#pragma unroll
        for (int x = 0; x < kBlocks; ++x) acc[mt][x] *= alpha;
      }
      const float ref = m[mt] == -__builtin_huge_valf() ? 0.f : m[mt];
      float e[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[4 * h + i] = __builtin_amdgcn_exp2f(fmaf(st[mt][h][i], mult, -ref));
      }
      l[mt] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
#pragma unroll
      for (int i = 0; i < 4; ++i) p[mt][i] = bf16_pack2(e[2 * i], e[2 * i + 1]);
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
      }
    }
  }
};

template <int DP, int MT, bool kExact>
__global__ __launch_bounds__(kF4Threads) void k_fp4_attn(Fp4AttnArgs a) {
  using Wave = Fp4Wave<DP, MT, kExact>;
  __shared__ Fp4Smem<DP> sm;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x) / kWave, lane = threadIdx.x % kWave;
  // block -> (chunk unit, row block): a unit's row blocks, which read the same
  // pages, follow one another on one XCD (block i runs on XCD i % 8)
  const int n_units = a.B * a.Hkv * a.chunks;
  const int turn = blockIdx.x >> 3, in_turn = turn % a.row_blocks;
  const int unit = (turn / a.row_blocks) * 8 + (blockIdx.x & 7);
  if (unit >= n_units) return;  // uniform
  const int rb = a.row_blocks - 1 - in_turn;
  const int chunk = unit % a.chunks, bh = unit / a.chunks;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int r0 = rb * 16 * MT;
  const Fp4Span sp = fp4_span(a, b, r0, 16 * MT);
  const int n_chunks = fp4_chunks(a, sp);
  if (chunk >= max(n_chunks, 1)) return;  // uniform
  const int t_lo = sp.tile0 + chunk * a.chunk_tiles;
  const int t_hi = chunk == a.chunks - 1 ? sp.tile0 + sp.tiles : min(t_lo + a.chunk_tiles, sp.tile0 + sp.tiles);
  Wave w(a, sp, b, hk, r0);
  uint16_t* vt = reinterpret_cast<uint16_t*>(sm.tile[wave]);
  // this wave's tiles t_lo + wave, + 4, ...; the page ids of 32 of them at a time
  typename Wave::Raw raw;
  int page = -1, slot = 0;
  const int n = t_hi > t_lo + wave ? (t_hi - t_lo - wave + kF4Waves - 1) / kF4Waves : 0;
  const auto ids = [&](int i) {  // lane 2 j + h: half h of tile i + j
    const int t = t_lo + wave + (i + (lane >> 1)) * kF4Waves;
    w.lookup(b, min(t, t_hi) * kF4Tile + 16 * (lane & 1), page, slot);
  };
  const auto fetch = [&](int i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = 2 * (i & 31) + h;
      w.load(raw, h, __builtin_amdgcn_readlane(page, at), __builtin_amdgcn_readlane(slot, at));
    }
  };
  if (n > 0) {
    ids(0);
    fetch(0);
  }
  for (int i = 0; i < n; ++i) {
    typename Wave::Raw cur = raw;
    if (i + 1 < n) {
      if (((i + 1) & 31) == 0) ids(i + 1);
      fetch(i + 1);
    }
    w.tile(cur, (t_lo + wave + i * kF4Waves) * kF4Tile, vt);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  }
  // join the waves: maxima and sums of every row, then the outputs, a row tile at a time
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const float l = fp4_sum_groups(w.l[mt]);
    if (w.grp == 0) {
      sm.m[wave][16 * mt + w.col] = w.m[mt];
      sm.l[wave][16 * mt + w.col] = l;
    }
  }
  const float ninf = -__builtin_huge_valf();
  const int64_t part_row = (static_cast<int64_t>(unit) * a.row_blocks + rb) * (16 * MT);
  const int64_t part_rows = static_cast<int64_t>(n_units) * a.row_blocks * (16 * MT);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    __syncthreads();  // the tiles (or the last row tile's outputs) have been read, the maxima are written
    f32x4* o = reinterpret_cast<f32x4*>(sm.tile[wave]);
#pragma unroll
    for (int x = 0; x < Wave::kBlocks; ++x) o[w.col * (DP / 4) + ((4 * x + w.grp) ^ (w.col & 7))] = w.acc[mt][x];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (DP / 4); i += kF4Threads) {
      const int row = i / (DP / 4), c = i % (DP / 4), r = r0 + 16 * mt + row;
      const int d = 4 * c;
      if (r >= sp.r_end || (!kExact && d >= a.D)) continue;
      const int t = r / a.G, h = hk * a.G + r - t * a.G;
      float top = ninf;
#pragma unroll
      for (int k = 0; k < kF4Waves; ++k) top = fmaxf(top, sm.m[k][16 * mt + row]);
      const bool one = a.chunks == 1;
      const float sink = one && a.sink ? a.sink[h] * kF4Log2e : ninf;
      const float ref = fmaxf(top, sink) == ninf ? 0.f : fmaxf(top, sink);
      float den = 0.f;
      f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kF4Waves; ++k) {
        const float f = __builtin_amdgcn_exp2f(sm.m[k][16 * mt + row] - ref);
        const float lk = sm.l[k][16 * mt + row];
        den += f == 0.f && lk == 0.f ? 0.f : f * lk;
        if (lk != lk) den = lk;  // NaN keys alone: no maximum
        v += reinterpret_cast<const f32x4*>(sm.tile[k])[row * (DP / 4) + (c ^ (row & 7))] * f;
      }
      if (one) {
        if (sink != ninf) den += __builtin_amdgcn_exp2f(sink - ref);
        const float inv = den == 0.f ? 0.f : 1.f / den;
        u32x2 y;
        y[0] = bf16_pack2(v[0] * inv, v[1] * inv);
        y[1] = bf16_pack2(v[2] * inv, v[3] * inv);
        *reinterpret_cast<u32x2*>(a.out + ((static_cast<int64_t>(b) * a.T + t) * a.H + h) * (kExact ? DP : a.D) + d) = y;
      } else {
        const int64_t pr = part_row + 16 * mt + row;
        if (c == 0) {
          a.part[2 * pr] = top;
          a.part[2 * pr + 1] = den;
        }
        reinterpret_cast<f32x4*>(a.part + 2 * part_rows)[pr * ((kExact ? DP : a.D) / 4) + c] = v;
      }
    }
  }
}

// Joins the chunks of every row: one wave per row, four rows a workgroup.
__global__ __launch_bounds__(kF4Threads) void k_fp4_attn_join(Fp4AttnArgs a, int rows_per_block) {
  const int lane = threadIdx.x % kWave;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kF4Waves + threadIdx.x / kWave;
  const int R = a.T * a.G;
  const int bh = static_cast<int>(item / R), r = static_cast<int>(item - static_cast<int64_t>(bh) * R);
  if (bh >= a.B * a.Hkv) return;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int t = r / a.G, h = hk * a.G + r - t * a.G;
  const int rb = r / rows_per_block;
  const Fp4Span sp = fp4_span(a, b, rb * rows_per_block, rows_per_block);
  const int n = fp4_chunks(a, sp);
  const int64_t part_rows = static_cast<int64_t>(a.B) * a.Hkv * a.chunks * a.row_blocks * rows_per_block;
  const auto row_of = [&](int c) {
    return ((static_cast<int64_t>(bh) * a.chunks + c) * a.row_blocks + rb) * rows_per_block + (r - rb * rows_per_block);
  };
  const float ninf = -__builtin_huge_valf();
  float top = ninf;
  for (int c = lane; c < n; c += kWave) top = fmaxf(top, a.part[2 * row_of(c)]);
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  const float sink = a.sink ? a.sink[h] * kF4Log2e : ninf;
  const float ref = fmaxf(top, sink) == ninf ? 0.f : fmaxf(top, sink);
  float den = 0.f;
  for (int c = lane; c < n; c += kWave) {
    const float f = __builtin_amdgcn_exp2f(a.part[2 * row_of(c)] - ref), l = a.part[2 * row_of(c) + 1];
    den += l != l ? l : f == 0.f ? 0.f : f * l;
  }
  for (int off = 32; off > 0; off >>= 1) den += __shfl_xor(den, off);
  if (sink != ninf) den += __builtin_amdgcn_exp2f(sink - ref);
  const float inv = den == 0.f ? 0.f : 1.f / den;
  const f32x4* o = reinterpret_cast<const f32x4*>(a.part + 2 * part_rows);
  for (int d = lane; d < a.D / 4; d += kWave) {
    f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < n; ++c) {
      const int64_t pr = row_of(c);
      v += o[pr * (a.D / 4) + d] * __builtin_amdgcn_exp2f(a.part[2 * pr] - ref);
    }
    u32x2 y;
    y[0] = bf16_pack2(v[0] * inv, v[1] * inv);
    y[1] = bf16_pack2(v[2] * inv, v[3] * inv);
    *reinterpret_cast<u32x2*>(a.out + ((static_cast<int64_t>(b) * a.T + t) * a.H + h) * a.D + 4 * d) = y;
  }
}

struct Fp4AttnPlan {
  int dims, mt;  // padded dims, row tiles of a workgroup
  int64_t row_blocks, chunks, chunk_tiles;
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
  const int64_t D = d->cache.head_dim, rows = d->n_queries * (d->n_heads / hkv);
  p.dims = D <= 64 ? 64 : D <= 128 ? 128 : D <= 256 ? 256 : 512;
  const int most = p.dims <= 128 ? 4 : p.dims == 256 ? 2 : 1;
  p.mt = std::min(most, rows <= 16 ? 1 : rows <= 32 ? 2 : 4);
  p.row_blocks = ceil_div(rows, 16 * p.mt);
  // positions that a row block may see, in tiles (two may be cut at the ends)
  const int64_t capacity = d->cache.bt_stride * d->cache.block_size;
  int64_t len = d->max_len > 0 ? std::min(d->max_len, capacity) : capacity;
  if (d->window > 0) len = std::min(len, d->window + ceil_div(16 * p.mt, d->n_heads / hkv));
  const int64_t tiles = ceil_div(len, kF4Tile) + 1;
  const int64_t blocks = std::max<int64_t>(1, d->cache.batch * hkv * p.row_blocks);
  int64_t chunks = d->splits;
  if (chunks == 0) {
    chunks = std::max<int64_t>(1, ceil_div(16 * device_cus(), blocks));
    chunks = std::min(chunks, ceil_div(tiles, 2 * kF4Waves));
  }
  chunks = std::min<int64_t>(std::min(chunks, tiles), 1024);
  p.chunk_tiles = ceil_div(tiles, chunks);
  p.chunks = ceil_div(tiles, p.chunk_tiles);
  if (blocks * p.chunks >= (1 << 28)) return set_error(SKV_EINVAL, "%s: too many workgroups", what);
  p.ws_bytes = p.chunks > 1 ? blocks * p.chunks * 16 * p.mt * (D + 2) * 4 : 0;
  return SKV_OK;
}

// The part launch for padded dims DP and mt row tiles (at most those that plan gives).
template <int DP, bool kExact>
void launch_rows(const Fp4AttnArgs& a, int mt, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(ceil_div(static_cast<int64_t>(a.B) * a.Hkv * a.chunks, 8) * 8 * a.row_blocks));
  if (mt == 1) hipLaunchKernelGGL((k_fp4_attn<DP, 1, kExact>), grid, dim3(kF4Threads), 0, s, a);
  if constexpr (DP <= 256) {
    if (mt == 2) hipLaunchKernelGGL((k_fp4_attn<DP, 2, kExact>), grid, dim3(kF4Threads), 0, s, a);
  }
  if constexpr (DP <= 128) {
    if (mt == 4) hipLaunchKernelGGL((k_fp4_attn<DP, 4, kExact>), grid, dim3(kF4Threads), 0, s, a);
  }
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
  a.B = static_cast<int32_t>(d->cache.batch);
  a.part = static_cast<float*>(workspace);
  a.row_blocks = static_cast<int32_t>(p.row_blocks);
  a.chunks = static_cast<int32_t>(p.chunks);
  a.chunk_tiles = static_cast<int32_t>(p.chunk_tiles);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.D != p.dims) {
    if (p.dims == 64) launch_rows<64, false>(a, p.mt, s);
    if (p.dims == 128) launch_rows<128, false>(a, p.mt, s);
    if (p.dims == 256) launch_rows<256, false>(a, p.mt, s);
    if (p.dims == 512) launch_rows<512, false>(a, p.mt, s);
  } else {
    if (p.dims == 64) launch_rows<64, true>(a, p.mt, s);
    if (p.dims == 128) launch_rows<128, true>(a, p.mt, s);
    if (p.dims == 256) launch_rows<256, true>(a, p.mt, s);
    if (p.dims == 512) launch_rows<512, true>(a, p.mt, s);
  }
  if (const int rc = check_launch(what)) return rc;
  if (p.chunks == 1) return SKV_OK;
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hkv * a.T * a.G;
  hipLaunchKernelGGL(k_fp4_attn_join, dim3(static_cast<unsigned>(ceil_div(rows, kF4Waves))), dim3(kF4Threads), 0, s, a,
                     16 * p.mt);
  return check_launch(what);
}
