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
//   64 sequences of 1k - 32k, 64 heads on 8 of 128 dims                    131 (117)
//   4 of 256k - 1M, 4 tokens, 16 heads on 4 of 64                          93 (74)
//   16 of 64k, 64 heads on 1 of 128                                        78 (25, products)
//   2 prompts' 1000 tokens over 16k, 32 heads on 8 of 128                  510 (367, products)
//   1 prompt's 512 tokens over 200k, the same heads                        1567 (1200, products)
//   32 windows of 128, 64 heads on 1 of 512                                20 (1)
// and dropped: two row groups of two waves with half the tiles each for 33 - 64 rows (68 ->
// 74 us for the 64k sequences, before their weights had rests: a tile's latency is then seen by
// all four waves); the next tile's scores ahead of a tile's weights (1%); a prologue that loads
// the queries last.
#include "skv_fp4_attn.h"

namespace skv {

// The first workgroup of an item's head, and how many have a piece of it.
struct Fp4Pieces {
  int first, n;
};
__device__ __forceinline__ Fp4Pieces fp4_pieces(const Fp4AttnArgs& a, int items, int item, int hk) {
  const int total = a.sched[items], p0 = a.sched[item], n = (a.sched[item + 1] - p0) / a.Hkv, small = a.sched[items + 1];
  if (small < 0) return {p0 + hk * n, n};  // counted in pieces, a workgroup each
  if (n - a.lead <= small) return {0, 1};
  const int groups = fp4_groups(a, total);
  const int x0 = p0 + hk * n;
  const int w0 = fp4_owner(x0 + min(fp4_early(a), n - 1), total, groups);
  return {w0, fp4_owner(x0 + n - 1, total, groups) - w0 + 1};
}

// Joins the pieces of a cut item's row: the pieces' weights, then the weighted sum
// of their outputs with D / 4 threads to a piece, as many pieces at a time as the
// row's kThreads threads have room for.  (256 threads a row where there are few rows,
// a wave where there are many.)
template <int kThreads, bool kShared>
__global__ __launch_bounds__(kF4Threads) void k_fp4_attn_join(Fp4AttnArgs a, int rows_per_block, int rows_per_group) {
  constexpr int kRows = kF4Threads / kThreads;
  __shared__ alignas(16) f32x4 sum[kF4Threads];
  const int items = a.B * a.row_blocks;
  const int item = blockIdx.x / a.Hkv, hk = blockIdx.x - item * a.Hkv;
  const int b = item / a.row_blocks, rb = item - b * a.row_blocks;
  const auto [w0, pieces] = fp4_pieces(a, items, item, hk);
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
    const int row = live ? at : 0, wave_rows = rows_per_block / kF4Waves;
    const auto piece = [&](int k) {
      const int64_t slot = k == 0 ? 2 * static_cast<int64_t>(w0) + 1 : 2 * static_cast<int64_t>(w0 + k);
      if constexpr (kShared) {
        return Fp4Part{a.part + (slot * rows_per_block + row / wave_rows * wave_rows) * pitch, wave_rows, a.D / 16};
      } else {
        return a.part + (slot * rows_per_block + row) * pitch;
      }
    };
    const auto m_of = [&](auto p) {
      if constexpr (kShared) return *p.m(row % wave_rows); else return p[0];
    };
    const auto l_of = [&](auto p) {
      if constexpr (kShared) return *p.l(row % wave_rows); else return p[1];
    };
    const auto quad_of = [&](auto p, int d) {
      if constexpr (kShared) return *p.quad(row % wave_rows, d); else return reinterpret_cast<const f32x4*>(p + 4)[d];
    };
    // every wave of the row works the weights' sum out for itself
    float top = kF4None;
    for (int k = lane; k < pieces; k += kWave) top = fmaxf(top, m_of(piece(k)));
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    const float sink = a.sink ? a.sink[h] * kF4Log2e : ninf;
    const float ref = fmaxf(top, sink) == kF4None ? 0.f : fmaxf(top, sink);
    float den = 0.f;
    for (int k = lane; k < pieces; k += kWave) {
      const float f = __builtin_amdgcn_exp2f(m_of(piece(k)) - ref), l = l_of(piece(k));
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
            const auto p = piece(min(k0 + k * sets, pieces - 1));
            m[k] = m_of(p);
            x[k] = quad_of(p, d);
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

// The same for many rows of shared tiles: a workgroup has an item's 16-dim blocks of 16 rows, a wave those of
// the wave that wrote them, in its lanes' order, so that a load is one run of 1 KB, and a lane works its row's
// weights out for itself.  32 trees' 256 rows on 8 heads, 1k - 16k tokens (1024 pieces, 69 MB): 13 us, 31 with a
// wave to a row of parts that lie row by row (whose writing took 31 us more of the first launch, too).
__global__ __launch_bounds__(kF4Threads) void k_fp4_attn_join_blocks(Fp4AttnArgs a, int rows_per_block, int blocks_per_group) {
  const int items = a.B * a.row_blocks;
  const int item = blockIdx.x / a.Hkv, hk = blockIdx.x - item * a.Hkv;
  const int b = item / a.row_blocks, rb = item - b * a.row_blocks;
  const auto [w0, pieces] = fp4_pieces(a, items, item, hk);
  if (pieces == 1) return;  // uniform
  const int wave = threadIdx.x / kWave, col = threadIdx.x % kWave >> 2, grp = threadIdx.x & 3;
  const int wave_rows = rows_per_block / kF4Waves, per_row = a.D / 16;
  const int64_t pitch = a.D + 4;
  const float ninf = -__builtin_huge_valf();
  const auto piece = [&](int k) {
    const int64_t slot = k == 0 ? 2 * static_cast<int64_t>(w0) + 1 : 2 * static_cast<int64_t>(w0 + k);
    return Fp4Part{a.part + (slot * kF4Waves + wave) * wave_rows * pitch, wave_rows, per_row};
  };
  const int first = blockIdx.y * blocks_per_group, last = min(first + blocks_per_group, wave_rows / 16 * per_row);
  for (int block = first; block < last;) {  // of one 16 rows at a time
    const int mt = block / per_row, end = min(last, (mt + 1) * per_row), row = 16 * mt + col;
    const int r = (rb * kF4Waves + wave) * wave_rows + row;
    const bool live = r < a.T * a.G;
    const int t = live ? r / a.G : 0, h = live ? hk * a.G + r - t * a.G : 0;
    const float sink = a.sink ? a.sink[h] * kF4Log2e : ninf;
    constexpr int kAhead = 4, kBlocks = 2;  // pieces in flight, of so many blocks
    for (; block < end; block += kBlocks) {
      // one pass over the pieces with the running maximum and sum of their softmax
      float top = kF4None, den = 0.f;
      f32x4 v[kBlocks] = {};
      for (int k0 = 0; k0 < pieces; k0 += kAhead) {
        float m[kAhead], l[kAhead];
        f32x4 x[kAhead][kBlocks];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const Fp4Part p = piece(min(k0 + k, pieces - 1));
          m[k] = *p.m(row);
          l[k] = *p.l(row);
#pragma unroll
          for (int i = 0; i < kBlocks; ++i) x[k][i] = *p.quad(row, 4 * (min(block + i, end - 1) - mt * per_row) + grp);
        }
        float up = top;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) up = fmaxf(up, m[k]);
        const float down = __builtin_amdgcn_exp2f(top - up);
        top = up;
        den *= down;
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) v[i] *= down;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          if (k0 + k >= pieces) break;
          const float f = __builtin_amdgcn_exp2f(m[k] - top);
          den += l[k] != l[k] ? l[k] : f == 0.f ? 0.f : f * l[k];
#pragma unroll
          for (int i = 0; i < kBlocks; ++i) v[i] += x[k][i] * f;
        }
      }
      const float ref = fmaxf(top, sink) == kF4None ? 0.f : fmaxf(top, sink), down = __builtin_amdgcn_exp2f(top - ref);
      den *= down;
      if (sink != ninf) den += __builtin_amdgcn_exp2f(sink - ref);
      const float inv = den == 0.f ? 0.f : down / den;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        if (!live || block + i >= end) break;
        u32x2 y;
        y[0] = bf16_pack2(v[i][0] * inv, v[i][1] * inv);
        y[1] = bf16_pack2(v[i][2] * inv, v[i][3] * inv);
        const int d = 16 * (block + i - mt * per_row) + 4 * grp;
        *reinterpret_cast<u32x2*>(a.out + ((static_cast<int64_t>(b) * a.T + t) * a.H + h) * a.D + d) = y;
      }
    }
    block = end;
  }
}

// a row to a workgroup where that makes few of them, else to a wave, up to about 8,192 workgroups
void fp4_attn_join(const Fp4AttnArgs& a, const Fp4AttnPlan& p, hipStream_t s) {
  const int64_t units = p.items * a.Hkv, block_rows = std::min<int64_t>(p.rows, static_cast<int64_t>(a.T) * a.G);
  const bool few = units * block_rows <= 2048;
  if (p.shared && !few) {  // up to about 2,048 workgroups
    const int64_t blocks = p.rows / (16 * kF4Waves) * (a.D / 16);
    const int64_t each = std::max<int64_t>(1, blocks * units / 2048);
    const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>(ceil_div(blocks, each)));
    hipLaunchKernelGGL(k_fp4_attn_join_blocks, grid, dim3(kF4Threads), 0, s, a, p.rows, static_cast<int>(each));
    return;
  }
  const int64_t per = few ? 1 : std::min(block_rows, std::max<int64_t>(kF4Waves, ceil_div(units * block_rows, 8192)));
  const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>(ceil_div(block_rows, per)));
  const auto go = [&](auto* kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kF4Threads), 0, s, a, p.rows, static_cast<int>(per)); };
  if (p.shared) return go(&k_fp4_attn_join<kF4Threads, true>);
  if (few) return go(&k_fp4_attn_join<kF4Threads, false>);
  go(&k_fp4_attn_join<kWave, false>);
}

}  // namespace skv

using namespace skv;

extern "C" int64_t skv_fp4_attention_desc_size(void) { return static_cast<int64_t>(sizeof(skv_fp4_attention_desc)); }

extern "C" int64_t skv_fp4_attention_workspace(const skv_fp4_attention_desc* d) {
  Fp4AttnPlan p;
  return fp4_attn_plan(d, nullptr, p) == SKV_OK ? p.ws_bytes : -1;
}

extern "C" int skv_fp4_attention(const skv_fp4_attention_desc* d, void* workspace, int64_t ws_bytes, void* stream) {
  return fp4_attn_call<false>(d, nullptr, workspace, ws_bytes, stream);
}
