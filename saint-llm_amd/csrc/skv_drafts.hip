// A step's drafted tokens as a tree: what each of them sees, which of them the model accepts, and the accepted
// ones moved together in the 4-bit pages.
//
// Node t of a sequence's tree is the t-th of its newest tokens, parents[t] < t the node that it follows (-1: the
// tokens before the tree).
//   masks  : bit j of node t's words for itself and every ancestor j; its depth is their number less one.
//   accept : from node 0 on, the child whose token is the one that the model picked after its parent.
//   keep   : the tokens path[0] < path[1] < ... of the newest n become the newest k of them: path[i]'s row, in every
//            layer's pages, moves to row i of the n, the length is cut behind row k - 1 and the pages behind it go
//            on the free stack.
// All of it is the latency of a few dependent reads; MI355X: 64 trees of up to 64 nodes take 4.2 us for their masks, 5.5
// for their paths (320 nodes accepted), 8.4 for the plan of what is kept and 6.0 to move its rows (184 in each of 8 layers, 8
// heads of 128 dims); with longer paths (618 accepted, 482 moved, onto each other's places) 8.0, 8.5 and 8.7.
#include <algorithm>

#include "skv_fp4.h"

namespace skv {

constexpr int kDraftThreads = 256;
constexpr int kDraftMaxNodes = 1024;

// grid: batch.  A node's walk up the tree passes its bits from the last word to the first.
__global__ __launch_bounds__(kDraftThreads) void k_draft_tree(const int32_t* __restrict__ parents, const int32_t* __restrict__ n_new,
                                                              uint64_t* __restrict__ tree, int32_t* __restrict__ depths, int T,
                                                              int words) {
  __shared__ int32_t up[kDraftMaxNodes];
  const int64_t b = blockIdx.x;
  const int n = n_new ? min(max(n_new[b], 0), T) : T;
  for (int t = threadIdx.x; t < T; t += kDraftThreads) up[t] = parents[b * T + t];
  __syncthreads();
  for (int t = threadIdx.x; t < T; t += kDraftThreads) {
    uint64_t* out = tree + (b * T + t) * words;
    int depth = -1;
    if (t < n) {
      uint64_t bits = 0;
      int w = words - 1, j = t;
      for (;;) {
        for (; w > j >> 6; --w) {
          out[w] = bits;
          bits = 0;
        }
        bits |= 1ull << (j & 63);
        ++depth;
        const int p = up[j];
        if (p < 0 || p >= j) {
          if (p != -1) depth = -1;  // not an earlier node: t is none of a tree
          break;
        }
        j = p;
      }
      for (; w >= 0; --w) {
        out[w] = bits;
        bits = 0;
      }
    }
    if (depth < 0) {
      for (int w = 0; w < words; ++w) out[w] = 0;
    }
    depths[b * T + t] = max(depth, 0);
  }
}

// Token ids of either width.
struct DraftIds {
  const void* data;
  int64_t seq_stride, tok_stride;  // in ids
  int32_t wide;
  __device__ __forceinline__ int64_t at(int64_t b, int t) const {
    const int64_t i = b * seq_stride + t * tok_stride;
    return wide ? static_cast<const int64_t*>(data)[i] : static_cast<const int32_t*>(data)[i];
  }
};

// grid: batch; a wave.  A lane has the nodes lane, lane + 64, ...; a child comes after its parent.
__global__ __launch_bounds__(kWave) void k_accept_drafts(const int32_t* __restrict__ parents, DraftIds tokens, DraftIds picks,
                                                         const int32_t* __restrict__ n_new, int32_t* __restrict__ path,
                                                         int32_t* __restrict__ n_keep, void* __restrict__ next, int T) {
  __shared__ int32_t up[kDraftMaxNodes];
  __shared__ int64_t token[kDraftMaxNodes], pick[kDraftMaxNodes];
  const int64_t b = blockIdx.x;
  const int lane = threadIdx.x;
  const int n = n_new ? min(max(n_new[b], 0), T) : T;
  for (int t = lane; t < T; t += kWave) {
    up[t] = parents[b * T + t];
    token[t] = tokens.at(b, t);
    pick[t] = picks.at(b, t);
  }
  __syncthreads();
  int kept = 0, at = n > 0 ? 0 : -1;
  int64_t last = -1;
  while (at >= 0) {  // uniform; `at` grows
    if (lane == 0) path[b * T + kept] = at;
    ++kept;
    last = pick[at];
    int child = -1;
    for (int t0 = (at + 1) & ~(kWave - 1); t0 < n && child < 0; t0 += kWave) {
      const int t = t0 + lane;
      const uint64_t hit = __ballot(t > at && t < n && up[t] == at && token[t] == last);
      if (hit) child = t0 + __ffsll(static_cast<unsigned long long>(hit)) - 1;
    }
    at = child;
  }
  for (int t = kept + lane; t < T; t += kWave) path[b * T + t] = -1;
  if (lane == 0) {
    n_keep[b] = kept;
    if (picks.wide) {
      static_cast<int64_t*>(next)[b] = last;
    } else {
      static_cast<int32_t*>(next)[b] = static_cast<int32_t>(last);
    }
  }
}

constexpr int kKeepThreads = 1024;
constexpr int kKeepMax = 4096;  // sequences
constexpr int kKeepPools = 32;

struct KeepArgs {
  int32_t* stack;
  int32_t* top;
  int64_t n_pages;
  const int32_t* refs;  // or null
  int32_t* bt;
  int64_t bt_stride;
  int32_t* lens;
  const int32_t* n_new;
  int32_t n_uni;
  const int32_t* path;
  int64_t path_stride;
  const int32_t* n_keep;
  int batch, bs;
  int4* moves;  // [batch, path_stride]: a kept token's page and slot, from and to
  int32_t* status;
};

// One workgroup: checks every sequence, then the rows' places, the pages that are cut, and only when all are good
// writes the lengths, the tables and the stack.  The kept tokens and the cut pages of all sequences are numbered
// through by prefix sums, so that a round of loads serves 1024 of them.
__global__ __launch_bounds__(kKeepThreads) void k_keep_plan(KeepArgs a) {
  __shared__ int base[kKeepMax];         // positions before the newest tokens
  __shared__ int kept_at[kKeepMax + 1];  // kept tokens of the sequences before
  __shared__ int cut_at[kKeepMax + 1];   // pages past the new length's whole ones, of the sequences before
  __shared__ int free_at[kKeepMax + 1];  // of these those that are left without a token
  __shared__ int scan_lds[17];
  __shared__ int bad_all;
  const int tid = threadIdx.x;
  if (tid == 0) bad_all = 0;
  const int top = *a.top;
  int bad = top < 0 || top > a.n_pages ? SKV_STATUS_BADARG : 0;
  int kept_all = 0, cut_all = 0, free_all = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kKeepThreads) {
    const int b = b0 + tid;
    int k = 0, cut = 0, freed = 0;
    if (b < a.batch) {
      const int L = a.lens[b], n = a.n_new ? a.n_new[b] : a.n_uni;
      k = a.n_keep[b];
      if (L < 0 || L > a.bt_stride * a.bs || n < 0 || n > L || k < 0 || k > n || k > a.path_stride) {
        bad |= SKV_STATUS_BADARG;
        k = 0;
        base[b] = 0;
      } else {
        base[b] = L - n;
        const int left = L - n + k, held = static_cast<int>(ceil_div(L, a.bs));
        if (left < L) {
          cut = held - left / a.bs;
          freed = held - static_cast<int>(ceil_div(left, a.bs));
        }
      }
    }
    int tot;
    int ex = block_exclusive_scan(k, scan_lds, &tot);
    if (b < a.batch) kept_at[b] = kept_all + ex;
    kept_all += tot;
    ex = block_exclusive_scan(cut, scan_lds, &tot);
    if (b < a.batch) cut_at[b] = cut_all + ex;
    cut_all += tot;
    ex = block_exclusive_scan(freed, scan_lds, &tot);
    if (b < a.batch) free_at[b] = free_all + ex;
    free_all += tot;
  }
  if (tid == 0) {
    kept_at[a.batch] = kept_all;
    cut_at[a.batch] = cut_all;
    free_at[a.batch] = free_all;
  }
  if (!bad && top + static_cast<int64_t>(free_all) > a.n_pages) bad = SKV_STATUS_STACK;
  if (bad) atomicOr(&bad_all, bad);
  __syncthreads();
  // the sequence of item i
  const auto owner = [&](const int* at, int i) {
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (at[mid] <= i) lo = mid; else hi = mid - 1;
    }
    return lo;
  };
  const auto page_of = [&](int b, int j) { return a.bt[b * a.bt_stride + j]; };
  const auto good = [&](int32_t p) { return p >= 0 && p < a.n_pages; };
  if (!bad_all) {  // uniform
    for (int i = tid; i < kept_all; i += kKeepThreads) {
      const int b = owner(kept_at, i), k = i - kept_at[b];
      const int32_t* path = a.path + b * a.path_stride;
      const int n = a.n_new ? a.n_new[b] : a.n_uni, p = path[k], before = k > 0 ? path[k - 1] : -1;
      int4 move = make_int4(0, 0, 0, 0);
      if (p <= before || p >= n) {
        bad |= SKV_STATUS_BADARG;
      } else if (p != k) {
        const int src = base[b] + p, dst = base[b] + k;
        const int32_t sp = page_of(b, src / a.bs), dp = page_of(b, dst / a.bs);
        if (!good(sp) || !good(dp) || (a.refs && a.refs[dp] != 0)) {
          bad |= SKV_STATUS_BADARG;
        } else {
          move = make_int4(sp, src % a.bs, dp, dst % a.bs);
        }
      }
      a.moves[b * a.path_stride + k] = move;
    }
    for (int i = tid; i < cut_all; i += kKeepThreads) {
      const int b = owner(cut_at, i);
      const int left = base[b] + kept_at[b + 1] - kept_at[b];
      const int32_t p = page_of(b, left / a.bs + i - cut_at[b]);
      if (!good(p) || (a.refs && a.refs[p] != 0)) bad |= SKV_STATUS_BADARG;
    }
  }
  __syncthreads();  // bad_all has been read
  if (bad) atomicOr(&bad_all, bad);
  __syncthreads();
  if (bad_all) {
    if (tid == 0) *a.status = bad_all;
    return;
  }
  // sequences ascending, a sequence's pages from its last to its first
  for (int i = tid; i < free_all; i += kKeepThreads) {
    const int b = owner(free_at, i);
    const int left = base[b] + kept_at[b + 1] - kept_at[b];
    const int j = static_cast<int>(ceil_div(left, a.bs)) + free_at[b + 1] - 1 - i;
    a.stack[top + i] = page_of(b, j);
    a.bt[b * a.bt_stride + j] = -1;
  }
  for (int b = tid; b < a.batch; b += kKeepThreads) a.lens[b] = base[b] + kept_at[b + 1] - kept_at[b];
  if (tid == 0) {
    *a.top = top + free_all;
    *a.status = 0;
  }
}

struct KeepPools {
  uint8_t* base[kKeepPools];
};

constexpr int kKeepAhead = 8;  // rows of a column in flight

// A column of kept rows: Vec bytes of a plane of one head.  A thread moves all rows of it, in their order:
// row i goes to a place that is at most its own, so that no row is written over before it is read.
template <class Vec>
__device__ __forceinline__ void keep_column(uint8_t* head, int64_t page_bytes, int row_bytes, const int4* moves, int n) {
  for (int i0 = 0; i0 < n; i0 += kKeepAhead) {
    int4 m[kKeepAhead];
    Vec v[kKeepAhead];
#pragma unroll
    for (int i = 0; i < kKeepAhead; ++i) m[i] = moves[min(i0 + i, n - 1)];
#pragma unroll
    for (int i = 0; i < kKeepAhead; ++i) v[i] = *reinterpret_cast<const Vec*>(head + m[i].x * page_bytes + m[i].y * row_bytes);
#pragma unroll
    for (int i = 0; i < kKeepAhead; ++i) {
      if (i0 + i < n && (m[i].x != m[i].z || m[i].y != m[i].w)) {
        *reinterpret_cast<Vec*>(head + m[i].z * page_bytes + m[i].w * row_bytes) = v[i];
      }
    }
  }
}

// grid: (columns of all pools, batch).  A head's row has D / 32 columns of 16 bytes of the key's codes, as many of
// the value's, and `scale_cols` of the scale bytes, of the largest power of two that divides them.
__global__ __launch_bounds__(kDraftThreads) void k_keep_move(KeepArgs a, KeepPools pools, int n_pools, int heads, int dim, int scale_width) {
  if (*a.status != 0) return;  // refused: uniform
  const int b = blockIdx.y;
  const int n = a.n_keep[b];
  if (n == 0) return;
  const int codes = dim / 32, scales = dim / 16 / scale_width, columns = 2 * codes + scales;
  int c = blockIdx.x * kDraftThreads + threadIdx.x;
  const int q = c / (columns * heads);
  if (q >= n_pools) return;
  c -= q * columns * heads;
  const int h = c / columns;
  c -= h * columns;
  const Fp4Page pg = fp4_page(a.bs, heads, dim);
  uint8_t* head = pools.base[q] + h * pg.head;
  const int4* moves = a.moves + b * a.path_stride;
  if (c < 2 * codes) {
    const bool value = c >= codes;
    keep_column<u32x4>(head + (value ? pg.v_codes : 0) + 16 * (value ? c - codes : c), pg.page, dim / 2, moves, n);
    return;
  }
  head += pg.scales + (c - 2 * codes) * scale_width;
  if (scale_width == 16) keep_column<u32x4>(head, pg.page, dim / 16, moves, n);
  if (scale_width == 8) keep_column<u32x2>(head, pg.page, dim / 16, moves, n);
  if (scale_width == 4) keep_column<uint32_t>(head, pg.page, dim / 16, moves, n);
  if (scale_width == 2) keep_column<uint16_t>(head, pg.page, dim / 16, moves, n);
}

int check_tree(const char* what, int64_t batch, int64_t n_nodes) {
  if (batch < 0 || batch > 65535) return set_error(SKV_EINVAL, "%s: batch must be in [0, 65535]; got %lld", what, (long long)batch);
  if (n_nodes < 1 || n_nodes > kDraftMaxNodes) {
    return set_error(SKV_EINVAL, "%s: n_nodes must be in [1, %d]; got %lld", what, kDraftMaxNodes, (long long)n_nodes);
  }
  return SKV_OK;
}

}  // namespace skv

using namespace skv;

extern "C" int skv_draft_tree(const int32_t* parents, const int32_t* n_new, int64_t batch, int64_t n_nodes, uint64_t* tree,
                              int32_t* depths, void* stream) {
  const char* what = "skv_draft_tree";
  if (const int rc = check_tree(what, batch, n_nodes)) return rc;
  if (batch == 0) return SKV_OK;
  if (!parents || !tree || !depths) return set_error(SKV_EINVAL, "%s: NULL pointer", what);
  hipLaunchKernelGGL(k_draft_tree, dim3(static_cast<unsigned>(batch)), dim3(kDraftThreads), 0, static_cast<hipStream_t>(stream),
                     parents, n_new, tree, depths, static_cast<int>(n_nodes), static_cast<int>(ceil_div(n_nodes, 64)));
  return check_launch(what);
}

extern "C" int skv_accept_drafts(const int32_t* parents, const skv_token_ids* tokens, const skv_token_ids* picks,
                                 const int32_t* n_new, int64_t batch, int64_t n_nodes, int32_t* path, int32_t* n_keep, void* next,
                                 void* stream) {
  const char* what = "skv_accept_drafts";
  if (const int rc = check_tree(what, batch, n_nodes)) return rc;
  if (!tokens || !picks) return set_error(SKV_EINVAL, "%s: NULL pointer", what);
  if (batch == 0) return SKV_OK;
  if (!parents || !tokens->data || !picks->data || !path || !n_keep || !next) return set_error(SKV_EINVAL, "%s: NULL pointer", what);
  const DraftIds t{tokens->data, tokens->seq_stride, tokens->tok_stride, tokens->wide};
  const DraftIds p{picks->data, picks->seq_stride, picks->tok_stride, picks->wide};
  hipLaunchKernelGGL(k_accept_drafts, dim3(static_cast<unsigned>(batch)), dim3(kWave), 0, static_cast<hipStream_t>(stream), parents,
                     t, p, n_new, path, n_keep, next, static_cast<int>(n_nodes));
  return check_launch(what);
}

extern "C" int64_t skv_keep_tokens_workspace(int64_t batch, int64_t path_stride) {
  if (batch < 0 || batch > kKeepMax || path_stride < 1 || path_stride > kDraftMaxNodes) {
    return set_error(SKV_EINVAL, "skv_keep_tokens: batch must be in [0, %d], path_stride in [1, %d]; got %lld and %lld", kKeepMax,
                     kDraftMaxNodes, (long long)batch, (long long)path_stride), -1;
  }
  return batch * path_stride * 16;
}

extern "C" int skv_keep_tokens(int32_t* free_stack, int32_t* free_top, const int32_t* refs, const skv_fp4_cache* cache,
                               int32_t* block_table, int32_t* seq_lens, const int32_t* n_new, int32_t n_new_uniform,
                               const int32_t* path, int64_t path_stride, const int32_t* n_keep, void* const* pools,
                               int32_t n_pools, int32_t* status, void* workspace, int64_t ws_bytes, void* stream) {
  const char* what = "skv_keep_tokens";
  if (!cache) return set_error(SKV_EINVAL, "%s: NULL cache", what);
  const int64_t need = skv_keep_tokens_workspace(cache->batch, path_stride);
  if (need < 0) return SKV_EINVAL;
  skv_fp4_cache c = *cache;
  c.block_table = block_table;
  if (n_pools < 1 || n_pools > kKeepPools || !pools) {
    return set_error(SKV_EINVAL, "%s: n_pools must be in [1, %d]; got %d", what, kKeepPools, n_pools);
  }
  KeepPools kp{};
  for (int q = 0; q < n_pools; ++q) {
    c.pool = pools[q];
    if (const int rc = fp4_check_cache(&c, what)) return rc;
    kp.base[q] = static_cast<uint8_t*>(pools[q]);
  }
  if (c.batch * c.bt_stride > INT32_MAX) return set_error(SKV_EINVAL, "%s: block_table has more than 2^31 - 1 entries", what);
  if (!n_new && n_new_uniform < 0) return set_error(SKV_EINVAL, "%s: n_new_uniform must be >= 0", what);
  if (c.batch == 0) return SKV_OK;
  if (!free_stack || !free_top || !block_table || !seq_lens || !path || !n_keep || !status) {
    return set_error(SKV_EINVAL, "%s: NULL pointer", what);
  }
  if (!workspace || ws_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)) {
    return set_error(SKV_EINVAL, "%s: a 16-byte aligned workspace of %lld bytes is needed", what, (long long)need);
  }
  const KeepArgs a{free_stack, free_top, c.n_pages, refs, block_table, c.bt_stride, seq_lens, n_new, n_new_uniform, path, path_stride,
                   n_keep, static_cast<int>(c.batch), static_cast<int>(c.block_size), static_cast<int4*>(workspace), status};
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(k_keep_plan, dim3(1), dim3(kKeepThreads), 0, s, a);
  if (const int rc = check_launch(what)) return rc;
  const int heads = static_cast<int>(c.n_kv_heads), dim = static_cast<int>(c.head_dim), scale = dim / 16;
  const int width = std::min(16, scale & -scale);
  const int64_t columns = static_cast<int64_t>(n_pools) * heads * (dim / 16 + scale / width);
  hipLaunchKernelGGL(k_keep_move, dim3(static_cast<unsigned>(ceil_div(columns, kDraftThreads)), static_cast<unsigned>(c.batch)),
                     dim3(kDraftThreads), 0, s, a, kp, n_pools, heads, dim, width);
  return check_launch(what);
}
