// Eviction (release of finished sequences to the free list) and compaction
// (defragmenting copy of live pages + block-table rewrite).
//
// No reference counterpart: the reference keeps contiguous per-layer tensors
// (kv_cache.py:59-60) and plans a block layout and state cache only
// (saint_llm_inference/__init__.py:5-9).  Policies, fixed here and restated by
// the CPU oracle:
//   release : push order ascending sequence, within a sequence from its last
//             logical page to its first; released tables become -1, lengths 0.
//   compact : with n_live live pages, the live pages whose id is >= n_live
//             ("movers", ascending) move into the free ids < n_live ("holes",
//             ascending); other pages keep their ids.  Afterwards the live set
//             is exactly [0, n_live) and pops return n_live, n_live+1, ...
//             Sources are all >= n_live and destinations all < n_live, so the
//             page copies are independent and run fully in parallel.
#include <algorithm>

#include "skv_common.h"

namespace skv {

constexpr int kEvictThreads = 1024;
constexpr int kEvictMaxBatch = 4096;
constexpr int kMaxPools = 16;

__device__ __forceinline__ int owner_of(const int* off, int batch, int t) {
  int lo = 0, hi = batch;  // off[lo] <= t < off[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kEvictThreads) void k_release(
    int32_t* __restrict__ stack, int32_t* __restrict__ top_ptr, int64_t n_pages,
    int32_t* __restrict__ bt, int64_t bt_stride, int32_t* __restrict__ lens,
    const uint8_t* __restrict__ mask, int batch, int bs, int32_t* __restrict__ status) {
  __shared__ int off[kEvictMaxBatch + 1];
  __shared__ int cnt[kEvictMaxBatch];
  __shared__ int scan_lds[17];
  __shared__ int bad_all;
  const int tid = threadIdx.x;
  if (tid == 0) bad_all = 0;
  int carry = 0;
  for (int base = 0; base < batch; base += kEvictThreads) {
    const int b = base + tid;
    int c = 0;
    if (b < batch && mask[b]) {
      c = static_cast<int>(min<int64_t>(ceil_div(max(lens[b], 0), bs), bt_stride));
    }
    int tot;
    const int ex = block_exclusive_scan(c, scan_lds, &tot);
    if (b < batch) {
      off[b] = carry + ex;
      cnt[b] = c;
    }
    carry += tot;
  }
  if (tid == 0) off[batch] = carry;
  __syncthreads();
  const int top = *top_ptr;
  int bad = (top < 0 || static_cast<int64_t>(top) + carry > n_pages) ? SKV_STATUS_STACK : 0;
  for (int t = tid; t < carry && !bad; t += kEvictThreads) {
    const int b = owner_of(off, batch, t);
    const int32_t page = bt[static_cast<int64_t>(b) * bt_stride + (t - off[b])];
    if (page < 0 || page >= n_pages) bad = SKV_STATUS_BADARG;
  }
  if (bad) atomicOr(&bad_all, bad);
  __syncthreads();
  if (bad_all) {
    if (tid == 0 && status) *status = bad_all;
    return;
  }
  for (int t = tid; t < carry; t += kEvictThreads) {
    const int b = owner_of(off, batch, t);
    const int j = t - off[b];
    stack[top + off[b] + (cnt[b] - 1 - j)] = bt[static_cast<int64_t>(b) * bt_stride + j];
  }
  __syncthreads();  // every page id is read before the tables are cleared
  for (int t = tid; t < carry; t += kEvictThreads) {
    const int b = owner_of(off, batch, t);
    bt[static_cast<int64_t>(b) * bt_stride + (t - off[b])] = -1;
  }
  for (int b = tid; b < batch; b += kEvictThreads) {
    if (mask[b]) lens[b] = 0;
  }
  if (tid == 0) {
    *top_ptr = top + carry;
    if (status) *status = 0;
  }
}

// k_release over shared pages (refs[p]: holders beyond the first), in two launches.
//
// k_release_drop takes every released entry's page a holder: scattered atomics, which
// one CU does at 1.6 ns each and many do at once.  A page whose holders have all left
// is then at -1, one released more often than it was held below that.
//
// k_release_shared, one workgroup, checks that, pushes the pages at -1 and clears the
// tables, or gives the counts back.  Push order is ascending b, within b from the last
// logical page; of a page's releases the last place u pushes it, found by a minimum over
// -2 - u in the count itself, so that the stack does not depend on the order in which
// the atomics run.  A wave takes 64 entries of one sequence's table (a unit) at a time,
// kReleaseAhead of them together; a release of up to kReleaseStep units keeps its
// entries in registers from pass to pass.  Which entries' pages have dropped is noted
// for the first kReleaseNoted units, so that later passes touch those alone.  48 sequences
// of 8k - 64k tokens, 22,000 entries: 142 us with every entry by a thread in turn, 66 with
// units and all in one launch, 5 + 44 so; with 24 units together 36, but 27 instead of 13
// for a release of 1,600 entries.
constexpr int kReleaseAhead = 8;
constexpr int kReleaseStep = kEvictThreads / kWave * kReleaseAhead;
constexpr int kReleaseNoted = 1024;
constexpr int kDropThreads = 256;
constexpr int kDropEntries = 4 * kDropThreads;

__device__ __forceinline__ int released_pages(const int32_t* lens, const uint8_t* mask, int64_t bt_stride, int b, int bs) {
  return mask[b] ? static_cast<int>(min<int64_t>(ceil_div(max(lens[b], 0), bs), bt_stride)) : 0;
}

// grid: (parts of a table row, batch)
__global__ __launch_bounds__(kDropThreads) void k_release_drop(int64_t n_pages, int32_t* refs, const int32_t* __restrict__ bt,
                                                               int64_t bt_stride, const int32_t* __restrict__ lens,
                                                               const uint8_t* __restrict__ mask, int bs) {
  const int b = blockIdx.y, n = released_pages(lens, mask, bt_stride, b, bs);
#pragma unroll
  for (int k = 0; k < kDropEntries / kDropThreads; ++k) {
    const int64_t j = static_cast<int64_t>(blockIdx.x) * kDropEntries + k * kDropThreads + static_cast<int>(threadIdx.x);
    if (j >= n) return;
    const int32_t page = bt[b * bt_stride + j];
    if (page >= 0 && page < n_pages) atomicSub(&refs[page], 1);
  }
}

__global__ __launch_bounds__(kEvictThreads) void k_release_shared(
    int32_t* __restrict__ stack, int32_t* __restrict__ top_ptr, int64_t n_pages, int32_t* refs, int32_t* bt,
    int64_t bt_stride, int32_t* __restrict__ lens, const uint8_t* __restrict__ mask, int batch, int bs,
    int32_t* __restrict__ status) {
  __shared__ int off[kEvictMaxBatch + 1];  // units before each sequence
  __shared__ int cnt[kEvictMaxBatch];      // its pages
  __shared__ uint64_t noted[kReleaseNoted];
  __shared__ int scan_lds[17];
  __shared__ int bad_all;
  const int tid = threadIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  if (tid == 0) bad_all = 0;
  int units = 0;
  for (int base = 0; base < batch; base += kEvictThreads) {
    const int b = base + tid, c = b < batch ? released_pages(lens, mask, bt_stride, b, bs) : 0;
    int tot;
    const int ex = block_exclusive_scan((c + kWave - 1) / kWave, scan_lds, &tot);
    if (b < batch) {
      off[b] = units + ex;
      cnt[b] = c;
    }
    units += tot;
  }
  if (tid == 0) off[batch] = units;
  __syncthreads();
  const int top = *top_ptr;
  // all of them loaded before any is used: else each load sinks into its use's branch
  const auto together = [](int32_t* x) {
    static_assert(kReleaseAhead % 8 == 0);
#pragma unroll
    for (int k = 0; k < kReleaseAhead; k += 8) {
      asm volatile("" : "+v"(x[k]), "+v"(x[k + 1]), "+v"(x[k + 2]), "+v"(x[k + 3]), "+v"(x[k + 4]), "+v"(x[k + 5]),
                        "+v"(x[k + 6]), "+v"(x[k + 7]));
    }
  };
  // the thread's entries of the step from unit `at` on: places (-1: no entry), indices in the table, page ids
  int at = -1, first = 0, u[kReleaseAhead];
  int entry[kReleaseAhead];
  int32_t page[kReleaseAhead];
  // f() for every step; all threads take the same steps
  const auto steps = [&](auto&& f) {
    for (int base = 0; base < units; base += kReleaseStep) {
      if (at != base) {
        at = base;
        first = base + wave * kReleaseAhead;
        int b = first < units ? owner_of(off, batch, first) : 0;
#pragma unroll
        for (int k = 0; k < kReleaseAhead; ++k) {
          u[k] = -1;
          entry[k] = 0;
          if (first + k < units) {  // uniform
            while (first + k >= off[b + 1]) ++b;
            const int j = (first + k - off[b]) * kWave + lane;
            if (j < cnt[b]) {
              u[k] = (first + k) * kWave + lane;
              entry[k] = static_cast<int>(b * bt_stride) + cnt[b] - 1 - j;
            }
          }
        }
#pragma unroll
        for (int k = 0; k < kReleaseAhead; ++k) page[k] = bt[entry[k]];
        together(page);
      }
      f();
    }
  };
  // of the k-th entries those that may have a noted property (past the noted units: any)
  const auto may = [&](int k) {
    return u[k] >= 0 && (first + k >= kReleaseNoted || ((noted[min(first + k, kReleaseNoted - 1)] >> lane) & 1));
  };
  const auto note = [&](int k, bool yes) {
    const uint64_t lanes = __ballot(yes);
    if (lane == 0 && first + k < kReleaseNoted) noted[first + k] = lanes;
    return lanes;
  };
  const auto known = [&](int k) { return u[k] >= 0 && page[k] >= 0 && page[k] < n_pages; };
  const auto counts = [&](const bool* ask, int32_t* count) {
#pragma unroll
    for (int k = 0; k < kReleaseAhead; ++k) count[k] = refs[ask[k] ? page[k] : 0];
    together(count);
  };
  const auto refuse = [&](int bad) {  // the whole workgroup's answer
    if (bad) atomicOr(&bad_all, bad);
    __syncthreads();
    if (!bad_all) return false;
    if (tid == 0 && status) *status = bad_all;
    steps([&] {  // the counts as they were
#pragma unroll
      for (int k = 0; k < kReleaseAhead; ++k) {
        if (known(k)) atomicAdd(&refs[page[k]], 1);
      }
    });
    return true;
  };
  int bad = (top < 0 || top > n_pages) ? SKV_STATUS_STACK : 0;
  steps([&] {
    bool ask[kReleaseAhead];
    int32_t count[kReleaseAhead];
#pragma unroll
    for (int k = 0; k < kReleaseAhead; ++k) ask[k] = known(k);
    counts(ask, count);
#pragma unroll
    for (int k = 0; k < kReleaseAhead; ++k) {
      if (u[k] >= 0 && (!ask[k] || count[k] < -1)) bad = SKV_STATUS_BADARG;
      note(k, ask[k] && count[k] < 0);
    }
  });
  if (refuse(bad)) return;
  // between a pass that changes counts and one that reads them: the changes have been
  // made, and the L1 cache holds no count
  const auto fresh = [] {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  };
  steps([&] {
#pragma unroll
    for (int k = 0; k < kReleaseAhead; ++k) {
      if (may(k) && (first + k < kReleaseNoted || refs[page[k]] < 0)) atomicMin(&refs[page[k]], -2 - u[k]);
    }
  });
  fresh();
  int mine = 0;  // pages that the wave will push
  steps([&] {
    bool ask[kReleaseAhead];
    int32_t count[kReleaseAhead];
#pragma unroll
    for (int k = 0; k < kReleaseAhead; ++k) ask[k] = may(k);
    counts(ask, count);
#pragma unroll
    for (int k = 0; k < kReleaseAhead; ++k) mine += __popcll(note(k, ask[k] && count[k] == -2 - u[k]));
  });
  const int pushes = block_reduce_sum(lane == 0 ? mine : 0, scan_lds);
  const bool full = static_cast<int64_t>(top) + pushes > n_pages;
  if (full) {  // uniform: the places leave the counts again
    steps([&] {
#pragma unroll
      for (int k = 0; k < kReleaseAhead; ++k) {
        if (may(k) && refs[page[k]] == -2 - u[k]) refs[page[k]] = -1;
      }
    });
    fresh();
  }
  if (refuse(full ? SKV_STATUS_STACK : 0)) return;
  int to = top;
  steps([&] {
    uint64_t push[kReleaseAhead];
    int n = 0;  // the wave's
#pragma unroll
    for (int k = 0; k < kReleaseAhead; ++k) {
      push[k] = __ballot(may(k) && (first + k < kReleaseNoted || refs[page[k]] == -2 - u[k]));
      n += __popcll(push[k]);
    }
    int tot;
    const int ex = block_exclusive_scan(lane == 0 ? n : 0, scan_lds, &tot);
    int slot = to + __builtin_amdgcn_readfirstlane(ex);
#pragma unroll
    for (int k = 0; k < kReleaseAhead; ++k) {
      if ((push[k] >> lane) & 1) {
        stack[slot + __popcll(push[k] & ((uint64_t{1} << lane) - 1))] = page[k];
        refs[page[k]] = 0;
      }
      slot += __popcll(push[k]);
      if (u[k] >= 0) bt[entry[k]] = -1;  // read by this thread alone
    }
    to += tot;
  });
  for (int b = tid; b < batch; b += kEvictThreads) {
    if (mask[b]) lens[b] = 0;
  }
  if (tid == 0) {
    *top_ptr = top + pushes;
    if (status) *status = 0;
  }
}

// ---- compaction -------------------------------------------------------------
// The pools of a copy launch, or the parts of their pages that it copies: page_bytes
// from page to page, part_bytes of each from base on.
struct PoolRefs {
  uint8_t* base[kMaxPools];
  int64_t page_bytes[kMaxPools], part_bytes[kMaxPools];
  int n;
};

// The plan runs one workgroup per block of kPlanSpan page ids.  A count
// launch before it writes the live pages of every block (counts: the last
// n_blocks words of the workspace, which the movers' list never reaches:
// n_moved <= n / 2), so that each plan workgroup knows how many live pages
// precede its block without waiting for another workgroup.
constexpr int kPlanPer = 4;                          // ids per thread: one 16-byte load of marks
constexpr int kPlanShift = 12;
constexpr int kPlanSpan = 1 << kPlanShift;           // ids per plan workgroup
static_assert(kPlanSpan == kEvictThreads * kPlanPer, "a plan workgroup covers its block in one pass");

__host__ __device__ __forceinline__ int64_t plan_blocks(int64_t n) { return (n + kPlanSpan - 1) >> kPlanShift; }

// grid: (ceil(bt_stride / 256), batch)
__global__ void k_mark_live(const int32_t* __restrict__ bt, int64_t bt_stride,
                            const int32_t* __restrict__ lens, int bs, int64_t n_pages,
                            int32_t* __restrict__ mark) {
  const int b = blockIdx.y;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t np = min<int64_t>(ceil_div(max(lens[b], 0), bs), bt_stride);
  if (j >= np) return;
  const int32_t p = bt[b * bt_stride + j];
  if (p >= 0 && p < n_pages) mark[p] = 1;
}

// The marks of ids [i0, i0 + kPlanPer) (0 past n).
__device__ __forceinline__ void load_run(const int32_t* mark, int64_t i0, int64_t n, int* v) {
  if (i0 + kPlanPer <= n) {  // whole run in range: one 16-byte load (i0 is a multiple of 4)
    const int4 w = *reinterpret_cast<const int4*>(mark + i0);
    v[0] = w.x;
    v[1] = w.y;
    v[2] = w.z;
    v[3] = w.w;
  } else {
#pragma unroll
    for (int k = 0; k < kPlanPer; ++k) v[k] = (i0 + k < n) ? mark[i0 + k] : 0;
  }
}

// Workgroup g writes the live pages of ids [g * kPlanSpan, (g + 1) * kPlanSpan).
__global__ __launch_bounds__(kEvictThreads) void k_count_live(const int32_t* __restrict__ mark, int64_t n,
                                                              int32_t* __restrict__ counts) {
  __shared__ int scan_lds[17];
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kPlanSpan + static_cast<int64_t>(threadIdx.x) * kPlanPer;
  int v[kPlanPer];
  load_run(mark, i0, n, v);
  int c = 0;
#pragma unroll
  for (int k = 0; k < kPlanPer; ++k) c += (v[k] != 0) ? 1 : 0;
  c = block_reduce_sum(c, scan_lds);
  if (threadIdx.x == 0) counts[blockIdx.x] = c;
}

// Workgroup g: ids [g * kPlanSpan, (g + 1) * kPlanSpan).
// ws: [0, n) marks -> movers' ranks, [n, 2n) holes, [2n, 3n) movers; counts
// as above.  A hole's rank is the number of holes before it (its id less the
// live pages before it); a mover's rank is the number of live pages in
// [n_live, id), i.e. the live pages before it less those before n_live.
// A mover's mark becomes its rank, which the copy launch's table rewrite
// reads and clears; the copy launch also clears the marks below n_live (other
// plan workgroups read them here), so words [0, n) are zero again after the
// compaction.  The free stack is rebuilt so that pops return
// n_live, n_live + 1, ...; info = {n_live, n_moved} (workgroup 0).
__global__ __launch_bounds__(kEvictThreads) void k_compact_plan(int32_t* __restrict__ ws, int64_t n,
                                                                int32_t* __restrict__ stack,
                                                                int32_t* __restrict__ top_ptr,
                                                                int32_t* __restrict__ info) {
  __shared__ int scan_lds[17];
  const int tid = threadIdx.x;
  const int g = blockIdx.x;
  const int n_blocks = static_cast<int>(plan_blocks(n));
  int32_t* mark = ws;
  int32_t* holes = ws + n;
  int32_t* movers = ws + 2 * n;
  const int32_t* counts = ws + 3 * n - n_blocks;
  // every load of the first round trip: the block counts and this block's marks
  constexpr int kCntPer = (1 << 24) / kPlanSpan / kEvictThreads;  // n < 2^24 pages
  int cnt[kCntPer];
#pragma unroll
  for (int k = 0; k < kCntPer; ++k) {
    const int i = tid + k * kEvictThreads;
    cnt[k] = (i < n_blocks) ? counts[i] : 0;
  }
  const int64_t i0 = static_cast<int64_t>(g) * kPlanSpan + static_cast<int64_t>(tid) * kPlanPer;
  int v[kPlanPer];
  load_run(mark, i0, n, v);
  int total = 0, before = 0;
#pragma unroll
  for (int k = 0; k < kCntPer; ++k) {
    total += cnt[k];
    before += (tid + k * kEvictThreads < g) ? cnt[k] : 0;
  }
  const int64_t n_live = block_reduce_sum(total, scan_lds);
  before = block_reduce_sum(before, scan_lds);
  // live pages before n_live: the blocks before its block, then that block up to n_live
  const int gs = static_cast<int>(n_live >> kPlanShift);
  int pre = 0;
#pragma unroll
  for (int k = 0; k < kCntPer; ++k) pre += (tid + k * kEvictThreads < gs) ? cnt[k] : 0;
  int w[kPlanPer];
  const int64_t j0 = static_cast<int64_t>(gs) * kPlanSpan + static_cast<int64_t>(tid) * kPlanPer;
  load_run(mark, j0, n_live, w);
#pragma unroll
  for (int k = 0; k < kPlanPer; ++k) pre += (w[k] != 0) ? 1 : 0;
  const int live_below = block_reduce_sum(pre, scan_lds);  // live pages with id < n_live
  const int n_moved = static_cast<int>(n_live) - live_below;
  // this block's ids
  int c = 0;
#pragma unroll
  for (int k = 0; k < kPlanPer; ++k) c += (v[k] != 0) ? 1 : 0;
  int tot;
  int lb = before + block_exclusive_scan(c, scan_lds, &tot);  // live pages before id i0
#pragma unroll
  for (int k = 0; k < kPlanPer; ++k) {
    const int64_t i = i0 + k;
    if (i >= n) break;
    const bool live = v[k] != 0;
    if (i < n_live) {
      if (!live) holes[i - lb] = static_cast<int32_t>(i);
    } else {
      if (live) {
        const int r = lb - live_below;
        movers[r] = static_cast<int32_t>(i);
        mark[i] = r;
      }
      stack[n - 1 - i] = static_cast<int32_t>(i);
    }
    lb += live ? 1 : 0;
  }
  if (g == 0 && tid == 0) {
    *top_ptr = static_cast<int32_t>(n - n_live);
    info[0] = static_cast<int32_t>(n_live);
    info[1] = n_moved;
  }
}

constexpr int kCompactCopyThreads = 256;
constexpr int kCopySlice = kCompactCopyThreads * 16;  // bytes per copy slice: 16 per thread
constexpr int kCopySlices = 8;                        // slices per workgroup per iteration

// Slices of the page copies: mover rank r owns slices [r * per_mover, (r+1) *
// per_mover); slices [first[q], first[q+1]) of a mover are pool q's page.
struct CopySlices {
  int32_t first[kMaxPools + 1];
  int32_t per_mover;
};

// Persistent grid over 4 KB slices of (mover, pool) pages.  A workgroup takes
// kCopySlices slices per iteration, all loads issued before any store; the
// hole / mover ids of its next iteration are loaded before this iteration's
// stores, so only the first iteration waits for them.  The same grid first
// rewrites the block tables (every table entry of a live page at or above
// n_live takes the hole of its rank, which it then clears) and clears the
// plan's marks below n_live.  Slices are counted below 2^24: more of them are
// copied by more launches, which come with no table (batch 0).
struct TableRef {
  int32_t* bt;
  const int32_t* lens;
  int32_t bt_stride;
  int32_t batch;
  int32_t block_size;
};

__device__ __forceinline__ void slice_ids(const CopySlices& cs, const int32_t* movers, const int32_t* holes,
                                          int s0, int total, int32_t* src_id, int32_t* dst_id) {
#pragma unroll
  for (int k = 0; k < kCopySlices; ++k) {
    const int s = min(s0 + k, total - 1);
    const int r = static_cast<int>(udiv24(s, cs.per_mover));
    src_id[k] = movers[r];
    dst_id[k] = holes[r];
  }
}

// kShared: several tables may hold a page, so the rewrite leaves the marks to
// k_compact_finish.
template <bool kShared>
__global__ __launch_bounds__(kCompactCopyThreads) void k_compact_copy(PoolRefs pools, CopySlices cs, TableRef tr,
                                                                     int32_t* __restrict__ ws, int64_t n,
                                                                     const int32_t* __restrict__ info) {
  const int n_live = info[0];
  const int n_moved = info[1];
  int32_t* remap = ws;
  const int32_t* holes = ws + n;
  const int32_t* movers = ws + 2 * n;
  const int total = n_moved * cs.per_mover;  // < 2^24 (checked on the host)
  // the moved pages' stores: plain (allocating) stores when the move writes
  // 96-256 MiB, where the written pages stay in the 256 MiB last-level
  // cache (fp8 1M-token pools: 227 MiB moved, 115 -> 104 us per release +
  // compaction on MI355X), nontemporal stores otherwise (the same limits as
  // the decode gather's rows)
  const int64_t moved_bytes = static_cast<int64_t>(total) * kCopySlice;
  const bool wb = moved_bytes >= (static_cast<int64_t>(96) << 20) && moved_bytes <= (static_cast<int64_t>(256) << 20);
  const int tid = threadIdx.x;
  const int gtid = blockIdx.x * kCompactCopyThreads + tid;
  const int gsize = gridDim.x * kCompactCopyThreads;
  int s0 = blockIdx.x * kCopySlices;
  int32_t src_id[kCopySlices], dst_id[kCopySlices];
  if (s0 < total) slice_ids(cs, movers, holes, s0, total, src_id, dst_id);  // in flight during the rewrite
  const int entries = tr.batch * tr.bt_stride;  // <= 2^30 (checked on the host)
  const bool far = entries >= 1 << 24;
  for (int t = gtid; t < entries; t += gsize) {
    const int b = far ? t / tr.bt_stride : static_cast<int>(udiv24(t, tr.bt_stride));
    const int j = t - b * tr.bt_stride;
    const int np = static_cast<int>(min<int64_t>(ceil_div24(max(tr.lens[b], 0), tr.block_size), tr.bt_stride));
    if (j < np) {
      const int32_t p = tr.bt[t];
      if (p >= n_live && p < n) {
        tr.bt[t] = holes[remap[p]];
        if constexpr (!kShared) remap[p] = 0;
      }
    }
  }
  if constexpr (!kShared) {
    for (int i = gtid; i < n_live; i += gsize) remap[i] = 0;
  }
  for (; s0 < total; s0 += gridDim.x * kCopySlices) {
    int q_of[kCopySlices], off[kCopySlices];
#pragma unroll
    for (int k = 0; k < kCopySlices; ++k) {
      const int s = min(s0 + k, total - 1);
      const int r = static_cast<int>(udiv24(s, cs.per_mover));
      const int j = s - r * cs.per_mover;
      int q = 0;
      for (int qq = 1; qq < pools.n; ++qq) q += (j >= cs.first[qq]) ? 1 : 0;
      q_of[k] = q;
      off[k] = (j - cs.first[q]) * kCopySlice + tid * 16;
    }
    u32x4 v[kCopySlices];
#pragma unroll
    for (int k = 0; k < kCopySlices; ++k) {
      const int64_t pb = pools.page_bytes[q_of[k]];
      const bool live = s0 + k < total && off[k] < pools.part_bytes[q_of[k]];
      const uint8_t* src = pools.base[q_of[k]] + static_cast<int64_t>(src_id[k]) * pb + (live ? off[k] : 0);
      v[k] = ld_stream(reinterpret_cast<const u32x4*>(src));
    }
    int32_t next_src[kCopySlices], next_dst[kCopySlices];
    const int s1 = s0 + gridDim.x * kCopySlices;
    if (s1 < total) slice_ids(cs, movers, holes, s1, total, next_src, next_dst);
#pragma unroll
    for (int k = 0; k < kCopySlices; ++k) {
      const int64_t pb = pools.page_bytes[q_of[k]];
      if (s0 + k < total && off[k] < pools.part_bytes[q_of[k]]) {
        u32x4* dst = reinterpret_cast<u32x4*>(pools.base[q_of[k]] + static_cast<int64_t>(dst_id[k]) * pb + off[k]);
        if (wb) {
          *dst = v[k];
        } else {
          st_stream(dst, v[k]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kCopySlices; ++k) {
      src_id[k] = next_src[k];
      dst_id[k] = next_dst[k];
    }
  }
}

// Clears the marks and moves the counts of the pages that moved.
__global__ __launch_bounds__(kCompactCopyThreads) void k_compact_finish(int32_t* __restrict__ ws, int64_t n,
                                                                       const int32_t* __restrict__ info,
                                                                       int32_t* __restrict__ refs) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kCompactCopyThreads + threadIdx.x;
  if (i >= n) return;
  ws[i] = 0;
  if (i < info[1]) {
    const int32_t hole = ws[n + i], mover = ws[2 * n + i];
    refs[hole] = refs[mover];
    refs[mover] = 0;
  }
}

}  // namespace skv

using namespace skv;

extern "C" int skv_release(int32_t* free_stack, int32_t* free_top, int64_t n_pages,
                           int32_t* block_table, int64_t bt_stride, int32_t* seq_lens,
                           const uint8_t* release_mask, int64_t batch, int64_t block_size,
                           int32_t* status, void* stream) {
  if (batch < 0 || batch > kEvictMaxBatch) {
    return set_error(SKV_EINVAL, "skv_release: batch must be in [0, %d]; got %lld", kEvictMaxBatch,
                     (long long)batch);
  }
  if (block_size <= 0 || bt_stride <= 0 || n_pages <= 0 || n_pages > INT32_MAX) {
    return set_error(SKV_EINVAL, "skv_release: bad block_size/bt_stride/n_pages");
  }
  if (!release_mask) return set_error(SKV_EINVAL, "skv_release: release_mask is NULL");
  if (batch == 0) return SKV_OK;
  hipLaunchKernelGGL(k_release, dim3(1), dim3(kEvictThreads), 0, static_cast<hipStream_t>(stream),
                     free_stack, free_top, n_pages, block_table, bt_stride, seq_lens, release_mask,
                     static_cast<int>(batch), static_cast<int>(block_size), status);
  return check_launch("skv_release");
}

extern "C" int skv_release_shared(int32_t* free_stack, int32_t* free_top, int64_t n_pages, int32_t* refs,
                                  int32_t* block_table, int64_t bt_stride, int32_t* seq_lens,
                                  const uint8_t* release_mask, int64_t batch, int64_t block_size, int32_t* status,
                                  void* stream) {
  const char* what = "skv_release_shared";
  if (batch < 0 || batch > kEvictMaxBatch) {
    return set_error(SKV_EINVAL, "%s: batch must be in [0, %d]; got %lld", what, kEvictMaxBatch, (long long)batch);
  }
  if (block_size <= 0 || block_size > INT32_MAX || bt_stride <= 0 || n_pages <= 0 || n_pages > INT32_MAX ||
      batch * (bt_stride + kWave) > INT32_MAX - kEvictThreads) {
    return set_error(SKV_EINVAL, "%s: bad block_size/bt_stride/n_pages", what);
  }
  if (!free_stack || !free_top || !refs || (batch > 0 && (!block_table || !seq_lens || !release_mask))) {
    return set_error(SKV_EINVAL, "%s: NULL pointer", what);
  }
  if (batch == 0) return SKV_OK;
  hipLaunchKernelGGL(k_release_drop, dim3(static_cast<unsigned>(ceil_div(bt_stride, kDropEntries)), static_cast<unsigned>(batch)),
                     dim3(kDropThreads), 0, static_cast<hipStream_t>(stream), n_pages, refs, block_table, bt_stride, seq_lens,
                     release_mask, static_cast<int>(block_size));
  if (const int rc = check_launch(what)) return rc;
  hipLaunchKernelGGL(k_release_shared, dim3(1), dim3(kEvictThreads), 0, static_cast<hipStream_t>(stream), free_stack,
                     free_top, n_pages, refs, block_table, bt_stride, seq_lens, release_mask, static_cast<int>(batch),
                     static_cast<int>(block_size), status);
  return check_launch(what);
}

// The launches of skv_compact and, with refs, skv_compact_shared.
static int compact(const char* what, const skv_pool_ref* pools, int32_t n_pools, int32_t* block_table, int64_t bt_stride,
                   const int32_t* seq_lens, int64_t batch, int64_t block_size, int64_t n_pages, int32_t* free_stack,
                   int32_t* free_top, int32_t* refs, int32_t* workspace, int32_t* info, void* stream) {
  if (n_pools < 1 || n_pools > kMaxPools || !pools) {
    return set_error(SKV_EINVAL, "%s: n_pools must be in [1, %d]; got %d", what, kMaxPools, n_pools);
  }
  if (batch < 0 || batch > 65535 || block_size <= 0 || bt_stride <= 0 || n_pages <= 0 ||
      n_pages > INT32_MAX) {
    return set_error(SKV_EINVAL, "%s: bad batch/block_size/bt_stride/n_pages", what);
  }
  if (!workspace || !info || !free_stack || !free_top) {
    return set_error(SKV_EINVAL, "%s: NULL workspace/info/free list", what);
  }
  for (int q = 0; q < n_pools; ++q) {
    if (!pools[q].base || pools[q].page_bytes <= 0 || (pools[q].page_bytes & 15) ||
        (reinterpret_cast<uintptr_t>(pools[q].base) & 15)) {
      return set_error(SKV_EINVAL, "%s: pool %d needs a 16-byte aligned base and page_bytes", what, q);
    }
  }
  if (n_pages >= (1 << 24)) return set_error(SKV_EINVAL, "%s: n_pages must stay below 2^24", what);
  if (bt_stride > (1 << 30) || batch * bt_stride > (1 << 30)) {
    return set_error(SKV_EINVAL, "%s: batch x bt_stride must be at most 2^30", what);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  int rc;
  const dim3 tgrid(static_cast<unsigned>(ceil_div(bt_stride, 256)), static_cast<unsigned>(batch));
  if (batch > 0) {
    hipLaunchKernelGGL(k_mark_live, tgrid, dim3(256), 0, s, block_table, bt_stride, seq_lens,
                       static_cast<int>(block_size), n_pages, workspace);
    if ((rc = check_launch(what))) return rc;
  }
  const dim3 pgrid(static_cast<unsigned>(plan_blocks(n_pages)));
  hipLaunchKernelGGL(k_count_live, pgrid, dim3(kEvictThreads), 0, s, workspace, n_pages,
                     workspace + 3 * n_pages - plan_blocks(n_pages));
  if ((rc = check_launch(what))) return rc;
  hipLaunchKernelGGL(k_compact_plan, pgrid, dim3(kEvictThreads), 0, s, workspace, n_pages,
                     free_stack, free_top, info);
  if ((rc = check_launch(what))) return rc;
  const TableRef tables{block_table, seq_lens, static_cast<int32_t>(bt_stride), static_cast<int32_t>(batch),
                        static_cast<int32_t>(block_size)};
  const int64_t per_launch = std::min<int64_t>(((1 << 24) - 1) / n_pages, 1 << 18);  // slices of a page: 1 GB at most
  int64_t done = 0;  // bytes of pool q's page
  for (int q = 0; q < n_pools;) {
    const bool first = q == 0 && done == 0;
    PoolRefs pr{};
    CopySlices cs{};
    for (; q < n_pools && cs.per_mover < per_launch; ++pr.n) {
      const int64_t left = pools[q].page_bytes - done;
      const int64_t slices = std::min<int64_t>(ceil_div(left, kCopySlice), per_launch - cs.per_mover);
      pr.base[pr.n] = static_cast<uint8_t*>(pools[q].base) + done;
      pr.page_bytes[pr.n] = pools[q].page_bytes;
      pr.part_bytes[pr.n] = std::min(left, slices * kCopySlice);
      cs.per_mover += static_cast<int32_t>(slices);
      cs.first[pr.n + 1] = cs.per_mover;
      done += pr.part_bytes[pr.n];
      if (done == pools[q].page_bytes) {
        done = 0;
        ++q;
      }
    }
    TableRef tr = tables;
    if (!first) tr.batch = 0;
    if (refs || !first) {
      hipLaunchKernelGGL((k_compact_copy<true>), dim3(kPersistentBlocks), dim3(kCompactCopyThreads), 0, s, pr, cs, tr,
                         workspace, n_pages, info);
    } else {
      hipLaunchKernelGGL((k_compact_copy<false>), dim3(kPersistentBlocks), dim3(kCompactCopyThreads), 0, s, pr, cs, tr,
                         workspace, n_pages, info);
    }
    if ((rc = check_launch(what))) return rc;
  }
  if (!refs) return SKV_OK;
  hipLaunchKernelGGL(k_compact_finish, dim3(static_cast<unsigned>(ceil_div(n_pages, kCompactCopyThreads))),
                     dim3(kCompactCopyThreads), 0, s, workspace, n_pages, info, refs);
  return check_launch(what);
}

extern "C" int skv_compact(const skv_pool_ref* pools, int32_t n_pools, int32_t* block_table,
                           int64_t bt_stride, const int32_t* seq_lens, int64_t batch,
                           int64_t block_size, int64_t n_pages, int32_t* free_stack,
                           int32_t* free_top, int32_t* workspace, int32_t* info, void* stream) {
  return compact("skv_compact", pools, n_pools, block_table, bt_stride, seq_lens, batch, block_size, n_pages, free_stack,
                 free_top, nullptr, workspace, info, stream);
}

extern "C" int skv_compact_shared(const skv_pool_ref* pools, int32_t n_pools, int32_t* block_table, int64_t bt_stride,
                                  const int32_t* seq_lens, int64_t batch, int64_t block_size, int64_t n_pages,
                                  int32_t* free_stack, int32_t* free_top, int32_t* refs, int32_t* workspace,
                                  int32_t* info, void* stream) {
  const char* what = "skv_compact_shared";
  if (!refs) return set_error(SKV_EINVAL, "%s: refs is NULL", what);
  return compact(what, pools, n_pools, block_table, bt_stride, seq_lens, batch, block_size, n_pages, free_stack,
                 free_top, refs, workspace, info, stream);
}
