// Forking sequences onto shared pages: whole pages are shared by a count of
// their holders, the last, begun page is copied.  (skv_evict.hip frees and
// compacts shared pages.)
//
// A page is shared only when it is whole, and appends write behind the whole
// pages, so that no shared page is ever written: a fork needs no copy on write.
//
// Two launches: one workgroup checks the forks and pops the pages (4 us, a chain of
// round trips), then table rows, counts and pages are copied by as many workgroups as
// they have slices (48 forks of 8k - 64k tokens in 8 pools: 22,000 entries and 13 MB in
// 8 us, of the counts' atomics).
#include <algorithm>

#include "skv_common.h"

namespace skv {

constexpr int kForkThreads = 1024;
constexpr int kForkMax = 4096;  // sequences, and forks of a call
constexpr int kForkPools = 32;  // 16 layers of two streams

struct ForkArgs {
  int32_t* stack;
  int32_t* top;
  int64_t n_pages;
  int32_t* refs;
  int32_t* bt;
  int64_t bt_stride;
  int32_t* lens;
  const int32_t* src;
  const int32_t* dst;
  int batch, bs, n;
  int32_t* status;
};

// One workgroup: checks the forks, pops a page for every begun one in the
// forks' order and writes it and the length.  The copy launch finds the page
// in dst's table.
__global__ __launch_bounds__(kForkThreads) void k_fork_plan(ForkArgs a) {
  __shared__ int len[kForkMax];    // of each fork's source
  __shared__ int page[kForkMax];   // rank of its page among the popped, then the page; -1 none
  __shared__ int taken[kForkMax];  // sequences that a fork goes to
  __shared__ int scan_lds[17];
  __shared__ int bad_all;
  const int tid = threadIdx.x;
  if (tid == 0) bad_all = 0;
  for (int b = tid; b < a.batch; b += kForkThreads) taken[b] = 0;
  __syncthreads();
  const int top = *a.top;
  int bad = (top < 0 || top > a.n_pages) ? SKV_STATUS_BADARG : 0;
  int carry = 0;
  for (int base = 0; base < a.n; base += kForkThreads) {
    const int f = base + tid;
    int need = 0;
    if (f < a.n) {
      const int s = a.src[f], d = a.dst[f];
      int L = 0;
      if (s < 0 || s >= a.batch || d < 0 || d >= a.batch) {
        bad |= SKV_STATUS_BADARG;
      } else {
        L = a.lens[s];
        if (a.lens[d] != 0 || atomicExch(&taken[d], 1) != 0) bad |= SKV_STATUS_BADARG;
        if (L < 0 || ceil_div(L, a.bs) > a.bt_stride) {
          bad |= SKV_STATUS_BADARG;
          L = 0;
        }
        need = L % a.bs != 0 ? 1 : 0;
        if (need) {
          const int32_t old = a.bt[s * a.bt_stride + L / a.bs];
          if (old < 0 || old >= a.n_pages) bad |= SKV_STATUS_BADARG;
        }
      }
      len[f] = L;
    }
    int tot;
    const int ex = block_exclusive_scan(need, scan_lds, &tot);
    if (f < a.n) page[f] = need ? carry + ex : -1;
    carry += tot;
  }
  if (!bad && carry > top) bad = SKV_STATUS_NOSPC;
  if (bad) atomicOr(&bad_all, bad);
  __syncthreads();
  if (!bad_all) {  // uniform: the pages to be popped, in their ranks' place
    for (int f = tid; f < a.n; f += kForkThreads) {
      if (page[f] < 0) continue;
      page[f] = a.stack[top - 1 - page[f]];
      if (page[f] < 0 || page[f] >= a.n_pages) bad = SKV_STATUS_STACK;
    }
    __syncthreads();  // bad_all has been read
    if (bad) atomicOr(&bad_all, bad);
    __syncthreads();
  }
  if (bad_all) {
    if (tid == 0) *a.status = bad_all;
    return;
  }
  for (int f = tid; f < a.n; f += kForkThreads) {
    const int d = a.dst[f];
    if (page[f] >= 0) a.bt[d * a.bt_stride + len[f] / a.bs] = page[f];
    a.lens[d] = len[f];
  }
  if (tid == 0) {
    *a.top = top - carry;
    *a.status = 0;
  }
}

constexpr int kForkCopyThreads = 256;
constexpr int kForkChunks = 4;                                         // 16-byte chunks per thread
constexpr int kForkSlice = kForkCopyThreads * kForkChunks * 16;        // bytes of a page per workgroup
constexpr int kForkEntries = kForkCopyThreads * kForkChunks;           // table entries per workgroup

struct ForkPools {
  uint8_t* base[kForkPools];
  int64_t page_bytes[kForkPools];
  int32_t first[kForkPools + 1];  // slices before pool q's
  int n;
};

// Bytes [off, off + kForkSlice) of n from src to dst, 16 bytes at a time (n a
// multiple of 16).
__device__ __forceinline__ void copy_slice(uint8_t* dst, const uint8_t* src, int64_t off, int64_t n) {
  u32x4 v[kForkChunks];
#pragma unroll
  for (int k = 0; k < kForkChunks; ++k) {
    const int64_t o = off + (k * kForkCopyThreads + static_cast<int>(threadIdx.x)) * 16;
    v[k] = *reinterpret_cast<const u32x4*>(src + (o < n ? o : 0));
  }
#pragma unroll
  for (int k = 0; k < kForkChunks; ++k) {
    const int64_t o = off + (k * kForkCopyThreads + static_cast<int>(threadIdx.x)) * 16;
    if (o < n) *reinterpret_cast<u32x4*>(dst + o) = v[k];
  }
}

// grid: (table parts, then the slices of the pools' pages; forks)
__global__ __launch_bounds__(kForkCopyThreads) void k_fork_copy(ForkArgs a, ForkPools pools, int table_parts) {
  if (*a.status != 0) return;  // refused: uniform
  const int f = blockIdx.y;
  const int64_t s = a.src[f], d = a.dst[f];
  const int L = a.lens[d];  // the plan's
  const int full = L / a.bs;
  int part = blockIdx.x;
  if (part < table_parts) {
#pragma unroll
    for (int k = 0; k < kForkChunks; ++k) {
      const int j = part * kForkEntries + k * kForkCopyThreads + static_cast<int>(threadIdx.x);
      if (j < full) {
        const int32_t p = a.bt[s * a.bt_stride + j];
        a.bt[d * a.bt_stride + j] = p;
        if (p >= 0 && p < a.n_pages) atomicAdd(&a.refs[p], 1);
      }
    }
    return;
  }
  if (L % a.bs == 0) return;
  part -= table_parts;
  int q = 0;
  while (q + 1 < pools.n && part >= pools.first[q + 1]) ++q;
  const int64_t pb = pools.page_bytes[q];
  const int32_t old = a.bt[s * a.bt_stride + full], fresh = a.bt[d * a.bt_stride + full];
  copy_slice(pools.base[q] + fresh * pb, pools.base[q] + old * pb, static_cast<int64_t>(part - pools.first[q]) * kForkSlice, pb);
}

struct SlotArrays {
  uint8_t* base[kForkPools];
  int64_t bytes[kForkPools];
};

// grid: (slices of the largest slot, forks, arrays)
__global__ __launch_bounds__(kForkCopyThreads) void k_copy_slots(SlotArrays arrays, int64_t n_slots,
                                                                 const int32_t* __restrict__ src,
                                                                 const int32_t* __restrict__ dst) {
  const int64_t s = src[blockIdx.y], d = dst[blockIdx.y];
  if (s < 0 || s >= n_slots || d < 0 || d >= n_slots || s == d) return;
  const int64_t n = arrays.bytes[blockIdx.z];
  const int64_t off = static_cast<int64_t>(blockIdx.x) * kForkSlice;
  if (off >= n) return;
  uint8_t* base = arrays.base[blockIdx.z];
  uint8_t* to = base + d * n;
  const uint8_t* from = base + s * n;
  if (((reinterpret_cast<uintptr_t>(base) | static_cast<uintptr_t>(n)) & 15) == 0) {
    copy_slice(to, from, off, n);
  } else {  // counts and the like
    for (int64_t o = off + threadIdx.x; o < min(n, off + kForkSlice); o += kForkCopyThreads) to[o] = from[o];
  }
}

}  // namespace skv

using namespace skv;

extern "C" int skv_fork(int32_t* free_stack, int32_t* free_top, int64_t n_pages, int32_t* refs, int32_t* block_table,
                        int64_t bt_stride, int32_t* seq_lens, int64_t batch, int64_t block_size, const int32_t* src,
                        const int32_t* dst, int64_t n_forks, const skv_pool_ref* pools, int32_t n_pools, int32_t* status,
                        void* stream) {
  const char* what = "skv_fork";
  if (batch < 0 || batch > kForkMax || n_forks < 0 || n_forks > kForkMax) {
    return set_error(SKV_EINVAL, "%s: batch and n_forks must be in [0, %d]; got %lld and %lld", what, kForkMax,
                     (long long)batch, (long long)n_forks);
  }
  if (block_size <= 0 || block_size > INT32_MAX || bt_stride <= 0 || bt_stride > INT32_MAX || n_pages <= 0 ||
      n_pages > INT32_MAX) {
    return set_error(SKV_EINVAL, "%s: bad block_size/bt_stride/n_pages", what);
  }
  if (n_pools < 0 || n_pools > kForkPools || (n_pools > 0 && !pools)) {
    return set_error(SKV_EINVAL, "%s: n_pools must be in [0, %d]; got %d", what, kForkPools, n_pools);
  }
  if (!free_stack || !free_top || !refs || !block_table || !seq_lens || !status || (n_forks > 0 && (!src || !dst))) {
    return set_error(SKV_EINVAL, "%s: NULL pointer", what);
  }
  ForkPools fp{};
  fp.n = n_pools;
  int64_t slices = 0;
  for (int q = 0; q < n_pools; ++q) {
    if (!pools[q].base || pools[q].page_bytes <= 0 || (pools[q].page_bytes & 15) ||
        (reinterpret_cast<uintptr_t>(pools[q].base) & 15)) {
      return set_error(SKV_EINVAL, "%s: pool %d needs a 16-byte aligned base and page_bytes", what, q);
    }
    fp.base[q] = static_cast<uint8_t*>(pools[q].base);
    fp.page_bytes[q] = pools[q].page_bytes;
    slices += ceil_div(pools[q].page_bytes, kForkSlice);
    if (slices >= (1 << 24)) return set_error(SKV_EINVAL, "%s: pages too large", what);
    fp.first[q + 1] = static_cast<int32_t>(slices);
  }
  // the copies' grid, which is counted before the plan has popped a page
  const int64_t table_parts = ceil_div(bt_stride, kForkEntries);
  if (table_parts + slices >= (1 << 24)) return set_error(SKV_EINVAL, "%s: pages and tables too large", what);
  if (batch == 0 && n_forks > 0) return set_error(SKV_EINVAL, "%s: forks in an empty batch", what);
  if (n_forks == 0) return SKV_OK;
  const ForkArgs a{free_stack, free_top, n_pages, refs, block_table, bt_stride, seq_lens, src, dst,
                   static_cast<int>(batch), static_cast<int>(block_size), static_cast<int>(n_forks), status};
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(k_fork_plan, dim3(1), dim3(kForkThreads), 0, s, a);
  if (const int rc = check_launch(what)) return rc;
  hipLaunchKernelGGL(k_fork_copy, dim3(static_cast<unsigned>(table_parts + slices), static_cast<unsigned>(n_forks)),
                     dim3(kForkCopyThreads), 0, s, a, fp, static_cast<int>(table_parts));
  return check_launch(what);
}

extern "C" int skv_copy_slots(const skv_pool_ref* arrays, int64_t n_arrays, int64_t n_slots, const int32_t* src,
                              const int32_t* dst, int64_t n_forks, void* stream) {
  const char* what = "skv_copy_slots";
  if (n_arrays < 0 || n_slots < 0 || n_forks < 0 || n_forks > 65535) {
    return set_error(SKV_EINVAL, "%s: bad n_arrays/n_slots/n_forks", what);
  }
  if ((n_arrays > 0 && !arrays) || (n_forks > 0 && (!src || !dst))) return set_error(SKV_EINVAL, "%s: NULL pointer", what);
  for (int64_t i = 0; i < n_arrays; ++i) {
    if (!arrays[i].base || arrays[i].page_bytes <= 0 || arrays[i].page_bytes > (int64_t{1} << 37)) {
      return set_error(SKV_EINVAL, "%s: array %lld needs a base and a slot size of at most 2^37", what, (long long)i);
    }
  }
  if (n_forks == 0 || n_slots == 0) return SKV_OK;
  for (int64_t i0 = 0; i0 < n_arrays; i0 += kForkPools) {
    SlotArrays sa{};
    const int n = static_cast<int>(std::min<int64_t>(kForkPools, n_arrays - i0));
    int64_t most = 0;
    for (int i = 0; i < n; ++i) {
      sa.base[i] = static_cast<uint8_t*>(arrays[i0 + i].base);
      sa.bytes[i] = arrays[i0 + i].page_bytes;
      most = std::max(most, sa.bytes[i]);
    }
    hipLaunchKernelGGL(k_copy_slots,
                       dim3(static_cast<unsigned>(ceil_div(most, kForkSlice)), static_cast<unsigned>(n_forks),
                            static_cast<unsigned>(n)),
                       dim3(kForkCopyThreads), 0, static_cast<hipStream_t>(stream), sa, n_slots, src, dst);
    if (const int rc = check_launch(what)) return rc;
  }
  return SKV_OK;
}
