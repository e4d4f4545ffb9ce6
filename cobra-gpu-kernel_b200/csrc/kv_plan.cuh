// kv_plan.cuh -- block tables and slot maps of a paged cache from the requests'
// lengths, in one launch and without a round trip to the host.
//
// For request r, growing from old to new tokens (or shrinking: finished, or
// guessed tokens taken back), with P tokens a page:
//   held = ceil(old / P), want = ceil(new / P), n = max(new - old, 0)
//   given back: held - want pages, pushed on the stack of free pages in order
//   taken: want - held pages, popped from its top
//   token i: position old + i, slot = page(position) * P + position % P
// Everything is a function of exclusive sums over the requests, which every
// block computes for itself in shared memory (reading 8 bytes a request from
// L2), so blocks need not wait for one another; then all blocks share the
// flattened lists of pages and tokens, finding each item's owner by bisection.
//
// What the call reads of the table and of the stack it does not write: pops
// come from below the old top, or from the pages given back, which are read in
// the table rows that they are leaving; pushes go above the old top; new table
// entries lie past the old ones. So a repeated call gives the same answer, and
// the caller keeps a step by adopting its lengths and its count of free pages.
//
// Bound: latency. 32 requests with a token each take 2.4 us (launch and one block's
// sums), 4096 requests with 281 thousand new tokens 12 us, of which writing the 12
// bytes a token would be 0.7.
#pragma once

#include "kv_common.cuh"

namespace b200l {

struct KvPlanArgs {
  const int* old_lens;
  const int* new_lens;
  int* table;
  long long table_stride;
  int* free_pages;
  const int* free_count;
  int* cu_new;
  int* cu_pages;
  int* positions;
  long long* slots;
  int* info;             // free pages after the step, pages that were missing
  int* unplaced;         // new tokens past max_tokens, or NULL
  int requests, width, page, log2_page, capacity, max_tokens;
};

// Exclusive sums over the block's threads, totals in tot: of tokens (64 bits) and of
// three counts of pages.
struct KvSums {
  long long tokens;
  int take, give, pages;
};
__device__ __forceinline__ KvSums operator+(KvSums a, const KvSums& b) {
  a.tokens += b.tokens;
  a.take += b.take;
  a.give += b.give;
  a.pages += b.pages;
  return a;
}
__device__ __forceinline__ KvSums warp_scan(KvSums v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    KvSums y;
    y.tokens = __shfl_up_sync(0xffffffffu, v.tokens, o);
    y.take = __shfl_up_sync(0xffffffffu, v.take, o);
    y.give = __shfl_up_sync(0xffffffffu, v.give, o);
    y.pages = __shfl_up_sync(0xffffffffu, v.pages, o);
    if (lane >= o) v = v + y;
  }
  return v;
}
__device__ __forceinline__ void block_scan(KvSums& v, KvSums& tot, KvSums* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const KvSums inc = warp_scan(v, lane);
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const KvSums s = warp_scan(lane < nw ? part[lane] : KvSums{0, 0, 0, 0}, lane);
    __syncwarp();
    part[lane] = s;
  }
  __syncthreads();
  const KvSums before = warp ? part[warp - 1] : KvSums{0, 0, 0, 0};
  tot = part[nw - 1];
  v = KvSums{before.tokens + inc.tokens - v.tokens, before.take + inc.take - v.take, before.give + inc.give - v.give,
             before.pages + inc.pages - v.pages};
}

__global__ void __launch_bounds__(1024) kv_plan_kernel(KvPlanArgs a) {
  pdl_wait_then_release();
  extern __shared__ int sm_plan[];
  __shared__ KvSums part[32];
  __shared__ unsigned long long s_over;
  const int R = a.requests;
  int* s_new = sm_plan;              // exclusive sums, R + 1 each: new tokens,
  int* s_take = s_new + R + 1;       // pages taken,
  int* s_give = s_take + R + 1;      // pages given back
  const int cap = a.width << a.log2_page, mask = a.page - 1;
  auto length = [&](const int* p, int r) { return min(max(p[r], 0), cap); };
  auto pages = [&](int len) { return (int)(((unsigned)len + mask) >> a.log2_page); };

  const int per = (R + blockDim.x - 1) / blockDim.x;
  const int r0 = min(R, (int)threadIdx.x * per), r1 = min(R, r0 + per);
  KvSums v{0, 0, 0, 0}, tot;
  long long over = 0;                // pages past the table's width
  for (int r = r0; r < r1; ++r) {
    const int o = length(a.old_lens, r), n = length(a.new_lens, r), po = pages(o), pn = pages(n);
    v = v + KvSums{max(n - o, 0), max(pn - po, 0), max(po - pn, 0), n > o ? pn : 0};
    if (blockIdx.x == 0 && a.new_lens[r] > cap) over += ((long long)a.new_lens[r] + mask) / a.page - a.width;
  }
  if (threadIdx.x == 0) s_over = 0;
  block_scan(v, tot, part);
  if (over) atomicAdd(&s_over, (unsigned long long)over);
  auto clip = [](long long x) { return (int)(x < 0x7fffffffLL ? x : 0x7fffffffLL); };
  const bool first = blockIdx.x == 0;
  for (int r = r0; r < r1; ++r) {
    const int o = length(a.old_lens, r), n = length(a.new_lens, r), po = pages(o), pn = pages(n);
    s_new[r] = clip(v.tokens);
    s_take[r] = v.take;
    s_give[r] = v.give;
    if (first) {
      a.cu_new[r] = clip(v.tokens);
      a.cu_pages[r] = v.pages;
    }
    v = v + KvSums{max(n - o, 0), max(pn - po, 0), max(po - pn, 0), n > o ? pn : 0};
  }
  const int total = clip(tot.tokens), take = tot.take, give = tot.give;
  const int count = min(max(*a.free_count, 0), a.capacity), top = count + give;
  if (threadIdx.x == 0) {
    s_new[R] = total;
    s_take[R] = take;
    s_give[R] = give;
    if (first) {
      a.cu_new[R] = total;
      a.cu_pages[R] = tot.pages;
    }
  }
  __syncthreads();
  if (first && threadIdx.x == 0) {
    a.info[0] = max(top - take, 0);
    a.info[1] = clip(max(take - top, 0) + (long long)s_over);
    if (a.unplaced) *a.unplaced = max(total - a.max_tokens, 0);
  }

  // Page at height i of the stack with the pages given back on top of it.
  auto given = [&](int i) {          // i-th page given back
    const int r = find_owner(s_give, R, i);
    return a.table[r * a.table_stride + pages(length(a.new_lens, r)) + (i - s_give[r])];
  };
  auto stack = [&](int i) { return i < 0 ? -1 : i < count ? a.free_pages[i] : given(i - count); };

  const int t0 = blockIdx.x * blockDim.x + threadIdx.x, step = gridDim.x * blockDim.x;
  for (int i = t0; i < take; i += step) {
    const int r = find_owner(s_take, R, i);
    a.table[r * a.table_stride + pages(length(a.old_lens, r)) + (i - s_take[r])] = stack(top - 1 - i);
  }
  for (int i = t0; i < give; i += step)
    if (count + i < a.capacity) a.free_pages[count + i] = given(i);
  for (int i = t0; i < a.max_tokens; i += step) {
    int pos = -1;
    long long slot = -1;
    if (i < total) {
      const int r = find_owner(s_new, R, i);
      const int o = length(a.old_lens, r), held = pages(o);
      pos = o + (i - s_new[r]);
      const int p = pos >> a.log2_page;
      const int id = p < held ? a.table[r * a.table_stride + p] : stack(top - 1 - (s_take[r] + p - held));
      if (id >= 0) slot = ((long long)id << a.log2_page) + (pos & mask);
    }
    a.positions[i] = pos;
    a.slots[i] = slot;
  }
}

}  // namespace b200l
