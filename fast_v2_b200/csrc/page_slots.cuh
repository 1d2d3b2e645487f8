// Block tables and slot maps of a paged KV cache, built on the device.
//
// A sequence of len tokens holds ceil(len / page) pages of the pool; table
// [b, i] is the page of its tokens i * page .. i * page + page - 1.  Free
// pages are a stack: free_pages[0 .. count), the next one taken is the last.
// For n_new[b] tokens more per sequence (packed rows, sequence after
// sequence):
//   cu[b]    = sum_{i<b} n_new[i]                      row of b's first token
//   need[b]  = ceil((len + n) / page) - ceil(len / page)  new pages
//   at[b]    = sum_{i<b} need[i]                       order of the pages
//   table[b, ceil(len/page) + j] = free_pages[count - 1 - at[b] - j]
//   pos[t]   = len[b] + t - cu[b],  slot[t] = table[b, pos / page] * page + pos % page
//
// Every CTA scans the B lengths itself (three loads per sequence and one block
// scan) and keeps cu and at in shared memory, so one launch does it all with
// any number of CTAs: each new page has exactly one token at its first
// position (pages are new from ceil(len / page) * page >= len on), and the
// thread of that token writes the table entry.  The lengths and the count
// are read by all CTAs and may be updated in place, so the CTA that finishes
// last writes them (a ticket next to the count, left at zero).
#pragma once
#include "common.cuh"
#include "device_util.cuh"

namespace fdl {

constexpr int kSlotsThreads = 256;
constexpr int kSlotsMaxBatch = 4096;

struct PageSlotsArgs {
  const int32_t* lens;
  const int32_t* n_new;
  int32_t* table;
  int64_t table_sb;
  const int32_t* free_pages;
  int32_t* count;  // [0] free pages, [1] ticket (0 between calls)
  int64_t* slots;
  int64_t* pos;
  int32_t* cu;
  int32_t* new_lens;
  int32_t* new_count;
  int B, max_pages, n_free;
  FastDiv page;
  int64_t T;
};

struct SlotSums {
  int64_t tokens;
  int64_t pages;
};

// Inclusive block scan of (tokens, pages) over kSlotsThreads threads.
__device__ __forceinline__ SlotSums block_scan(SlotSums v, SlotSums* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, v.tokens, off);
    const int64_t p = __shfl_up_sync(0xffffffffu, v.pages, off);
    if (lane >= off) {
      v.tokens += t;
      v.pages += p;
    }
  }
  if (lane == 31) sh[warp] = v;
  __syncthreads();
  SlotSums base{0, 0};
  for (int w = 0; w < warp; ++w) {
    base.tokens += sh[w].tokens;
    base.pages += sh[w].pages;
  }
  v.tokens += base.tokens;
  v.pages += base.pages;
  return v;
}

// n_new and new pages of every sequence, the latter -1 for a request that
// cannot be: a length below 0 or past the table's width, or a first token whose
// page, begun before, is missing in the table.  A thread takes kEach sequences a
// round: their lengths and then their entries are on their way together (one
// token each, one by one / so: 1000 sequences 8.9 / 6.7 us, 4000 21.2 / 13.5).
template <int kEach>
__device__ __forceinline__ void slot_requests(const PageSlotsArgs& a, int32_t* s_n, int32_t* s_pages) {
  const int64_t width = static_cast<int64_t>(a.max_pages) * a.page.d;
  for (int b0 = threadIdx.x; b0 < a.B; b0 += kEach * kSlotsThreads) {
    int len[kEach], n[kEach], entry[kEach];
    uint32_t i[kEach], begun[kEach];
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int b = min(b0 + u * kSlotsThreads, a.B - 1);
      len[u] = a.lens[b];
      n[u] = a.n_new[b];
    }
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int b = min(b0 + u * kSlotsThreads, a.B - 1);
      const bool fits = len[u] >= 0 && n[u] >= 0 && static_cast<int64_t>(len[u]) + n[u] <= width;
      a.page.divmod(static_cast<uint32_t>(max(len[u], 0)), i[u], begun[u]);
      entry[u] = fits ? 0 : -1;
      if (fits && n[u] > 0 && begun[u] > 0) entry[u] = a.table[b * a.table_sb + i[u]];  // (the tokens read it again, from L1)
    }
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int b = b0 + u * kSlotsThreads;
      if (b < a.B) {
        s_n[b] = max(n[u], 0);
        s_pages[b] = entry[u] < 0 ? -1
                                  : static_cast<int>(a.page.div(static_cast<uint32_t>(len[u]) + n[u] + a.page.d - 1) -
                                                     i[u] - (begun[u] > 0));
      }
    }
  }
}

__global__ void __launch_bounds__(kSlotsThreads) page_slots_kernel(const __grid_constant__ PageSlotsArgs a) {
  extern __shared__ int32_t s_buf[];
  int32_t* s_cu = s_buf;            // [B + 1], saturated at the largest int32; n_new before the scan
  int32_t* s_at = s_buf + a.B + 1;  // [B]: order of b's first new page, -1 = refused; new pages before the scan
  __shared__ SlotSums sh_scan[kSlotsThreads / 32];
  __shared__ int sh_last, sh_taken;
  await_stream();
  release_stream();
  const int count = min(max(a.count[0], 0), a.n_free);
  if (threadIdx.x == 0) sh_taken = 0;
  if (a.B <= kSlotsThreads)
    slot_requests<1>(a, s_cu, s_at);
  else if (a.B <= 4 * kSlotsThreads)
    slot_requests<4>(a, s_cu, s_at);
  else
    slot_requests<8>(a, s_cu, s_at);
  __syncthreads();
  const int per = (a.B + kSlotsThreads - 1) / kSlotsThreads | 1;  // odd: no two threads on a bank
  const int b0 = threadIdx.x * per, b1 = min(a.B, b0 + per);
  SlotSums sum{0, 0};
  for (int b = b0; b < b1; ++b) {
    sum.tokens += s_cu[b];
    sum.pages += max(s_at[b], 0);
  }
  const SlotSums incl = block_scan(sum, sh_scan);
  SlotSums run{incl.tokens - sum.tokens, incl.pages - sum.pages};
  int taken = 0;
  for (int b = b0; b < b1; ++b) {
    const SlotSums r{s_cu[b], max(s_at[b], 0)};
    const bool ok = s_at[b] >= 0;
    // A request is served whole or not at all: its pages have to be in the
    // pool and its rows in the slot map.
    const bool served = ok && (r.pages == 0 || run.pages + r.pages <= count) && run.tokens + r.tokens <= a.T;
    s_cu[b] = static_cast<int32_t>(min(run.tokens, static_cast<int64_t>(INT32_MAX)));
    s_at[b] = served ? (r.pages ? static_cast<int32_t>(run.pages) : 0) : -1;
    if (served && r.pages) taken = static_cast<int>(run.pages + r.pages);
    if (!served && blockIdx.x == 0) report(FDL_DEV_LENGTH, b);
    run.tokens += r.tokens;
    run.pages += r.pages;
  }
  if (b1 == a.B && b0 < b1) s_cu[a.B] = static_cast<int32_t>(min(run.tokens, static_cast<int64_t>(INT32_MAX)));
  if (taken) atomicMax(&sh_taken, taken);
  __syncthreads();

  const int64_t total = s_cu[a.B];
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kSlotsThreads;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kSlotsThreads + threadIdx.x; t < a.T; t += stride) {
    int64_t slot = -1, p = 0;
    if (t < total) {
      int lo = 0, hi = a.B;  // last b with s_cu[b] <= t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= t) lo = mid; else hi = mid;
      }
      const int len = a.lens[lo];
      p = static_cast<int64_t>(len) + (t - s_cu[lo]);
      if (s_at[lo] >= 0) {
        uint32_t i, r;
        a.page.divmod(static_cast<uint32_t>(p), i, r);
        const uint32_t old = a.page.div(static_cast<uint32_t>(len) + a.page.d - 1);
        int32_t* entry = a.table + lo * a.table_sb + i;
        int32_t page;
        if (i < old) {
          page = *entry;
        } else {
          page = a.free_pages[count - 1 - s_at[lo] - static_cast<int>(i - old)];
          if (r == 0) *entry = page;
        }
        if (page >= 0)
          slot = static_cast<int64_t>(page) * a.page.d + r;
        else
          report(FDL_DEV_INDEX, page);  // the stack of free pages holds it
      }
    }
    a.slots[t] = slot;
    a.pos[t] = p;
  }
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b <= a.B; b += kSlotsThreads) a.cu[b] = s_cu[b];
  // The last CTA to get here writes what every CTA has read.
  __syncthreads();
  if (gridDim.x > 1) {
    if (threadIdx.x == 0) {
      __threadfence();
      sh_last = atomicAdd(a.count + 1, 1) == static_cast<int>(gridDim.x) - 1;
    }
    __syncthreads();
    if (!sh_last) return;
    if (threadIdx.x == 0) a.count[1] = 0;
  }
  for (int b = threadIdx.x; b < a.B; b += kSlotsThreads) {
    const int len = a.lens[b];
    a.new_lens[b] = s_at[b] >= 0 ? len + a.n_new[b] : len;
  }
  if (threadIdx.x == 0) {
    a.new_count[0] = count - sh_taken;
    a.new_count[1] = 0;  // the ticket of a call that takes it as its count
  }
}

// Pages of finished sequences go back on the stack, in the order of the rows
// and of the pages in a row; their table entries become -1 and their lengths
// 0.  One CTA (a finished row is rare and short next to a step): a warp per
// row counts the row's pages, one scan orders the rows, and the warps write.
// A row whose length does not fit its table is left alone and reported, and
// so is the whole call when the stack has no room for the pages.
struct PageReleaseArgs {
  const uint8_t* done;
  int32_t* lens;
  int32_t* table;
  int64_t table_sb;
  int32_t* free_pages;
  int32_t* count;
  int B, max_pages, n_free;
  FastDiv page;
};

__global__ void __launch_bounds__(kSlotsThreads) page_release_kernel(const __grid_constant__ PageReleaseArgs a) {
  extern __shared__ int32_t s_n[];  // [B] pages of the row, then their order
  __shared__ SlotSums sh_scan[kSlotsThreads / 32];
  __shared__ int64_t sh_total;
  await_stream();
  release_stream();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int b = warp; b < a.B; b += kSlotsThreads / 32) {
    int n = -1;
    if (a.done[b]) {
      const int len = a.lens[b];
      if (len < 0 || len > static_cast<int64_t>(a.max_pages) * a.page.d) {
        if (lane == 0) report(FDL_DEV_LENGTH, b);
      } else {
        const int pages = a.page.div(static_cast<uint32_t>(len) + a.page.d - 1);
        n = 0;
        for (int i = lane; i - lane < pages; i += 32)
          n += __popc(__ballot_sync(0xffffffffu, i < pages && a.table[b * a.table_sb + i] >= 0));
      }
    }
    if (lane == 0) s_n[b] = n;
  }
  __syncthreads();
  const int per = (a.B + kSlotsThreads - 1) / kSlotsThreads;
  const int b0 = threadIdx.x * per, b1 = min(a.B, b0 + per);
  SlotSums sum{0, 0};
  for (int b = b0; b < b1; ++b) sum.pages += max(s_n[b], 0);
  const SlotSums incl = block_scan(sum, sh_scan);
  int64_t at = incl.pages - sum.pages;
  for (int b = b0; b < b1; ++b) {
    const int n = s_n[b];
    if (n >= 0) s_n[b] = static_cast<int32_t>(at);
    at += max(n, 0);
  }
  if (threadIdx.x == kSlotsThreads - 1) sh_total = incl.pages;
  __syncthreads();
  const int64_t count = min(max(a.count[0], 0), a.n_free);
  if (count + sh_total > a.n_free) {
    if (threadIdx.x == 0) report(FDL_DEV_INDEX, count + sh_total);
    return;
  }
  for (int b = warp; b < a.B; b += kSlotsThreads / 32) {
    if (s_n[b] < 0) continue;
    const int pages = a.page.div(static_cast<uint32_t>(a.lens[b]) + a.page.d - 1);
    int64_t to = count + s_n[b];
    for (int i = lane; i - lane < pages; i += 32) {
      const int32_t page = i < pages ? a.table[b * a.table_sb + i] : -1;
      const unsigned have = __ballot_sync(0xffffffffu, page >= 0);
      if (page >= 0) a.free_pages[to + __popc(have & ((1u << lane) - 1))] = page;
      if (i < pages) a.table[b * a.table_sb + i] = -1;
      to += __popc(have);
    }
    __syncwarp();
    if (lane == 0) a.lens[b] = 0;
  }
  __syncthreads();
  if (threadIdx.x == 0) a.count[0] = static_cast<int32_t>(count + sh_total);
}

}  // namespace fdl
