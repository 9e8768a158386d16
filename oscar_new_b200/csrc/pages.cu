// Page pool of the paged cache on the device: requests forked copy-on-write, grown,
// released, and their pages compacted.  (The reference leaves paging to its host engine
// and refuses shared pages, oscar_ascend/backend.py:41-64, because a request's BF16
// window lives in its first page; a fork here gives every request its own first page.)
//
// State, one int32 arena: a reference count per page (page 0 is never handed out), a
// length per request row, and the block table.  A row of L tokens holds ceil(L / Bp)
// pages in table order.  Fresh pages are the free pages of the lowest numbers, handed out
// in the order of the call's list, so every result is determined by the state and the
// list alone: the small decisions (validity, prefix sums, the search for free pages) run
// in one block, and only the pages' bytes and table rows are spread over the GPU.
//
// Bytes: a page's used slots (tokens * H * 160, contiguous in the K stripe) and, for a
// first page, the window (contiguous in the V stripe) are moved as 16 KiB slices: 131 MB (most of
// it written) of 60 forks in 28 us, 4.6 TB/s, behind 8 us of decisions; 145 MB of a compaction
// in 26 us.  The next slice's job fetched ahead of this one's stores: 28 us too, not kept.
#include <algorithm>

#include "common.cuh"

namespace oscar {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kSliceBytes = 16384;

struct PageJob {  // one page to copy: `tokens` slots, the window when `window` is set
  int32_t src, dst, tokens, window;
};

struct Pool {
  int32_t *refs, *lens, *table;          // state
  int32_t *head, *claim, *remap, *used;  // workspace
  int32_t *list;                         // [num_pages]: free pages found / holes
  PageJob *jobs;
  int32_t num_pages, max_reqs, columns;
  int32_t block_tokens, per_page;        // tokens per page, 128-token blocks per page
};

int64_t up4(int64_t x) { return (x + 3) / 4 * 4; }

bool pool_offsets(int64_t num_pages, int64_t max_reqs, int64_t columns, int64_t (&off)[10]) {
  if (num_pages < 1 || max_reqs < 1 || columns < 1 || num_pages > (1 << 24) || max_reqs > (1 << 20) ||
      columns > (1 << 24) || max_reqs * columns > INT32_MAX)  // sums of pages over all rows are int32
    return false;
  const int64_t jobs = std::max(2 * max_reqs, num_pages);
  off[0] = 0;                                   // reference counts
  off[1] = off[0] + up4(num_pages);             // lengths
  off[2] = off[1] + up4(max_reqs);              // table
  off[3] = off[2] + up4(max_reqs * columns);    // end of the state; head
  off[4] = off[3] + 8;                          // claim
  off[5] = off[4] + up4(max_reqs);              // remap
  off[6] = off[5] + up4(num_pages);             // used
  off[7] = off[6] + up4(num_pages);             // list
  off[8] = off[7] + up4(num_pages);             // jobs
  off[9] = off[8] + 4 * jobs;                   // words
  return true;
}

bool make_pool(Pool &p, int32_t *arena, int32_t num_pages, int32_t max_reqs, int32_t columns, int32_t block_tokens) {
  int64_t off[10];
  if (!arena || (reinterpret_cast<uintptr_t>(arena) & 15) || block_tokens <= 0 || block_tokens % kKernelBlock ||
      !pool_offsets(num_pages, max_reqs, columns, off))
    return false;
  p.refs = arena + off[0], p.lens = arena + off[1], p.table = arena + off[2], p.head = arena + off[3];
  p.claim = arena + off[4], p.remap = arena + off[5], p.used = arena + off[6], p.list = arena + off[7];
  p.jobs = reinterpret_cast<PageJob *>(arena + off[8]);
  p.num_pages = num_pages, p.max_reqs = max_reqs, p.columns = columns;
  p.block_tokens = block_tokens, p.per_page = block_tokens / kKernelBlock;
  return true;
}

// unsigned: tokens (not negative) may be up to 2^31 - 1
OSCAR_DEVINL int pages_of(const Pool &p, int tokens) {
  return (int)(((uint32_t)tokens + p.block_tokens - 1) / (uint32_t)p.block_tokens);
}
// tokens a table row can hold
OSCAR_DEVINL int64_t row_tokens(const Pool &p) { return (int64_t)(p.columns / p.per_page) * p.block_tokens; }
OSCAR_DEVINL int table_page(const Pool &p, int row, int page) {
  return p.table[(int64_t)row * p.columns + (int64_t)page * p.per_page] / p.per_page;
}
OSCAR_DEVINL bool page_ok(const Pool &p, int page) { return page > 0 && page < p.num_pages; }

// Inclusive scan over the block (kPlanThreads threads); `total` is the block's sum.
OSCAR_DEVINL int block_scan(int v, int &total) {
  __shared__ int32_t sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();  // the previous scan's readers are done
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  int s = sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  total = __shfl_sync(0xffffffffu, s, 31);
  const int before = __shfl_sync(0xffffffffu, s, (warp + 31) & 31);
  return v + (warp ? before : 0);
}

// list[0 .. found) = the lowest free pages, at most `want`; returns found.  Four pages per
// thread and step (the counts are 16-byte aligned and padded).
OSCAR_DEVINL int find_free(const Pool &p, int want) {
  int found = 0;
  for (int base = 0; base < p.num_pages && found < want; base += 4 * kPlanThreads) {
    const int page = base + 4 * threadIdx.x;
    int4 c = make_int4(1, 1, 1, 1);
    if (page < p.num_pages) c = __ldcg(reinterpret_cast<const int4 *>(p.refs + page));
    const bool f[4] = {c.x == 0 && page > 0, c.y == 0 && page + 1 < p.num_pages, c.z == 0 && page + 2 < p.num_pages,
                       c.w == 0 && page + 3 < p.num_pages};
    const int mine = f[0] + f[1] + f[2] + f[3];
    int total;
    int at = found + block_scan(mine, total) - mine;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (f[k] && at < want)
        p.list[at++] = page + k;
    found += total;
  }
  __syncthreads();
  return min(found, want);
}

// claim[row] = the first list entry that names `row` (entries out of range claim nothing)
OSCAR_DEVINL void claim_rows(const Pool &p, const int32_t *rows, int count) {
  for (int i = threadIdx.x; i < count; i += kPlanThreads)
    if (rows[i] >= 0 && rows[i] < p.max_reqs) p.claim[rows[i]] = INT32_MAX;
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kPlanThreads)
    if (rows[i] >= 0 && rows[i] < p.max_reqs) atomicMin(p.claim + rows[i], i);
  __syncthreads();
}

// ---- fork -------------------------------------------------------------------------

__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const Pool p, const int32_t *__restrict__ parents,
                                                                 const int32_t *__restrict__ children, int count,
                                                                 int32_t *__restrict__ result) {
  claim_rows(p, children, count);
  // pages each pair needs (0: not a valid pair), judged on the state before the call
  int carry = 0;
  for (int base = 0; base < count; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int need = 0;
    if (i < count) {
      const int a = parents[i], c = children[i];
      if (a >= 0 && a < p.max_reqs && c >= 0 && c < p.max_reqs && __ldcg(p.claim + c) == i) {
        const int n = p.lens[a];
        if (n > 0 && n <= row_tokens(p) && p.lens[c] == 0) need = n > p.block_tokens && n % p.block_tokens ? 2 : 1;
      }
    }
    int total;
    const int upto = carry + block_scan(need, total);
    if (i < count) {
      p.jobs[2 * i].tokens = need;  // until the pages are known
      p.jobs[2 * i].src = upto;
    }
    carry += total;
  }
  __syncthreads();
  const int have = find_free(p, carry);
  for (int i = threadIdx.x; i < count; i += kPlanThreads) {
    const int need = p.jobs[2 * i].tokens, upto = p.jobs[2 * i].src;
    PageJob first{0, 0, 0, 0}, last{0, 0, 0, 0};
    if (need > 0 && upto <= have) {
      const int n = p.lens[parents[i]], c = children[i];
      first.src = table_page(p, parents[i], 0);
      first.dst = p.list[upto - need];
      first.tokens = min(n, p.block_tokens);
      first.window = 1;
      p.refs[first.dst] = 1;
      if (need == 2) {
        last.src = table_page(p, parents[i], n / p.block_tokens);
        last.dst = p.list[upto - 1];
        last.tokens = n % p.block_tokens;
        p.refs[last.dst] = 1;
      }
      result[i] = 1;
      p.claim[c] = n;  // the child's length, published once every pair has been judged
    } else {
      result[i] = need > 0 ? 0 : -1;
    }
    p.jobs[2 * i] = first;
    p.jobs[2 * i + 1] = last;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kPlanThreads)
    if (result[i] == 1) p.lens[children[i]] = p.claim[children[i]];
  if (threadIdx.x == 0) p.head[0] = 2 * count;
}

// Table rows of the forked children and the counts of the pages they share.
OSCAR_DEVINL void fork_row(const Pool &p, int i, int parent, int child) {
  const PageJob first = p.jobs[2 * i], last = p.jobs[2 * i + 1];
  if (!first.dst) return;
  const int n = p.lens[child], pages = pages_of(p, n), cols = pages * p.per_page;
  const int32_t *src = p.table + (int64_t)parent * p.columns;
  int32_t *dst = p.table + (int64_t)child * p.columns;
  for (int c = threadIdx.x; c < p.columns; c += blockDim.x) {
    const int page = c / p.per_page, in = c % p.per_page;
    int block = 0;
    if (c < cols) {
      block = src[c];
      if (page == 0) {
        block = first.dst * p.per_page + in;
      } else if (last.dst && page == pages - 1) {
        block = last.dst * p.per_page + in;
      } else if (in == 0 && page_ok(p, block / p.per_page)) {
        atomicAdd(p.refs + block / p.per_page, 1);
      }
    }
    dst[c] = block;
  }
}

// ---- copies -----------------------------------------------------------------------

struct CopyParams {
  Pool p;
  uint8_t *history, *window;
  int64_t page_bytes;
  int32_t slot_row;       // H * 160: bytes of one token's slots
  int32_t window_bytes;
  int32_t slices_h, slices_w;  // most slices of a page's history and window
  const int32_t *parents, *children;  // fork rows (nullable)
  int32_t rows;
  int32_t marked;  // compact: a job's tokens and window are the marks of its source page
};

__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const CopyParams C) {
  const Pool &p = C.p;
  for (int i = blockIdx.x; i < C.rows; i += gridDim.x) fork_row(p, i, C.parents[i], C.children[i]);
  const int per_job = C.slices_h + C.slices_w;
  const int64_t units = (int64_t)p.head[0] * per_job;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    PageJob job = p.jobs[u / per_job];
    const int s = (int)(u % per_job);
    if (!page_ok(p, job.src) || !page_ok(p, job.dst)) continue;
    if (C.marked) {
      job.tokens = p.used[job.src], job.window = p.list[job.src];
      // no row holds it, its count alone does: what it keeps is not known here
      if (job.tokens == 0) job.tokens = p.block_tokens, job.window = 1;
    }
    const bool hist = s < C.slices_h;
    const int64_t at = (int64_t)(hist ? s : s - C.slices_h) * kSliceBytes;
    const int64_t bytes = hist ? (int64_t)job.tokens * C.slot_row : (job.window ? C.window_bytes : 0);
    if (at >= bytes) continue;
    uint8_t *base = hist ? C.history : C.window;
    const uint4 *src = reinterpret_cast<const uint4 *>(base + job.src * C.page_bytes + at);
    uint4 *dst = reinterpret_cast<uint4 *>(base + job.dst * C.page_bytes + at);
    const int vecs = (int)(min(bytes - at, (int64_t)kSliceBytes) / 16);
    constexpr int V = kSliceBytes / 16 / kCopyThreads;
    uint4 x[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int v = threadIdx.x + k * kCopyThreads;
      if (v < vecs) x[k] = __ldg(src + v);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int v = threadIdx.x + k * kCopyThreads;
      if (v < vecs) dst[v] = x[k];
    }
  }
}

// ---- resize -----------------------------------------------------------------------

// A warp takes 16 list entries at a time: lane k < 16 judges entry k, then the whole warp
// walks the entries that change the table, the loads of four of them in flight and a lane per
// page of a released row.  512 entries, 192 releases of 11 pages and 320 growths by 3 (one
// block): 19 us; a lane per table word of a released row, each divided by the blocks of a
// page, 24 us.
constexpr int kEntries = 16;

__global__ void __launch_bounds__(kPlanThreads) resize_kernel(const Pool p, const int32_t *__restrict__ rows,
                                                              const int32_t *__restrict__ lens, int count,
                                                              int32_t *__restrict__ result) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, step = kEntries * kPlanThreads / 32;
  claim_rows(p, rows, count);
  // releases first: their pages serve the growth of the same call
  for (int base = 0; base < count; base += step) {
    const int i = base + warp * kEntries + lane;
    int state = 0, cols = 0, r = 0;  // state 0: no entry, -1 refused, 1 release, 2 + pages needed
    if (lane < kEntries && i < count) {
      r = rows[i];
      const int want = lens[i];
      state = -1;
      if (r >= 0 && r < p.max_reqs && __ldcg(p.claim + r) == i) {
        const int n = p.lens[r];
        if (want == 0 && n >= 0 && n <= row_tokens(p)) {
          state = 1;
          cols = pages_of(p, n) * p.per_page;
          p.lens[r] = 0;
        } else if (want > 0 && want >= n && n >= 0 && want <= row_tokens(p)) {
          state = 2 + pages_of(p, want) - pages_of(p, n);
        }
      }
      result[i] = state;
    }
    uint32_t left = __ballot_sync(0xffffffffu, cols > 0);
    while (left) {
      int32_t *row[4];
      int n[4], most = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int e = left ? __ffs(left) - 1 : -1;
        left &= left - 1;  // 0 stays 0
        row[k] = p.table + (int64_t)__shfl_sync(0xffffffffu, r, e & 31) * p.columns;
        n[k] = __shfl_sync(0xffffffffu, cols, e & 31);
        if (e < 0) n[k] = 0;
        most = max(most, n[k]);
      }
      for (int c = lane * p.per_page; c < most; c += 32 * p.per_page) {  // a lane per page
        int block[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c < n[k]) block[k] = row[k][c];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c < n[k] && page_ok(p, block[k] / p.per_page)) atomicSub(p.refs + block[k] / p.per_page, 1);
      }
      __syncwarp();  // the blocks are read
      for (int c = lane; c < most; c += 32)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c < n[k]) row[k][c] = 0;
    }
  }
  __syncthreads();
  int carry = 0;
  for (int base = 0; base < count; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    const int need = i < count ? result[i] - 2 : -1;  // < 0: nothing to grow
    int total;
    const int upto = carry + block_scan(max(need, 0), total);
    if (i < count) p.jobs[i].src = upto;
    carry += total;
  }
  __syncthreads();
  const int have = find_free(p, carry);
  for (int base = 0; base < count; base += step) {
    const int i = base + warp * kEntries + lane;
    int first = 0, words = 0;  // first fresh page in the list, table words to write
    int64_t at = 0;
    if (lane < kEntries && i < count) {
      const int need = result[i] - 2, upto = p.jobs[i].src;
      if (need >= 0) {
        const bool ok = need == 0 || upto <= have;
        if (ok) {
          const int r = rows[i];
          first = upto - need, words = need * p.per_page;
          at = (int64_t)r * p.columns + (int64_t)pages_of(p, p.lens[r]) * p.per_page;
          p.lens[r] = lens[i];
        }
        result[i] = ok;
      }
    }
    uint32_t left = __ballot_sync(0xffffffffu, words > 0);
    while (left) {
      int32_t *row[4];
      int from[4], n[4], most = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int e = left ? __ffs(left) - 1 : -1;
        left &= left - 1;
        row[k] = p.table + __shfl_sync(0xffffffffu, at, e & 31);
        from[k] = __shfl_sync(0xffffffffu, first, e & 31);
        n[k] = __shfl_sync(0xffffffffu, words, e & 31);
        if (e < 0) n[k] = 0;
        most = max(most, n[k]);
      }
      for (int c = lane; c < most; c += 32) {
        int page[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c < n[k]) page[k] = p.list[from[k] + c / p.per_page];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c < n[k]) {
            row[k][c] = page[k] * p.per_page + c % p.per_page;
            if (c % p.per_page == 0) p.refs[page[k]] = 1;
          }
      }
    }
  }
}

// ---- compact ----------------------------------------------------------------------

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const Pool p, int32_t *__restrict__ summary,
                                                                    int32_t *__restrict__ moved_to) {
  int mine = 0;
  for (int page = 1 + threadIdx.x; page < p.num_pages; page += kPlanThreads) mine += __ldcg(p.refs + page) > 0;
  int live;
  block_scan(mine, live);
  int holes = 0, movers = 0;
  for (int base = 0; base < p.num_pages; base += kPlanThreads) {
    const int page = base + threadIdx.x;
    const bool in = page < p.num_pages;
    const bool used = in && page > 0 && __ldcg(p.refs + page) > 0;
    const bool hole = in && page > 0 && !used && page <= live, mover = used && page > live;
    int total;
    // holes and movers never share a page: one scan counts both (16 bits each per block)
    const int at = block_scan((hole ? 1 : 0) + (mover ? 1 << 16 : 0), total);
    if (hole) p.list[holes + (at & 0xffff) - 1] = page;
    if (mover) p.jobs[movers + (at >> 16) - 1].src = page;
    if (in) {
      p.used[page] = 0;
      p.remap[page] = used || page == 0 ? page : -1;
    }
    holes += total & 0xffff;
    movers += total >> 16;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < movers; k += kPlanThreads) {
    const int src = p.jobs[k].src, dst = p.list[k];
    p.jobs[k].dst = dst;
    p.remap[src] = dst;
    p.refs[dst] = __ldcg(p.refs + src);
    p.refs[src] = 0;
  }
  __syncthreads();
  for (int page = threadIdx.x; page < p.num_pages; page += kPlanThreads) {
    moved_to[page] = p.remap[page];
    p.list[page] = 0;  // from here on: pages that own a window
  }
  if (threadIdx.x == 0) {
    p.head[0] = movers;
    summary[0] = live;
    summary[1] = movers;
  }
}

// used[page] = most tokens a request keeps in a page (0: no request does), list[page] = 1
// when a request starts in it (its window), both by the old page numbers; the table's blocks
// follow their pages
__global__ void __launch_bounds__(kCopyThreads) compact_rows_kernel(const Pool p) {
  const int r = blockIdx.x;
  const int n = (int)min((int64_t)max(p.lens[r], 0), row_tokens(p));
  const int cols = pages_of(p, n) * p.per_page;
  int32_t *row = p.table + (int64_t)r * p.columns;
  for (int c = threadIdx.x; c < p.columns; c += kCopyThreads) {
    const int block = row[c], page = block / p.per_page, at = c / p.per_page;
    if (c >= cols) {
      if (block) row[c] = 0;
      continue;
    }
    if (!page_ok(p, page)) continue;
    if (c % p.per_page == 0) atomicMax(p.used + page, min(n - at * p.block_tokens, p.block_tokens));
    if (c == 0) atomicExch(p.list + page, 1);
    const int to = p.remap[page];
    if (to >= 0 && to != page) row[c] = to * p.per_page + block % p.per_page;
  }
}

}  // namespace
}  // namespace oscar

using namespace oscar;

namespace {

// Launch of the copies of p.jobs[0 .. head[0]), at most `jobs` of them.
int launch_copies(const Pool &p, const oscar_geometry &geo, void *history, void *window, int64_t jobs,
                  const int32_t *parents, const int32_t *children, int32_t rows, int32_t marked, cudaStream_t st) {
  CopyParams C{};
  C.p = p;
  C.history = reinterpret_cast<uint8_t *>(history), C.window = reinterpret_cast<uint8_t *>(window);
  C.page_bytes = geo.page_bytes;
  C.slot_row = geo.kv_heads * geo.slot_bytes;
  C.window_bytes = (geo.sink + geo.ring) * 2 * geo.kv_heads * kDim * 2;
  C.slices_h = (int32_t)(((int64_t)geo.block_tokens * C.slot_row + kSliceBytes - 1) / kSliceBytes);
  C.slices_w = (C.window_bytes + kSliceBytes - 1) / kSliceBytes;
  C.parents = parents, C.children = children, C.rows = rows, C.marked = marked;
  const int64_t units = std::max<int64_t>(jobs * (C.slices_h + C.slices_w), rows);
  if (units == 0) return OSCAR_OK;  // a pool of one page has none to move
  const int grid = (int)std::min<int64_t>(units, 148 * 8);
  copy_pages_kernel<<<grid, kCopyThreads, 0, st>>>(C);
  OSCAR_CHECK_LAUNCH();
  return OSCAR_OK;
}

bool stripes_ok(const oscar_geometry &geo, const void *history, const void *window) {
  return paged_geometry_ok(geo) && history && window &&
         !((reinterpret_cast<uintptr_t>(history) | reinterpret_cast<uintptr_t>(window)) & 15) &&
         (int64_t)geo.block_tokens * geo.kv_heads * geo.slot_bytes <= geo.page_bytes &&
         ((int64_t)geo.sink + geo.ring) * 2 * geo.kv_heads * kDim * 2 <= geo.page_bytes &&
         geo.page_bytes <= INT32_MAX;
}

}  // namespace

extern "C" int oscar_page_pool_layout(int32_t num_pages, int32_t max_reqs, int32_t columns, int64_t *offsets) {
  int64_t off[10];
  if (!offsets || !pool_offsets(num_pages, max_reqs, columns, off)) return OSCAR_ERR_INVALID;
  for (int i = 0; i < 4; ++i) offsets[i] = off[i];
  offsets[4] = off[9];
  return OSCAR_OK;
}

extern "C" int oscar_fork_requests(int32_t *arena, int32_t num_pages, int32_t max_reqs, int32_t columns,
                                   const int32_t *parents, const int32_t *children, int32_t count, void *history,
                                   void *window, oscar_geometry geo, int32_t *result, void *stream) {
  Pool p;
  if (!make_pool(p, arena, num_pages, max_reqs, columns, geo.block_tokens) || !stripes_ok(geo, history, window) ||
      count < 0 || count > max_reqs)
    return OSCAR_ERR_INVALID;
  if (count == 0) return OSCAR_OK;
  if (!parents || !children || !result) return OSCAR_ERR_INVALID;
  cudaStream_t st = (cudaStream_t)stream;
  fork_plan_kernel<<<1, kPlanThreads, 0, st>>>(p, parents, children, count, result);
  OSCAR_CHECK_LAUNCH();
  return launch_copies(p, geo, history, window, 2 * (int64_t)count, parents, children, count, 0, st);
}

extern "C" int oscar_resize_requests(int32_t *arena, int32_t num_pages, int32_t max_reqs, int32_t columns,
                                     int32_t block_tokens, const int32_t *rows, const int32_t *lens, int32_t count,
                                     int32_t *result, void *stream) {
  Pool p;
  if (!make_pool(p, arena, num_pages, max_reqs, columns, block_tokens) || count < 0 || count > max_reqs)
    return OSCAR_ERR_INVALID;
  if (count == 0) return OSCAR_OK;
  if (!rows || !lens || !result) return OSCAR_ERR_INVALID;
  resize_kernel<<<1, kPlanThreads, 0, (cudaStream_t)stream>>>(p, rows, lens, count, result);
  OSCAR_CHECK_LAUNCH();
  return OSCAR_OK;
}

extern "C" int oscar_compact_pages(int32_t *arena, int32_t num_pages, int32_t max_reqs, int32_t columns, void *history,
                                   void *window, oscar_geometry geo, int32_t *summary, int32_t *moved_to,
                                   void *stream) {
  Pool p;
  if (!make_pool(p, arena, num_pages, max_reqs, columns, geo.block_tokens) || !stripes_ok(geo, history, window) ||
      !summary || !moved_to)
    return OSCAR_ERR_INVALID;
  cudaStream_t st = (cudaStream_t)stream;
  compact_plan_kernel<<<1, kPlanThreads, 0, st>>>(p, summary, moved_to);
  OSCAR_CHECK_LAUNCH();
  compact_rows_kernel<<<max_reqs, kCopyThreads, 0, st>>>(p);
  OSCAR_CHECK_LAUNCH();
  return launch_copies(p, geo, history, window, num_pages / 2, nullptr, nullptr, 0, 1, st);
}
