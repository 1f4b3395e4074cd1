// Tables of pages from the lengths that requests ask for, and the places of a step's rows, on the device.
//
// Tables.  A sequence of `len` tokens has the first ceil(len / page) entries of its row of the table.  For lengths w asked for:
//   gone_b = max(ceil(len_b / page) - ceil(w_b / page), 0),  more_b the other way round
//   pages that are given back lie on a stack in their order, the first one on top; then the sequences take theirs from the top,
//   one sequence behind the other, as long as more_0 + ... + more_b <= what the stack holds
// Both orders count from the top, so the x-th page given back is the x-th taken: a thread has the x-th of either and moves it from the
// place it leaves to the place it goes to, and no thread reads what another writes.  Sums over the sequences come first, by one
// workgroup; where the table is small it moves the pages too, else a second launch does.
//
// Slots.  Row t of sequence b is its token j = len_b - rows_b + (t - starts_b), on place table[b][j / page] * page + j % page.
//
// Both move few bytes; they are bound by their launches and by the loads that wait for one another.
#include "cbk_cache_attn.h"
#include "cbk_cache_check.h"

namespace cbk {

struct DPages {
  int32_t *table, *lens, *free, *count;
  int64_t ld, pages;
  int seqs, cols, page, shift;
};
struct PagePlan { int64_t count, gone, taken, moves; };             // pages on the stack before, given back, taken; the larger of the two

constexpr int PLAN_THREADS = 1024;
constexpr int64_t INLINE_MOVES = 8192;      // entries of a table whose pages the first launch moves

struct Change { int have, need, now; };     // pages before and asked for; the length asked for
__device__ inline Change change_of(const DPages& p, const int32_t* want, int len, int b) {
  const int cap = p.cols * p.page;
  len = min(max(len, 0), cap);
  Change c;
  const int w = want[b];
  c.now = w < 0 || w > cap ? len : w;                               // (negative: stays; more than the table holds: refused)
  c.have = (len + p.page - 1) >> p.shift;
  c.need = (c.now + p.page - 1) >> p.shift;
  return c;
}

// Sum of a workgroup's threads up to and with this one, and of all (sh: a word a wavefront and one more)
__device__ inline int64_t block_scan(int64_t x, int64_t* sh, int64_t& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  x = scan64(x, lane);
  __syncthreads();
  if (lane == 63) sh[wave] = x;
  __syncthreads();
  int64_t before = 0;
  all = 0;
#pragma unroll
  for (int i = 0; i < PLAN_THREADS / 64; ++i) {
    const int64_t y = sh[i];
    before += i < wave ? y : 0;
    all += y;
  }
  return x + before;
}

// The sequence whose share of a running sum `ends` has x, and the sum before it
__device__ inline int share_of(const int64_t* ends, int n, int64_t x, int64_t& before) {
  int lo = 0, hi = n - 1;                                           // the first b with ends[b] > x
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (ends[mid] > x) hi = mid; else lo = mid + 1;
  }
  before = lo ? ends[lo - 1] : 0;
  return lo;
}

// The x-th page: from where it is given back, or from the stack, to where it is taken, or to the stack
__device__ inline void move_page(const DPages& p, const PagePlan& plan, const int64_t* gone_ends, const int64_t* more_ends, const int32_t* firsts, int64_t x) {
  const int64_t place = plan.count + plan.gone - 1 - x;             // from the top of the stack, with what is given back on it
  if (place < 0 || place >= p.pages) return;                        // (more given back than the pool has pages: not a table of this pool)
  int32_t id;
  if (x < plan.gone) {
    int64_t before;
    const int b = share_of(gone_ends, p.seqs, x, before);
    int32_t* const from = p.table + (int64_t)b * p.ld + firsts[b] + (x - before);
    id = *from;
    *from = -1;
    p.free[place] = id;
  } else {
    id = p.free[place];
  }
  if (x < plan.taken) {
    int64_t before;
    const int b = share_of(more_ends, p.seqs, x, before);
    p.table[(int64_t)b * p.ld + firsts[b] + (x - before)] = id;
  }
}

__global__ __launch_bounds__(PLAN_THREADS) void pages_plan_kernel(DPages p, const int32_t* want, int32_t* starts, uint8_t* ws, int inline_moves) {
  __shared__ int64_t sh[PLAN_THREADS / 64];
  PagePlan* const out = (PagePlan*)ws;
  int64_t* const gone_ends = (int64_t*)(ws + 64);
  int64_t* const more_ends = gone_ends + p.seqs;
  int32_t* const firsts = (int32_t*)(more_ends + p.seqs);
  const int tid = threadIdx.x, each = (p.seqs + PLAN_THREADS - 1) / PLAN_THREADS;
  const int b0 = (int)min((int64_t)tid * each, (int64_t)p.seqs), b1 = min(b0 + each, p.seqs);
  const int64_t count = min(max((int64_t)*p.count, (int64_t)0), p.pages);
  int64_t gone = 0, more = 0, all_gone, all_more;
  for (int b = b0; b < b1; ++b) {
    const Change c = change_of(p, want, p.lens[b], b);
    gone += max(c.have - c.need, 0);
    more += max(c.need - c.have, 0);
  }
  int64_t gone_at = block_scan(gone, sh, all_gone) - gone, more_at = block_scan(more, sh, all_more) - more;
  const int64_t there = min(count + all_gone, p.pages);
  // who is served, and what each gains
  int64_t gained = 0, taken = 0, all_gained, all_taken;
  int64_t at = more_at;
  for (int b = b0; b < b1; ++b) {
    const int len = min(max(p.lens[b], 0), p.cols * p.page);
    const Change c = change_of(p, want, len, b);
    const int m = max(c.need - c.have, 0);
    at += m;
    if (m == 0 || at <= there) {
      gained += max(c.now - len, 0);
      taken += m;
    }
  }
  int64_t row = block_scan(gained, sh, all_gained) - gained;
  block_scan(taken, sh, all_taken);
  if (starts && tid == 0) starts[p.seqs] = (int32_t)min(all_gained, (int64_t)0x7fffffff);
  at = more_at;
  int64_t took = min(more_at, all_taken);
  for (int b = b0; b < b1; ++b) {
    const int len = min(max(p.lens[b], 0), p.cols * p.page);
    const Change c = change_of(p, want, len, b);
    const int m = max(c.need - c.have, 0);
    at += m;
    const bool served = m == 0 || at <= there;
    if (starts) starts[b] = (int32_t)min(row, (int64_t)0x7fffffff);
    row += served ? max(c.now - len, 0) : 0;
    gone_at += max(c.have - c.need, 0);
    took += served ? m : 0;
    gone_ends[b] = gone_at;
    more_ends[b] = took;
    firsts[b] = min(c.have, c.need);
    p.lens[b] = served ? c.now : len;
  }
  PagePlan plan{count, all_gone, all_taken, max(all_gone, all_taken)};
  if (tid == 0) *p.count = (int32_t)max(there - all_taken, (int64_t)0);
  if (!inline_moves) {
    if (tid == 0) *out = plan;
    return;
  }
  __syncthreads();
  for (int64_t x = tid; x < plan.moves; x += PLAN_THREADS) move_page(p, plan, gone_ends, more_ends, firsts, x);
}

__global__ __launch_bounds__(256) void pages_move_kernel(DPages p, const uint8_t* ws) {
  const PagePlan plan = *(const PagePlan*)ws;
  const int64_t* const gone_ends = (const int64_t*)(ws + 64);
  const int64_t* const more_ends = gone_ends + p.seqs;
  const int32_t* const firsts = (const int32_t*)(more_ends + p.seqs);
  for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < plan.moves; x += (int64_t)gridDim.x * 256)
    move_page(p, plan, gone_ends, more_ends, firsts, x);
}

static int to_dpages(const cbk_pages* in, DPages* p, bool need_device_ptrs) {
  if (!in) return CBK_ERR_NULL;
  if (in->page < 16 || in->page > 256 || (in->page & (in->page - 1))) return CBK_ERR_LAYOUT;
  if (in->pages < 1 || in->pages > INT32_MAX || in->seqs < 0 || in->seqs >= 1 << 24 || in->table_cols < 0 || in->ld_table < in->table_cols)
    return CBK_ERR_SHAPE;
  if (in->table_cols > (1 << 30) / in->page) return CBK_ERR_SHAPE;
  if (need_device_ptrs && in->seqs > 0) {
    if (!in->lens || !in->free_pages || !in->free_count || (in->table_cols && !in->table)) return CBK_ERR_NULL;
    if (((uintptr_t)in->lens | (uintptr_t)in->table | (uintptr_t)in->free_pages | (uintptr_t)in->free_count) & 3) return CBK_ERR_ALIGN;
  }
  *p = DPages{(int32_t*)in->table, (int32_t*)in->lens, (int32_t*)in->free_pages, (int32_t*)in->free_count, in->ld_table, in->pages, in->seqs,
              in->table_cols, in->page, __builtin_ctz((unsigned)in->page)};
  return CBK_OK;
}

// ------------------------------------------------------------------ slots
constexpr int SLOT_ROWS = 4;                // rows a thread

// The last sequence that begins at or before row t (its offsets ascend); -1: none does
__device__ inline int begins_before(const DRows& r, int t, int lo, int hi) {
  while (lo < hi) {                                                 // the answer is in [lo - 1, hi - 1]
    const int mid = (lo + hi) / 2;
    if (r.starts[mid] <= t) lo = mid + 1; else hi = mid;
  }
  return lo - 1;
}

__global__ __launch_bounds__(256) void cache_slots_kernel(DRows r, int64_t pages, int shift, int64_t* slots, int32_t* positions) {
  const int64_t first = (int64_t)blockIdx.x * (256 * SLOT_ROWS);
  int lo = 0, hi = 0;
  if (r.starts) {                                                   // the sequences that the workgroup's rows can be of
    lo = begins_before(r, (int)first, 0, r.seqs + 1);
    hi = begins_before(r, (int)min(first + 256 * SLOT_ROWS, (int64_t)r.tokens) - 1, max(lo, 0), r.seqs + 1);
  }
#pragma unroll
  for (int u = 0; u < SLOT_ROWS; ++u) {
    const int64_t row = first + u * 256 + threadIdx.x;
    if (row >= r.tokens) return;
    const int t = (int)row;
    const int b = r.starts ? (lo == hi ? lo : begins_before(r, t, max(lo, 0), hi + 1)) : t / r.per;
    int64_t slot = -1;
    int pos = 0;
    if (b >= 0 && b < r.seqs) {
      const int end = r.starts ? r.starts[b + 1] : (b + 1) * r.per;
      const int64_t j = (int64_t)max(r.lens[b], 0) - ((int64_t)end - t);
      if (t < end) {                                                // (its begin is at or before t)
        pos = (int)max(j, (int64_t)0);
        if (j >= 0 && j < r.cap) {
          const int page = r.table[(int64_t)b * r.ld + (j >> shift)];
          if (page >= 0 && page < pages) slot = ((int64_t)page << shift) + (j & ((1 << shift) - 1));
        }
      }
    }
    if (slots) slots[row] = slot;
    if (positions) positions[row] = pos;
  }
}

}  // namespace cbk

using namespace cbk;

extern "C" {

size_t cbk_cache_pages_workspace_bytes(const cbk_pages* pages) {
  DPages p;
  if (to_dpages(pages, &p, false) || p.seqs == 0) return 0;
  return 64 + (size_t)p.seqs * 20;
}

int cbk_cache_pages(const cbk_pages* pages, const void* want, void* starts, void* workspace, size_t workspace_bytes, void* stream) {
  DPages p;
  const int rc = to_dpages(pages, &p, true);
  if (rc) return rc;
  if (p.seqs == 0) return CBK_OK;
  if (!want) return CBK_ERR_NULL;
  if (((uintptr_t)want | (uintptr_t)starts) & 3 || (uintptr_t)workspace & 255) return CBK_ERR_ALIGN;
  if (!workspace || workspace_bytes < 64 + (size_t)p.seqs * 20) return CBK_ERR_WORKSPACE;
  const int64_t entries = (int64_t)p.seqs * p.cols;                 // pages moved, at most
  const bool here = entries <= INLINE_MOVES;
  hipLaunchKernelGGL(pages_plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, (hipStream_t)stream, p, (const int32_t*)want, (int32_t*)starts,
                     (uint8_t*)workspace, (int)here);
  if (!here) {
    const int64_t most = (entries + 255) / 256;
    hipLaunchKernelGGL(pages_move_kernel, dim3((unsigned)(most < 1024 ? most : 1024)), dim3(256), 0, (hipStream_t)stream, p, (const uint8_t*)workspace);
  }
  return hipGetLastError() == hipSuccess ? CBK_OK : CBK_ERR_HIP;
}

int cbk_cache_slots(const cbk_rows* rows, int64_t pages, int page, void* slots, void* positions, void* stream) {
  if (page < 16 || page > 256 || (page & (page - 1))) return CBK_ERR_LAYOUT;
  if (pages < 1 || pages > INT32_MAX) return CBK_ERR_SHAPE;
  DRows r;
  const int rc = to_drows(rows, page, &r, true);
  if (rc) return rc;
  if (((uintptr_t)slots & 7) || ((uintptr_t)positions & 3)) return CBK_ERR_ALIGN;
  if (r.tokens == 0 || (!slots && !positions)) return CBK_OK;
  const unsigned grid = (unsigned)(((int64_t)r.tokens + 256 * SLOT_ROWS - 1) / (256 * SLOT_ROWS));
  hipLaunchKernelGGL(cache_slots_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, r, pages, __builtin_ctz((unsigned)page), (int64_t*)slots,
                     (int32_t*)positions);
  return hipGetLastError() == hipSuccess ? CBK_OK : CBK_ERR_HIP;
}

}  // extern "C"
