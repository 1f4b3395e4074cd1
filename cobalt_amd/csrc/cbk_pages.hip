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
// Both move few bytes; they are bound by their launches and by the loads that wait for one another: a step of 32 sequences 3.5 us in one kernel, 1024
// sequences of up to 60000 tokens in pages of 16 (3.8 million entries, 15 % of them end, 15 % begin) 4.7 + 6.5 us; slots of 32 rows 2.8, of a million rows 6.6 us.
#include "cbk_cache_attn.h"
#include "cbk_cache_check.h"

namespace cbk {

struct DPages {
  int32_t *table, *lens, *free, *count;
  int64_t ld, pages;
  int seqs, cols, page, shift;
};
// Pages on the stack before, given back, taken (and the larger of the two); all below 2^31, as the table's entries are
struct PagePlan { int64_t count, gone, taken, moves; };
// Behind the plan in the workspace, or in LDS: running sums over the sequences, and the entry that a sequence's pages leave from or go to
struct PageEnds { int32_t *gone, *more, *first; };

// Entries and rows of a table whose pages the first launch moves.  A step moves few of a table's pages, and one launch takes 6.4 us with 256 threads, 7.8 with
// 1024 (timed with the call), two 10 to 11; where all move, one workgroup is the bottleneck: 2048 entries 10.2 and 8.5 us, 4096 entries 14 and 9.6, 8192
// entries 24 and 12, 32768 entries 76 and 28.  So 256 threads to a quarter of the entries, 1024 to all of them, two launches above.
constexpr int INLINE_ENTRIES = 8192, INLINE_SEQS = 1024;

struct Change { int len, now, have, need; };                        // tokens before and asked for, and their pages
__device__ inline Change change_of(const DPages& p, const int32_t* want, int b) {
  const int cap = p.cols * p.page, w = want[b];
  Change c;
  c.len = min(max(p.lens[b], 0), cap);
  c.now = w < 0 || w > cap ? c.len : w;                             // (negative: stays; more than the table holds: refused)
  c.have = (c.len + p.page - 1) >> p.shift;
  c.need = (c.now + p.page - 1) >> p.shift;
  return c;
}

template <class X>
__device__ inline X wave_scan(X x, int lane) {                      // sum of the lanes up to and with this one
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const X y = __shfl_up(x, o);
    x += lane >= o ? y : 0;
  }
  return x;
}
// Two such sums over a workgroup's T threads, and of all
template <int T, class X>
__device__ inline void block_scan(X& x, int& y, X& all_x, int& all_y, X* shx, int* shy) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  x = wave_scan(x, lane);
  y = wave_scan(y, lane);
  if (lane == 63) { shx[wave] = x; shy[wave] = y; }
  __syncthreads();
  X bx = 0;
  int by = 0;
  all_x = 0; all_y = 0;
#pragma unroll
  for (int i = 0; i < T / 64; ++i) {
    if (i < wave) { bx += shx[i]; by += shy[i]; }
    all_x += shx[i]; all_y += shy[i];
  }
  x += bx; y += by;
}

// The first b in [lo, hi] with ends[b] > x (there is one)
__device__ inline int share_of(const int32_t* ends, int lo, int hi, int x) {
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (ends[mid] > x) hi = mid; else lo = mid + 1;
  }
  return lo;
}
// The entry of the table that the x-th page of a list leaves or goes to, if sequence b has it
__device__ inline int32_t* entry_of(const DPages& p, const int32_t* ends, const int32_t* first, int b, int x) {
  return p.table + (int64_t)b * p.ld + first[b] + (x - (b ? ends[b - 1] : 0));
}

// The pages from the base-th on, U a thread of T, neighbours side by side, from the place each leaves (the table, or the stack) to the one it goes
// to (the stack, the table): the loads of all first.  Those given back are of sequences g0 to g1, those taken of m0 to m1.
template <int U, int T>
__device__ inline void move_pages(const DPages& p, const PagePlan& plan, const PageEnds& ends, int64_t base, int g0, int g1, int m0, int m1) {
  int32_t id[U];
  int32_t* from[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t x = base + u * T + threadIdx.x, place = plan.count + plan.gone - 1 - x;   // from the top of the stack, with what is given back on it
    from[u] = nullptr;
    if (x >= plan.moves || place < 0 || place >= p.pages) continue; // (more given back than the pool has pages: not a table of this pool)
    if (x < plan.gone) from[u] = entry_of(p, ends.gone, ends.first, share_of(ends.gone, g0, g1, (int)x), (int)x);
    id[u] = *(x < plan.gone ? from[u] : p.free + place);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t x = base + u * T + threadIdx.x, place = plan.count + plan.gone - 1 - x;
    if (x >= plan.moves || place < 0 || place >= p.pages) continue;
    int32_t* const to = x < plan.taken ? entry_of(p, ends.more, ends.first, share_of(ends.more, m0, m1, (int)x), (int)x) : nullptr;
    if (x < plan.gone) {
      *from[u] = -1;
      p.free[place] = id[u];
    }
    if (to) *to = id[u];
  }
}

// T threads; ONE: no more sequences than that, one a thread; HERE: the pages are moved too, not by a second launch
template <int T, bool ONE, bool HERE>
__global__ __launch_bounds__(T) void pages_plan_kernel(DPages p, const int32_t* want, int32_t* starts, uint8_t* ws) {
  __shared__ int sha[T / 64], shb[T / 64], shd[T / 64];
  __shared__ int64_t shc[T / 64];
  __shared__ int32_t ends_sh[HERE ? 3 * T : 1];
  int32_t* const of = HERE ? ends_sh : (int32_t*)(ws + sizeof(PagePlan));
  const int n = HERE ? T : p.seqs;
  const PageEnds ends{of, of + n, of + 2 * n};
  const int tid = threadIdx.x, each = ONE ? 1 : (p.seqs + T - 1) / T;
  const int b0 = ONE ? min(tid, p.seqs) : (int)min((int64_t)tid * each, (int64_t)p.seqs), b1 = min(b0 + each, p.seqs);
  const int64_t count = min(max((int64_t)*p.count, (int64_t)0), p.pages);
  Change mine{};
  int gone = 0, more = 0, all_gone, all_more;
  for (int b = b0; b < b1; ++b) {
    mine = change_of(p, want, b);
    gone += max(mine.have - mine.need, 0);
    more += max(mine.need - mine.have, 0);
  }
  int gone_at = gone, more_at = more;
  block_scan<T>(gone_at, more_at, all_gone, all_more, sha, shb);
  gone_at -= gone; more_at -= more;                                 // before this thread's sequences
  const int64_t there = min(count + all_gone, p.pages);
  // who is served, and what each gains
  int64_t gained = 0, all_gained;
  int taken = 0, all_taken, at = more_at;
  for (int b = b0; b < b1; ++b) {
    const Change c = ONE ? mine : change_of(p, want, b);
    const int m = max(c.need - c.have, 0);
    at += m;
    if (m == 0 || at <= there) { gained += max(c.now - c.len, 0); taken += m; }
  }
  int64_t row = gained;
  int took = taken;
  block_scan<T>(row, took, all_gained, all_taken, shc, shd);
  row -= gained; took -= taken;
  constexpr int64_t most = 0x7fffffff;
  if (starts && tid == 0) starts[p.seqs] = (int32_t)min(all_gained, most);
  at = more_at;
  for (int b = b0; b < b1; ++b) {
    const Change c = ONE ? mine : change_of(p, want, b);
    const int m = max(c.need - c.have, 0);
    at += m;
    const bool served = m == 0 || at <= there;
    if (starts) starts[b] = (int32_t)min(row, most);
    row += served ? max(c.now - c.len, 0) : 0;
    gone_at += max(c.have - c.need, 0);
    took += served ? m : 0;
    ends.gone[b] = gone_at;
    ends.more[b] = took;
    ends.first[b] = min(c.have, c.need);
    p.lens[b] = served ? c.now : c.len;
  }
  const PagePlan plan{count, all_gone, all_taken, max(all_gone, all_taken)};
  if (tid == 0) *p.count = (int32_t)max(there - all_taken, (int64_t)0);
  if constexpr (!HERE) {
    if (tid == 0) *(PagePlan*)ws = plan;
    return;
  }
  __syncthreads();
  for (int64_t base = 0; base < plan.moves; base += T) move_pages<1, T>(p, plan, ends, base, 0, p.seqs - 1, 0, p.seqs - 1);
}

// For two numbers that are the same in all lanes, the first i < n whose entry of an ascending list passes them (n: none does):
// a 64th of the list a step.  above(i, x): whether entry i passes x.
template <class F>
__device__ inline void first_above(int n, int lane, int x0, int x1, int& i0, int& i1, F above) {
  int lo0 = 0, lo1 = 0, width = n;                                  // the answer is in [lo, lo + width]
  while (width > 0) {
    const int step = (width + 63) / 64;
    const int a = lo0 + (lane + 1) * step - 1, b = lo1 + (lane + 1) * step - 1;
    const bool pa = a >= n || above(a, x0), pb = b >= n || above(b, x1);
    const uint64_t ma = __ballot(pa), mb = __ballot(pb);
    lo0 += (ma ? __ffsll((unsigned long long)ma) - 1 : 64) * step;
    lo1 += (mb ? __ffsll((unsigned long long)mb) - 1 : 64) * step;
    width = step - 1;
  }
  i0 = min(lo0, n); i1 = min(lo1, n);
}

constexpr int MOVES = 2;                    // pages a thread at a time (half a million moved: 1 22.2 us, 2 21.8, 4 22.4)

// A workgroup takes neighbours, of few sequences.  SMALL: at most INLINE_SEQS sequences, whose sums come into LDS at once instead of by loads that wait for one another.
template <bool SMALL>
__global__ __launch_bounds__(256) void pages_move_kernel(DPages p, uint8_t* ws) {
  __shared__ int32_t of_sh[SMALL ? 3 * INLINE_SEQS : 1];
  int32_t* const of = (int32_t*)(ws + sizeof(PagePlan));
  const int lane = threadIdx.x & 63;
  constexpr int N = SMALL ? 3 * INLINE_SEQS / 256 : 1;
  int32_t part[N];
  if constexpr (SMALL)
#pragma unroll
    for (int i = 0; i < N; ++i) part[i] = of[min(i * 256 + (int)threadIdx.x, 3 * p.seqs - 1)];
  const PagePlan plan = *(const PagePlan*)ws;
  if ((int64_t)blockIdx.x * (256 * MOVES) >= plan.moves) return;
  if constexpr (SMALL) {
#pragma unroll
    for (int i = 0; i < N; ++i) of_sh[i * 256 + threadIdx.x] = part[i];
    __syncthreads();
  }
  int32_t* const sums = SMALL ? of_sh : of;
  const PageEnds ends{sums, sums + p.seqs, sums + 2 * p.seqs};
  for (int64_t base = (int64_t)blockIdx.x * (256 * MOVES); base < plan.moves; base += (int64_t)gridDim.x * (256 * MOVES)) {
    const int x0 = (int)base, x1 = (int)min(base + 256 * MOVES, plan.moves) - 1;
    int g0 = 0, g1 = 0, m0 = 0, m1 = 0;                             // the sequences that they can be of
    if (x0 < plan.gone) first_above(p.seqs, lane, x0, (int)min((int64_t)x1, plan.gone - 1), g0, g1, [&](int i, int x) { return ends.gone[i] > x; });
    if (x0 < plan.taken) first_above(p.seqs, lane, x0, (int)min((int64_t)x1, plan.taken - 1), m0, m1, [&](int i, int x) { return ends.more[i] > x; });
    move_pages<MOVES, 256>(p, plan, ends, base, g0, g1, m0, m1);
  }
}

static size_t pages_workspace(const DPages& p) {                    // 0: the pages are moved by the first launch
  const bool here = p.seqs <= INLINE_SEQS && (int64_t)p.seqs * p.cols <= INLINE_ENTRIES;
  return here || p.seqs == 0 ? 0 : sizeof(PagePlan) + (size_t)p.seqs * 12;
}

static int to_dpages(const cbk_pages* in, DPages* p, bool need_device_ptrs) {
  if (!in) return CBK_ERR_NULL;
  if (in->page < 16 || in->page > 256 || (in->page & (in->page - 1))) return CBK_ERR_LAYOUT;
  if (in->pages < 1 || in->pages > INT32_MAX || in->seqs < 0 || in->seqs >= 1 << 24 || in->table_cols < 0 || in->ld_table < in->table_cols)
    return CBK_ERR_SHAPE;
  if (in->table_cols > (1 << 30) / in->page || (int64_t)in->seqs * in->table_cols > INT32_MAX) return CBK_ERR_SHAPE;
  if (need_device_ptrs && in->seqs > 0) {
    if (!in->lens || !in->free_pages || !in->free_count || (in->table_cols && !in->table)) return CBK_ERR_NULL;
    if (((uintptr_t)in->lens | (uintptr_t)in->table | (uintptr_t)in->free_pages | (uintptr_t)in->free_count) & 3) return CBK_ERR_ALIGN;
  }
  *p = DPages{(int32_t*)in->table, (int32_t*)in->lens, (int32_t*)in->free_pages, (int32_t*)in->free_count, in->ld_table, in->pages, in->seqs,
              in->table_cols, in->page, __builtin_ctz((unsigned)in->page)};
  return CBK_OK;
}

// ------------------------------------------------------------------ slots
constexpr int SLOT_ROWS = 2;                // rows a thread (a million rows of 1024 sequences: 1 11.1 us, 2 9.6, 4 10.3; of 8 sequences 9.0, 8.3, 8.5)

// SMALL: at most SLOT_SEQS sequences with offsets, which come into LDS at once
constexpr int SLOT_SEQS = 768;
template <bool SMALL>
__global__ __launch_bounds__(256) void cache_slots_kernel(DRows r, int64_t pages, int shift, int64_t* slots, int32_t* positions) {
  __shared__ int32_t starts_sh[SMALL ? SLOT_SEQS + 256 : 1], lens_sh[SMALL ? SLOT_SEQS : 1];
  const int64_t first = (int64_t)blockIdx.x * (256 * SLOT_ROWS);
  if constexpr (SMALL) {
    int32_t a[SLOT_SEQS / 256 + 1], b[SLOT_SEQS / 256];
#pragma unroll
    for (int i = 0; i <= SLOT_SEQS / 256; ++i) a[i] = r.starts[min(i * 256 + (int)threadIdx.x, r.seqs)];
#pragma unroll
    for (int i = 0; i < SLOT_SEQS / 256; ++i) b[i] = r.lens[min(i * 256 + (int)threadIdx.x, r.seqs - 1)];
#pragma unroll
    for (int i = 0; i <= SLOT_SEQS / 256; ++i) starts_sh[i * 256 + threadIdx.x] = a[i];
#pragma unroll
    for (int i = 0; i < SLOT_SEQS / 256; ++i) lens_sh[i * 256 + threadIdx.x] = b[i];
    __syncthreads();
  }
  const int32_t *const starts = SMALL ? starts_sh : r.starts, *const lens = SMALL ? lens_sh : r.lens;
  int lo = 0, hi = 0;                                               // offsets that pass the workgroup's first and last row: its rows are of sequences [lo - 1, hi)
  if (starts)
    first_above(r.seqs + 1, threadIdx.x & 63, (int)first, (int)min(first + 256 * SLOT_ROWS, (int64_t)r.tokens) - 1, lo, hi,
                [&](int i, int t) { return starts[i] > t; });
  int64_t slot[SLOT_ROWS];
  int pos[SLOT_ROWS];
  int page[SLOT_ROWS];
#pragma unroll
  for (int u = 0; u < SLOT_ROWS; ++u) {
    const int64_t row = first + u * 256 + threadIdx.x;
    const int t = (int)min(row, (int64_t)r.tokens - 1);
    int b = hi;
    if (SMALL || r.starts) {
      for (int l = lo; l < b;) {                                    // (starts[hi] passes t if anything does)
        const int mid = (l + b) / 2;
        if (starts[mid] > t) b = mid; else l = mid + 1;
      }
      --b;
    } else {
      b = t / r.per;
    }
    const bool is = b >= 0 && b < r.seqs;
    const int at = is ? b : 0, end = !is ? 0 : r.starts ? starts[b + 1] : (b + 1) * r.per;
    const int64_t j = is ? (int64_t)max(lens[at], 0) - ((int64_t)end - t) : -1;
    pos[u] = is && t < end ? (int)max(j, (int64_t)0) : 0;           // (its begin is at or before t)
    page[u] = is && t < end && j >= 0 && j < r.cap ? r.table[(int64_t)b * r.ld + (j >> shift)] : -1;
    slot[u] = j & ((1 << shift) - 1);
  }
#pragma unroll
  for (int u = 0; u < SLOT_ROWS; ++u) {
    const int64_t row = first + u * 256 + threadIdx.x;
    if (row >= r.tokens) return;
    if (slots) slots[row] = page[u] >= 0 && page[u] < pages ? ((int64_t)page[u] << shift) + slot[u] : -1;
    if (positions) positions[row] = pos[u];
  }
}

}  // namespace cbk

using namespace cbk;

extern "C" {

size_t cbk_cache_pages_workspace_bytes(const cbk_pages* pages) {
  DPages p;
  return to_dpages(pages, &p, false) ? 0 : pages_workspace(p);
}

int cbk_cache_pages(const cbk_pages* pages, const void* want, void* starts, void* workspace, size_t workspace_bytes, void* stream) {
  DPages p;
  const int rc = to_dpages(pages, &p, true);
  if (rc) return rc;
  if (p.seqs == 0) return CBK_OK;
  if (!want) return CBK_ERR_NULL;
  if (((uintptr_t)want | (uintptr_t)starts) & 3 || (uintptr_t)workspace & 255) return CBK_ERR_ALIGN;
  const size_t need = pages_workspace(p);
  if (need > workspace_bytes || (need && !workspace)) return CBK_ERR_WORKSPACE;
  uint8_t* const ws = need ? (uint8_t*)workspace : nullptr;
  const hipStream_t st = (hipStream_t)stream;
  auto plan = [&](auto kernel, int threads) { hipLaunchKernelGGL(kernel, dim3(1), dim3(threads), 0, st, p, (const int32_t*)want, (int32_t*)starts, ws); };
  if (!need && p.seqs <= 256 && (int64_t)p.seqs * p.cols <= INLINE_ENTRIES / 4) plan(pages_plan_kernel<256, true, true>, 256);
  else if (!need) plan(pages_plan_kernel<1024, true, true>, 1024);
  else if (p.seqs <= 256) plan(pages_plan_kernel<256, true, false>, 256);
  else if (p.seqs <= 1024) plan(pages_plan_kernel<1024, true, false>, 1024);
  else plan(pages_plan_kernel<1024, false, false>, 1024);
  if (need) {
    const int64_t most = ((int64_t)p.seqs * p.cols + 256 * MOVES - 1) / (256 * MOVES);   // pages moved, at most
    const dim3 grid((unsigned)(most < 4096 ? (most ? most : 1) : 4096));
    if (p.seqs <= INLINE_SEQS) hipLaunchKernelGGL(pages_move_kernel<true>, grid, dim3(256), 0, st, p, ws);
    else hipLaunchKernelGGL(pages_move_kernel<false>, grid, dim3(256), 0, st, p, ws);
  }
  return hipGetLastError() == hipSuccess ? CBK_OK : CBK_ERR_HIP;
}

int cbk_cache_slots(const cbk_rows* rows, int64_t pages, int page, void* slots, void* positions, void* stream) {
  if (page < 16 || page > 256 || (page & (page - 1))) return CBK_ERR_LAYOUT;
  if (pages < 1 || pages > INT32_MAX || (rows && rows->seqs >= 1 << 30)) return CBK_ERR_SHAPE;
  DRows r;
  const int rc = to_drows(rows, page, &r, true);
  if (rc) return rc;
  if (((uintptr_t)slots & 7) || ((uintptr_t)positions & 3)) return CBK_ERR_ALIGN;
  if (r.tokens == 0 || (!slots && !positions)) return CBK_OK;
  const unsigned grid = (unsigned)(((int64_t)r.tokens + 256 * SLOT_ROWS - 1) / (256 * SLOT_ROWS));
  if (r.starts && r.seqs > 0 && r.seqs <= SLOT_SEQS)
    hipLaunchKernelGGL(cache_slots_kernel<true>, dim3(grid), dim3(256), 0, (hipStream_t)stream, r, pages, __builtin_ctz((unsigned)page),
                       (int64_t*)slots, (int32_t*)positions);
  else
    hipLaunchKernelGGL(cache_slots_kernel<false>, dim3(grid), dim3(256), 0, (hipStream_t)stream, r, pages, __builtin_ctz((unsigned)page),
                       (int64_t*)slots, (int32_t*)positions);
  return hipGetLastError() == hipSuccess ? CBK_OK : CBK_ERR_HIP;
}

}  // extern "C"
