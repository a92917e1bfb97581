// One step of the page allocator on the device (b200_page_step): lengths in, block tables, slots and row maps out.
//
// Every CTA adds up all sequences (new rows, pages taken, pages given back: three prefix sums in shared memory) and then writes its share of
// the outputs; a row, a page or a place of the stack finds its sequence by binary search.  Table entries and places of the stack that are read
// (below a sequence's old end, below the old top) are not those that are written; lengths and the top may be written where they were read, by
// one CTA, after the others where there are any: a second launch of its own.
// 24 sequences that grow by one: 4.5 us; 2000, a tenth of them by prompts of up to 500 rows (102 thousand places of the row maps): 9.8 us.  Latencies bound the
// one, the searches' instructions the other.
#include "kv4.cuh"

#include <algorithm>

namespace b200 {

namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32, kMostCtas = 148;

struct Sums {
  long long rows, taken, given;
};
__device__ __forceinline__ Sums operator+(Sums a, Sums b) { return {a.rows + b.rows, a.taken + b.taken, a.given + b.given}; }
__device__ __forceinline__ Sums up(Sums a, int o) {
  return {__shfl_up_sync(0xffffffffu, a.rows, o), __shfl_up_sync(0xffffffffu, a.taken, o), __shfl_up_sync(0xffffffffu, a.given, o)};
}

// (positions and a page's size: 2^31 - 1 each at most)
__device__ __forceinline__ int pages_of(int positions, int page) { return (int)(((uint32_t)positions + (uint32_t)page - 1) / (uint32_t)page); }

// The last i of 0 .. n - 1 with first[i] <= x (first does not decrease, first[0] <= x < first[n]): never a sequence without any.
__device__ __forceinline__ int owner(const int32_t *first, int n, int x) {
  int lo = 0, hi = n;   // first[lo] <= x < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// what: 1 rows, tables, stack and status; 2 lengths and the stack's top
__global__ void __launch_bounds__(kThreads) page_step_kernel(const __grid_constant__ b200_page_step_args p, const int what) {
  extern __shared__ int32_t s_all[];
  __shared__ Sums s_warp[kWarps];
  __shared__ int s_over, s_state;
  const int n = p.n_seqs, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads / 32;
  int32_t *s_row = s_all, *s_take = s_row + n + 1, *s_give = s_take + n + 1, *s_held = s_give + n + 1;
  kernel_go();
  if (tid == 0)
    s_over = s_state = 0;
  kernel_wait();
  __syncthreads();

  // ---- this thread's sequences, then all before them ------------------------------------------------------------------------
  const int per = (n + threads - 1) / threads, first = min(n, tid * per), last = min(n, first + per);
  const long long room = (long long)p.table_stride * p.page;
  Sums mine{0, 0, 0};
  bool over = false, bad = false;
  const int n_free = *p.n_free;
  for (int s = first; s < last; ++s) {
    const long long held = p.held[s], add = p.add[s];
    bad = bad || held < 0 || held > room;
    over = over || (add > 0 && held + add > room);
    const long long have = (held + p.page - 1) / p.page;
    mine = mine + (add < 0 ? Sums{0, 0, have} : Sums{add, (held + add + p.page - 1) / p.page - have, 0});
    s_held[s] = (int32_t)held;
  }
  if (over)
    s_over = 1;
  if (bad)
    s_state = 1;
  Sums sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Sums v = up(sum, o);
    if (lane >= o)
      sum = sum + v;
  }
  if (lane == 31)
    s_warp[warp] = sum;
  __syncthreads();
  Sums upto = lane < warps ? s_warp[lane] : Sums{0, 0, 0};   // (every warp adds up the warps' sums)
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Sums v = up(upto, o);
    if (lane >= o)
      upto = upto + v;
  }
  const Sums total{__shfl_sync(0xffffffffu, upto.rows, 31), __shfl_sync(0xffffffffu, upto.taken, 31), __shfl_sync(0xffffffffu, upto.given, 31)};
  const int one = max(warp - 1, 0);
  Sums before{__shfl_sync(0xffffffffu, upto.rows, one), __shfl_sync(0xffffffffu, upto.taken, one), __shfl_sync(0xffffffffu, upto.given, one)};
  if (warp == 0)
    before = Sums{0, 0, 0};
  const int status = s_state || n_free < 0 || n_free > p.n_pages || n_free + total.given > p.n_pages ? B200_PAGES_STATE
                     : s_over                                                                        ? B200_PAGES_TABLE
                     : total.rows > p.max_rows                                                       ? B200_PAGES_ROWS
                     : total.taken > n_free + total.given                                            ? B200_PAGES_EXHAUSTED
                                                                                                     : B200_PAGES_OK;
  const bool ok = status == B200_PAGES_OK;
  if (ok) {   // (then all sums fit 32 bits)
    Sums at = {before.rows + sum.rows - mine.rows, before.taken + sum.taken - mine.taken, before.given + sum.given - mine.given};
    for (int s = first; s < last; ++s) {
      const int held = s_held[s], add = p.add[s], have = pages_of(held, p.page);
      s_row[s] = (int32_t)at.rows;
      s_take[s] = (int32_t)at.taken;
      s_give[s] = (int32_t)at.given;
      at = at + (add < 0 ? Sums{0, 0, have} : Sums{add, (int)(((long long)held + add + p.page - 1) / p.page) - have, 0});
    }
    if (tid == 0) {
      s_row[n] = (int32_t)total.rows;
      s_take[n] = (int32_t)total.taken;
      s_give[n] = (int32_t)total.given;
    }
  }
  __syncthreads();
  const int rows = ok ? (int)total.rows : 0, taken = ok ? (int)total.taken : 0, given = ok ? (int)total.given : 0, top = n_free + given;

  // ---- outputs ------------------------------------------------------------------------------------------------------------------
  auto returned = [&](int i) {   // the i-th page that is given back
    const int s = owner(s_give, n, i);
    return p.block_table[(int64_t)s * p.table_stride + i - s_give[s]];
  };
  auto new_page = [&](int i) {   // the i-th page that is taken
    const int at = top - 1 - i;
    return at < n_free ? p.free_pages[at] : returned(at - n_free);
  };
  const uint32_t at0 = blockIdx.x * threads + tid, step = gridDim.x * threads;   // (counted without sign: the last step of a loop may pass 2^31)
  if (what & 1) {
    for (uint32_t r = at0; r < (uint32_t)p.max_rows; r += step) {
      int64_t slot = -1;
      int seq = -1, pos = -1;
      if (r < (uint32_t)rows) {
        seq = owner(s_row, n, (int)r);
        pos = s_held[seq] + (int)r - s_row[seq];
        const int have = pages_of(s_held[seq], p.page), at = pos / p.page;
        const int page = at < have ? p.block_table[(int64_t)seq * p.table_stride + at] : new_page(s_take[seq] + at - have);
        slot = (int64_t)page * p.page + pos % p.page;
      }
      p.slots[r] = slot;
      if (p.row_seq != nullptr)
        p.row_seq[r] = seq;
      if (p.row_pos != nullptr)
        p.row_pos[r] = pos;
    }
    for (uint32_t i = at0; i < (uint32_t)taken; i += step) {
      const int s = owner(s_take, n, (int)i), have = pages_of(s_held[s], p.page);
      p.block_table[(int64_t)s * p.table_stride + have + (int)i - s_take[s]] = new_page((int)i);
    }
    for (uint32_t i = at0; (int64_t)i < (int64_t)given - taken; i += step)   // what stays on the stack of them
      p.free_pages[n_free + (int)i] = returned((int)i);
    for (uint32_t s = at0; s <= (uint32_t)n; s += step)
      p.row_start[s] = ok ? s_row[s] : 0;
    if (at0 == 0)
      *p.status = status;
  }
  if (what & 2) {
    for (uint32_t s = at0; s < (uint32_t)n; s += step)
      p.held_out[s] = !ok ? s_held[s] : s_row[s + 1] > s_row[s] ? s_held[s] + s_row[s + 1] - s_row[s] : p.add[s] < 0 ? 0 : s_held[s];
    if (at0 == 0)
      *p.n_free_out = ok ? top - taken : n_free;
  }
}

RaisedOn g_raised;

} // namespace

int page_step_launch(const b200_page_step_args &a, cudaStream_t st) {
  const int bytes = 4 * (4 * a.n_seqs + 3);
  if (int rc = raise_shared_limit(g_raised, (const void *)page_step_kernel, 4 * (4 * B200_PAGE_STEP_MAX_SEQS + 3)))
    return rc;
  // one CTA up to 2048 rows, a small one for a few sequences, then one for every 1024
  const int ctas = a.max_rows <= 2048 ? 1 : std::min(kMostCtas, (a.max_rows - 1) / kThreads + 1);
  const int threads = ctas == 1 && a.n_seqs <= 256 && a.max_rows <= 512 ? 256 : kThreads;
  const bool apart = ctas > 1 && (a.held_out == a.held || a.n_free_out == a.n_free);
  if (int rc = launch_after(page_step_kernel, dim3(ctas), threads, bytes, st, a, apart ? 1 : 3))
    return rc;
  return apart ? launch_after(page_step_kernel, dim3(1), kThreads, bytes, st, a, 2) : B200_OK;
}

} // namespace b200

using namespace b200;

extern "C" int b200_page_step(const b200_page_step_args *a, void *stream) {
  if (!a || !a->held || !a->add || !a->held_out || !a->block_table || !a->free_pages || !a->n_free || !a->n_free_out || !a->row_start || !a->status ||
      (a->max_rows > 0 && !a->slots))
    return fail(B200_EINVAL, "page_step: null pointer");
  if (a->n_seqs < 1 || a->page < 1 || a->table_stride < 1 || a->n_pages < 1 || a->max_rows < 0)
    return fail(B200_EINVAL, "page_step: %d sequences, pages of %d, tables of %d, %d pages, %d rows", a->n_seqs, a->page, a->table_stride, a->n_pages,
                a->max_rows);
  if ((int64_t)a->table_stride * a->page > INT32_MAX)
    return fail(B200_EINVAL, "page_step: a table of %d pages of %d positions: more than 2^31 - 1 positions", a->table_stride, a->page);
  if (a->n_seqs > B200_PAGE_STEP_MAX_SEQS)
    return fail(B200_ELIMIT, "page_step: %d sequences (at most %d)", a->n_seqs, B200_PAGE_STEP_MAX_SEQS);
  if (a->add == a->held_out || (const void *)a->slots == a->held || a->row_start == a->held_out)
    return fail(B200_EINVAL, "page_step: arrays overlap");
  if (((uintptr_t)a->held | (uintptr_t)a->add | (uintptr_t)a->held_out | (uintptr_t)a->block_table | (uintptr_t)a->free_pages | (uintptr_t)a->n_free |
       (uintptr_t)a->n_free_out | (uintptr_t)a->row_start | (uintptr_t)a->row_seq | (uintptr_t)a->row_pos | (uintptr_t)a->status) &
          3 ||
      (uintptr_t)a->slots & 7)
    return fail(B200_EINVAL, "page_step: a pointer is not aligned to its elements");
  if (int rc = ensure_device())
    return rc;
  return page_step_launch(*a, (cudaStream_t)stream);
}
