// Paged key/value cache in 4 bits: the plan of a step, rows in and out, attention (dfl_kv4.h has
// the format, the layout and the arithmetic of the work split).
#include "dfl_kv4.h"

#include <float.h>

#include "dfl_common.h"

namespace dfl {

namespace {

typedef __bf16 bf16_t;
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ step
//
// Block tables and slot maps from the lengths alone, in whole numbers.  With pages(n) =
// ceil(n / page), sequence s puts back its pages from place pages(keep) on and then takes
// pages(keep + grow) - pages(keep).  The free pages are a stack: the pages put back lie on it with
// the first sequence's first page on top, and are handed out again from the top, sequence by
// sequence, so a step that puts back what it takes leaves every table as it was.
//
// Phases, each over all sequences: scan (totals, then offsets), check, move, rows.  The check looks
// at every page id that the step will touch, and puts the pages that come back on the stack, above
// its top as it was; only when all are pages of the pool does anything else change (if not, those
// places of the stack, which hold no page, are cleared).  A phase reads what the one before wrote,
// so for many sequences or rows they are launches of their own; up to STEP_ONE_SEQS and
// STEP_ONE_ROWS one workgroup does them all, with the offsets in LDS.  In both forms the pages and
// rows of all sequences are numbered through and found by a search in the offsets, so that no thread
// waits for a long sequence.
//
// Bound by latencies: launches and a handful of reads that follow on each other.  One workgroup
// against launches, us (sequences x new rows of each; every page put back and taken again):
//   8 x 16 5.2, 12.4;  256 x 16 11.6, 19.1;  1024 x 8 16.9, 23.3;  8 x 1024 11.3, 14.5;
//   1024 x 32 39.5, 22.2;  64 x 512 29.3, 15.9;  8 x 4096 22.3, 14.5.
// (Of these the check takes 0.2 in one workgroup, where a thread keeps the move that it has looked at
// in registers, and 1 in launches.)

constexpr int STEP_ONE_SEQS = 1024, STEP_ONE_ROWS = 8192;
// Steps of one workgroup that move more pages than it has threads: a thread has STEP_N moves under
// way at once, and STEP_L threads clear what a table gives up.  64 tables of 256 pages put back 36 us
// (one move at once 53), 1024 of 64 61 (79); STEP_L 4, 8, 16, 64: 1024 of 8 16.5, 17.2, 18.7, 28.6,
// one of 1000 13.9, 10.8, 9.2, 7.9.
constexpr int STEP_N = 4, STEP_L = 16;

// Sums over the workgroup's threads of three counts at once (inclusive), and their totals.
struct Sum3 { long long a, b, c; };
DFL_DEV Sum3 block_scan3(Sum3 v, Sum3* lds /* 16 */, Sum3& total) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, nw = blockDim.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long x = __shfl_up(v.a, o, 64), y = __shfl_up(v.b, o, 64), z = __shfl_up(v.c, o, 64);
    if (lane >= o) { v.a += x; v.b += y; v.c += z; }
  }
  __syncthreads();
  if (lane == 63) lds[wv] = v;
  __syncthreads();
  total = Sum3{0, 0, 0};
  for (int w = 0; w < nw; ++w) {
    const Sum3 x = lds[w];
    if (w < wv) { v.a += x.a; v.b += x.b; v.c += x.c; }
    total.a += x.a; total.b += x.b; total.c += x.c;
  }
  return v;
}

DFL_DEV bool step_ask(const Kv4StepArgs& a, int s, Kv4Ask& q) {
  const int len = a.lens[s];
  return kv4_ask(len, a.keep ? a.keep[s] : len, a.grow ? a.grow[s] : 0, a.width, a.page_shift, q);
}
// Why a step cannot be done (0: it can), from its totals.
DFL_DEV int step_error(const Kv4StepArgs& a, bool bad, const Sum3& all, int n_free) {
  int err = bad ? KV4_ERR_LEN : 0;
  // (freed pages beyond the pool, or a free count beyond it: the state is not a step's)
  if (n_free < 0 || n_free > a.n_pages || n_free + all.a > a.n_pages) err |= KV4_ERR_PAGE;
  else if (all.b > n_free + all.a) err |= KV4_ERR_POOL;
  if (all.c > a.max_rows) err |= KV4_ERR_ROWS;
  return err;
}
// The last of the ascending n numbers at (n > 0, at[0] <= v) that is not above v, of equals the last.
DFL_DEV int step_search(const int* at, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= v) lo = mid; else hi = mid;
  }
  return lo;
}
// Offsets of all sequences: kept lengths, pages put back and taken before each (n_seq), new rows
// before each (n_seq + 1).
struct StepView { int *base, *f_at, *t_at, *starts; };
// Moves i, i + n, .. of a step, N of them at once (the searches do not wait for each other): page i of
// those put back and page i of those taken, which is the same one if both are there (they have one
// place on the stack, `top` less i with the stack's top after all are put back).
template <int N> struct StepMoves {
  int *from[N], *to[N];   // their places in the tables (null: from the stack, it stays there)
  int page[N];
  bool again[N];          // the step puts another page into `from`
};
template <int N>
DFL_DEV void step_search(const int* at, int n_seq, int i, int n, int past, int (&s)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) s[k] = 0;
  for (int step = n_seq > 1 ? 1 << (31 - __clz(n_seq - 1)) : 0; step; step >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int mid = min(s[k] + step, n_seq - 1);
      if (at[mid] <= min(i + k * n, past - 1)) s[k] = mid;
    }
}
// Where pages that are put back come from.
template <int N>
DFL_DEV void step_from(const Kv4StepArgs& a, const StepView& v, int i, int n, int freed, StepMoves<N>& m) {
  int s[N];
  step_search<N>(v.f_at, a.n_seq, i, n, freed, s);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int at = kv4_pages(v.base[s[k]], a.page_shift) + (i + k * n - v.f_at[s[k]]);
    m.again[k] = at < kv4_pages(v.base[s[k]] + (v.starts[s[k] + 1] - v.starts[s[k]]), a.page_shift);
    m.from[k] = i + k * n < freed ? a.table + (long long)s[k] * a.width + at : nullptr;
  }
}
// Where pages that are taken go.
template <int N>
DFL_DEV void step_to(const Kv4StepArgs& a, const StepView& v, int i, int n, int taken, StepMoves<N>& m) {
  int s[N];
  step_search<N>(v.t_at, a.n_seq, i, n, taken, s);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int at = kv4_pages(v.base[s[k]], a.page_shift) + (i + k * n - v.t_at[s[k]]);
    m.to[k] = i + k * n < taken ? a.table + (long long)s[k] * a.width + at : nullptr;
  }
}
DFL_DEV bool step_page_ok(const Kv4StepArgs& a, int page) { return page >= 0 && page < a.n_pages; }
// The pages, and whether all are the pool's.
template <int N>
DFL_DEV bool step_look(const Kv4StepArgs& a, const StepView& v, int i, int n, int freed, int taken, int top, StepMoves<N>& m) {
  step_from<N>(a, v, i, n, freed, m);
  bool ok = true;
#pragma unroll
  for (int k = 0; k < N; ++k)
    m.page[k] = m.from[k] ? *m.from[k] : i + k * n < taken ? a.free_pages[top - (i + k * n)] : 0;
#pragma unroll
  for (int k = 0; k < N; ++k) ok = step_page_ok(a, m.page[k]) && ok;
  return ok;
}
// With the pages that are put back on the stack.
template <int N>
DFL_DEV bool step_put(const Kv4StepArgs& a, const StepView& v, int i, int n, int freed, int taken, int top) {
  StepMoves<N> m;
  const bool ok = step_look<N>(a, v, i, n, freed, taken, top, m);
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (m.from[k]) a.free_pages[top - (i + k * n)] = m.page[k];
  return ok;
}
template <int N>
DFL_DEV void step_move(const Kv4StepArgs& a, int i, int n, int top, const StepMoves<N>& m) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    if (m.from[k] && !m.again[k]) *m.from[k] = -1;
    if (m.to[k]) *m.to[k] = m.page[k];
    if (m.from[k] || m.to[k]) a.free_pages[top - (i + k * n)] = m.to[k] ? -1 : m.page[k];
  }
}
// After step_put: the pages that are taken, and the places that are given up.
template <int N>
DFL_DEV void step_take(const Kv4StepArgs& a, const StepView& v, int i, int n, int taken, int top) {
  StepMoves<N> m;
  step_to<N>(a, v, i, n, taken, m);
#pragma unroll
  for (int k = 0; k < N; ++k) m.page[k] = m.to[k] ? a.free_pages[top - (i + k * n)] : 0;
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (m.to[k]) {
      *m.to[k] = m.page[k];
      a.free_pages[top - (i + k * n)] = -1;
    }
}
DFL_DEV void step_clear(const Kv4StepArgs& a, const StepView& v, int i, int freed) {
  StepMoves<1> m;
  step_from<1>(a, v, i, 0, freed, m);
  if (!m.again[0]) *m.from[0] = -1;
}
// The page that new rows of sequence s go on in; 0 if there is none.
DFL_DEV int step_kept(const Kv4StepArgs& a, const StepView& v, int s) {
  if (v.starts[s] == v.starts[s + 1] || !(v.base[s] & ((1 << a.page_shift) - 1))) return 0;
  return a.table[(long long)s * a.width + (v.base[s] >> a.page_shift)];
}
// Slot and position of new row r of sequence s.
struct StepRow { int slot, pos; };
DFL_DEV StepRow step_row(const Kv4StepArgs& a, const StepView& v, int s, int r) {
  const int pos = v.base[s] + (r - v.starts[s]);
  const int pg = a.table[(long long)s * a.width + (pos >> a.page_shift)];
  return StepRow{(pg << a.page_shift) + (pos & ((1 << a.page_shift) - 1)), pos};
}

// One workgroup, a thread to a sequence.  Eight sequences of up to 16 new rows: 11.1 us with the
// offsets in memory and a wave to each sequence's pages, 5.3 so.
__global__ __launch_bounds__(1024) void kv4_step_one_kernel(Kv4StepArgs a) {
  __shared__ Sum3 lds[16];
  __shared__ int offsets[4][STEP_ONE_SEQS + 1];
  const StepView v{offsets[0], offsets[1], offsets[2], offsets[3]};
  const int s = threadIdx.x, nt = blockDim.x;
  Kv4Ask q{0, 0, 0, 0};
  bool bad = false;
  if (s < a.n_seq) bad = !step_ask(a, s, q);
  const int n_free = *a.n_free;
  Sum3 all;
  const Sum3 in = block_scan3(Sum3{q.freed, q.taken, q.grow}, lds, all);
  int err = step_error(a, __syncthreads_or(bad), all, n_free);
  if (!err) {
    if (s < a.n_seq) {
      v.base[s] = q.keep;
      v.f_at[s] = (int)(in.a - q.freed);
      v.t_at[s] = (int)(in.b - q.taken);
      v.starts[s] = (int)(in.c - q.grow);
    }
    if (s == 0) v.starts[a.n_seq] = (int)all.c;
    const int freed = (int)all.a, taken = (int)all.b, moves = max(freed, taken), top = n_free + freed - 1;
    __syncthreads();
    const int kept = s < a.n_seq ? step_kept(a, v, s) : 0;
    bool ok = true;
    StepMoves<1> m;   // (of few moves, in registers)
    if (moves <= nt) {
      ok = step_look<1>(a, v, s, nt, freed, taken, top, m);
      step_to<1>(a, v, s, nt, taken, m);
    } else {
      for (int i = s; i < moves; i += STEP_N * nt) ok = step_put<STEP_N>(a, v, i, nt, freed, taken, top) && ok;
    }
    ok = step_page_ok(a, kept) && ok;
    if (__syncthreads_or(!ok)) {
      err = KV4_ERR_PAGE;
      if (moves > nt)
        for (int i = s; i < freed; i += nt) a.free_pages[top - i] = -1;
    } else {
      if (moves <= nt) step_move<1>(a, s, nt, top, m);
      else {
        for (int i = s; i < taken; i += STEP_N * nt) step_take<STEP_N>(a, v, i, nt, taken, top);
        for (int k = s / STEP_L; k < a.n_seq; k += nt / STEP_L) {   // (stores: nothing waits)
          const int kept_k = kv4_pages(v.base[k], a.page_shift);
          const int from = kv4_pages(v.base[k] + (v.starts[k + 1] - v.starts[k]), a.page_shift);
          const int past = kept_k + (k + 1 < a.n_seq ? v.f_at[k + 1] : freed) - v.f_at[k];
          for (int at = from + s % STEP_L; at < past; at += STEP_L) a.table[(long long)k * a.width + at] = -1;
        }
      }
      if (s < a.n_seq) a.lens[s] = q.keep + q.grow;
      if (s == 0) *a.n_free = (int)(n_free + all.a - all.b);
      __syncthreads();
    }
  }
  if (s < a.n_seq) a.starts[s] = err ? 0 : v.starts[s];
  if (s == 0) {
    a.starts[a.n_seq] = err ? 0 : (int)all.c;
    if (err) atomicOr(a.err, err);
  }
  const int rows = err ? 0 : (int)all.c;
  for (int r = s; r < a.max_rows; r += nt) {
    StepRow x{-1, -1};
    if (r < rows) x = step_row(a, v, step_search(v.starts, a.n_seq, r), r);
    a.slots[r] = x.slot;
    a.positions[r] = x.pos;
  }
}

// The same in launches.  scratch: the scan's error, pages put back and taken, free pages before, the
// check's error; then the offsets but for the rows', which are a.starts.
DFL_DEV StepView step_view(const Kv4StepArgs& a) {
  return StepView{a.scratch + 5, a.scratch + 5 + a.n_seq, a.scratch + 5 + 2 * a.n_seq, a.starts};
}
__global__ __launch_bounds__(1024) void kv4_step_scan_kernel(Kv4StepArgs a) {
  __shared__ Sum3 lds[16];
  const StepView v = step_view(a);
  const int nt = blockDim.x;
  Sum3 all{0, 0, 0};
  int bad = 0;
  for (int s0 = 0; s0 < a.n_seq; s0 += nt) {
    const int s = s0 + threadIdx.x;
    Kv4Ask q{0, 0, 0, 0};
    if (s < a.n_seq && !step_ask(a, s, q)) bad = 1;
    Sum3 t;
    const Sum3 in = block_scan3(Sum3{q.freed, q.taken, q.grow}, lds, t);
    if (s < a.n_seq) {
      v.base[s] = q.keep;
      v.f_at[s] = (int)(all.a + in.a - q.freed);
      v.t_at[s] = (int)(all.b + in.b - q.taken);
      v.starts[s] = (int)(all.c + in.c - q.grow);
    }
    all.a += t.a; all.b += t.b; all.c += t.c;
  }
  const int n_free = *a.n_free;
  const int err = step_error(a, __syncthreads_or(bad), all, n_free);
  if (threadIdx.x == 0) {
    v.starts[a.n_seq] = (int)all.c;
    a.scratch[0] = err;
    a.scratch[1] = (int)all.a;
    a.scratch[2] = (int)all.b;
    a.scratch[3] = n_free;
    a.scratch[4] = 0;
    if (err) atomicOr(a.err, err);
  }
}
__global__ __launch_bounds__(256) void kv4_step_check_kernel(Kv4StepArgs a) {
  if (a.scratch[0]) return;
  const StepView v = step_view(a);
  const int n_free = a.scratch[3], freed = a.scratch[1], taken = a.scratch[2], top = n_free + freed - 1;
  const int t = blockIdx.x * 256 + threadIdx.x, nt = gridDim.x * 256;
  bool ok = true;
  for (int s = t; s < a.n_seq; s += nt) ok = step_page_ok(a, step_kept(a, v, s)) && ok;
  for (int i = t; i < max(freed, taken); i += nt) ok = step_put<1>(a, v, i, nt, freed, taken, top) && ok;
  if (!ok) {
    atomicOr(a.scratch + 4, KV4_ERR_PAGE);
    atomicOr(a.err, KV4_ERR_PAGE);
  }
}
__global__ __launch_bounds__(256) void kv4_step_move_kernel(Kv4StepArgs a) {
  const StepView v = step_view(a);
  const int n_free = a.scratch[3], freed = a.scratch[1], taken = a.scratch[2], top = n_free + freed - 1;
  const int t = blockIdx.x * 256 + threadIdx.x, nt = gridDim.x * 256;
  if (a.scratch[0] | a.scratch[4]) {   // no rows, and the stack as it was
    for (int s = t; s <= a.n_seq; s += nt) v.starts[s] = 0;
    if (!a.scratch[0])
      for (int i = t; i < freed; i += nt) a.free_pages[top - i] = -1;
    return;
  }
  for (int i = t; i < taken; i += nt) step_take<1>(a, v, i, nt, taken, top);
  for (int i = t; i < freed; i += nt) step_clear(a, v, i, freed);
  for (int s = t; s < a.n_seq; s += nt) a.lens[s] = v.base[s] + (v.starts[s + 1] - v.starts[s]);
  if (t == 0) *a.n_free = n_free + freed - taken;
}
// 1024 rows a workgroup, 4 a thread; the sequences of the first and the last are found first, 64
// places at a time, those between them are few.  Two million rows of 1024 sequences: 17 us with a
// search of all sequences for each row, 11.2 so (16 MB, 3.3 us of a copy's time).
constexpr int STEP_ROWS = 1024;
__global__ __launch_bounds__(256) void kv4_step_rows_kernel(Kv4StepArgs a) {
  const StepView v = step_view(a);
  const int lane = threadIdx.x & 63, rows = v.starts[a.n_seq];
  for (long long c = (long long)blockIdx.x * STEP_ROWS; c < a.max_rows; c += (long long)gridDim.x * STEP_ROWS) {
    const int c0 = (int)c;   // (at most 2^31 - 1024)
    int s = 0, last = 0;
    if (c0 < rows) {
      const int r1 = min(c0 + (STEP_ROWS - 1), rows - 1);
      int n = a.n_seq, m = a.n_seq;   // sequences that s and last are still among
      while (n > 1 || m > 1) {
        const int i = (n + 63) >> 6, j = (m + 63) >> 6;
        const bool x = lane * i < n && v.starts[s + min(lane * i, n - 1)] <= c0;
        const bool y = lane * j < m && v.starts[last + min(lane * j, m - 1)] <= r1;
        const int k = max(0, __popcll(__ballot(x)) - 1) * i, l = max(0, __popcll(__ballot(y)) - 1) * j;
        s += k; n = min(i, n - k);
        last += l; m = min(j, m - l);
      }
    }
    StepRow x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = c0 + 256 * k + threadIdx.x;
      x[k] = StepRow{-1, -1};
      if (r < rows) x[k] = step_row(a, v, s + step_search(v.starts + s, last - s + 1, r), r);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = c0 + 256 * k + threadIdx.x;
      if (r < a.max_rows) {
        a.slots[r] = x[k].slot;
        a.positions[r] = x[k].pos;
      }
    }
  }
}

// ------------------------------------------------------------------ rows in and out
//
// A workgroup has 32 rows of one head's keys or values, 8 lanes a row; a lane has 8 values of the
// row's first half and 8 of its second, so that each load of a wave takes 8 times 128 bytes (fp16)
// in a row and each store of codes the 16-byte groups of 8 rows.  Groups are four lanes.  65521
// rows of 8 heads (bf16, 268 MB to 71 MB): 82 us to append, 72 to read, 4.2 and 4.7 TB/s (copies
// reach 5.1); 16 lanes a row, each of 8 values in a row, took 112 and 111.

template <int DT> struct RowT;
template <> struct RowT<0> { typedef float t; };
template <> struct RowT<1> { typedef half_t t; };
template <> struct RowT<2> { typedef bf16_t t; };

template <int DT>
DFL_DEV void load8(const void* base, long long at, float (&x)[8]) {
  typedef typename RowT<DT>::t E;
  typedef E vec __attribute__((ext_vector_type(DT == 0 ? 4 : 8)));
  const vec* p = reinterpret_cast<const vec*>(reinterpret_cast<const E*>(base) + at);
#pragma unroll
  for (int i = 0; i < (DT == 0 ? 2 : 1); ++i) {
    const vec v = p[i];
#pragma unroll
    for (int j = 0; j < (DT == 0 ? 4 : 8); ++j) x[4 * i + j] = (float)v[j];
  }
}

// Where a slot's row lies; false (and the error bit) for a slot outside the pool, -1 is no error.
DFL_DEV bool slot_at(const Kv4RowsArgs& a, int slot, int head, unsigned char*& blk, int& r) {
  if (slot < 0 || slot >= (a.n_pages << a.page_shift)) {
    if (slot != -1) atomicOr(a.err, KV4_ERR_SLOT);
    return false;
  }
  const int in = slot & ((1 << a.page_shift) - 1);
  blk = a.pool + kv4_block_at(kv4_block_no(slot >> a.page_shift, a.n_kv, head, a.page_shift - 5, in >> 5));
  r = in & 31;
  return true;
}

constexpr int ROWS_WG = 32;   // rows of a workgroup

template <int DT>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4RowsArgs a) {
  const int head = blockIdx.x >> 1, v = blockIdx.x & 1;
  const int part = threadIdx.x & 7;
  for (long long row = (long long)blockIdx.y * ROWS_WG + (threadIdx.x >> 3); row < a.rows;
       row += (long long)gridDim.y * ROWS_WG) {
    unsigned char* blk;
    int r;
    if (!slot_at(a, a.slots[row], head, blk, r)) continue;   // (one answer for the row's lanes)
    const long long at = row * (v ? a.v_row : a.k_row) + head * (v ? a.v_head : a.k_head) + 8 * part;
    float x[2][8];
    load8<DT>(v ? a.v : a.k, at, x[0]);
    load8<DT>(v ? a.v : a.k, at + 64, x[1]);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      // |x| orders as its bits do; an infinity or a NaN is at or past 0x7f800000
      int top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, (int)(__float_as_uint(x[half][j]) & 0x7fffffffu));
      top = max(top, __shfl_xor(top, 1, 64));
      top = max(top, __shfl_xor(top, 2, 64));
      const bool bad = top >= 0x7f800000;
      const int b = bad ? 255 : max(0, (top >> 23) - 2 + ((top & 0x7fffff) > 0x600000 ? 1 : 0));
      const float s = __uint_as_float((uint32_t)b << 23);   // (the conversion reads the exponent alone)
      uint32_t w = 0;
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[half][0], x[half][1], s, 0);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[half][2], x[half][3], s, 1);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[half][4], x[half][5], s, 2);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[half][6], x[half][7], s, 3);
      const int g = 2 * half + (part >> 2);
      *reinterpret_cast<uint32_t*>(blk + kv4_code_at(r, g, v) + 4 * (part & 3)) = bad ? 0u : w;
      if ((part & 3) == 0) blk[kv4_scale_at(r, g, v)] = (unsigned char)b;
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4RowsArgs a) {
  const int head = blockIdx.x >> 1, v = blockIdx.x & 1;
  const int part = threadIdx.x & 7;
  for (long long row = (long long)blockIdx.y * ROWS_WG + (threadIdx.x >> 3); row < a.rows;
       row += (long long)gridDim.y * ROWS_WG) {
    unsigned char* blk;
    int r;
    const bool ok = slot_at(a, a.slots[row], head, blk, r);
    typedef typename RowT<DT>::t E;
    E* out = reinterpret_cast<E*>(v ? a.ov : a.ok) + (row * a.n_kv + head) * KV4_D + 8 * part;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int g = 2 * half + (part >> 2);
      uint32_t w = 0;
      float s = 1.f;
      if (ok) {
        w = *reinterpret_cast<const uint32_t*>(blk + kv4_code_at(r, g, v) + 4 * (part & 3));
        s = __uint_as_float((uint32_t)blk[kv4_scale_at(r, g, v)] << 23);
      }
      if constexpr (DT == 0) {
        const floatx2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0);
        const floatx2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
        const floatx2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2);
        const floatx2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
        reinterpret_cast<floatx4*>(out + 64 * half)[0] = (floatx4){p0.x, p0.y, p1.x, p1.y};
        reinterpret_cast<floatx4*>(out + 64 * half)[1] = (floatx4){p2.x, p2.y, p3.x, p3.y};
      } else {
        u32x4 o;
        if constexpr (DT == 1) {
          o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0));
          o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1));
          o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2));
          o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3));
        } else {
          o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
          o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
          o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
          o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
        }
        *reinterpret_cast<u32x4*>(out + 64 * half) = o;
      }
    }
  }
}

// ------------------------------------------------------------------ attention
//
// O = softmax(scale * Q K^T) V over each sequence's cached rows, K and V in 4 bits.
//
// A unit is a tile of query rows (row = token * ratio + head in group) of one sequence and kv
// head; a workgroup takes a run of key blocks of a unit (32 keys each).  Of a block:
//   S^T = K Q^T   matrix instructions with keys on the M axis;
//   softmax       fp32, log2 domain, the reference maximum raised only when a block exceeds it by
//                 more than KV4_SLACK; weights rounded to the type of Q, and summed as rounded;
//   O^T += V^T P  V converted in registers, written to LDS as rows, read back transposed
//                 (ds_read_b64_tr_b16); P from the S^T accumulators as they lie: the rows of V that
//                 a lane's weights stand for are those whose keys its accumulators hold.
// Two kernels: kv4_attn_kernel for up to 32 rows (single tokens, small blocks), where HBM and
// latency count, and kv4_tile_kernel for more, where the matrix and vector units do.

constexpr float KV4_SLACK = 6.f;
// Weights are 2^(s - m + KV4_LIFT) <= 2^15 for a reference m: fp16 then keeps 2^-23 of the
// largest weight as a normal number and 2^-34 as the rounding of the smallest, so that a million
// keys far below one large one still add up.
constexpr float KV4_LIFT = 9.f;

template <typename T> struct Mat;
template <> struct Mat<half_t> {
  // Codes convert to half their value: a group whose largest fp16 value is above 3.5 * 2^14 holds
  // 2^16, past fp16's range.  (The product keeps the exponent 255 of NaN.)
  // V below 2^-21 are rounded to steps of 2^-23, half an output's smallest step off at most.
  static constexpr float kUnit = 0.5f;
  static constexpr uint32_t kVNan = 142;   // (the largest code is 4 or 6: halved, 2^16 or more)
  static constexpr float kVUp = 0x1p113f;  // 2^(255 - kVNan)
  // Whether codes of a group with exponent byte b, halved, may not be numbers of fp16 (those of 105,
  // down to 2^-24, to 141, up to 49152, are; groups of zeros have 0, which stands for 2^-127).
  static DFL_DEV bool past(uint32_t b) { return (b - 105u > 141u - 105u) & (b != 0); }
  typedef half8_t v8;
  typedef half2_t v2;
  static DFL_DEV floatx4 mfma(v8 a, v8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static DFL_DEV floatx16 mfma(v8 a, v8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static DFL_DEV v8 dequant(uint32_t w, float s) {
    const v2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0);
    const v2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1);
    const v2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2);
    const v2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3);
    return (v8){p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
  }
  static DFL_DEV float sum2(v2 p, float c) {
    return __builtin_amdgcn_fdot2(p, (v2){(half_t)1.f, (half_t)1.f}, c, false);
  }
};
template <> struct Mat<bf16_t> {
  static constexpr float kUnit = 1.f;
  static constexpr uint32_t kVNan = 253;   // (2^128 or more)
  static constexpr float kVUp = 0x1p2f;
  static DFL_DEV bool past(uint32_t) { return false; }   // (all of them are bf16's)
  typedef bf16x8_t v8;
  typedef bf16x2_t v2;
  static DFL_DEV floatx4 mfma(v8 a, v8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static DFL_DEV floatx16 mfma(v8 a, v8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static DFL_DEV v8 dequant(uint32_t w, float s) {
    const v2 p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0);
    const v2 p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1);
    const v2 p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2);
    const v2 p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
    return (v8){p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
  }
  static DFL_DEV float sum2(v2 p, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(p, (v2){(bf16_t)1.f, (bf16_t)1.f}, c, false);
  }
};
// Two 4-key halves of a V operand, read transposed: the lanes' addresses are those of rows, what
// they get is 4 keys of one value.
template <typename T>
DFL_DEV typename Mat<T>::v8 read_vt(const unsigned char* lo, const unsigned char* hi) {
  typedef __attribute__((address_space(3))) short4_t* lp;
  typedef short short8_t __attribute__((ext_vector_type(8)));
  const short4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)lo);
  const short4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)hi);
  return __builtin_bit_cast(typename Mat<T>::v8, (short8_t){a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w});
}
DFL_DEV float exponent(uint32_t b) { return __uint_as_float(b << 23); }
// What V converts with.  A group of exponent byte M::kVNan or more has a value past the type's range:
// it is NaN as a whole, so that its infinity does not reach rows that do not see it, as 0 * infinity
// (where some row does not, groups that are NaN are left out and set by hand).
template <typename M>
DFL_DEV float v_unit(uint32_t b) {
  return exponent(b) * M::kVUp * (M::kUnit / M::kVUp);
}

// An int that no kernel writes while this one runs, at a uniform address: a scalar load.
DFL_DEV int load_const(const int* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) int*>(reinterpret_cast<uintptr_t>(p));
}
// The lane's number, anew: what is made of it in a walk's steps is not kept in registers between them.
DFL_DEV int lane_again() {
  int lane;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
  return lane;
}
DFL_DEV long long lane_value(long long v, int lane) {
  const uint32_t lo = __builtin_amdgcn_ds_bpermute(4 * lane, (int)v);
  const uint32_t hi = __builtin_amdgcn_ds_bpermute(4 * lane, (int)(v >> 32));
  return (long long)((unsigned long long)hi << 32 | lo);
}
// Inclusive sum over the wave's lanes, and a lane's.
DFL_DEV long long wave_scan_ll(long long v) {
  const int lane = lane_again();
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long x = lane_value(v, lane - o);
    if (lane >= o) v += x;
  }
  return v;
}
DFL_DEV long long pick_ll(long long v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)v, lane), hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
  return (long long)((unsigned long long)hi << 32 | lo);
}
DFL_DEV int pick(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
// Sequences one lane each, 64 at a time: sequence s0 + lane's row range and length, and its places.
struct Lanes { int q0, q1, len; long long cost; };
DFL_DEV Lanes attn_lanes(const Kv4AttnArgs& a, int tile_rows, int s0, bool report) {
  const int s = s0 + lane_again();
  Lanes l{0, 0, 0, 0};
  if (s < a.n_seq) {
    l = Lanes{a.starts[s], a.starts[s + 1], a.lens[s], 0};
    const Kv4Seq q = kv4_seq(l.q0, l.q1, l.len, a.n_rows, a.width, a.page_shift, a.n_heads / a.n_kv,
                             tile_rows, a.causal);
    if (q.bad && report) atomicOr(a.err, KV4_ERR_PAGE);
    l.cost = kv4_cost(q, a.n_kv);
  }
  return l;
}
// The sequence among the 64 whose places hold pos (in: their inclusive sums, after acc places):
// its number of them and the places before it; -1 if there is none.
DFL_DEV int attn_among(const Lanes& l, long long in, long long acc, long long pos, long long& before) {
  const unsigned long long past = __ballot(acc + in > pos);
  if (!past) return -1;
  const int k = __ffsll((unsigned long long)past) - 1;
  before = acc + pick_ll(in - l.cost, k);
  return k;
}
// The tile of a head at its place r: the last that has begun.  Every lane tries one, 64 at a time.
DFL_DEV int attn_tile(const Kv4Seq& s, long long r) {
  const int lane = lane_again();
  int lo = 0, n = s.tiles;   // the tile is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 63) >> 6;
    const int t = lo + lane * step;
    const unsigned long long begun = __ballot(t < lo + n && kv4_begun(s, t, r));
    const int k = max(0, __popcll(begun) - 1);
    n = min(step, n - k * step);
    lo += k * step;
  }
  return lo;
}

// Visible keys of a token of a sequence (they grow with the token).
DFL_DEV int attn_visible(const Kv4AttnArgs& a, const Kv4Seq& q, int token) {
  return a.causal ? max(0, min(q.len, q.len - q.qlen + token + 1)) : q.len;
}

// A unit, and where its places are.
struct Unit {
  Kv4Seq sq;
  int s, head, tile, nblk;
  long long r0;        // place of its first block
  long long head0;     // place at which its head begins
};
DFL_DEV void unit_places(Unit& u) {
  const long long p0 = kv4_places(u.sq, u.tile);
  u.nblk = (int)(kv4_places(u.sq, u.tile + 1) - p0) - KV4_PAD;
  u.r0 = u.head0 + p0 + KV4_PAD;
}
// The unit of sequence s (row range and length q0, q1, len) at a place, the sequence's first being
// at place `at`.
DFL_DEV void unit_of(const Kv4AttnArgs& a, int tile_rows, int s, int q0, int q1, int len, long long at,
                     long long pos, Unit& u) {
  u.s = s;
  u.sq = kv4_seq(q0, q1, len, a.n_rows, a.width, a.page_shift, a.n_heads / a.n_kv, tile_rows, a.causal);
  const long long of_head = kv4_places(u.sq, u.sq.tiles);
  u.head = (int)kv4_div(pos - at, of_head);
  u.head0 = at + u.head * of_head;
  u.tile = u.sq.tiles > 1 ? __builtin_amdgcn_readfirstlane(attn_tile(u.sq, pos - u.head0)) : 0;
  unit_places(u);
}
// The unit at a place (uniform); false if there is none.
DFL_DEV bool unit_at(const Kv4AttnArgs& a, int tile_rows, long long pos, Unit& u) {
  long long acc = 0;
  for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
    const Lanes l = attn_lanes(a, tile_rows, s0, false);
    const long long in = wave_scan_ll(l.cost);
    long long at;
    const int k = attn_among(l, in, acc, pos, at);
    if (k >= 0) {
      unit_of(a, tile_rows, s0 + k, pick(l.q0, k), pick(l.q1, k), pick(l.len, k), at, pos, u);
      return true;
    }
    acc += pick_ll(in, 63);
  }
  return false;
}

// A worker's walk over its places: run after run of blocks [b0, b1) of a unit.
struct Run : Unit {
  int b0, b1;
  int whole;           // all of the unit's blocks
};
struct Walk { long long pos, end, per; };
// Which worker a workgroup is.  Workgroups go to the 8 dies of the chip in turn, each with an L2 of
// its own, and workers that follow on each other read the same keys (the tiles of a head): so
// each die has an eighth of all places, one after the other.  (In turn, and
// so, us: one token over 500 keys 11.0, 10.6; 32 rows of 40 heads over 32800 keys 55.4, 53.6; two
// prompts of 4096 and 777 rows 196, 190.)
static_assert(KV4_CUS % 8 == 0, "workers in eight parts");
DFL_DEV int worker_of(const Kv4AttnArgs& a, int workgroup) {
  return (workgroup & 7) * (a.workers >> 3) + (workgroup >> 3);
}
// Begins at the worker's first place; false if it has none.
DFL_DEV bool walk_begin(const Kv4AttnArgs& a, int tile_rows, Walk& k, Run& r) {
  const bool report = blockIdx.x == 0;
  Lanes l = attn_lanes(a, tile_rows, 0, report);
  long long in = wave_scan_ll(l.cost);
  long long total = pick_ll(in, 63);
  for (int s0 = 64; s0 < a.n_seq; s0 += 64)
    total += pick_ll(wave_scan_ll(attn_lanes(a, tile_rows, s0, report).cost), 63);
  k.per = kv4_per(total, a.workers);
  k.pos = worker_of(a, blockIdx.x) * k.per;
  k.end = min(total, k.pos + k.per);
  if (k.pos >= k.end) return false;
  if (a.n_seq > 64) return unit_at(a, tile_rows, k.pos, r);
  long long at;
  const int s = attn_among(l, in, 0, k.pos, at);
  if (s < 0) return false;
  unit_of(a, tile_rows, s, pick(l.q0, s), pick(l.q1, s), pick(l.len, s), at, k.pos, r);
  return true;
}
// The run of the unit at hand; false if only places before its first block are this worker's.
DFL_DEV bool walk_run(const Walk& k, Run& r) {
  r.b0 = (int)max(0ll, k.pos - r.r0);
  r.b1 = (int)min((long long)r.nblk, k.end - r.r0);
  r.whole = r.b0 == 0 && r.b1 == r.nblk;
  return r.b1 > 0;
}
// On to the next unit; false at the end.  (Everything here is uniform over the workgroup.)
DFL_DEV bool walk_next(const Kv4AttnArgs& a, int tile_rows, Walk& k, Run& r) {
  k.pos = r.r0 + r.nblk;
  if (k.pos >= k.end) return false;
  if (r.tile + 1 < r.sq.tiles) {
    ++r.tile;
  } else if (r.head + 1 < a.n_kv) {
    r.head0 = k.pos;
    ++r.head;
    r.tile = 0;
  } else {
    // the next sequence that has rows begins here
    for (int s0 = r.s + 1;; s0 += 64) {
      if (s0 >= a.n_seq) return false;
      const Lanes l = attn_lanes(a, tile_rows, s0, false);
      const unsigned long long some = __ballot(l.cost > 0);
      if (!some) continue;
      const int i = __ffsll(some) - 1;
      r.s = s0 + i;
      r.sq = kv4_seq(pick(l.q0, i), pick(l.q1, i), pick(l.len, i), a.n_rows, a.width, a.page_shift,
                     a.n_heads / a.n_kv, tile_rows, a.causal);
      r.head = r.tile = 0;
      r.head0 = k.pos;
      break;
    }
  }
  unit_places(r);
  return true;
}
// What the merge needs to know of the unit that a worker begins and others go on with (w1: the
// last of them; -1: there is none).  The notes lie behind the partials.
DFL_DEV Kv4Note* kv4_notes(const Kv4AttnArgs& a, int tile_rows) {
  return reinterpret_cast<Kv4Note*>(a.ws + 2ll * a.workers * kv4_piece_floats(tile_rows));
}
DFL_DEV void walk_no_note(const Kv4AttnArgs& a, int tile_rows, int wave) {
  if (wave == 0 && lane_again() == 0) kv4_notes(a, tile_rows)[worker_of(a, blockIdx.x)].w1 = -1;
}
DFL_DEV void walk_note(const Kv4AttnArgs& a, int tile_rows, int wave, long long per, const Run& r) {
  if (wave || lane_again()) return;
  kv4_notes(a, tile_rows)[worker_of(a, blockIdx.x)] = Kv4Note{
      (int)kv4_div(r.r0 + r.nblk - 1, per), r.head, r.tile, r.sq.q0, r.sq.qlen, r.sq.len, 0, 0};
}
// The page of block b of a run's keys; -1: there is no such page (its keys are absent).
DFL_DEV int page_of(const Kv4AttnArgs& a, const Run& r, int b) {
  const int page = load_const(a.table + (long long)r.s * a.width + (b >> (a.page_shift - 5)));
  return page >= a.n_pages || page < 0 ? -1 : page;
}
// Address of block b in a page (for page -1 some address in the pool).
DFL_DEV const unsigned char* block_in(const Kv4AttnArgs& a, const Run& r, int b, int page) {
  const int sh = a.page_shift - 5;
  return a.pool + kv4_block_at(kv4_block_no(max(page, 0), a.n_kv, r.head, sh, b & ((1 << sh) - 1)));
}

// ---- up to 32 query rows
//
// The four waves of a workgroup take every fourth block of a run each, a wave's whole work on a
// block in its own registers and its own 9 KiB of LDS (no barrier in the loop); their states are
// joined at the run's end.  The next block's codes load while this one computes.
//
// Long caches are bound by HBM: sixteen tokens of 64 heads over 65 thousand keys each (1.14 GB) take
// 203 us, 5.6 TB/s; 64 ragged tokens (379 MB) 80, 4.7.  One token over 500 keys takes 7.4 us, a
// chain of latencies: launch, lengths, pages, blocks, join.

constexpr int VROW = 288;                 // bytes of a V row in LDS: 8 banks apart, so that the 8
                                          // rows of a half wave's transposing read do not collide
constexpr int VWAVE = 32 * VROW;

template <typename T, int NT>
__global__ __launch_bounds__(256, NT == 1 ? 3 : 2) void kv4_attn_kernel(Kv4AttnArgs a) {
  typedef Mat<T> M;
  typedef typename M::v8 v8;
  typedef typename M::v2 v2;
  constexpr int ROWS = 16 * NT;
  __shared__ __attribute__((aligned(16))) unsigned char lds[4 * VWAVE];
  __shared__ float mls[4][2][ROWS];
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ratio = a.n_heads / a.n_kv;
  unsigned char* vbuf = lds + wv * VWAVE;
  const unsigned char* vread = vbuf + (4 * g + (i >> 2)) * VROW + 8 * (i & 3);
  unsigned char* vwrite = vbuf + i * VROW + 64 * g;
  const float scale = a.scale_log2 * (1.f / M::kUnit);

  Walk walk;
  Run run;
  bool more = walk_begin(a, ROWS, walk, run);
  walk_no_note(a, ROWS, wv);
  for (; more; more = walk_next(a, ROWS, walk, run)) {
    if (!walk_run(walk, run)) break;   // (the worker's last places)
    if (run.b0 == 0 && !run.whole) walk_note(a, ROWS, wv, walk.per, run);
    const Kv4Seq& sq = run.sq;
    // query fragments: step st covers values 32 g + 8 st ..; visible keys of this lane's rows
    v8 qf[NT][4];
    int vis[NT];
    const int n_row = sq.qlen * ratio;   // rows of the sequence and kv head
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = min((run.tile * NT + n) * 16 + i, n_row - 1);
      const int tok = r / ratio;
      const T* qp = reinterpret_cast<const T*>(a.q) + (long long)(sq.q0 + tok) * a.q_row +
                    (long long)(run.head * ratio + r - tok * ratio) * a.q_head + 32 * g;
#pragma unroll
      for (int st = 0; st < 4; ++st) qf[n][st] = *reinterpret_cast<const v8*>(qp + 8 * st);
      vis[n] = attn_visible(a, sq, tok);
    }
    const int vmin = attn_visible(a, sq, run.tile * ROWS / ratio);
    const int vmax = attn_visible(a, sq, (min(run.tile * ROWS + ROWS, n_row) - 1) / ratio);

    floatx4 o[NT][8];
    float mrun[NT], lrun[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      mrun[n] = -FLT_MAX;
      lrun[n] = 0.f;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[n][d] = (floatx4){0.f, 0.f, 0.f, 0.f};
    }
    u32x4 kc[2], vc[2];
    uint32_t sc = 0;
    int pg = 0;
    auto load_block = [&](int b) {
      pg = page_of(a, run, b);
      const unsigned char* p = block_in(a, run, b, pg);
      kc[0] = load_vec(p + kv4_code_at(i, g, 0));
      kc[1] = load_vec(p + kv4_code_at(16 + i, g, 0));
      vc[0] = load_vec(p + kv4_code_at(i, g, 1));
      vc[1] = load_vec(p + kv4_code_at(16 + i, g, 1));
      sc = *reinterpret_cast<const uint32_t*>(p + KV4_SC + 4 * lane);
    };
    // blocks that no row of the tile sees add nothing
    const int b_end = min(run.b1, (vmax + KV4_KEYS - 1) / KV4_KEYS);
    int b = run.b0 + wv;
    if (b < b_end) load_block(b);
    for (; b < b_end; b += 4) {
      u32x4 k0 = kc[0], k1 = kc[1], v0 = vc[0], v1 = vc[1];
      uint32_t s4 = sc;
      const int page = pg;
      if (b + 4 < b_end) load_block(b + 4);
      const int kbase = b * KV4_KEYS;
      const bool masked = kbase + KV4_KEYS > vmin || page < 0;   // (uniform)
      if (masked) {
        if (page < 0 && lane == 0) atomicOr(a.err, KV4_ERR_PAGE);
        // V rows that nobody may see, and groups that stand for NaN (they must not reach a row
        // that does not see them, as 0 * NaN): zero codes; the rows that do see one are set here
        const int lim = page < 0 ? 0 : sq.len;
        const bool gone0 = kbase + i >= lim, gone1 = kbase + 16 + i >= lim;
        const bool nan0 = !gone0 && ((s4 >> 16) & 255) >= M::kVNan, nan1 = !gone1 && (s4 >> 24) >= M::kVNan;
        if (gone0 || nan0) { v0 = (u32x4){0, 0, 0, 0}; s4 &= 0xff00ffffu; }
        if (gone1 || nan1) { v1 = (u32x4){0, 0, 0, 0}; s4 &= 0x00ffffffu; }
        const float nan = __builtin_nanf("");
        if (__ballot(nan0 || nan1)) {
#pragma unroll 1
          for (int key = 0; key < KV4_KEYS; ++key) {
            const unsigned long long hit = __ballot(key < 16 ? nan0 : nan1) >> (key & 15);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              if (kbase + key < vis[n])
                static_for<0, 4>([&](auto group) {
                  constexpr int gr = group;
                  if ((hit >> (16 * gr)) & 1)
                    o[n][2 * gr] = o[n][2 * gr + 1] = (floatx4){nan, nan, nan, nan};
                });
          }
        }
      }
      const uint32_t e0 = s4 & 255u, e1 = (s4 >> 8) & 255u;
      const float sv0 = v_unit<M>((s4 >> 16) & 255u), sv1 = v_unit<M>(s4 >> 24);
      floatx4 sa[NT], sb[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) sa[n] = sb[n] = (floatx4){0.f, 0.f, 0.f, 0.f};
      // Keys past fp16's range, in a cache that was filled from bf16 or fp32: as bf16, which holds
      // them, against Q in two parts of bf16, which hold every fp16 value.  To see that there are none
      // costs, us: eight blocks of 8 rows 26.3 for 25.8, one token over 500 keys 10.6 for 10.3 (code);
      // this path for all blocks 27.7 and 10.9.
      const bool wide = __ballot(M::past(e0) | M::past(e1)) != 0;
      if (__builtin_expect(wide, 0)) {
        typedef Mat<bf16_t> W;
        static_for<0, 4>([&](auto step) {
          constexpr int st = step;
          const bf16x8_t f0 = W::dequant(k0[st], exponent(e0)), f1 = W::dequant(k1[st], exponent(e1));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            u32x4 qw = __builtin_bit_cast(u32x4, qf[n][st]);
            asm volatile("" : "+v"(qw));   // (made here, not kept over the loop)
            const v8 x = __builtin_bit_cast(v8, qw);
            bf16x8_t hi, lo;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              hi[j] = (bf16_t)(float)x[j];
              lo[j] = (bf16_t)((float)x[j] - (float)hi[j]);
            }
            sa[n] = W::mfma(f0, hi, W::mfma(f0, lo, sa[n]));
            sb[n] = W::mfma(f1, hi, W::mfma(f1, lo, sb[n]));
          }
        });
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          sa[n] *= M::kUnit;
          sb[n] *= M::kUnit;
        }
      } else {
        const float sk0 = M::kUnit * exponent(e0), sk1 = M::kUnit * exponent(e1);
        static_for<0, 4>([&](auto step) {
          constexpr int st = step;
          const v8 f0 = M::dequant(k0[st], sk0), f1 = M::dequant(k1[st], sk1);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            sa[n] = M::mfma(f0, qf[n][st], sa[n]);
            sb[n] = M::mfma(f1, qf[n][st], sb[n]);
          }
        });
      }
      __builtin_amdgcn_sched_barrier(0);   // (fewer operands in flight: 168 registers)
      static_for<0, 4>([&](auto step) {
        constexpr int st = step;
        *reinterpret_cast<v8*>(vwrite + 16 * st) = M::dequant(v0[st], sv0);
        *reinterpret_cast<v8*>(vwrite + 16 * VROW + 16 * st) = M::dequant(v1[st], sv1);
      });
      // softmax of this lane's 8 keys (4 g .. 4 g + 3 and 16 on) for its row i of each tile
      v8 pf[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float v[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          v[r] = sa[n][r];
          v[4 + r] = sb[n][r];
        }
        if (masked) {
          asm volatile("");   // (a branch: as selects these are a part of every step)
          const int lim = page < 0 ? 0 : vis[n];
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (kbase + 4 * g + (r & 3) + 16 * (r >> 2) >= lim) v[r] = -INFINITY;
        }
        // (scale > 0: the largest logit is the largest product's)
        float top = scale * fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])),
                                  fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
        if (!__all(top <= mrun[n] + KV4_SLACK)) {
          top = fmaxf(top, __shfl_xor(top, 16, 64));
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          const float mnew = top > mrun[n] + KV4_SLACK ? top : mrun[n];
          const float alpha = __builtin_amdgcn_exp2f(mrun[n] - mnew);
          lrun[n] *= alpha;
#pragma unroll
          for (int d = 0; d < 8; ++d) o[n][d] *= alpha;
          mrun[n] = mnew;
        }
        const float ref = KV4_LIFT - mrun[n];
#pragma unroll
        for (int r = 0; r < 8; r += 2) {
          const v2 p = __builtin_convertvector(
              ((floatx2){__builtin_amdgcn_exp2f(__builtin_fmaf(v[r], scale, ref)),
                         __builtin_amdgcn_exp2f(__builtin_fmaf(v[r + 1], scale, ref))}), v2);
          lrun[n] = M::sum2(p, lrun[n]);
          pf[n][r] = p.x;
          pf[n][r + 1] = p.y;
        }
      }
      static_for<0, 8>([&](auto dt) {
        constexpr int d = dt;
        const v8 vf = read_vt<T>(vread + 32 * d, vread + 16 * VROW + 32 * d);
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][d] = M::mfma(vf, pf[n], o[n][d]);
      });
    }

    // join the four waves: a row's reference is its largest, the states are brought to it
    int ge = g;
    asm volatile("" : "+v"(ge));   // (addresses of the end are not kept in registers over the loop)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float l = lrun[n];
      l += __shfl_xor(l, 16, 64);
      l += __shfl_xor(l, 32, 64);
      if (g == 0) {
        mls[wv][0][16 * n + i] = mrun[n];
        mls[wv][1][16 * n + i] = l;
      }
    }
    __syncthreads();
    float* piece = a.ws + kv4_piece(worker_of(a, blockIdx.x), walk.per, run.r0) * kv4_piece_floats(ROWS);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int c = 16 * n + i;
      const float m0 = mls[0][0][c], m1 = mls[1][0][c], m2 = mls[2][0][c], m3 = mls[3][0][c];
      const float m = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
      const float l = mls[0][1][c] * __builtin_amdgcn_exp2f(m0 - m) +
                      mls[1][1][c] * __builtin_amdgcn_exp2f(m1 - m) +
                      mls[2][1][c] * __builtin_amdgcn_exp2f(m2 - m) +
                      mls[3][1][c] * __builtin_amdgcn_exp2f(m3 - m);
      const float f = __builtin_amdgcn_exp2f(mrun[n] - m) * (1.f / M::kUnit);
      float* mine = reinterpret_cast<float*>(vbuf);
#pragma unroll
      for (int d = 0; d < 8; ++d)
        *reinterpret_cast<floatx4*>(mine + (d * 64 + lane) * 4) = o[n][d] * f;
      __syncthreads();
      floatx4 sum[2];
#pragma unroll
      for (int dd = 0; dd < 2; ++dd) {
        const int at = ((2 * wv + dd) * 64 + lane) * 16;
        sum[dd] = *reinterpret_cast<const floatx4*>(lds + at) +
                  *reinterpret_cast<const floatx4*>(lds + VWAVE + at) +
                  *reinterpret_cast<const floatx4*>(lds + 2 * VWAVE + at) +
                  *reinterpret_cast<const floatx4*>(lds + 3 * VWAVE + at);
      }
      __syncthreads();
      const int r = run.tile * ROWS + c;
      if (!run.whole) {   // (a.ws holds two pieces a worker; rows past the unit's are not read)
#pragma unroll
        for (int dd = 0; dd < 2; ++dd)
          *reinterpret_cast<floatx4*>(piece + ((n * 8 + 2 * wv + dd) * 64 + lane) * 4) = sum[dd];
        if (wv == 0 && g == 0)
          *reinterpret_cast<floatx2*>(piece + ROWS * KV4_D + 2 * c) = (floatx2){m, l};
      } else if (r < n_row) {
        const int tok = r / ratio;
        const long long orow = (long long)(sq.q0 + tok) * a.n_heads + run.head * ratio + r - tok * ratio;
        const bool none = l == 0.f;   // a row that sees no key: zeros, and the sum of none
        T* op = reinterpret_cast<T*>(a.out) + orow * KV4_D + 4 * ge;
#pragma unroll
        for (int dd = 0; dd < 2; ++dd) {
          typedef T v4 __attribute__((ext_vector_type(4)));
          v4 x;
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = (T)(none ? 0.f : sum[dd][k] / l);
          *reinterpret_cast<v4*>(op + 16 * (2 * wv + dd)) = x;
        }
        if (a.lse && wv == 0 && g == 0)
          a.lse[orow] = none ? -INFINITY : (m - KV4_LIFT + __log2f(l)) * 0.69314718056f;
      }
    }
    __syncthreads();   // mls is written again
  }
}

// ---- more query rows
//
// Four waves of 32 rows each go over the same keys, two blocks a step (one block's chain of products
// leaves the matrix unit half idle, two interleaved fill it).  Blocks come as they lie in the pool
// into a ring in LDS, TDEPTH steps of them on their way while one computes.  K goes into the
// products as it is cached (see split_q); V is converted once for all, a part by each wave, into
// one of two LDS buffers; one barrier a step.  Accumulator r of lane (q, h) is key 8 (r / 4) + 4 h +
// r % 4 of the block.
//
// The logits are summed onto the negative reference, so that a weight is the power of what the
// products leave.  S^T of the next step is made between the weights of this one.
//
// Two workgroups a CU (LDS and 256 registers).  Two prompts of 4096 and 777 rows, 32 heads: 185 to
// 210 us by card with the merge's 15, 800 to 910 TF (a large product of 16-bit matrices reaches 1210).
// A step of both workgroups takes 1.8 us, 3400 cycles: for each SIMD 1790 of products and 1700 of
// vector instructions, for the CU 1900 of LDS.  No one of them is full: two waves a SIMD do not
// fill each other's gaps, and there are no registers for a third.  Eight blocks of 32 rows over
// 811 .. 7844 keys: 37 us and 11; of the 37 3 go to finding the first unit, 4.3 to its queries and
// first blocks, 20 to the steps, and both kernels move 36 MB of partials.  With K converted in
// registers as V is (64 conversions a step and wave), the prompts took 233 us, the blocks 54 in all.

constexpr int TROW = 320;                 // bytes of a V row in LDS: 16 banks apart, so that the 4
                                          // rows of a half wave's transposing read do not collide
constexpr int VTILE = 32 * TROW;
constexpr int TPAIR = 2 * KV4_BLOCK;
constexpr int TDEPTH = 3;                 // steps loaded ahead
constexpr int TRING = TDEPTH + 1;
constexpr int TILE_LDS = TRING * TPAIR + 4 * VTILE;
typedef __attribute__((address_space(3))) void* lds_ptr_t;

// 16 (4) bytes a lane from global memory, from + 16 lane (from + past + 4 lane), into LDS at to + 16
// lane (to + 4 lane); from, to and past uniform, at = 16 lane.  In assembly, because the compiler
// waits for all loads of the builtin before it lets any LDS read go by; these have no result
// registers, and the waits are wait_loads'.
DFL_DEV void load_to_lds16(const unsigned char* from, int at, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :: "v"(at), "s"(from), "s"(to) : "memory", "m0");
}
DFL_DEV void load_to_lds4(const unsigned char* from, int past, int at, uint32_t to) {
  uint32_t at4;
  asm volatile("s_mov_b32 m0, %3\n\tv_lshrrev_b32 %0, 2, %1\n\tv_add_u32 %0, %4, %0\n\t"
               "global_load_lds_dword %0, %2"
               : "=&v"(at4) : "v"(at), "s"(from), "s"(to), "s"(past) : "memory", "m0");
}

// Waits until at most N of this wave's loads are outstanding.
template <int N>
DFL_DEV void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(N | (7 << 4) | (15 << 8));
  asm volatile("" ::: "memory");
}
// Barrier that leaves loads on their way; LDS writes of this wave are done before it.
DFL_DEV void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4) | (0 << 8));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Q in 6 bits, thrice.  The matrix instructions that take 4-bit operands as they lie, with a power
// of two for each 32 of them, want the other operand in 8 bits or fewer, and are with 6 bits as
// fast as without: 64 values in the time that 16-bit ones need for 16.  So a group x of 32 values
// of Q (times the softmax's scale) is split into x = (p0 + p1 / 16 + p2 / 512) 2^b, each part the
// nearest of the numbers with 4 bits of which 7.5 is the largest: with a <= 7.5 for the largest
// |x| = a 2^b, what p0 leaves is at most 1/4, 4 units of p1, which leaves at most 1/8, 4 units of
// p2, which leaves at most 1/8 of its own, 2^-12 2^b.  As a > 3.75, every value is held to 2^-13.9
// of its group's largest: finer than half a step of fp16 (2^-11 of a value) down to 1/7 of that
// largest, of bf16 (2^-8) down to 1/59, and coarser for the small values beside a large one.  Under
// fp16 queries with a channel of each group 20 to 1000 times the rest (4000 keys, logits of some 5)
// results are off by 2.9e-4 of their norm, by 2.0e-4 if Q is held as it is, which is what rounding
// them to fp16 takes alone; under normal queries by 2.9e-4 and 2.7e-4.  A fourth part would bring the
// 2.9e-4 to 2.1e-4 (2^-18.9), and take eight blocks from 45.6 to 48.4 us, fp16 prompts from 190 to
// 207: it needs the reference's registers, so that the logits begin at zero.
typedef int int8v_t __attribute__((ext_vector_type(8)));
typedef unsigned uint6v_t __attribute__((ext_vector_type(6)));
typedef float float32v_t __attribute__((ext_vector_type(32)));
struct Q6 { uint6v_t part[3]; uint32_t exps; };   // exps: an exponent byte for each part
// Values 2 i in lo, 2 i + 1 in hi, divided by 2^(b - 127).  (In assembly: the builtin's result may be
// put into registers of its operands, which the instruction still reads when it has written them.)
DFL_DEV uint6v_t to_fp6(floatx16 lo, floatx16 hi, uint32_t b) {
  uint6v_t r;
  asm("v_cvt_scalef32_2xpk16_fp6_f32 %0, %1, %2, %3" : "=&v"(r) : "v"(lo), "v"(hi), "v"(b << 23));
  return r;
}
DFL_DEV float32v_t from_fp6(uint6v_t x, uint32_t b) {
  float32v_t r;
  asm("v_cvt_scalef32_pk32_f32_fp6 %0, %1, %2" : "=&v"(r) : "v"(x), "v"(b << 23));
  return r;
}
template <typename V8>
DFL_DEV Q6 split_q(const V8 (&x)[4], float scale) {
  floatx16 lo, hi;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    lo[i] = scale * (float)x[i >> 2][2 * (i & 3)];
    hi[i] = scale * (float)x[i >> 2][2 * (i & 3) + 1];
    top = max(max(top, __float_as_uint(lo[i]) & 0x7fffffffu), __float_as_uint(hi[i]) & 0x7fffffffu);
  }
  // (10: p2's exponent must not go below that of the byte 0.  Groups below 2^-115 keep fewer bits.)
  const uint32_t b = max(10, (int)(top >> 23) - 2 + ((top & 0x7fffff) > 0x700000 ? 1 : 0));
  Q6 q;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const uint32_t bk = k == 0 ? b : k == 1 ? b - 4 : b - 9;
    q.part[k] = to_fp6(lo, hi, bk);
    if (k < 2) {
      const float32v_t held = from_fp6(q.part[k], bk);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        lo[i] -= held[2 * i];
        hi[i] -= held[2 * i + 1];
      }
    }
  }
  // an infinity or a NaN, or what the scale makes one, is a NaN in all products of the row
  q.exps = top >= 0x7f800000u ? 0xffffffu : b | (b - 4) << 8 | (b - 9) << 16;
  return q;
}
// c + K Q^T of 64 values a row: 32 keys of K as they are cached, a lane's key and half of the
// values, and the exponent in ke's lowest byte.
template <int PART>
DFL_DEV floatx16 mfma_part(u32x4 k, uint32_t ke, const Q6& q, floatx16 c) {
  const int8v_t x = {(int)k.x, (int)k.y, (int)k.z, (int)k.w};
  const uint6v_t p = q.part[PART];
  const int8v_t y = {(int)p[0], (int)p[1], (int)p[2], (int)p[3], (int)p[4], (int)p[5]};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 2, 0, (int)ke, PART, (int)q.exps);
}

// What all lanes hold alike, into scalar registers.
template <typename S>
DFL_DEV S scalars(const S& v) {
  constexpr int N = sizeof(S) / 4;
  static_assert(sizeof(S) % 4 == 0, "words");
  struct Words { int w[N]; };
  Words x = __builtin_bit_cast(Words, v);
#pragma unroll
  for (int i = 0; i < N; ++i) x.w[i] = __builtin_amdgcn_readfirstlane(x.w[i]);
  return __builtin_bit_cast(S, x);
}
// The kernel's arguments, read again: what a run's begin and end need of them is not kept in scalar
// registers over its steps, which have few.
DFL_DEV const Kv4AttnArgs& args_again() {
  auto p = reinterpret_cast<const __attribute__((address_space(4))) Kv4AttnArgs*>(
      (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(p));
  return *(const Kv4AttnArgs*)p;
}

template <typename T>
__global__ __launch_bounds__(256, 2) void kv4_tile_kernel(Kv4AttnArgs args) {
  typedef Mat<T> M;
  typedef typename M::v8 v8;
  typedef typename M::v2 v2;
  constexpr int ROWS = 128;
  extern __shared__ __attribute__((aligned(1024))) unsigned char tile_lds[];   // TILE_LDS bytes
  unsigned char* const ring = tile_lds;                      // [TRING][TPAIR]
  unsigned char* const vbuf = tile_lds + TRING * TPAIR;      // [2][2][VTILE]
  const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // K: row i of a block, groups h and 2 + h.  V: of block vu of the step row i, group 2 vj + h.
  const int koff = 16 * lane;
  const int soff = KV4_SC + 4 * ((i & 15) + 16 * h) + (i >> 4);   // K's exponent (V's is 2 further)
  const int vu = wv >> 1, vj = wv & 1;
  const int vwrite = i * TROW + 64 * h;
  const int vread = (4 * h + ((lane & 15) >> 2)) * TROW + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);

  // (as with the arguments: a wave's place in its walk is kept in LDS over a run's steps)
  struct Kept { Walk walk; Run run; };
  __shared__ Kept kept_of[4];
  Kept& kept = kept_of[wv];
  bool more;
  {
    Walk walk;
    Run run;
    more = walk_begin(args, ROWS, walk, run);
    kept = Kept{walk, run};
  }
  walk_no_note(args, ROWS, wv);
  while (more) {
    Walk walk = scalars(kept.walk);
    Run run = scalars(kept.run);
    const Kv4AttnArgs& a = args_again();
    const int ratio = a.n_heads / a.n_kv;
    if (!walk_run(walk, run)) break;   // (the worker's last places)
    if (run.b0 == 0 && !run.whole) walk_note(a, ROWS, wv, walk.per, run);
    kept.run = run;
    const Kv4Seq& sq = run.sq;
    const int n_row = sq.qlen * ratio;
    const int row0 = run.tile * ROWS + 32 * wv;     // this wave's first row (may be past the last)
    int le = lane_again();   // (addresses of a run's begin and end are not kept over others)
    const int row = min(row0 + (le & 31), n_row - 1), tok = row / ratio;
    v8 qin[2][4];   // groups h and 2 + h of the row
    const T* qp = reinterpret_cast<const T*>(a.q) + (long long)(sq.q0 + tok) * a.q_row +
                  (long long)(run.head * ratio + row - tok * ratio) * a.q_head + 32 * (le >> 5);
#pragma unroll
    for (int st = 0; st < 8; ++st) qin[st >> 2][st & 3] = *reinterpret_cast<const v8*>(qp + 8 * (st & 3) + 64 * (st >> 2));
    // keys that the lane's row sees (made again where it is needed: rarely)
    auto visible = [&]() __attribute__((always_inline)) {
      const int l = lane_again();
      const Kv4AttnArgs& e = args_again();
      const Run r = scalars(kept.run);
      const Kv4Seq& q = r.sq;
      const int ratio = e.n_heads / e.n_kv;
      return attn_visible(e, q, min(r.tile * ROWS + 32 * wv + (l & 31), q.qlen * ratio - 1) / ratio);
    };
    // fewest and most keys that rows of the tile see
    const int tmin = attn_visible(a, sq, run.tile * ROWS / ratio);
    const int tmax = attn_visible(a, sq, (min(run.tile * ROWS + ROWS, n_row) - 1) / ratio);
    const int b_end = min(run.b1, (tmax + KV4_KEYS - 1) / KV4_KEYS);

    floatx16 o[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) o[d] = (floatx16){};
    float lrun = -INFINITY;   // (the row has no weight yet)
    // What the logits are summed onto: KV4_LIFT less the reference (in all 16: the instruction's
    // operand), 0 while the row has no weight.
    floatx16 ref = {};

    // Addresses of blocks, 64 at a time, a lane each (past the last block the last one again, so
    // that the count of loads under way is always the same).
    const int subs = a.page_shift - 5;
    const int* trow = a.table + (long long)run.s * a.width;
    const uint32_t per_page = (uint32_t)a.n_kv << subs, of_head = (uint32_t)run.head << subs;
    int abase = 0;                       // the first of the 64
    uint32_t mine = 0;                   // (their numbers: a register less)
    // Blocks before this one are in pages of the pool, in the run, and seen whole by all rows of the
    // tile; steps past it look closer.
    int full = min(b_end, tmin / KV4_KEYS);
    auto no_page = [&](int page) { return page < 0 || page >= a.n_pages; };
    auto absent = [&](int b) { return b >= b_end || no_page(load_const(trow + (b >> subs))); };
    auto addresses = [&](int b) {
      const int k = max(0, min(b + lane_again(), b_end - 1));   // (b_end may be 0: then nothing is loaded)
      const int page = b_end > 0 ? trow[k >> subs] : 0;
      const bool no = no_page(page);
      mine = (no ? 0u : (uint32_t)page * per_page) + of_head + (uint32_t)(k & ((1 << subs) - 1));
      abase = b;
      if (__ballot(no)) {
        full = 0;
        int bit = KV4_ERR_PAGE;
        asm volatile("" : "+v"(bit));   // (no register for it over the steps)
        if (no) atomicOr(a.err, bit);
      }
    };
    // A wave's loads of the step that begins with block b, into a place of the ring: KiB wv of both
    // blocks, and the exponents of block wv % 2 (two waves load the same, so that all count alike).
    constexpr int LOADS = 3;
    const unsigned char* const pool_w = a.pool + 1024 * wv;
    const uint32_t ring_w = (uint32_t)(uintptr_t)(lds_ptr_t)ring + 1024 * wv;
    auto issue = [&](int b, int place) __attribute__((always_inline)) {
      if (__builtin_expect(b - abase >= 64, 0)) addresses(b);
      const int k = b - abase;           // (even: the pair is within the 64)
      const unsigned char* const p0 = pool_w + kv4_block_at((uint32_t)__builtin_amdgcn_readlane(mine, k));
      const unsigned char* const p1 = pool_w + kv4_block_at((uint32_t)__builtin_amdgcn_readlane(mine, k + 1));
      const uint32_t to = ring_w + place;
      load_to_lds16(p0, koff, to);
      load_to_lds16(p1, koff, to + KV4_BLOCK);
      const uintptr_t p = wv & 1 ? (uintptr_t)p1 : (uintptr_t)p0;
      load_to_lds4(reinterpret_cast<const unsigned char*>(p), KV4_SC - 1024 * wv, koff,
                   to + (wv & 1) * KV4_BLOCK + KV4_SC - 1024 * wv);
    };
    // V of the step that begins with block b, from a place of the ring: codes and exponent, then
    // into buffers `to`.  In a block that some row of the tile does not see whole: zeros for rows
    // past the sequence and for NaN groups, as there 0 * NaN would reach rows that do not see them;
    // the rows that do see a NaN are set when the block is used.
    u32x4 vc;
    uint32_t ve;
    auto read_v = [&](int place) __attribute__((always_inline)) {
      const unsigned char* vb = ring + place + vu * KV4_BLOCK;
      ve = vb[128 * vj + soff + 2];
      vc = *reinterpret_cast<const u32x4*>(vb + 2048 + 1024 * vj + koff);
    };
    auto mask_v = [&](int b) __attribute__((always_inline)) {
      if (__builtin_expect(b + 2 > full, 0)) {
        const bool gone = absent(b + vu);
        if (ve >= M::kVNan || gone || (b + vu) * KV4_KEYS + (lane_again() & 31) >= sq.len) {
          ve = 0;
          vc = (u32x4){0, 0, 0, 0};
        }
      }
    };
    auto convert_v = [&](int b, int to) __attribute__((always_inline)) {
      mask_v(b);
      unsigned char* at = vbuf + (2 * to + vu) * VTILE + 128 * vj + vwrite;
      const float unit = v_unit<M>(ve);
      static_for<0, 4>([&](auto word) {
        constexpr int w = word;
        *reinterpret_cast<v8*>(at + 16 * w) = M::dequant(vc[w], unit);
      });
    };
    // S^T of the two blocks in a place of the ring: codes and exponents, then the products.
    Q6 qf[2];
    u32x4 kc[4];
    uint32_t ke[4];
    auto read_k = [&](int place) __attribute__((always_inline)) {
      const unsigned char* kb = ring + place;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          ke[2 * u + j] = kb[u * KV4_BLOCK + soff + 128 * j];
          kc[2 * u + j] = *reinterpret_cast<const u32x4*>(kb + u * KV4_BLOCK + koff + 1024 * j);
        }
    };
    // Product n of 12 for the S^T t of both blocks, begun on ref: half the values, one part of Q.
    auto product = [&](auto n, floatx16 (&t)[2]) __attribute__((always_inline)) {
      constexpr int st = decltype(n)::value / 6, part = 2 - decltype(n)::value % 6 / 2, u = decltype(n)::value & 1;
      t[u] = mfma_part<part>(kc[2 * u + st], ke[2 * u + st], qf[st],
                             decltype(n)::value < 2 ? ref : t[u]);
    };
    const bool idle = row0 >= n_row;   // a wave past the sequence's rows only loads and converts
    floatx16 s[2] = {};
    addresses(run.b0);
    if (run.b0 < b_end) {
#pragma unroll
      for (int j = 0; j < TDEPTH; ++j) issue(run.b0 + 2 * j, j * TPAIR);
    }
    qf[0] = split_q(qin[0], a.scale_log2);
    qf[1] = split_q(qin[1], a.scale_log2);
    // The queries are there: from here on the ring's loads alone are counted.  (The compiler's waits
    // do not know of them; one statement, so that it has none in the loop.)
    asm volatile(""
                 : "+v"(qf[0].part[0]), "+v"(qf[0].part[1]), "+v"(qf[0].part[2]), "+v"(qf[0].exps),
                   "+v"(qf[1].part[0]), "+v"(qf[1].part[1]), "+v"(qf[1].part[2]), "+v"(qf[1].exps) :: "memory");
    if (run.b0 < b_end) {
      wait_loads<LOADS * (TDEPTH - 1)>();
      lds_barrier();
      read_v(0);
      read_k(0);
      convert_v(run.b0, 0);
      static_for<0, 12>([&](auto n) { product(n, s); });
    }
    // Step `odd` of a pair (s: S^T of its two blocks): their weights, between which (they do not wait
    // for each other) go the products of the next step's S^T t, then the products with V.  A pair of
    // steps has half of the ring (h0, the other is h1; bytes), a step one of V's buffers.
    int h0 = 0, h1 = 2 * TPAIR;
    auto do_step = [&](auto which, int b, floatx16 (&s)[2], floatx16 (&t)[2]) __attribute__((always_inline)) {
      constexpr int odd = which, to = odd;
      const int kbase = b * KV4_KEYS, next = odd ? h1 : h0 + TPAIR;
      __builtin_amdgcn_s_setprio(0);
      wait_loads<LOADS * (TDEPTH - 2)>();
      // the next step's blocks and V of this one's are there, and nobody reads those of the last
      // step any more
      lds_barrier();
      read_v(next);   // (after the last step those are blocks read once too often)
      read_k(next);
      issue(b + 2 * TDEPTH, odd ? h0 : h1 + TPAIR);
      convert_v(b + 2, to ^ 1);   // (while K is on its way from LDS)
      if (__builtin_expect(!idle, 1)) {
        if (__builtin_expect(b + 2 > full, 0)) {
          const bool gone0 = absent(b), gone1 = absent(b + 1);
          const int vis = visible();   // (volatile: a branch; as selects the masks are a third of the loop)
          // groups h, 2 + h of row i of either block that stand for NaN
          const unsigned char* kb = ring + h0 + odd * TPAIR + soff;
          const int l = lane_again(), i = l & 31, h = l >> 5;
          const bool there0 = !gone0 && kbase + i < sq.len;
          const bool there1 = !gone1 && kbase + KV4_KEYS + i < sq.len;
          auto nan_at = [&](int at) { return kb[at + 2] >= M::kVNan; };
          const bool n0 = there0 && nan_at(0), n1 = there0 && nan_at(128);
          const bool n2 = there1 && nan_at(KV4_BLOCK), n3 = there1 && nan_at(KV4_BLOCK + 128);
          if (__ballot(n0 || n1 || n2 || n3)) {
            const float nan = __builtin_nanf("");
#pragma unroll 1
            for (int r = 0; r < 2 * KV4_KEYS; ++r) {
              const unsigned long long lo = __ballot(r < 32 ? n0 : n2) >> (r & 31);
              const unsigned long long hi = __ballot(r < 32 ? n1 : n3) >> (r & 31);
              if (kbase + r < vis)
                static_for<0, 4>([&](auto group) {
                  constexpr int gr = group;
                  if (((gr & 2 ? hi : lo) >> (32 * (gr & 1))) & 1)
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[gr][k] = nan;
                });
            }
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int lim = (u ? gone1 : gone0) ? 0 : vis;
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (kbase + 32 * u + 4 * h + (r & 3) + 8 * (r >> 2) >= lim) s[u][r] = -INFINITY;
          }
        }
        v8 p[4], vf[2][4];
        float sum = 0.f;
        auto weights = [&](int n) __attribute__((always_inline)) {   // two of 32
          const int u = n >> 3, r = 2 * (n & 7);
          const v2 x = __builtin_convertvector(
              ((floatx2){__builtin_amdgcn_exp2f(s[u][r]), __builtin_amdgcn_exp2f(s[u][r + 1])}), v2);
          sum = M::sum2(x, sum);
          p[n >> 2][r & 7] = x.x;
          p[n >> 2][(r & 7) + 1] = x.y;
        };
        const unsigned char* vb = vbuf + 2 * to * VTILE + vread;
        auto read_vf = [&](int q) __attribute__((always_inline)) {   // operands of V for 16 keys
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const unsigned char* at = vb + (q >> 1) * VTILE + 16 * (q & 1) * TROW + 64 * d;
            vf[q & 1][d] = read_vt<T>(at, at + 8 * TROW);
          }
        };
        // (the order is held by the barriers: left to itself the compiler puts all products first and
        // each read right before its use; eight blocks then take 52 us for 51)
        constexpr int AHEAD = 4;   // weights made while K is on its way
        static_for<0, AHEAD>([&](auto w) { weights(w); });
        __builtin_amdgcn_sched_barrier(0);
        static_for<0, 12>([&](auto n) {
          constexpr int k = n;
          product(n, t);
          static_for<AHEAD + (16 - AHEAD) * k / 12, AHEAD + (16 - AHEAD) * (k + 1) / 12>([&](auto w) { weights(w); });
          __builtin_amdgcn_sched_barrier(0);
        });
        read_vf(0);
        // Weights above 2^15 (the sum of 32 says so; an infinity and a NaN do too), or none so far:
        // the row's reference is raised to the largest logit (more than KV4_SLACK above it), or set,
        // and they are made again.  So no maximum is taken in the steps in which none is needed, and
        // a row's references do not depend on the other rows.
        if (__builtin_expect(!__all((sum <= 1048576.f) & (lrun + sum >= 0.f)), 0)) {
          float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
          for (int r = 1; r < 16; ++r) top = fmaxf(fmaxf(top, s[0][r]), s[1][r]);
          top = fmaxf(top, __int_as_float(__builtin_amdgcn_ds_bpermute(4 * (lane_again() ^ 32), __float_as_int(top))));
          top -= KV4_LIFT;
          const bool none = lrun == -INFINITY;   // (both lanes of the row)
          const unsigned long long past = __ballot(!(sum <= 1048576.f));
          const bool over = (past | past >> 32 | past << 32) >> lane_again() & 1;
          const float up = (over && top > KV4_SLACK) || (none && top > -INFINITY) ? top : 0.f;
          const float alpha = none ? 1.f : __builtin_amdgcn_exp2f(-up);
          lrun = none && top > -INFINITY ? 0.f : lrun * alpha;
#pragma unroll
          for (int d = 0; d < 4; ++d) o[d] *= alpha;
          ref -= up;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            s[u] -= up;
            t[u] -= up;
          }
          sum = 0.f;
#pragma unroll
          for (int n = 0; n < 16; ++n) weights(n);
        }
        lrun += sum;
        __builtin_amdgcn_s_setprio(1);   // (before the other workgroup's conversions: eight blocks 49.7 -> 48.9 us)
        static_for<0, 4>([&](auto quarter) {
          constexpr int q = quarter;
          if constexpr (q < 3) read_vf(q + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int d = 0; d < 4; ++d) o[d] = M::mfma(vf[q & 1][d], p[q], o[d]);
          __builtin_amdgcn_sched_barrier(0);
        });
      }
    };
    floatx16 t[2];
    for (int b = run.b0; b < b_end; b += 4) {
      do_step(std::integral_constant<int, 0>{}, b, s, t);
      if (__builtin_expect(b + 2 < b_end, 1)) do_step(std::integral_constant<int, 1>{}, b + 2, t, s);
      const int h = h0;
      h0 = h1;
      h1 = h;
    }
    __builtin_amdgcn_s_waitcnt(0);   // (the loads past the last block)

    {
      const Kv4AttnArgs& e = args_again();
      walk = scalars(kept.walk);
      run = scalars(kept.run);
      const Kv4Seq& sq = run.sq;
      const int ratio = e.n_heads / e.n_kv, n_row = sq.qlen * ratio, row0 = run.tile * ROWS + 32 * wv;
      lrun += __shfl_xor(lrun, 32, 64);
      const float mrun = lrun == -INFINITY ? -FLT_MAX : KV4_LIFT - ref[0];
      if (lrun == -INFINITY) lrun = 0.f;
      le = lane_again();
      if (!run.whole) {
        float* piece = e.ws + kv4_piece(worker_of(e, blockIdx.x), walk.per, run.r0) * kv4_piece_floats(ROWS);
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<floatx4*>(piece + (((wv * 4 + d) * 4 + k) * 64 + le) * 4) =
                (floatx4){o[d][4 * k], o[d][4 * k + 1], o[d][4 * k + 2], o[d][4 * k + 3]} * (1.f / M::kUnit);
        if (le < 32)
          *reinterpret_cast<floatx2*>(piece + ROWS * KV4_D + 2 * (32 * wv + le)) = (floatx2){mrun, lrun};
      } else if (row0 + (le & 31) < n_row) {
        const int row = row0 + (le & 31), tok = row / ratio;
        const long long orow = (long long)(sq.q0 + tok) * e.n_heads + (run.head - tok) * ratio + row;
        const bool none = lrun == 0.f;   // a row that sees no key: zeros, and the sum of none
        const float f = (1.f / M::kUnit) / lrun;
        T* op = reinterpret_cast<T*>(e.out) + orow * KV4_D + 4 * (le >> 5);
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            typedef T v4 __attribute__((ext_vector_type(4)));
            v4 x;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = (T)(none ? 0.f : o[d][4 * k + j] * f);
            *reinterpret_cast<v4*>(op + 32 * d + 8 * k) = x;
          }
        if (e.lse && le < 32)
          e.lse[orow] = none ? -INFINITY : (mrun - KV4_LIFT + __log2f(lrun)) * 0.69314718056f;
      }
      more = walk_next(e, ROWS, walk, run);
      kept = Kept{walk, run};
    }
    __syncthreads();   // the buffers are written again
  }
}

// Units that several workers share: their partial states joined in the order of the keys, by the
// note of the worker that began with the unit.  A thread has 4 values of a row.  TILE: the partials
// are kv4_tile_kernel's.  Bound by them: eight blocks leave 550 of 66 KB, 10.6 us with the launch.
// Two partials (most of a prompt's) or eight are loaded at once: one by one two prompts' took 30 us
// for 16.  Which they are is in notes: every workgroup finding its unit by itself took 40 us more.
template <typename T, bool TILE>
__global__ __launch_bounds__(256) void kv4_merge_kernel(Kv4AttnArgs a, int tile_rows) {
  const int lane = threadIdx.x & 63;
  const int ratio = a.n_heads / a.n_kv;
  const int groups = tile_rows / 8;                 // workgroups of a unit
  // (the worker, whose partials its own die's L2 may still hold)
  const int w0 = (blockIdx.x & 7) * (a.workers >> 3) + (blockIdx.x >> 3) / groups;
  const int f = (int)((blockIdx.x >> 3) % groups) * 256 + threadIdx.x;   // which 4 values of the tile
  const int c = TILE ? 32 * (f >> 10) + (lane & 31) : 16 * (f >> 9) + (lane & 15);
  const int col = TILE ? 32 * ((f >> 8) & 3) + 8 * ((f >> 6) & 3) + 4 * (lane >> 5)
                       : 16 * ((f >> 6) & 7) + 4 * (lane >> 4);
  const Kv4Note& n = kv4_notes(a, tile_rows)[w0];
  const int w1 = n.w1, head = n.head, r = n.tile * tile_rows + c;
  if (w1 < 0 || r >= n.qlen * ratio) return;
  const long long pf = kv4_piece_floats(tile_rows);
  float m = -FLT_MAX, l = 0.f;
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  // N pieces from w on, all loads under way together
  auto join = [&](int w, auto count) __attribute__((always_inline)) {
    constexpr int N = count;
    floatx4 x[N];
    floatx2 y[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int k = min(w + j, w1);   // (that of the first lies behind its other one)
      const float* p = a.ws + (2ll * k + (k == w0 ? 1 : 0)) * pf;
      x[j] = *reinterpret_cast<const floatx4*>(p + 4 * f);
      y[j] = *reinterpret_cast<const floatx2*>(p + tile_rows * KV4_D + 2 * c);
    }
    float mn = m;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (w + j > w1) {   // (0 * what lies there may be NaN)
        x[j] = (floatx4){0.f, 0.f, 0.f, 0.f};
        y[j] = (floatx2){-INFINITY, 0.f};
      }
      mn = fmaxf(mn, y[j].x);
    }
    const float k = __builtin_amdgcn_exp2f(m - mn);
    o *= k;
    l *= k;
    m = mn;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float e = __builtin_amdgcn_exp2f(y[j].x - m);
      l += e * y[j].y;
      o += e * x[j];
    }
  };
  if (w1 == w0 + 1) {
    join(w0, std::integral_constant<int, 2>{});
  } else {
    for (int w = w0; w <= w1; w += 8) join(w, std::integral_constant<int, 8>{});
  }
  const int tok = r / ratio;
  const long long orow = (long long)(n.q0 + tok) * a.n_heads + head * ratio + r - tok * ratio;
  const bool none = l == 0.f;
  typedef T v4 __attribute__((ext_vector_type(4)));
  v4 x;
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = (T)(none ? 0.f : o[j] / l);
  *reinterpret_cast<v4*>(reinterpret_cast<T*>(a.out) + orow * KV4_D + col) = x;
  if (a.lse && col == 0)
    a.lse[orow] = none ? -INFINITY : (m - KV4_LIFT + __log2f(l)) * 0.69314718056f;
}

template <typename T>
void attend(const Kv4AttnArgs& a, const Kv4Cut& c, hipStream_t st) {
  const dim3 grid(a.workers), block(256), mgrid(a.workers * (c.tile_rows / 8));
  switch (c.tile_rows) {
    case 16: hipLaunchKernelGGL((kv4_attn_kernel<T, 1>), grid, block, 0, st, a); break;
    case 32: hipLaunchKernelGGL((kv4_attn_kernel<T, 2>), grid, block, 0, st, a); break;
    default: hipLaunchKernelGGL((kv4_tile_kernel<T>), grid, block, TILE_LDS, st, a);
  }
  if (c.tile_rows <= 32) hipLaunchKernelGGL((kv4_merge_kernel<T, false>), mgrid, block, 0, st, a, c.tile_rows);
  else hipLaunchKernelGGL((kv4_merge_kernel<T, true>), mgrid, block, 0, st, a, c.tile_rows);
}

}  // namespace

void launch_kv4_step(const Kv4StepArgs& a, hipStream_t st) {
  if (a.n_seq <= STEP_ONE_SEQS && a.max_rows <= STEP_ONE_ROWS) {
    const int threads = a.n_seq <= 256 && a.max_rows <= 1024 ? 256 : 1024;
    hipLaunchKernelGGL(kv4_step_one_kernel, dim3(1), dim3(threads), 0, st, a);
    return;
  }
  // (what a step moves is known on the device alone: at most the pool's pages)
  const dim3 pages(min(1024, (max(a.n_pages, a.n_seq) + 255) / 256)), block(256);
  hipLaunchKernelGGL(kv4_step_scan_kernel, dim3(1), dim3(1024), 0, st, a);
  hipLaunchKernelGGL(kv4_step_check_kernel, pages, block, 0, st, a);
  hipLaunchKernelGGL(kv4_step_move_kernel, pages, block, 0, st, a);
  if (a.max_rows > 0)
    hipLaunchKernelGGL(kv4_step_rows_kernel, dim3(min(65536, a.max_rows / STEP_ROWS + 1)), block, 0, st, a);
}

static dim3 rows_grid(const Kv4RowsArgs& a) {
  const long long chunks = ((long long)a.rows + ROWS_WG - 1) / ROWS_WG;
  return dim3(2 * a.n_kv, (unsigned)(chunks < 65535 ? chunks : 65535));
}
void launch_kv4_append(const Kv4RowsArgs& a, hipStream_t st) {
  const dim3 grid = rows_grid(a), block(256);
  if (a.dtype == 0) hipLaunchKernelGGL((kv4_append_kernel<0>), grid, block, 0, st, a);
  else if (a.dtype == 1) hipLaunchKernelGGL((kv4_append_kernel<1>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((kv4_append_kernel<2>), grid, block, 0, st, a);
}
void launch_kv4_read(const Kv4RowsArgs& a, hipStream_t st) {
  const dim3 grid = rows_grid(a), block(256);
  if (a.dtype == 0) hipLaunchKernelGGL((kv4_read_kernel<0>), grid, block, 0, st, a);
  else if (a.dtype == 1) hipLaunchKernelGGL((kv4_read_kernel<1>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((kv4_read_kernel<2>), grid, block, 0, st, a);
}
void launch_kv4_attend(const Kv4AttnArgs& a_in, hipStream_t st) {
  Kv4AttnArgs a = a_in;
  const Kv4Cut c = kv4_cut(a.n_rows, a.n_heads, a.n_kv, a.n_seq);
  a.workers = c.workers;
  if (a.dtype == 1) attend<half_t>(a, c, st);
  else attend<bf16_t>(a, c, st);
}

}  // namespace dfl
