// Step of a paged 4-bit cache whose sequences share pages (dfl_kv4.h): sequences go on from others'
// rows, pages are counted, a shared page is copied for the sequence that writes into it.
//
// Sequence s keeps the first keep[s] rows of sequence parent[s] as it was before the step, in the same
// pages, and grows by grow[s].  refs[p] is the number of table places that hold page p; pages with none
// are free, and are taken lowest number first, sequence by sequence (a sequence's copied page, then
// the pages of its new rows).  New rows that begin inside a page go into it: of the sequences that hold
// it after the step, if all write into it, the first does, and the others (or, if some do not write,
// all that do) get a page of their own with the kept rows' blocks copied.
//
// Phases, each over all sequences: scan (what each asks, the pages that are written into); count (a
// holder more or less for every place that changes, pages kept from others noted, as their tables change
// too; the writers); ask (who copies; free pages); list (free pages by rank); place (tables, counts,
// slots); then the copies, in a launch of their own.  Nothing but the counts changes before it is known
// that the step can be done, and they are set back if it cannot.
//
// Bound by latencies, as the plain step: for few sequences, rows, pages and places (FORK_ONE_..) one
// workgroup does all phases with the offsets in LDS, past that each is a launch.  Places of all
// sequences are numbered through and found by a search in the offsets.  One workgroup and launches, us of a
// step in a graph (sequences x kept pages that all but the group's first keep from it): 8 x 64 7, 23; 64 x 43
// 15, 27; 64 x 121 21, 28; 256 x 15 20, 30; 256 x 62 37, 31; 1024 x 93 195, 42.  Sequences that begin so, with
// no pages before, take as long as those that hold the same pages already; with pages of other texts, which
// all change hands, 256 x 62 take 45, 31 and 1024 x 31 114, 41.  (With an atomic for each kept page, whether
// it changes hands or not, the 1024 x 93 that hold theirs already took 335 and 59.)  The host knows the
// places that the tables have, not those that a step looks at: the 64 x 43 in tables of 512 pages each take
// the launches, 26 where one workgroup would take 15 (17 and 10 if none forks).
#include "dfl_kv4.h"

#include "dfl_common.h"
#include "dfl_kv4_scan.h"

namespace dfl {

namespace {

DFL_DEV int load_agent(const int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
DFL_DEV void store_agent(int* p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Numbers of each sequence: kept rows, parent, pages before the step, the page that its rows go on in
// (-1: none), places counted and places written before it, pages taken before it, copies before it
// (own[s]: whether it has one), new rows before it (n_seq + 1).
struct ForkView { int *base, *par, *old, *edge, *count_at, *place_at, *take_at, *copy_at, *own, *starts; };
constexpr int FORK_ARRAYS = 9;   // (starts come on top)
// Totals and errors, in LDS or at the scratch's start.
struct ForkTotals { int err, counted, placed, rows, bad, need, copies, pad; };

struct ForkScratch {   // in memory
  ForkTotals* totals;
  int *copy_src, *copy_dst, *copy_blocks, *writers, *first, *list, *chunks, *kept;
  ForkView view;
};
DFL_DEV ForkScratch fork_scratch(const Kv4ForkArgs& a) {
  int* p = a.scratch;
  auto take = [&](long long n) { int* q = p; p += n; return q; };
  ForkScratch x;
  x.totals = reinterpret_cast<ForkTotals*>(take(KV4_FORK_TOTALS));
  x.copy_src = take(a.n_seq);
  x.copy_dst = take(a.n_seq);
  x.copy_blocks = take(a.n_seq);
  ForkView& v = x.view;
  for (int** q : {&v.base, &v.par, &v.old, &v.edge, &v.count_at, &v.place_at, &v.take_at, &v.copy_at, &v.own})
    *q = take(a.n_seq);
  v.starts = a.starts;
  x.writers = take(a.n_pages);
  x.first = take(a.n_pages);
  x.list = take(a.n_pages);
  x.chunks = take(kv4_fork_chunks(a.n_pages));
  x.kept = take(0);   // [n_seq][width], only with parents
  return x;
}

DFL_DEV bool fork_page_ok(const Kv4ForkArgs& a, int page) { return page >= 0 && page < a.n_pages; }
DFL_DEV bool fork_ask(const Kv4ForkArgs& a, int s, Kv4ForkAsk& q) {
  const int par = a.parent ? a.parent[s] : s;
  const bool ok = par >= 0 && par < a.n_seq;
  const int from = a.lens[ok ? par : s], len = a.lens[s];
  return kv4_fork_ask(s, ok ? par : -1, from, len, a.keep ? a.keep[s] : from, a.grow ? a.grow[s] : 0, a.width,
                      a.page_shift, q);
}
DFL_DEV void fork_note(const Kv4ForkAsk& q, const Sum3& in, int s, const ForkView& v) {
  v.base[s] = q.keep;
  v.par[s] = q.parent;
  v.old[s] = q.old;
  v.count_at[s] = (int)(in.a - q.counted);
  v.place_at[s] = (int)(in.b - q.placed);
  v.starts[s] = (int)(in.c - q.grow);
}
DFL_DEV int fork_grow(const ForkView& v, int s) { return v.starts[s + 1] - v.starts[s]; }

// Place i of those that are looked at: the page that the sequence gives up there and the one that it
// holds from now on, kept from its parent (-1: none).  A sequence that goes on from one that it shares
// pages with mostly has the same in both.
struct ForkCount { int gives, holds; int* keep_at; };
DFL_DEV ForkCount fork_count_at(const Kv4ForkArgs& a, const ForkScratch& x, const ForkView& v, int s, int i) {
  const int kept = kv4_pages(v.base[s], a.page_shift), j = i - v.count_at[s], par = v.par[s];
  const long long at = (long long)s * a.width + j;
  if (par == s) return ForkCount{a.table[at + kept], -1, nullptr};
  return ForkCount{j < v.old[s] ? a.table[at] : -1, j < kept ? a.table[(long long)par * a.width + j] : -1,
                   j < kept ? x.kept + at : nullptr};
}
constexpr int FORK_N = 4;   // places of a thread under way at once
// Counts (sign 1) or sets the counts back (-1); whether all pages are the pool's.
DFL_DEV bool fork_count(const Kv4ForkArgs& a, const ForkScratch& x, const ForkView& v, int total, int t, int nt,
                        int sign) {
  bool ok = true;
  for (int i0 = t; i0 < total; i0 += FORK_N * nt) {
    int s[FORK_N];
    step_search<FORK_N>(v.count_at, a.n_seq, i0, nt, total, s);
    ForkCount c[FORK_N];
#pragma unroll
    for (int k = 0; k < FORK_N; ++k)
      c[k] = i0 + k * nt < total ? fork_count_at(a, x, v, s[k], i0 + k * nt) : ForkCount{0, 0, nullptr};
#pragma unroll
    for (int k = 0; k < FORK_N; ++k) {
      if (i0 + k * nt >= total) break;
      // (a place past the sequence's old pages gives up none, one past its kept ones holds none)
      const bool own = v.par[s[k]] == s[k], gives = own || i0 + k * nt - v.count_at[s[k]] < v.old[s[k]];
      const bool holds = c[k].keep_at != nullptr;
      if ((gives && !fork_page_ok(a, c[k].gives)) || (holds && !fork_page_ok(a, c[k].holds))) {
        ok = false;   // (neither is counted: nor are they when the counts are set back)
        continue;
      }
      if (holds) *c[k].keep_at = c[k].holds;
      if (c[k].gives == c[k].holds) continue;
      if (gives) atomicAdd(a.refs + c[k].gives, -sign);
      if (holds) atomicAdd(a.refs + c[k].holds, sign);
    }
  }
  return ok;
}
// The page that a sequence's new rows begin inside; its marks are cleared.
DFL_DEV bool fork_edge(const Kv4ForkArgs& a, const ForkScratch& x, const ForkView& v, int s, const Kv4ForkAsk& q) {
  int e = -1;
  bool ok = true;
  if (q.grow > 0 && (q.keep & ((1 << a.page_shift) - 1))) {
    e = a.table[(long long)q.parent * a.width + (q.keep >> a.page_shift)];
    ok = fork_page_ok(a, e);
    if (ok) {
      store_agent(x.writers + e, 0);
      store_agent(x.first + e, INT32_MAX);
    } else {
      e = -1;
    }
  }
  v.edge[s] = e;
  return ok;
}
DFL_DEV void fork_mark(const ForkScratch& x, const ForkView& v, int s) {
  const int e = v.edge[s];
  if (e < 0) return;
  atomicAdd(x.writers + e, 1);
  atomicMin(x.first + e, s);
}
// Whether a sequence copies its edge page, and the pages that it takes.
DFL_DEV int fork_need(const Kv4ForkArgs& a, const ForkScratch& x, const ForkView& v, int s, int& copies) {
  const int e = v.edge[s], keep = v.base[s];
  copies = e >= 0 && !(load_agent(x.writers + e) == load_agent(a.refs + e) && load_agent(x.first + e) == s);
  return kv4_pages(keep + fork_grow(v, s), a.page_shift) - kv4_pages(keep, a.page_shift) + copies;
}
// Place i of the tables that are written.
DFL_DEV void fork_place(const Kv4ForkArgs& a, const ForkScratch& x, const ForkView& v, int s, int i) {
  const int keep = v.base[s], kept = kv4_pages(keep, a.page_shift), own = v.own[s];
  const int now = kv4_pages(keep + fork_grow(v, s), a.page_shift);
  const int j = i - v.place_at[s] + (v.par[s] == s ? kept : 0);
  const long long at = (long long)s * a.width + j;
  if (j < kept) {
    if (!(own && j == kept - 1)) a.table[at] = x.kept[at];
  } else if (j < now) {
    const int page = x.list[v.take_at[s] + own + j - kept];
    a.table[at] = page;
    a.refs[page] = 1;
  } else {
    a.table[at] = -1;
  }
}
// A sequence's copied page, and its length.
DFL_DEV void fork_own(const Kv4ForkArgs& a, const ForkScratch& x, const ForkView& v, int s) {
  const int keep = v.base[s];
  if (v.own[s]) {
    const int page = x.list[v.take_at[s]], e = v.edge[s], c = v.copy_at[s];
    a.table[(long long)s * a.width + (keep >> a.page_shift)] = page;
    a.refs[page] = 1;
    atomicAdd(a.refs + e, -1);
    x.copy_src[c] = e;
    x.copy_dst[c] = page;
    x.copy_blocks[c] = ((keep & ((1 << a.page_shift) - 1)) + 31) >> 5;
  }
  a.lens[s] = keep + fork_grow(v, s);
}
DFL_DEV void fork_row(const Kv4ForkArgs& a, const ForkScratch& x, const ForkView& v, int s, int r) {
  const int keep = v.base[s], pos = keep + (r - v.starts[s]), kept = kv4_pages(keep, a.page_shift);
  const int j = pos >> a.page_shift;
  int page;
  if (j < kept && !v.own[s]) page = v.edge[s];
  else page = x.list[v.take_at[s] + (j < kept ? 0 : v.own[s] + j - kept)];
  a.slots[r] = (page << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
  a.positions[r] = pos;
}

constexpr int FORK_ONE_PLACES = 16384, FORK_ONE_SEQS = 1024, FORK_ONE_ROWS = 8192, FORK_ONE_PAGES = 65536;

__global__ __launch_bounds__(1024) void kv4_fork_one_kernel(Kv4ForkArgs a) {
  __shared__ Sum3 lds[16];
  __shared__ int arrays[FORK_ARRAYS + 1][FORK_ONE_SEQS + 1];
  const ForkScratch x = fork_scratch(a);
  const ForkView v{arrays[0], arrays[1], arrays[2], arrays[3], arrays[4],
                   arrays[5], arrays[6], arrays[7], arrays[8], arrays[9]};
  const int s = threadIdx.x, nt = blockDim.x;
  const bool mine = s < a.n_seq;
  Kv4ForkAsk q{};
  const bool bad = mine && !fork_ask(a, s, q);
  Sum3 all;
  const Sum3 in = block_scan3(Sum3{q.counted, q.placed, q.grow}, lds, all);
  int err = __syncthreads_or(bad) ? KV4_ERR_LEN : 0;
  if (all.c > a.max_rows) err |= KV4_ERR_ROWS;
  const int counted = (int)all.a, placed = (int)all.b, rows = (int)all.c;
  int copies = 0;
  if (!err) {
    if (mine) fork_note(q, in, s, v);
    if (s == 0) v.starts[a.n_seq] = rows;
    __syncthreads();
    bool ok = !mine || fork_edge(a, x, v, s, q);
    __syncthreads();
    if (mine) fork_mark(x, v, s);
    ok = fork_count(a, x, v, counted, s, nt, 1) && ok;
    if (__syncthreads_or(!ok)) err = KV4_ERR_PAGE;
    // a thread's pages: some in a row
    const int per = (a.n_pages + nt - 1) / nt, p0 = min(s * per, a.n_pages), p1 = min(p0 + per, a.n_pages);
    int zeros = 0;
#pragma unroll 8
    for (int p = p0; p < p1; ++p) zeros += load_agent(a.refs + p) == 0;
    int own = 0;
    const int need = mine ? fork_need(a, x, v, s, own) : 0;
    Sum3 sum;
    const Sum3 upto = block_scan3(Sum3{need, own, zeros}, lds, sum);
    if (mine) {
      v.own[s] = own;
      v.take_at[s] = (int)(upto.a - need);
      v.copy_at[s] = (int)(upto.b - own);
    }
    if (!err && sum.a > sum.c) err = KV4_ERR_POOL;
    if (err) {
      fork_count(a, x, v, counted, s, nt, -1);
    } else {
      int rank = (int)(upto.c - zeros);
      for (int p = p0; p < p1 && rank < sum.a; ++p)
        if (load_agent(a.refs + p) == 0) x.list[rank++] = p;
      copies = (int)sum.b;
      __syncthreads();
      for (int i0 = s; i0 < placed; i0 += FORK_N * nt) {
        int of[FORK_N];
        step_search<FORK_N>(v.place_at, a.n_seq, i0, nt, placed, of);
#pragma unroll
        for (int k = 0; k < FORK_N; ++k)
          if (i0 + k * nt < placed) fork_place(a, x, v, of[k], i0 + k * nt);
      }
      if (mine) fork_own(a, x, v, s);
      if (s == 0) *a.n_free = (int)(sum.c - sum.a);
    }
  }
  if (mine) a.starts[s] = err ? 0 : v.starts[s];
  if (s == 0) {
    a.starts[a.n_seq] = err ? 0 : rows;
    x.totals->copies = copies;
    if (err) atomicOr(a.err, err);
  }
  for (int r = s; r < a.max_rows; r += nt) {
    if (!err && r < rows) fork_row(a, x, v, step_search(v.starts, a.n_seq, r), r);
    else a.slots[r] = a.positions[r] = -1;
  }
}

// The same in launches.
__global__ __launch_bounds__(1024) void kv4_fork_scan_kernel(Kv4ForkArgs a) {
  __shared__ Sum3 lds[16];
  const ForkScratch x = fork_scratch(a);
  const int nt = blockDim.x;
  Sum3 all{0, 0, 0};
  int bad = 0;
  for (int s0 = 0; s0 < a.n_seq; s0 += nt) {
    const int s = s0 + threadIdx.x;
    Kv4ForkAsk q{};
    if (s < a.n_seq && !fork_ask(a, s, q)) bad = 1;
    Sum3 t;
    Sum3 in = block_scan3(Sum3{q.counted, q.placed, q.grow}, lds, t);
    in.a += all.a; in.b += all.b; in.c += all.c;
    if (s < a.n_seq) {
      fork_note(q, in, s, x.view);
      if (!fork_edge(a, x, x.view, s, q)) bad |= 2;
    }
    all.a += t.a; all.b += t.b; all.c += t.c;
  }
  int err = __syncthreads_or(bad & 1) ? KV4_ERR_LEN : 0;
  if (all.c > a.max_rows) err |= KV4_ERR_ROWS;
  if (!err && __syncthreads_or(bad)) err = KV4_ERR_PAGE;   // (err is the same in all threads)
  if (threadIdx.x == 0) {
    x.view.starts[a.n_seq] = (int)all.c;
    *x.totals = ForkTotals{err, (int)all.a, (int)all.b, (int)all.c, 0, 0, 0, 0};
    if (err) atomicOr(a.err, err);
  }
}
__global__ __launch_bounds__(256) void kv4_fork_count_kernel(Kv4ForkArgs a) {
  const ForkScratch x = fork_scratch(a);
  if (x.totals->err) return;
  const int t = blockIdx.x * 256 + threadIdx.x, nt = gridDim.x * 256;
  for (int s = t; s < a.n_seq; s += nt) fork_mark(x, x.view, s);
  if (!fork_count(a, x, x.view, x.totals->counted, t, nt, 1)) {
    atomicOr(&x.totals->bad, KV4_ERR_PAGE);
    atomicOr(a.err, KV4_ERR_PAGE);
  }
}
// Free pages of every KV4_FORK_CHUNK, 4 a thread.
DFL_DEV int fork_free4(const Kv4ForkArgs& a, int chunk, bool (&free)[4]) {
  int n = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int p = chunk * KV4_FORK_CHUNK + 4 * threadIdx.x + k;
    free[k] = p < a.n_pages && load_agent(a.refs + p) == 0;
    n += free[k];
  }
  return n;
}
__global__ __launch_bounds__(256) void kv4_fork_ask_kernel(Kv4ForkArgs a) {
  __shared__ Sum3 lds[16];
  const ForkScratch x = fork_scratch(a);
  if (x.totals->err) return;
  const ForkView& v = x.view;
  for (int s = blockIdx.x * 256 + threadIdx.x; s < a.n_seq; s += gridDim.x * 256) {
    int own;
    v.take_at[s] = fork_need(a, x, v, s, own);   // (sums of these follow)
    v.own[s] = own;
  }
  for (int c = blockIdx.x; c < kv4_fork_chunks(a.n_pages); c += gridDim.x) {
    bool free[4];
    Sum3 all;
    block_scan3(Sum3{fork_free4(a, c, free), 0, 0}, lds, all);
    if (threadIdx.x == 0) x.chunks[c] = (int)all.a;
  }
}
__global__ __launch_bounds__(1024) void kv4_fork_sum_kernel(Kv4ForkArgs a) {
  __shared__ Sum3 lds[16];
  const ForkScratch x = fork_scratch(a);
  if (x.totals->err) return;
  const ForkView& v = x.view;
  const int chunks = kv4_fork_chunks(a.n_pages), nt = blockDim.x;
  Sum3 all{0, 0, 0};
  for (int i0 = 0; i0 < max(a.n_seq, chunks); i0 += nt) {
    const int i = i0 + threadIdx.x;
    const int need = i < a.n_seq ? v.take_at[i] : 0, own = i < a.n_seq ? v.own[i] : 0;
    const int zeros = i < chunks ? x.chunks[i] : 0;
    Sum3 t;
    const Sum3 in = block_scan3(Sum3{need, own, zeros}, lds, t);
    if (i < a.n_seq) {
      v.take_at[i] = (int)min(all.a + in.a - need, 0x7fffffffll);
      v.copy_at[i] = (int)(all.b + in.b - own);
    }
    if (i < chunks) x.chunks[i] = (int)(all.c + in.c - zeros);
    all.a += t.a; all.b += t.b; all.c += t.c;
  }
  if (threadIdx.x == 0) {
    int bad = x.totals->bad;
    if (!bad && all.a > all.c) {
      bad = KV4_ERR_POOL;
      atomicOr(a.err, bad);
    }
    x.totals->bad = bad;
    x.totals->need = bad ? 0 : (int)all.a;
    x.totals->copies = bad ? 0 : (int)all.b;
    if (!bad) *a.n_free = (int)(all.c - all.a);
  }
}
__global__ __launch_bounds__(256) void kv4_fork_list_kernel(Kv4ForkArgs a) {
  __shared__ Sum3 lds[16];
  const ForkScratch x = fork_scratch(a);
  if (x.totals->err) return;
  const int t = blockIdx.x * 256 + threadIdx.x, nt = gridDim.x * 256;
  if (x.totals->bad) {   // as it was
    fork_count(a, x, x.view, x.totals->counted, t, nt, -1);
    return;
  }
  for (int c = blockIdx.x; c < kv4_fork_chunks(a.n_pages); c += gridDim.x) {
    if (x.chunks[c] >= x.totals->need) break;
    bool free[4];
    const int n = fork_free4(a, c, free);
    Sum3 all;
    int rank = x.chunks[c] + (int)block_scan3(Sum3{n, 0, 0}, lds, all).a - n;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (free[k] && rank < x.totals->need) x.list[rank] = c * KV4_FORK_CHUNK + 4 * threadIdx.x + k;
      rank += free[k];
    }
  }
}
__global__ __launch_bounds__(256) void kv4_fork_place_kernel(Kv4ForkArgs a) {
  const ForkScratch x = fork_scratch(a);
  const ForkView& v = x.view;
  const int t = blockIdx.x * 256 + threadIdx.x, nt = gridDim.x * 256;
  const bool none = x.totals->err || x.totals->bad;
  const int rows = none ? 0 : x.totals->rows, placed = none ? 0 : x.totals->placed;
  for (int i0 = t; i0 < placed; i0 += FORK_N * nt) {
    int of[FORK_N];
    step_search<FORK_N>(v.place_at, a.n_seq, i0, nt, placed, of);
#pragma unroll
    for (int k = 0; k < FORK_N; ++k)
      if (i0 + k * nt < placed) fork_place(a, x, v, of[k], i0 + k * nt);
  }
  for (int s = t; s <= a.n_seq; s += nt) {
    if (none) a.starts[s] = 0;
    else if (s < a.n_seq) fork_own(a, x, v, s);
  }
  for (long long r = t; r < a.max_rows; r += nt) {
    if (r < rows) fork_row(a, x, v, step_search(v.starts, a.n_seq, (int)r), (int)r);
    else a.slots[r] = a.positions[r] = -1;
  }
}
// The copied pages: a workgroup takes the kept rows' blocks of one layer's head, which follow on each
// other.
__global__ __launch_bounds__(256) void kv4_fork_copy_kernel(Kv4ForkArgs a) {
  const ForkScratch x = fork_scratch(a);
  const int per = a.n_layers * a.n_kv, sh = a.page_shift - 5;
  const long long items = (long long)x.totals->copies * per;
  for (long long i = blockIdx.x; i < items; i += gridDim.x) {
    const int c = (int)(i / per), k = (int)(i - (long long)c * per), layer = k / a.n_kv, head = k - layer * a.n_kv;
    unsigned char* pool = a.pool + layer * a.layer_bytes;
    const u32x4* from = reinterpret_cast<const u32x4*>(pool + kv4_block_at(kv4_block_no(x.copy_src[c], a.n_kv, head, sh, 0)));
    u32x4* to = reinterpret_cast<u32x4*>(pool + kv4_block_at(kv4_block_no(x.copy_dst[c], a.n_kv, head, sh, 0)));
    const int n = x.copy_blocks[c] * (KV4_BLOCK / 16);
    for (int j = threadIdx.x; j < n; j += 4 * 256) {
      u32x4 w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) w[u] = from[min(j + 256 * u, n - 1)];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j + 256 * u < n) to[j + 256 * u] = w[u];
    }
  }
}

}  // namespace

void launch_kv4_fork(const Kv4ForkArgs& a, hipStream_t st) {
  const dim3 block(256);
  // (the places that a step may look at; without parents only those that lengths give up and take)
  const long long places = a.parent ? (long long)a.n_seq * a.width : 0;
  if (a.n_seq <= FORK_ONE_SEQS && a.max_rows <= FORK_ONE_ROWS && a.n_pages <= FORK_ONE_PAGES && places <= FORK_ONE_PLACES) {
    const int threads = a.n_seq <= 256 && a.max_rows <= 1024 && a.n_pages <= 4096 && places <= 2048 ? 256 : 1024;
    hipLaunchKernelGGL(kv4_fork_one_kernel, dim3(1), dim3(threads), 0, st, a);
  } else {
    // (how many places a step counts and writes is known on the device alone)
    const dim3 wide(512);
    const dim3 pages(min(1024, max(kv4_fork_chunks(a.n_pages), (a.n_seq + 255) / 256)));
    hipLaunchKernelGGL(kv4_fork_scan_kernel, dim3(1), dim3(1024), 0, st, a);
    hipLaunchKernelGGL(kv4_fork_count_kernel, wide, block, 0, st, a);
    hipLaunchKernelGGL(kv4_fork_ask_kernel, pages, block, 0, st, a);
    hipLaunchKernelGGL(kv4_fork_sum_kernel, dim3(1), dim3(1024), 0, st, a);
    hipLaunchKernelGGL(kv4_fork_list_kernel, wide, block, 0, st, a);
    hipLaunchKernelGGL(kv4_fork_place_kernel, wide, block, 0, st, a);
  }
  const long long most = (long long)a.n_seq * a.n_layers * a.n_kv;
  hipLaunchKernelGGL(kv4_fork_copy_kernel, dim3((unsigned)(most < 2048 ? most : 2048)), block, 0, st, a);
}

}  // namespace dfl
