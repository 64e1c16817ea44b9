// Paged key/value cache in 4 bits: layout, launch interface and host checks.
//
// Format.  A row of one head (128 values) is four groups of 32.  A group is a shared exponent
// byte b and 32 four-bit codes, standing for code * 2^(b - 127) with the code a sign and one of
// 0, 0.5, 1, 1.5, 2, 3, 4, 6 (the 4-bit floats of gfx950's conversions; the OCP microscaling
// layout of 32 elements to an e8m0 scale).  b is the smallest exponent >= 0 for which the group's
// largest magnitude is at most 7 * 2^(b - 127): what lies in (6, 7] rounds to 6, nothing is
// clipped further than half a step.  b = 255 marks a group that held an infinity or a NaN and
// stands for NaN.
//
// Layout.  The pool is [layer][page][kv head][page / 32] blocks of 4352 bytes, a block being 32
// consecutive rows (keys) of one head:
//   bytes    0 .. 2047   K codes: 16 bytes of each row's group 0, then of group 1, 2, 3
//   bytes 2048 .. 4095   V codes, the same
//   bytes 4096 .. 4351   exponent bytes, 4 a word: word i + 16 g holds group g of the rows i and
//                        16 + i: bytes K0, K1, V0, V1
// In a group's 16 bytes the byte e holds values 2e (low nibble) and 2e + 1.  A lane's operand of a
// matrix product is a row's group, so a wave reads a block in pieces of 1 KiB in which lane after
// lane takes 16 bytes, from memory as from LDS.
//
// Everything here but the launchers is plain host code too, so that it can be tested on a CPU.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dfl {

#define DFL_HD __host__ __device__ inline

constexpr int KV4_D = 128;                 // head dimension
constexpr int KV4_KEYS = 32;               // rows of a block
constexpr int KV4_V = 2048, KV4_SC = 4096; // V codes and exponent bytes of a block
constexpr int KV4_BLOCK = 4352;            // bytes of a block
constexpr int KV4_CUS = 256;               // compute units of an MI355X
constexpr int KV4_MAX_SEQS = 65536;

// error bits (they follow the library's bits 0 .. 2)
constexpr int KV4_ERR_LEN = 8;       // step: a length out of range
constexpr int KV4_ERR_POOL = 16;     // step: not enough free pages
constexpr int KV4_ERR_ROWS = 32;     // step: more new rows than the slot map holds
constexpr int KV4_ERR_SLOT = 64;     // append, read: a slot outside the pool
constexpr int KV4_ERR_PAGE = 128;    // attend, step: a page, length, row range or free count out of bounds

// Offsets in a block, of K (v = 0) or V (v = 1): the 16 code bytes of group g of row r, and its
// exponent byte.
DFL_HD int kv4_code_at(int r, int g, int v) { return v * KV4_V + g * 512 + r * 16; }
DFL_HD int kv4_scale_at(int r, int g, int v) {
  return KV4_SC + 4 * ((r & 15) + 16 * g) + 2 * v + (r >> 4);
}
// Number and byte offset in a layer's pool of block `sub` of a page's head (check_kv4_pool keeps
// the number within 32 bits).
DFL_HD uint32_t kv4_block_no(uint32_t page, int n_kv, int head, int sub_shift, int sub) {
  return ((page * (uint32_t)n_kv + (uint32_t)head) << sub_shift) + (uint32_t)sub;
}
DFL_HD unsigned long long kv4_block_at(uint32_t no) { return (unsigned long long)no * KV4_BLOCK; }

DFL_HD int kv4_pages(int n, int page_shift) { return (int)(((long long)n + (1 << page_shift) - 1) >> page_shift); }

// ---- step (block tables and slot maps) ----
struct Kv4StepArgs {
  int n_seq, page_shift, width, n_pages, max_rows;
  const int *keep, *grow;      // [n_seq], either may be null (keep everything, grow by nothing)
  int *lens, *table, *free_pages, *n_free;
  int *starts, *slots, *positions;
  int* scratch;                // kv4_step_scratch(n_seq) ints
  int* err;
};
// scratch: the scan's error, freed and taken totals, free pages before, the check's error; then
// [n_seq] kept lengths, freed and taken pages before each sequence
DFL_HD long long kv4_step_scratch(int n_seq) { return 5 + 3ll * n_seq; }

// What one sequence asks of a step; false if a length is out of range.
struct Kv4Ask { int keep, grow, freed, taken; };
DFL_HD bool kv4_ask(int len, int keep, int grow, int width, int page_shift, Kv4Ask& a) {
  const bool ok = len >= 0 && (long long)len <= ((long long)width << page_shift) && keep >= 0 &&
                  keep <= len && grow >= 0 &&
                  (long long)keep + grow <= ((long long)width << page_shift);
  a = Kv4Ask{ok ? keep : 0, ok ? grow : 0, 0, 0};
  if (!ok) return false;
  const int pk = kv4_pages(keep, page_shift);
  a.freed = kv4_pages(len, page_shift) - pk;
  a.taken = kv4_pages(keep + grow, page_shift) - pk;
  return true;
}

// ---- step of sequences that share pages ----
struct Kv4ForkArgs {
  int n_seq, page_shift, width, n_pages, max_rows, n_kv, n_layers;
  const int *parent, *keep, *grow;   // [n_seq], any may be null (itself, all of the parent's, nothing)
  int *lens, *table, *refs, *n_free;
  int *starts, *slots, *positions;
  unsigned char* pool;               // all layers
  long long layer_bytes;             // of a layer's pages
  int* scratch;                      // kv4_fork_scratch(..) ints
  int* err;
};
constexpr int KV4_FORK_TOTALS = 8;
constexpr int KV4_FORK_CHUNK = 1024;   // pages whose free ones are counted together
DFL_HD int kv4_fork_chunks(int n_pages) { return (int)(((long long)n_pages + KV4_FORK_CHUNK - 1) / KV4_FORK_CHUNK); }
// totals; [n_seq] the copies (3), the view (9); [n_pages] writers, first writer, list of free pages; free
// pages of the chunks; with parents the kept pages [n_seq][width]
DFL_HD long long kv4_fork_scratch(int n_seq, int width, int n_pages, bool parents) {
  return KV4_FORK_TOTALS + 12ll * n_seq + 3ll * n_pages + kv4_fork_chunks(n_pages) + (parents ? (long long)n_seq * width : 0);
}
// What one sequence asks of a step: places whose pages may gain or lose a holder (counted), places that
// are written (placed; its last kept page's apart), pages that it had (old); false if a length is out of
// range.
struct Kv4ForkAsk { int keep, grow, parent, old, counted, placed; };
DFL_HD bool kv4_fork_ask(int s, int parent, int from, int len, int keep, int grow, int width, int page_shift,
                         Kv4ForkAsk& a) {
  const long long cap = (long long)width << page_shift;
  const bool ok = parent >= 0 && len >= 0 && len <= cap && from >= 0 && from <= cap && keep >= 0 && keep <= from &&
                  grow >= 0 && (long long)keep + grow <= cap;
  a = Kv4ForkAsk{0, 0, s, 0, 0, 0};
  if (!ok) return false;
  const int kept = kv4_pages(keep, page_shift), now = kv4_pages(keep + grow, page_shift);
  a = Kv4ForkAsk{keep, grow, parent, kv4_pages(len, page_shift), 0, 0};
  const int most = now > a.old ? now : a.old;
  a.counted = parent == s ? a.old - kept : a.old > kept ? a.old : kept;
  a.placed = parent == s ? most - kept : most;
  return true;
}

// ---- append / read ----
struct Kv4RowsArgs {
  const void *k, *v;           // append: rows in; read: unused
  void *ok, *ov;               // read: rows out
  long long k_row, k_head, v_row, v_head;   // strides in elements
  int dtype;                   // 0 fp32, 1 fp16, 2 bf16
  int rows, n_kv, page_shift, n_pages;
  const int* slots;
  unsigned char* pool;         // one layer's pages
  int* err;
};

// ---- attention ----
struct Kv4AttnArgs {
  const void* q;
  void* out;
  float* lse;                  // [n_rows][n_heads] or null
  long long q_row, q_head;     // strides in elements (out is contiguous)
  int dtype;                   // 1 fp16, 2 bf16
  int n_rows, n_heads, n_kv, n_seq, causal;
  float scale_log2;
  const int *starts, *lens, *table;
  int width, page_shift, n_pages;
  const unsigned char* pool;   // one layer's pages
  float* ws;
  int workers;                 // workgroups that share the places (Kv4Cut)
  int* err;
  const int* ends;             // where the sequences' rows end (starts + 1)
  // attention with shared keys: the first n_groups of the n_seq sequences are groups' shared keys, not
  // causal, the others the sequences' own rest
  int n_groups;
  const long long* row_of;     // [n_seq] where a sequence's pages begin in the table
  const int* skip;             // [n_seq - n_groups] pages of a sequence that its group's keys hold
  struct Kv4Rec* recs;         // [2][n_rows][n_heads] where a row's rest and shared part lie
  float *state_o, *state_ml;   // [2][n_rows][n_heads] states of parts that one worker has whole: sums
                               // [128], (reference, sum of weights)
  int* seq_of;                 // [n_rows] the sequence of a row (any value for rows of none)
  float* shared_ws;            // partials of the shared parts
};
// Workers (w0 .. w1) that have partials of a row's unit and its place in them; w0 -1: in the states, -2:
// it is written already.
struct Kv4Rec { int w0, w1, c, pad; };

// The work of a launch.  Sequence s contributes, for each kv head and each of its query tiles, one
// unit; units are numbered sequence by sequence, head by head, tile by tile.  A unit takes up
// KV4_PAD + nblk places in a row: the first KV4_PAD stand for what a unit costs besides its key
// blocks (finding it, its queries, the first loads' latency, its result), so that a worker with
// many short units has no more to do than one with a part of a long one; then one for each key
// block that its rows see, and now and then one more.  Worker w takes the places
// [w * per, (w + 1) * per); a unit whose blocks several workers share leaves one partial result
// with each (slot kv4_piece), which the merge joins.
//
// The places of a head's tiles 0 .. t - 1 are KV4_PAD t + floor((slope t (t - 1) / 2 + base t) / m)
// with m = 32 ratio.  Tile t sees ceil(v / 32) blocks, v = len - qlen + 1 + floor((tile_rows (t + 1)
// - 1) / ratio) the keys that its last row's token sees; that is floor((slope t + base) / m) with
// slope = tile_rows and base = ratio (len - qlen + 32) + tile_rows - 1, and the floor of a sum is
// not below the sum of floors.  Where every row sees all keys, slope = 0 and base = ratio (len + 31).
// (Keys before the first row at least 0, keys at least 1: every unit has a block, so that rows that
// see nothing are written too.)
//
// KV4_PAD 8, 10 and 12 (KV4_MIN_PLACES 12, 12, 14) as measured, us: eight blocks of 32 rows over
// 5000 keys (32 heads on 8) 48.6, 47.3, 45.5; sixteen of 8 rows over 300 keys 16.7, 17.3, 18.2; one
// token over 2000 keys 12.6, 12.8, 14.8; 64 tokens over 1000 keys 26.0, 24.0, 24.5.
constexpr int KV4_PAD = 10;
struct Kv4Seq {
  int q0, qlen, len, tiles;
  long long slope, base, m;
  int bad;
};
DFL_HD Kv4Seq kv4_seq(int q0, int q1, int len, int n_rows, int width, int page_shift, int ratio,
                      int tile_rows, bool causal) {
  Kv4Seq s;
  const long long cap = (long long)width << page_shift;
  s.bad = q0 < 0 || q1 < q0 || q1 > n_rows || len < 0 || (long long)len > cap;
  s.q0 = s.bad ? 0 : q0;
  s.qlen = s.bad ? 0 : q1 - q0;
  s.len = s.bad ? 0 : len;
  s.tiles = (int)(((long long)s.qlen * ratio + tile_rows - 1) / tile_rows);
  const long long before = s.len > s.qlen ? s.len - s.qlen : 0;
  s.slope = causal ? tile_rows : 0;
  s.base = causal ? ratio * (before + KV4_KEYS) + tile_rows - 1
                  : ratio * ((long long)(s.len > 1 ? s.len : 1) + KV4_KEYS - 1);
  s.m = (long long)KV4_KEYS * ratio;
  return s;
}
// slope t (t - 1) / 2 + base t
DFL_HD long long kv4_sum(const Kv4Seq& s, long long t) { return s.slope * (t * (t - 1) / 2) + s.base * t; }
// floor(n / d) for 0 <= n < 2^52, 0 < d: both are whole in a double, and a quotient below a whole
// number is below it by at least 1 / d, more than the rounding.  (The wide whole-number division is
// some 170 instructions, and there are seven of them.)
DFL_HD long long kv4_div(long long n, long long d) { return (long long)((double)n / (double)d); }
// Places of a head's first t tiles, and of a sequence's units.
DFL_HD long long kv4_places(const Kv4Seq& s, long long t) {
  return KV4_PAD * t + kv4_div(kv4_sum(s, t), s.m);
}
DFL_HD long long kv4_cost(const Kv4Seq& s, int n_kv) { return n_kv * kv4_places(s, s.tiles); }
// Whether tile t begins at or before place r of its head.
DFL_HD bool kv4_begun(const Kv4Seq& s, long long t, long long r) {
  return kv4_sum(s, t) < (r - KV4_PAD * t + 1) * s.m;
}
// Fewest places of a worker: 10, 12, 16 and 32 take, us, for one token over 500 keys 10.4, 9.8, 10.9,
// 14.3, for a block of 32 rows over 500 keys 21.6, 21.8, 24.1, 34.0.
constexpr int KV4_MIN_PLACES = 12;
DFL_HD long long kv4_per(long long total, int workers) {
  const long long per = kv4_div(total + workers - 1, workers);
  return per < KV4_MIN_PLACES ? KV4_MIN_PLACES : per;
}
// Partial slot of worker w for a shared unit whose first block is at place r0: a worker has at
// most one unit that it goes on with, and one that it begins and leaves.
DFL_HD long long kv4_piece(long long w, long long per, long long r0) {
  return 2 * w + (r0 < w * per ? 0 : 1);
}
// Floats of one partial: O [tile rows][128] in the order of the kernel's registers, then (max,
// sum) a row.
DFL_HD long long kv4_piece_floats(int tile_rows) { return (long long)tile_rows * (KV4_D + 2); }
// What a worker notes of a shared unit for the merge.
struct Kv4Note { int w1, head, tile, q0, qlen, len, pad[2]; };
// Bytes of a launch's workspace.
DFL_HD long long kv4_ws_bytes(int tile_rows, int workers) {
  return workers * (2 * kv4_piece_floats(tile_rows) * (long long)sizeof(float) + (long long)sizeof(Kv4Note));
}
// Whether every count above stays below 2^52, for any lengths that the launch can have.
DFL_HD bool kv4_counts_fit(int n_rows, int ratio, int n_kv, int n_seq, int width, int page_shift, int tile_rows) {
  const double cap = (double)((long long)width << page_shift) + KV4_KEYS;
  const double tiles = (double)n_rows * ratio / tile_rows + n_seq + 1;
  const double sum = tile_rows * tiles * tiles + (ratio * cap + tile_rows) * tiles;
  return sum < 4e15 && (sum / KV4_KEYS + KV4_PAD * tiles) * n_kv < 4e15;
}

// How a launch is cut (what its workspace holds follows from it).
struct Kv4Cut {
  int tile_rows;   // query rows of a unit: 16 or 32 (each wave has them all and a fourth of the
                   // keys) or 128 (each wave has 32 of them and all keys)
  int workers;     // workgroups
};
inline Kv4Cut kv4_cut(int n_rows, int n_heads, int n_kv, int n_seq) {
  Kv4Cut c{};
  // Rows of a kv head in a sequence, on average over those that can have any.  Which sequences have
  // rows, and which rows are a sequence's, is known on the device alone: idle sequences and spare
  // rows count, and a call takes longer with many of them, us: a prompt of 4096 rows among 1024
  // sequences 314 (alone 160), eight blocks of 32 rows among 64 57 (46), 64 tokens over 2000 keys in
  // a call of 2048 rows 55 (34); one such block among 64 is faster in tiles of 16, 22 (34).
  const long long seqs = n_seq < n_rows ? n_seq : n_rows;
  const long long rows = ((long long)n_rows * (n_heads / n_kv) + seqs - 1) / seqs;
  // us, eight sequences of 5000 keys, 8 kv heads: 16 rows in tiles of 16 and 32 22.2, 27.1; 32 rows
  // in tiles of 32 27.9, 40 rows in tiles of 128 41.0; tiles of 64 (two waves, else as those of 128)
  // took 40.4 and at 64 rows 40.3 for 41.5.  Workgroups for each CU: as many as fit at once with
  // tiles of 32 and 128 (LDS and registers); of four that fit with 16, three: 64 ragged tokens take
  // 93 us with two, 89, 100 with four; sixteen tokens over 65 thousand keys 214, 216, 253.
  c.tile_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 128;
  c.workers = KV4_CUS * (c.tile_rows == 16 ? 3 : 2);
  return c;
}

// How an attention with shared keys is cut.  Groups and sequences are in one launch, in tiles of as
// many rows, or the groups are in one of tiles of 128 and the sequences in one of 16.
struct Kv4SharedCut {
  int own, shared;     // query rows of a unit in the sequences' own parts and the shared ones; 0: not shared
  int workers, shared_workers;
};
inline Kv4SharedCut kv4_shared_cut(int n_rows, int n_heads, int n_kv, int n_seq, int n_groups) {
  // Sequences of more than 16 rows of a kv head fill their tiles: keys read once more cost them
  // little, and the group's states are written and read on top.  Us, attended apart and together (in
  // tiles of 128): 16 sequences of 32 rows over 1651 to 7844 shared keys 37, 49; 8 over 32000 73, 69; 16
  // of 64 rows over 8000 79, 73.
  const Kv4Cut own = kv4_cut(n_rows, n_heads, n_kv, n_seq);
  if (own.tile_rows != 16) return Kv4SharedCut{0, 0, 0, 0};
  // Rows of a kv head in a group, on average.  Us in tiles of 16, 32 and 128, over 1024, 4096, 16384 and
  // 32768 shared keys, one group, 8 kv heads in bf16:
  //    64 rows  27 30 37 46    28 31 38 46    40 48 58 66
  //   128       28 33 47 68    29 34 45 61    43 53 63 70
  //   256       33 42 69 107   34 41 62 91    53 59 70 85
  //   512       41 57 112 184  45 57 100 154  62 71 91 121
  //  1024       50 77 184 318  52 74 160 260  64 73 116 173
  // The borders lie where long texts turn: past 512 rows a text of 4096 keys takes 14 us more than in
  // tiles of 32, as the host does not know its length.  The average is over all groups that the call
  // names, also those of one sequence or with nothing in common, of which the host knows as little: 1024
  // rows behind 32768 keys take 173 us, 242 and 309 with 4 and 8 single sequences named as groups beside
  // them, 177 and 173 with those outside of the boundaries (without groups 520).
  const long long groups = n_groups < n_rows ? n_groups : n_rows, rows = (long long)n_rows * (n_heads / n_kv);
  if (rows >= 512 * groups) return Kv4SharedCut{16, 128, own.workers, 2 * KV4_CUS};
  if (rows >= 128 * groups) return Kv4SharedCut{32, 32, 2 * KV4_CUS, 0};
  return Kv4SharedCut{16, 16, own.workers, 0};
}
// Its workspace (offsets).
struct Kv4SharedWs { long long own, shared, state_o, state_ml, recs, row_of, q0, q1, len, skip, seq_of, bytes; };
inline Kv4SharedWs kv4_shared_ws(int n_rows, int n_heads, int n_kv, int n_seq, int n_groups) {
  const Kv4SharedCut c = kv4_shared_cut(n_rows, n_heads, n_kv, n_seq, n_groups);
  const long long rows = (long long)n_rows * n_heads, all = (long long)n_groups + n_seq;
  Kv4SharedWs w{};
  if (!c.own) {   // (that of an attention without groups)
    const Kv4Cut d = kv4_cut(n_rows, n_heads, n_kv, n_seq);
    w.bytes = kv4_ws_bytes(d.tile_rows, d.workers);
    return w;
  }
  long long at = 0;
  auto take = [&](long long n) { const long long p = at; at += (n + 15) / 16 * 16; return p; };
  w.own = take(kv4_ws_bytes(c.own, c.workers));
  w.shared = c.shared_workers ? take(kv4_ws_bytes(c.shared, c.shared_workers)) : w.own;
  w.state_o = take(2 * rows * KV4_D * 4);
  w.state_ml = take(2 * rows * 8);
  w.recs = take(2 * rows * (long long)sizeof(Kv4Rec));
  w.row_of = take(8 * all);
  w.q0 = take(4 * all);
  w.q1 = take(4 * all);
  w.len = take(4 * all);
  w.skip = take(4ll * n_seq);
  w.seq_of = take(4ll * n_rows);
  w.bytes = at;
  return w;
}

inline const char* check_kv4_pool(int n_kv, int page_shift, int n_pages) {
  if (n_kv < 1 || n_kv > 1024) return "kv heads outside [1, 1024]";
  if (page_shift < 5 || page_shift > 8) return "page rows must be 32, 64, 128 or 256";
  if (n_pages < 1 || ((long long)n_pages << page_shift) > 0x7fffffffll ||
      (((long long)n_pages * n_kv) << (page_shift - 5)) > 0xffffffffll)
    return "pool pages out of range (at least one, slots below 2^31, blocks below 2^32)";
  return nullptr;
}
inline const char* check_kv4_step(const Kv4StepArgs& a) {
  if (const char* e = check_kv4_pool(1, a.page_shift, a.n_pages)) return e;
  if (a.n_seq < 1 || a.n_seq > KV4_MAX_SEQS) return "sequences outside [1, 65536]";
  if (a.width < 1 || ((long long)a.width << a.page_shift) > 0x7fffffffll)
    return "table width out of range";
  if (a.max_rows < 0) return "negative row capacity";
  if (!a.lens || !a.table || !a.free_pages || !a.n_free || !a.starts || !a.scratch || !a.err)
    return "null pointer";
  if (a.max_rows > 0 && (!a.slots || !a.positions)) return "null slot map";
  return nullptr;
}
inline const char* check_kv4_fork(const Kv4ForkArgs& a) {
  if (const char* e = check_kv4_pool(a.n_kv, a.page_shift, a.n_pages)) return e;
  if (a.n_seq < 1 || a.n_seq > KV4_MAX_SEQS) return "sequences outside [1, 65536]";
  if (a.width < 1 || ((long long)a.width << a.page_shift) > 0x7fffffffll) return "table width out of range";
  if ((long long)a.n_seq * a.width >= (1ll << 29)) return "2^29 places in the table or more";
  if (a.n_layers < 1 || a.n_layers > 65536) return "layers outside [1, 65536]";
  if (a.layer_bytes < (((long long)a.n_pages * a.n_kv) << (a.page_shift - 5)) * KV4_BLOCK || (a.layer_bytes & 15))
    return "a layer's bytes do not hold its pages, or are no multiple of 16";
  if (a.max_rows < 0) return "negative row capacity";
  if (!a.lens || !a.table || !a.refs || !a.n_free || !a.starts || !a.pool || !a.scratch || !a.err)
    return "null pointer";
  if (a.max_rows > 0 && (!a.slots || !a.positions)) return "null slot map";
  if (reinterpret_cast<uintptr_t>(a.pool) & 15) return "the pool must be 16-byte aligned";
  return nullptr;
}
inline const char* check_kv4_rows(const Kv4RowsArgs& a, bool append) {
  if (const char* e = check_kv4_pool(a.n_kv, a.page_shift, a.n_pages)) return e;
  if (a.rows < 0) return "negative row count";
  if (a.dtype < 0 || a.dtype > 2) return "dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)";
  if (!a.slots || !a.pool || !a.err) return "null pointer";
  if (append ? (!a.k || !a.v) : (!a.ok || !a.ov)) return "null rows";
  auto mis = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  if (mis(a.k) || mis(a.v) || mis(a.ok) || mis(a.ov) || mis(a.pool))
    return "rows and pool must be 16-byte aligned";
  if ((a.k_row | a.k_head | a.v_row | a.v_head) & 7) return "row and head strides must be multiples of 8";
  return nullptr;
}
// n_groups: 0, or those of a launch with shared keys.
inline const char* check_kv4_attn(const Kv4AttnArgs& a, int n_groups = 0) {
  if (const char* e = check_kv4_pool(a.n_kv, a.page_shift, a.n_pages)) return e;
  if (a.n_rows < 0) return "negative row count";
  if (a.n_heads < 1 || a.n_heads % a.n_kv) return "query heads must be a multiple of the kv heads";
  if (a.n_heads / a.n_kv > 1024) return "more than 1024 query heads to a kv head";
  if ((long long)a.n_rows * a.n_heads > 0x7fffffffll) return "too many query rows";
  if (a.dtype != 1 && a.dtype != 2) return "dtype must be 1 (fp16) or 2 (bf16)";
  if (a.n_seq < 1 || a.n_seq > KV4_MAX_SEQS) return "sequences outside [1, 65536]";
  if (a.width < 1 || ((long long)a.width << a.page_shift) > 0x7fffffffll)
    return "table width out of range";
  if (n_groups < 0 || n_groups > a.n_seq) return "more groups than sequences";
  // (with shared keys every row is in two sequences)
  if (n_groups && a.n_rows > 0x3fffffff) return "too many query rows";
  if (a.n_rows > 0 && !kv4_counts_fit(n_groups ? 2 * a.n_rows : a.n_rows, a.n_heads / a.n_kv, a.n_kv, a.n_seq + n_groups,
                                      a.width, a.page_shift, kv4_cut(a.n_rows, a.n_heads, a.n_kv, a.n_seq).tile_rows))
    return "too many query rows for so long a table";
  if (!(a.scale_log2 > 0.f) || a.scale_log2 > 1e30f) return "scale must be positive and finite";
  if (!a.q || !a.out || !a.starts || !a.lens || !a.table || !a.pool || !a.err) return "null pointer";
  auto mis = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  if (mis(a.q) || mis(a.out) || mis(a.pool) || mis(a.ws)) return "rows, pool and workspace must be 16-byte aligned";
  if ((a.q_row | a.q_head) & 7) return "row and head strides must be multiples of 8";
  return nullptr;
}

void launch_kv4_step(const Kv4StepArgs& a, hipStream_t st);
void launch_kv4_fork(const Kv4ForkArgs& a, hipStream_t st);
void launch_kv4_append(const Kv4RowsArgs& a, hipStream_t st);
void launch_kv4_read(const Kv4RowsArgs& a, hipStream_t st);
void launch_kv4_attend(const Kv4AttnArgs& a, hipStream_t st);
void launch_kv4_attend_shared(const Kv4AttnArgs& a, const int* groups, int n_groups, hipStream_t st);

}  // namespace dfl
