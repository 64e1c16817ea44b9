// Host checks of the paged 4-bit cache: the layout's index maps, what a step asks of lengths that
// do not fit, the even split of the attention's work, and the launch argument rules.  No GPU.
#include <cstdio>
#include <cstdlib>
#include <string>
#include <vector>

#include "dfl_kv4.h"

using namespace dfl;

static void must(bool ok, const char* what) {
  if (!ok) {
    std::printf("FAIL: %s\n", what);
    std::exit(1);
  }
}
static bool says(const char* got, const char* needle) {
  if (!got) return false;
  return std::string(got).find(needle) != std::string::npos;
}

static void layout() {
  std::vector<int> bytes(KV4_BLOCK, 0);
  for (int r = 0; r < 32; ++r)
    for (int v = 0; v < 2; ++v)
      for (int g = 0; g < 4; ++g) {
        for (int b = 0; b < 16; ++b) must(!bytes[kv4_code_at(r, g, v) + b]++, "codes overlap");
        const int at = kv4_scale_at(r, g, v);
        must(at >= KV4_SC && at < KV4_BLOCK && !bytes[at]++, "exponent bytes overlap");
      }
  for (int b : bytes) must(b == 1, "a block has no gaps");
  must(kv4_block_at(kv4_block_no(70000, 8, 7, 3, 7)) == ((70000ull * 8 + 7) * 8 + 7) * KV4_BLOCK,
       "offsets past 32 bits");
  must(kv4_block_at(kv4_block_no(0x1ffffffu, 16, 15, 3, 7)) == 0xffffffffull * KV4_BLOCK, "the last block");
}

static void asks() {
  Kv4Ask a;
  const int big = 0x7fffffff;
  must(kv4_ask(100, 40, 50, 4, 5, a) && a.freed == 2 && a.taken == 1, "pages back and taken");
  must(kv4_ask(96, 96, 0, 3, 5, a) && a.freed == 0 && a.taken == 0, "nothing to do");
  must(kv4_ask(0, 0, 96, 3, 5, a) && a.taken == 3, "a full table");
  for (auto t : {std::vector<int>{0, 0, 97}, {0, 1, 0}, {10, 11, 0}, {10, -1, 0}, {10, 5, -1},
                 {97, 0, 0}, {-1, 0, 0}, {50, 50, big}, {big, big, big}, {-big - 1, 0, 0}}) {
    must(!kv4_ask(t[0], t[1], t[2], 3, 5, a), "a length out of range");
    must(a.freed == 0 && a.taken == 0 && a.grow == 0 && a.keep == 0, "asks for nothing then");
  }
  must(kv4_ask(0, 0, 0x7fffffe0, 0x3ffffff, 5, a), "the longest table");
}

// Keys that the last row of a tile sees, from the definition.
static long long seen(const Kv4Seq& s, int ratio, int rows, int t, bool causal) {
  long long last = (long long)(t + 1) * rows - 1;
  if (last > (long long)s.qlen * ratio - 1) last = (long long)s.qlen * ratio - 1;
  long long v = causal ? s.len - s.qlen + last / ratio + 1 : s.len;
  return v < 0 ? 0 : v > s.len ? s.len : v;
}

// Every block of every unit is one worker's; the pieces of a shared unit are different slots, and
// those that the merge reads are those that the workers write.
static void split(const std::vector<int>& q, const std::vector<int>& lens, int heads, int kv, int rows, int workers,
                  bool causal) {
  struct U { long long r0; int nblk; };
  std::vector<U> units;
  int at = 0, n = 0;
  for (int m : q) n += m;
  long long total = 0;
  for (size_t i = 0; i < q.size(); ++i) {
    const Kv4Seq s = kv4_seq(at, at + q[i], lens[i], n, 1 << 20, 5, heads / kv, rows, causal);
    must(!s.bad, "the rows fit");
    at += q[i];
    const long long head = kv4_places(s, s.tiles);
    for (int h = 0; h < kv; ++h)
      for (int t = 0; t < s.tiles; ++t) {
        const long long p0 = kv4_places(s, t), p1 = kv4_places(s, t + 1);
        const int nblk = (int)(p1 - p0) - KV4_PAD;
        const long long need = (seen(s, heads / kv, rows, t, causal) + 31) / 32;
        must(nblk >= 1 && nblk >= need, "a place for each block");
        must(lens[i] < q[i] || nblk <= need + 2, "few places besides");
        for (long long r = p0; r < p1; r += r + 97 < p1 ? 97 : 1)
          must(kv4_begun(s, t, r) && (t + 1 == s.tiles || !kv4_begun(s, t + 1, r)), "a place is its tile's");
        units.push_back({total + h * head + p0 + KV4_PAD, nblk});
      }
    total += kv4_cost(s, kv);
  }
  const long long per = kv4_per(total, workers);
  must(per >= KV4_MIN_PLACES && per * workers >= total, "the workers cover the places");
  std::vector<int> done(total, 0), slot(2ll * workers, 0), want(2ll * workers, 0);
  long long end_of_last = 0;
  for (const U& u : units) {
    must(u.r0 - KV4_PAD == end_of_last, "units lie one behind the other");
    end_of_last = u.r0 + u.nblk;
    int shared = 0;
    for (long long w = (u.r0 - KV4_PAD) / per; w * per < u.r0 + u.nblk; ++w) {   // as the walk cuts it
      const long long pos = w * per > u.r0 - KV4_PAD ? w * per : u.r0 - KV4_PAD;
      const long long end = (w + 1) * per < total ? (w + 1) * per : total;
      const long long b0 = pos > u.r0 ? pos - u.r0 : 0, b1 = u.nblk < end - u.r0 ? u.nblk : end - u.r0;
      if (b1 <= 0) continue;
      must(b1 > b0, "a run is not empty");
      for (long long b = b0; b < b1; ++b) ++done[u.r0 + b];
      if (b0 > 0 || b1 < u.nblk) {
        const long long p = kv4_piece(w, per, u.r0);
        must(p >= 0 && p < 2ll * workers && !slot[p]++, "two pieces in one slot");
        ++shared;
      }
    }
    // the merge: the worker that begins inside the unit's blocks first
    int merged = 0;
    for (long long first = u.r0 / per; first * per < u.r0 + u.nblk; ++first) {
      const long long pos = first * per;
      if (first < 1 || pos <= u.r0 || pos - per > u.r0) continue;
      must(++merged == 1, "one worker's affair");
      for (long long w = first - 1; w <= (u.r0 + u.nblk - 1) / per; ++w) ++want[kv4_piece(w, per, u.r0)];
    }
    must(merged == (shared > 0), "merged if shared");
    for (int k = -KV4_PAD; k < u.nblk; ++k) must(done[u.r0 + k] == (k >= 0), "each block once");
  }
  must(end_of_last == total && slot == want, "the merge reads what was written");
}

static void seqs() {
  // row ranges and lengths that do not fit make a sequence without rows
  for (auto t : {std::vector<int>{-1, 3, 5}, {3, 2, 5}, {0, 11, 5}, {0, 1, -1}, {0, 1, 97}, {0, 0x7fffffff, 1}})
    for (bool causal : {false, true}) {
      const Kv4Seq s = kv4_seq(t[0], t[1], t[2], 10, 3, 5, 4, 16, causal);
      must(s.bad && s.qlen == 0 && s.tiles == 0 && kv4_cost(s, 8) == 0, "a bad sequence has no work");
    }
  const Kv4Seq e = kv4_seq(2, 3, 0, 10, 3, 5, 4, 16, false);
  must(!e.bad && e.tiles == 1 && kv4_places(e, 1) == KV4_PAD + 1, "a row without keys is still written");
  must(kv4_cost(kv4_seq(0, 0, 90, 10, 3, 5, 4, 16, true), 8) == 0, "a sequence without rows costs nothing");
  must(kv4_counts_fit(1 << 20, 8, 8, 64, 1 << 15, 6, 128), "large launches fit");
  must(kv4_counts_fit(65536, 1024, 1, 1024, 1 << 14, 6, 128), "with a thousand heads to a kv head too");
  must(!kv4_counts_fit(0x7fffffff, 1024, 1, 65536, 0x3ffffff, 5, 16), "launches past 52 bits do not");
  for (long long d : {1ll, 3ll, 7ll, 1024ll, 32768ll, 1000003ll, (1ll << 40) + 1})
    for (long long q : {0ll, 1ll, 2ll, 12345ll, (1ll << 52) / d - 2})
      for (long long r : {0ll, 1ll, d / 2, d - 1})
        if (q >= 0 && r < d && q * d + r < (1ll << 52)) must(kv4_div(q * d + r, d) == q, "division");
}

static void rules() {
  alignas(16) static unsigned char mem[64];
  int* ip = reinterpret_cast<int*>(mem);
  Kv4StepArgs s{};
  s.n_seq = 2; s.page_shift = 5; s.width = 4; s.n_pages = 9; s.max_rows = 3;
  s.lens = s.table = s.free_pages = s.n_free = s.starts = s.slots = s.positions = s.scratch = s.err = ip;
  must(!check_kv4_step(s), "a good step");
  auto step = [&](auto f, const char* why) { Kv4StepArgs x = s; f(x); must(says(check_kv4_step(x), why), why); };
  step([](Kv4StepArgs& x) { x.page_shift = 4; }, "page rows");
  step([](Kv4StepArgs& x) { x.page_shift = -1; }, "page rows");
  step([](Kv4StepArgs& x) { x.page_shift = 9; }, "page rows");
  step([](Kv4StepArgs& x) { x.n_pages = 0; }, "pool pages");
  step([](Kv4StepArgs& x) { x.n_pages = 1 << 26; }, "pool pages");
  step([](Kv4StepArgs& x) { x.n_seq = 0; }, "sequences");
  step([](Kv4StepArgs& x) { x.n_seq = 65537; }, "sequences");
  step([](Kv4StepArgs& x) { x.width = 0; }, "width");
  step([](Kv4StepArgs& x) { x.width = 1 << 26; }, "width");
  step([](Kv4StepArgs& x) { x.max_rows = -1; }, "negative");
  step([](Kv4StepArgs& x) { x.lens = nullptr; }, "null");
  step([](Kv4StepArgs& x) { x.scratch = nullptr; }, "null");
  step([](Kv4StepArgs& x) { x.slots = nullptr; }, "null slot map");
  Kv4StepArgs none = s;
  none.max_rows = 0;
  none.slots = none.positions = nullptr;
  must(!check_kv4_step(none), "no slot map is needed for no rows");

  Kv4RowsArgs r{};
  r.k = r.v = r.ok = r.ov = mem; r.dtype = 1; r.rows = 4; r.n_kv = 8; r.page_shift = 6; r.n_pages = 3;
  r.slots = r.err = ip; r.pool = mem; r.k_row = r.v_row = 1024; r.k_head = r.v_head = 128;
  must(!check_kv4_rows(r, true) && !check_kv4_rows(r, false), "good rows");
  auto row = [&](auto f, const char* why) { Kv4RowsArgs x = r; f(x); must(says(check_kv4_rows(x, true), why), why); };
  row([](Kv4RowsArgs& x) { x.dtype = 3; }, "dtype");
  row([](Kv4RowsArgs& x) { x.rows = -1; }, "negative");
  row([](Kv4RowsArgs& x) { x.n_kv = 0; }, "kv heads");
  row([](Kv4RowsArgs& x) { x.n_kv = 1024; x.n_pages = 0x1ffffff; }, "pool pages");
  row([](Kv4RowsArgs& x) { x.k_row = 1028; }, "strides");
  row([](Kv4RowsArgs& x) { x.v_head = 4; }, "strides");
  row([](Kv4RowsArgs& x) { x.k = mem + 8; }, "aligned");
  row([](Kv4RowsArgs& x) { x.pool = mem + 1; }, "aligned");
  row([](Kv4RowsArgs& x) { x.v = nullptr; }, "null rows");
  row([](Kv4RowsArgs& x) { x.slots = nullptr; }, "null");

  Kv4AttnArgs a{};
  a.q = a.out = mem; a.q_row = 4096; a.q_head = 128; a.dtype = 2; a.n_rows = 3; a.n_heads = 32; a.n_kv = 8;
  a.n_seq = 2; a.scale_log2 = 0.1f; a.starts = a.lens = a.table = a.err = ip; a.width = 4; a.page_shift = 5;
  a.n_pages = 9; a.pool = mem; a.ws = reinterpret_cast<float*>(mem);
  must(!check_kv4_attn(a), "a good attention");
  auto att = [&](auto f, const char* why) { Kv4AttnArgs x = a; f(x); must(says(check_kv4_attn(x), why), why); };
  att([](Kv4AttnArgs& x) { x.dtype = 0; }, "dtype");
  att([](Kv4AttnArgs& x) { x.n_heads = 33; }, "multiple");
  att([](Kv4AttnArgs& x) { x.n_heads = 0; }, "multiple");
  att([](Kv4AttnArgs& x) { x.n_kv = 1; x.n_heads = 1025; }, "1024");
  att([](Kv4AttnArgs& x) { x.n_rows = 1 << 27; }, "too many");
  att([](Kv4AttnArgs& x) { x.n_rows = -1; }, "negative");
  att([](Kv4AttnArgs& x) { x.n_seq = 0; }, "sequences");
  att([](Kv4AttnArgs& x) { x.scale_log2 = 0.f; }, "scale");
  att([](Kv4AttnArgs& x) { x.scale_log2 = -1.f; }, "scale");
  att([](Kv4AttnArgs& x) { x.scale_log2 = __builtin_nanf(""); }, "scale");
  att([](Kv4AttnArgs& x) { x.scale_log2 = __builtin_inff(); }, "scale");
  att([](Kv4AttnArgs& x) { x.q_head = 132; }, "strides");
  att([](Kv4AttnArgs& x) { x.out = nullptr; }, "null");
  att([](Kv4AttnArgs& x) { x.q = mem + 2; }, "aligned");
}

int main() {
  layout();
  asks();
  seqs();
  for (int workers : {1, 3, 256, 768})
    for (int rows : {16, 32, 128})
      for (bool causal : {false, true}) {
        split({1}, {1}, 32, 8, rows, workers, causal);
        split({1}, {33000}, 32, 8, rows, workers, causal);
        split({32, 0, 7, 1, 300}, {500, 90, 0, 1, 4097}, 40, 8, rows, workers, causal);
        split({1, 1, 1, 1, 1, 1, 1}, {511, 512, 513, 16, 100000, 3, 2000}, 5, 1, rows, workers, causal);
        split({700, 64, 5}, {700, 3000, 2}, 21, 3, rows, workers, causal);
        split({333}, {90}, 2, 2, rows, workers, causal);
      }
  rules();
  std::printf("ok\n");
  return 0;
}
