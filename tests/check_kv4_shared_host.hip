// Host program: what a step of sequences that share pages asks of each, its scratch, the workspace of an
// attention with shared keys and how it is cut, the argument rules; the cut of a verification.
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "dfl_kv4.h"
#include "dfl_verify.h"

using namespace dfl;

static void must(bool ok, const char* what) {
  if (!ok) {
    std::printf("failed: %s\n", what);
    std::exit(1);
  }
}
static bool says(const char* e, const char* what) { return e && std::strstr(e, what); }

static void asks() {
  Kv4ForkAsk a;
  // itself: 100 rows, 40 kept, 50 more, pages of 32
  must(kv4_fork_ask(3, 3, 100, 100, 40, 50, 4, 5, a) && a.old == 4 && a.counted == 2 && a.placed == 2, "itself");
  // from a sequence of 200 rows: the 4 old places are looked at, of 6 kept
  must(kv4_fork_ask(3, 1, 200, 100, 170, 10, 8, 5, a) && a.old == 4 && a.counted == 6 && a.placed == 6, "from another");
  must(kv4_fork_ask(3, 1, 200, 250, 30, 0, 8, 5, a) && a.counted == 8 && a.placed == 8, "fewer than before");
  must(kv4_fork_ask(0, 0, 0, 0, 0, 0, 1, 5, a) && a.counted == 0 && a.placed == 0, "nothing");
  must(kv4_fork_ask(0, 0, 32, 32, 32, 1, 2, 5, a) && a.counted == 0 && a.placed == 1, "a new page");
  const int bad[][6] = {{-1, 10, 10, 0, 0, 0}, {0, 10, 10, 11, 0, 0}, {0, 10, 10, -1, 0, 0}, {0, 10, 10, 5, -1, 0},
                        {0, 10, 10, 5, 124, 0}, {0, -1, 10, 0, 0, 0}, {0, 10, -1, 0, 0, 0}, {0, 129, 10, 0, 0, 0},
                        {0, 10, 129, 0, 0, 0}, {0, 10, 10, 5, 0x7fffffff, 0}};
  for (const auto& t : bad)
    must(!kv4_fork_ask(2, t[0], t[1], t[2], t[3], t[4], 4, 5, a) && a.counted == 0 && a.placed == 0 && a.grow == 0 &&
             a.parent == 2, "a length out of range");
  must(kv4_fork_chunks(1) == 1 && kv4_fork_chunks(1024) == 1 && kv4_fork_chunks(1025) == 2 &&
           kv4_fork_chunks(0x7fffffff) == 2097152, "chunks");
  must(kv4_fork_scratch(10, 7, 100, true) - kv4_fork_scratch(10, 7, 100, false) == 70, "kept pages");
  must(kv4_fork_scratch(65536, 8191, 1, true) > 65536ll * 8191, "scratch past 32 bits of bytes");
}

static void cuts() {
  for (int rows : {1, 5, 64, 4096})
    for (int seqs : {1, 3, 64, 1000})
      for (int groups : {1, 2, 64})
        for (int heads : {1, 8, 64}) {
          if (groups > seqs) continue;
          const Kv4SharedCut c = kv4_shared_cut(rows, heads, 1, seqs, groups);
          const Kv4SharedWs w = kv4_shared_ws(rows, heads, 1, seqs, groups);
          const Kv4Cut d = kv4_cut(rows, heads, 1, seqs);
          if (!c.own) {
            must(d.tile_rows != 16 && w.bytes == kv4_ws_bytes(d.tile_rows, d.workers), "apart");
            continue;
          }
          must(d.tile_rows == 16 && (c.shared_workers ? c.own == 16 && c.shared == 128 : c.own == c.shared), "tiles");
          must(c.workers % 8 == 0 && c.shared_workers % 8 == 0, "workers by die");
          const long long at[] = {w.own, w.shared, w.state_o, w.state_ml, w.recs, w.row_of, w.q0, w.q1, w.len, w.skip, w.seq_of};
          for (long long p : at) must(p % 16 == 0, "aligned");
          const long long orows = (long long)rows * heads, all = seqs + groups;
          must(c.shared_workers ? w.shared - w.own >= kv4_ws_bytes(16, c.workers) &&
                                      w.state_o - w.shared >= kv4_ws_bytes(128, c.shared_workers)
                                : w.shared == w.own && w.state_o - w.own >= kv4_ws_bytes(c.own, c.workers), "partials");
          must(w.state_ml - w.state_o >= 2 * orows * 512 && w.recs - w.state_ml >= 2 * orows * 8 &&
                   w.row_of - w.recs >= 2 * orows * 16 && w.q0 - w.row_of >= 8 * all && w.q1 - w.q0 >= 4 * all &&
                   w.len - w.q1 >= 4 * all && w.skip - w.len >= 4 * all && w.seq_of - w.skip >= 4ll * seqs &&
                   w.bytes - w.seq_of >= 4ll * rows, "parts do not overlap");
        }
}

static void verify_cuts() {
  VerifyArgs a{};
  for (int rows : {1, 16, 2048, 1 << 20})
    for (int vocab : {1, 7, 4096, 4097, 151936, VF_MAX_VOCAB})
      for (int dt : {0, 1, 2})
        for (bool draft : {false, true}) {
          a.n_rows = rows;
          a.n_seq = rows < 64 ? rows : 64;
          a.vocab = vocab;
          a.target_dtype = dt;
          a.draft = draft ? &a : nullptr;
          a.draft_dtype = 2 - dt;
          vf_cut(a);
          const long long round = VF_THREADS * VF_VECS;
          must(a.t_chunks >= 1 && (long long)a.t_chunks * a.t_rounds * round * vf_elems(dt) >= vocab, "a row's parts hold it");
          must((long long)(a.t_chunks - 1) * a.t_rounds * round * vf_elems(dt) < vocab, "no part is empty");
          must(draft ? (long long)a.d_chunks * a.d_rounds * round * vf_elems(2 - dt) >= vocab : a.d_chunks == 0, "the draft's");
          must((long long)a.draw_chunks * VF_DRAW >= vocab, "the draw's");
          const VfWs w = vf_ws(a);
          must(w.draws - w.parts >= (long long)rows * (a.t_chunks + a.d_chunks) * 16 &&
                   w.sums - w.draws >= a.n_seq * (long long)sizeof(VfDraw) &&
                   w.states - w.sums >= 24ll * a.n_seq * a.draw_chunks && w.bytes - w.states >= 4ll * rows &&
                   w.draws % 16 == 0 && w.sums % 16 == 0 && w.states % 16 == 0, "the workspace");
        }
}

static void rules() {
  alignas(16) static unsigned char mem[64];
  int* ip = reinterpret_cast<int*>(mem);
  Kv4ForkArgs f{};
  f.n_seq = 4; f.page_shift = 5; f.width = 8; f.n_pages = 9; f.max_rows = 3; f.n_kv = 2; f.n_layers = 3;
  f.lens = f.table = f.refs = f.n_free = f.starts = f.slots = f.positions = f.scratch = f.err = ip;
  f.pool = mem;
  f.layer_bytes = 9 * 2 * KV4_BLOCK;
  must(!check_kv4_fork(f), "a good step");
  auto fork = [&](auto g, const char* why) { Kv4ForkArgs x = f; g(x); must(says(check_kv4_fork(x), why), why); };
  fork([](Kv4ForkArgs& x) { x.page_shift = 4; }, "page rows");
  fork([](Kv4ForkArgs& x) { x.n_pages = 0; }, "pool pages");
  fork([](Kv4ForkArgs& x) { x.n_kv = 0; }, "kv heads");
  fork([](Kv4ForkArgs& x) { x.n_seq = 0; }, "sequences");
  fork([](Kv4ForkArgs& x) { x.n_seq = 65537; }, "sequences");
  fork([](Kv4ForkArgs& x) { x.width = 0; }, "width");
  fork([](Kv4ForkArgs& x) { x.n_seq = 65536; x.width = 8192; }, "2^29");
  fork([](Kv4ForkArgs& x) { x.n_layers = 0; }, "layers");
  fork([](Kv4ForkArgs& x) { x.layer_bytes -= 16; }, "bytes");
  fork([](Kv4ForkArgs& x) { x.layer_bytes += 8; }, "bytes");
  fork([](Kv4ForkArgs& x) { x.max_rows = -1; }, "negative");
  fork([](Kv4ForkArgs& x) { x.refs = nullptr; }, "null");
  fork([](Kv4ForkArgs& x) { x.pool = nullptr; }, "null");
  fork([](Kv4ForkArgs& x) { x.slots = nullptr; }, "null slot map");
  fork([](Kv4ForkArgs& x) { x.pool = mem + 4; }, "aligned");
}

int main() {
  asks();
  cuts();
  verify_cuts();
  rules();
  std::printf("ok\n");
  return 0;
}
