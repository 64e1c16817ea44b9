// Verification of drafted blocks against the target's distributions: sizes, workspace, host checks.
// Everything here but the launcher is plain host code too, so that it can be tested on a CPU.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dfl {

struct VerifyArgs {
  const void *target, *draft;        // [n_rows][vocab] logits; draft may be null
  long long target_row, draft_row;   // row strides in elements
  int target_dtype, draft_dtype;     // 0 fp32, 1 fp16, 2 bf16
  int n_rows, vocab, n_seq;
  const int *ids, *starts;
  const float* uniforms;
  const float *temps, *draft_temps;  // [n_seq], or null: one for all
  float temp, draft_temp;
  int *accepted, *next_ids;
  float* chances;
  void* ws;
  // from here on set by the launcher
  int t_chunks, d_chunks;            // parts of a row in the first pass, for each matrix
  int t_rounds, d_rounds;            // rounds of a part
  int draw_chunks;                   // parts of a row in the draw
};

constexpr int VF_THREADS = 256;
constexpr int VF_VECS = 2;           // 16-byte loads of a thread and round
constexpr int VF_DRAW = 2048;        // values of a part in the draw: 8 a thread
constexpr int VF_MAX_VOCAB = 1 << 24, VF_MAX_ROWS = 1 << 24, VF_MAX_SEQS = 65536;

inline int vf_elems(int dtype) { return dtype == 0 ? 4 : 8; }   // values of 16 bytes
// Rounds of a row (one at least).
inline int vf_rounds(int vocab, int dtype) {
  const int round = VF_THREADS * vf_elems(dtype) * VF_VECS;
  return (vocab + round - 1) / round;
}
inline int vf_draw_chunks(int vocab) { return (vocab + VF_DRAW - 1) / VF_DRAW; }

// What the first pass leaves of a part of a row: its largest logit and, softmax, the sum of its
// weights relative to that one's (offset_of), greedy, the largest's first place.  A sum or
// place that is no number marks a row without a distribution.
struct VfPart { float top, pad; double sum; };
// What a sequence's draw needs.
struct VfDraw {
  int kind;          // 0: nothing to draw; 1: from p but for one token; 2: from max(p - q, 0)
  int row, draft;    // rows of target and draft
  int not_this;      // the token that is left out (-1: none)
  float p_top, q_top;   // the rows' largest logits
  float u, pad;
  double pc, qc;        // log2(e) / T
  double ratio;         // sum of p's weights over that of q's (kind 2)
};
struct VfWs { long long parts, draws, sums, states, bytes; };   // offsets
inline VfWs vf_ws(const VerifyArgs& a) {
  VfWs w{};
  long long at = 0;
  auto take = [&](long long n) { const long long p = at; at += (n + 15) / 16 * 16; return p; };
  w.parts = take((long long)a.n_rows * (a.t_chunks + a.d_chunks) * (long long)sizeof(VfPart));
  w.draws = take((long long)a.n_seq * (long long)sizeof(VfDraw));
  w.sums = take(3ll * a.n_seq * a.draw_chunks * 8);   // p, q, max(p - q, 0)
  w.states = take(4ll * a.n_rows);
  w.bytes = at;
  return w;
}
// How the call is cut: into parts of as many rounds as leave VF_PARTS of them, what the chip holds at
// once.  768, 1024, 1536 and 4096 parts, us: 8 blocks of 32 rows without a draft's logits 32, 32, 35, 51;
// 48 ragged ones of a vocabulary of 32003 41, 43, 43, 69; one block of 16 rows 30 with each.  (Rounds of
// 1, 2, 3 and 4 loads with 768: the blocks 33, 32, 31, 32, the ragged ones 44, 41, 41, 43, 64 blocks of 32
// rows 283, 259, 257, 257.)
constexpr int VF_PARTS = 768;
// At most so many values of a thread and part: each of its four sums then has 128 additions.
constexpr int VF_MOST = 512;
inline void vf_cut(VerifyArgs& a) {
  const int t = vf_rounds(a.vocab, a.target_dtype), d = a.draft ? vf_rounds(a.vocab, a.draft_dtype) : 0;
  const long long each = (long long)a.n_rows * (t + d) / VF_PARTS;
  auto cut = [&](int rounds, int dtype, int& per, int& chunks) {
    const int most = VF_MOST / (VF_VECS * vf_elems(dtype));
    per = each < 1 ? 1 : each < most ? (int)each : most;
    chunks = (rounds + per - 1) / per;
    per = chunks ? (rounds + chunks - 1) / chunks : 1;   // (parts alike)
    chunks = (rounds + per - 1) / per;
  };
  cut(t, a.target_dtype, a.t_rounds, a.t_chunks);
  cut(d, a.draft_dtype, a.d_rounds, a.d_chunks);
  a.draw_chunks = vf_draw_chunks(a.vocab);
}

inline const char* check_verify(const VerifyArgs& a) {
  if (a.n_rows < 0 || a.n_rows > VF_MAX_ROWS) return "rows outside [0, 2^24]";
  if (a.vocab < 1 || a.vocab > VF_MAX_VOCAB) return "vocabulary outside [1, 2^24]";
  if (a.n_seq < 1 || a.n_seq > VF_MAX_SEQS) return "sequences outside [1, 65536]";
  if (a.target_dtype < 0 || a.target_dtype > 2 || (a.draft && (a.draft_dtype < 0 || a.draft_dtype > 2)))
    return "dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)";
  VerifyArgs cut = a;
  vf_cut(cut);
  if ((long long)a.n_rows * (cut.t_chunks + cut.d_chunks) > 0x7fffffffll ||
      (long long)a.n_seq * cut.draw_chunks > 0x7fffffffll)
    return "too many rows for so large a vocabulary";
  if (!a.starts || !a.accepted || !a.next_ids) return "null pointer";
  if (a.n_rows > 0 && (!a.target || !a.ids || !a.uniforms || !a.chances)) return "null pointer";
  if (a.n_rows > 1 && (a.target_row < a.vocab || (a.draft && a.draft_row < a.vocab)))
    return "rows overlap (a row stride below the vocabulary)";
  auto mis = [](const void* p, int dtype) {
    return (reinterpret_cast<uintptr_t>(p) & (dtype ? 1 : 3)) != 0;
  };
  if (mis(a.target, a.target_dtype) || mis(a.draft, a.draft_dtype)) return "logits are not aligned to their type";
  auto number = [](float t) { return t >= 0.f && t <= 3.4028235e38f; };
  if (!a.temps && !number(a.temp)) return "temperature must be finite and not negative";
  if (a.draft && !a.draft_temps && !number(a.draft_temp))
    return "draft temperature must be finite and not negative";
  return nullptr;
}

void launch_verify(const VerifyArgs& a, hipStream_t st);

}  // namespace dfl
