// Verification of drafted blocks (dfl_verify.h): which drafted tokens the target's distributions
// accept, by given uniform numbers, and the token that follows them.
//
// With p the softmax of a target row over its temperature and q the draft's, row t's token x is
// accepted if u q(x) < p(x), p of row t - 1: with the chance min(1, p / q).  The first rejected row
// has its token drawn anew from max(p - q, 0), which makes every token a draw from p; behind a block
// that is accepted whole one more is drawn from p.  A draw is the first token whose running sum
// exceeds u times the whole.
//
// First pass (all rows): the sum of exponentials of parts of a row, in fp32; the judge joins them
// in 64 bits and takes the sequence's first rejected row.  That sum is off by 2^-15.9 at most: a
// test that such an error could turn is made again with sums in 64 bits.  A draw has no such slack, as
// some token's running sum almost always lies within 2^-20 of any number: it is made in 64 bits
// throughout, over the one row of a sequence that needs it.
//
// Bound by HBM: the logits are read once, the row that is drawn from two or three times more.
#include "dfl_verify.h"

#include "dfl_common.h"

namespace dfl {

namespace {

typedef __bf16 bf16_t;

constexpr double LOG2E = 1.44269504088896340736;
constexpr float GREEDY = 1e-5f;   // temperatures below are those of the largest logit alone

template <int DT> struct LogitT;
template <> struct LogitT<0> { typedef float t; };
template <> struct LogitT<1> { typedef half_t t; };
template <> struct LogitT<2> { typedef bf16_t t; };

DFL_DEV float logit_at(const void* base, int dtype, long long at) {
  if (dtype == 0) return reinterpret_cast<const float*>(base)[at];
  if (dtype == 1) return (float)reinterpret_cast<const half_t*>(base)[at];
  return (float)reinterpret_cast<const bf16_t*>(base)[at];
}
// Temperature of a sequence: log2(e) / T, 0 for the largest logit alone, -1 for a number on the device that
// is no temperature (negative, infinite, NaN): no part of the sequence's rows is then summed, so that they
// have no distribution.
DFL_DEV double scale_of(const float* temps, float temp, int s) {
  const float t = temps ? temps[s] : temp;
  if (!(t >= 0.f && t < INFINITY)) return -1.0;
  return t >= GREEDY ? LOG2E / (double)fminf(t, 1e30f) : 0.0;
}
// 2^x: the series of 2^f around a whole number, |f| <= 1/2, to f^12 (the next term is below 2^-52 of
// it), half of the library's code.  0 for -infinity; any number for NaN.
DFL_DEV double pow2_64(double x) {
  x = fmax(x, -2000.0);
  const double k = __builtin_rint(x), f = x - k;
  double p = 2.5678435993488206e-11;
  p = __builtin_fma(p, f, 4.4455382718708116e-10);
  p = __builtin_fma(p, f, 7.054911620801123e-09);
  p = __builtin_fma(p, f, 1.01780860092397e-07);
  p = __builtin_fma(p, f, 1.321548679014431e-06);
  p = __builtin_fma(p, f, 1.5252733804059841e-05);
  p = __builtin_fma(p, f, 0.0001540353039338161);
  p = __builtin_fma(p, f, 0.0013333558146428443);
  p = __builtin_fma(p, f, 0.009618129107628477);
  p = __builtin_fma(p, f, 0.05550410866482158);
  p = __builtin_fma(p, f, 0.24022650695910072);
  p = __builtin_fma(p, f, 0.6931471805599453);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)k);
}
// The scale log2(e) / T is taken as c + d in two parts, d > 0, so that a logit of -infinity stays one
// in both steps of an exponent.
DFL_DEV float scale_hi(double scale) { return __uint_as_float(__float_as_uint((float)scale) - 1u); }
// Exponents in 32 bits are relative to the largest logit's, rounded as it may be: fl(c top).  This is
// how far that is below top log2(e) / T: the weight of a logit x is 2^((x - top) log2(e) / T + it).
// (Past 2^16 the rounding is too much; there differences of logits are taken first.)
DFL_DEV bool is_moderate(float ref) { return fabsf(ref) < 0x1p16f; }
DFL_DEV double offset_of(float top, double scale) {
  const float r = top * scale_hi(scale);
  return is_moderate(r) ? __builtin_fma((double)top, scale, -(double)r) : 0.0;
}
// The sequence of a row, by all lanes of a wave: the last that begins at or before it; -1 if the
// row is none's.
DFL_DEV int seq_of(const VerifyArgs& a, int row) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = a.n_seq;
  while (n > 1) {
    const int step = (n + 63) >> 6, i = lane * step;
    const bool begun = i < n && a.starts[lo + i] <= row;
    const int k = max(0, (int)__popcll(__ballot(begun)) - 1) * step;   // (the count is unsigned)
    lo += k;
    n = min(step, n - k);
  }
  return a.starts[lo] <= row && row < a.starts[lo + 1] ? lo : -1;
}

// A sum of weights relative to `top`, made one relative to `to` >= top.
DFL_DEV double moved_sum(double sum, float top, float to, double scale) {
  return sum == 0.0 || top == to ? sum : sum * pow2_64(((double)top - to) * scale + (offset_of(to, scale) - offset_of(top, scale)));
}

// Two parts joined (in the order of their places).
DFL_DEV VfPart join(const VfPart& x, const VfPart& y, double scale) {
  if (scale == 0.0) {
    if (!(x.sum == x.sum) || !(y.sum == y.sum)) return VfPart{fmaxf(x.top, y.top), 0.f, __builtin_nan("")};
    return y.top > x.top || (y.top == x.top && y.sum < x.sum) ? y : x;
  }
  const float top = fmaxf(x.top, y.top);
  return VfPart{top, 0.f, moved_sum(x.sum, x.top, top, scale) + moved_sum(y.sum, y.top, top, scale)};
}
// ---- first pass: parts of rows
//
// A workgroup goes over its part of a row in rounds of VF_VECS loads of 16 bytes a thread; the next
// round's loads are on their way while this one's exponentials are made.  Bound by HBM where there is
// enough to read (1.2 GB in bf16: 186 us, 6.6 TB/s; 65 MB 16, 4 TB/s), else by the begin and end of the
// workgroups.  With all of a part's loads at once and two barriers' sums for each 32 KiB the 1.2 GB
// took 293 us.

template <int DT> struct Vec {
  typedef typename LogitT<DT>::t E;
  static constexpr int N = DT == 0 ? 4 : 8;   // values of 16 bytes
  typedef E vec __attribute__((ext_vector_type(N)));
};
// Vectors v, v + VF_THREADS, .. of a row's `n`; -infinity past the last.
template <int DT>
DFL_DEV void load_round(const typename Vec<DT>::vec* p, int v, int n, bool inside, typename Vec<DT>::vec (&x)[VF_VECS]) {
  if (inside) {
#pragma unroll
    for (int j = 0; j < VF_VECS; ++j) x[j] = __builtin_nontemporal_load(p + v + j * VF_THREADS);
    return;
  }
#pragma unroll
  for (int j = 0; j < VF_VECS; ++j) {
#pragma unroll
    for (int i = 0; i < Vec<DT>::N; ++i) x[j][i] = (typename Vec<DT>::E)-INFINITY;
    if (v + j * VF_THREADS < n) x[j] = p[v + j * VF_THREADS];
  }
}
// The weights' sum of a wave's part, relative to a logit that is raised to the largest so far when
// that is more than twice its weight.
struct SoftState {
  float top, at, ref;   // this lane's largest; the logit that weights are relative to, and fl(c at)
  float sum[4];
};
template <int VECS, int N, typename V>
DFL_DEV void soft_round(const V (&x)[VECS], SoftState& s, float c, float d, double scale) {
  float top = s.top;
#pragma unroll
  for (int j = 0; j < VECS; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, (float)x[j][i]);
  s.top = top;
  if (!__all(is_moderate(s.ref) ? top * c <= s.ref + 1.f : top <= s.at)) {
    const float to = wave_max(top);
    if (to > s.at) {
      if (s.at > -INFINITY) {
        const float k = (float)moved_sum(1.0, s.at, to, scale);
#pragma unroll
        for (int i = 0; i < 4; ++i) s.sum[i] *= k;
      }
      s.at = to;
      s.ref = to * c;
    }
  }
  if (__builtin_expect(is_moderate(s.ref), 1)) {
#pragma unroll
    for (int j = 0; j < VECS; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float v = (float)x[j][i];
        s.sum[i & 3] += __builtin_amdgcn_exp2f(__builtin_fmaf(v, d, __builtin_fmaf(v, c, -s.ref)));
      }
  } else {   // nothing but -infinity so far, or large logits
    const float both = (float)scale;
#pragma unroll
    for (int j = 0; j < VECS; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float v = (float)x[j][i];
        s.sum[i & 3] += v == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((v - s.at) * both);
      }
  }
}
// (scale_at: the row's log2(e) / T, found while the first loads are on their way; below 0: the row is not
// wanted, or has no temperature)
template <int DT, typename F>
DFL_DEV VfPart part_of_row(const VerifyArgs& a, const void* base, long long stride, int row, int chunk, int rounds,
                           F scale_at, float (&lds)[2][4]) {
  typedef Vec<DT> V;
  constexpr int ROUND = VF_THREADS * VF_VECS;   // vectors
  const typename V::E* p = reinterpret_cast<const typename V::E*>(base) + row * stride;
  // whole vectors of the row, and the values before and behind them (the first part takes those)
  const int head = min(a.vocab, (int)(-(reinterpret_cast<uintptr_t>(p) / sizeof(typename V::E)) & (V::N - 1)));
  const int n = (a.vocab - head) / V::N, tail = head + n * V::N;
  const typename V::vec* body = reinterpret_cast<const typename V::vec*>(p + head);
  const int begin = chunk * rounds * ROUND, end = min(begin + rounds * ROUND, n);
  const int tid = threadIdx.x, wv = threadIdx.x >> 6;
  auto inside = [&](int v) { return v + ROUND <= n; };
  // (threads 0 .. 7: the values before; 8 .. 15: those behind)
  const int edge = tid < V::N ? tid : tail + tid - V::N;
  const bool at_edge = chunk == 0 && (tid < V::N ? tid < head : edge < a.vocab && tid < 2 * V::N);
  typename V::vec x[VF_VECS], y[VF_VECS];
  load_round<DT>(body, begin + tid, n, inside(begin), x);
  const float extra = at_edge ? (float)p[edge] : -INFINITY;
  const double scale = scale_at();
  VfPart out{-INFINITY, 0.f, 0.0};
  if (scale < 0.0) return out;
  if (scale == 0.0) {   // the largest and its first place
    bool bad = false;
    float top = -INFINITY;
    int at = INT32_MAX;
    auto take = [&](float v, int place) {
      bad |= !(v < INFINITY);
      if (v > top) {
        top = v;
        at = place;
      }
    };
    if (tid < V::N) take(extra, edge);
    for (int v = begin; v < end; v += ROUND) {
      if (v + ROUND < end) load_round<DT>(body, v + ROUND + tid, n, inside(v + ROUND), y);
#pragma unroll
      for (int j = 0; j < VF_VECS; ++j)
#pragma unroll
        for (int i = 0; i < V::N; ++i)
          take((float)x[j][i], head + (v + tid + j * VF_THREADS) * V::N + i);
#pragma unroll
      for (int j = 0; j < VF_VECS; ++j) x[j] = y[j];
    }
    if (tid >= V::N) take(extra, edge);
    const float of_wave = wave_max(top);
    if (top != of_wave) at = INT32_MAX;
#pragma unroll
    for (int o = 32; o; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
    if (__ballot(bad)) at = -1;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      lds[0][wv] = of_wave;
      lds[1][wv] = __int_as_float(at);
    }
    __syncthreads();
    for (int w = 0; w < 4; ++w) {
      const int i = __float_as_int(lds[1][w]);
      out = join(out, VfPart{lds[0][w], 0.f, i < 0 ? __builtin_nan("") : (double)i}, 0.0);
    }
    return out;
  }
  const float c = scale_hi(scale), d = (float)(scale - (double)c);
  SoftState s{-INFINITY, -INFINITY, -INFINITY, {0.f, 0.f, 0.f, 0.f}};
  if (chunk == 0 && n * V::N < a.vocab) {
    const floatx2 one[1] = {{extra, extra}};
    soft_round<1, 1>(one, s, c, d, scale);
  }
  for (int v = begin; v < end; v += ROUND) {
    if (v + ROUND < end) load_round<DT>(body, v + ROUND + tid, n, inside(v + ROUND), y);
    soft_round<VF_VECS, V::N>(x, s, c, d, scale);
#pragma unroll
    for (int j = 0; j < VF_VECS; ++j) x[j] = y[j];
  }
  const float top = wave_max(s.top), sum = wave_sum((s.sum[0] + s.sum[1]) + (s.sum[2] + s.sum[3]));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    lds[0][wv] = top;
    lds[1][wv] = top == s.at ? sum : (float)moved_sum(sum, s.at, top, scale);
  }
  __syncthreads();
  for (int w = 0; w < 4; ++w) out.top = fmaxf(out.top, lds[0][w]);
  for (int w = 0; w < 4; ++w) out.sum += moved_sum(lds[1][w], lds[0][w], out.top, scale);
  return out;
}

__global__ __launch_bounds__(VF_THREADS) void verify_parts_kernel(VerifyArgs a, VfPart* parts) {
  __shared__ float lds[2][4];
  const uint32_t t_items = (uint32_t)a.n_rows * a.t_chunks, items = t_items + (uint32_t)a.n_rows * a.d_chunks;
  for (uint32_t i = blockIdx.x; i < items; i += gridDim.x) {   // (below 2^31, as the grid)
    const bool drafted = i >= t_items;
    const uint32_t chunks = drafted ? a.d_chunks : a.t_chunks, k = drafted ? i - t_items : i;
    const int row = (int)(k / chunks), chunk = (int)(k - row * chunks);
    auto scale = [&]() {
      const int s = seq_of(a, row);
      if (s < 0 || (drafted && a.starts[s] == row)) return -1.0;   // (a first row has no draft)
      return drafted ? scale_of(a.draft_temps, a.draft_temp, s) : scale_of(a.temps, a.temp, s);
    };
    const void* base = drafted ? a.draft : a.target;
    const long long stride = drafted ? a.draft_row : a.target_row;
    const int dt = drafted ? a.draft_dtype : a.target_dtype, rounds = drafted ? a.d_rounds : a.t_rounds;
    VfPart out;
    if (dt == 0) out = part_of_row<0>(a, base, stride, row, chunk, rounds, scale, lds);
    else if (dt == 1) out = part_of_row<1>(a, base, stride, row, chunk, rounds, scale, lds);
    else out = part_of_row<2>(a, base, stride, row, chunk, rounds, scale, lds);
    if (threadIdx.x == 0) parts[i] = out;
  }
}

// ---- the judge
//
// A workgroup to a sequence, a wave to a row.  Bound by latencies: starts, temperatures and parts, the
// tokens' logits, the states; 7.5 us for rows of 16, 12 for 64 sequences of 32.

// The parts of a row joined, by a wave: what VfPart is, of the whole row.
DFL_DEV VfPart own_part(const VfPart* parts, int chunks) {   // (a lane's first, for join_parts)
  const int lane = threadIdx.x & 63;
  return lane < chunks ? parts[lane] : VfPart{-INFINITY, 0.f, 0.0};
}
DFL_DEV VfPart join_parts(const VfPart* parts, int chunks, double scale, VfPart r) {
  for (int i = (threadIdx.x & 63) + 64; i < chunks; i += 64) r = join(r, parts[i], scale);
  const float top = wave_max(r.top);
  if (scale == 0.0) {
    int at = r.top == top ? (int)r.sum : INT32_MAX;   // (of a NaN any)
#pragma unroll
    for (int o = 32; o; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
    return VfPart{top, 0.f, __ballot(!(r.sum == r.sum)) ? __builtin_nan("") : (double)at};
  }
  r.sum = moved_sum(r.sum, r.top, top, scale);
#pragma unroll
  for (int o = 32; o; o >>= 1) r.sum += __shfl_xor(r.sum, o, 64);
  return VfPart{top, 0.f, r.sum};
}
DFL_DEV bool has_distribution(const VfPart& r, bool greedy) {
  return greedy ? r.sum == r.sum && r.top > -INFINITY : r.sum > 0.0 && r.sum < INFINITY;
}
// The probability of token x, whose logit is l, in a row (x outside the vocabulary: 0).
DFL_DEV double chance_of(float l, int x, int vocab, double scale, const VfPart& r) {
  if (x < 0 || x >= vocab) return 0.0;
  if (scale == 0.0) return (double)x == r.sum ? 1.0 : 0.0;
  return pow2_64(((double)l - r.top) * scale + offset_of(r.top, scale)) / r.sum;
}
// Sum over the workgroup's threads in 64 bits, the same in all.
DFL_DEV double block_sum64(double v, double* lds /* 16 */) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) v += lds[w];
  return v;
}
// The probability of a token with the sum in 64 bits, by the whole workgroup.
DFL_DEV double chance64(const void* base, int dtype, long long stride, int vocab, int row, int x, double scale,
                        const VfPart& r, double* lds) {
  if (scale == 0.0 || x < 0 || x >= vocab) return chance_of(0.f, x, vocab, scale, r);
  double v = 0.0;
  for (int i = threadIdx.x; i < vocab; i += blockDim.x)
    v += pow2_64(((double)logit_at(base, dtype, row * stride + i) - r.top) * scale);
  return pow2_64(((double)logit_at(base, dtype, row * stride + x) - r.top) * scale) / block_sum64(v, lds);
}

constexpr int JUDGE = 1024, JUDGE_KEPT = 64;
enum { ROW_YES = 0, ROW_NO = 1, ROW_CLOSE = 2 };
// What the first pass's sums can change in a test.  Exponents down to -40 matter (smaller weights add
// up to V 2^-40), rounded twice (three times past 2^16): 2^-24 40 ln 2 each time, 5.0e-6 in all; the
// power is off by 2^-23, a thread's sum by 128 additions, 7.6e-6, and at most 40 rescalings, 2.4e-6,
// the wave's by 8 more, 5e-7: 1.6e-5, 2^-15.9, of p's sum and of q's.
constexpr double VF_CLOSE = 0x1p-14;

__global__ __launch_bounds__(JUDGE) void verify_judge_kernel(VerifyArgs a, const VfPart* parts, VfDraw* draws,
                                                             int* states) {
  __shared__ double lds[JUDGE / 64];
  __shared__ VfPart p_kept[JUDGE_KEPT], q_kept[JUDGE_KEPT];   // of the sequence's first rows
  const int s = blockIdx.x, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int q0 = a.starts[s], q1 = a.starts[s + 1];
  VfDraw draw{};
  if (q0 < 0 || q1 <= q0 || q1 > a.n_rows) {
    if (threadIdx.x == 0) {
      a.accepted[s] = 0;
      a.next_ids[s] = -1;
      draws[s] = draw;
    }
    return;
  }
  const double pc = scale_of(a.temps, a.temp, s), qc = a.draft ? scale_of(a.draft_temps, a.draft_temp, s) : 0.0;
  const VfPart* d_parts = parts + (long long)a.n_rows * a.t_chunks;
  auto t_at = [&](int row) { return parts + (long long)row * a.t_chunks; };
  auto d_at = [&](int row) { return d_parts + (long long)row * a.d_chunks; };
  auto target = [&](int row) {
    return row - q0 < JUDGE_KEPT ? p_kept[row - q0] : join_parts(t_at(row), a.t_chunks, pc, own_part(t_at(row), a.t_chunks));
  };
  auto drafted = [&](int row) {
    return row - q0 < JUDGE_KEPT ? q_kept[row - q0] : join_parts(d_at(row), a.d_chunks, qc, own_part(d_at(row), a.d_chunks));
  };
  for (int row = q0 + wv; row < q1; row += JUDGE / 64) {
    // (the first row has no test: its wave joins the last one's target, which no test needs)
    const int before = row > q0 ? row - 1 : q1 - 1;
    const bool with_draft = a.draft && row > q0;
    // loads that do not wait for each other, then those of the token's logits
    VfPart pr = own_part(t_at(before), a.t_chunks), qr{0.f, 0.f, 0.0};
    if (with_draft) qr = own_part(d_at(row), a.d_chunks);
    const int x = a.ids[row];
    const double u = a.uniforms[row];
    const bool in = x >= 0 && x < a.vocab;
    const float pl = in ? logit_at(a.target, a.target_dtype, before * a.target_row + x) : 0.f;
    const float ql = in && with_draft ? logit_at(a.draft, a.draft_dtype, row * a.draft_row + x) : 0.f;
    pr = join_parts(t_at(before), a.t_chunks, pc, pr);
    if (with_draft) qr = join_parts(d_at(row), a.d_chunks, qc, qr);
    int state = ROW_YES;
    double chance = 1.0;
    if (row > q0) {
      if (!has_distribution(pr, pc == 0.0) || (a.draft && !has_distribution(qr, qc == 0.0))) {
        state = ROW_NO;
        chance = 0.0;
      } else {
        const double p = chance_of(pl, x, a.vocab, pc, pr), q = a.draft ? chance_of(ql, x, a.vocab, qc, qr) : 1.0;
        chance = p > 0.0 ? fmin(1.0, p / fmax(q, 1e-300)) : 0.0;
        state = u * q < p ? ROW_YES : ROW_NO;
        if ((pc != 0.0 || qc != 0.0) && fabs(u * q - p) <= VF_CLOSE * p && p > 0.0) state = ROW_CLOSE;
      }
    }
    if (lane == 0) {
      a.chances[row] = (float)chance;
      states[row] = state;
      if (before - q0 < JUDGE_KEPT) p_kept[before - q0] = pr;
      if (row - q0 < JUDGE_KEPT) q_kept[row - q0] = qr;
    }
  }
  int stop = q0 + 1;   // the first rejected row, or the end (the first row has no test)
  __syncthreads();
  while (true) {
    while (stop < q1) {   // (every wave the same, 64 rows at a time)
      const int row = stop + lane;
      const unsigned long long no = __ballot(row < q1 && states[row] != ROW_YES);
      stop = no ? stop + __ffsll(no) - 1 : min(stop + 64, q1);
      if (no) break;
    }
    if (stop >= q1 || states[stop] == ROW_NO) break;
    // too close for the sums in 32 bits
    const int x = a.ids[stop];
    const double p = chance64(a.target, a.target_dtype, a.target_row, a.vocab, stop - 1, x, pc, target(stop - 1), lds);
    const double q = a.draft ? chance64(a.draft, a.draft_dtype, a.draft_row, a.vocab, stop, x, qc, drafted(stop), lds) : 1.0;
    if (!((double)a.uniforms[stop] * q < p)) break;
    ++stop;
  }
  if (wv) return;
  const int last = stop - 1;
  const bool some = stop < q1;
  const VfPart pr = target(last);
  draw.row = last;
  draw.draft = stop;
  draw.u = a.uniforms[q0];
  draw.not_this = -1;
  draw.pc = pc;
  draw.qc = qc;
  draw.p_top = pr.top;
  bool ok = has_distribution(pr, pc == 0.0);
  draw.kind = 1;
  if (some && !a.draft) draw.not_this = a.ids[stop];
  if (some && a.draft) {
    const VfPart qr = drafted(stop);
    ok = ok && has_distribution(qr, qc == 0.0);
    if (qc == 0.0) draw.not_this = (int)qr.sum;
    else draw.kind = 2;
    draw.q_top = qr.top;
  }
  if (!ok || pc == 0.0) draw.kind = 0;   // (what is left of all weight on one token is that token)
  if (lane == 0) {
    a.accepted[s] = last - q0;
    a.next_ids[s] = ok && pc == 0.0 ? (int)pr.sum : -1;
    draws[s] = draw;
  }
}

// ---- the draw
//
// Parts of VF_DRAW tokens, 8 in a row to a thread, in 64 bits: sums of p's and q's weights, sums of what is
// left, then the part and the token.  Three launches, as each needs all sums of the one before; 4 to 5 us
// each where latency counts.

// The 16 powers of 2^(1/16), which the draw's kernels keep in LDS.
__constant__ const double kRoots[16] = {
    1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916,
    1.189207115002721, 1.241857812073484, 1.2968395546510096, 1.3542555469368927,
    1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543,
    1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474,
};
typedef double Roots[16];
DFL_DEV void load_roots(Roots& lds) {
  if (threadIdx.x < 16) lds[threadIdx.x] = kRoots[threadIdx.x];
  __syncthreads();
}
// 2^(y / 16): the series around a whole number of y, to the 6th power (the next term is below 2^-50 of
// it), times a root.  What bounds the draw's kernels is their 64-bit instructions: the sums of 64 rows of
// 151936 take 23 us with this, 25 with pow2_64, 48 ragged sequences 42 and 46 in all.
DFL_DEV double pow2_16(double y, const Roots& roots) {
  y = fmax(y, -32000.0);
  const double k = __builtin_rint(y), f = y - k;
  const int n = (int)k;
  double p = 9.181219573844438e-12;
  p = __builtin_fma(p, f, 1.2715871950558131e-09);
  p = __builtin_fma(p, f, 1.467610032291943e-07);
  p = __builtin_fma(p, f, 1.3550807779497457e-05);
  p = __builtin_fma(p, f, 0.0009383847928089872);
  p = __builtin_fma(p, f, 0.04332169878499658);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_ldexp(p * roots[n & 15], n >> 4);
}

// Logits i0 .. i0 + 7 of a row (-infinity past its end).  Rows may begin at any value's address; the
// card loads 16 bytes from those too.
template <typename E>
DFL_DEV void logits8(const E* p, int vocab, int i0, float (&x)[8]) {
  constexpr int N = 16 / sizeof(E);
  typedef E vec __attribute__((ext_vector_type(N), aligned(sizeof(E))));
  if (i0 + 8 <= vocab) {
#pragma unroll
    for (int j = 0; j < 8 / N; ++j) {
      const vec v = reinterpret_cast<const vec*>(p + i0)[j];
#pragma unroll
      for (int i = 0; i < N; ++i) x[N * j + i] = (float)v[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i0 + i < vocab ? (float)p[i0 + i] : -INFINITY;
  }
}
DFL_DEV void weights8(const void* base, int dtype, long long stride, int vocab, int row, int i0, double scale,
                      float top, const Roots& roots, double (&w)[8]) {
  float x[8];
  if (dtype == 0) logits8(reinterpret_cast<const float*>(base) + row * stride, vocab, i0, x);
  else if (dtype == 1) logits8(reinterpret_cast<const half_t*>(base) + row * stride, vocab, i0, x);
  else logits8(reinterpret_cast<const bf16_t*>(base) + row * stride, vocab, i0, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pow2_16(((double)x[i] - top) * (16.0 * scale), roots);
}
DFL_DEV void p_weights(const VerifyArgs& a, const VfDraw& d, int i0, const Roots& roots, double (&w)[8]) {
  weights8(a.target, a.target_dtype, a.target_row, a.vocab, d.row, i0, d.pc, d.p_top, roots, w);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i0 + i == d.not_this) w[i] = 0.0;
}
DFL_DEV void q_weights(const VerifyArgs& a, const VfDraw& d, int i0, const Roots& roots, double (&w)[8]) {
  weights8(a.draft, a.draft_dtype, a.draft_row, a.vocab, d.draft, i0, d.qc, d.q_top, roots, w);
}
DFL_DEV double sum8(const double (&w)[8]) {
  double v = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) v += w[i];
  return v;
}
// Sums of p's and q's weights.
__global__ __launch_bounds__(VF_THREADS) void verify_sums_kernel(VerifyArgs a, const VfDraw* draws, double* sums) {
  __shared__ Roots roots;
  load_roots(roots);
  __shared__ double lds[4];
  const long long all = (long long)a.n_seq * a.draw_chunks;
  for (long long i = blockIdx.x; i < all; i += gridDim.x) {
    const int s = (int)(i / a.draw_chunks), chunk = (int)(i - (long long)s * a.draw_chunks);
    const VfDraw d = draws[s];
    if (!d.kind) continue;
    const int i0 = chunk * VF_DRAW + 8 * threadIdx.x;
    double w[8];
    p_weights(a, d, i0, roots, w);
    const double p = block_sum64(sum8(w), lds);
    if (threadIdx.x == 0) sums[i] = p;
    if (d.kind == 2) {
      q_weights(a, d, i0, roots, w);
      const double q = block_sum64(sum8(w), lds);
      if (threadIdx.x == 0) sums[all + i] = q;
    }
  }
}
DFL_DEV void sums_of(const double* x, const double* y, int n, double (*lds)[2], double& sx, double& sy) {
  sx = sy = 0.0;
  for (int i = threadIdx.x; i < n; i += VF_THREADS) {
    sx += x[i];
    sy += y[i];
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    sx += __shfl_xor(sx, o, 64);
    sy += __shfl_xor(sy, o, 64);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    lds[threadIdx.x >> 6][0] = sx;
    lds[threadIdx.x >> 6][1] = sy;
  }
  __syncthreads();
  sx = sy = 0.0;
  for (int w = 0; w < VF_THREADS / 64; ++w) {
    sx += lds[w][0];
    sy += lds[w][1];
  }
}
// max(p - q, 0) times the sum of p's weights; ratio: that over the sum of q's.
DFL_DEV void left_weights(const VerifyArgs& a, const VfDraw& d, int i0, double ratio, const Roots& roots, double (&w)[8]) {
  double q[8];
  p_weights(a, d, i0, roots, w);
  q_weights(a, d, i0, roots, q);
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = fmax(w[i] - q[i] * ratio, 0.0);
}
__global__ __launch_bounds__(VF_THREADS) void verify_left_kernel(VerifyArgs a, VfDraw* draws, double* sums) {
  __shared__ Roots roots;
  load_roots(roots);
  __shared__ double lds[4][2];
  const long long all = (long long)a.n_seq * a.draw_chunks;
  for (long long i = blockIdx.x; i < all; i += gridDim.x) {
    const int s = (int)(i / a.draw_chunks), chunk = (int)(i - (long long)s * a.draw_chunks);
    const VfDraw d = draws[s];   // (but its ratio)
    if (d.kind != 2) continue;
    double zp, zq;
    sums_of(sums + i - chunk, sums + all + i - chunk, a.draw_chunks, lds, zp, zq);
    double w[8];
    left_weights(a, d, chunk * VF_DRAW + 8 * threadIdx.x, zp / zq, roots, w);
    const double r = block_sum64(sum8(w), lds[0]);
    if (threadIdx.x == 0) {
      sums[2 * all + i] = r;
      if (chunk == 0) draws[s].ratio = zp / zq;
    }
  }
}
// The first thread of the workgroup for which `hit`, and the last for which `any`; -1: there is none.
struct Ends { int first, last; };
DFL_DEV Ends block_ends(bool hit, bool any, Ends* lds /* 4 */) {
  const unsigned long long h = __ballot(hit), y = __ballot(any);
  const int wv = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
    lds[wv] = Ends{h ? 64 * wv + __ffsll(h) - 1 : -1, y ? 64 * wv + 63 - __clzll((long long)y) : -1};
  __syncthreads();
  Ends e{-1, -1};
  for (int w = 0; w < VF_THREADS / 64; ++w) {
    if (e.first < 0) e.first = lds[w].first;
    e.last = max(e.last, lds[w].last);
  }
  return e;
}
// Sum over the threads before this one, and the whole.
DFL_DEV double block_before64(double v, double* lds /* 4 */, double& all) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  double in = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double x = __shfl_up(in, o, 64);
    if (lane >= o) in += x;
  }
  double before = __shfl_up(in, 1, 64);
  if (lane == 0) before = 0.0;
  __syncthreads();
  if (lane == 63) lds[wv] = in;
  __syncthreads();
  all = 0.0;
  for (int w = 0; w < VF_THREADS / 64; ++w) {
    if (w < wv) before += lds[w];
    all += lds[w];
  }
  return before;
}
__global__ __launch_bounds__(VF_THREADS) void verify_draw_kernel(VerifyArgs a, const VfDraw* draws, const double* sums) {
  __shared__ Roots roots;
  load_roots(roots);
  __shared__ double lds[4];
  __shared__ Ends ends[4];
  const int s = blockIdx.x, n = a.draw_chunks;
  const long long all = (long long)a.n_seq * n;
  const double* p_sums = sums + (long long)s * n;
  // (loaded before it is known which are wanted: they do not wait for each other)
  const int mine = min((int)threadIdx.x, n - 1);
  const double x_p = p_sums[mine], x_left = a.draft ? p_sums[2 * all + mine] : 0.0;
  VfDraw d = draws[s];
  if (!d.kind) return;
  const double* parts = d.kind == 2 ? p_sums + 2 * all : p_sums;
  double whole = 0.0;
  // running sums of the parts, VF_THREADS at a time (a vocabulary of half a million: once)
  double x = 0.0, b = 0.0;
  auto scan = [&](int c0) {
    const int c = c0 + (int)threadIdx.x;
    x = c >= n ? 0.0 : c0 ? parts[c] : d.kind == 2 ? x_left : x_p;
    double some;
    b = block_before64(x, lds, some);
    return some;
  };
  for (int c0 = 0; c0 < n; c0 += VF_THREADS) whole += scan(c0);
  if (!(whole > 0.0)) {
    if (d.kind == 1) {   // all of p's weight is on the token that is left out
      if (threadIdx.x == 0) a.next_ids[s] = d.not_this;
      return;
    }
    d.kind = 1;          // p and q are the same
    parts = p_sums;
    whole = 0.0;
    for (int c0 = 0; c0 < n; c0 += VF_THREADS) whole += scan(c0);
  }
  const double v = (double)d.u * whole;
  // the part in which the running sum exceeds v (the last that has any weight if none does)
  int chunk = -1, last = 0;
  double done = 0.0;
  for (int c0 = 0; c0 < n && chunk < 0; c0 += VF_THREADS) {
    double some = 0.0;
    if (n > VF_THREADS) some = scan(c0);
    const Ends e = block_ends(x > 0.0 && done + b + x > v, x > 0.0, ends);
    if (e.first >= 0) {
      chunk = c0 + e.first;
      if ((int)threadIdx.x == e.first) lds[0] = done + b;
    }
    if (e.last >= 0) last = c0 + e.last;
    done += some;
  }
  __syncthreads();
  const double rest = chunk < 0 ? INFINITY : v - lds[0];
  if (chunk < 0) chunk = last;
  const int i0 = chunk * VF_DRAW + 8 * threadIdx.x;
  double w[8], some;
  if (d.kind == 2) left_weights(a, d, i0, d.ratio, roots, w);
  else p_weights(a, d, i0, roots, w);
  double sum = block_before64(sum8(w), lds, some);
  int hit = -1, any = -1;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    sum += w[i];
    if (w[i] > 0.0) {
      if (hit < 0 && sum > rest) hit = i0 + i;
      any = i0 + i;
    }
  }
  const Ends e = block_ends(hit >= 0, any >= 0, ends);
  const int thread = e.first >= 0 ? e.first : max(e.last, 0);
  if ((int)threadIdx.x == thread) a.next_ids[s] = e.first >= 0 ? hit : any;
}

}  // namespace

void launch_verify(const VerifyArgs& a_in, hipStream_t st) {
  VerifyArgs a = a_in;
  vf_cut(a);
  const VfWs w = vf_ws(a);
  char* ws = static_cast<char*>(a.ws);
  VfPart* parts = reinterpret_cast<VfPart*>(ws + w.parts);
  VfDraw* draws = reinterpret_cast<VfDraw*>(ws + w.draws);
  double* sums = reinterpret_cast<double*>(ws + w.sums);
  int* states = reinterpret_cast<int*>(ws + w.states);
  const long long items = (long long)a.n_rows * (a.t_chunks + a.d_chunks);
  const dim3 block(VF_THREADS), grid((unsigned)(items < (1 << 20) ? items : 1 << 20));
  if (items > 0) {
    hipLaunchKernelGGL(verify_parts_kernel, grid, block, 0, st, a, parts);
  }
  hipLaunchKernelGGL(verify_judge_kernel, dim3(a.n_seq), dim3(JUDGE), 0, st, a, (const VfPart*)parts, draws, states);
  if (a.n_rows == 0) return;
  const long long draws_n = (long long)a.n_seq * a.draw_chunks;
  const dim3 dgrid((unsigned)(draws_n < (1 << 20) ? draws_n : 1 << 20));
  hipLaunchKernelGGL(verify_sums_kernel, dgrid, block, 0, st, a, (const VfDraw*)draws, sums);
  if (a.draft) hipLaunchKernelGGL(verify_left_kernel, dgrid, block, 0, st, a, draws, sums);
  hipLaunchKernelGGL(verify_draw_kernel, dim3(a.n_seq), block, 0, st, a, (const VfDraw*)draws, (const double*)sums);
}

}  // namespace dfl
