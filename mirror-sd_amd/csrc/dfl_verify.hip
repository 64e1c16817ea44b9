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
// in 64 bits and takes the sequence's first rejected row.  That sum is off by less than 2^-16: a
// test that such an error could turn is made again with sums in 64 bits.  A draw has no such slack, as
// some token's running sum almost always lies within 2^-20 of any number: it is made in 64 bits
// throughout, over the one row of a sequence that needs it.
//
// Bound by HBM: the logits are read once, the row that is drawn from two or three times more.
#include "dfl_verify.h"

#include <float.h>

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
// Temperature of a sequence: log2(e) / T, 0 for the largest logit alone.
DFL_DEV double scale_of(const float* temps, float temp, int s) {
  const float t = temps ? temps[s] : temp;
  return t >= GREEDY ? LOG2E / (double)fminf(t, 1e30f) : 0.0;
}
// 2^x to the last bits: the series of 2^f around a whole number, |f| <= 1/2, to f^13 (the next term
// is below 2^-57).  A third of the library's code; 0 for -infinity, NaN for NaN.
DFL_DEV double pow2_64(double x) {
  x = x < -1100.0 ? -1100.0 : x;
  const double k = __builtin_rint(x), f = x - k;
  double p = 1.3691488853904128e-12;
  p = __builtin_fma(p, f, 2.5678435993488206e-11);
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

// ---- first pass: parts of rows
//
// A thread has VECS loads of 16 bytes, all under way together; a wave has its own reference.
template <int DT, int VECS>
DFL_DEV void part_of_row(const VerifyArgs& a, const void* base, long long stride, int row, int chunk,
                         double scale, VfPart& out, float (&lds)[2][4]) {
  typedef typename LogitT<DT>::t E;
  constexpr int N = DT == 0 ? 4 : 8;
  typedef E vec __attribute__((ext_vector_type(N)));
  const E* p = reinterpret_cast<const E*>(base) + row * stride;
  const int pad = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(E));
  const int e0 = chunk * (VF_THREADS * VECS * N) - pad + N * threadIdx.x;   // this thread's first value
  vec x[VECS];
  if (chunk > 0 && (chunk + 1) * (VF_THREADS * VECS * N) - pad <= a.vocab) {
#pragma unroll
    for (int j = 0; j < VECS; ++j)
      x[j] = __builtin_nontemporal_load(reinterpret_cast<const vec*>(p + e0 + j * (VF_THREADS * N)));
  } else {
#pragma unroll
    for (int j = 0; j < VECS; ++j) {
      const int e = e0 + j * (VF_THREADS * N);
      if (e >= 0 && e + N <= a.vocab) {
        x[j] = *reinterpret_cast<const vec*>(p + e);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[j][i] = e + i >= 0 && e + i < a.vocab ? p[e + i] : (E)-INFINITY;
      }
    }
  }
  const int wv = threadIdx.x >> 6;
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < VECS; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, (float)x[j][i]);
  if (scale == 0.0) {   // the largest and its first place
    bool bad = false;
    int at = INT32_MAX;
    top = wave_max(top);
#pragma unroll
    for (int j = VECS - 1; j >= 0; --j)
#pragma unroll
      for (int i = N - 1; i >= 0; --i) {
        const float v = (float)x[j][i];
        bad |= !(v < INFINITY);
        if (v == top) at = e0 + j * (VF_THREADS * N) + i;
      }
#pragma unroll
    for (int o = 32; o; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
    at = __ballot(bad) ? -1 : max(at, 0);   // (of a wave without values it is no place)
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      lds[0][wv] = top;
      lds[1][wv] = __int_as_float(at);
    }
    __syncthreads();
    out = VfPart{-INFINITY, 0.f, 0.0};
    for (int w = 0; w < 4; ++w) {
      const int i = __float_as_int(lds[1][w]);
      if (i < 0) out.sum = __builtin_nan("");
      const float m = lds[0][w];
      if (m > out.top || (m == out.top && i < out.sum)) {
        out.top = m;
        if (out.sum == out.sum) out.sum = i;
      }
    }
    return;
  }
  top = wave_max(top);
  const float c = scale_hi(scale), d = (float)(scale - (double)c), ref = top * c;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (__builtin_expect(is_moderate(ref), 1)) {
#pragma unroll
    for (int j = 0; j < VECS; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float v = (float)x[j][i];
        sum[i & 3] += __builtin_amdgcn_exp2f(__builtin_fmaf(v, d, __builtin_fmaf(v, c, -ref)));
      }
  } else {   // nothing but -infinity, or large logits
    const float both = (float)scale;
#pragma unroll
    for (int j = 0; j < VECS; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float v = (float)x[j][i];
        sum[i & 3] += v == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((v - top) * both);
      }
  }
  const float s = wave_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    lds[0][wv] = top;
    lds[1][wv] = s;
  }
  __syncthreads();
  out = VfPart{lds[0][0], 0.f, 0.0};
  for (int w = 1; w < 4; ++w) out.top = fmaxf(out.top, lds[0][w]);
  for (int w = 0; w < 4; ++w) out.sum += moved_sum(lds[1][w], lds[0][w], out.top, scale);
}

template <int VECS>
__global__ __launch_bounds__(VF_THREADS) void verify_parts_kernel(VerifyArgs a, VfPart* parts) {
  __shared__ float lds[2][4];
  const uint32_t t_items = (uint32_t)a.n_rows * a.t_chunks, items = t_items + (uint32_t)a.n_rows * a.d_chunks;
  for (uint32_t i = blockIdx.x; i < items; i += gridDim.x) {   // (below 2^31, as the grid)
    const bool drafted = i >= t_items;
    const uint32_t chunks = drafted ? a.d_chunks : a.t_chunks, k = drafted ? i - t_items : i;
    const int row = (int)(k / chunks), chunk = (int)(k - row * chunks);
    const int s = seq_of(a, row);
    if (s < 0 || (drafted && a.starts[s] == row)) continue;   // (a first row has no draft)
    const double scale = drafted ? scale_of(a.draft_temps, a.draft_temp, s) : scale_of(a.temps, a.temp, s);
    const void* base = drafted ? a.draft : a.target;
    const long long stride = drafted ? a.draft_row : a.target_row;
    const int dt = drafted ? a.draft_dtype : a.target_dtype;
    VfPart out;
    if (dt == 0) part_of_row<0, VECS>(a, base, stride, row, chunk, scale, out, lds);
    else if (dt == 1) part_of_row<1, VECS>(a, base, stride, row, chunk, scale, out, lds);
    else part_of_row<2, VECS>(a, base, stride, row, chunk, scale, out, lds);
    if (threadIdx.x == 0) parts[i] = out;
  }
}

// ---- the judge
//
// A workgroup to a sequence, a wave to a row.

// Two parts joined (in the order of their places).
DFL_DEV VfPart join(const VfPart& x, const VfPart& y, double scale) {
  if (scale == 0.0) {
    if (!(x.sum == x.sum) || !(y.sum == y.sum)) return VfPart{fmaxf(x.top, y.top), 0.f, __builtin_nan("")};
    return y.top > x.top || (y.top == x.top && y.sum < x.sum) ? y : x;
  }
  const float top = fmaxf(x.top, y.top);
  return VfPart{top, 0.f, moved_sum(x.sum, x.top, top, scale) + moved_sum(y.sum, y.top, top, scale)};
}
// The parts of a row joined, by a wave: what VfPart is, of the whole row.
DFL_DEV VfPart join_parts(const VfPart* parts, int chunks, double scale) {
  const int lane = threadIdx.x & 63;
  VfPart r{-INFINITY, 0.f, 0.0};
  for (int i = lane; i < chunks; i += 64) r = join(r, parts[i], scale);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const VfPart x{__shfl_xor(r.top, o, 64), 0.f, __shfl_xor(r.sum, o, 64)};
    r = lane & o ? join(x, r, scale) : join(r, x, scale);   // (the same in both of a pair)
  }
  return r;
}
DFL_DEV bool has_distribution(const VfPart& r, bool greedy) {
  return greedy ? r.sum == r.sum && r.top > -INFINITY : r.sum > 0.0 && r.sum < INFINITY;
}
// The probability of a token (any lane alone).
DFL_DEV double chance_of(const void* base, int dtype, long long stride, int vocab, int row, int x,
                         double scale, const VfPart& r) {
  if (x < 0 || x >= vocab) return 0.0;
  if (scale == 0.0) return (double)x == r.sum ? 1.0 : 0.0;
  return pow2_64(((double)logit_at(base, dtype, row * stride + x) - r.top) * scale + offset_of(r.top, scale)) / r.sum;
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
  if (scale == 0.0 || x < 0 || x >= vocab) return chance_of(base, dtype, stride, vocab, row, x, scale, r);
  double v = 0.0;
  for (int i = threadIdx.x; i < vocab; i += blockDim.x)
    v += pow2_64(((double)logit_at(base, dtype, row * stride + i) - r.top) * scale);
  return pow2_64(((double)logit_at(base, dtype, row * stride + x) - r.top) * scale) / block_sum64(v, lds);
}

constexpr int JUDGE = 1024;
enum { ROW_YES = 0, ROW_NO = 1, ROW_CLOSE = 2 };
// What the first pass's sums (each off by 2^-16 at most: exponents of at most 40 that matter, each
// rounded twice, 2^-17.6, the power's 2^-22, a thread's additions 2^-18) can change in a quotient.
constexpr double VF_CLOSE = 0x1p-14;

__global__ __launch_bounds__(JUDGE) void verify_judge_kernel(VerifyArgs a, const VfPart* parts, VfDraw* draws,
                                                             int* states) {
  __shared__ double lds[JUDGE / 64];
  __shared__ int found;
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
  auto target = [&](int row) { return join_parts(parts + (long long)row * a.t_chunks, a.t_chunks, pc); };
  auto drafted = [&](int row) { return join_parts(d_parts + (long long)row * a.d_chunks, a.d_chunks, qc); };
  auto p_of = [&](int row, int x, const VfPart& r) {
    return chance_of(a.target, a.target_dtype, a.target_row, a.vocab, row, x, pc, r);
  };
  auto q_of = [&](int row, int x, const VfPart& r) {
    return chance_of(a.draft, a.draft_dtype, a.draft_row, a.vocab, row, x, qc, r);
  };
  for (int row = q0 + wv; row < q1; row += JUDGE / 64) {
    int state = ROW_YES;
    double chance = 1.0;
    if (row > q0) {
      const int x = a.ids[row];
      const VfPart pr = target(row - 1), qr = a.draft ? drafted(row) : VfPart{0.f, 0.f, (double)x};
      if (!has_distribution(pr, pc == 0.0) || (a.draft && !has_distribution(qr, qc == 0.0))) {
        state = ROW_NO;
        chance = 0.0;
      } else {
        const double p = p_of(row - 1, x, pr), q = a.draft ? q_of(row, x, qr) : 1.0;
        const double u = a.uniforms[row];
        chance = p > 0.0 ? fmin(1.0, p / fmax(q, 1e-300)) : 0.0;
        state = u * q < p ? ROW_YES : ROW_NO;
        if ((pc != 0.0 || qc != 0.0) && fabs(u * q - p) <= VF_CLOSE * p && p > 0.0) state = ROW_CLOSE;
      }
    }
    if (lane == 0) {
      a.chances[row] = (float)chance;
      states[row] = state;
    }
  }
  int stop = q0;   // the first rejected row, or the end
  while (true) {
    __syncthreads();
    if (threadIdx.x == 0) found = q1;
    __syncthreads();
    for (int row = stop + threadIdx.x; row < q1; row += JUDGE)
      if (states[row] != ROW_YES) {
        atomicMin(&found, row);
        break;
      }
    __syncthreads();
    stop = found;
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
// Parts of VF_DRAW tokens, 8 in a row to a thread, in 64 bits.

DFL_DEV void weights8(const void* base, int dtype, long long stride, int vocab, int row, int i0, double scale,
                      float top, double (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    w[i] = i0 + i < vocab ? pow2_64(((double)logit_at(base, dtype, row * stride + i0 + i) - top) * scale) : 0.0;
}
DFL_DEV void p_weights(const VerifyArgs& a, const VfDraw& d, int i0, double (&w)[8]) {
  weights8(a.target, a.target_dtype, a.target_row, a.vocab, d.row, i0, d.pc, d.p_top, w);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i0 + i == d.not_this) w[i] = 0.0;
}
DFL_DEV void q_weights(const VerifyArgs& a, const VfDraw& d, int i0, double (&w)[8]) {
  weights8(a.draft, a.draft_dtype, a.draft_row, a.vocab, d.draft, i0, d.qc, d.q_top, w);
}
DFL_DEV double sum8(const double (&w)[8]) {
  double v = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) v += w[i];
  return v;
}
// Sums of p's and q's weights.
__global__ __launch_bounds__(VF_THREADS) void verify_sums_kernel(VerifyArgs a, const VfDraw* draws, double* sums) {
  __shared__ double lds[4];
  const long long all = (long long)a.n_seq * a.draw_chunks;
  for (long long i = blockIdx.x; i < all; i += gridDim.x) {
    const int s = (int)(i / a.draw_chunks), chunk = (int)(i - (long long)s * a.draw_chunks);
    const VfDraw d = draws[s];
    if (!d.kind) continue;
    const int i0 = chunk * VF_DRAW + 8 * threadIdx.x;
    double w[8];
    p_weights(a, d, i0, w);
    const double p = block_sum64(sum8(w), lds);
    if (threadIdx.x == 0) sums[i] = p;
    if (d.kind == 2) {
      q_weights(a, d, i0, w);
      const double q = block_sum64(sum8(w), lds);
      if (threadIdx.x == 0) sums[all + i] = q;
    }
  }
}
DFL_DEV double sum_of(const double* at, int n, double* lds) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) v += at[i];
  return block_sum64(v, lds);
}
// max(p - q, 0)
DFL_DEV void left_weights(const VerifyArgs& a, const VfDraw& d, int i0, double zp, double zq, double (&w)[8]) {
  double q[8];
  p_weights(a, d, i0, w);
  q_weights(a, d, i0, q);
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = fmax(w[i] / zp - q[i] / zq, 0.0);
}
__global__ __launch_bounds__(VF_THREADS) void verify_left_kernel(VerifyArgs a, const VfDraw* draws, double* sums) {
  __shared__ double lds[4];
  const long long all = (long long)a.n_seq * a.draw_chunks;
  for (long long i = blockIdx.x; i < all; i += gridDim.x) {
    const int s = (int)(i / a.draw_chunks), chunk = (int)(i - (long long)s * a.draw_chunks);
    const VfDraw d = draws[s];
    if (d.kind != 2) continue;
    const double zp = sum_of(sums + i - chunk, a.draw_chunks, lds);
    const double zq = sum_of(sums + all + i - chunk, a.draw_chunks, lds);
    double w[8];
    left_weights(a, d, chunk * VF_DRAW + 8 * threadIdx.x, zp, zq, w);
    const double r = block_sum64(sum8(w), lds);
    if (threadIdx.x == 0) sums[2 * all + i] = r;
  }
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
  __shared__ double lds[4];
  __shared__ int first, last;
  const int s = blockIdx.x;
  VfDraw d = draws[s];
  if (!d.kind) return;
  const long long all = (long long)a.n_seq * a.draw_chunks, at = (long long)s * a.draw_chunks;
  double zp = 1.0, zq = 1.0;
  const double* parts = sums + at;
  if (d.kind == 2) {
    zp = sum_of(parts, a.draw_chunks, lds);
    zq = sum_of(sums + all + at, a.draw_chunks, lds);
    parts = sums + 2 * all + at;
  }
  double whole = sum_of(parts, a.draw_chunks, lds);
  if (!(whole > 0.0)) {
    if (d.kind == 1) {   // all of p's weight is on the token that is left out
      if (threadIdx.x == 0) a.next_ids[s] = d.not_this;
      return;
    }
    d.kind = 1;          // p and q are the same
    parts = sums + at;
    whole = zp;
  }
  const double v = (double)a.uniforms[a.starts[s]] * whole;
  // the part in which the running sum exceeds v (the last that has any weight if none does)
  if (threadIdx.x == 0) {
    first = INT32_MAX;
    last = 0;
  }
  double done = 0.0, before = 0.0;
  int mine = -1;
  for (int c0 = 0; c0 < a.draw_chunks; c0 += VF_THREADS) {
    const int c = c0 + threadIdx.x;
    const double x = c < a.draw_chunks ? parts[c] : 0.0;
    double some;
    const double b = done + block_before64(x, lds, some);
    if (x > 0.0) {
      if (b + x > v) atomicMin(&first, c);
      atomicMax(&last, c);
    }
    done += some;
    __syncthreads();
    const int hit = first;
    if (hit != INT32_MAX) {
      if (c == hit) {
        mine = c;
        before = b;
      }
      break;
    }
  }
  __syncthreads();
  const int chunk = first != INT32_MAX ? first : last;
  const bool past = first == INT32_MAX;
  if (mine >= 0) lds[0] = before;
  __syncthreads();
  const double rest = past ? INFINITY : v - lds[0];
  __syncthreads();
  if (threadIdx.x == 0) {
    first = INT32_MAX;
    last = 0;
  }
  const int i0 = chunk * VF_DRAW + 8 * threadIdx.x;
  double w[8], some;
  if (d.kind == 2) left_weights(a, d, i0, zp, zq, w);
  else p_weights(a, d, i0, w);
  double sum = block_before64(sum8(w), lds, some);
  int hit = INT32_MAX, any = -1;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    sum += w[i];
    if (w[i] > 0.0) {
      if (hit == INT32_MAX && sum > rest) hit = i0 + i;
      any = i0 + i;
    }
  }
  if (hit != INT32_MAX) atomicMin(&first, hit);
  if (any >= 0) atomicMax(&last, any);
  __syncthreads();
  if (threadIdx.x == 0) a.next_ids[s] = first != INT32_MAX ? first : last;
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
    if (a.vecs == 2) hipLaunchKernelGGL((verify_parts_kernel<2>), grid, block, 0, st, a, parts);
    else hipLaunchKernelGGL((verify_parts_kernel<8>), grid, block, 0, st, a, parts);
  }
  hipLaunchKernelGGL(verify_judge_kernel, dim3(a.n_seq), dim3(JUDGE), 0, st, a, (const VfPart*)parts, draws, states);
  if (a.n_rows == 0) return;
  const long long draws_n = (long long)a.n_seq * a.draw_chunks;
  const dim3 dgrid((unsigned)(draws_n < (1 << 20) ? draws_n : 1 << 20));
  hipLaunchKernelGGL(verify_sums_kernel, dgrid, block, 0, st, a, (const VfDraw*)draws, sums);
  if (a.draft) hipLaunchKernelGGL(verify_left_kernel, dgrid, block, 0, st, a, (const VfDraw*)draws, sums);
  hipLaunchKernelGGL(verify_draw_kernel, dim3(a.n_seq), block, 0, st, a, (const VfDraw*)draws, (const double*)sums);
}

}  // namespace dfl
