// Sums and searches over the sequences of a step, shared by its two forms.
#pragma once

#include "dfl_common.h"

namespace dfl {

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

// The last of the ascending n numbers at (n > 0, at[0] <= v) that is not above v, of equals the last.
DFL_DEV int step_search(const int* at, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= v) lo = mid; else hi = mid;
  }
  return lo;
}
// The same for i, i + n, .. (those below `past`) in the n_seq ascending numbers at `at`, N of them at
// once, so that the searches do not wait for each other.
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
}  // namespace dfl
