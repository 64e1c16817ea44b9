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
// Phases, each over all sequences: scan (totals, then offsets), free, take, rows.  A phase reads
// what the one before wrote, so they are launches of their own, or for a few sequences one
// workgroup with barriers between them.

// Inclusive sums over the workgroup's threads of three counts at once.
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
    if (w < wv) { v.a += lds[w].a; v.b += lds[w].b; v.c += lds[w].c; }
    total.a += lds[w].a; total.b += lds[w].b; total.c += lds[w].c;
  }
  return v;
}

struct StepView { int *base, *f_at, *t_at; };
DFL_DEV StepView step_view(const Kv4StepArgs& a) {
  return StepView{a.scratch + 4, a.scratch + 4 + a.n_seq, a.scratch + 4 + 2 * a.n_seq};
}
DFL_DEV bool step_ask(const Kv4StepArgs& a, int s, Kv4Ask& q) {
  const int len = a.lens[s];
  return kv4_ask(len, a.keep ? a.keep[s] : len, a.grow ? a.grow[s] : 0, a.width, a.page_shift, q);
}

// One workgroup: status and totals into scratch[0 .. 3], offsets and starts; all or nothing.
DFL_DEV void step_scan(const Kv4StepArgs& a, Sum3* lds) {
  const int nt = blockDim.x;
  Sum3 all{0, 0, 0};
  int bad = 0;
  for (int s0 = 0; s0 < a.n_seq; s0 += nt) {
    const int s = s0 + threadIdx.x;
    Kv4Ask q{0, 0, 0, 0};
    if (s < a.n_seq && !step_ask(a, s, q)) bad = 1;
    Sum3 t;
    block_scan3(Sum3{q.freed, q.taken, q.grow}, lds, t);
    all.a += t.a; all.b += t.b; all.c += t.c;
  }
  bad = __syncthreads_or(bad);
  const int n_free = *a.n_free;
  int err = bad ? KV4_ERR_LEN : 0;
  // (freed pages beyond the pool, or a free count beyond it: the state is not a step's)
  if (n_free < 0 || n_free > a.n_pages || n_free + all.a > a.n_pages) err |= KV4_ERR_PAGE;
  else if (all.b > n_free + all.a) err |= KV4_ERR_POOL;
  if (all.c > a.max_rows) err |= KV4_ERR_ROWS;
  const StepView v = step_view(a);
  Sum3 at{0, 0, 0};
  for (int s0 = 0; s0 < a.n_seq; s0 += nt) {
    const int s = s0 + threadIdx.x;
    Kv4Ask q{0, 0, 0, 0};
    if (s < a.n_seq) step_ask(a, s, q);
    Sum3 t;
    const Sum3 in = block_scan3(Sum3{q.freed, q.taken, q.grow}, lds, t);
    if (s < a.n_seq) {
      v.base[s] = q.keep;
      v.f_at[s] = (int)(at.a + in.a - q.freed);
      v.t_at[s] = (int)(at.b + in.b - q.taken);
      a.starts[s] = err ? 0 : (int)(at.c + in.c - q.grow);
    }
    at.a += t.a; at.b += t.b; at.c += t.c;
  }
  if (threadIdx.x == 0) {
    a.starts[a.n_seq] = err ? 0 : (int)all.c;
    a.scratch[0] = err;
    a.scratch[1] = (int)all.a;
    a.scratch[2] = (int)all.b;
    a.scratch[3] = n_free;
    if (err) atomicOr(a.err, err);
  }
}
// Waves wave, wave + n_waves, ..: one sequence each.
DFL_DEV void step_free(const Kv4StepArgs& a, int wave, int n_waves) {
  if (a.scratch[0]) return;
  const int lane = threadIdx.x & 63;
  const int top = a.scratch[3] + a.scratch[1] - 1;
  const StepView v = step_view(a);
  for (int s = wave; s < a.n_seq; s += n_waves) {
    const int pk = kv4_pages(v.base[s], a.page_shift);
    const int n = kv4_pages(a.lens[s], a.page_shift) - pk;
    int* row = a.table + (long long)s * a.width + pk;
    for (int j = lane; j < n; j += 64) {
      const int p = row[j];
      if (p < 0 || p >= a.n_pages) atomicOr(a.err, KV4_ERR_PAGE);
      a.free_pages[top - (v.f_at[s] + j)] = p;
      row[j] = -1;
    }
  }
}
DFL_DEV void step_take(const Kv4StepArgs& a, int wave, int n_waves) {
  if (a.scratch[0]) return;
  const int lane = threadIdx.x & 63;
  const int top = a.scratch[3] + a.scratch[1] - 1;
  const StepView v = step_view(a);
  for (int s = wave; s < a.n_seq; s += n_waves) {
    const int keep = v.base[s], grow = a.starts[s + 1] - a.starts[s];
    const int pk = kv4_pages(keep, a.page_shift);
    const int n = kv4_pages(keep + grow, a.page_shift) - pk;
    int* row = a.table + (long long)s * a.width + pk;
    for (int j = lane; j < n; j += 64) {
      const int i = top - (v.t_at[s] + j);
      row[j] = a.free_pages[i];
      a.free_pages[i] = -1;
    }
    if (lane == 0) a.lens[s] = keep + grow;
  }
  if (wave == 0 && lane == 0) *a.n_free = a.scratch[3] + a.scratch[1] - a.scratch[2];
}
// Rows t, t + n, .. of the slot map; those past the step's rows get -1.
DFL_DEV void step_rows(const Kv4StepArgs& a, long long t, long long n) {
  const StepView v = step_view(a);
  const int total = a.starts[a.n_seq];
  for (long long r = t; r < a.max_rows; r += n) {
    int slot = -1, pos = -1;
    if (r < total) {
      int lo = 0, hi = a.n_seq;   // the last sequence that starts at or before r
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.starts[mid] <= r) lo = mid; else hi = mid;
      }
      pos = v.base[lo] + (int)(r - a.starts[lo]);
      const int pg = a.table[(long long)lo * a.width + (pos >> a.page_shift)];
      const int mask = (1 << a.page_shift) - 1;
      slot = pg < 0 || pg >= a.n_pages ? -1 : (pg << a.page_shift) + (pos & mask);
    }
    a.slots[r] = slot;
    a.positions[r] = pos;
  }
}

__global__ __launch_bounds__(1024) void kv4_step_scan_kernel(Kv4StepArgs a) {
  __shared__ Sum3 lds[16];
  step_scan(a, lds);
}
__global__ __launch_bounds__(256) void kv4_step_free_kernel(Kv4StepArgs a) {
  step_free(a, blockIdx.x * 4 + (threadIdx.x >> 6), gridDim.x * 4);
}
__global__ __launch_bounds__(256) void kv4_step_take_kernel(Kv4StepArgs a) {
  step_take(a, blockIdx.x * 4 + (threadIdx.x >> 6), gridDim.x * 4);
}
__global__ __launch_bounds__(256) void kv4_step_rows_kernel(Kv4StepArgs a) {
  step_rows(a, (long long)blockIdx.x * 256 + threadIdx.x, (long long)gridDim.x * 256);
}
__global__ __launch_bounds__(1024) void kv4_step_small_kernel(Kv4StepArgs a) {
  __shared__ Sum3 lds[16];
  step_scan(a, lds);
  __syncthreads();
  step_free(a, threadIdx.x >> 6, blockDim.x >> 6);
  __syncthreads();
  step_take(a, threadIdx.x >> 6, blockDim.x >> 6);
  __syncthreads();
  step_rows(a, threadIdx.x, blockDim.x);
}

// ------------------------------------------------------------------ rows in and out
//
// 16 threads to a row of one head, 8 values (one code word) each; a group is a quad of lanes.

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

// Where slot's row lies; false (and the error bit) for a slot outside the pool, -1 is no error.
DFL_DEV bool slot_at(const Kv4RowsArgs& a, int slot, int head, unsigned char*& blk, int& r) {
  if (slot < 0 || slot >= (a.n_pages << a.page_shift)) {
    if (slot != -1) atomicOr(a.err, KV4_ERR_SLOT);
    return false;
  }
  const int in = slot & ((1 << a.page_shift) - 1);
  blk = a.pool + kv4_block_at(slot >> a.page_shift, a.n_kv, head, 1 << (a.page_shift - 5), in >> 5);
  r = kv4_row(in & 31);
  return true;
}

template <int DT>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4RowsArgs a) {
  const long long n = (long long)a.rows * 2 * a.n_kv * 16;
  const long long step = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += step) {
    const int part = (int)i & 15;
    const long long item = i >> 4;
    const int head = (int)(item % a.n_kv);
    const long long rv = item / a.n_kv;
    const int v = (int)rv & 1;
    const long long row = rv >> 1;
    unsigned char* blk;
    int r;
    const bool ok = slot_at(a, a.slots[row], head, blk, r);   // (one answer for the quad's lanes)
    if (!ok) continue;
    float x[8];
    load8<DT>(v ? a.v : a.k, row * (v ? a.v_row : a.k_row) + head * (v ? a.v_head : a.k_head) + 8 * part, x);
    // |x| orders as its bits do; an infinity or a NaN is at or past 0x7f800000
    int top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, (int)(__float_as_uint(x[j]) & 0x7fffffffu));
    top = max(top, __shfl_xor(top, 1, 64));
    top = max(top, __shfl_xor(top, 2, 64));
    const bool bad = top >= 0x7f800000;
    const int b = bad ? 255 : max(0, (top >> 23) - 2 + ((top & 0x7fffff) > 0x600000 ? 1 : 0));
    const float s = __uint_as_float((uint32_t)b << 23);   // (the conversion reads the exponent alone)
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
    *reinterpret_cast<uint32_t*>(blk + v * KV4_V + r * 64 + part * 4) = bad ? 0u : w;
    if ((part & 3) == 0) blk[kv4_scale_at(r, part >> 2, v)] = (unsigned char)b;
  }
}

template <int DT>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4RowsArgs a) {
  const long long n = (long long)a.rows * 2 * a.n_kv * 16;
  const long long step = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += step) {
    const int part = (int)i & 15;
    const long long item = i >> 4;
    const int head = (int)(item % a.n_kv);
    const long long rv = item / a.n_kv;
    const int v = (int)rv & 1;
    const long long row = rv >> 1;
    unsigned char* blk;
    int r;
    uint32_t w = 0;
    float s = 1.f;
    if (slot_at(a, a.slots[row], head, blk, r)) {
      w = *reinterpret_cast<const uint32_t*>(blk + v * KV4_V + r * 64 + part * 4);
      s = __uint_as_float((uint32_t)blk[kv4_scale_at(r, part >> 2, v)] << 23);
    }
    typedef typename RowT<DT>::t E;
    E* out = reinterpret_cast<E*>(v ? a.ov : a.ok) + (row * a.n_kv + head) * KV4_D + 8 * part;
    if constexpr (DT == 0) {
      const floatx2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0);
      const floatx2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
      const floatx2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2);
      const floatx2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
      reinterpret_cast<floatx4*>(out)[0] = (floatx4){p0.x, p0.y, p1.x, p1.y};
      reinterpret_cast<floatx4*>(out)[1] = (floatx4){p2.x, p2.y, p3.x, p3.y};
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
      *reinterpret_cast<u32x4*>(out) = o;
    }
  }
}

// ------------------------------------------------------------------ attention
//
// O = softmax(scale * Q K^T) V over each sequence's cached rows, K and V in 4 bits.
//
// A unit is a tile of 16 NT query rows (row = token * ratio + head in group) of one sequence and
// kv head.  A workgroup takes a run of key blocks of a unit, its four waves every fourth block
// each, with a wave's whole work on a block in its own registers and its own 9 KiB of LDS (no
// barrier in the loop):
//   S^T = K Q^T   v_mfma 16x16x32, keys on the M axis, K converted from codes in registers (two
//                 values an instruction, their power of two applied by it: exact);
//   softmax       fp32, log2 domain, reference maximum raised only when a block exceeds it by
//                 more than KV4_SLACK; weights rounded to the type of Q, and summed as rounded;
//   O^T += V^T P  V converted in registers, written to LDS as rows, read back transposed
//                 (ds_read_b64_tr_b16); P from the S^T accumulators as they lie (kv4_row).
// The next block's codes load while this one computes.

constexpr float KV4_SLACK = 6.f;
// Weights are 2^(s - m + KV4_LIFT) <= 2^15 for a reference m: fp16 then keeps 2^-23 of the
// largest weight as a normal number and 2^-34 as the rounding of the smallest, so that a million
// keys far below one large one still add up.
constexpr float KV4_LIFT = 9.f;
constexpr int VROW = 288;                 // bytes of a V row in LDS: 8 banks apart, so that the 8
                                          // rows of a half wave's transposing read do not collide
constexpr int VWAVE = 32 * VROW;

template <typename T> struct Mat;
template <> struct Mat<half_t> {
  // Codes convert to half their value: a group whose largest fp16 value is above 3.5 * 2^14 holds
  // 2^16, past fp16's range.  (The product keeps the exponent 255 of NaN.)
  static constexpr float kUnit = 0.5f;
  typedef half8_t v8;
  typedef half2_t v2;
  static DFL_DEV floatx4 mfma(v8 a, v8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
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
  typedef bf16x8_t v8;
  typedef bf16x2_t v2;
  static DFL_DEV floatx4 mfma(v8 a, v8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static DFL_DEV v8 dequant(uint32_t w, float s) {
    const v2 p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0);
    const v2 p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1);
    const v2 p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2);
    const v2 p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
    return (v8){p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
  }
  static DFL_DEV float sum2(v2 p, float c) { return c + ((float)p.x + (float)p.y); }
};

// Sequence s of the launch, and (lane 0 of the caller's choice) its error bit.
DFL_DEV Kv4Seq attn_seq(const Kv4AttnArgs& a, int s, int tile_rows) {
  return kv4_seq(a.starts[s], a.starts[s + 1], a.lens[s], a.n_rows, a.width, a.page_shift,
                 a.n_heads / a.n_kv, tile_rows);
}
DFL_DEV long long wave_sum_ll(long long v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// Key blocks of all units; every lane gets the sum.
DFL_DEV long long attn_total(const Kv4AttnArgs& a, int tile_rows) {
  const int lane = threadIdx.x & 63;
  long long t = 0;
  for (int s = lane; s < a.n_seq; s += 64) {
    const Kv4Seq q = attn_seq(a, s, tile_rows);
    if (q.bad) atomicOr(a.err, KV4_ERR_PAGE);
    t += kv4_cost(q, a.n_kv);
  }
  return wave_sum_ll(t);
}
// The sequence that holds position pos of a cumulative count (blocks: its blocks; else its units),
// and the count before it.  pos must lie below the total.
template <bool UNITS>
DFL_DEV int attn_find(const Kv4AttnArgs& a, int tile_rows, long long pos, long long& before) {
  const int lane = threadIdx.x & 63;
  long long acc = 0;
  for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
    long long c = 0;
    if (s0 + lane < a.n_seq) {
      const Kv4Seq q = attn_seq(a, s0 + lane, tile_rows);
      c = UNITS ? (long long)q.tiles * a.n_kv : kv4_cost(q, a.n_kv);
    }
    long long in = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const long long x = __shfl_up(in, o, 64);
      if (lane >= o) in += x;
    }
    const unsigned long long past = __ballot(acc + in > pos);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      before = acc + __shfl(in - c, l, 64);
      return s0 + l;
    }
    acc += __shfl(in, 63, 64);
  }
  before = acc;
  return a.n_seq;
}

// Visible keys of row `row` (token * ratio + head) of a sequence.
DFL_DEV int attn_visible(const Kv4AttnArgs& a, const Kv4Seq& q, int token) {
  return a.causal ? max(0, min(q.len, q.len - q.qlen + token + 1)) : q.len;
}

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
  const long long total = attn_total(a, ROWS);
  const long long per = kv4_per(total, a.workers);
  const long long w = blockIdx.x;
  long long pos = w * per;
  const long long end = min(total, pos + per);
  while (pos < end) {
    // the unit at pos, and the run [b0, b1) of its blocks
    long long s_at;
    const int s = __builtin_amdgcn_readfirstlane(attn_find<false>(a, ROWS, pos, s_at));
    if (s >= a.n_seq) break;   // (cannot be: pos < total)
    const Kv4Seq sq = attn_seq(a, s, ROWS);
    const long long unit = (pos - s_at) / sq.nblk;
    const long long u0 = s_at + unit * sq.nblk;
    const int b0 = (int)(pos - u0), b1 = (int)min((long long)sq.nblk, b0 + (end - pos));
    const int head = (int)(unit / sq.tiles), tile = (int)(unit - (long long)head * sq.tiles);
    pos += b1 - b0;
    const bool whole = b0 == 0 && b1 == sq.nblk;

    // query fragments: step st covers values 32 g + 8 st ..; visible keys of this lane's rows
    v8 qf[NT][4];
    int vis[NT];
    int vmin = 0x7fffffff, vmax = 0;
    const int n_row = sq.qlen * ratio;   // rows of the sequence and kv head
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = (tile * NT + n) * 16 + i;
      const int rr = min(r, n_row - 1);
      const int tok = rr / ratio;
      const T* qp = reinterpret_cast<const T*>(a.q) + (long long)(sq.q0 + tok) * a.q_row +
                    (long long)(head * ratio + rr - tok * ratio) * a.q_head + 32 * g;
#pragma unroll
      for (int st = 0; st < 4; ++st) qf[n][st] = *reinterpret_cast<const v8*>(qp + 8 * st);
      vis[n] = attn_visible(a, sq, tok);
      vmin = min(vmin, vis[n]);
      vmax = max(vmax, vis[n]);
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      vmin = min(vmin, __shfl_xor(vmin, o, 64));
      vmax = max(vmax, __shfl_xor(vmax, o, 64));
    }
    vmin = __builtin_amdgcn_readfirstlane(vmin);
    vmax = __builtin_amdgcn_readfirstlane(vmax);

    floatx4 o[NT][8];
    float mrun[NT], lrun[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      mrun[n] = -FLT_MAX;
      lrun[n] = 0.f;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[n][d] = (floatx4){0.f, 0.f, 0.f, 0.f};
    }

    const int subs_shift = a.page_shift - 5;
    const int* trow = a.table + (long long)s * a.width;
    // block b's address; pg < 0: no such page (its keys are absent)
    auto block_ptr = [&](int b, int& pg) {
      pg = trow[b >> subs_shift];
      if (pg >= a.n_pages) pg = -1;
      return a.pool + kv4_block_at(max(pg, 0), a.n_kv, head, 1 << subs_shift,
                                   b & ((1 << subs_shift) - 1));
    };
    u32x4 kc[2], vc[2];
    uint32_t sc = 0;
    int pg = 0;
    auto load_block = [&](int b) {
      const unsigned char* p = block_ptr(b, pg);
      kc[0] = load_vec(p + 16 * (4 * i + g));
      kc[1] = load_vec(p + 1024 + 16 * (4 * i + g));
      vc[0] = load_vec(p + KV4_V + 16 * (4 * i + g));
      vc[1] = load_vec(p + KV4_V + 1024 + 16 * (4 * i + g));
      sc = *reinterpret_cast<const uint32_t*>(p + KV4_SC + 4 * lane);
    };
    // blocks that no row of the tile sees add nothing
    const int b_end = min(b1, (vmax + KV4_KEYS - 1) / KV4_KEYS);
    int b = b0 + wv;
    if (b < b_end) load_block(b);
    for (; b < b_end; b += 4) {
      u32x4 k0 = kc[0], k1 = kc[1], v0 = vc[0], v1 = vc[1];
      uint32_t s4 = sc;
      const int page = pg;
      if (b + 4 < b_end) load_block(b + 4);
      const int kbase = b * KV4_KEYS;
      const bool masked = kbase + KV4_KEYS > vmin || page < 0;   // (uniform)
      unsigned long long poison = 0;
      if (masked) {
        if (page < 0 && lane == 0) atomicOr(a.err, KV4_ERR_PAGE);
        // V rows that nobody may see, and groups that stand for NaN (they must not reach a row
        // that does not see them, as 0 * NaN): zero codes; the rows that do see one are set below
        const int lim = page < 0 ? 0 : sq.len;
        const bool gone0 = kbase + kv4_key(i, 0) >= lim, gone1 = kbase + kv4_key(i, 1) >= lim;
        const bool nan0 = !gone0 && ((s4 >> 16) & 255) == 255, nan1 = !gone1 && (s4 >> 24) == 255;
        if (gone0 || nan0) { v0 = (u32x4){0, 0, 0, 0}; s4 &= 0xff00ffffu; }
        if (gone1 || nan1) { v1 = (u32x4){0, 0, 0, 0}; s4 &= 0x00ffffffu; }
        poison = __ballot(nan0 || nan1);
        if (poison) {
          // o of every row that sees such a key, in the values of that group
#pragma unroll 1
          for (int key = 0; key < KV4_KEYS; ++key) {
            const int r = kv4_row(key);
            const unsigned long long hit = __ballot((r >> 4) ? nan1 : nan0);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              if (kbase + key < vis[n])
                static_for<0, 4>([&](auto group) {
                  constexpr int gr = group;
                  if ((hit >> ((r & 15) + 16 * gr)) & 1) {
                    o[n][2 * gr] = o[n][2 * gr + 1] =
                        (floatx4){__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
                  }
                });
          }
        }
      }
      const float sk0 = M::kUnit * __uint_as_float((s4 & 255u) << 23);
      const float sk1 = M::kUnit * __uint_as_float(((s4 >> 8) & 255u) << 23);
      const float sv0 = M::kUnit * __uint_as_float(((s4 >> 16) & 255u) << 23);
      const float sv1 = M::kUnit * __uint_as_float((s4 >> 24) << 23);
      floatx4 sa[NT], sb[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) sa[n] = sb[n] = (floatx4){0.f, 0.f, 0.f, 0.f};
      static_for<0, 4>([&](auto step) {
        constexpr int st = step;
        const v8 f0 = M::dequant(k0[st], sk0), f1 = M::dequant(k1[st], sk1);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          sa[n] = M::mfma(f0, qf[n][st], sa[n]);
          sb[n] = M::mfma(f1, qf[n][st], sb[n]);
        }
      });
      static_for<0, 4>([&](auto step) {
        constexpr int st = step;
        *reinterpret_cast<v8*>(vwrite + 16 * st) = M::dequant(v0[st], sv0);
        *reinterpret_cast<v8*>(vwrite + 16 * VROW + 16 * st) = M::dequant(v1[st], sv1);
      });
      // softmax of this lane's 8 keys (kbase + 8 g ..) for its row i of each tile
      v8 pf[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float v[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          v[r] = sa[n][r] * scale;
          v[4 + r] = sb[n][r] * scale;
        }
        if (masked) {
          const int lim = page < 0 ? 0 : vis[n];
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (kbase + 8 * g + r >= lim) v[r] = -INFINITY;
        }
        float top = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])),
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
        const float ref = mrun[n] - KV4_LIFT;
#pragma unroll
        for (int r = 0; r < 8; r += 2) {
          const v2 p = __builtin_convertvector(
              ((floatx2){__builtin_amdgcn_exp2f(v[r] - ref), __builtin_amdgcn_exp2f(v[r + 1] - ref)}), v2);
          lrun[n] = M::sum2(p, lrun[n]);
          pf[n][r] = p.x;
          pf[n][r + 1] = p.y;
        }
      }
      static_for<0, 8>([&](auto dt) {
        constexpr int d = dt;
        typedef __attribute__((address_space(3))) short4_t* lp;
        const short4_t t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(vread + 32 * d));
        const short4_t t1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(vread + 16 * VROW + 32 * d));
        typedef short short8_t __attribute__((ext_vector_type(8)));
        const v8 vf = __builtin_bit_cast(
            v8, (short8_t){t0.x, t0.y, t0.z, t0.w, t1.x, t1.y, t1.z, t1.w});
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][d] = M::mfma(vf, pf[n], o[n][d]);
      });
    }

    // join the four waves: a row's reference is its largest, the states are brought to it
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
    const long long piece = kv4_piece(w, per, u0);
    float* wsO = a.ws + piece * kv4_piece_floats(ROWS);
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
      const int r = tile * ROWS + c;
      if (r < n_row) {
        if (whole) {
          const int tok = r / ratio;
          const long long orow = (long long)(sq.q0 + tok) * a.n_heads + head * ratio + r - tok * ratio;
          const bool none = vis[n] <= 0;   // a row that sees no key: zeros, and the sum of none
          T* op = reinterpret_cast<T*>(a.out) + orow * KV4_D + 4 * g;
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
        } else {
          // (a.ws holds two pieces a worker)
#pragma unroll
          for (int dd = 0; dd < 2; ++dd)
            *reinterpret_cast<floatx4*>(wsO + c * KV4_D + 16 * (2 * wv + dd) + 4 * g) = sum[dd];
          if (wv == 0 && g == 0) {
            wsO[ROWS * KV4_D + 2 * c] = m;
            wsO[ROWS * KV4_D + 2 * c + 1] = l;
          }
        }
      }
    }
    __syncthreads();   // mls is written again
  }
}

// A row of a unit that several workers share: their partial states joined in the order of the
// keys.  One wave to a row, two values a lane.
template <typename T>
__global__ __launch_bounds__(256) void kv4_merge_kernel(Kv4AttnArgs a, int tile_rows) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int ratio = a.n_heads / a.n_kv;
  const int groups = tile_rows / 4;                 // workgroups of a unit
  const long long unit = blockIdx.x / groups;
  const int c = (int)(blockIdx.x % groups) * 4 + wv;
  long long before;
  const int s = __builtin_amdgcn_readfirstlane(attn_find<true>(a, tile_rows, unit, before));
  if (s >= a.n_seq) return;
  const Kv4Seq sq = attn_seq(a, s, tile_rows);
  const long long u = unit - before;
  const int head = (int)(u / sq.tiles), tile = (int)(u - (long long)head * sq.tiles);
  const int r = tile * tile_rows + c;
  if (r >= sq.qlen * ratio) return;
  // block numbers: those of the sequences before s, then of the units before this one
  long long t = 0, all = 0;
  for (int k = lane; k < a.n_seq; k += 64) {
    const long long cost = kv4_cost(attn_seq(a, k, tile_rows), a.n_kv);
    all += cost;
    if (k < s) t += cost;
  }
  const long long total = wave_sum_ll(all);
  const long long u0 = wave_sum_ll(t) + u * sq.nblk, u1 = u0 + sq.nblk;
  const long long per = kv4_per(total, a.workers);
  const long long w0 = u0 / per, w1 = (u1 - 1) / per;
  if (w0 == w1) return;   // one worker had it all
  const long long pf = kv4_piece_floats(tile_rows);
  float m = -FLT_MAX;
  for (long long w = w0 + lane; w <= w1; w += 64)
    m = fmaxf(m, a.ws[kv4_piece(w, per, u0) * pf + tile_rows * KV4_D + 2 * c]);
  m = wave_max(m);
  float l = 0.f;
  floatx2 o = {0.f, 0.f};
  for (long long w = w0; w <= w1; ++w) {
    const float* p = a.ws + kv4_piece(w, per, u0) * pf;
    const float f = __builtin_amdgcn_exp2f(p[tile_rows * KV4_D + 2 * c] - m);
    const floatx2 x = *reinterpret_cast<const floatx2*>(p + c * KV4_D + 2 * lane);
    l += f * p[tile_rows * KV4_D + 2 * c + 1];
    o.x += f * x.x;
    o.y += f * x.y;
  }
  const int tok = r / ratio;
  const long long orow = (long long)(sq.q0 + tok) * a.n_heads + head * ratio + r - tok * ratio;
  const bool none = attn_visible(a, sq, tok) <= 0;
  typedef T o2 __attribute__((ext_vector_type(2)));
  *reinterpret_cast<o2*>(reinterpret_cast<T*>(a.out) + orow * KV4_D + 2 * lane) =
      (o2){(T)(none ? 0.f : o.x / l), (T)(none ? 0.f : o.y / l)};
  if (a.lse && lane == 0)
    a.lse[orow] = none ? -INFINITY : (m - KV4_LIFT + __log2f(l)) * 0.69314718056f;
}

// Units that a launch can have at most.
long long max_units(const Kv4AttnArgs& a, int tile_rows) {
  const long long rows = (long long)a.n_rows * (a.n_heads / a.n_kv);
  // a tile of a sequence holds a row of its own
  const long long tiles = rows / tile_rows + (a.n_seq < a.n_rows ? a.n_seq : a.n_rows);
  return tiles * a.n_kv;
}

template <typename T>
void attend(const Kv4AttnArgs& a, hipStream_t st) {
  const int tr = kv4_tile_rows(a.n_rows, a.n_heads, a.n_kv, a.n_seq);
  const dim3 grid(a.workers), block(256);
  if (tr == 16) hipLaunchKernelGGL((kv4_attn_kernel<T, 1>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((kv4_attn_kernel<T, 2>), grid, block, 0, st, a);
  hipLaunchKernelGGL((kv4_merge_kernel<T>), dim3((unsigned)(max_units(a, tr) * (tr / 4))), block, 0, st, a,
                     tr);
}

}  // namespace

int kv4_tile_rows(int n_rows, int n_heads, int n_kv, int n_seq) {
  // rows of a kv head in a sequence, on average
  const long long rows = ((long long)n_rows * (n_heads / n_kv) + n_seq - 1) / n_seq;
  return rows <= 16 ? 16 : 32;
}
int kv4_workers(int n_rows, int n_heads, int n_kv, int n_seq) {
  const int tr = kv4_tile_rows(n_rows, n_heads, n_kv, n_seq);
  return KV4_CUS * (tr == 16 ? 3 : 2);
}

void launch_kv4_step(const Kv4StepArgs& a, hipStream_t st) {
  if (a.n_seq <= 64 && a.max_rows <= 4096) {
    hipLaunchKernelGGL(kv4_step_small_kernel, dim3(1), dim3(1024), 0, st, a);
    return;
  }
  hipLaunchKernelGGL(kv4_step_scan_kernel, dim3(1), dim3(1024), 0, st, a);
  const int wgs = min(1024, (a.n_seq + 3) / 4);
  hipLaunchKernelGGL(kv4_step_free_kernel, dim3(wgs), dim3(256), 0, st, a);
  hipLaunchKernelGGL(kv4_step_take_kernel, dim3(wgs), dim3(256), 0, st, a);
  if (a.max_rows > 0)
    hipLaunchKernelGGL(kv4_step_rows_kernel, dim3(min(2048, (a.max_rows + 255) / 256)), dim3(256), 0, st, a);
}

static dim3 rows_grid(const Kv4RowsArgs& a) {
  const long long wgs = ((long long)a.rows * 2 * a.n_kv * 16 + 255) / 256;
  return dim3((unsigned)(wgs < 65536 ? wgs : 65536));
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
void launch_kv4_attend(const Kv4AttnArgs& a, hipStream_t st) {
  if (a.dtype == 1) attend<half_t>(a, st);
  else attend<bf16_t>(a, st);
}

}  // namespace dfl
