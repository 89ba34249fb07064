// mg_policy.hip — the clipped policy loss with its gradient, and the draw of actions (include/minigrid_ops.h).
//
// A row's distribution enters through three sums around its largest logit m:  s = sum e^{l - m},  t = sum e^{l - m} (l - m); then log-sum-exp = m + log s,
// entropy = log s - t / s.  Both are gathered in one pass over the logits, the maximum running along.  What the loss decides by (is the ratio
// beyond the clipping border?) and what the draw decides by (where does the running sum pass u s?) is decided in 64 bits: a value next to a border
// falls on the side that the mathematics says.  The draw's sums and those of a loss over up to 64 columns are 64-bit throughout; longer rows of a loss
// are summed from 32-bit exponentials, and a row whose ratio lies within their error of its border is summed again in 64 bits (row_result).
#include "mg_ops.h"

namespace mgo {

constexpr int SMALL_VOCAB = 64;          // up to here a lane owns a row
constexpr float NEG_INF = -__builtin_inff();

// e^d for d <= 0 (or -inf, or NaN) in 64 bits: d = k ln 2 + r with |r| <= ln 2 / 2, e^r as its Taylor sum up to r^12 (what is left out is below 2e-16)
__device__ __forceinline__ double exp_neg(double d) {
  const double k = __builtin_rint(d * 1.44269504088896340736);
  const double r = __builtin_fma(k, -2.3190468138462996e-17, __builtin_fma(k, -LN2, d));     // ln 2 in two parts
  double p = 1.0 / 479001600.0;
  p = __builtin_fma(p, r, 1.0 / 39916800.0);
  p = __builtin_fma(p, r, 1.0 / 3628800.0);
  p = __builtin_fma(p, r, 1.0 / 362880.0);
  p = __builtin_fma(p, r, 1.0 / 40320.0);
  p = __builtin_fma(p, r, 1.0 / 5040.0);
  p = __builtin_fma(p, r, 1.0 / 720.0);
  p = __builtin_fma(p, r, 1.0 / 120.0);
  p = __builtin_fma(p, r, 1.0 / 24.0);
  p = __builtin_fma(p, r, 1.0 / 6.0);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  const double e = __builtin_amdgcn_ldexp(p, (int)k);
  return d < -745.2 ? 0.0 : e;
}

struct Saved { double lse; float dlp, entropy; };       // of a row, for the backward pass; one more behind the rows holds their number (in lse)
static_assert(sizeof(Saved) == 16, "the header promises 16 bytes a row");

struct LossArgs {
  const void* logits; int64_t ld; const void* action; int32_t action_dtype;
  const float *old_lp, *adv, *ref_lp; const uint8_t* mask;
  double lo, hi, kl, ent;                // 1 - clip_lo, 1 + clip_hi, kl_coef, ent_coef
  Saved* save;
  int64_t rows, vocab;
};

template <class A> __device__ __forceinline__ int64_t action_of(const A& a, int64_t i) {
  return a.action_dtype == MG_DT_U8 ? ((const uint8_t*)a.action)[i] : a.action_dtype == MG_DT_I32 ? ((const int32_t*)a.action)[i] : ((const int64_t*)a.action)[i];
}

struct Terms { double policy, kl, entropy, clipped, count; };

// The loss terms of a row that counts, from its statistics; what its backward pass needs is returned.  error: the ratio is known up to the factor 1 +- error.  Where
// that leaves open whether it is beyond its border (`open`), nothing is added.  (A border of 0 or infinity leaves nothing open, nor does an error of 0.)
__device__ __forceinline__ Saved row_terms(const LossArgs& a, int64_t i, double lse, double entropy, double chosen, double error, bool& open, Terms& sum) {
  const double lp = chosen - lse, adv = a.adv[i], q = exp(lp - (double)a.old_lp[i]), border = adv >= 0.0 ? a.hi : a.lo;
  open = q > border * (1.0 - error) && q < border * (1.0 + error);
  if (open) return {};
  const bool clipped = adv >= 0.0 ? q > border : q < border;
  const double policy = -(clipped ? border : q) * adv;
  double dlp = clipped ? 0.0 : -q * adv, kl = 0.0;
  if (a.ref_lp) {
    const double gap = (double)a.ref_lp[i] - lp, e = exp(gap);
    kl = e - gap - 1.0;
    dlp += a.kl * (1.0 - e);
  }
  sum.policy += policy; sum.kl += kl; sum.entropy += entropy; sum.clipped += clipped ? 1.0 : 0.0; sum.count += 1.0;
  return {lse, (float)dlp, (float)entropy};
}

__device__ __forceinline__ void write_out(const LossArgs& a, const Terms& t, float* out) {
  if (a.save) a.save[a.rows] = {t.count, 0.0f, 0.0f};
  const double inv = t.count > 0.0 ? 1.0 / t.count : 0.0, p = t.policy * inv, k = t.kl * inv, h = t.entropy * inv;
  out[0] = (float)(p + a.kl * k - a.ent * h); out[1] = (float)p; out[2] = (float)k; out[3] = (float)h; out[4] = (float)(t.clipped * inv); out[5] = (float)t.count;
}

__device__ __forceinline__ void wave_sum(Terms& t) {
  t.policy = wave_sum(t.policy); t.kl = wave_sum(t.kl); t.entropy = wave_sum(t.entropy); t.clipped = wave_sum(t.clipped); t.count = wave_sum(t.count);
}

// partial sums: five arrays of n
__device__ __forceinline__ void put_part(double* part, int64_t n, int64_t at, const Terms& t) {
  part[at] = t.policy; part[n + at] = t.kl; part[2 * n + at] = t.entropy; part[3 * n + at] = t.clipped; part[4 * n + at] = t.count;
}

// the workgroups' sums in their order (each lane every 1024th of them, then the lanes): one workgroup
__global__ __launch_bounds__(1024) void k_loss_out(LossArgs a, int64_t n, const double* part, float* out) {
  __shared__ Terms s[16];
  Terms t = {};
#pragma unroll 2
  for (int64_t u = threadIdx.x; u < n; u += 1024) {
    t.policy += part[u]; t.kl += part[n + u]; t.entropy += part[2 * n + u]; t.clipped += part[3 * n + u]; t.count += part[4 * n + u];
  }
  wave_sum(t);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    Terms r = {};
    for (int w = 0; w < 16; w++) { r.policy += s[w].policy; r.kl += s[w].kl; r.entropy += s[w].entropy; r.clipped += s[w].clipped; r.count += s[w].count; }
    write_out(a, r, out);
  }
}

// `rows` rows of logits into LDS, row stride vocab | 1 (odd: a lane per row reads without bank conflicts), read as they lie in memory
template <class T>
__device__ __forceinline__ void stage_rows(const T* logits, int64_t ld, int64_t first, int rows, int vocab, float* lds) {
  const int n = rows * vocab;
  for (int u = threadIdx.x; u < n; u += blockDim.x) {
    const int r = u / vocab, c = u - r * vocab;
    lds[r * (vocab | 1) + c] = (float)logits[(first + r) * ld + c];
  }
}

// few columns: a lane owns a row, 64-bit throughout (seven exponentials a row are nothing)
template <class T>
__global__ void k_loss_small(LossArgs a, double* part, float* out) {
  extern __shared__ float lds[];
  const int vocab = (int)a.vocab, R = blockDim.x;
  const int64_t first = (int64_t)blockIdx.x * R;
  const int rows = (int)min((int64_t)R, a.rows - first);
  stage_rows((const T*)a.logits, a.ld, first, rows, vocab, lds);
  __syncthreads();
  Terms sum = {};
  const int64_t i = first + threadIdx.x;
  if ((int)threadIdx.x < rows && (!a.mask || a.mask[i])) {
    const float* l = lds + threadIdx.x * (vocab | 1);
    float m = NEG_INF;
    for (int c = 0; c < vocab; c++) m = fmaxf(m, l[c]);
    double s = 0.0, t = 0.0;
    for (int c = 0; c < vocab; c++) {
      const double d = (double)l[c] - (double)m, e = exp_neg(d);
      s += e;
      t += e == 0.0 ? 0.0 : e * d;                              // a closed column: e^-inf (-inf) counts 0
    }
    const double ls = log(s);
    const int64_t act = action_of(a, i);
    bool open;
    const Saved k = row_terms(a, i, (double)m + ls, ls - t / s, act >= 0 && act < vocab ? (double)l[act] : __builtin_nan(""), 0.0, open, sum);
    if (a.save) a.save[i] = k;
  }
  // the workgroup's sums; LDS is free again
  wave_sum(sum);
  Terms* w = (Terms*)lds;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    Terms r = {};
    for (int v = 0; v < R / 64; v++) { r.policy += w[v].policy; r.kl += w[v].kl; r.entropy += w[v].entropy; r.clipped += w[v].clipped; r.count += w[v].count; }
    if (gridDim.x == 1) write_out(a, r, out);
    else put_part(part, gridDim.x, blockIdx.x, r);
  }
}

// ---- long rows ----
struct Sums { float m; double s, t; };

template <int N>
__device__ __forceinline__ void add_chunk(Sums& a, const float (&x)[N]) {
  float top = x[0];
#pragma unroll
  for (int u = 1; u < N; u++) top = fmaxf(top, x[u]);
  if (top > a.m) {
    if (a.s != 0.0) {
      const double d = (double)a.m - (double)top, f = exp_neg(d);
      a.t = f * (a.t + d * a.s);
      a.s = f * a.s;
    }
    a.m = top;
  }
  if (a.m == NEG_INF) {                                          // nothing but -inf so far; a NaN must not get lost
#pragma unroll
    for (int u = 0; u < N; u++)
      if (x[u] != x[u]) a.s = a.t = __builtin_nan("");
    return;
  }
  constexpr int G = N < 8 ? N : 8;
#pragma unroll
  for (int g = 0; g < N; g += G) {
    float s = 0.0f, t = 0.0f;                                    // eight terms in 32 bits, then into the 64-bit sum
#pragma unroll
    for (int u = g; u < g + G; u++) {
      float d = x[u] - a.m;
      d = d < -200.0f ? -200.0f : d;                             // e^-200 is 0 in 32 bits, and 0 * -200 is 0 (keeps a NaN)
      const float e = __builtin_amdgcn_exp2f(d * LOG2E);
      s += e;
      t = __builtin_fmaf(e, d, t);
    }
    a.s += (double)s;
    a.t += (double)t;
  }
}

template <class T> struct Pack { static constexpr int N = 16 / sizeof(T); };

// the sums of elements [from, to) of a row over NT lanes
template <class T, int NT>
__device__ __forceinline__ Sums row_sums(const T* row, int64_t from, int64_t to, int tid) {
  constexpr int N = Pack<T>::N;
  Sums a = {NEG_INF, 0.0, 0.0};
  const int64_t skew = (int64_t)(((uintptr_t)(row + from) & 15) / sizeof(T));
  const int64_t head = min(to, from + (skew ? N - skew : 0)), body = head + (to - head) / N * N;
  if (from + tid < head) { const float x[1] = {(float)row[from + tid]}; add_chunk(a, x); }
  int64_t c = head + (int64_t)tid * N;
  for (; c + 3 * NT * N < body; c += (int64_t)4 * NT * N) {       // four chunks on their way at a time, one look at the maximum
    T v[4][N];
#pragma unroll
    for (int g = 0; g < 4; g++) __builtin_memcpy(v[g], __builtin_assume_aligned(row + c + g * NT * N, 16), 16);
    float x[4 * N];
#pragma unroll
    for (int u = 0; u < 4 * N; u++) x[u] = (float)v[u / N][u % N];
    add_chunk(a, x);
  }
  for (; c < body; c += (int64_t)NT * N) {
    T v[N];
    __builtin_memcpy(v, __builtin_assume_aligned(row + c, 16), 16);
    float x[N];
#pragma unroll
    for (int u = 0; u < N; u++) x[u] = (float)v[u];
    add_chunk(a, x);
  }
  if (body + tid < to) { const float x[1] = {(float)row[body + tid]}; add_chunk(a, x); }
  return a;
}

__device__ __forceinline__ void wave_join(Sums& a) {
  const float M = wave_max(a.m);
  const double d = a.m == NEG_INF ? 0.0 : (double)a.m - (double)M, f = exp_neg(d);
  a.t = wave_sum(f * (a.t + d * a.s));
  a.s = wave_sum(f * a.s);
  a.m = M;
}

// d loss / d logit_j = g / count (dlp (1[j = action] - p_j) + ent p_j (l_j - lse + H)), p_j = e^{l_j - lse}
struct GradArgs {
  const void* logits; int64_t ld; const void* action; int32_t action_dtype; const uint8_t* mask;
  const Saved* save; const float* grad; void* dlogits;
  float ent; int64_t rows, vocab;
};
__device__ __forceinline__ float grad_of(float l, double lse, float entropy, float dlp, float ent, bool chosen) {
  float d = (float)((double)l - lse);
  d = d < -200.0f ? -200.0f : d;
  const float p = __builtin_amdgcn_exp2f(d * LOG2E);
  return p * (ent * (d + entropy) - dlp) + (chosen ? dlp : 0.0f);
}

template <class T>
__global__ void k_grad_small(GradArgs a) {
  extern __shared__ float lds[];
  const int vocab = (int)a.vocab, R = blockDim.x;
  const int64_t first = (int64_t)blockIdx.x * R;
  const int rows = (int)min((int64_t)R, a.rows - first);
  stage_rows((const T*)a.logits, a.ld, first, rows, vocab, lds);
  __syncthreads();
  if ((int)threadIdx.x < rows) {
    float* l = lds + threadIdx.x * (vocab | 1);
    const int64_t i = first + threadIdx.x;
    if (!a.mask || a.mask[i]) {
      const Saved s = a.save[i];
      const float share = a.grad[0] / (float)a.save[a.rows].lse, dlp = s.dlp * share, ent = a.ent * share;
      const int64_t act = action_of(a, i);
      for (int c = 0; c < vocab; c++) l[c] = grad_of(l[c], s.lse, s.entropy, dlp, ent, c == act);
    } else {
      for (int c = 0; c < vocab; c++) l[c] = 0.0f;
    }
  }
  __syncthreads();
  T* d = (T*)a.dlogits + first * vocab;
  for (int u = threadIdx.x; u < rows * vocab; u += R) {
    const int r = u / vocab, c = u - r * vocab;
    d[u] = (T)lds[r * (vocab | 1) + c];
  }
}

// The gradient of a long row, in powers of two: with y = (l - lse) log2 e it is 2^y (ent ln 2 (y + H log2 e) - dlp), plus dlp at the action.  lse comes in
// two parts: l - hi is as good as exact where p is large.
struct GradRow {
  float hi, lo2, ent2, k, dlp;
  __device__ __forceinline__ GradRow(const Saved& s, float dlp_, float ent) : hi((float)s.lse), ent2(ent * (float)LN2), dlp(dlp_) {
    lo2 = (float)(s.lse - (double)hi) * LOG2E;
    k = __builtin_fmaf(ent, s.entropy, -dlp_);
  }
  __device__ __forceinline__ float operator()(float l) const {
    const float y = __builtin_fmaf(l - hi, LOG2E, -lo2);
    return __builtin_amdgcn_exp2f(y) * __builtin_fmaf(ent2, fmaxf(y, -300.0f), k);           // (a NaN is in the first factor, and a closed column's is 0)
  }
  // the chunk of columns c..c + N
  template <class T, int N> __device__ __forceinline__ void chunk(T* x, int64_t c, int64_t act) const {
    float g[N];
#pragma unroll
    for (int u = 0; u < N; u++) g[u] = (*this)((float)x[u]);
    if ((uint64_t)(act - c) < N)                                 // (rarely: no lane of the wave has it)
#pragma unroll
      for (int u = 0; u < N; u++) g[u] += c + u == act ? dlp : 0.0f;
#pragma unroll
    for (int u = 0; u < N; u++) x[u] = (T)g[u];
  }
};

// the gradient of elements [from, to) of a row that counts, or zeros
template <class T, int NT>
__device__ __forceinline__ void grad_run(const T* row, T* d, int64_t from, int64_t to, bool on, const GradRow& g, int64_t act) {
  constexpr int N = Pack<T>::N;
  // whole 16-byte stores: the run is counted from the gradient's alignment, the logits may lie at any
  const int64_t skew = (int64_t)(((uintptr_t)(d + from) & 15) / sizeof(T));
  const int64_t head = min(to, from + (skew ? N - skew : 0)), body = head + (to - head) / N * N;
  auto one = [&](int64_t c) {
    T x[1] = {(T)0.0f};
    if (on) {
      x[0] = row[c];
      g.chunk<T, 1>(x, c, act);
    }
    d[c] = x[0];
  };
  if (from + threadIdx.x < head) one(from + threadIdx.x);
#pragma unroll 2
  for (int64_t c = head + (int64_t)threadIdx.x * N; c < body; c += NT * N) {
    T v[N] = {};
    if (on) {
      __builtin_memcpy(v, row + c, 16);
      g.chunk<T, N>(v, c, act);
    }
    __builtin_memcpy(__builtin_assume_aligned(d + c, 16), v, 16);
  }
  if (body + threadIdx.x < to) one(body + threadIdx.x);
}

// how many rows count: one workgroup
__global__ __launch_bounds__(1024) void k_count(const uint8_t* mask, int64_t rows, double* count) {
  __shared__ int64_t w[16];
  int64_t n = 0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < rows; i += 1024) n += mask[i] ? 1 : 0;
#pragma unroll
  for (int m = 32; m; m >>= 1) n += __shfl_xor((int)n, m);       // (a lane has less than 2^21 of them)
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    n = 0;
    for (int v = 0; v < 16; v++) n += w[v];
    *count = (double)n;
  }
}

// what a row's thread 0 makes of its sums; error and open as in row_terms
template <class T>
__device__ __forceinline__ Saved row_result(const LossArgs& a, int64_t i, const T* row, float m, double s, double t, double error, bool& open, Terms& sum) {
  const double ls = log(s);
  const int64_t act = action_of(a, i);
  const Saved k = row_terms(a, i, (double)m + ls, ls - t / s, act >= 0 && act < a.vocab ? (double)(float)row[act] : __builtin_nan(""), error, open, sum);
  if (a.save && !open) a.save[i] = k;
  return k;
}

// The sums of a long row are made in 32 bits: d = l - m is rounded (2^-24 |d|), so is d log2 e (2^-24 |d|, and its constant another 1.4e-8 |d|), the exponential is
// good to 2^-23, and up to eight terms are added in 32 bits (7 x 2^-24).  So s, and with it the ratio, is off by at most 2^-24 (9 + 2.3 D) of itself, D = -t / s
// the mean of |d| under the row's distribution.  Where that leaves open whether the ratio is beyond its border (a row in 10^5 or so), the row's first wave sums
// it again with 64-bit exponentials.  (Where every row lies on its border, a clip of 0 and a policy that has not moved, 16 384 x 40 961 bf16 take 3.2 ms.)
__device__ __forceinline__ double sums_error(double s, double t) { return 0x1p-24 * (16.0 - 4.0 * (t / s)); }
struct Sums64 { double s, t; };
template <class T>
__device__ __noinline__ Sums64 wave_sums_64(const T* row, int64_t vocab, float m) {
  double s = 0.0, t = 0.0;
#pragma unroll 4
  for (int64_t c = threadIdx.x; c < vocab; c += 64) {
    const double d = (double)(float)row[c] - (double)m, e = exp_neg(d);
    s += e;
    t += e == 0.0 ? 0.0 : e * d;
  }
  return {wave_sum(s), wave_sum(t)};
}

// By the row's first wave, with arguments and results in LDS.  (Called, not inlined: the constants of its exp and log would be held in registers over the whole
// loop, next to the row.)
struct LossShared { LossArgs a; Terms sum; Saved saved; };
template <class T>
__device__ __noinline__ void row_result_call(LossShared* sh, int64_t i, const T* row, float m, double s, double t) {
  bool open = false;
  if (threadIdx.x == 0) sh->saved = row_result(sh->a, i, row, m, s, t, sums_error(s, t), open, sh->sum);
  if (!__ballot(open)) return;
  const Sums64 w = wave_sums_64<T>(row, sh->a.vocab, m);
  if (threadIdx.x == 0) sh->saved = row_result(sh->a, i, row, m, w.s, w.t, 0.0, open, sh->sum);
}

// A workgroup per row at a time, every gridDim-th row: rows of up to C x NT 16-byte chunks are held in registers, so the maximum, the sums and, where
// dlogits is wanted, the gradient (for the factor 1) take one trip to memory.  16 384 x 40 961 bf16, a quarter masked: 2.35 GB in 517 us, 4.5 TB/s, bound by
// memory and by about twenty vector instructions an element together (two workgroups a CU, 127 registers).  The loss and the gradient from two readings
// took 719 us, a second reading through the caches 814.  (Handed to the call per row in scratch memory and not in LDS, the arguments cost 100 us of that, and of
// 65 536 x 1 000 f32 424 us where it is 282.)
// count: how many rows count (where dlogits and a mask are there), else all do.
template <class T, int NT, int C>
__global__ __launch_bounds__(NT, 4) void k_loss_held(LossArgs a, double* part, const double* count, T* dlogits) {
  constexpr int N = Pack<T>::N, W = NT / 64;
  typedef T VT __attribute__((ext_vector_type(N)));
  __shared__ float wm[W];
  __shared__ double ws[W], wt[W];
  __shared__ LossShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) { sh.a = a; sh.sum = {}; }                         // (the first wave reads it behind the first barrier)
  float share = 0.0f;
  if (dlogits) share = 1.0f / (float)(a.mask ? *count : (double)a.rows);
  for (int64_t i = blockIdx.x; i < a.rows; i += gridDim.x) {
    const T* row = (const T*)a.logits + i * a.ld;
    T* d = dlogits + i * a.vocab;
    // whole 16-byte chunks as the gradient's alignment deals them (the logits may lie at any); in front of and behind them less than a chunk
    const int skew = dlogits ? (int)(((uintptr_t)d & 15) / sizeof(T)) : (int)(((uintptr_t)(i * a.vocab * sizeof(T)) & 15) / sizeof(T));
    const int vocab = (int)a.vocab, head = min(vocab, skew ? N - skew : 0), body = head + (vocab - head) / N * N;
    if (a.mask && !a.mask[i]) {                                  // (uniform in the workgroup)
      if (dlogits) {
        if (tid < head) d[tid] = (T)0.0f;
        for (int c = head + tid * N; c < body; c += NT * N) *(u32x4*)__builtin_assume_aligned(d + c, 16) = (u32x4)(0u);
        if (body + tid < vocab) d[body + tid] = (T)0.0f;
      }
      continue;
    }
    u32x4 v[C];
    T edge = (T)NEG_INF;
    // the chunk's elements, widened where they are used: otherwise they would be kept widened, and not fit
    auto chunk = [&](int q) __attribute__((always_inline)) {
      asm volatile("" : "+v"(v[q]));
      return __builtin_bit_cast(VT, v[q]);
    };
    const int at = tid < head ? tid : tid >= 64 && body + tid - 64 < vocab ? body + tid - 64 : -1;      // an element of the head, or of the rest
#pragma unroll
    for (int q = 0; q < C; q++) {
      const int c = head + (q * NT + tid) * N;
      v[q] = (u32x4)(sizeof(T) == 4 ? 0xff800000u : std::is_same_v<T, bf16> ? 0xff80ff80u : 0xfc00fc00u);        // -inf
      if (c < body) __builtin_memcpy(&v[q], row + c, 16);
    }
    if (at >= 0) edge = row[at];
    float m = (float)edge;
#pragma unroll
    for (int q = 0; q < C; q++) {
      const VT x = chunk(q);
#pragma unroll
      for (int u = 0; u < N; u++) m = fmaxf(m, (float)x[u]);
    }
    m = wave_max(m);
    if (lane == 0) wm[wave] = m;
    __syncthreads();
    m = wm[0];
#pragma unroll
    for (int w = 1; w < W; w++) m = fmaxf(m, wm[w]);
    double s = 0.0, t = 0.0;
    auto add = [&](float x, float& e8, float& t8) __attribute__((always_inline)) {
      const float z = (x - m) * LOG2E, e = __builtin_amdgcn_exp2f(z);
      e8 += e;
      t8 = __builtin_fmaf(e, fmaxf(z, -300.0f), t8);             // (2^-300 is 0 in 32 bits; a NaN is in e)
    };
#pragma unroll
    for (int q = 0; q < C; q++) {
      if (head + (q * NT + (tid & ~63)) * N >= body) break;      // (uniform in the wave)
      const VT x = chunk(q);
      float e8 = 0.0f, t8 = 0.0f;                                // at most eight terms in 32 bits, then into the 64-bit sum
#pragma unroll
      for (int u = 0; u < N; u++) add((float)x[u], e8, t8);
      s += (double)e8;
      t += (double)t8;
    }
    {
      float e8 = 0.0f, t8 = 0.0f;
      if (at >= 0) add((float)edge, e8, t8);
      s += (double)e8;
      t += (double)t8;
    }
    s = wave_sum(s);
    t = wave_sum(t);
    if (lane == 0) { ws[wave] = s; wt[wave] = t; }
    __syncthreads();
    if (tid < 64) {
#pragma unroll
      for (int w = 1; w < W; w++) { s += ws[w]; t += wt[w]; }
      row_result_call<T>(&sh, i, row, m, s, t * LN2);
    }
    if (!dlogits) continue;                                      // (the first wave has read what the next row overwrites before it comes to the next barrier)
    __syncthreads();
    const GradRow g(sh.saved, sh.saved.dlp * share, (float)a.ent * share);
    const int act = (int)min((int64_t)0x7fffffff, max((int64_t)-1, action_of(a, i)));
#pragma unroll
    for (int q = 0; q < C; q++) {
      const int c = head + (q * NT + tid) * N;
      if (c < body) {
        T x[N];
        const VT h = chunk(q);
        __builtin_memcpy(x, &h, sizeof x);
        g.chunk<T, N>(x, c, act);
        __builtin_memcpy(__builtin_assume_aligned(d + c, 16), x, 16);
      }
    }
    if (at >= 0) {
      T x[1] = {edge};
      g.chunk<T, 1>(x, at, act);
      d[at] = x[0];
    }
  }
  if (tid == 0) put_part(part, gridDim.x, blockIdx.x, sh.sum);
}

// rows that no workgroup's registers hold: their sums alone, the maximum running along
template <class T>
__global__ __launch_bounds__(256, 4) void k_loss_rows(LossArgs a, double* part) {
  __shared__ Sums w[4];
  Terms sum = {};
  for (int64_t i = blockIdx.x; i < a.rows; i += gridDim.x) {
    if (a.mask && !a.mask[i]) continue;                          // (uniform in the workgroup)
    const T* row = (const T*)a.logits + i * a.ld;
    Sums s = row_sums<T, 256>(row, 0, a.vocab, threadIdx.x);
    wave_join(s);
    __syncthreads();                                             // (the row before is done with w)
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x < 64) {
      s = threadIdx.x < 4 ? w[threadIdx.x] : Sums{NEG_INF, 0.0, 0.0};
      wave_join(s);
      for (double error = sums_error(s.s, s.t);; error = 0.0) {
        bool open = false;
        if (threadIdx.x == 0) row_result(a, i, row, s.m, s.s, s.t, error, open, sum);
        if (!__ballot(open)) break;
        const Sums64 again = wave_sums_64<T>(row, a.vocab, s.m);
        s.s = again.s; s.t = again.t;
      }
    }
  }
  if (threadIdx.x == 0) put_part(part, gridDim.x, blockIdx.x, sum);
}

constexpr int64_t GRAD_RUN = 16384;      // elements of a row per workgroup at a time

// unless_one: nothing is to be done for the factor 1
template <class T>
__global__ __launch_bounds__(256) void k_grad_rows(GradArgs a, int64_t runs, int unless_one) {
  if (unless_one && a.grad[0] == 1.0f) return;
  for (int64_t u = blockIdx.x; u < a.rows * runs; u += gridDim.x) {
    // (the last rows first: the forward pass has just left them in the cache behind the L2s)
    const int64_t i = a.rows - 1 - u / runs, from = u % runs * GRAD_RUN, to = min(a.vocab, from + GRAD_RUN);
    const bool on = !a.mask || a.mask[i];
    Saved s = {0.0, 0.0f, 0.0f};
    float dlp = 0.0f, ent = 0.0f;
    int64_t act = -1;
    if (on) {
      s = a.save[i];
      const float share = a.grad[0] / (float)a.save[a.rows].lse;
      dlp = s.dlp * share; ent = a.ent * share; act = action_of(a, i);
    }
    grad_run<T, 256>((const T*)a.logits + i * a.ld, (T*)a.dlogits + i * a.vocab, from, to, on, GradRow(s, dlp, ent), act);
  }
}

// ---- the draw ----
__device__ __forceinline__ void store_action(void* action, int64_t vocab, int64_t i, int64_t k) {
  if (vocab <= 256) ((uint8_t*)action)[i] = (uint8_t)k;
  else ((int32_t*)action)[i] = (int32_t)k;
}

template <class T>
__global__ void k_sample_small(const T* logits, int64_t ld, int64_t rows_all, int vocab, const float* u, void* action, float* lp) {
  extern __shared__ float lds[];
  const int R = blockDim.x;
  const int64_t first = (int64_t)blockIdx.x * R;
  const int rows = (int)min((int64_t)R, rows_all - first);
  stage_rows(logits, ld, first, rows, vocab, lds);
  __syncthreads();
  if ((int)threadIdx.x >= rows) return;
  const int64_t i = first + threadIdx.x;
  const float* l = lds + threadIdx.x * (vocab | 1);
  float m = NEG_INF;
  int best = 0;
  for (int c = 0; c < vocab; c++)
    if (l[c] > m) { m = l[c]; best = c; }
  double s = 0.0;
  for (int c = 0; c < vocab; c++) s += exp_neg((double)l[c] - (double)m);
  int k = best;
  if (u) {
    const double target = (double)u[i] * s;
    double run = 0.0;
    int last = 0;
    k = -1;
    for (int c = 0; c < vocab && k < 0; c++) {
      const double e = exp_neg((double)l[c] - (double)m);
      run += e;
      if (e > 0.0) { last = c; if (run > target) k = c; }
    }
    if (k < 0) k = last;                                         // u s was reached by rounding only
  }
  const bool fine = s > 0.0 && s < __builtin_inf();              // (false for NaN)
  store_action(action, vocab, i, fine ? k : 0);
  lp[i] = fine ? (float)((double)l[k] - (double)m - log(s)) : __builtin_nanf("");
}

// Long rows: a row is cut into 64 pieces, a wave per piece finds its maximum and its sum against it; from the 64 pairs one wave finds the piece in which the
// running sum passes the border, and walks that piece alone.  Few rows: the pieces of a row are dealt to up to sixteen workgroups, and a second kernel
// walks; more rows: one workgroup of four waves does both; many: a wave does.  Bound by the 64-bit exponentials for many rows, by two short launches for few.
constexpr int PIECES = 64, E = 4;        // E: elements of a lane at a time
struct Piece { float m; int32_t at; double s; };          // the largest logit, its first index, sum e^{l - m}
static_assert(sizeof(Piece) == 16, "the workspace is counted in these");

// (a piece is at least what a wave reads at once: 256 elements; the pieces behind the row's end are empty)
__host__ __device__ __forceinline__ int64_t piece_length(int64_t vocab) {
  const int64_t n = ((vocab + PIECES - 1) / PIECES + E - 1) / E * E;
  return n < 64 * E ? 64 * E : n;
}

template <class T>
__device__ __forceinline__ void load_some(const T* row, int64_t c, int64_t to, float (&x)[E]) {
  if (c + E <= to) {
    T v[E];
    __builtin_memcpy(v, row + c, sizeof v);
#pragma unroll
    for (int q = 0; q < E; q++) x[q] = (float)v[q];
  } else {
#pragma unroll
    for (int q = 0; q < E; q++) x[q] = c + q < to ? (float)row[c + q] : NEG_INF;
  }
}

template <class T>
__device__ __forceinline__ Piece look_at(const T* row, int64_t from, int64_t to) {
  const int lane = threadIdx.x & 63;
  float m = NEG_INF;
  int64_t at = to;
  double s = 0.0;
#pragma unroll 2
  for (int64_t c0 = from; c0 < to; c0 += 64 * E) {
    const int64_t c = c0 + lane * E;
    float x[E];
    load_some(row, c, to, x);
    float top = m;
#pragma unroll
    for (int q = 0; q < E; q++)
      if (x[q] > top) { top = x[q]; at = c + q; }
    const double M = top == NEG_INF ? 0.0 : (double)top;
    s *= m == NEG_INF ? 1.0 : exp_neg((double)m - M);            // (without a finite logit so far the sum is 0 or NaN)
#pragma unroll
    for (int q = 0; q < E; q++) s += exp_neg((double)x[q] - M);
    m = top;
  }
  const float M = wave_max(m);
  int first = m == M && m != NEG_INF ? (int)(at - from) : 0x7fffffff;
#pragma unroll
  for (int b = 32; b; b >>= 1) first = min(first, __shfl_xor(first, b));
  s = wave_sum(s * (m == NEG_INF ? 1.0 : exp_neg((double)m - (double)M)));
  return {M, (int32_t)(from + first), s};
}

// by one wave, lane q with the row's piece q
template <class T>
__device__ __forceinline__ void choose(const T* row, int64_t vocab, Piece mine, int64_t i, const float* u, void* action, float* lp) {
  const int lane = threadIdx.x & 63;
  const float M = wave_max(mine.m);
  const double share = mine.s * (mine.m == NEG_INF ? 1.0 : exp_neg((double)mine.m - (double)M));
  double upto = share;                                           // inclusive over the pieces
#pragma unroll
  for (int b = 1; b < 64; b <<= 1) {
    const double o = __hiloint2double(__shfl_up(__double2hiint(upto), b), __shfl_up(__double2loint(upto), b));
    if (lane >= b) upto += o;
  }
  auto of_lane = [](double v, int l) { return __hiloint2double(__shfl(__double2hiint(v), l), __shfl(__double2loint(v), l)); };
  const double S = of_lane(upto, 63);
  if (!(S > 0.0 && S < __builtin_inf())) {                       // (false for NaN)
    if (lane == 0) { store_action(action, vocab, i, 0); lp[i] = __builtin_nanf(""); }
    return;
  }
  int64_t k = __shfl(mine.at, __ffsll((long long)__ballot(mine.m == M)) - 1);
  if (u) {
    const double target = (double)u[i] * S;
    const int64_t len = piece_length(vocab);
    const unsigned long long over = __ballot(upto > target && share > 0.0), some = __ballot(share > 0.0);
    // beyond every piece by rounding only: the last element that has a share, in the last piece that has one
    const int p = over ? __ffsll((long long)over) - 1 : 63 - __builtin_clzll(some);
    double before = p ? of_lane(upto, p - 1) : 0.0;
    const int64_t from = p * len, to = min(vocab, from + len);
    int64_t last = -1;
    bool found = false;
    for (int64_t c0 = from; c0 < to && !found; c0 += 64 * E) {
      float x[E];
      load_some(row, c0 + lane * E, to, x);
      double e[E], sum = 0.0;
#pragma unroll
      for (int q = 0; q < E; q++) { e[q] = exp_neg((double)x[q] - (double)M); sum += e[q]; }
      double run = sum;
#pragma unroll
      for (int b = 1; b < 64; b <<= 1) {
        const double o = __hiloint2double(__shfl_up(__double2hiint(run), b), __shfl_up(__double2loint(run), b));
        if (lane >= b) run += o;
      }
      // the running sum as the lane's elements see it: exact enough to be compared lane by lane, and what a lane passes is passed by its last element
      double r = before + (run - sum);
      int pick = -1, any = -1;
#pragma unroll
      for (int q = 0; q < E; q++) {
        r += e[q];
        if (e[q] > 0.0) { any = q; if (pick < 0 && r > target) pick = q; }
      }
      const unsigned long long hit = __ballot(pick >= 0), has = __ballot(any >= 0);
      if (hit) {
        const int w = __ffsll((long long)hit) - 1;
        last = c0 + w * E + __shfl(pick, w);
        found = true;
      } else if (has) {
        const int w = 63 - __builtin_clzll(has);
        last = c0 + w * E + __shfl(any, w);
      }
      before += of_lane(run, 63);
    }
    if (last >= 0) k = last;
  }
  if (lane == 0) {
    store_action(action, vocab, i, k);
    lp[i] = (float)((double)(float)row[k] - (double)M - log(S));
  }
}

// grid (rows, groups): every wave of a row's groups looks at every (4 groups)-th piece; a single group chooses at once
template <class T>
__global__ __launch_bounds__(256) void k_sample_rows(const T* logits, int64_t ld, int64_t rows, int64_t vocab, const float* u, Piece* pieces, void* action, float* lp) {
  __shared__ Piece all[PIECES];
  const int w = threadIdx.x >> 6;
  const int64_t len = piece_length(vocab);
  for (int64_t i = blockIdx.x; i < rows; i += gridDim.x) {
    const T* row = logits + i * ld;
    for (int p = blockIdx.y * 4 + w; p < PIECES; p += 4 * gridDim.y) {
      const int64_t from = min(vocab, p * len), to = min(vocab, from + len);
      const Piece q = from < to ? look_at(row, from, to) : Piece{NEG_INF, 0, 0.0};
      if ((threadIdx.x & 63) == 0) {
        if (pieces) pieces[i * PIECES + p] = q;
        else all[p] = q;
      }
    }
    if (pieces) continue;
    __syncthreads();
    if (w == 0) choose(row, vocab, all[threadIdx.x & 63], i, u, action, lp);
    __syncthreads();
  }
}

// Many rows, or short ones: a wave per row, so that none waits for another
template <class T>
__global__ __launch_bounds__(256) void k_sample_waves(const T* logits, int64_t ld, int64_t rows, int64_t vocab, const float* u, void* action, float* lp) {
  const int64_t len = piece_length(vocab);
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < rows; i += (int64_t)gridDim.x * 4) {
    const T* row = logits + i * ld;
    Piece mine = {NEG_INF, 0, 0.0};
    for (int p = 0; p * len < vocab; p++) {
      const Piece q = look_at(row, p * len, min(vocab, (p + 1) * len));
      if ((int)(threadIdx.x & 63) == p) mine = q;
    }
    choose(row, vocab, mine, i, u, action, lp);
  }
}

template <class T>
__global__ __launch_bounds__(64) void k_sample_choose(const T* logits, int64_t ld, int64_t vocab, const float* u, const Piece* pieces, void* action, float* lp) {
  const int64_t i = blockIdx.x;
  choose(logits + i * ld, vocab, pieces[i * PIECES + threadIdx.x], i, u, action, lp);
}

// workgroups per row: four of them a CU, each of its four waves with at least one piece (64 x 40 961 f32: 10.5 us with two of them a CU)
static int sample_groups(int64_t rows, int64_t vocab) {
  const int64_t pieces = (vocab + piece_length(vocab) - 1) / piece_length(vocab);
  int g = 1;
  while (g * 4 < pieces && rows * g < 1024) g *= 2;
  return g;
}

// A wave per row, or a workgroup (or several)?  4 096 x 1 000: 16 us against 33, 262 144 x 100: 361 against 1 682, 16 384 x 4 096: 139 against 200; for fewer
// rows only where they are short: 512 x 197: 6.7 against 8.4, 1 024 x 5 000: 29 against 20, 2 048 x 32 000: 165 against 126.
static bool wave_per_row(int64_t rows, int64_t vocab) { return rows >= 4096 || (rows >= 512 && vocab <= 1024); }

static int check_logits(int dtype, int64_t rows, int64_t vocab, int64_t ld) {
  if (dtype != MG_DT_F32 && dtype != MG_DT_BF16 && dtype != MG_DT_F16) return fail(MG_ERR_INVALID, "logits must be f32, bf16 or f16");
  if (rows < 0 || rows > 0x7fffffffll || vocab < 1 || vocab > 0x7fffffffll) return fail(MG_ERR_INVALID, "sizes must be 0 <= rows, 1 <= vocab, below 2^31");
  if (ld < vocab) return fail(MG_ERR_INVALID, "the row stride is smaller than a row");
  return MG_OK;
}

static int check_action(int t) { return t == MG_DT_U8 || t == MG_DT_I32 || t == MG_DT_I64 ? MG_OK : fail(MG_ERR_INVALID, "action must be u8, i32 or i64"); }

static int small_rows(int64_t vocab) { return vocab < 32 ? 256 : 64; }            // rows per workgroup: at most 32 KB of LDS

template <class F> static int by_type(int dtype, F f) {
  return dtype == MG_DT_F32 ? f((const float*)nullptr) : dtype == MG_DT_BF16 ? f((const bf16*)nullptr) : f((const f16*)nullptr);
}

// workgroups of the loss over its rows: for long rows at most 4096, each with its share of them
static int64_t loss_groups(int64_t rows, int64_t vocab) {
  if (vocab <= SMALL_VOCAB) return (rows + small_rows(vocab) - 1) / small_rows(vocab);
  const int64_t per = (rows + 4095) / 4096;
  return per ? (rows + per - 1) / per : 0;
}
constexpr int64_t HELD_BYTES = 160 * 1024;  // the longest row that a workgroup's registers hold

static size_t small_lds(int R, int64_t vocab) { return std::max<size_t>((size_t)R * (vocab | 1) * 4, 4 * sizeof(Terms)); }

}  // namespace mgo

using namespace mgo;

extern "C" {

int mg_op_policy_loss_workspace(int64_t rows, int64_t vocab, int64_t* bytes) {
  const int rc = check_logits(MG_DT_F32, rows, vocab, vocab);
  if (rc != MG_OK) return rc;
  if (!bytes) return fail(MG_ERR_INVALID, "bytes must not be NULL");
  *bytes = loss_groups(rows, vocab) * (int64_t)sizeof(Terms) + 16;          // (behind the sums: the number of rows that count)
  return MG_OK;
}

int mg_op_policy_loss_makes_gradient(int dtype, int64_t vocab) { return vocab > SMALL_VOCAB && vocab * dtype_bytes(dtype) <= HELD_BYTES; }

int mg_op_policy_loss_with_gradient(int device, void* stream, int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, const void* action, int action_dtype,
                                    const float* old_lp, const float* adv, const float* ref_lp, const uint8_t* mask, double clip_lo, double clip_hi, double kl_coef,
                                    double ent_coef, float* out, void* save, void* ws, int64_t ws_bytes, void* dlogits) {
  int rc = check_logits(dtype, rows, vocab, ld);
  if (rc == MG_OK) rc = check_action(action_dtype);
  if (rc != MG_OK) return rc;
  if (!out || (rows && (!logits || !action || !old_lp || !adv))) return fail(MG_ERR_INVALID, "logits, action, old_lp, adv and out must not be NULL");
  if (dlogits && !mg_op_policy_loss_makes_gradient(dtype, vocab)) return fail(MG_ERR_INVALID, "no gradient comes with the loss for rows of this length");
  int64_t need = 0;
  mg_op_policy_loss_workspace(rows, vocab, &need);
  if (ws_bytes < need || !ws || ((uintptr_t)ws & 15)) return fail(MG_ERR_INVALID, "workspace: %lld bytes are needed", (long long)need);
  DeviceGuard g(device);
  if (g.rc != MG_OK) return g.rc;
  hipStream_t st = (hipStream_t)stream;
  LossArgs a = {logits, ld, action, action_dtype, old_lp, adv, ref_lp, mask, 1.0 - clip_lo, 1.0 + clip_hi, kl_coef, ent_coef, (Saved*)save, rows, vocab};
  const int64_t parts = loss_groups(rows, vocab);
  if (rows && vocab <= SMALL_VOCAB) {
    const int R = small_rows(vocab);
    by_type(dtype, [&](auto* t) {
      typedef std::remove_cv_t<std::remove_pointer_t<decltype(t)>> T;
      k_loss_small<T><<<(unsigned)parts, R, small_lds(R, vocab), st>>>(a, (double*)ws, out);
      return 0;
    });
    if (parts == 1) return launched("policy loss");
  } else if (rows) {
    double* count = (double*)ws + parts * 5;
    if (dlogits && mask) k_count<<<1, 1024, 0, st>>>(mask, rows, count);
    by_type(dtype, [&](auto* t) {
      typedef std::remove_cv_t<std::remove_pointer_t<decltype(t)>> T;
      // The smallest workgroup that holds a row, counted in whole 16-byte chunks (less than a chunk of it lies in front of them and behind them).  Where two of them hold it
      // (f32, unmasked, with gradient): 16 384 x 4 096 in 256 threads 119 us, in 512 181; 8 192 x 8 192 in 512 x 4 chunks 130, x 10 136, in 1 024 211; 3 276 x 20 480 in 512
      // 125, in 1 024 149; 65 536 x 65 in 256 234, in 1 024 1 207.
      const int64_t bytes = vocab * (int64_t)sizeof(T), chunks = bytes / 16;
#define MG_HELD(NT, C) k_loss_held<T, NT, C><<<(unsigned)parts, NT, 0, st>>>(a, (double*)ws, count, (T*)dlogits)
      if (chunks <= 256 * 4) MG_HELD(256, 4);
      else if (chunks <= 512 * 4) MG_HELD(512, 4);
      else if (chunks <= 512 * 10) MG_HELD(512, 10);
      else if (bytes <= HELD_BYTES) MG_HELD(1024, 10);
      else k_loss_rows<T><<<(unsigned)parts, 256, 0, st>>>(a, (double*)ws);
#undef MG_HELD
      return 0;
    });
  }
  k_loss_out<<<1, 1024, 0, st>>>(a, parts, (const double*)ws, out);
  return launched("policy loss");
}

int mg_op_policy_loss(int device, void* stream, int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, const void* action, int action_dtype, const float* old_lp,
                      const float* adv, const float* ref_lp, const uint8_t* mask, double clip_lo, double clip_hi, double kl_coef, double ent_coef, float* out,
                      void* save, void* ws, int64_t ws_bytes) {
  return mg_op_policy_loss_with_gradient(device, stream, dtype, rows, vocab, logits, ld, action, action_dtype, old_lp, adv, ref_lp, mask, clip_lo, clip_hi, kl_coef, ent_coef, out,
                                         save, ws, ws_bytes, nullptr);
}

static int loss_backward(int device, void* stream, int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, const void* action, int action_dtype, const uint8_t* mask,
                         double ent_coef, const void* save, const float* grad, void* dlogits, bool unless_one) {
  int rc = check_logits(dtype, rows, vocab, ld);
  if (rc == MG_OK) rc = check_action(action_dtype);
  if (rc != MG_OK || rows == 0) return rc;
  if (!logits || !action || !save || !grad || !dlogits) return fail(MG_ERR_INVALID, "no pointer but mask may be NULL");
  if (unless_one && !mg_op_policy_loss_makes_gradient(dtype, vocab)) return fail(MG_ERR_INVALID, "no gradient comes with the loss for rows of this length");
  DeviceGuard g(device);
  if (g.rc != MG_OK) return g.rc;
  hipStream_t st = (hipStream_t)stream;
  GradArgs a = {logits, ld, action, action_dtype, mask, (const Saved*)save, grad, dlogits, (float)ent_coef, rows, vocab};
  return by_type(dtype, [&](auto* t) {
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(t)>> T;
    if (vocab <= SMALL_VOCAB) {
      const int R = small_rows(vocab);
      k_grad_small<T><<<(unsigned)((rows + R - 1) / R), R, small_lds(R, vocab), st>>>(a);
    } else {
      const int64_t runs = (vocab + GRAD_RUN - 1) / GRAD_RUN;
      k_grad_rows<T><<<(unsigned)std::min<int64_t>(rows * runs, unless_one ? 2048 : 1 << 20), 256, 0, st>>>(a, runs, unless_one);
    }
    return launched("policy loss backward");
  });
}

int mg_op_policy_loss_backward(int device, void* stream, int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, const void* action, int action_dtype,
                               const uint8_t* mask, double ent_coef, const void* save, const float* grad, void* dlogits) {
  return loss_backward(device, stream, dtype, rows, vocab, logits, ld, action, action_dtype, mask, ent_coef, save, grad, dlogits, false);
}

int mg_op_policy_loss_rescale(int device, void* stream, int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, const void* action, int action_dtype,
                              const uint8_t* mask, double ent_coef, const void* save, const float* grad, void* dlogits) {
  return loss_backward(device, stream, dtype, rows, vocab, logits, ld, action, action_dtype, mask, ent_coef, save, grad, dlogits, true);
}

int mg_op_sample_workspace(int64_t rows, int64_t vocab, int64_t* bytes) {
  const int rc = check_logits(MG_DT_F32, rows, vocab, vocab);
  if (rc != MG_OK) return rc;
  if (!bytes) return fail(MG_ERR_INVALID, "bytes must not be NULL");
  *bytes = vocab > SMALL_VOCAB && !wave_per_row(rows, vocab) && sample_groups(rows, vocab) > 1 ? rows * PIECES * (int64_t)sizeof(Piece) : 0;
  return MG_OK;
}

int mg_op_sample(int device, void* stream, int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, const float* u, void* action, float* lp, void* ws,
                 int64_t ws_bytes) {
  int rc = check_logits(dtype, rows, vocab, ld);
  if (rc != MG_OK || rows == 0) return rc;
  if (!logits || !action || !lp) return fail(MG_ERR_INVALID, "logits, action and lp must not be NULL");
  int64_t need = 0;
  mg_op_sample_workspace(rows, vocab, &need);
  if (need && (ws_bytes < need || !ws || ((uintptr_t)ws & 255))) return fail(MG_ERR_INVALID, "workspace: %lld bytes, 256-byte aligned, are needed", (long long)need);
  DeviceGuard g(device);
  if (g.rc != MG_OK) return g.rc;
  hipStream_t st = (hipStream_t)stream;
  return by_type(dtype, [&](auto* t) {
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(t)>> T;
    const T* x = (const T*)logits;
    if (vocab <= SMALL_VOCAB) {
      const int R = small_rows(vocab);
      k_sample_small<T><<<(unsigned)((rows + R - 1) / R), R, (size_t)R * (vocab | 1) * 4, st>>>(x, ld, rows, (int)vocab, u, action, lp);
    } else if (wave_per_row(rows, vocab)) {
      k_sample_waves<T><<<(unsigned)std::min<int64_t>((rows + 3) / 4, 1 << 22), 256, 0, st>>>(x, ld, rows, vocab, u, action, lp);
    } else {
      const int groups = sample_groups(rows, vocab);
      Piece* pieces = groups > 1 ? (Piece*)ws : nullptr;
      k_sample_rows<T><<<dim3((unsigned)std::min<int64_t>(rows, 1 << 22), groups), 256, 0, st>>>(x, ld, rows, vocab, u, pieces, action, lp);
      if (pieces) k_sample_choose<T><<<(unsigned)rows, 64, 0, st>>>(x, ld, vocab, u, pieces, action, lp);
    }
    return launched("sample");
  });
}

}  // extern "C"
