// mg_linear.h — the tile product behind the linear layer and its two gradients, for gfx950's matrix instructions.
//
//   C (i, j) = sum_s A(i, s) B(j, s)
//     forward      A = x (rows, k),  B = w (n, k)      both contiguous along s            y = act(C + b) + r
//     dx = dz w    A = dz (rows, n), B(j, s) = w[s][j] B contiguous along j
//     dw = dzT x   A(i, s) = dz[s][i], B(j, s) = x[s][j]: both contiguous along i / j
//
// An operand that is contiguous along s ("rows") lies in LDS as 128-byte rows of one tile row each; one that is contiguous along i / j ("cols") lies
// there as one row per s and is turned by the transposing LDS read (16-bit types) or read element by element (f32).  Both are swizzled so that the
// fragment reads of a wave spread over all banks.
//
// Three kernels.  k_product takes results at least as large as its tile and at least one tile deep, and then needs no bounds check at all: a tile that would
// stick out is moved back inside (its first rows belong to a neighbour and are not stored), and a last piece of the summed axis is loaded as the last
// whole one with what was summed already set to zero.  Its global loads go through registers: rows may start at any address, and bytes are widened on the
// way.  k_product_direct is the 256-tile of it whose rows are 16-byte aligned: memory to LDS without registers in between.  k_product_guarded checks the
// chunks of tiles that are not whole and takes the rest.
#pragma once
#include "mg_ops.h"

namespace mgo {

typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <class T> struct Chunk;                          // 16 bytes of an operand: what a lane loads and what a lane feeds
template <> struct Chunk<bf16> { typedef bf16x8 V; static constexpr int N = 8; };
template <> struct Chunk<f16> { typedef f16x8 V; static constexpr int N = 8; };
template <> struct Chunk<float> { typedef f32x4 V; static constexpr int N = 4; };

struct Operand {
  const void* p;
  int64_t ld;      // elements between rows of memory
  int32_t extent;  // i (or j): rows of the result this operand feeds
};

struct Epilogue {
  const void* b;   // (n) or null
  const void* r;   // (rows, n) or null
  void* c;         // result of T, row stride ldc
  void* z;         // values in front of the activation (contiguous, of KeptOf<T, act>), or null
  float* part;     // split sums: f32 (splits, rows, n), contiguous; null = store the result
  int64_t ldr, ldc;
  int32_t act;
  int32_t narrow;  // 256 rows of c, r, z and part span less than 2 GiB
};

// ---- activations ----
// What a backward pass keeps of z.  For most activations z in the operands' type: the slope at a rounded z is off by less than dz's own rounding (by a third of it for
// gelu and silu at z of 1).  tanh's slope falls as e^{-2 |z|}, so at a rounded z it is off by 2 |z| half steps of itself: for MG_ACTIVATION_TANH_Z32 z stays in 32 bits.  (dx and
// dw of 2 049 x 300 x 136 bf16 are off by 2.55e-3 of their norm with a rounded z, 2.33e-3 without, by 1.66e-3 where they alone are rounded; the forward and backward
// pass of 65 536 x 512 x 512 take 238 and 253 us.)
template <class T, int ACT> using KeptOf = std::conditional_t<ACT == MG_ACTIVATION_TANH_Z32, float, T>;

// exp2 with a result of 0 far below the smallest number: v_exp_f32, one ulp
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }

// The normal distribution function at -|x|: e^{-x^2/2} q(t), t = 1 / (1 + 0.3 |x|).  q is 0.5 erfcx(|x| / sqrt 2) as a polynomial of degree 8 without a
// constant term, fitted here for the least largest RELATIVE error on |x| <= 13.5 (1.3e-7; 2.9e-7 evaluated in 32 bits); beyond, e^{-x^2/2} is 0 in f32.  The exponential
// adds what rounding its argument to 32 bits makes: gelu(-x) is off by 7e-7 of itself up to 3, 2e-6 at 6, 8e-6 at 13, where it is 1e-37.  (tanh's slope, from
// e^{-2 |z|}: 6e-7 up to 3, 1.1e-6 at 9, 4e-6 at 40; silu: 6e-7 at -9, 2e-6 at -40.)
__device__ __forceinline__ float phi_tail(float a, float* density) {
  const float t = rcp_fast(__builtin_fmaf(0.3f, a, 1.0f));
  float q = 0.03593193367123604f;
  q = __builtin_fmaf(q, t, -0.1582767814397812f);
  q = __builtin_fmaf(q, t, 0.2082078605890274f);
  q = __builtin_fmaf(q, t, -0.05539492145180702f);
  q = __builtin_fmaf(q, t, 0.12946972250938416f);
  q = __builtin_fmaf(q, t, 0.09963735193014145f);
  q = __builtin_fmaf(q, t, 0.12079837918281555f);
  q = __builtin_fmaf(q, t, 0.11962638795375824f);
  const float e = exp2_fast(a * a * (-0.5f * 1.44269504f));
  *density = e * 0.398942280f;
  return q * t * e;
}

__device__ __forceinline__ float tanh_act(float z) {
  // 1 - 2 / (e^{2|z|} + 1) loses the leading bits of a small result: the odd power series up to z^11 below 0.3 (its next term is 4e-9 of the value)
  const float a = fabsf(z), e = exp2_fast(a * (-2.0f * 1.44269504f));
  const float big = copysignf((1.0f - e) * rcp_fast(1.0f + e), z), s = z * z;
  float p = -0.00886323553f;                              // -1382 / 155925
  p = __builtin_fmaf(p, s, 0.0218694885f);                // 62 / 2835
  p = __builtin_fmaf(p, s, -0.0539682540f);               // -17 / 315
  p = __builtin_fmaf(p, s, 0.133333333f);                 // 2 / 15
  p = __builtin_fmaf(p, s, -0.333333333f);                // -1 / 3
  return a < 0.3f ? __builtin_fmaf(z * s, p, z) : (z != z ? z : big);
}

__device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case MG_ACTIVATION_RELU: return z < 0.0f ? 0.0f : z;                       // (keeps a NaN)
    case MG_ACTIVATION_TANH: case MG_ACTIVATION_TANH_Z32: return tanh_act(z);
    case MG_ACTIVATION_GELU: {
      float d;
      const float t = phi_tail(fabsf(z), &d);
      return z * (z < 0.0f ? t : 1.0f - t);
    }
    case MG_ACTIVATION_SILU: return z * rcp_fast(1.0f + exp2_fast(z * -1.44269504f));
    default: return z;
  }
}

// (An infinite z is one that did not fit 16 bits: the slope there is the limit, 0 or 1, not infinity times 0.  Beyond the bounds that z is held in the other factor is 0.)
__device__ __forceinline__ float activate_grad(int act, float z) {
  switch (act) {
    case MG_ACTIVATION_RELU: return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
    case MG_ACTIVATION_TANH: case MG_ACTIVATION_TANH_Z32: {
      const float t = tanh_act(z), e = exp2_fast(fabsf(z) * (-2.0f * 1.44269504f)), q = rcp_fast(1.0f + e);
      return fabsf(z) < 0.3f ? 1.0f - t * t : 4.0f * e * q * q;                // 1 - tanh^2 = 4 e^{-2|z|} / (1 + e^{-2|z|})^2
    }
    case MG_ACTIVATION_GELU: {
      float d;
      const float t = phi_tail(fabsf(z), &d);
      return (z < 0.0f ? t : 1.0f - t) + fminf(fmaxf(z, -16.0f), 16.0f) * d;        // (a NaN is in t)
    }
    case MG_ACTIVATION_SILU: {
      const float p = rcp_fast(1.0f + exp2_fast(z * -1.44269504f));
      return p * __builtin_fmaf(fminf(fmaxf(z, -200.0f), 200.0f), 1.0f - p, 1.0f);  // (a NaN is in p)
    }
    default: return 1.0f;
  }
}

// ---- global loads ----
// N consecutive elements of a memory row as T, element e valid where at + e < end
template <class T, class S>
__device__ __forceinline__ typename Chunk<T>::V load_chunk(const S* row, int64_t at, int64_t end, bool inside) {
  constexpr int N = Chunk<T>::N;
  typename Chunk<T>::V v = {};
  if (!inside || at >= end) return v;
  if constexpr (sizeof(S) == sizeof(T)) {
    if (at + N <= end) {
      __builtin_memcpy(&v, row + at, 16);
      return v;
    }
  } else if (at + N <= end) {
    uint8_t u[N];
    __builtin_memcpy(u, row + at, N);
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = (T)(float)u[e];
    return v;
  }
#pragma unroll
  for (int e = 0; e < N; e++)
    if (at + e < end) v[e] = (T)(float)row[at + e];
  return v;
}

// One operand's tile: EXT rows of the result x 128 / sizeof(T) summed elements = EXT x 128 bytes of LDS.
template <class T, bool COLS, int EXT>
struct Lds {
  typedef typename Chunk<T>::V V;
  static constexpr int N = Chunk<T>::N, BK = 8 * N, BYTES = EXT * 128, CPR = COLS ? EXT / N : 8;       // CPR: chunks per row of memory

  // LDS byte address of the chunk (row i, s = c * N ..) / (s, i = c * N ..)
  static __device__ __forceinline__ int addr_rows(int i, int c) { return i * 128 + ((c ^ (i & 7)) << 4); }
  static __device__ __forceinline__ int swz(int s) {
    if constexpr (sizeof(T) == 4) return EXT > 32 ? ((s >> 2) & 1) << 7 : 0;               // the two halves of a wave read rows four apart
    return (((s & 3) | ((s >> 1) & 4)) & (EXT / 16 - 1)) << 5;                            // the sixteen rows of a transposing read: eight 32-byte blocks
  }
  static __device__ __forceinline__ int addr_cols(int s, int byte) { return s * (EXT * (int)sizeof(T)) + (byte ^ swz(s)); }

  // chunk u of the tile, in the order of memory
  static __device__ __forceinline__ void put(char* lds, int u, V v) {
    *(V*)(lds + (COLS ? addr_cols(u / CPR, (u % CPR) * 16) : addr_rows(u / CPR, u % CPR))) = v;
  }
  // what lane l feeds in step c of the tile: row i0 + l % 32, the N summed elements (2 c + l / 32) * N ..
  static __device__ __forceinline__ V frag(const char* lds, int i0, int c) {
    const int l = threadIdx.x & 63, h = l >> 5;
    if constexpr (!COLS) {
      return *(const V*)(lds + addr_rows(i0 + (l & 31), 2 * c + h));
    } else if constexpr (sizeof(T) == 2) {
      // lane j of a group of sixteen names 4 elements of row s = j / 4, and receives column j of the group's 4 rows x 16 columns
      const int j = l & 15, s = (2 * c + h) * 8 + (j >> 2), byte = (i0 + (l & 16)) * 2 + (j & 3) * 8;
      typedef __attribute__((address_space(3))) s16x4* P;
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(lds + addr_cols(s, byte)));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(lds + addr_cols(s + 4, byte)));
      return __builtin_bit_cast(V, (s16x8)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      V v;
#pragma unroll
      for (int e = 0; e < N; e++) v[e] = *(const float*)(lds + addr_cols((2 * c + h) * 4 + e, (i0 + (l & 31)) * 4));
      return v;
    }
  }
};

// A thread's chunks of a tile on their way from memory to LDS, every one checked
template <class T, class S, bool COLS, int EXT, int THREADS>
struct GuardedLoader {
  typedef Lds<T, COLS, EXT> L;
  static constexpr int PER = EXT * 8 / THREADS;
  static_assert(EXT * 8 % THREADS == 0, "whole chunks per thread");
  typename L::V hold[PER];
  __device__ __forceinline__ void load(const Operand& o, int i0, int64_t s0, int64_t send) {
    const S* p = (const S*)o.p;
    if (i0 + (int64_t)EXT <= o.extent && s0 + L::BK <= send) {      // (uniform: a whole tile, nothing to check)
#pragma unroll
      for (int q = 0; q < PER; q++) {
        const int u = q * THREADS + (int)threadIdx.x, r = u / L::CPR, c = (u % L::CPR) * L::N;
        hold[q] = load_chunk<T, S>(p + (COLS ? (s0 + r) * o.ld + i0 : (i0 + r) * o.ld + s0), c, (int64_t)1 << 62, true);
      }
      return;
    }
#pragma unroll
    for (int q = 0; q < PER; q++) {
      const int u = q * THREADS + (int)threadIdx.x, r = u / L::CPR, c = (u % L::CPR) * L::N;
      if constexpr (!COLS) hold[q] = load_chunk<T, S>(p + (int64_t)(i0 + r) * o.ld, s0 + c, send, i0 + r < o.extent);
      else hold[q] = load_chunk<T, S>(p + (s0 + r) * o.ld, (int64_t)i0 + c, o.extent, s0 + r < send);
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int q = 0; q < PER; q++) L::put(lds, q * THREADS + (int)threadIdx.x, hold[q]);
  }
};

// The same without checks: the tile lies inside the operand.  One 32-bit offset per thread (the host has checked that a tile spans less than 2 GiB); what
// differs between a thread's chunks and between tiles is uniform.
template <class T, class S, bool COLS, int EXT, int THREADS>
struct Loader {
  typedef Lds<T, COLS, EXT> L;
  static constexpr int PER = EXT * 8 / THREADS, N = L::N, BK = L::BK;
  static_assert(EXT * 8 % THREADS == 0 && THREADS % L::CPR == 0, "whole chunks and rows per pass of the threads");
  typedef uint8_t Bytes __attribute__((ext_vector_type(N)));
  typedef std::conditional_t<sizeof(S) == 1, Bytes, typename L::V> Raw;
  Raw hold[PER];
  const char* base;            // of the tile that is loaded next
  int64_t pass, step;          // bytes between a thread's chunks, and between tiles
  uint32_t off;
  __device__ __forceinline__ void start(const Operand& o, int i0, int64_t s0) {
    const int r = (int)threadIdx.x / L::CPR, c = (int)threadIdx.x % L::CPR;
    off = (uint32_t)(r * (int)(o.ld * sizeof(S)) + c * (int)(N * sizeof(S)));
    pass = (int64_t)(THREADS / L::CPR) * o.ld * sizeof(S);
    step = (COLS ? BK * o.ld : BK) * (int64_t)sizeof(S);
    base = (const char*)o.p + (COLS ? s0 * o.ld + i0 : (int64_t)i0 * o.ld + s0) * (int64_t)sizeof(S);
  }
  __device__ __forceinline__ void back(const Operand& o, int64_t by) { base -= (COLS ? by * o.ld : by) * (int64_t)sizeof(S); }
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int q = 0; q < PER; q++) __builtin_memcpy(&hold[q], base + q * pass + off, sizeof(Raw));
    base += step;
  }
  // done: so many leading elements of the summed axis were summed before
  __device__ __forceinline__ void store(char* lds, int done) const {
#pragma unroll
    for (int q = 0; q < PER; q++) {
      const int u = q * THREADS + (int)threadIdx.x;
      typename L::V v;
      if constexpr (sizeof(S) == 1) {
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = (T)(float)hold[q][e];
      } else v = hold[q];
      if (done) {
        const int at = COLS ? u / L::CPR : (u % L::CPR) * N;
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = at + (COLS ? 0 : e) < done ? (T)0.0f : v[e];
      }
      L::put(lds, u, v);
    }
  }
};

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f32x4 a, f32x4 b, f32x16 c) {   // both operands deal the summed index alike, so its order does not matter
#pragma unroll
  for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// one element of the result; the sum comes in 32 bits and each result is rounded to T once
template <class T>
__device__ __forceinline__ void finish(const Epilogue& e, int64_t i, int64_t j, int64_t n, float v) {
  if (e.b) v += (float)((const T*)e.b)[j];
  if (e.z) {
    if (e.act == MG_ACTIVATION_TANH_Z32) ((float*)e.z)[i * n + j] = v;
    else ((T*)e.z)[i * n + j] = (T)v;
  }
  v = activate(e.act, v);
  if (e.r) v += (float)((const T*)e.r)[i * e.ldr + j];
  ((T*)e.c)[i * e.ldc + j] = (T)v;
}

// W neighbours of a row at any alignment, those from `skip` up to `count`
template <class T, int W>
__device__ __forceinline__ void store_some(T* p, const float (&v)[W], int skip, int count) {
  T t[W];
#pragma unroll
  for (int u = 0; u < W; u++) t[u] = (T)v[u];
  if (skip <= 0 && count >= W) __builtin_memcpy(p, t, sizeof t);
  else
#pragma unroll
    for (int u = 0; u < W; u++)
      if (u >= skip && u < count) p[u] = t[u];
}
template <class T, int W>
__device__ __forceinline__ void load_row(const T* p, T (&t)[W], int skip, int count) {
  if (skip <= 0 && count >= W) __builtin_memcpy(t, p, sizeof t);
  else
#pragma unroll
    for (int u = 0; u < W; u++) t[u] = u >= skip && u < count ? p[u] : (T)0.0f;
}

// Workgroups go to the eight XCDs in turn: each XCD takes one contiguous run of tiles, ordered in bands of eight tile rows with the row running fastest, so
// that what is multiplied at the same time on an XCD is a block of tiles that shares rows of both operands in its L2.
struct TileAt { int i, j; };
__device__ __forceinline__ TileAt tile_at(int ti, int tj) {
  const int tiles = gridDim.x, x = blockIdx.x & 7, run = tiles >> 3, more = tiles & 7;
  const int t = x * run + min(x, more) + ((int)blockIdx.x >> 3);
  const int band = t / (8 * tj), in = t - band * 8 * tj, high = min(8, ti - band * 8);
  return {band * 8 + in % high, in / high};
}

// Lane l holds column l % 32 and rows 8 (q / 4) + 4 (l / 32) + q % 4 of a 32 x 32 block.  The sums pass through LDS, 32 rows of a wave at a time, so
// that a lane ends with eight neighbours of one row: 16-byte accesses, whole lines.  (Row stride + 8: the two halves of a wave write disjoint banks.)  A lane
// keeps its columns, so their bias is loaded once; its rows go by in groups of G, the residual of the next group on its way while one is finished.  (The
// groups are a loop: unrolled, an activation's code alone would be larger than the instruction cache.)  Rows below iown and columns below jown belong to
// a neighbour.
template <class T, int ACT, int MI, int MJ>
__device__ __forceinline__ void store_tile(const Epilogue& ep, f32x16 (&acc)[MI][MJ], float* stage, int64_t i0, int64_t iown, int64_t rows, int64_t j0, int64_t jown, int64_t n) {
  constexpr int W = 8, STRIDE = MJ * 32 + 8, LPR = MJ * 32 / W, RPP = 64 / LPR, P = 32 / RPP, G = P < 2 ? 1 : 2;
  const int l = threadIdx.x & 63, r0 = l / LPR, col = (l % LPR) * W;
  const int64_t j = j0 + col;
  const int count = (int)min((int64_t)W, n - j), skip = (int)min((int64_t)W, jown - j);
  const bool some = count > 0 && skip < W;
  float bias[W];
#pragma unroll
  for (int u = 0; u < W; u++) bias[u] = 0.0f;
  if (ep.b && !ep.part && some) {
    T t[W];
    load_row<T, W>((const T*)ep.b + j, t, skip, count);
#pragma unroll
    for (int u = 0; u < W; u++) bias[u] = (float)t[u];
  }
  const bool residual = ep.r && !ep.part && some;
  T next[G][W];
  auto residuals = [&](int p) {                                  // of the group that starts with the p-th of this lane's rows
    if (residual)
#pragma unroll
      for (int u = 0; u < G; u++) {
        const int64_t i = i0 + (p + u) * RPP + r0;
        if (i >= iown && i < rows) load_row<T, W>((const T*)ep.r + i * ep.ldr + j, next[u], skip, count);
      }
  };
  residuals(0);
#pragma unroll
  for (int a = 0; a < MI; a++) {
#pragma unroll
    for (int b = 0; b < MJ; b++)
#pragma unroll
      for (int q = 0; q < 16; q++) stage[(8 * (q >> 2) + 4 * (l >> 5) + (q & 3)) * STRIDE + b * 32 + (l & 31)] = acc[a][b][q];
    __builtin_amdgcn_wave_barrier();                             // (a wave's LDS operations happen in order)
#pragma unroll 1
    for (int p = 0; p < P; p += G) {
      float v[G][W];
      T res[G][W];
#pragma unroll
      for (int u = 0; u < G; u++) {
        __builtin_memcpy(v[u], __builtin_assume_aligned(stage + ((p + u) * RPP + r0) * STRIDE + col, 16), sizeof v[u]);
        __builtin_memcpy(res[u], next[u], sizeof res[u]);
      }
      if (a * P + p + G < MI * P) residuals(a * P + p + G);
#pragma unroll
      for (int u = 0; u < G; u++) {
        const int64_t i = i0 + (a * P + p + u) * RPP + r0;
        if (!some || i < iown || i >= rows) continue;
        if (ep.part) {
          store_some<float, W>(ep.part + ((int64_t)blockIdx.y * rows + i) * n + j, v[u], skip, count);
          continue;
        }
#pragma unroll
        for (int e = 0; e < W; e++) v[u][e] += bias[e];
        if (ep.z) store_some<KeptOf<T, ACT>, W>((KeptOf<T, ACT>*)ep.z + i * n + j, v[u], skip, count);
#pragma unroll
        for (int e = 0; e < W; e++) v[u][e] = activate(ACT, v[u][e]);
        if (residual)
#pragma unroll
          for (int e = 0; e < W; e++) v[u][e] += (float)res[u][e];
        store_some<T, W>((T*)ep.c + i * ep.ldc + j, v[u], skip, count);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- the same where nothing has to be asked of a lane ----
// Aligned: every row of the result, the residual and z is 16-byte aligned and n a multiple of 8.  Memory is reached through buffer descriptors, and a lane
// that owns nothing (a tile that was moved back inside) has an offset outside of them.
constexpr uint32_t OUTSIDE = 0x80000000u;
struct Aligned {                 // rows of elements from (i, j) on
  __amdgpu_buffer_rsrc_t rsrc;
  uint32_t row;                  // bytes
  __device__ __forceinline__ Aligned(const void* p, int64_t i, int64_t j, int64_t ld, int size)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc((void*)((const char*)p + (i * ld + j) * size), 0, 0x7fffffff, 0x00027000)), row((uint32_t)(ld * size)) {}
  __device__ __forceinline__ u32x4 get(uint32_t lane, uint32_t at) const { return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, lane, at, 0)); }
  __device__ __forceinline__ void put(bool own, uint32_t lane, uint32_t at, u32x4 d) const { __builtin_amdgcn_raw_buffer_store_b128(d, rsrc, own ? lane : OUTSIDE, at, 0); }
};
// Inside: a whole tile at any alignment.  (Eight columns of which only the last are a tile's own are stored by its neighbour too: the same sums in the
// same order, so the same bits.)
struct Inside {
  char* base;
  uint32_t row;
  __device__ __forceinline__ Inside(const void* p, int64_t i, int64_t j, int64_t ld, int size) : base((char*)p + (i * ld + j) * size), row((uint32_t)(ld * size)) {}
  __device__ __forceinline__ u32x4 get(uint32_t lane, uint32_t at) const {
    u32x4 d;
    __builtin_memcpy(&d, base + at + lane, 16);
    return d;
  }
  __device__ __forceinline__ void put(bool own, uint32_t lane, uint32_t at, u32x4 d) const {
    if (own) __builtin_memcpy(base + at + lane, &d, 16);
  }
};

// The sums pass through LDS as in store_tile, up to 64 rows at a time, and a lane ends with the same eight columns of every (64 / LPR)-th row.  (A row's
// halves of 32 columns change places where bit 2 of the row is set: the two halves of a wave write disjoint banks.)  The residual is asked for before the
// first store, since a load behind a store would wait for the store.  Measured at 65 536 x 512 x 512 with gelu, z and residual: 115 -> 73 us.
// stage: the wave's own LDS; i0 / j0: where the wave's tile begins; iown / jown: the first row and column that it owns, counted from there
template <class T, int ACT, bool RES, class VIEW, int MI, int MJ>
__device__ __forceinline__ void store_wave(const Epilogue& ep, f32x16 (&acc)[MI][MJ], float* stage, int64_t i0, int iown, int64_t j0, int jown, int64_t rows, int64_t n) {
  typedef T V8 __attribute__((ext_vector_type(8)));
  constexpr int COLS = MJ * 32, LPR = COLS / 8, RPP = 64 / LPR, H = MI > 2 ? MI / 2 : 1, MH = MI / H, P = MH * 32 / RPP, SZ = sizeof(T), SWAP = MJ > 1 ? 32 : 0;
  const int l = threadIdx.x & 63, r0 = l / LPR, col = (l % LPR) * 8;
  const bool mine = col + 8 > jown;
  auto put_stage = [&](int h) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < MH; a++)
#pragma unroll
      for (int b = 0; b < MJ; b++)
#pragma unroll
        for (int q = 0; q < 16; q++) stage[(a * 32 + 8 * (q >> 2) + 4 * (l >> 5) + (q & 3)) * COLS + ((b * 32 + (l & 31)) ^ ((l >> 5) * SWAP))] = acc[h * MH + a][b][q];
    __builtin_amdgcn_wave_barrier();                             // (a wave's LDS operations happen in order)
  };
  auto staged = [&](int row) __attribute__((always_inline)) { return stage + row * COLS + (col ^ (((row >> 2) & 1) * SWAP)); };
  if (ep.part) {                                                 // 32-bit sums of a split: two 16-byte stores a row
    const VIEW part(ep.part + (int64_t)blockIdx.y * rows * n, i0, j0, n, 4);
    const uint32_t off = r0 * part.row + col * 4;
#pragma unroll
    for (int h = 0; h < H; h++) {
      put_stage(h);
#pragma unroll 4
      for (int p = 0; p < P; p++) {
        const int row = p * RPP + r0;
        u32x4 sums[2];
        __builtin_memcpy(sums, __builtin_assume_aligned(staged(row), 16), sizeof sums);
        const bool own = mine && h * MH * 32 + row >= iown;
        const uint32_t at = (h * P + p) * RPP * part.row;
        part.put(own, off, at, sums[0]);
        part.put(own, off + 16, at, sums[1]);
      }
      __builtin_amdgcn_wave_barrier();
    }
    return;
  }
  typedef KeptOf<T, ACT> Z;
  typedef Z Z8 __attribute__((ext_vector_type(8)));
  const VIEW c(ep.c, i0, j0, ep.ldc, SZ), z(ep.z, i0, j0, n, sizeof(Z)), r(ep.r, i0, j0, ep.ldr, SZ);
  float bias[8] = {};
  if (ep.b) {
    V8 t;
    __builtin_memcpy(&t, (const T*)ep.b + j0 + col, sizeof t);
#pragma unroll
    for (int e = 0; e < 8; e++) bias[e] = (float)t[e];
  }
  const uint32_t oc = r0 * c.row + col * SZ, oz = r0 * z.row + col * sizeof(Z);
  constexpr int W = SZ / 2;                                      // 16-byte words of eight elements
  // (as many rows as registers hold: all of them, of 32-bit elements a half)
  constexpr int AHEAD = SZ == 2 ? H * P : P;
  u32x4 res[RES ? AHEAD : 1][W];
  auto residuals = [&](int first) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < AHEAD; p++)
#pragma unroll
      for (int w = 0; w < W; w++) res[p][w] = r.get(r0 * r.row + col * SZ + w * 16, (first + p) * RPP * r.row);       // (rows and columns that are not its own lie inside too)
  };
  if constexpr (RES) residuals(0);
  auto put8 = [&](const VIEW& v, bool own, uint32_t lane, uint32_t at, const auto& t) __attribute__((always_inline)) {
    u32x4 d[sizeof t / 16];
    __builtin_memcpy(d, &t, sizeof d);
#pragma unroll
    for (int w = 0; w < (int)(sizeof t / 16); w++) v.put(own, lane + w * 16, at, d[w]);
  };
  auto finish_row = [&](int h, int p, const u32x4 (&residual)[W]) __attribute__((always_inline)) {
    const int row = p * RPP + r0;
    float v[8];
    __builtin_memcpy(v, __builtin_assume_aligned(staged(row), 16), sizeof v);
    const bool own = mine && h * MH * 32 + row >= iown;
    const uint32_t step = (h * P + p) * RPP;
    V8 t, add;
    __builtin_memcpy(&add, residual, sizeof add);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] += bias[e];
    if (ep.z) {
      Z8 kept;
#pragma unroll
      for (int e = 0; e < 8; e++) kept[e] = (Z)v[e];
      put8(z, own, oz, step * z.row, kept);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
      v[e] = activate(ACT, v[e]);
      if constexpr (RES) v[e] += (float)add[e];
      t[e] = (T)v[e];
    }
    put8(c, own, oc, step * c.row, t);
  };
#pragma unroll
  for (int h = 0; h < H; h++) {
    put_stage(h);
    if constexpr (RES) {
#pragma unroll
      for (int p = 0; p < P; p++) finish_row(h, p, res[(h * P + p) % AHEAD]);
      if (h + 1 < H && AHEAD < H * P) residuals((h + 1) * P);
    } else {
#pragma unroll 4
      for (int p = 0; p < P; p++) finish_row(h, p, res[0]);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <class T, bool PLAIN, class VIEW, int MI, int MJ>
__device__ __forceinline__ void store_wave_any(const Epilogue& ep, f32x16 (&acc)[MI][MJ], float* stage, int64_t i0, int iown, int64_t j0, int jown, int64_t rows, int64_t n) {
#define MG_ACT(A) \
  if (ep.r) store_wave<T, A, true, VIEW, MI, MJ>(ep, acc, stage, i0, iown, j0, jown, rows, n); \
  else store_wave<T, A, false, VIEW, MI, MJ>(ep, acc, stage, i0, iown, j0, jown, rows, n)
  if constexpr (!PLAIN) {
    switch (ep.part ? MG_ACTIVATION_NONE : ep.act) {
      case MG_ACTIVATION_RELU: MG_ACT(MG_ACTIVATION_RELU); return;
      case MG_ACTIVATION_TANH: MG_ACT(MG_ACTIVATION_TANH); return;
      case MG_ACTIVATION_TANH_Z32:                               // (32-bit operands: the same as tanh, which is asked for)
        if constexpr (sizeof(T) == 2) { MG_ACT(MG_ACTIVATION_TANH_Z32); }
        return;
      case MG_ACTIVATION_GELU: MG_ACT(MG_ACTIVATION_GELU); return;
      case MG_ACTIVATION_SILU: MG_ACT(MG_ACTIVATION_SILU); return;
      default: MG_ACT(MG_ACTIVATION_NONE); return;
    }
  } else {
    store_wave<T, MG_ACTIVATION_NONE, false, VIEW, MI, MJ>(ep, acc, stage, i0, iown, j0, jown, rows, n);
  }
#undef MG_ACT
}

template <class T, bool PLAIN, int MI, int MJ>
__device__ __forceinline__ void store_tile_any(const Epilogue& ep, f32x16 (&acc)[MI][MJ], float* stage, int64_t i0, int64_t iown, int64_t rows, int64_t j0, int64_t jown, int64_t n) {
#define MG_ACT(A) store_tile<T, A, MI, MJ>(ep, acc, stage, i0, iown, rows, j0, jown, n)
  if constexpr (!PLAIN) {
    switch (ep.part ? MG_ACTIVATION_NONE : ep.act) {
      case MG_ACTIVATION_RELU: MG_ACT(MG_ACTIVATION_RELU); return;
      case MG_ACTIVATION_TANH: MG_ACT(MG_ACTIVATION_TANH); return;
      case MG_ACTIVATION_TANH_Z32:                               // (32-bit operands: the same as tanh, which is asked for)
        if constexpr (sizeof(T) == 2) { MG_ACT(MG_ACTIVATION_TANH_Z32); }
        return;
      case MG_ACTIVATION_GELU: MG_ACT(MG_ACTIVATION_GELU); return;
      case MG_ACTIVATION_SILU: MG_ACT(MG_ACTIVATION_SILU); return;
      default: break;
    }
  }
  MG_ACT(MG_ACTIVATION_NONE);
#undef MG_ACT
}

template <class LA, class LB, int MI, int MJ>
__device__ __forceinline__ void multiply(const char* la, const char* lb, int wi, int wj, int c, f32x16 (&acc)[MI][MJ]) {
  typename LA::V fa[MI];
  typename LB::V fb[MJ];
#pragma unroll
  for (int a = 0; a < MI; a++) fa[a] = LA::frag(la, wi + a * 32, c);
#pragma unroll
  for (int b = 0; b < MJ; b++) fb[b] = LB::frag(lb, wj + b * 32, c);
#pragma unroll
  for (int a = 0; a < MI; a++)
#pragma unroll
    for (int b = 0; b < MJ; b++) acc[a][b] = mma(fa[a], fb[b], acc[a][b]);
}

// grid: (tiles, splits); WI x WJ waves of (BI / WI) x (BJ / WJ) each; A.extent >= BI, B.extent >= BJ, depth >= BK
template <class T, class SA, class SB, bool ACOLS, bool BCOLS, int BI, int BJ, int WI, int WJ>
__global__ __launch_bounds__(WI * WJ * 64) void k_product(Operand A, Operand B, int64_t depth, int32_t tiles_per_split, Epilogue ep) {
  constexpr int THREADS = WI * WJ * 64, MI = BI / WI / 32, MJ = BJ / WJ / 32;
  typedef Loader<T, SA, ACOLS, BI, THREADS> TA;
  typedef Loader<T, SB, BCOLS, BJ, THREADS> TB;
  typedef typename TA::L LA;
  typedef typename TB::L LB;
  constexpr int BK = LA::BK, BUF = LA::BYTES + LB::BYTES;
  __shared__ __attribute__((aligned(16))) char lds[2 * BUF];
  const TileAt at = tile_at((A.extent + BI - 1) / BI, (B.extent + BJ - 1) / BJ);
  const int i0 = min(at.i * BI, A.extent - BI), j0 = min(at.j * BJ, B.extent - BJ);
  const int64_t first = (int64_t)blockIdx.y * tiles_per_split, deep = (depth + BK - 1) / BK;
  const int tiles = (int)(min(deep, first + tiles_per_split) - first);
  // (the last tile of the axis, if it is not whole, starts `over` earlier)
  const int over = first + tiles == deep ? (int)(deep * BK - depth) : 0;
  const int wave = threadIdx.x >> 6, wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);

  f32x16 acc[MI][MJ];
#pragma unroll
  for (int a = 0; a < MI; a++)
#pragma unroll
    for (int b = 0; b < MJ; b++) acc[a][b] = (f32x16)(0.0f);

  TA ta;
  TB tb;
  ta.start(A, i0, first * BK);
  tb.start(B, j0, first * BK);
  auto fetch = [&](int t) {
    if (over && t == tiles - 1) { ta.back(A, over); tb.back(B, over); }
    ta.load();
    tb.load();
  };
  auto put = [&](int t) {
    char* p = lds + (t & 1) * BUF;
    const int done = t == tiles - 1 ? over : 0;
    ta.store(p, done);
    tb.store(p + LA::BYTES, done);
  };
  fetch(0);
  put(0);
  if (tiles > 1) fetch(1);
  __syncthreads();
  // while tile t is multiplied, tile t + 1 goes from registers to the other half of LDS and tile t + 2 is on its way from memory
  for (int t = 0; t < tiles; t++) {
    const char* la = lds + (t & 1) * BUF;
    const char* lb = la + LA::BYTES;
    multiply<LA, LB>(la, lb, wi, wj, 0, acc);
    multiply<LA, LB>(la, lb, wi, wj, 1, acc);
    if (t + 1 < tiles) put(t + 1);
    if (t + 2 < tiles) fetch(t + 2);
    multiply<LA, LB>(la, lb, wi, wj, 2, acc);
    multiply<LA, LB>(la, lb, wi, wj, 3, acc);
    __syncthreads();
  }
  static_assert(WI * WJ * 32 * (MJ * 32 + 8) * 4 <= (int)sizeof lds, "staging fits");
  constexpr int STAGED = (MI > 2 ? 64 : MI * 32) * MJ * 32;
  static_assert(WI * WJ * STAGED * 4 <= (int)sizeof lds, "staging fits");
  store_wave_any<T, BCOLS, Inside, MI, MJ>(ep, acc, (float*)lds + wave * STAGED, i0 + wi, at.i * BI - i0 - wi, j0 + wj, at.j * BJ - j0 - wj, A.extent, B.extent);
}

// An operand's tile from memory straight into LDS, 16 bytes a lane: no registers in between, and nothing waits for it but the wait that is written down.
// A wave's 64 chunks land one behind the other, so the swizzle is in which chunk a lane asks for.  Needs 16-byte aligned rows and tiles (the host checks).
template <class T, bool COLS, int EXT, int THREADS>
struct DirectLoader {
  typedef Lds<T, COLS, EXT> L;
  static constexpr int PER = EXT * 8 / THREADS, RPP = THREADS / L::CPR;      // RPP: memory rows per pass of the threads
  static_assert(sizeof(T) == 2 && EXT == 256 && (!COLS || RPP == 8 || RPP == 16), "the swizzle below");
  const char* base;            // of the tile that is loaded next
  int64_t pass, step;
  uint32_t off[2];             // (cols: bit 3 of a tile row is the parity of the pass where a pass has 8 rows)
  __device__ __forceinline__ void start(const Operand& o, int i0, int64_t s0) {
    const int r = (int)threadIdx.x / L::CPR, p = (int)threadIdx.x % L::CPR;
#pragma unroll
    for (int q = 0; q < 2; q++) {
      const int at = COLS ? (p * 16) ^ L::swz(r + q * RPP) : (p ^ (r & 7)) * 16;
      off[q] = (uint32_t)(r * (int)(o.ld * 2) + at);
    }
    pass = (int64_t)RPP * o.ld * 2;
    step = (COLS ? L::BK * o.ld : L::BK) * 2;
    base = (const char*)o.p + (COLS ? s0 * o.ld + i0 : (int64_t)i0 * o.ld + s0) * 2;
  }
  // pass q of the tile at LDS byte address lds (uniform, like the wave's number)
  __device__ __forceinline__ void load(int q, uint32_t lds, int wave) {
    const uint32_t at = lds + q * (THREADS * 16) + wave * 1024;
    // (m0 is named so that nothing of the compiler's is expected to outlive the statement in it; it warns that it saves no such register for us, which nothing asks for)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(off[COLS ? q & 1 : 0]), "s"(base + q * pass) : "memory", "m0");
#pragma clang diagnostic pop
  }
  __device__ __forceinline__ void advance() { base += step; }
};

// The 256-tile where every row is 16-byte aligned: four waves of 128 x 128, so that a fragment read from LDS feeds four matrix instructions (what a CU reads
// from LDS takes half as long as what it multiplies; with eight waves of 128 x 64 the two take the same time).  One wave per SIMD: the fragments of a step
// are read while the step before is multiplied, and the tile after next is on its way to LDS from the moment its buffer is free.  One barrier per tile: it
// stands where the last fragments of tile t have been read and tile t + 1 has landed.
template <class T, bool ACOLS, bool BCOLS>
__global__ __launch_bounds__(256, 1) void k_product_direct(Operand A, Operand B, int64_t depth, int32_t tiles_per_split, Epilogue ep) {
  constexpr int BI = 256, BJ = 256, THREADS = 256, MI = 4, MJ = 4;
  typedef DirectLoader<T, ACOLS, BI, THREADS> TA;
  typedef DirectLoader<T, BCOLS, BJ, THREADS> TB;
  typedef typename TA::L LA;
  typedef typename TB::L LB;
  constexpr int BK = LA::BK, BUF = LA::BYTES + LB::BYTES;
  __shared__ __attribute__((aligned(1024))) char lds[2 * BUF];
  const TileAt at = tile_at((A.extent + BI - 1) / BI, (B.extent + BJ - 1) / BJ);
  const int i0 = min(at.i * BI, A.extent - BI), j0 = min(at.j * BJ, B.extent - BJ);
  const int64_t first = (int64_t)blockIdx.y * tiles_per_split, last = min((depth + BK - 1) / BK, first + tiles_per_split);
  const int tiles = (int)(min(depth / BK, last) - first);          // whole tiles; what is left of the axis comes behind them
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = (wave >> 1) * 128, wj = (wave & 1) * 128;
  const uint32_t l0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

  f32x16 acc[MI][MJ];
#pragma unroll
  for (int a = 0; a < MI; a++)
#pragma unroll
    for (int b = 0; b < MJ; b++) acc[a][b] = (f32x16)(0.0f);

  TA ta;
  TB tb;
  ta.start(A, i0, first * BK);
  tb.start(B, j0, first * BK);
  typename LA::V fa[2][MI];
  typename LB::V fb[2][MJ];
  auto read = [&](int s, const char* p, int c, int u) __attribute__((always_inline)) {
    fa[s][u] = LA::frag(p, wi + u * 32, c);
    fb[s][u] = LB::frag(p + LA::BYTES, wj + u * 32, c);
  };
  // a pass of both operands' next tile, numbered through
  auto fetch = [&](int q, int t) __attribute__((always_inline)) {
    const uint32_t p = l0 + (t & 1) * BUF;
    if (q < TA::PER) ta.load(q, p, wave);
    else tb.load(q - TA::PER, p + LA::BYTES, wave);
    if (q == TA::PER - 1) ta.advance();
    if (q == TA::PER + TB::PER - 1) tb.advance();
  };
  constexpr int PASSES = TA::PER + TB::PER, SLOTS = 8;
  // A step: 16 matrix instructions, four at a time, between them the reads of the next step's fragments and, over two steps, the passes that bring the tile
  // after next.  Measured at 32 768 x 2048 x 4096 (dx): all passes one behind the other 608 us (the wave waits for the memory pipe to take them), over four
  // groups 496, over eight 460, over twelve 468 (the last ones land late).
  auto step = [&](int s, bool reads, const char* p, int c, int slot, bool fetches, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 4; u++) {
      if (reads) read(s ^ 1, p, c, u);
      if (fetches && slot >= 0)
#pragma unroll
        for (int q = 0; q < PASSES; q++)
          if (q >= (slot + u) * PASSES / SLOTS && q < (slot + u + 1) * PASSES / SLOTS) fetch(q, t);
#pragma unroll
      for (int b = 0; b < MJ; b++) acc[u][b] = mma(fa[s][u], fb[s][b], acc[u][b]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // tile t; `ahead`: the tile behind it exists; rest / begin: tile t + 1's later passes and tile t + 2's first ones are due
  auto tile = [&](int t, bool ahead, bool rest, bool begin) __attribute__((always_inline)) {
    const char* p = lds + (t & 1) * BUF;
    const char* n = lds + ((t + 1) & 1) * BUF;
    step(0, true, p, 1, 4, rest, t + 1);
    step(1, true, p, 2, -1, false, 0);
    step(0, true, p, 3, -1, false, 0);
    // (the last fragments are in registers, the next tile has landed, and every wave has come as far)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    step(1, ahead, n, 0, 0, begin, t + 2);
  };
  if (tiles > 0) {
#pragma unroll
    for (int q = 0; q < PASSES; q++) fetch(q, 0);
    if (tiles > 1) {
#pragma unroll
      for (int q = 0; q < PASSES / 2; q++) fetch(q, 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PASSES / 2) : "memory");
    }
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int u = 0; u < 4; u++) read(0, lds, 0, u);
    int t = 0;
    for (; t + 2 < tiles; t++) tile(t, true, true, true);
    if (t + 1 < tiles) tile(t++, true, true, false);
    tile(t, false, false, false);
  }
  if (first + tiles < last) {                                      // the last piece of the axis, loaded as the last whole one; what was summed is zeroed
    const int over = (int)(last * BK - depth);
    Loader<T, T, ACOLS, BI, THREADS> ra;
    Loader<T, T, BCOLS, BJ, THREADS> rb;
    ra.start(A, i0, depth - BK);
    ra.load();
    ra.store(lds, over);
    rb.start(B, j0, depth - BK);
    rb.load();
    rb.store(lds + LA::BYTES, over);
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 4; c++) {
#pragma unroll
      for (int u = 0; u < 4; u++) read(0, lds, c, u);
      step(0, false, lds, 0, -1, false, 0);
    }
    __syncthreads();
  }
  static_assert(2 * BUF == 4 * 64 * 128 * 4, "staging fits");
  store_wave_any<T, BCOLS, Aligned, MI, MJ>(ep, acc, (float*)lds + wave * 64 * 128, i0 + wi, at.i * BI - i0 - wi, j0 + wj, at.j * BJ - j0 - wj, A.extent, B.extent);
}

template <class T, class SA, class SB, bool ACOLS, bool BCOLS, int BI, int BJ, int WI, int WJ>
__global__ __launch_bounds__(WI * WJ * 64) void k_product_guarded(Operand A, Operand B, int64_t depth, int32_t tiles_per_split, Epilogue ep) {
  constexpr int THREADS = WI * WJ * 64, MI = BI / WI / 32, MJ = BJ / WJ / 32;
  typedef GuardedLoader<T, SA, ACOLS, BI, THREADS> TA;
  typedef GuardedLoader<T, SB, BCOLS, BJ, THREADS> TB;
  typedef typename TA::L LA;
  typedef typename TB::L LB;
  constexpr int BK = LA::BK, BUF = LA::BYTES + LB::BYTES;
  __shared__ __attribute__((aligned(16))) char lds[2 * BUF];
  const TileAt at = tile_at((A.extent + BI - 1) / BI, (B.extent + BJ - 1) / BJ);
  // (whole tiles where there are some: the last ones are moved back inside)
  const bool whole = A.extent >= BI && B.extent >= BJ && ep.narrow;
  const int i0 = whole ? min(at.i * BI, A.extent - BI) : at.i * BI, j0 = whole ? min(at.j * BJ, B.extent - BJ) : at.j * BJ;
  const int64_t s_begin = (int64_t)blockIdx.y * tiles_per_split * BK, s_end = min(depth, s_begin + (int64_t)tiles_per_split * BK);
  const int wave = threadIdx.x >> 6, wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);
  f32x16 acc[MI][MJ];
#pragma unroll
  for (int a = 0; a < MI; a++)
#pragma unroll
    for (int b = 0; b < MJ; b++) acc[a][b] = (f32x16)(0.0f);
  TA ta;
  TB tb;
  ta.load(A, i0, s_begin, s_end);
  tb.load(B, j0, s_begin, s_end);
  int cur = 0;
  for (int64_t s = s_begin; s < s_end; s += BK) {
    char* la = lds + cur * BUF;
    char* lb = la + LA::BYTES;
    ta.store(la);
    tb.store(lb);
    if (s + BK < s_end) {
      ta.load(A, i0, s + BK, s_end);
      tb.load(B, j0, s + BK, s_end);
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 4; c++) multiply<LA, LB>(la, lb, wi, wj, c, acc);
    cur ^= 1;
  }
  __syncthreads();
  constexpr int STAGED = (MI > 2 ? 64 : MI * 32) * MJ * 32;
  static_assert(WI * WJ * STAGED * 4 <= (int)sizeof lds && WI * WJ * 32 * (MJ * 32 + 8) * 4 <= (int)sizeof lds, "staging fits");
  if (whole) {
    store_wave_any<T, BCOLS, Inside, MI, MJ>(ep, acc, (float*)lds + wave * STAGED, i0 + wi, at.i * BI - i0 - wi, j0 + wj, at.j * BJ - j0 - wj, A.extent, B.extent);
    return;
  }
  float* stage = (float*)lds + wave * 32 * (MJ * 32 + 8);
  store_tile_any<T, BCOLS, MI, MJ>(ep, acc, stage, i0 + wi, 0, A.extent, j0 + wj, 0, B.extent);
}

// Few rows (a step of a handful of environments): a wave per result column, its lanes along k in chunks of 16 bytes of the weight, one sum per row and lane,
// joined over the lanes at the end.  Bound by the weight's bytes where it is large, by one trip to memory and back where it is small.
template <class T, class S, int ROWS>
__global__ __launch_bounds__(256) void k_few_rows(int rows, int64_t k, int64_t n, const S* x, int64_t ldx, const T* w, int64_t ldw, Epilogue ep) {
  constexpr int N = Chunk<T>::N;
  const int lane = threadIdx.x & 63;
  for (int64_t j = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); j < n; j += (int64_t)gridDim.x * 4) {
    const T* wj = w + j * ldw;
    float s[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) s[i] = 0.0f;
    for (int64_t c = (int64_t)lane * N; c < k; c += 64 * N) {
      const auto b = load_chunk<T, T>(wj, c, k, true);
#pragma unroll
      for (int i = 0; i < ROWS; i++) {
        if (i < rows) {
          const auto a = load_chunk<T, S>(x + i * ldx, c, k, true);
#pragma unroll
          for (int e = 0; e < N; e++) s[i] = __builtin_fmaf((float)a[e], (float)b[e], s[i]);
        }
      }
    }
    float mine = 0.0f;
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
#pragma unroll
      for (int m = 32; m; m >>= 1) s[i] += __shfl_xor(s[i], m);
      mine = lane == i ? s[i] : mine;
    }
    if (lane < rows) finish<T>(ep, lane, j, n, mine);
  }
}

// The splits' sums, added in an order that the sizes fix, and the epilogue.  A workgroup takes 256 neighbouring results: a wave reads a quarter of the splits,
// four results a lane, and the four sums of a result meet in LDS.
template <class T>
__global__ __launch_bounds__(256) void k_join(int64_t total, int64_t n, int splits, Epilogue ep) {
  __shared__ float sum[4][256];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int64_t u0 = (int64_t)blockIdx.x * 256; u0 < total; u0 += (int64_t)gridDim.x * 256) {
    const int64_t u = u0 + lane * 4;
    f32x4 s = (f32x4)(0.0f);
    if (u + 4 <= total) {
#pragma unroll 4
      for (int q = w; q < splits; q += 4) {
        f32x4 v;
        __builtin_memcpy(&v, ep.part + (int64_t)q * total + u, 16);
        s += v;
      }
    } else {
      for (int q = w; q < splits; q += 4)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (u + e < total) s[e] += ep.part[(int64_t)q * total + u + e];
    }
    *(f32x4*)&sum[w][lane * 4] = s;
    __syncthreads();
    const int64_t at = u0 + threadIdx.x;
    if (at < total) {
      finish<T>(ep, at / n, at % n, n, (sum[0][threadIdx.x] + sum[1][threadIdx.x]) + (sum[2][threadIdx.x] + sum[3][threadIdx.x]));
    }
    __syncthreads();
  }
}

// ---- what mg_linear.hip asks of the translation unit of a type ----
enum { TILE_GUARDED_32_128, TILE_GUARDED_128_32, TILE_GUARDED_128_128, TILE_64, TILE_128, TILE_256, TILE_DIRECT, TILES };
enum { FORM_FORWARD, FORM_DX, FORM_DW };          // A rows B rows, A rows B cols, A cols B cols
struct Plan {
  int tile, splits, per;       // how many ways the summed axis is split, tiles of that axis per split
  int64_t part_bytes;
};
constexpr int TILE_I[TILES] = {32, 128, 128, 64, 128, 256, 256}, TILE_J[TILES] = {128, 32, 128, 64, 128, 256, 256};
constexpr int FEW_ROWS = 8;
template <class T> struct Linear {
  static void product(hipStream_t st, int form, bool bytes, const Plan& p, const Operand& A, const Operand& B, int64_t depth, const Epilogue& ep);
  static void few_rows(hipStream_t st, bool bytes, int rows, int64_t k, int64_t n, const void* x, int64_t ldx, const void* w, int64_t ldw, const Epilogue& ep);
  static void join(hipStream_t st, int64_t rows, int64_t n, int splits, const Epilogue& ep);
  static void dz(hipStream_t st, int act, int64_t rows, int64_t n, const void* dy, int64_t lddy, const void* z, void* dz, void* db, float* part);
};
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// dz = dy act'(z) and the column sums of dz: a workgroup takes `lanes` chunks of eight columns and every 256 / lanes-th row of a run
struct DzPlan { int lanes_log2; int64_t strips, run, runs; };
inline DzPlan dz_plan(int64_t rows, int64_t n) {
  DzPlan p;
  const int64_t chunks = ceil_div(n, 8);
  p.lanes_log2 = 0;
  while (p.lanes_log2 < 6 && (1 << p.lanes_log2) < chunks) p.lanes_log2++;
  p.strips = ceil_div(chunks, 1 << p.lanes_log2);
  // about four workgroups a CU, each with at least four rows a thread
  const int64_t runs = std::max<int64_t>(1, 1024 / p.strips), least = 4 * (256 >> p.lanes_log2);
  p.run = std::max<int64_t>(least, ceil_div(std::max<int64_t>(rows, 1), runs));
  p.runs = ceil_div(std::max<int64_t>(rows, 1), p.run);
  return p;
}

}  // namespace mgo
