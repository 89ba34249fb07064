// mg_linear.h — the tile product behind the linear layer and its two gradients, for gfx950's matrix instructions.
//
//   C (i, j) = sum_s A(i, s) B(j, s)
//     forward      A = x (rows, k),  B = w (n, k)      both contiguous along s            y = act(C + b) + r
//     dx = dz w    A = dz (rows, n), B(j, s) = w[s][j] B contiguous along j
//     dw = dzT x   A(i, s) = dz[s][i], B(j, s) = x[s][j]: both contiguous along i / j
//
// An operand that is contiguous along s ("rows") lies in LDS as 128-byte rows of one tile row each; one that is contiguous along i / j ("cols") lies
// there as one row per s and is turned by the transposing LDS read (16-bit types) or read element by element (f32).  Both are swizzled so that the
// fragment reads of a wave spread over all banks.  Global loads go through registers: they may be unaligned, partial (guarded), or bytes that are
// widened on the way.  The loads of tile t + 1 are in flight while tile t is multiplied (two LDS buffers, one barrier per tile).
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
  void* z;         // values in front of the activation (contiguous), or null
  float* part;     // split sums: f32 (splits, rows, n), contiguous; null = store the result
  int64_t ldr, ldc;
  int32_t act;
  int32_t wide;    // n and every row stride divide by 8 and every pointer by 16 bytes
};

// ---- activations ----
// exp2 with a result of 0 far below the smallest number: v_exp_f32, one ulp
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }

// The normal distribution function at -|x|: e^{-x^2/2} q(t), t = 1 / (1 + 0.3 |x|).  q is 0.5 erfcx(|x| / sqrt 2) as a polynomial of degree 8 without a
// constant term, fitted here for the least largest RELATIVE error on |x| <= 13.5 (1.3e-7; 2.9e-7 evaluated in 32 bits); beyond, e^{-x^2/2} is 0 in f32.
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
    case MG_ACTIVATION_TANH: return tanh_act(z);
    case MG_ACTIVATION_GELU: {
      float d;
      const float t = phi_tail(fabsf(z), &d);
      return z * (z < 0.0f ? t : 1.0f - t);
    }
    case MG_ACTIVATION_SILU: return z * rcp_fast(1.0f + exp2_fast(z * -1.44269504f));
    default: return z;
  }
}

__device__ __forceinline__ float activate_grad(int act, float z) {
  switch (act) {
    case MG_ACTIVATION_RELU: return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
    case MG_ACTIVATION_TANH: {
      const float t = tanh_act(z), e = exp2_fast(fabsf(z) * (-2.0f * 1.44269504f)), q = rcp_fast(1.0f + e);
      return fabsf(z) < 0.3f ? 1.0f - t * t : 4.0f * e * q * q;                // 1 - tanh^2 = 4 e^{-2|z|} / (1 + e^{-2|z|})^2
    }
    case MG_ACTIVATION_GELU: {
      float d;
      const float t = phi_tail(fabsf(z), &d);
      return (z < 0.0f ? t : 1.0f - t) + z * d;
    }
    case MG_ACTIVATION_SILU: {
      const float p = rcp_fast(1.0f + exp2_fast(z * -1.44269504f));
      return p * __builtin_fmaf(z, 1.0f - p, 1.0f);
    }
    default: return 1.0f;
  }
}

// ---- global loads ----
// N consecutive elements of a memory row as T, element e valid where at + e < end; VEC: 16-byte aligned and never partial
template <class T, class S, bool VEC>
__device__ __forceinline__ typename Chunk<T>::V load_chunk(const S* row, int64_t at, int64_t end, bool inside) {
  constexpr int N = Chunk<T>::N;
  typename Chunk<T>::V v = {};
  if (!inside || at >= end) return v;
  if constexpr (sizeof(S) == sizeof(T)) {
    if (VEC || at + N <= end) {
      __builtin_memcpy(&v, VEC ? __builtin_assume_aligned(row + at, 16) : (const void*)(row + at), 16);
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
template <class T, class S, bool COLS, bool VEC, int EXT, int THREADS>
struct Tile {
  typedef typename Chunk<T>::V V;
  static constexpr int N = Chunk<T>::N, BK = 8 * N, BYTES = EXT * 128, PER = EXT * 8 / THREADS;
  static_assert(EXT * 8 % THREADS == 0, "whole chunks per thread");
  V hold[PER];

  // LDS byte address of the chunk (row i, s = c * N ..) / (s, i = c * N ..)
  static __device__ __forceinline__ int addr_rows(int i, int c) { return i * 128 + ((c ^ (i & 7)) << 4); }
  static __device__ __forceinline__ int swz(int s) {
    if constexpr (sizeof(T) == 4) return EXT > 32 ? ((s >> 2) & 1) << 7 : 0;               // the two halves of a wave read rows four apart
    return (((s & 3) | ((s >> 1) & 4)) & (EXT / 16 - 1)) << 5;                            // the sixteen rows of a transposing read: eight 32-byte blocks
  }
  static __device__ __forceinline__ int addr_cols(int s, int byte) { return s * (EXT * (int)sizeof(T)) + (byte ^ swz(s)); }

  __device__ __forceinline__ void load(const Operand& o, int i0, int64_t s0, int64_t send) {
    const S* p = (const S*)o.p;
#pragma unroll
    for (int q = 0; q < PER; q++) {
      const int u = q * THREADS + (int)threadIdx.x;
      if constexpr (!COLS) {
        const int i = u >> 3, c = u & 7;
        hold[q] = load_chunk<T, S, VEC>(p + (int64_t)(i0 + i) * o.ld, s0 + c * N, send, i0 + i < o.extent);
      } else {
        constexpr int CPR = EXT / N;                      // chunks per row of memory
        const int s = u / CPR, c = u % CPR;
        hold[q] = load_chunk<T, S, VEC>(p + (s0 + s) * o.ld, (int64_t)i0 + c * N, o.extent, s0 + s < send);
      }
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int q = 0; q < PER; q++) {
      const int u = q * THREADS + (int)threadIdx.x;
      int a;
      if constexpr (!COLS) a = addr_rows(u >> 3, u & 7);
      else { constexpr int CPR = EXT / N; a = addr_cols(u / CPR, (u % CPR) * 16); }
      *(V*)(lds + a) = hold[q];
    }
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

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f32x4 a, f32x4 b, f32x16 c) {   // both operands deal the summed index alike, so its order does not matter
#pragma unroll
  for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// W consecutive elements (i, j ..) of the result, `count` of them inside; the sums come in 32 bits and each result is rounded to T once.  WIDE: all of
// them inside and every row 16-byte aligned.
template <class T, int W, bool WIDE>
__device__ __forceinline__ void finish(const Epilogue& e, int64_t i, int64_t j, int64_t n, int count, float (&v)[W]) {
  T t[W];
  if (e.b) {
#pragma unroll
    for (int u = 0; u < W; u++)
      if (WIDE || u < count) v[u] += (float)((const T*)e.b)[j + u];
  }
  if (e.z) {
    T* z = (T*)e.z + i * n + j;
#pragma unroll
    for (int u = 0; u < W; u++) t[u] = (T)v[u];
    if constexpr (WIDE) __builtin_memcpy(__builtin_assume_aligned(z, 16), t, sizeof t);
    else
#pragma unroll
      for (int u = 0; u < W; u++)
        if (u < count) z[u] = t[u];
  }
  switch (e.act) {
#define MG_ACT(A) case A: _Pragma("unroll") for (int u = 0; u < W; u++) v[u] = activate(A, v[u]); break;
    MG_ACT(MG_ACTIVATION_RELU) MG_ACT(MG_ACTIVATION_TANH) MG_ACT(MG_ACTIVATION_GELU) MG_ACT(MG_ACTIVATION_SILU)
#undef MG_ACT
    default: break;
  }
  if (e.r) {
    const T* r = (const T*)e.r + i * e.ldr + j;
    if constexpr (WIDE) {
      __builtin_memcpy(t, __builtin_assume_aligned(r, 16), sizeof t);
#pragma unroll
      for (int u = 0; u < W; u++) v[u] += (float)t[u];
    } else {
#pragma unroll
      for (int u = 0; u < W; u++)
        if (u < count) v[u] += (float)r[u];
    }
  }
  T* c = (T*)e.c + i * e.ldc + j;
#pragma unroll
  for (int u = 0; u < W; u++) t[u] = (T)v[u];
  if constexpr (WIDE) __builtin_memcpy(__builtin_assume_aligned(c, 16), t, sizeof t);
  else
#pragma unroll
    for (int u = 0; u < W; u++)
      if (u < count) c[u] = t[u];
}

// grid: (tiles, splits); WI x WJ waves of (BI / WI) x (BJ / WJ) each
template <class T, class SA, class SB, bool ACOLS, bool BCOLS, bool VEC, int BI, int BJ, int WI, int WJ>
__global__ __launch_bounds__(WI * WJ * 64) void k_product(Operand A, Operand B, int64_t depth, int32_t depth_tiles_per_split, Epilogue ep) {
  constexpr int THREADS = WI * WJ * 64, MI = BI / WI / 32, MJ = BJ / WJ / 32;
  typedef Tile<T, SA, ACOLS, VEC, BI, THREADS> TA;
  typedef Tile<T, SB, BCOLS, VEC, BJ, THREADS> TB;
  constexpr int BK = TA::BK;
  __shared__ __attribute__((aligned(16))) char lds[2 * (TA::BYTES + TB::BYTES)];

  // workgroups go to the eight XCDs in turn: each XCD takes one contiguous run of tiles (j fastest), so that what shares rows of A shares an L2
  const int tj = (B.extent + BJ - 1) / BJ, tiles = gridDim.x;
  int t = blockIdx.x;
  {
    const int x = t & 7, run = tiles >> 3, more = tiles & 7;
    t = x * run + min(x, more) + (t >> 3);
  }
  const int i0 = (t / tj) * BI, j0 = (t % tj) * BJ;
  const int64_t s_begin = (int64_t)blockIdx.y * depth_tiles_per_split * BK, s_end = min(depth, s_begin + (int64_t)depth_tiles_per_split * BK);
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
    char* la = lds + cur * (TA::BYTES + TB::BYTES);
    char* lb = la + TA::BYTES;
    ta.store(la);
    tb.store(lb);
    if (s + BK < s_end) {
      ta.load(A, i0, s + BK, s_end);
      tb.load(B, j0, s + BK, s_end);
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 4; c++) {
      typename TA::V fa[MI];
      typename TB::V fb[MJ];
#pragma unroll
      for (int a = 0; a < MI; a++) fa[a] = TA::frag(la, wi + a * 32, c);
#pragma unroll
      for (int b = 0; b < MJ; b++) fb[b] = TB::frag(lb, wj + b * 32, c);
#pragma unroll
      for (int a = 0; a < MI; a++)
#pragma unroll
        for (int b = 0; b < MJ; b++) acc[a][b] = mma(fa[a], fb[b], acc[a][b]);
    }
    cur ^= 1;
  }

  // Lane l holds column l % 32 and rows 8 (q / 4) + 4 (l / 32) + q % 4 of a 32 x 32 block.  The sums pass through LDS, 32 rows of a wave at a time, so
  // that a lane ends with eight neighbours of one row: whole 16-byte accesses, whole lines.  (Row stride + 8: the two halves of a wave write disjoint banks.)
  constexpr int W = 8, COLS = BJ / WJ, STRIDE = COLS + 8, LPR = COLS / W, RPP = 64 / LPR;
  static_assert(WI * WJ * 32 * STRIDE * 4 <= (int)sizeof lds, "staging fits");
  const int l = threadIdx.x & 63;
  float* stage = (float*)lds + wave * 32 * STRIDE;
  __syncthreads();
#pragma unroll
  for (int a = 0; a < MI; a++) {
#pragma unroll
    for (int b = 0; b < MJ; b++)
#pragma unroll
      for (int q = 0; q < 16; q++) stage[(8 * (q >> 2) + 4 * (l >> 5) + (q & 3)) * STRIDE + b * 32 + (l & 31)] = acc[a][b][q];
    __syncthreads();
#pragma unroll 1
    for (int p = 0; p < 32; p += RPP) {
      const int row = p + l / LPR, col = (l % LPR) * W;
      const int64_t i = i0 + wi + a * 32 + row, j = j0 + wj + col;
      float v[W];
      __builtin_memcpy(v, __builtin_assume_aligned(stage + row * STRIDE + col, 16), sizeof v);
      const int count = (int)min((int64_t)W, (int64_t)B.extent - j);
      if (i < A.extent && count > 0) {
        if (ep.part) {
          float* d = ep.part + ((int64_t)blockIdx.y * A.extent + i) * B.extent + j;
          if (ep.wide) __builtin_memcpy(__builtin_assume_aligned(d, 16), v, sizeof v);
          else
#pragma unroll
            for (int u = 0; u < W; u++)
              if (u < count) d[u] = v[u];
        } else if (ep.wide) finish<T, W, true>(ep, i, j, B.extent, W, v);
        else finish<T, W, false>(ep, i, j, B.extent, count, v);
      }
    }
    __syncthreads();
  }
}

// the splits' sums, added in their order, and the epilogue
template <class T>
__global__ __launch_bounds__(256) void k_join(int64_t rows, int64_t n, int splits, Epilogue ep) {
  const int64_t total = rows * n;
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < total; u += (int64_t)gridDim.x * 256) {
    float v[1] = {0.0f};
    for (int s = 0; s < splits; s++) v[0] += ep.part[(int64_t)s * total + u];
    finish<T, 1, false>(ep, u / n, u % n, n, 1, v);
  }
}

}  // namespace mgo
