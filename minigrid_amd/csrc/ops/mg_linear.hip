// mg_linear.hip — the linear layer and its gradients (include/minigrid_ops.h): argument checks, the choice of tile and split, the elementwise part of
// the backward pass.
#include "mg_linear.h"

namespace mgo {

// dz = dy act'(z), and the column sums of dz: a workgroup takes 64 columns and a run of rows, its four waves every fourth row; the sums of the runs are
// added in their order by k_column_sums.  Bound by memory: reads dy and z, writes dz.
template <class T>
__global__ __launch_bounds__(256) void k_dz(int64_t rows, int64_t n, int act, const T* dy, int64_t lddy, const T* z, T* dz, float* part, int64_t run) {
  __shared__ float sum[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t j = (int64_t)blockIdx.x * 64 + lane, i1 = min(rows, ((int64_t)blockIdx.y + 1) * run);
  float s = 0.0f;
  if (j < n)
    for (int64_t i = (int64_t)blockIdx.y * run + w; i < i1; i += 4) {
      float v = (float)dy[i * lddy + j];
      if (z) v *= activate_grad(act, (float)z[i * n + j]);
      if (dz) dz[i * n + j] = (T)v;
      s += v;
    }
  if (part) {
    sum[w][lane] = s;
    __syncthreads();
    if (w == 0 && j < n) part[(int64_t)blockIdx.y * n + j] = (sum[0][lane] + sum[1][lane]) + (sum[2][lane] + sum[3][lane]);
  }
}

template <class T>
__global__ __launch_bounds__(64) void k_column_sums(int64_t n, int runs, const float* part, T* db) {
  const int64_t j = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (j >= n) return;
  float s = 0.0f;
  for (int r = 0; r < runs; r++) s += part[(int64_t)r * n + j];
  db[j] = (T)s;
}

struct Plan {
  int bi, bj, splits, per;     // tile, number of splits of the summed axis, tiles of that axis per split
  int64_t part_bytes;
};

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The tile follows the result's shape; where the tiles of the result do not fill the 256 CUs twice, the summed axis is split so that they do, in runs of
// at least four tiles.
static Plan plan_product(int64_t ri, int64_t rj, int64_t depth, int dtype) {
  Plan p;
  p.bi = ri <= 32 ? 32 : 128;
  p.bj = rj <= 32 && p.bi == 128 ? 32 : 128;
  const int64_t tiles = ceil_div(ri, p.bi) * ceil_div(rj, p.bj), deep = ceil_div(depth, 128 / dtype_bytes(dtype));
  int64_t splits = tiles >= 512 ? 1 : ceil_div(512, tiles);
  if (splits > deep / 4) splits = deep / 4;
  if (splits < 1) splits = 1;
  p.per = (int)ceil_div(deep, splits);
  p.splits = (int)(p.per ? ceil_div(deep, p.per) : 1);
  if (p.splits < 1) p.splits = 1;
  p.part_bytes = p.splits > 1 ? (int64_t)p.splits * ri * rj * 4 : 0;
  return p;
}

static bool row_vec(const void* p, int64_t ld, int64_t elem, int64_t extent_along) {
  const int64_t n = 16 / elem;
  return ((uintptr_t)p & 15) == 0 && ld % n == 0 && extent_along % n == 0;
}

template <class T, class SA, class SB, bool ACOLS, bool BCOLS, bool VEC>
static int launch_product(hipStream_t st, const Plan& p, const Operand& A, const Operand& B, int64_t depth, const Epilogue& ep) {
  const dim3 grid((unsigned)(ceil_div(A.extent, p.bi) * ceil_div(B.extent, p.bj)), p.splits);
  if (p.bi == 32) k_product<T, SA, SB, ACOLS, BCOLS, VEC, 32, 128, 1, 4><<<grid, 256, 0, st>>>(A, B, depth, p.per, ep);
  else if (p.bj == 32) k_product<T, SA, SB, ACOLS, BCOLS, VEC, 128, 32, 4, 1><<<grid, 256, 0, st>>>(A, B, depth, p.per, ep);
  else k_product<T, SA, SB, ACOLS, BCOLS, VEC, 128, 128, 2, 2><<<grid, 256, 0, st>>>(A, B, depth, p.per, ep);
  return launched("product");
}

template <class T, class SA, class SB, bool ACOLS, bool BCOLS>
static int product(hipStream_t st, const Operand& A, const Operand& B, int64_t depth, int dtype, bool vec, Epilogue ep, void* ws, int64_t ws_bytes) {
  if (A.extent == 0 || B.extent == 0) return MG_OK;
  const Plan p = plan_product(A.extent, B.extent, depth, dtype);
  if (p.part_bytes > ws_bytes || (p.part_bytes && (!ws || ((uintptr_t)ws & 255)))) return fail(MG_ERR_INVALID, "workspace: %lld bytes, 256-byte aligned, are needed", (long long)p.part_bytes);
  if (ceil_div(A.extent, p.bi) * ceil_div(B.extent, p.bj) > 0x7fffffffll) return fail(MG_ERR_INVALID, "the result has too many tiles");
  Epilogue first = ep;
  if (p.splits > 1) {
    first.part = (float*)ws;
    first.wide = B.extent % 8 == 0;
  }
  const int rc = vec ? launch_product<T, SA, SB, ACOLS, BCOLS, true>(st, p, A, B, depth, first) : launch_product<T, SA, SB, ACOLS, BCOLS, false>(st, p, A, B, depth, first);
  if (rc != MG_OK || p.splits == 1) return rc;
  ep.part = (float*)ws;
  const int64_t total = (int64_t)A.extent * B.extent;
  k_join<T><<<(unsigned)std::min<int64_t>(ceil_div(total, 256), 4096), 256, 0, st>>>(A.extent, B.extent, p.splits, ep);
  return launched("join");
}

static int check_sizes(int64_t rows, int64_t k, int64_t n, int dtype) {
  if (dtype != MG_DT_F32 && dtype != MG_DT_BF16 && dtype != MG_DT_F16) return fail(MG_ERR_INVALID, "dtype must be f32, bf16 or f16");
  if (rows < 0 || k < 1 || n < 1 || rows > 0x7fffff00ll || k > 0x7fffff00ll || n > 0x7fffff00ll) return fail(MG_ERR_INVALID, "sizes must be 0 <= rows, 1 <= k, 1 <= n, below 2^31 - 256");
  return MG_OK;
}

template <class F> static int by_type(int dtype, F f) {
  return dtype == MG_DT_F32 ? f((float*)nullptr) : dtype == MG_DT_BF16 ? f((bf16*)nullptr) : f((f16*)nullptr);
}

constexpr int DZ_RUNS = 1024;
static int64_t dz_run(int64_t rows, int64_t n) {           // rows per workgroup: about 2048 workgroups, at least 16 rows each
  const int64_t strips = ceil_div(n, 64);
  int64_t runs = std::min<int64_t>(std::max<int64_t>(1, 2048 / strips), DZ_RUNS);
  return std::max<int64_t>(16, ceil_div(rows, runs));
}

}  // namespace mgo

using namespace mgo;

extern "C" {

int mg_op_linear_workspace(int64_t rows, int64_t k, int64_t n, int dtype, int64_t* forward, int64_t* backward_input, int64_t* backward_weight) {
  const int rc = check_sizes(rows, k, n, dtype);
  if (rc != MG_OK) return rc;
  if (forward) *forward = rows ? plan_product(rows, n, k, dtype).part_bytes : 0;
  if (backward_input) *backward_input = rows ? plan_product(rows, k, n, dtype).part_bytes : 0;
  if (backward_weight) *backward_weight = plan_product(n, k, rows, dtype).part_bytes;
  return MG_OK;
}

int mg_op_linear(int device, void* stream, int dtype, int x_dtype, int act, int64_t rows, int64_t k, int64_t n, const void* x, int64_t ldx, const void* w,
                 int64_t ldw, const void* b, const void* r, int64_t ldr, void* y, int64_t ldy, void* z, void* ws, int64_t ws_bytes) {
  int rc = check_sizes(rows, k, n, dtype);
  if (rc != MG_OK) return rc;
  if (x_dtype != dtype && x_dtype != MG_DT_U8) return fail(MG_ERR_INVALID, "x must have w's type or be bytes");
  if (act < MG_ACTIVATION_NONE || act > MG_ACTIVATION_SILU) return fail(MG_ERR_INVALID, "unknown activation %d", act);
  if (rows == 0) return MG_OK;
  if (!x || !w || !y) return fail(MG_ERR_INVALID, "x, w and y must not be NULL");
  if (ldx < k || ldw < k || ldy < n || (r && ldr < n)) return fail(MG_ERR_INVALID, "a row stride is smaller than its row");
  DeviceGuard g(device);
  if (g.rc != MG_OK) return g.rc;
  hipStream_t st = (hipStream_t)stream;
  const int eb = dtype_bytes(dtype);
  Epilogue ep = {b, r, y, z, nullptr, ldr, ldy, act, 0};
  ep.wide = row_vec(y, ldy, 2, n) && (!r || row_vec(r, ldr, 2, n)) && (!z || row_vec(z, n, 2, n));      // (eight elements: 16 bytes or twice 16)
  const Operand A = {x, ldx, (int32_t)rows}, B = {w, ldw, (int32_t)n};
  const bool vb = row_vec(w, ldw, eb, k);
  return by_type(dtype, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    if (x_dtype == MG_DT_U8) return product<T, uint8_t, T, false, false>(st, A, B, k, dtype, false, ep, ws, ws_bytes);
    return product<T, T, T, false, false>(st, A, B, k, dtype, vb && row_vec(x, ldx, eb, k), ep, ws, ws_bytes);
  });
}

int mg_op_linear_dz_workspace(int64_t rows, int64_t n, int64_t* bytes) {
  if (rows < 0 || n < 1 || !bytes) return fail(MG_ERR_INVALID, "sizes must be 0 <= rows, 1 <= n");
  *bytes = ceil_div(std::max<int64_t>(rows, 1), dz_run(rows, n)) * n * 4;
  return MG_OK;
}

int mg_op_linear_dz(int device, void* stream, int dtype, int act, int64_t rows, int64_t n, const void* dy, int64_t lddy, const void* z, void* dz, void* db,
                    void* ws, int64_t ws_bytes) {
  int rc = check_sizes(rows, 1, n, dtype);
  if (rc != MG_OK) return rc;
  if (act < MG_ACTIVATION_NONE || act > MG_ACTIVATION_SILU) return fail(MG_ERR_INVALID, "unknown activation %d", act);
  if (act != MG_ACTIVATION_NONE && !z && rows) return fail(MG_ERR_INVALID, "the values in front of the activation are needed");
  if ((!dy && rows) || lddy < n) return fail(MG_ERR_INVALID, "dy must not be NULL and its row stride not smaller than its row");
  DeviceGuard g(device);
  if (g.rc != MG_OK) return g.rc;
  hipStream_t st = (hipStream_t)stream;
  const int64_t run = dz_run(rows, n), runs = ceil_div(rows, run);
  if (db && (runs * n * 4 > ws_bytes || (runs && (!ws || ((uintptr_t)ws & 255))))) return fail(MG_ERR_INVALID, "workspace: %lld bytes, 256-byte aligned, are needed", (long long)(runs * n * 4));
  const int64_t strips = ceil_div(n, 64);
  return by_type(dtype, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    if (runs) k_dz<T><<<dim3((unsigned)strips, (unsigned)runs), 256, 0, st>>>(rows, n, act, (const T*)dy, lddy, act == MG_ACTIVATION_NONE ? nullptr : (const T*)z, (T*)dz, db ? (float*)ws : nullptr, run);
    if (db) k_column_sums<T><<<(unsigned)strips, 64, 0, st>>>(n, (int)runs, (const float*)ws, (T*)db);
    return launched("dz");
  });
}

int mg_op_linear_dx(int device, void* stream, int dtype, int64_t rows, int64_t k, int64_t n, const void* dz, int64_t lddz, const void* w, int64_t ldw, void* dx,
                    void* ws, int64_t ws_bytes) {
  int rc = check_sizes(rows, k, n, dtype);
  if (rc != MG_OK) return rc;
  if (rows == 0) return MG_OK;
  if (!dz || !w || !dx || lddz < n || ldw < k) return fail(MG_ERR_INVALID, "dz, w and dx must not be NULL and a row stride not smaller than its row");
  DeviceGuard g(device);
  if (g.rc != MG_OK) return g.rc;
  const int eb = dtype_bytes(dtype);
  Epilogue ep = {nullptr, nullptr, dx, nullptr, nullptr, 0, k, MG_ACTIVATION_NONE, row_vec(dx, k, 2, k)};
  const Operand A = {dz, lddz, (int32_t)rows}, B = {w, ldw, (int32_t)k};
  return by_type(dtype, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    return product<T, T, T, false, true>((hipStream_t)stream, A, B, n, dtype, row_vec(dz, lddz, eb, n) && row_vec(w, ldw, eb, k), ep, ws, ws_bytes);
  });
}

int mg_op_linear_dw(int device, void* stream, int dtype, int x_dtype, int64_t rows, int64_t k, int64_t n, const void* dz, int64_t lddz, const void* x, int64_t ldx,
                    void* dw, void* ws, int64_t ws_bytes) {
  int rc = check_sizes(rows, k, n, dtype);
  if (rc != MG_OK) return rc;
  if (x_dtype != dtype && x_dtype != MG_DT_U8) return fail(MG_ERR_INVALID, "x must have w's type or be bytes");
  if (!dw || (rows && (!dz || !x)) || lddz < n || ldx < k) return fail(MG_ERR_INVALID, "dz, x and dw must not be NULL and a row stride not smaller than its row");
  DeviceGuard g(device);
  if (g.rc != MG_OK) return g.rc;
  hipStream_t st = (hipStream_t)stream;
  const int eb = dtype_bytes(dtype);
  Epilogue ep = {nullptr, nullptr, dw, nullptr, nullptr, 0, k, MG_ACTIVATION_NONE, row_vec(dw, k, 2, k)};
  const Operand A = {dz, lddz, (int32_t)n}, B = {x, ldx, (int32_t)k};
  return by_type(dtype, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    if (x_dtype == MG_DT_U8) return product<T, T, uint8_t, true, true>(st, A, B, rows, dtype, false, ep, ws, ws_bytes);
    return product<T, T, T, true, true>(st, A, B, rows, dtype, row_vec(dz, lddz, eb, n) && row_vec(x, ldx, eb, k), ep, ws, ws_bytes);
  });
}

}  // extern "C"
