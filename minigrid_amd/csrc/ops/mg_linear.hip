// mg_linear.hip — the linear layer and its gradients (include/minigrid_ops.h): argument checks and the choice of tile and split.  The kernels are in
// mg_linear.h, one translation unit per element type (mg_linear_tu.inc).
#include "mg_linear.h"

namespace mgo {

// The unchecked kernel needs a whole tile of every axis, and a tile of an operand that spans less than 2 GiB (one 32-bit offset per thread).
static bool fits(int tile, int64_t ri, int64_t rj, int64_t depth, int bk) { return ri >= TILE_I[tile] && rj >= TILE_J[tile] && depth >= bk; }

// A tile and how the summed axis is split: as often as the CUs hold workgroups that the tiles of the result alone do not fill (in runs of at least four tiles).  A
// CU holds one workgroup of the 256-tile, two of 128, four of 64.
static Plan with_tile(int tile, int64_t ri, int64_t rj, int64_t deep) {
  const int64_t slots = tile == TILE_256 ? 256 : tile == TILE_64 ? 1024 : 512, tiles = ceil_div(ri, TILE_I[tile]) * ceil_div(rj, TILE_J[tile]);
  Plan p;
  p.tile = tile;
  const int64_t splits = std::max<int64_t>(1, std::min(slots / tiles, deep / 4));
  p.per = (int)ceil_div(deep, splits);
  p.splits = p.per ? (int)ceil_div(deep, p.per) : 1;
  p.part_bytes = p.splits > 1 ? (int64_t)p.splits * ri * rj * 4 : 0;
  return p;
}

// About how many us the product takes: rounds of one workgroup a CU (two of a CU share its matrix units), each as long as its piece of the summed axis, and the splits'
// sums, which are written and read at 4 TB/s.  ns per summed element and workgroup, measured with the CUs full: 4 096 x 4 096 x 8 192 bf16 in 199 us with 256-tiles, 317
// with 128; 4 096 x 4 096 x 2 048 f32 in 510 and 545.
static double about_us(const Plan& p, int64_t ri, int64_t rj, int64_t depth, int dtype) {
  const bool f32 = dtype == MG_DT_F32, large = p.tile == TILE_256;
  const double ns = large ? (f32 ? 250.0 : 24.6) : (f32 ? 66.0 : 9.7);
  const int64_t rounds = ceil_div(ceil_div(ri, TILE_I[p.tile]) * ceil_div(rj, TILE_J[p.tile]) * p.splits, 256);
  return rounds * (double)std::min<int64_t>(depth, (int64_t)p.per * (128 / dtype_bytes(dtype))) * ns * 1e-3 + 2.0 * p.part_bytes * 0.25e-6;
}

// 256-tiles or 128?  For 16-bit operands the large ones multiply faster, but leave more CUs idle in the last round, and need more splits.  The estimates decide, with 5 % for
// the large ones.  Over 257 products (25 shapes of 256 x 512 to 65 536 x 512, 512 to 65 536 summed, bf16 and f32), forward and dw, what they choose is 0.4 % slower than the
// better of the two in the mean, at most 15 %: 3 328 x 3 328 x 2 048 bf16 256 46 us (128: 68), 3 297 x 1 483 x 2 048 bf16 128 41 (256: 48), 2 304 x 2 304 x 4 096 bf16 256 62
// (128: 76), 6 000 x 3 003 x 1 001 f32 128 345 (256: 513).
static Plan plan_product(int64_t ri, int64_t rj, int64_t depth, int dtype) {
  const int bk = 128 / dtype_bytes(dtype);
  const int64_t deep = ceil_div(depth, bk);
  auto work = [&](int t) { return ceil_div(ri, TILE_I[t]) * ceil_div(rj, TILE_J[t]) * deep; };
  if (fits(TILE_128, ri, rj, depth, bk) && work(TILE_128) >= 256 * 4) {
    const Plan p = with_tile(TILE_128, ri, rj, deep);
    if (!fits(TILE_256, ri, rj, depth, bk) || work(TILE_256) < 256 * 8) return p;
    const Plan large = with_tile(TILE_256, ri, rj, deep);
    return about_us(large, ri, rj, depth, dtype) <= 1.05 * about_us(p, ri, rj, depth, dtype) ? large : p;
  }
  if (fits(TILE_64, ri, rj, depth, bk)) return with_tile(TILE_64, ri, rj, deep);
  return with_tile(ri <= 32 ? TILE_GUARDED_32_128 : rj <= 32 ? TILE_GUARDED_128_32 : TILE_GUARDED_128_128, ri, rj, deep);
}

template <class F> static int by_type(int dtype, F f) {
  return dtype == MG_DT_F32 ? f((float*)nullptr) : dtype == MG_DT_BF16 ? f((bf16*)nullptr) : f((f16*)nullptr);
}

static int product(hipStream_t st, int form, bool bytes, const Operand& A, const Operand& B, int64_t depth, int dtype, Epilogue ep, void* ws, int64_t ws_bytes) {
  if (A.extent == 0 || B.extent == 0) return MG_OK;
  ep.narrow = std::max({ep.ldc, ep.r ? ep.ldr : 0, (int64_t)B.extent}) < (1 << 21);
  Plan p = plan_product(A.extent, B.extent, depth, dtype);
  if (p.part_bytes > ws_bytes || (p.part_bytes && (!ws || ((uintptr_t)ws & 255)))) return fail(MG_ERR_INVALID, "workspace: %lld bytes, 256-byte aligned, are needed", (long long)p.part_bytes);
  // (rows so far apart that a tile of them, or of the result, spans 2 GiB: the kernel with 64-bit offsets, same splits)
  if (p.tile >= TILE_64 && (!ep.narrow || std::max(A.ld, B.ld) * TILE_I[p.tile] * 4 >= 0x7fffffffll)) p.tile = TILE_GUARDED_128_128;
  // Four waves of 128 x 128 or eight of 128 x 64?  The four multiply faster (65 536 x 1024 x 512: 69 us against 78; 32 768 x 2048 x 4096: 448 against 521),
  // the eight get a tile's z and residual through faster, which decides up to 512 summed elements (65 536 x 256 x 512 with both: 61 us against 54,
  // 65 536 x 512 x 512 from cold memory: 99 against 87; 65 536 x 768 x 512: 95 against 102).
  const bool busy = (ep.z || ep.r) && depth <= 512;
  // 16-byte chunks at 16-byte addresses throughout: the operand itself, its rows, and the tiles that were moved back inside
  auto aligned = [](const Operand& o, bool cols) { return !((uintptr_t)o.p & 15) && o.ld % 8 == 0 && (!cols || o.extent % 8 == 0); };
  auto row = [](const void* q, int64_t ld) { return !q || (!((uintptr_t)q & 15) && ld % 8 == 0); };
  if (p.tile == TILE_256 && dtype != MG_DT_F32 && !bytes && aligned(A, form == FORM_DW) && aligned(B, form != FORM_FORWARD) && B.extent % 8 == 0 && ep.narrow &&
      row(ep.c, ep.ldc) && row(ep.z, 0) && row(ep.r, ep.ldr) && row(ep.b, 0) && !busy)
    p.tile = TILE_DIRECT;
  // (a launch holds less than 2^32 threads along an axis)
  if (ceil_div(A.extent, TILE_I[p.tile]) * ceil_div(B.extent, TILE_J[p.tile]) * 512 > 0xffffffffll) return fail(MG_ERR_INVALID, "the result has too many tiles");
  Epilogue first = ep;
  if (p.splits > 1) first.part = (float*)ws;
  return by_type(dtype, [&](auto* t) {
    typedef Linear<std::remove_pointer_t<decltype(t)>> L;
    L::product(st, form, bytes, p, A, B, depth, first);
    if (p.splits > 1) {
      ep.part = (float*)ws;
      L::join(st, A.extent, B.extent, p.splits, ep);
    }
    return launched("product");
  });
}

static bool known(int act) { return (act >= MG_ACTIVATION_NONE && act <= MG_ACTIVATION_SILU) || act == MG_ACTIVATION_TANH_Z32; }
// (a z of 32-bit operands is f32 either way)
static int kernel_act(int act, int dtype) { return act == MG_ACTIVATION_TANH_Z32 && dtype == MG_DT_F32 ? MG_ACTIVATION_TANH : act; }

static int check_sizes(int64_t rows, int64_t k, int64_t n, int dtype) {
  if (dtype != MG_DT_F32 && dtype != MG_DT_BF16 && dtype != MG_DT_F16) return fail(MG_ERR_INVALID, "dtype must be f32, bf16 or f16");
  if (rows < 0 || k < 1 || n < 1 || rows > 0x7fffff00ll || k > 0x7fffff00ll || n > 0x7fffff00ll) return fail(MG_ERR_INVALID, "sizes must be 0 <= rows, 1 <= k, 1 <= n, below 2^31 - 256");
  return MG_OK;
}

}  // namespace mgo

using namespace mgo;

extern "C" {

int mg_op_linear_workspace(int64_t rows, int64_t k, int64_t n, int dtype, int64_t* forward, int64_t* backward_input, int64_t* backward_weight) {
  const int rc = check_sizes(rows, k, n, dtype);
  if (rc != MG_OK) return rc;
  if (forward) *forward = rows > FEW_ROWS ? plan_product(rows, n, k, dtype).part_bytes : 0;
  if (backward_input) *backward_input = rows ? plan_product(rows, k, n, dtype).part_bytes : 0;
  if (backward_weight) *backward_weight = plan_product(n, k, rows, dtype).part_bytes;
  return MG_OK;
}

int mg_op_linear(int device, void* stream, int dtype, int x_dtype, int act, int64_t rows, int64_t k, int64_t n, const void* x, int64_t ldx, const void* w,
                 int64_t ldw, const void* b, const void* r, int64_t ldr, void* y, int64_t ldy, void* z, void* ws, int64_t ws_bytes) {
  int rc = check_sizes(rows, k, n, dtype);
  if (rc != MG_OK) return rc;
  if (x_dtype != dtype && x_dtype != MG_DT_U8) return fail(MG_ERR_INVALID, "x must have w's type or be bytes");
  if (!known(act)) return fail(MG_ERR_INVALID, "unknown activation %d", act);
  if (rows == 0) return MG_OK;
  if (!x || !w || !y) return fail(MG_ERR_INVALID, "x, w and y must not be NULL");
  if (ldx < k || ldw < k || ldy < n || (r && ldr < n)) return fail(MG_ERR_INVALID, "a row stride is smaller than its row");
  DeviceGuard g(device);
  if (g.rc != MG_OK) return g.rc;
  hipStream_t st = (hipStream_t)stream;
  Epilogue ep = {b, r, y, z, nullptr, ldr, ldy, kernel_act(act, dtype), 0};
  const bool bytes = x_dtype == MG_DT_U8;
  if (rows <= FEW_ROWS)
    return by_type(dtype, [&](auto* t) {
      Linear<std::remove_pointer_t<decltype(t)>>::few_rows(st, bytes, (int)rows, k, n, x, ldx, w, ldw, ep);
      return launched("linear");
    });
  const Operand A = {x, ldx, (int32_t)rows}, B = {w, ldw, (int32_t)n};
  return product(st, FORM_FORWARD, bytes, A, B, k, dtype, ep, ws, ws_bytes);
}

int mg_op_linear_dz_workspace(int64_t rows, int64_t n, int64_t* bytes) {
  if (rows < 0 || n < 1 || !bytes) return fail(MG_ERR_INVALID, "sizes must be 0 <= rows, 1 <= n");
  *bytes = dz_plan(rows, n).runs * n * 4;
  return MG_OK;
}

int mg_op_linear_dz(int device, void* stream, int dtype, int act, int64_t rows, int64_t n, const void* dy, int64_t lddy, const void* z, void* dz, void* db,
                    void* ws, int64_t ws_bytes) {
  int rc = check_sizes(rows, 1, n, dtype);
  if (rc != MG_OK) return rc;
  if (!known(act)) return fail(MG_ERR_INVALID, "unknown activation %d", act);
  if (act != MG_ACTIVATION_NONE && !z && rows) return fail(MG_ERR_INVALID, "the values in front of the activation are needed");
  if ((!dy && rows) || lddy < n) return fail(MG_ERR_INVALID, "dy must not be NULL and its row stride not smaller than its row");
  DeviceGuard g(device);
  if (g.rc != MG_OK) return g.rc;
  hipStream_t st = (hipStream_t)stream;
  const DzPlan p = dz_plan(rows, n);
  const int64_t need = p.runs * n * 4;
  if (db && (need > ws_bytes || !ws || ((uintptr_t)ws & 255))) return fail(MG_ERR_INVALID, "workspace: %lld bytes, 256-byte aligned, are needed", (long long)need);
  if (p.strips > 0x7fffffffll || p.runs > 65535) return fail(MG_ERR_INVALID, "too many rows or columns");
  return by_type(dtype, [&](auto* t) {
    Linear<std::remove_pointer_t<decltype(t)>>::dz(st, kernel_act(act, dtype), rows, n, dy, lddy, z, dz, db, db ? (float*)ws : nullptr);
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
  Epilogue ep = {nullptr, nullptr, dx, nullptr, nullptr, 0, k, MG_ACTIVATION_NONE, 0};
  const Operand A = {dz, lddz, (int32_t)rows}, B = {w, ldw, (int32_t)k};
  return product((hipStream_t)stream, FORM_DX, false, A, B, n, dtype, ep, ws, ws_bytes);
}

int mg_op_linear_dw(int device, void* stream, int dtype, int x_dtype, int64_t rows, int64_t k, int64_t n, const void* dz, int64_t lddz, const void* x, int64_t ldx,
                    void* dw, void* ws, int64_t ws_bytes) {
  int rc = check_sizes(rows, k, n, dtype);
  if (rc != MG_OK) return rc;
  if (x_dtype != dtype && x_dtype != MG_DT_U8) return fail(MG_ERR_INVALID, "x must have w's type or be bytes");
  if (!dw || (rows && (!dz || !x)) || lddz < n || ldx < k) return fail(MG_ERR_INVALID, "dz, x and dw must not be NULL and a row stride not smaller than its row");
  DeviceGuard g(device);
  if (g.rc != MG_OK) return g.rc;
  Epilogue ep = {nullptr, nullptr, dw, nullptr, nullptr, 0, k, MG_ACTIVATION_NONE, 0};
  const Operand A = {dz, lddz, (int32_t)n}, B = {x, ldx, (int32_t)k};
  return product((hipStream_t)stream, FORM_DW, x_dtype == MG_DT_U8, A, B, rows, dtype, ep, ws, ws_bytes);
}

}  // extern "C"
