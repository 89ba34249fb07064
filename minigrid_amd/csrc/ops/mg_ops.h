// mg_ops.h — what the learning operators' translation units share: element types, argument checks, the device guard of a C entry, small device
// helpers.  The operators (include/minigrid_ops.h) are stateless: every buffer, the workspace among them, belongs to the caller, every launch goes to
// the caller's stream, and nothing is allocated, so that a call may be captured into a graph.
#pragma once
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "../../../include/minigrid_ops.h"

namespace mgo {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));   // sets mg_ops_last_error() of this thread
int launched(const char* what);                                                   // MG_OK, or what hipGetLastError says

// The device of the tensors is current for the duration of a C entry; the caller's device is current again afterwards.
struct DeviceGuard {
  int before = -1, rc = MG_OK;
  bool moved = false;
  explicit DeviceGuard(int device) {
    if (hipGetDevice(&before) != hipSuccess) { (void)hipGetLastError(); rc = fail(MG_ERR_NO_DEVICE, "no HIP device"); return; }
    if (device != before) {
      if (hipSetDevice(device) != hipSuccess) { (void)hipGetLastError(); rc = fail(MG_ERR_INVALID, "device %d does not exist", device); return; }
      moved = true;
    }
  }
  ~DeviceGuard() { if (moved) (void)hipSetDevice(before); }
  DeviceGuard(const DeviceGuard&) = delete;
};

inline int dtype_bytes(int d) { return d == MG_DT_F32 || d == MG_DT_I32 ? 4 : d == MG_DT_BF16 || d == MG_DT_F16 ? 2 : d == MG_DT_F64 || d == MG_DT_I64 ? 8 : d == MG_DT_U8 ? 1 : 0; }

// ---- wave reductions ----
__device__ __forceinline__ double shfl_xor_f64(double v, int m) {
  int lo = __double2loint(v), hi = __double2hiint(v);
  lo = __shfl_xor(lo, m); hi = __shfl_xor(hi, m);
  return __hiloint2double(hi, lo);
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += shfl_xor_f64(v, m);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}

constexpr float LOG2E = 1.44269504f;
constexpr double LN2 = 0.693147180559945309417232;

}  // namespace mgo
