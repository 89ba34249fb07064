// mg_advantages.hip — generalised advantages of a rollout (include/minigrid_ops.h), and the operators' error text.
//
//   delta_t = r_t + gamma V_{t+1} [not terminated at t] - V_t,   A_t = delta_t + gamma lam [no end at t] A_{t+1},   A_t = 0 where step t only resets
//
// a linear recurrence from the last step to the first: A_t = b_t + a_t A_{t+1}.  Stretches of it compose: (a, b) of a stretch = (a1 a2, b1 + a1 b2).
#include "mg_ops.h"

#include <string>

namespace mgo {

static thread_local std::string g_error;

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  g_error = buf;
  return code;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MG_OK : fail(MG_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

template <class T> __device__ __forceinline__ double at(const void* p, const int64_t* s, int64_t t, int64_t e) { return (double)((const T*)p)[t * s[0] + e * s[1]]; }

struct Step { double a, b, value; bool valid; };

template <class R, class V>
__device__ __forceinline__ Step one_step(const mg_advantages_args& g, int64_t t, int64_t e, double next_value) {
  const int64_t* st = g.s_term;
  const int64_t* su = g.s_trunc;
  const bool term = g.terminated[t * st[0] + e * st[1]] != 0, trunc = g.truncated[t * su[0] + e * su[1]] != 0;
  bool valid = true;
  double worth = next_value;
  if (g.next_step) {
    const bool before = t ? (g.terminated[(t - 1) * st[0] + e * st[1]] | g.truncated[(t - 1) * su[0] + e * su[1]]) != 0 : g.done0 && g.done0[e] != 0;
    valid = !before;
    if (term) worth = 0.0;
  } else {
    if (term) worth = 0.0;
    else if (trunc) worth = g.final_value ? at<V>(g.final_value, g.s_final, t, e) : 0.0;
  }
  const double value = at<V>(g.value, g.s_value, t, e);
  if (!valid) return {0.0, 0.0, value, false};
  return {term || trunc ? 0.0 : g.gamma * g.lam, at<R>(g.reward, g.s_reward, t, e) + g.gamma * worth - value, value, true};
}

// a lane per environment walks its rollout from the end
template <class R, class V>
__global__ __launch_bounds__(64) void k_advantages(mg_advantages_args g) {
  const int64_t e = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (e >= g.envs) return;
  double next = (double)((const V*)g.last_value)[e], run = 0.0;
  for (int64_t t = g.steps - 1; t >= 0; t--) {
    const Step s = one_step<R, V>(g, t, e, next);
    run = s.b + s.a * run;
    const int64_t o = t * g.envs + e;
    g.advantage[o] = (float)run;
    g.ret[o] = (float)(run + s.value);
    g.valid[o] = s.valid ? 1 : 0;
    next = s.value;
  }
}

}  // namespace mgo

using namespace mgo;

extern "C" {

const char* mg_ops_last_error(void) { return g_error.c_str(); }

int mg_op_advantages(int device, void* stream, const mg_advantages_args* args) {
  if (!args) return fail(MG_ERR_INVALID, "args must not be NULL");
  const mg_advantages_args g = *args;
  if (g.steps < 0 || g.envs < 0 || g.envs > 0x7fffffc0ll) return fail(MG_ERR_INVALID, "sizes must be 0 <= steps, 0 <= envs < 2^31 - 64");
  if (g.steps == 0 || g.envs == 0) return MG_OK;
  if (!g.reward || !g.value || !g.terminated || !g.truncated || !g.last_value || !g.advantage || !g.ret || !g.valid) return fail(MG_ERR_INVALID, "only done0 and final_value may be NULL");
  if (g.reward_dtype != MG_DT_F64 && g.reward_dtype != MG_DT_F32) return fail(MG_ERR_INVALID, "reward must be f64 or f32");
  if (g.value_dtype != MG_DT_F32 && g.value_dtype != MG_DT_BF16 && g.value_dtype != MG_DT_F16) return fail(MG_ERR_INVALID, "value must be f32, bf16 or f16");
  if (g.final_value && g.next_step) return fail(MG_ERR_INVALID, "final_value belongs to the same-step autoreset");
  DeviceGuard d(device);
  if (d.rc != MG_OK) return d.rc;
  hipStream_t st = (hipStream_t)stream;
  const unsigned grid = (unsigned)((g.envs + 63) / 64);
#define MG_GO(R, V) k_advantages<R, V><<<grid, 64, 0, st>>>(g)
  if (g.reward_dtype == MG_DT_F64) {
    if (g.value_dtype == MG_DT_F32) MG_GO(double, float); else if (g.value_dtype == MG_DT_BF16) MG_GO(double, bf16); else MG_GO(double, f16);
  } else {
    if (g.value_dtype == MG_DT_F32) MG_GO(float, float); else if (g.value_dtype == MG_DT_BF16) MG_GO(float, bf16); else MG_GO(float, f16);
  }
#undef MG_GO
  return launched("advantages");
}

}  // extern "C"
