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

// The two flags of a step: bit 0 terminated, bit 1 truncated.  PAIR: they are neighbouring bytes at an even address (fields of one step record), one load.
template <bool PAIR>
__device__ __forceinline__ uint32_t flags_at(const mg_advantages_args& g, int64_t t, int64_t e) {
  if constexpr (PAIR) {
    const uint32_t v = *(const uint16_t*)(g.terminated + t * g.s_term[0] + e * g.s_term[1]);
    return ((v & 0xffu) ? 1u : 0u) | ((v >> 8) ? 2u : 0u);
  } else {
    return (g.terminated[t * g.s_term[0] + e * g.s_term[1]] ? 1u : 0u) | (g.truncated[t * g.s_trunc[0] + e * g.s_trunc[1]] ? 2u : 0u);
  }
}

constexpr int SEG = 16;        // steps of a lane
constexpr int WAVES = 8;

// Reward and flags of a step at once where they are the fields of one 16-byte record (f64, then the two bytes): what the environments hand out.  Asked for one by
// one, a record's line is on its way twice (2 048 x 16: 15.8 us, at once 12.9; 128 x 65 536 is bound by memory either way).
__device__ __forceinline__ void record_at(const mg_advantages_args& g, int64_t t, int64_t e, double& reward, uint32_t& flags) {
  const u32x4 w = *(const u32x4*)((const double*)g.reward + t * g.s_reward[0] + e * g.s_reward[1]);
  reward = __hiloint2double((int)w[1], (int)w[0]);
  flags = ((w[2] & 0xffu) ? 1u : 0u) | ((w[2] & 0xff00u) ? 2u : 0u);
}
enum { FLAGS_APART, FLAGS_PAIR, FLAGS_RECORD };

// A workgroup owns EL environments and walks their rollout from the end, blockDim / EL stretches of SEG steps at a time.  A lane loads its stretch
// whole (every load in flight at once), folds it into one pair (a, b); the pairs of an environment are chained through LDS by one lane, and each lane
// unfolds its stretch from what the chain leaves behind it.  So the inputs are read once and the dependent chain is steps / SEG long.  Bound by
// memory: 128 x 65 536 (16-byte records) moves 243 MB in 55 us, 71 where nothing of it is in a cache yet.  EL = 64 has whole lines in every access; where that leaves most CUs without a workgroup, 16
// and 4 environments share a wave's lanes with the time axis.
template <class R, class V, int EL, int FLAGS>
__global__ __launch_bounds__(64 * WAVES) void k_advantages(mg_advantages_args g) {
  __shared__ double pa[64 * WAVES], pb[64 * WAVES], pc[64 * WAVES], carry[EL];
  const int el = threadIdx.x % EL, seg = threadIdx.x / EL, segs = blockDim.x / EL;
  const int64_t e = (int64_t)blockIdx.x * EL + el, span = (int64_t)segs * SEG;
  const bool on = e < g.envs;
  const double gl = g.gamma * g.lam;
  if (seg == 0) carry[el] = 0.0;
  // stretches are dealt from the end: the first block of `span` steps ends at g.steps
  for (int64_t top = g.steps; top > 0; top -= span) {
    const int64_t hi = top - (int64_t)seg * SEG, lo = hi > SEG ? hi - SEG : 0;      // this lane's steps lo..hi-1 (none where hi <= 0)
    const int n = on && hi > 0 ? (int)(hi - lo) : 0;
    double r[SEG];
    float v[SEG + 1];
    uint32_t f[SEG + 1];
    // index u counts from the end: step hi - 1 - u
#pragma unroll
    for (int u = 0; u < SEG; u++) {
      r[u] = 0.0; v[u + 1] = 0.0f; f[u] = 0;
      if (u < n) {
        const int64_t t = hi - 1 - u;
        if constexpr (FLAGS == FLAGS_RECORD) record_at(g, t, e, r[u], f[u]);
        else {
          r[u] = at<R>(g.reward, g.s_reward, t, e);
          f[u] = flags_at<FLAGS == FLAGS_PAIR>(g, t, e);
        }
        v[u + 1] = (float)at<V>(g.value, g.s_value, t, e);
      }
    }
    v[0] = 0.0f; f[SEG] = 0;
    uint32_t before = 0;                                                             // did the step in front of the stretch end an episode?
    if (n) {
      v[0] = hi < g.steps ? (float)at<V>(g.value, g.s_value, hi, e) : (float)((const V*)g.last_value)[e];
      if (g.next_step) before = lo ? flags_at<FLAGS != FLAGS_APART>(g, lo - 1, e) : g.done0 && g.done0[e] ? 1u : 0u;
    }
    double a = 1.0, b = 0.0;
    uint32_t valid = 0, open = 0;                                                    // bits: the step counts; the sum goes on behind it
#pragma unroll
    for (int u = 0; u < SEG; u++) {
      if (u < n) {
        const uint32_t end = f[u], prev = u + 1 < n ? f[u + 1] : before;
        const bool counts = !(g.next_step && prev);
        double worth = end & 1u ? 0.0 : (double)v[u];
        if (!g.next_step && (end & 2u) && !(end & 1u)) worth = g.final_value ? at<V>(g.final_value, g.s_final, hi - 1 - u, e) : 0.0;
        r[u] = counts ? r[u] + g.gamma * worth - (double)v[u + 1] : 0.0;
        const bool go = counts && !end;
        valid |= counts ? 1u << u : 0u;
        open |= go ? 1u << u : 0u;
        // (selected, not multiplied by 0: a NaN behind an end stays there)
        b = go ? r[u] + gl * b : r[u];
        a = go ? a * gl : 0.0;
      }
    }
    // (-inf says that the stretch holds an end: nothing behind it counts, not even a NaN)
    pa[seg * EL + el] = open == (1u << n) - 1 ? a : -__builtin_inf();
    pb[seg * EL + el] = b;
    __syncthreads();
    if (seg == 0) {
      double c = carry[el];
      constexpr int Q = 64 / EL < 8 ? 64 / EL : 8;                                         // (the number of stretches is a multiple of it)
      for (int q = 0; q < segs; q += Q) {
        double qa[Q], qb[Q];
#pragma unroll
        for (int u = 0; u < Q; u++) { qa[u] = pa[(q + u) * EL + el]; qb[u] = pb[(q + u) * EL + el]; }
#pragma unroll
        for (int u = 0; u < Q; u++) {
          pc[(q + u) * EL + el] = c;                                                 // what stands behind the stretch
          c = qa[u] == -__builtin_inf() ? qb[u] : qb[u] + qa[u] * c;
        }
      }
      carry[el] = c;
    }
    __syncthreads();
    double run = pc[seg * EL + el];
#pragma unroll
    for (int u = 0; u < SEG; u++) {
      if (u < n) {
        run = open >> u & 1u ? r[u] + gl * run : r[u];
        const int64_t o = (hi - 1 - u) * g.envs + e;
        g.advantage[o] = (float)run;
        g.ret[o] = (float)(run + (double)v[u + 1]);
        g.valid[o] = valid >> u & 1u;
      }
    }
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
  // neighbouring flag bytes at even addresses?
  const bool pair = g.truncated == g.terminated + 1 && !((uintptr_t)g.terminated & 1) && g.s_term[0] == g.s_trunc[0] && g.s_term[1] == g.s_trunc[1] &&
                    g.s_term[0] % 2 == 0 && g.s_term[1] % 2 == 0;
  const bool record = pair && g.reward_dtype == MG_DT_F64 && (const uint8_t*)g.reward + 8 == g.terminated && !((uintptr_t)g.reward & 15) && g.s_reward[0] % 2 == 0 &&
                      g.s_reward[1] % 2 == 0 && g.s_term[0] == 8 * g.s_reward[0] && g.s_term[1] == 8 * g.s_reward[1];
  // As many environments per workgroup as leave every CU two, or half of them one (128 x 20 000: 20 us with 16, 25 with 64; 53 x 58 162: 37 and 30;
  // 300 x 1 000: 13 with 4, 11 with 16, 22 with 64; 1 788 x 2: 13, 40 and 130); a short rollout has nothing to spread over the lanes.
  const int el = g.envs >= 64 * 512 || g.steps <= SEG ? 64 : g.envs >= 16 * 128 || g.steps <= 4 * SEG ? 16 : 4;
  const int64_t stretches = (g.steps + SEG - 1) / SEG;
  const int waves = (int)std::min<int64_t>(WAVES, (stretches * el + 63) / 64);
  const unsigned grid = (unsigned)((g.envs + el - 1) / el);
#define MG_GO3(R, V, EL) \
  (record && sizeof(R) == 8 ? k_advantages<R, V, EL, sizeof(R) == 8 ? FLAGS_RECORD : FLAGS_PAIR><<<grid, 64 * waves, 0, st>>>(g) \
   : pair ? k_advantages<R, V, EL, FLAGS_PAIR><<<grid, 64 * waves, 0, st>>>(g) : k_advantages<R, V, EL, FLAGS_APART><<<grid, 64 * waves, 0, st>>>(g))
#define MG_GO(R, V) (el == 64 ? MG_GO3(R, V, 64) : el == 16 ? MG_GO3(R, V, 16) : MG_GO3(R, V, 4))
  if (g.reward_dtype == MG_DT_F64) {
    if (g.value_dtype == MG_DT_F32) MG_GO(double, float); else if (g.value_dtype == MG_DT_BF16) MG_GO(double, bf16); else MG_GO(double, f16);
  } else {
    if (g.value_dtype == MG_DT_F32) MG_GO(float, float); else if (g.value_dtype == MG_DT_BF16) MG_GO(float, bf16); else MG_GO(float, f16);
  }
#undef MG_GO
#undef MG_GO3
  return launched("advantages");
}

}  // extern "C"
