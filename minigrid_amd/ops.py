"""The learning operators: what turns the batched environments' observations into actions and their trajectories into a gradient.

    linear          y = act(x W^T + b) + r, x may be the byte observations themselves; gradients of x, W, b and r
    sample_actions  one action per row of logits from one uniform number (or the greedy one), with its log-probability
    advantages      generalised advantages of a rollout, aware of the environments' autoreset
    policy_loss     the clipped policy loss with KL and entropy terms; gradient of the logits

All of them take torch tensors on an MI355X and run hand-written kernels of libminigrid_hip.so (include/minigrid_ops.h) on the tensors' device and its
current stream, in the manner of torch's own operators: nothing synchronises, results are new tensors, a call may be captured into a graph.  There is no
CPU fallback, and no forward-mode derivative: an argument that carries a tangent is refused.  So is a
call that is being traced (torch.jit.trace, make_fx): a trace would hold the result's memory and not what fills it.  What is checked and bound per call is C++ (csrc/ops/mg_torch.cpp).  `MiniGridVecEnv.rollout(policy=...)` and
`minigrid_amd.policy.ActorCritic` are built from them.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _binding as B

_ACTIVATIONS = {None: 0, "relu": 1, "tanh": 2, "gelu": 3, "silu": 4}

# every symbol include/minigrid_ops.h declares
SYMBOLS = ["mg_ops_last_error", "mg_op_linear_workspace", "mg_op_linear", "mg_op_linear_dz_workspace", "mg_op_linear_dz", "mg_op_linear_dx", "mg_op_linear_dw",
           "mg_op_policy_loss_workspace", "mg_op_policy_loss", "mg_op_policy_loss_makes_gradient", "mg_op_policy_loss_with_gradient", "mg_op_policy_loss_backward", "mg_op_policy_loss_rescale", "mg_op_sample_workspace", "mg_op_sample", "mg_op_advantages"]


class _AdvantagesArgs(C.Structure):
    _fields_ = [("steps", C.c_int64), ("envs", C.c_int64),
                ("reward", C.c_void_p), ("s_reward", C.c_int64 * 2), ("value", C.c_void_p), ("s_value", C.c_int64 * 2),
                ("final_value", C.c_void_p), ("s_final", C.c_int64 * 2), ("terminated", C.c_void_p), ("s_term", C.c_int64 * 2),
                ("truncated", C.c_void_p), ("s_trunc", C.c_int64 * 2), ("last_value", C.c_void_p), ("done0", C.c_void_p),
                ("advantage", C.c_void_p), ("ret", C.c_void_p), ("valid", C.c_void_p), ("gamma", C.c_double), ("lam", C.c_double),
                ("reward_dtype", C.c_int32), ("value_dtype", C.c_int32), ("next_step", C.c_int32), ("reserved", C.c_int32)]


_L = None


def _lib():
    global _L
    if _L is None:
        L = B.load()
        if not hasattr(L, "mg_op_linear"):
            raise B.MiniGridHipError("the loaded library does not hold the learning operators")
        vp, i, q, d = C.c_void_p, C.c_int, C.c_int64, C.c_double
        pq = C.POINTER(C.c_int64)
        L.mg_ops_last_error.argtypes, L.mg_ops_last_error.restype = [], C.c_char_p
        L.mg_op_linear_workspace.argtypes = [q, q, q, i, pq, pq, pq]
        L.mg_op_linear.argtypes = [i, vp, i, i, i, q, q, q, vp, q, vp, q, vp, vp, q, vp, q, vp, vp, q]
        L.mg_op_linear_dz_workspace.argtypes = [q, q, pq]
        L.mg_op_linear_dz.argtypes = [i, vp, i, i, q, q, vp, q, vp, vp, vp, vp, q]
        L.mg_op_linear_dx.argtypes = [i, vp, i, q, q, q, vp, q, vp, q, vp, vp, q]
        L.mg_op_linear_dw.argtypes = [i, vp, i, i, q, q, q, vp, q, vp, q, vp, vp, q]
        L.mg_op_policy_loss_workspace.argtypes = [q, q, pq]
        L.mg_op_policy_loss.argtypes = [i, vp, i, q, q, vp, q, vp, i, vp, vp, vp, vp, d, d, d, d, vp, vp, vp, q]
        L.mg_op_policy_loss_backward.argtypes = [i, vp, i, q, q, vp, q, vp, i, vp, d, vp, vp, vp]
        L.mg_op_policy_loss_makes_gradient.argtypes = [i, q]
        L.mg_op_policy_loss_with_gradient.argtypes = L.mg_op_policy_loss.argtypes + [vp]
        L.mg_op_policy_loss_rescale.argtypes = L.mg_op_policy_loss_backward.argtypes
        L.mg_op_sample_workspace.argtypes = [q, q, pq]
        L.mg_op_sample.argtypes = [i, vp, i, q, q, vp, q, vp, vp, vp, vp, q]
        L.mg_op_advantages.argtypes = [i, vp, C.POINTER(_AdvantagesArgs)]
        _L = L
    return _L


_X = None


def _ext():
    global _X
    if _X is None:
        import importlib.util

        from . import build as _build
        handle = _lib()._handle
        spec = importlib.util.spec_from_file_location("minigrid_amd._torch_ops", _build.build_torch_ops(missing_compiler_ok=True))
        x = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(x)
        x.bind_library(handle, B.MiniGridHipError)
        _X = x
    return _X


# ---- linear -----------------------------------------------------------------------------------------------------------------------------

def linear(x, weight, bias=None, *, activation: Optional[str] = None, residual=None):
    """act(x weight^T + bias) + residual as one operator.

    x (..., k): weight's dtype, or uint8 -- the observations as the environments hand them out (their values are exact in every float type here).
    weight (n, k), bias (n): float32, bfloat16 or float16; residual (..., n), the result's own shape and dtype.  activation: None, "relu", "tanh",
    "gelu" (x Phi(x) with the normal distribution function itself) or "silu".  Sums are held in 32 bits and the result is rounded once.

    Differentiable in x (unless bytes), weight, bias and residual, once.  For the backward pass of an activation the values in front of it are kept
    in weight's dtype (tanh: in float32, since its slope would lose most by that; relu without a residual: the result itself, which must then not be changed in place), and their gradient is rounded to it before the two products that use it (the matrix instructions take such operands);
    bias's gradient is summed before that rounding.  All sums run in a fixed order."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {[a for a in _ACTIVATIONS if a]} or None")
    return (_X or _ext()).linear(x, weight, bias, _ACTIVATIONS[activation], residual)


# ---- policy loss ------------------------------------------------------------------------------------------------------------------------

def policy_loss(logits, action, old_log_prob, advantage, *, mask=None, ref_log_prob=None, clip=0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0):
    """The clipped policy loss with a KL and an entropy term, averaged over the rows that count.

    logits (..., actions) float32, bfloat16 or float16, one row per transition (or token); action (...) uint8, int32 or int64; old_log_prob, advantage and
    ref_log_prob (...) float32; mask (...) bool or uint8, the rows that count (`advantages` returns it as `valid`).  With lp the log-probability of the
    action under the logits and q = exp(lp - old_log_prob), a row's loss is
        -min(q advantage, clamp(q, 1 - lo, 1 + hi) advantage) + kl_coef (exp(d) - d - 1) - entropy_coef H,       d = ref_log_prob - lp
    where clip is one number or the pair (lo, hi).  kl_coef needs ref_log_prob.

    Returns (loss, stats): stats are the means of the policy term, the KL term and the entropy, the share of clipped rows, and the number of rows that
    count.  Only the loss is differentiable, in the logits, once.  Rows that do not count are not read, whatever they hold, and get the gradient 0; with
    no row that counts everything is 0.  For more than 64 actions in rows of up to 160 KB of float32 or bfloat16 the gradient is made along with the loss, for the factor 1; a backward
    pass with another factor (a loss that was scaled) makes it anew.  Logits of -inf are closed actions.  A counted row whose action is not one of the columns makes the loss NaN."""
    lo, hi = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    return (_X or _ext()).policy_loss(logits, action, old_log_prob, advantage, mask, ref_log_prob, float(lo), float(hi), float(kl_coef), float(entropy_coef))


# ---- sampling ---------------------------------------------------------------------------------------------------------------------------

def sample_actions(logits, uniform=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One action per row of logits (..., actions), and its log-probability (float32).

    uniform (...) float32 in [0, 1): the action is the lowest one at which the running sum of the probabilities exceeds it (sums in 64 bits).  None: the most
    likely action, the lowest one of equals.  The actions are uint8 for up to 256 of them -- what `MiniGridVecEnv.step` takes --, int32 beyond.  Logits of
    -inf are never drawn.  A row with a NaN or +inf, or with nothing but -inf, gives action 0 and a NaN."""
    return (_X or _ext()).sample_actions(logits, uniform)


# ---- advantages -------------------------------------------------------------------------------------------------------------------------

def advantages(reward, value, last_value, terminated, truncated, *, gamma: float = 0.99, lam: float = 0.95, autoreset_mode: str = "next_step", done=None,
               final_value=None):
    """Generalised advantages of a rollout: (advantage, return, valid), each (steps, envs) -- float32, float32, bool.

    reward (steps, envs) float64 or float32, terminated and truncated (steps, envs) bool or uint8: what `step` returned, any strides.  value (steps, envs):
    the value of the observation each step was taken on; last_value (envs): of the observation behind the last step; float32, bfloat16 or float16.

    autoreset_mode="next_step" (the environments' default): the step behind an end of an episode only resets.  Such a row has valid = False and advantage 0,
    and the value at it is that of the observation the episode ended on, which a truncated step is bootstrapped from.  done (envs), bool or uint8: whether
    the step in front of the first row ended an episode.  "same_step": every row counts; a truncated step is bootstrapped from final_value (steps, envs), the
    value of the observation it ended on, or from 0 without it.  A terminated step is worth its reward.  return = advantage + value.

    The recurrence runs in 64 bits.  Not differentiable."""
    if autoreset_mode not in ("next_step", "same_step"):
        raise ValueError("autoreset_mode must be 'next_step' or 'same_step'")
    return (_X or _ext()).advantages(reward, value, last_value, terminated, truncated, float(gamma), float(lam), autoreset_mode == "next_step", done, final_value)
