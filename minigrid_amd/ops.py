"""The learning operators: what turns the batched environments' observations into actions and their trajectories into a gradient.

    linear          y = act(x W^T + b) + r, x may be the byte observations themselves; gradients of x, W, b and r
    sample_actions  one action per row of logits from one uniform number (or the greedy one), with its log-probability
    advantages      generalised advantages of a rollout, aware of the environments' autoreset
    policy_loss     the clipped policy loss with KL and entropy terms; gradient of the logits

All of them take torch tensors on an MI355X and run hand-written kernels of libminigrid_hip.so (include/minigrid_ops.h) on the tensors' device and its
current stream, in the manner of torch's own operators: nothing synchronises, results are new tensors, a call may be captured into a graph.  There is no
CPU fallback.  `MiniGridVecEnv.rollout(policy=...)` and `minigrid_amd.policy.ActorCritic` are built from them.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _binding as B

_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.uint8: 3, torch.float64: 4, torch.int32: 5, torch.int64: 6}
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_ACTIVATIONS = {None: 0, "relu": 1, "tanh": 2, "gelu": 3, "silu": 4}

# every symbol include/minigrid_ops.h declares
SYMBOLS = ["mg_ops_last_error", "mg_op_linear_workspace", "mg_op_linear", "mg_op_linear_dz_workspace", "mg_op_linear_dz", "mg_op_linear_dx", "mg_op_linear_dw",
           "mg_op_policy_loss_workspace", "mg_op_policy_loss", "mg_op_policy_loss_backward", "mg_op_sample", "mg_op_advantages"]


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
        L.mg_op_policy_loss_backward.argtypes = [i, vp, i, q, q, vp, q, vp, i, vp, d, vp, vp, vp, vp]
        L.mg_op_sample.argtypes = [i, vp, i, q, q, vp, q, vp, vp, vp]
        L.mg_op_advantages.argtypes = [i, vp, C.POINTER(_AdvantagesArgs)]
        _L = L
    return _L


def _check(rc: int):
    if rc != B.MG_OK:
        msg = (_lib().mg_ops_last_error() or b"").decode(errors="replace")
        if rc == B.MG_ERR_INVALID:
            raise ValueError(msg)
        raise B.MiniGridHipError(f"libminigrid_hip error {rc}: {msg}")


def _stream(device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _on_gpu(name, t, device=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU: minigrid_amd has no CPU fallback")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.layout is not torch.strided:
        raise ValueError(f"{name} must be a dense tensor")


def _matrix(t, cols):
    """t as (rows, cols) with contiguous columns and rows that do not overlap: a view where the strides allow it, else a copy."""
    t = t.reshape(-1, cols)
    if (cols > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t


def _ld(t):
    return max(t.stride(0), t.shape[1])          # (the stride of a single row means nothing)


def _scratch(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


# ---- linear -----------------------------------------------------------------------------------------------------------------------------

def _linear_forward(x, w, b, act, r, want_z):
    L, dev, (rows, k), n = _lib(), w.device, x.shape, w.shape[0]
    y = torch.empty((rows, n), dtype=w.dtype, device=dev)
    z = torch.empty((rows, n), dtype=w.dtype, device=dev) if want_z else None
    need = C.c_int64()
    _check(L.mg_op_linear_workspace(rows, k, n, _DT[w.dtype], C.byref(need), None, None))
    ws = _scratch(need.value, dev)
    _check(L.mg_op_linear(dev.index, _stream(dev), _DT[w.dtype], _DT[x.dtype], act, rows, k, n, _ptr(x), _ld(x), _ptr(w), _ld(w), _ptr(b), _ptr(r),
                          0 if r is None else _ld(r), _ptr(y), n, _ptr(z), _ptr(ws), need.value))
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, r, act):
        k, n = w.shape[1], w.shape[0]
        x2, w2 = _matrix(x, k), _matrix(w, k)
        y, z = _linear_forward(x2, w2, None if b is None else b.contiguous(), act, None if r is None else _matrix(r, n), act != 0)
        ctx.save_for_backward(x2, w2, z)
        ctx.act, ctx.shapes = act, (x.shape, None if r is None else r.shape)
        return y.view(x.shape[:-1] + (n,))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, z = ctx.saved_tensors
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        L, dev, dt, (rows, k), n = _lib(), w.device, _DT[w.dtype], x.shape, w.shape[0]
        g = _matrix(dy, n)
        dx = dw = db = None
        need_dx, need_dw = C.c_int64(), C.c_int64()
        _check(L.mg_op_linear_workspace(rows, k, n, dt, None, C.byref(need_dx), C.byref(need_dw)))
        if want_b or (ctx.act and (want_x or want_w)):
            need = C.c_int64()
            if want_b:
                db = torch.empty((n,), dtype=w.dtype, device=dev)
                _check(L.mg_op_linear_dz_workspace(rows, n, C.byref(need)))
            ws = _scratch(need.value, dev)
            dz = torch.empty((rows, n), dtype=w.dtype, device=dev) if ctx.act and (want_x or want_w) else None
            _check(L.mg_op_linear_dz(dev.index, _stream(dev), dt, ctx.act, rows, n, _ptr(g), _ld(g), _ptr(z), _ptr(dz), _ptr(db), _ptr(ws), need.value))
            if dz is not None:
                g = dz
        if want_x:
            dx = torch.empty((rows, k), dtype=w.dtype, device=dev)
            ws = _scratch(need_dx.value, dev)
            _check(L.mg_op_linear_dx(dev.index, _stream(dev), dt, rows, k, n, _ptr(g), _ld(g), _ptr(w), _ld(w), _ptr(dx), _ptr(ws), need_dx.value))
            dx = dx.view(ctx.shapes[0])
        if want_w:
            dw = torch.empty((n, k), dtype=w.dtype, device=dev)
            ws = _scratch(need_dw.value, dev)
            _check(L.mg_op_linear_dw(dev.index, _stream(dev), dt, _DT[x.dtype], rows, k, n, _ptr(g), _ld(g), _ptr(x), _ld(x), _ptr(dw), _ptr(ws), need_dw.value))
        return dx, dw, db, dy if want_r else None, None


def linear(x, weight, bias=None, *, activation: Optional[str] = None, residual=None):
    """act(x weight^T + bias) + residual as one operator.

    x (..., k): weight's dtype, or uint8 -- the observations as the environments hand them out (their values are exact in every float type here).
    weight (n, k), bias (n): float32, bfloat16 or float16; residual (..., n), the result's own shape and dtype.  activation: None, "relu", "tanh",
    "gelu" (x Phi(x) with the normal distribution function itself) or "silu".  Sums are held in 32 bits and the result is rounded once.

    Differentiable in x (unless bytes), weight, bias and residual, once.  For the backward pass of an activation the values in front of it are kept
    in weight's dtype, and their gradient is rounded to it before the two products that use it (the matrix instructions take such operands);
    bias's gradient is summed before that rounding.  All sums run in a fixed order."""
    _on_gpu("weight", weight)
    dev = weight.device
    _on_gpu("x", x, dev)
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {[a for a in _ACTIVATIONS if a]} or None")
    if weight.dtype not in _FLOATS or weight.dim() != 2 or weight.numel() == 0:
        raise ValueError("weight must be (n, k) of float32, bfloat16 or float16, n and k at least 1")
    n, k = weight.shape
    if x.dtype not in (weight.dtype, torch.uint8):
        raise ValueError(f"x must be {weight.dtype} (weight's dtype) or uint8, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"x must have {k} columns, got shape {tuple(x.shape)}")
    if bias is not None:
        _on_gpu("bias", bias, dev)
        if bias.dtype != weight.dtype or bias.shape != (n,):
            raise ValueError(f"bias must be ({n},) of {weight.dtype}")
    if residual is not None:
        _on_gpu("residual", residual, dev)
        if residual.dtype != weight.dtype or residual.shape != x.shape[:-1] + (n,):
            raise ValueError(f"residual must be {tuple(x.shape[:-1]) + (n,)} of {weight.dtype}: the result's shape, nothing is broadcast")
    act = _ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        return _Linear.apply(x, weight, bias, residual, act)
    y, _ = _linear_forward(_matrix(x, k), _matrix(weight, k), None if bias is None else bias.contiguous(), act,
                           None if residual is None else _matrix(residual, n), False)
    return y.view(x.shape[:-1] + (n,))


# ---- policy loss ------------------------------------------------------------------------------------------------------------------------

class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, action, old, adv, ref, mask, lo, hi, kl, ent):
        vocab = logits.shape[-1]
        x = _matrix(logits, vocab)
        keep = ctx.needs_input_grad[0]
        out, save = _loss_forward(x, action, old, adv, ref, mask, lo, hi, kl, ent, keep)
        loss, stats = out[0], out[1:]
        ctx.mark_non_differentiable(stats)
        if keep:
            ctx.save_for_backward(x, action, mask, out, save)
            ctx.ent, ctx.shape = ent, logits.shape
        return loss, stats

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _):
        x, action, mask, out, save = ctx.saved_tensors
        L, dev, (rows, vocab) = _lib(), x.device, x.shape
        d = torch.empty((rows, vocab), dtype=x.dtype, device=dev)
        _check(L.mg_op_policy_loss_backward(dev.index, _stream(dev), _DT[x.dtype], rows, vocab, _ptr(x), _ld(x), _ptr(action), _DT[action.dtype], _ptr(mask),
                                            ctx.ent, _ptr(out), _ptr(save), _ptr(g), _ptr(d)))
        return (d.view(ctx.shape),) + (None,) * 9


def _loss_forward(x, action, old, adv, ref, mask, lo, hi, kl, ent, keep):
    L, dev, (rows, vocab) = _lib(), x.device, x.shape
    out = torch.empty(6, dtype=torch.float32, device=dev)
    save = torch.empty((rows, 2), dtype=torch.float64, device=dev) if keep else None
    need = C.c_int64()
    _check(L.mg_op_policy_loss_workspace(rows, vocab, C.byref(need)))
    ws = _scratch(need.value, dev)
    _check(L.mg_op_policy_loss(dev.index, _stream(dev), _DT[x.dtype], rows, vocab, _ptr(x), _ld(x), _ptr(action), _DT[action.dtype], _ptr(old), _ptr(adv), _ptr(ref),
                               _ptr(mask), lo, hi, kl, ent, _ptr(out), _ptr(save), _ptr(ws), need.value))
    return out, save


def _per_row(name, t, shape, dtypes, device):
    _on_gpu(name, t, device)
    if t.shape != shape or t.dtype not in dtypes:
        raise ValueError(f"{name} must be {tuple(shape)} of {' or '.join(str(d) for d in dtypes)}, got {tuple(t.shape)} of {t.dtype}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} is a constant of this operator and gets no gradient: pass {name}.detach()")
    t = t.detach()
    if t.dtype is torch.bool:
        t = t.view(torch.uint8)
    return t.reshape(-1).contiguous()


def policy_loss(logits, action, old_log_prob, advantage, *, mask=None, ref_log_prob=None, clip=0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0):
    """The clipped policy loss with a KL and an entropy term, averaged over the rows that count.

    logits (..., actions) float32, bfloat16 or float16, one row per transition (or token); action (...) uint8, int32 or int64; old_log_prob, advantage and
    ref_log_prob (...) float32; mask (...) bool or uint8, the rows that count (`advantages` returns it as `valid`).  With lp the log-probability of the
    action under the logits and q = exp(lp - old_log_prob), a row's loss is
        -min(q advantage, clamp(q, 1 - lo, 1 + hi) advantage) + kl_coef (exp(d) - d - 1) - entropy_coef H,       d = ref_log_prob - lp
    where clip is one number or the pair (lo, hi).  kl_coef needs ref_log_prob.

    Returns (loss, stats): stats are the means of the policy term, the KL term and the entropy, the share of clipped rows, and the number of rows that
    count.  Only the loss is differentiable, in the logits, once.  Rows that do not count are not read, whatever they hold, and get the gradient 0; with
    no row that counts everything is 0.  Logits of -inf are closed actions.  A counted row whose action is not one of the columns makes the loss NaN."""
    _on_gpu("logits", logits)
    dev = logits.device
    if logits.dtype not in _FLOATS or logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must be (..., actions) of float32, bfloat16 or float16")
    lo, hi = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    lo, hi, kl, ent = float(lo), float(hi), float(kl_coef), float(entropy_coef)
    if not (0.0 <= lo <= 1.0 and hi >= 0.0):
        raise ValueError("clip must be a number in 0..1 or a pair (lo, hi) with lo in 0..1 and hi >= 0")
    if kl != 0.0 and ref_log_prob is None:
        raise ValueError("kl_coef needs ref_log_prob")
    shape = logits.shape[:-1]
    action = _per_row("action", action, shape, (torch.uint8, torch.int32, torch.int64), dev)
    old = _per_row("old_log_prob", old_log_prob, shape, (torch.float32,), dev)
    adv = _per_row("advantage", advantage, shape, (torch.float32,), dev)
    ref = None if ref_log_prob is None else _per_row("ref_log_prob", ref_log_prob, shape, (torch.float32,), dev)
    mask = None if mask is None else _per_row("mask", mask, shape, (torch.bool, torch.uint8), dev)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _PolicyLoss.apply(logits, action, old, adv, ref, mask, lo, hi, kl, ent)
    out, _ = _loss_forward(_matrix(logits, logits.shape[-1]), action, old, adv, ref, mask, lo, hi, kl, ent, False)
    return out[0], out[1:]


# ---- sampling ---------------------------------------------------------------------------------------------------------------------------

def sample_actions(logits, uniform=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One action per row of logits (..., actions), and its log-probability (float32).

    uniform (...) float32 in [0, 1): the action is the lowest one at which the running sum of the probabilities exceeds it (sums in 64 bits).  None: the most
    likely action, the lowest one of equals.  The actions are uint8 for up to 256 of them -- what `MiniGridVecEnv.step` takes --, int32 beyond.  Logits of
    -inf are never drawn.  A row with a NaN or +inf, or with nothing but -inf, gives action 0 and a NaN."""
    _on_gpu("logits", logits)
    dev = logits.device
    if logits.dtype not in _FLOATS or logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must be (..., actions) of float32, bfloat16 or float16")
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("a draw has no gradient: pass logits.detach(), or call it under torch.no_grad()")
    shape, vocab = logits.shape[:-1], logits.shape[-1]
    u = None if uniform is None else _per_row("uniform", uniform, shape, (torch.float32,), dev)
    x = _matrix(logits, vocab)
    action = torch.empty(shape, dtype=torch.uint8 if vocab <= 256 else torch.int32, device=dev)
    lp = torch.empty(shape, dtype=torch.float32, device=dev)
    _check(_lib().mg_op_sample(dev.index, _stream(dev), _DT[x.dtype], x.shape[0], vocab, _ptr(x), _ld(x), _ptr(u), _ptr(action), _ptr(lp)))
    return action, lp


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
    _on_gpu("value", value)
    dev = value.device
    if autoreset_mode not in ("next_step", "same_step"):
        raise ValueError("autoreset_mode must be 'next_step' or 'same_step'")
    if value.dim() != 2 or value.dtype not in _FLOATS:
        raise ValueError("value must be (steps, envs) of float32, bfloat16 or float16")
    steps, envs = value.shape

    def grid(name, t, dtypes):
        _on_gpu(name, t, dev)
        if t.shape != (steps, envs) or t.dtype not in dtypes:
            raise ValueError(f"{name} must be {(steps, envs)} of {' or '.join(str(d) for d in dtypes)}, got {tuple(t.shape)} of {t.dtype}")
        return t.view(torch.uint8) if t.dtype is torch.bool else t

    if torch.is_grad_enabled() and any(t is not None and isinstance(t, torch.Tensor) and t.requires_grad for t in (reward, value, last_value, final_value)):
        raise ValueError("the advantages have no gradient: pass detached tensors, or call it under torch.no_grad()")
    flags = (torch.bool, torch.uint8)
    reward, terminated, truncated = grid("reward", reward, (torch.float64, torch.float32)), grid("terminated", terminated, flags), grid("truncated", truncated, flags)
    last_value = _per_row("last_value", last_value, (envs,), (value.dtype,), dev)
    if final_value is not None:
        if autoreset_mode != "same_step":
            raise ValueError("final_value belongs to autoreset_mode='same_step': with 'next_step' the rows themselves hold it")
        grid("final_value", final_value, (value.dtype,))
    if done is not None:
        if autoreset_mode != "next_step":
            raise ValueError("done belongs to autoreset_mode='next_step'")
        done = _per_row("done", done, (envs,), flags, dev)
    adv = torch.empty((steps, envs), dtype=torch.float32, device=dev)
    ret = torch.empty_like(adv)
    valid = torch.empty((steps, envs), dtype=torch.bool, device=dev)
    two = C.c_int64 * 2
    st = lambda t: two(0, 0) if t is None else two(*t.stride())
    a = _AdvantagesArgs(steps, envs, _ptr(reward), st(reward), _ptr(value), st(value), _ptr(final_value), st(final_value), _ptr(terminated), st(terminated),
                        _ptr(truncated), st(truncated), _ptr(last_value), _ptr(done), _ptr(adv), _ptr(ret), _ptr(valid), float(gamma), float(lam),
                        _DT[reward.dtype], _DT[value.dtype], int(autoreset_mode == "next_step"), 0)
    _check(_lib().mg_op_advantages(dev.index, _stream(dev), C.byref(a)))
    return adv, ret, valid
