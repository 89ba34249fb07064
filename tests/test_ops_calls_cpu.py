"""Calls that the learning operators refuse before they look at anything else, so that no GPU is needed to see it."""
import pytest

torch = pytest.importorskip("torch")

import minigrid_amd as mg


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


# every floating-point argument of every operator
TANGENTS = {
    "linear x": lambda f: mg.linear(f(t(2, 3)), t(4, 3)), "linear weight": lambda f: mg.linear(t(2, 3), f(t(4, 3))),
    "linear bias": lambda f: mg.linear(t(2, 3), t(4, 3), f(t(4))), "linear residual": lambda f: mg.linear(t(2, 3), t(4, 3), residual=f(t(2, 4))),
    "loss logits": lambda f: mg.policy_loss(f(t(2, 7)), t(2, dtype=torch.int64), t(2), t(2)),
    "loss old_log_prob": lambda f: mg.policy_loss(t(2, 7), t(2, dtype=torch.int64), f(t(2)), t(2)),
    "loss advantage": lambda f: mg.policy_loss(t(2, 7), t(2, dtype=torch.int64), t(2), f(t(2))),
    "loss ref_log_prob": lambda f: mg.policy_loss(t(2, 7), t(2, dtype=torch.int64), t(2), t(2), ref_log_prob=f(t(2))),
    "draw logits": lambda f: mg.sample_actions(f(t(2, 7))), "draw uniform": lambda f: mg.sample_actions(t(2, 7), f(t(2))),
    "advantages reward": lambda f: mg.advantages(f(t(2, 3)), t(2, 3), t(3), t(2, 3).bool(), t(2, 3).bool()),
    "advantages value": lambda f: mg.advantages(t(2, 3), f(t(2, 3)), t(3), t(2, 3).bool(), t(2, 3).bool()),
    "advantages last_value": lambda f: mg.advantages(t(2, 3), t(2, 3), f(t(3)), t(2, 3).bool(), t(2, 3).bool()),
    "advantages final_value": lambda f: mg.advantages(t(2, 3), t(2, 3), t(3), t(2, 3).bool(), t(2, 3).bool(), autoreset_mode="same_step", final_value=f(t(2, 3))),
}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", list(TANGENTS))
def test_a_tangent_is_refused(name, grad):
    """there is no forward-mode derivative: a result without a tangent would be taken for a constant (torch.no_grad() does not turn forward mode off)"""
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(ValueError, match="forward-mode"):
            TANGENTS[name](lambda v: fw.make_dual(v, torch.ones_like(v)))


CALLS = {
    "linear": (lambda x: mg.linear(x, t(4, 3)), t(2, 3)), "policy_loss": (lambda x: mg.policy_loss(x, t(2, dtype=torch.int64), t(2), t(2)), t(2, 7)),
    "sample_actions": (lambda x: mg.sample_actions(x), t(2, 7)), "advantages": (lambda x: mg.advantages(x, x, t(3), t(2, 3).bool(), t(2, 3).bool()), t(2, 3)),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_a_trace_is_refused(name):
    """a trace would record the result's allocation and not the operator, and return uninitialised memory"""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, x = CALLS[name]
    with pytest.raises(ValueError, match="traced"):
        torch.jit.trace(f, (x,))
    with pytest.raises(ValueError, match="traced"):
        make_fx(f)(x)
    with pytest.raises(ValueError, match="no CPU fallback"):         # (not being traced, the call comes as far as its arguments)
        f(x)


@pytest.mark.parametrize("name", list(CALLS))
def test_tensors_without_memory_are_refused(name):
    """a fake tensor says that it is on the GPU and holds nothing that a kernel could read"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    f, x = CALLS[name]
    with FakeTensorMode(), torch.device("cuda"), pytest.raises(ValueError, match="has no memory"):
        f(torch.empty(x.shape))


def test_assembly_names_the_special_registers_that_it_writes():
    """a register that an asm statement writes and does not name may hold a value of the compiler's: m0 (the LDS address of a load into LDS) among them"""
    import glob
    import os
    import re

    from conftest import ROOT
    found = 0
    for path in glob.glob(os.path.join(ROOT, "minigrid_amd", "csrc", "ops", "*")):
        if not path.endswith((".h", ".hip", ".inc")):
            continue
        for m in re.finditer(r"\basm\s+volatile\s*\((.*?)\);", open(path).read(), re.S):
            text = m.group(1)
            for reg in ("m0", "vcc", "scc", "exec"):
                if re.search(r"\bs_mov_b\d+ +%s\b" % reg, text):
                    found += 1
                    assert '"%s"' % reg in text.split(":")[-1], (os.path.basename(path), text)
    assert found


def test_seeds_of_rollouts_are_their_own():
    from minigrid_amd.vector_env import _draw_seed
    assert _draw_seed(7, 0, 0) == 7 and _draw_seed(-3, 0, 0) == -3
    seen = {_draw_seed(s, t, b) for s in (0, 1, 2, -1, 2 ** 63) for t in (0, 1, 2, 128, 256, 2 ** 31) for b in (0, 1, 64, 2 ** 20)}
    assert len(seen) == 5 * 6 * 4 and all(-2 ** 63 <= v < 2 ** 64 for v in seen)
