"""The learning operators where no GPU is needed: the library exports what the header declares, and calls that cannot be right are refused -- by the
binding before anything reaches the library, and by the C entries before anything reaches the device."""
import ctypes as C
import os
import re

import pytest

torch = pytest.importorskip("torch")

import minigrid_amd as mg
from conftest import ROOT
from minigrid_amd import _binding as B
from minigrid_amd import ops


def test_library_exports_every_declared_operator():
    header = open(os.path.join(ROOT, "include", "minigrid_ops.h")).read()
    declared = set(re.findall(r"MG_API\s+(?:const char\*|int)\s+(mg_\w+)\s*\(", header))
    assert declared == set(ops.SYMBOLS)
    L = ops._lib()
    for name in declared:
        assert hasattr(L, name), name
    args = re.search(r"typedef struct mg_advantages_args \{(.*?)\} mg_advantages_args;", header, re.S).group(1)
    names = re.findall(r"(\w+)(?:\[2\])?\s*[;,]", args)
    assert names == [f[0] for f in ops._AdvantagesArgs._fields_]
    assert C.sizeof(ops._AdvantagesArgs) == 208        # 2 sizes, 5 strided arrays (24 bytes each), 5 pointers, 2 doubles, 4 numbers of 32 bits


def test_names_are_public_and_lazy():
    assert mg.linear is ops.linear and mg.policy_loss is ops.policy_loss and mg.sample_actions is ops.sample_actions and mg.advantages is ops.advantages
    with pytest.raises(AttributeError):
        mg.no_such_name


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("call", [
    lambda: mg.linear(t(2, 3), t(4, 3)), lambda: mg.policy_loss(t(2, 7), t(2, dtype=torch.int64), t(2), t(2)), lambda: mg.sample_actions(t(2, 7)),
    lambda: mg.advantages(t(2, 3), t(2, 3), t(3), t(2, 3, dtype=torch.bool), t(2, 3, dtype=torch.bool))])
def test_no_cpu_fallback(call):
    with pytest.raises(ValueError, match="no CPU fallback"):
        call()


def test_not_a_tensor():
    with pytest.raises(TypeError):
        mg.linear([[1.0]], [[1.0]])


def _rc(rc, text):
    assert rc == B.MG_ERR_INVALID, rc
    assert text in ops._lib().mg_ops_last_error().decode(), ops._lib().mg_ops_last_error()


def test_c_entries_refuse_before_the_device_is_touched():
    """(addresses that were never allocated: an entry that did not refuse would have no device here, or fault)"""
    L, p = ops._lib(), 4096
    lin = lambda **k: L.mg_op_linear(*[{**dict(dev=0, st=None, dt=0, xdt=0, act=0, rows=4, k=8, n=8, x=p, ldx=8, w=p, ldw=8, b=None, r=None, ldr=0, y=p, ldy=8, z=None, ws=None,
                                               wsb=0), **k}[q] for q in "dev st dt xdt act rows k n x ldx w ldw b r ldr y ldy z ws wsb".split()])
    _rc(lin(dt=3), "dtype must be")
    _rc(lin(xdt=1), "w's type or be bytes")
    _rc(lin(act=5), "unknown activation")
    _rc(lin(k=0), "sizes must be")
    _rc(lin(rows=-1), "sizes must be")
    _rc(lin(rows=1 << 31), "sizes must be")
    _rc(lin(x=None), "must not be NULL")
    _rc(lin(ldx=7), "row stride")
    _rc(lin(r=p, ldr=7), "row stride")
    assert lin(rows=0) == B.MG_OK
    need = C.c_int64()
    assert L.mg_op_linear_workspace(40, 4096, 8, 0, C.byref(need), None, None) == B.MG_OK and need.value > 0
    _rc(L.mg_op_linear_dz(0, None, 0, 3, 4, 8, p, 8, None, p, None, None, 0), "in front of the activation")
    _rc(L.mg_op_linear_dz(0, None, 0, 0, 4, 8, p, 7, None, p, None, None, 0), "row stride")
    _rc(L.mg_op_linear_dx(0, None, 0, 4, 8, 8, p, 8, None, 8, p, None, 0), "NULL")
    _rc(L.mg_op_linear_dw(0, None, 0, 4, 4, 8, 8, p, 8, p, 8, p, None, 0), "w's type")
    loss = lambda dt=0, rows=4, vocab=7, ld=7, action=p, adt=6, out=p, ws=p, wsb=1 << 20: L.mg_op_policy_loss(
        0, None, dt, rows, vocab, p, ld, action, adt, p, p, None, None, 0.2, 0.2, 0.0, 0.0, out, None, ws, wsb)
    _rc(loss(dt=3), "logits must be")
    _rc(loss(vocab=0, ld=0), "sizes must be")
    _rc(loss(ld=6), "row stride")
    _rc(loss(adt=0), "action must be")
    _rc(loss(action=None), "must not be NULL")
    _rc(loss(ws=None), "workspace")
    _rc(loss(wsb=8), "workspace")
    _rc(L.mg_op_policy_loss_backward(0, None, 0, 4, 7, p, 7, p, 6, None, 0.0, None, p, p), "NULL")
    # the gradient comes with the loss for rows of more than 64 columns and at most 160 KB
    with_gradient = lambda dt, vocab: L.mg_op_policy_loss_with_gradient(0, None, dt, 4, vocab, p, vocab, p, 6, p, p, None, None, 0.2, 0.2, 0.0, 0.0, p, None, p, 1 << 20, p)
    for dt, vocab, makes in ((0, 7, 0), (0, 64, 0), (0, 65, 1), (0, 40960, 1), (0, 40961, 0), (1, 81920, 1), (1, 81921, 0)):
        assert L.mg_op_policy_loss_makes_gradient(dt, vocab) == makes, (dt, vocab)
        if not makes:
            _rc(with_gradient(dt, vocab), "no gradient comes with the loss")
            _rc(L.mg_op_policy_loss_rescale(0, None, dt, 4, vocab, p, vocab, p, 6, None, 0.0, p, p, p), "no gradient comes with the loss")
    _rc(L.mg_op_policy_loss_rescale(0, None, 0, 4, 65, p, 65, p, 6, None, 0.0, None, p, p), "NULL")
    _rc(L.mg_op_sample(0, None, 0, 4, 7, p, 6, None, p, p, None, 0), "row stride")
    _rc(L.mg_op_sample(0, None, 0, 4, 7, p, 7, None, None, p, None, 0), "NULL")
    _rc(L.mg_op_sample(0, None, 0, 4, 3000, p, 3000, None, p, p, None, 0), "workspace")
    assert L.mg_op_sample(0, None, 0, 0, 7, None, 7, None, None, None, None, 0) == B.MG_OK
    _rc(L.mg_op_advantages(0, None, None), "args")
    a = ops._AdvantagesArgs(steps=2, envs=3)
    _rc(L.mg_op_advantages(0, None, C.byref(a)), "NULL")
    two = (C.c_int64 * 2)(3, 1)
    full = dict(steps=2, envs=3, reward=p, s_reward=two, value=p, s_value=two, terminated=p, s_term=two, truncated=p, s_trunc=two, last_value=p, advantage=p, ret=p, valid=p,
                reward_dtype=4, value_dtype=0, next_step=1)
    _rc(L.mg_op_advantages(0, None, C.byref(ops._AdvantagesArgs(**dict(full, reward_dtype=1)))), "reward must be")
    _rc(L.mg_op_advantages(0, None, C.byref(ops._AdvantagesArgs(**dict(full, value_dtype=4)))), "value must be")
    _rc(L.mg_op_advantages(0, None, C.byref(ops._AdvantagesArgs(**dict(full, final_value=p)))), "same-step")
    assert L.mg_op_advantages(0, None, C.byref(ops._AdvantagesArgs(steps=0, envs=3))) == B.MG_OK


def test_without_a_device_the_entries_say_so():
    if B.load().mg_device_count() > 0:
        pytest.skip("GPU present")
    p = 4096
    assert ops._lib().mg_op_sample(0, None, 0, 4, 7, p, 7, None, p, p, None, 0) == B.MG_ERR_NO_DEVICE
