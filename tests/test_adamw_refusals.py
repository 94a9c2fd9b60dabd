"""What the AdamW entry points refuse before any device work (no GPU needed)."""
import ctypes

import pytest
import torch

import manbo
from manbo import ops
from repo_b200 import _native as nat

CS_OK, CS_ERR_ARG = 0, 1


class CTensor(ctypes.Structure):
    _fields_ = [("param", ctypes.c_void_p), ("grad", ctypes.c_void_p),
                ("exp_avg", ctypes.c_void_p), ("exp_avg_sq", ctypes.c_void_p),
                ("exp_avg_scales", ctypes.c_void_p), ("exp_avg_sq_scales", ctypes.c_void_p),
                ("numel", ctypes.c_int64), ("dtype", ctypes.c_int32), ("group", ctypes.c_int32)]


class CGroup(ctypes.Structure):
    _fields_ = [("lr", ctypes.c_double), ("beta1", ctypes.c_double), ("beta2", ctypes.c_double),
                ("eps", ctypes.c_double), ("weight_decay", ctypes.c_double),
                ("step", ctypes.c_int64), ("lr_device", ctypes.c_void_p)]


class CGrad(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("numel", ctypes.c_int64), ("dtype", ctypes.c_int32),
                ("reserved", ctypes.c_int32)]


def _tensor(**kw):  # host addresses: every call here is refused before a launch
    f = dict(param=256, grad=512, exp_avg=1024, exp_avg_sq=2048, exp_avg_scales=4096,
             exp_avg_sq_scales=8192, numel=10, dtype=0, group=0)
    f.update(kw)
    return CTensor(**f)


def _group(**kw):
    f = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1, lr_device=None)
    f.update(kw)
    return CGroup(**f)


def _step(name, tensor, group=None, count=1, groups=1):
    t = (CTensor * 1)(tensor)
    g = (CGroup * 1)(group or _group())
    args = [ctypes.addressof(t), count, ctypes.addressof(g), groups, None]
    if name == "cs_adamw8_step":
        args.append(7)
    return nat.call(name, *args, None, None)


@pytest.mark.parametrize("name", ["cs_adamw_step", "cs_adamw8_step"])
def test_c_entries_refuse_bad_tables(name):
    for bad in (dict(numel=-1), dict(numel=(1 << 40) + 1), dict(dtype=3), dict(dtype=-1),
                dict(group=1), dict(group=-1), dict(param=None), dict(grad=None),
                dict(exp_avg=None), dict(exp_avg_sq=None), dict(param=258),
                dict(grad=513, dtype=1)):
        assert _step(name, _tensor(**bad)) == CS_ERR_ARG, bad
    for bad in (dict(beta1=1.0), dict(beta2=1.0), dict(beta1=-0.1), dict(beta2=float("nan")),
                dict(step=0)):
        assert _step(name, _tensor(), _group(**bad)) == CS_ERR_ARG, bad
    assert _step(name, _tensor(), count=-1) == CS_ERR_ARG
    assert _step(name, _tensor(), count=(1 << 22) + 1) == CS_ERR_ARG
    assert _step(name, _tensor(), groups=0) == CS_ERR_ARG
    assert _step(name, _tensor(), groups=17) == CS_ERR_ARG
    # nothing to do: no launch, no error
    assert _step(name, _tensor(numel=0, param=None)) == CS_OK
    assert _step(name, _tensor(), count=0) == CS_OK


def test_c_entries_refuse_missing_scales_counters_and_workspaces():
    assert _step("cs_adamw8_step", _tensor(exp_avg_scales=None)) == CS_ERR_ARG
    assert _step("cs_adamw8_step", _tensor(exp_avg_sq_scales=None)) == CS_ERR_ARG
    t = (CTensor * 1)(_tensor(dtype=1))
    assert nat.call("cs_adamw8_moments", ctypes.addressof(t), 1, None) == CS_ERR_ARG
    t = (CTensor * 1)(_tensor(param=None))
    assert nat.call("cs_adamw8_moments", ctypes.addressof(t), 1, None) == CS_ERR_ARG
    g = (CGroup * 2)(_group(), _group())
    same = (ctypes.c_void_p * 2)(256, 256)
    none = (ctypes.c_void_p * 1)(None)
    for steps, n, coef in ((same, 2, 64), (none, 1, 64), (same, 1, None), (same, 0, 64),
                           (same, 17, 64)):
        assert nat.call("cs_adamw_advance", ctypes.addressof(steps), ctypes.addressof(g), n, 0,
                        coef, None) == CS_ERR_ARG
    n = (CGrad * 1)(CGrad(256, 1 << 30, 0, 0))  # large enough to need a workspace
    at = ctypes.addressof(n)
    assert nat.call("cs_grad_norm_workspace_size", at, 1) >= 8
    assert nat.call("cs_grad_norm_workspace_size", at, 0) == 0
    for args in ((at, -1, 64, 64, 64), (None, 1, 64, 64, 64), (at, 1, None, 64, 64),
                 (at, 1, 64, 64, None), (at, 1, 64, 64, 68)):
        assert nat.call("cs_grad_norm", args[0], args[1], 1.0, 1e-6, *args[2:], None) == CS_ERR_ARG
    assert _step("cs_adamw_step", _tensor(exp_avg=1026)) == CS_ERR_ARG
    for bad in (CGrad(None, 4, 0, 0), CGrad(256, -4, 0, 0), CGrad(256, 4, 9, 0),
                CGrad(258, 4, 0, 0), CGrad(257, 4, 1, 0)):
        n = (CGrad * 1)(bad)
        assert nat.call("cs_grad_norm", ctypes.addressof(n), 1, 1.0, 1e-6, 64, 64, 64,
                        None) == CS_ERR_ARG
    few = (CGrad * 1)(CGrad(256, 1000, 0, 0))
    assert nat.call("cs_grad_norm_workspace_size", ctypes.addressof(few), 1) == 0


def _lists(k=2):
    return [[torch.zeros(4) for _ in range(k)] for _ in range(4)]


def test_operators_refuse_bad_arguments():
    p, g, m, v = _lists()
    with pytest.raises(ValueError, match="grads must have as many tensors as params \\(2\\), got 1"):
        ops.adamw_step(p, g[:1], m, v, step=1)
    with pytest.raises(ValueError, match="params must be a sequence of tensors"):
        ops.adamw_step(p[0], g, m, v, step=1)
    with pytest.raises(ValueError, match="params\\[0\\] must be a tensor"):
        ops.adamw_step([1], g[:1], m[:1], v[:1], step=1)
    for kw, msg in ((dict(step=0), "step must be >= 1"), (dict(step=1, lr=-1.0), "learning rate"),
                    (dict(step=1, betas=(1.0, 0.9)), "beta parameter at index 0"),
                    (dict(step=1, betas=(0.9, -0.1)), "beta parameter at index 1"),
                    (dict(step=1, eps=-1e-8), "epsilon"),
                    (dict(step=1, weight_decay=-1.0), "weight_decay"),
                    (dict(step=1, lr=float("nan")), "learning rate"),
                    (dict(step=torch.ones((), dtype=torch.int64)), "step must be an int"),
                    (dict(step=1, lr=torch.ones(())), "lr must be one float32 value")):
        with pytest.raises(ValueError, match=msg):
            ops.adamw_step(p, g, m, v, **kw)
        with pytest.raises(ValueError, match=msg):
            ops.adamw8_step(p, g, m, m, v, v, **kw)
    with pytest.raises(ValueError, match="params\\[0\\] must be a CUDA tensor"):
        ops.adamw_step(p, g, m, v, step=1)
    with pytest.raises(ValueError, match="params\\[0\\] must be a CUDA tensor"):
        ops.adamw8_step(p, g, m, m, v, v, step=1)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.grad_norm(g)
    with pytest.raises(ValueError, match="must not be empty"):
        ops.grad_norm([])
    with pytest.raises(ValueError, match="max_norm"):
        ops.grad_norm(g, max_norm=-1.0)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.adamw8_moments(m, m, v, v)
    ops.adamw_step([], [], [], [], step=1)  # nothing to do


def test_optimizer_validation():
    p = torch.zeros(3, requires_grad=True)
    for kw, msg in ((dict(lr=-1.0), "Invalid learning rate"), (dict(eps=-1.0), "Invalid epsilon"),
                    (dict(betas=(0.9, 1.0)), "Invalid beta parameter at index 1"),
                    (dict(weight_decay=-1.0), "Invalid weight_decay"),
                    (dict(max_grad_norm=-1.0), "Invalid max_grad_norm"),
                    (dict(state_bits=4), "state_bits must be 8 or 32"),
                    (dict(lr=torch.ones(())), "needs capturable")):
        with pytest.raises(ValueError, match=msg):
            manbo.AdamW([p], **kw)
    opt = manbo.AdamW([p])
    opt.step()  # no gradient yet: nothing to do
    p.grad = torch.ones(3)
    with pytest.raises(ValueError, match="CUDA"):
        opt.step()
    assert not opt.state[p]  # a refused step leaves no count behind


def test_optimizer_loads_state_without_casting_it():
    """Moments keep their types whatever the parameter's (host tensors here:
    loading needs no device)."""
    p = torch.zeros(5, 3, dtype=torch.bfloat16, requires_grad=True)
    q = torch.zeros(7, requires_grad=True)
    opt = manbo.AdamW([{"params": [p], "state_bits": 8}, {"params": [q], "lr": 0.5}])
    codes = torch.arange(15, dtype=torch.uint8).view(5, 3)
    saved = opt.state_dict()
    saved["state"] = {
        0: dict(exp_avg=codes, exp_avg_scales=torch.tensor([90], dtype=torch.uint8),
                exp_avg_sq=codes + 1, exp_avg_sq_scales=torch.tensor([80], dtype=torch.uint8),
                step=12),
        1: dict(exp_avg=torch.ones(7), exp_avg_sq=torch.full((7,), 2.0),
                step=torch.tensor(12.0))}
    opt.load_state_dict(saved)
    st = opt.state[p]
    assert st["exp_avg"].dtype == torch.uint8 and torch.equal(st["exp_avg"], codes)
    assert st["exp_avg"].data_ptr() != codes.data_ptr() and st["exp_avg_scales"].tolist() == [90]
    assert st["step"] == 12 and opt.state[q]["step"] == 12
    assert opt.state[q]["exp_avg"].dtype == torch.float32
    assert opt.param_groups[1]["lr"] == 0.5 and opt.param_groups[0]["state_bits"] == 8
    saved["state"][0]["exp_avg"] = codes.t().contiguous().t()
    with pytest.raises(ValueError, match="strides"):
        opt.load_state_dict(saved)
