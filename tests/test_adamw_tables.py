"""C calls whose tensors take more than one launch are refused as a whole, before
the first one (no GPU needed: host addresses that no launch may see)."""
import ctypes

import pytest

from repo_b200 import _native as nat
from test_adamw_refusals import CS_ERR_ARG, CS_OK, CGrad, CTensor, _group, _tensor

BAD = (dict(exp_avg=None), dict(exp_avg_sq=None), dict(param=None), dict(grad=None))


def _call(name, tensors):
    t = (CTensor * len(tensors))(*tensors)
    g = (type(_group()) * 1)(_group())
    args = [ctypes.addressof(t), len(tensors)]
    if name != "cs_adamw8_moments":
        args += [ctypes.addressof(g), 1, None]
    if name == "cs_adamw8_step":
        args.append(7)
    if name != "cs_adamw8_moments":
        args.append(None)
    return nat.call(name, *args, None)


@pytest.mark.parametrize("name,bad", [
    *(("cs_adamw_step", b) for b in (*BAD, dict(exp_avg=1026), dict(exp_avg_sq=2049))),
    *((n, b) for n in ("cs_adamw8_step", "cs_adamw8_moments")
      for b in (*BAD, dict(exp_avg_scales=None), dict(exp_avg_sq_scales=None)))])
def test_a_bad_tensor_behind_a_full_table_is_refused_before_any_launch(name, bad):
    assert _call(name, [_tensor()] * 1300 + [_tensor(**bad)]) == CS_ERR_ARG


def test_a_first_place_below_zero_is_refused():
    t, g = (CTensor * 1)(_tensor()), (type(_group()) * 1)(_group())
    for place, tensor, want in ((-1, _tensor(), CS_ERR_ARG), (5, _tensor(numel=0), CS_OK)):
        t[0] = tensor
        assert nat.call("cs_adamw8_step_at", ctypes.addressof(t), 1, ctypes.addressof(g), 1, None,
                        7, place, None, None) == want


@pytest.mark.parametrize("name", ["cs_adamw_step_counted", "cs_adamw8_step_counted"])
def test_counted_steps_refuse_missing_counters_and_workspaces(name):
    t = (CTensor * 600)(*[_tensor() for _ in range(600)])
    g = (type(_group()) * 1)(_group(step=0))  # the host's count is not read
    good = [256 + 8 * i for i in range(600)]

    def call(steps, work=4096, count=600, place=0):
        steps = steps and (ctypes.c_void_p * 600)(*steps)
        args = [ctypes.addressof(t), count, ctypes.addressof(g), 1,
                steps and ctypes.addressof(steps), work]
        if name == "cs_adamw8_step_counted":
            args += [7, place]
        return nat.call(name, *args, None, None)
    assert call(good[:-1] + [None]) == CS_ERR_ARG
    assert call(good[:-1] + [260]) == CS_ERR_ARG
    assert call(None) == CS_ERR_ARG
    assert call(good, work=None) == CS_ERR_ARG
    assert call(good, work=4098) == CS_ERR_ARG
    assert call(good, count=-1) == CS_ERR_ARG
    assert call(good, count=0) == CS_OK
    if name == "cs_adamw8_step_counted":
        assert call(good, place=-1) == CS_ERR_ARG
    t[599].exp_avg = None
    assert call(good) == CS_ERR_ARG


def test_misaligned_device_scalars_are_refused():
    g = (type(_group()) * 1)(_group())
    t = (CTensor * 1)(_tensor())
    at, gt = ctypes.addressof(t), ctypes.addressof(g)
    for name, more in (("cs_adamw_step", ()), ("cs_adamw8_step", (7,))):
        assert nat.call(name, at, 1, gt, 1, None, *more, 66, None) == CS_ERR_ARG  # grad_scale
        assert nat.call(name, at, 1, gt, 1, 66, *more, None, None) == CS_ERR_ARG  # coef
        bad = (type(_group()) * 1)(_group(lr_device=66))
        assert nat.call(name, at, 1, ctypes.addressof(bad), 1, None, *more, None,
                        None) == CS_ERR_ARG
    for step, coef in ((260, 64), (256, 66)):
        steps = (ctypes.c_void_p * 1)(step)
        assert nat.call("cs_adamw_advance", ctypes.addressof(steps), gt, 1, 0, coef,
                        None) == CS_ERR_ARG
    n = (CGrad * 1)(CGrad(256, 1000, 0, 0))
    for norm, scale in ((66, 64), (64, 66)):
        assert nat.call("cs_grad_norm", ctypes.addressof(n), 1, 1.0, 1e-6, norm, scale, None,
                        None) == CS_ERR_ARG
