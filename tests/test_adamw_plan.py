"""Which calls a step of manbo.AdamW makes: a stand-in for the binding records them,
on host tensors that say they are on a device (no GPU needed)."""
import pytest
import torch

import manbo
import manbo.optim


class OnDevice(torch.Tensor):
    """A host tensor that gives `where` as its device's index."""
    def get_device(self):
        return self.where


class Recorder:
    def __init__(self):
        self.calls = []

    def adamw_steps(self, calls, scale):
        assert scale is None
        self.calls.append(calls)


@pytest.fixture
def binding(monkeypatch):
    recorder = Recorder()
    monkeypatch.setattr(manbo.optim._ext, "load", lambda: recorder)
    return recorder


def _params(devices):
    out = []
    for d in devices:
        p = torch.zeros(300).as_subclass(OnDevice)
        p.where = d
        p.requires_grad_()
        p.grad = torch.ones(300)
        out.append(p)
    return out


def test_places_go_on_over_devices_and_launches(binding):
    """Calls of one seed: (first place, tensors) cover the step once; another seed
    starts anew."""
    ps = _params([0, 1] * 20)
    opt = manbo.AdamW([{"params": ps[i:i + 2], "lr": 1e-3 * (i + 1), "seed": 7 if i < 36 else 8}
                       for i in range(0, 40, 2)], state_bits=8)
    opt.step()
    (calls,) = binding.calls  # one binding call
    spans = {}
    for params, *_, seed, first in calls:
        assert len({p.get_device() for p in params}) == 1
        spans.setdefault(seed, []).append((first, first + len(params)))
    assert sorted(spans) == [7, 8]
    for seed, n in ((7, 36), (8, 4)):
        ends = sorted(spans[seed])
        assert ends[0][0] == 0 and ends[-1][1] == n
        assert all(a[1] == b[0] for a, b in zip(ends, ends[1:]))
    assert len(spans[7]) == 4  # two devices, 18 groups each: 16 and 2


@pytest.mark.parametrize("bits", [8, 32])
def test_capturable_parameters_of_a_group_are_one_call(binding, bits):
    """At whatever steps they are: the tensors' own counters go along, and no count
    is made on the host."""
    ps = _params([0] * 30)
    opt = manbo.AdamW(ps, state_bits=bits, capturable=True)
    for i in range(1, 30):
        ps[i].grad = None
    opt.step()
    for p in ps:
        p.grad = torch.ones(300)
    opt.step()
    (first,), (second,) = binding.calls
    assert len(first[0]) == 1 and len(second[0]) == 30 and len(second[4]) == 1
    assert len({x.data_ptr() for x in second[5]}) == 30
    assert all(opt.state[p]["step"] is x for p, x in zip(ps, second[5]))


def test_host_counts_rise_for_parameters_that_stepped(binding):
    ps = _params([0, 0, 0])
    opt = manbo.AdamW(ps)
    opt.step()
    ps[1].grad = None
    opt.step()
    ps[1].grad = torch.ones(300)
    opt.step()
    assert [opt.state[p]["step"] for p in ps] == [3, 2, 3]
    # the last step had parameters at two counts: a group for each, with its number
    assert sorted((g[0], g[6]) for g in binding.calls[2][0][4]) == [(1, 2), (2, 3)]
    assert binding.calls[2][0][5] is None
