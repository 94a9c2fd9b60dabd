"""manbo.AdamW.load_state_dict on host tensors (loading needs no device)."""
import copy

import pytest
import torch

import manbo


def _optimiser(**kw):
    p = torch.zeros(5, 3, requires_grad=True)
    q = torch.zeros(7, requires_grad=True)
    return (p, q), manbo.AdamW([{"params": [p], "state_bits": 8}, {"params": [q], "lr": 0.5}], **kw)


def _saved(opt, step=12):
    saved = opt.state_dict()
    codes = torch.arange(15, dtype=torch.uint8).view(5, 3)
    saved["state"] = {
        0: dict(exp_avg=codes, exp_avg_scales=torch.tensor([90], dtype=torch.uint8),
                exp_avg_sq=codes + 1, exp_avg_sq_scales=torch.tensor([80], dtype=torch.uint8),
                step=step),
        1: dict(exp_avg=torch.ones(7), exp_avg_sq=torch.full((7,), 2.0), step=step)}
    return saved


def test_a_pre_hook_changes_the_state_and_a_post_hook_sees_it():
    (p, q), opt = _optimiser()
    saved, seen = _saved(opt), []

    def pre(o, d):
        assert o is opt
        d = copy.deepcopy(d)
        d["state"][1]["exp_avg"].fill_(3.0)
        del d["state"][0]
        d["param_groups"][1]["lr"] = 0.25
        return d
    opt.register_load_state_dict_pre_hook(pre)
    opt.register_load_state_dict_post_hook(lambda o: seen.append(dict(o.state)))
    opt.load_state_dict(saved)
    assert not opt.state[p] and opt.state[q]["exp_avg"].tolist() == [3.0] * 7
    assert opt.param_groups[1]["lr"] == 0.25
    assert len(seen) == 1 and seen[0][q]["step"] == 12 and p not in seen[0]
    assert saved["state"][1]["exp_avg"].tolist() == [1.0] * 7
    opt.load_state_dict(saved)  # the hooks stay, none is left over
    assert len(seen) == 2 and len(opt._optimizer_load_state_dict_pre_hooks) == 1


def test_a_refused_load_changes_nothing():
    (p, q), opt = _optimiser()
    opt.load_state_dict(_saved(opt))
    kept = {k: {n: copy.deepcopy(x) for n, x in st.items()} for k, st in opt.state.items()}

    def strides(d):
        d["state"][0]["exp_avg"] = d["state"][0]["exp_avg"].t().contiguous().t()

    def kind(d):
        d["param_groups"][1]["amsgrad"] = True

    def groups(d):
        d["param_groups"] = d["param_groups"][:1]

    def fewer(d):
        d["param_groups"][1]["params"] = []
    for change in (strides, kind, groups, fewer):
        saved = _saved(opt, step=99)
        saved["param_groups"][1]["lr"] = 0.125
        change(saved)
        with pytest.raises(ValueError):
            opt.load_state_dict(saved)
        assert opt.param_groups[1]["lr"] == 0.5
        assert set(opt.state) == {p, q}
        for k, st in kept.items():
            assert set(opt.state[k]) == set(st)
            for n, x in st.items():
                y = opt.state[k][n]
                assert torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y
    opt.load_state_dict(_saved(opt, step=99))
    assert opt.state[p]["step"] == 99


def test_copies_of_an_optimiser_load_too():
    (p, q), opt = _optimiser()
    opt.load_state_dict(_saved(opt))
    other = copy.deepcopy(opt)
    ps = [x for g in other.param_groups for x in g["params"]]
    assert other.state[ps[0]]["step"] == 12
    other.load_state_dict(_saved(other, step=13))
    assert other.state[ps[0]]["step"] == 13 and opt.state[p]["step"] == 12
