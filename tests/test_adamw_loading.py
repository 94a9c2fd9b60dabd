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


def test_moments_of_16_bit_states_become_float32():
    p = torch.zeros(4, 6, dtype=torch.bfloat16).t().requires_grad_()
    opt = manbo.AdamW([p])
    old = torch.optim.AdamW([p], lr=0.5)
    p.grad = torch.randn(6, 4).bfloat16()
    old.step()
    opt.load_state_dict(old.state_dict())
    for k in ("exp_avg", "exp_avg_sq"):
        x = opt.state[p][k]
        assert x.dtype == torch.float32 and x.stride() == p.stride()
        assert torch.equal(x, old.state[p][k].float())
    assert opt.state[p]["step"] == 1 and opt.param_groups[0]["lr"] == 0.5


def test_states_that_a_step_could_not_take_are_refused():
    (p, q), opt = _optimiser()
    for i, change, msg in (
            (1, dict(exp_avg=torch.ones(8)), "exp_avg must have its parameter's shape"),
            (1, dict(exp_avg_sq=torch.ones(7, dtype=torch.uint8)), "state_bits=32"),
            (1, dict(exp_avg_sq=None), "exp_avg_sq"), (1, dict(step=None), "step"),
            (0, dict(exp_avg=torch.ones(5, 3)), "state_bits=8"),
            (0, dict(exp_avg_sq=torch.ones(5, 3)), "state_bits=8"),
            (0, dict(exp_avg_sq_scales=None), "exp_avg_sq_scales"),
            (0, dict(exp_avg_scales=torch.ones(2, dtype=torch.uint8)), "1 uint8 scales"),
            (0, dict(exp_avg_scales=torch.ones(1)), "1 uint8 scales"),
            (0, dict(exp_avg=torch.ones(3, 5, dtype=torch.uint8)), "parameter's shape")):
        saved = _saved(opt)
        for k, x in change.items():
            if x is None:
                del saved["state"][i][k]
            else:
                saved["state"][i][k] = x
        with pytest.raises(ValueError, match=msg):
            opt.load_state_dict(saved)
        assert not opt.state
    # a state of 32-bit moments for an optimiser that keeps 8-bit ones
    old = torch.optim.AdamW([q])
    q.grad = torch.ones(7)
    old.step()
    with pytest.raises(ValueError, match="state_bits=8"):
        manbo.AdamW([q], state_bits=8).load_state_dict(old.state_dict())
    opt.load_state_dict({**_saved(opt), "state": {0: {}}})  # empty: as if there were none
    assert not opt.state[p]


def test_strides_of_sizes_of_one_do_not_matter():
    p = torch.zeros(1, 5).as_strided((1, 5), (1, 1)).requires_grad_()
    opt = manbo.AdamW([p], state_bits=8)
    saved = opt.state_dict()
    codes = torch.arange(5, dtype=torch.uint8).view(1, 5)
    s = torch.tensor([90], dtype=torch.uint8)
    saved["state"] = {0: dict(exp_avg=codes, exp_avg_scales=s, exp_avg_sq=codes,
                              exp_avg_sq_scales=s, step=1)}
    opt.load_state_dict(saved)
    assert torch.equal(opt.state[p]["exp_avg"], codes)


@pytest.mark.parametrize("step", [3, 3.0, torch.tensor(3.0), torch.tensor([3])])
@pytest.mark.parametrize("capturable", [False, True])
def test_step_counts_of_every_kind(step, capturable):
    p = torch.zeros(7, requires_grad=True)
    opt = manbo.AdamW([p], capturable=capturable)
    saved = opt.state_dict()
    saved["state"] = {0: dict(exp_avg=torch.ones(7), exp_avg_sq=torch.ones(7), step=step)}
    opt.load_state_dict(saved)
    got = opt.state[p]["step"]
    if capturable:
        assert got.dtype == torch.int64 and got.shape == () and got is not step
    else:
        assert type(got) is int
    assert int(got) == 3


def test_learning_rates_that_are_tensors():
    ps = [torch.zeros(3, requires_grad=True) for _ in range(3)]
    rate = torch.tensor(0.25, dtype=torch.float64)

    def groups(**kw):
        return [{"params": [p], **kw} for p in ps[:2]] + [{"params": ps[2:], "lr": 0.5}]
    old = manbo.AdamW(groups(lr=rate), capturable=True)
    new = manbo.AdamW(groups(), capturable=True)
    new.load_state_dict(old.state_dict())
    a, b, c = (g["lr"] for g in new.param_groups)
    assert a is b and a is not rate and a.dtype == torch.float32 and float(a) == 0.25 and c == 0.5
    # torch takes a tensor without capturable, too
    new.load_state_dict(torch.optim.AdamW(groups(lr=torch.tensor(0.125)), foreach=False)
                        .state_dict())
    assert [g["lr"] for g in new.param_groups] == [0.125, 0.125, 0.5]
    assert type(new.param_groups[0]["lr"]) is float


def test_stored_optimisers_whose_parameters_share_a_counter_get_one_each():
    ps = [torch.zeros(3, requires_grad=True) for _ in range(3)]
    opt = manbo.AdamW(ps, capturable=True)
    shared = torch.tensor(5)
    for p in ps[:2]:
        opt.state[p] = dict(exp_avg=torch.zeros(3), exp_avg_sq=torch.zeros(3), step=shared)
    other = copy.deepcopy(opt)
    a, b = (other.state[p]["step"] for p in other.param_groups[0]["params"][:2])
    a += 1
    assert int(a) == 6 and int(b) == 5 and int(shared) == 5


def test_a_group_added_after_a_load_clips_with_the_others():
    ps = [torch.zeros(3, requires_grad=True) for _ in range(2)]
    old = manbo.AdamW(ps[:1], max_grad_norm=0.5)
    new = manbo.AdamW(ps[:1])
    new.load_state_dict(old.state_dict())
    new.add_param_group({"params": ps[1:]})
    assert [g["max_grad_norm"] for g in new.param_groups] == [0.5, 0.5]
