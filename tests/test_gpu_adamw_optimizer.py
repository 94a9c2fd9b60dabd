"""manbo.AdamW and the AdamW operators on the GPU where calls differ from one
another: parameters that skip steps, many groups, resumed and restarted
optimisers, refusals, and values at the ends of the float32 range.

Tolerances are those of test_gpu_adamw.py: oracle.adamw64's bounds, twice them
with 8-bit moments."""
import numpy as np
import pytest
import torch

import manbo
from manbo import ops
from oracle import adamw as oa
from test_gpu_adamw import BF16, F16, F32, HYPER, check_param, make, moments32, n64

pytestmark = pytest.mark.gpu


def params_of(sizes, dtype=F32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [make(n, dtype, gen, 0.3).requires_grad_() for n in sizes], gen


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lr", [1e-30, 1e-36, 1e-37, 1e-38, 1e-39, 1e-44])
def test_a_tiny_learning_rate_leaves_parameters_of_no_gradient(lr, dtype):
    gen = torch.Generator().manual_seed(8)
    for device_lr in (False, True):
        p, g = make(3000, dtype, gen, 0.3), make(3000, dtype, gen)
        g[::3] = 0
        old, rate = p.clone(), torch.tensor(lr, device="cuda") if device_lr else lr
        m, v = moments32(p, gen)
        st = ops.adamw8_state(p)
        ops.adamw8_step([p], [g], *[[x] for x in st], step=1, lr=rate)
        assert torch.equal(p, old) and st[0].any()
        ops.adamw_step([p], [g], [m], [v], step=1, lr=rate)
        assert torch.equal(p, old)


def test_a_learning_rate_of_zero_with_a_square_that_overflows():
    for dtype in (F32, BF16):
        p, g = torch.full((600,), 0.5, dtype=dtype, device="cuda"), None
        old = p.clone()
        g = torch.full_like(p, 1e21)
        g[::2] = 0
        st = ops.adamw8_state(p)
        ops.adamw8_step([p], [g], *[[x] for x in st], step=1, lr=0.0)
        assert torch.equal(p, old)
        m, v = torch.zeros(600, device="cuda"), torch.zeros(600, device="cuda")
        ops.adamw_step([p], [g], [m], [v], step=1, lr=0.0)
        assert torch.equal(p, old)


def test_lazily_negated_scalars_are_refused():
    p, g, m, v = (torch.ones(8, device="cuda") for _ in range(4))
    neg = torch._neg_view(torch.full((), 0.5, device="cuda"))
    st = ops.adamw8_state(p)
    for kw, name in ((dict(lr=neg), "lr"), (dict(grad_scale=neg), "grad_scale")):
        with pytest.raises(ValueError, match=f"{name} must not be a lazily negated"):
            ops.adamw_step([p], [g], [m], [v], step=1, **kw)
        with pytest.raises(ValueError, match=f"{name} must not be a lazily negated"):
            ops.adamw8_step([p], [g], *[[x] for x in st], step=1, **kw)
    count = torch._neg_view(torch.full((), 5, device="cuda"))
    with pytest.raises(ValueError, match="step must not be a lazily negated"):
        ops.adamw_step([p], [g], [m], [v], step=count)
    assert torch.equal(p, torch.ones_like(p))


def test_written_moments_and_counters_rise_in_version():
    p, g = torch.ones(600, device="cuda"), torch.ones(600, device="cuda")
    m, v = torch.zeros(600, device="cuda"), torch.zeros(600, device="cuda")
    count = torch.zeros((), dtype=torch.int64, device="cuda")
    x = torch.ones(600, device="cuda", requires_grad=True)
    y = (x * m).sum()
    ops.adamw_step([p], [g], [m], [v], step=count)
    assert all(t._version == 1 for t in (p, m, v, count)) and g._version == 0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    st = ops.adamw8_state(p)
    before = [t._version for t in st]
    ops.adamw8_step([p], [g], *[[t] for t in st], step=count)
    assert [t._version for t in st] == [b + 1 for b in before]
    assert p._version == 2 and count._version == 2 and g._version == 0
    out = [torch.zeros(600, device="cuda")], [torch.zeros(600, device="cuda")]
    ops.adamw8_moments(*[[t] for t in st], out=out)
    assert out[0][0]._version == 1 and out[1][0]._version == 1
    assert [t._version for t in st] == [b + 1 for b in before]


@pytest.mark.parametrize("capturable", [False, True])
def test_groups_beyond_one_launch_round_with_bits_of_their_own(capturable):
    """40 groups of one seed: each parameter's codes are those of its place in the
    whole step (of the restatement), not of its place in a launch."""
    ps, gen = params_of([600] * 40, seed=7)
    opt = manbo.AdamW([{"params": [p], "lr": 1e-3 * (i + 1)} for i, p in enumerate(ps)],
                      state_bits=8, capturable=capturable, seed=11)
    zeros, scales = np.zeros(600, np.uint8), np.zeros(3, np.uint8)
    state = [(zeros, scales, zeros, scales)] * 40
    for t in (1, 2):
        for i, p in enumerate(ps):
            p.grad = make(600, F32, gen)
            state[i] = oa.step8(p.grad.cpu().numpy(), *state[i], step=t, seed=11, place=i)[2:]
        opt.step()
        for p, want in zip(ps, state):
            st = opt.state[p]
            for k, w in zip(("exp_avg", "exp_avg_scales", "exp_avg_sq", "exp_avg_sq_scales"),
                            want):
                np.testing.assert_array_equal(st[k].cpu().numpy(), w)


@pytest.mark.parametrize("bits", [8, 32])
def test_groups_may_differ_in_capturable(bits):
    runs = []
    for mixed in (False, True):
        ps, gen = params_of((300, 700, 50), seed=6)
        opt = manbo.AdamW([{"params": [p], "capturable": mixed and i != 1, "seed": i}
                           for i, p in enumerate(ps)], lr=0.01, state_bits=bits)
        for _ in range(3):
            for p in ps:
                p.grad = make(p.numel(), F32, gen)
            opt.step()
        runs.append([x for p in ps for x in (p, *opt.moments(p))])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("bits", [8, 32])
def test_a_parameter_without_a_gradient_is_not_counted(bits):
    """The second parameter has a gradient in steps 1, 2 and 5 only, the third from
    step 3 on, but not in 4: counts on the device and on the host agree, and so do
    parameters and moments, bit for bit."""
    runs = []
    for capturable in (False, True):
        ps, gen = params_of((3000, 257, 700), seed=4)
        opt = manbo.AdamW(ps, lr=0.01, state_bits=bits, capturable=capturable, seed=3)
        for t in range(1, 6):
            here = (True, t in (1, 2, 5), t in (3, 5))
            for p, yes in zip(ps, here):
                g = make(p.numel(), F32, gen)
                p.grad = g if yes else None
            before = n64(ps[1]), opt.moments(ps[1]) if t > 1 else None
            opt.step()
            if t == 5:  # its third step
                (m, v), now = before[1], ps[1]
                want = oa.adamw64(before[0], n64(now.grad), n64(m), n64(v), 3, lr=0.01)
                assert (np.abs(n64(now) - want[0]) <= 2 * want[3][0]).all()
        assert [int(opt.state[p]["step"]) for p in ps] == [5, 3, 2]
        runs.append([x for p in ps for x in (p, *opt.moments(p))])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("bits", [8, 32])
def test_a_captured_step_counts_its_own_parameters_only(bits):
    """Captured while the second parameter has no gradient, replayed twice, then
    an eager step of both, then a replay: as eager steps without a graph."""
    runs = []
    for captured in (False, True):
        ps, gen = params_of((3000, 257), seed=5)
        for p in ps:
            p.grad = make(p.numel(), F32, gen)
        grads = [p.grad for p in ps]
        opt = manbo.AdamW(ps, lr=0.01, state_bits=bits, capturable=True, max_grad_norm=0.1)
        opt.step()
        ps[1].grad = None
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
        for both in (False, False, True, False):
            ps[1].grad = grads[1] if both else None
            graph.replay() if captured and not both else opt.step()
        assert [int(opt.state[p]["step"]) for p in ps] == [5, 2]
        runs.append([x for p in ps for x in (p, *opt.moments(p))])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("count", [1, 130, 1300])
def test_counts_of_many_parameters(count):
    """Counters on the device through every table size, each at another step."""
    runs = []
    for capturable in (False, True):
        ps, gen = params_of([1 + i % 37 for i in range(count)], seed=count)
        opt = manbo.AdamW(ps, lr=0.01, capturable=capturable)
        for t in range(4):
            for i, p in enumerate(ps):
                p.grad = make(p.numel(), F32, gen)
                if i % 4 < t:
                    p.grad = None
            if any(p.grad is not None for p in ps):
                opt.step()
        assert [int(opt.state[p]["step"]) for p in ps] == [1 + i % 4 for i in range(count)]
        runs.append([x for p in ps for x in (p, *opt.moments(p))])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_a_refused_step_moves_no_parameter():
    """The refusal is in another launch than the first: 8-bit moments after 32-bit
    ones, the 17th group, a device counter."""
    def build(n, **kw):
        ps, gen = params_of((300,) * n, seed=12)
        for p in ps:
            p.grad = make(300, F32, gen)
        return ps
    for n, groups in ((2, [{}, {"state_bits": 8}]), (20, [{"lr": 1e-3 * i} for i in range(1, 21)]),
                      (2, [{"capturable": True}, {"capturable": False}])):
        ps = build(n)
        opt = manbo.AdamW([{"params": [p], **g} for p, g in zip(ps, groups)])
        opt.step()
        old = [[x.clone() for x in (p, *opt.moments(p))] for p in ps]
        ps[-1].grad = ps[-1].grad.to_sparse()
        with pytest.raises(ValueError, match="must be a dense tensor"):
            opt.step()
        for p, o in zip(ps, old):
            assert all(torch.equal(a, b) for a, b in zip((p, *opt.moments(p)), o))
            assert int(opt.state[p]["step"]) == 1


def test_a_resumed_optimiser_still_clips():
    """max_grad_norm is in the saved groups, so it holds after a load, and where a
    group is given another value."""
    ps, gen = params_of((700, 50), seed=8)
    opt = manbo.AdamW(ps, lr=0.01, max_grad_norm=0.05)
    for p in ps:
        p.grad = make(p.numel(), F32, gen)
    opt.step()
    qs = [p.detach().clone().requires_grad_() for p in ps]
    other = manbo.AdamW(qs)
    other.load_state_dict(opt.state_dict())
    for p, q in zip(ps, qs):
        p.grad = make(p.numel(), F32, gen)
        q.grad = p.grad.clone()
    opt.step()
    other.step()
    assert torch.equal(opt.grad_norm, other.grad_norm) and float(opt.grad_norm) > 0.05
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    for o in (opt, other):
        for group in o.param_groups:
            group["max_grad_norm"] = 0.01 if o is opt else 0.0
    for q in qs:
        q.grad = None
    ps[1].grad = None
    p, g = ps[0], n64(ps[0].grad)
    old, (m, v) = n64(p), opt.moments(p)
    opt.step()
    _, c = oa.norm64([g], 0.01)
    want = oa.adamw64(old, g, n64(m), n64(v), 3, lr=0.01, scale=float(np.float32(c)))
    assert (np.abs(n64(p) - want[0]) <= 2 * want[3][0]).all()


def test_groups_that_disagree_on_max_grad_norm_are_refused():
    ps, gen = params_of((50, 60), seed=8)
    opt = manbo.AdamW([{"params": ps[:1], "max_grad_norm": 1.0}, {"params": ps[1:]}])
    for p in ps:
        p.grad = make(p.numel(), F32, gen)
    old = [p.clone() for p in ps]
    with pytest.raises(ValueError, match="max_grad_norm must be the same in every group"):
        opt.step()
    assert all(torch.equal(p, o) for p, o in zip(ps, old))
    for group in opt.param_groups:
        group["max_grad_norm"] = -1.0
    with pytest.raises(ValueError, match="Invalid max_norm"):
        opt.step()
    for group in opt.param_groups:
        group["max_grad_norm"] = 1.0
    opt.step()
    assert opt.grad_norm is not None


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("capturable", [False, True])
def test_state_of_torch_adamw_with_16_bit_parameters_continues(dtype, capturable):
    ps, gen = params_of((700, 50), dtype, seed=9)
    kw = dict(lr=1e-2, betas=(0.8, 0.99), weight_decay=0.1, capturable=capturable)
    old = torch.optim.AdamW(ps, **kw)
    for _ in range(2):
        for p in ps:
            p.grad = make(p.numel(), dtype, gen)
        old.step()
    opt = manbo.AdamW(ps)
    opt.load_state_dict(old.state_dict())
    for p in ps:
        m, v = opt.moments(p)
        assert m.dtype == v.dtype == F32
        assert torch.equal(m, old.state[p]["exp_avg"].float())
        p.grad = make(p.numel(), dtype, gen)
    kw.pop("capturable")
    wants = [oa.adamw64(n64(p), n64(p.grad), *map(n64, opt.moments(p)), 3, **kw) for p in ps]
    opt.step()
    for p, want in zip(ps, wants):
        # torch's own steps in float16 leave parameters that are infinite (v underflows):
        # these stay so, the others are within the bound
        ok = np.isfinite(want[0])
        assert ok.sum() > p.numel() // 2
        np.testing.assert_array_equal(n64(p)[~ok], want[0][~ok])
        check_param(p.detach()[torch.from_numpy(ok).cuda()], dtype, want[0][ok], want[3][0][ok])
        assert int(opt.state[p]["step"]) == 3


@pytest.mark.parametrize("bits", [8, 32])
def test_restart_zeroes_what_a_captured_step_writes(bits):
    ps, gen = params_of((700, 50), seed=10)
    opt = manbo.AdamW(ps, lr=0.01, state_bits=bits, capturable=True)
    for p in ps:
        p.grad = make(p.numel(), F32, gen)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    kept = [{k: x.data_ptr() for k, x in opt.state[p].items()} for p in ps]
    opt.restart_opt()
    for p, k in zip(ps, kept):
        assert {name: x.data_ptr() for name, x in opt.state[p].items()} == k
        assert all(not x.any() for x in opt.state[p].values())
    qs = [p.detach().clone().requires_grad_() for p in ps]
    fresh = manbo.AdamW(qs, lr=0.01, state_bits=bits)
    for _ in range(2):
        graph.replay()
        for p, q in zip(ps, qs):
            q.grad = p.grad.clone()
        fresh.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q) and int(opt.state[p]["step"]) == 2
        assert all(torch.equal(a, b) for a, b in zip(opt.moments(p), fresh.moments(q)))


def test_restart_drops_a_state_of_another_kind():
    ps, gen = params_of((700, 50), seed=10)
    opt = manbo.AdamW([{"params": [p]} for p in ps], lr=0.01)
    for p in ps:
        p.grad = make(p.numel(), F32, gen)
    opt.step()
    opt.param_groups[0].update(state_bits=8, capturable=True)
    opt.restart_opt()
    assert ps[0] not in opt.state and opt.state[ps[1]]["step"] == 0
    opt.step()
    assert opt.state[ps[0]]["exp_avg"].dtype == torch.uint8
    assert [int(opt.state[p]["step"]) for p in ps] == [1, 1]


def test_a_learning_rate_saved_from_the_device_and_read_on_the_host():
    """A checkpoint that was read with every tensor on the host continues."""
    ps, gen = params_of((700, 50), seed=13)
    opt = manbo.AdamW(ps, lr=torch.tensor(0.01, device="cuda"), capturable=True)
    for p in ps:
        p.grad = make(p.numel(), F32, gen)
    opt.step()
    saved = opt.state_dict()
    host = {"param_groups": [{**g, "lr": g["lr"].cpu()} for g in saved["param_groups"]],
            "state": {i: {k: x.cpu() for k, x in st.items()} for i, st in saved["state"].items()}}
    qs = [p.detach().clone().requires_grad_() for p in ps]
    other = manbo.AdamW(qs, capturable=True)
    other.load_state_dict(host)
    for p, q in zip(ps, qs):
        q.grad = p.grad.clone()
    opt.step()
    other.step()
    assert other.param_groups[0]["lr"].is_cuda
    for p, q in zip(ps, qs):
        assert torch.equal(p, q) and int(other.state[q]["step"]) == 2


@pytest.mark.parametrize("bits", [8, 32])
def test_gradients_from_an_iterator_live_until_the_step_has_run(bits):
    """Tensors that only the call holds, beside a workspace that it allocates (for a
    device counter) after it has read them."""
    runs = []
    for lazy in (False, True):
        ps, gen = params_of((4,) * 50 + (3000,), seed=14)
        ps = [p.detach() for p in ps]
        base = [make(p.numel(), F32, gen) for p in ps]
        if bits == 8:
            state = list(zip(*[ops.adamw8_state(p) for p in ps]))
        else:
            state = [[torch.zeros_like(p) for p in ps] for _ in range(2)]
        count = torch.zeros((), dtype=torch.int64, device="cuda")
        for _ in range(3):
            grads = (g * 0.5 for g in base) if lazy else [g * 0.5 for g in base]
            step = ops.adamw8_step if bits == 8 else ops.adamw_step
            step(ps, grads, *state, step=count, **HYPER)
        runs.append(ps)
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_non_finite_gradients_of_unaligned_parameters(dtype, shift):
    """Every path of a block (aligned, by way of shared memory, cut short): the
    element's parameter and the whole block's moments."""
    n = 256 * 5 + 100
    p = torch.ones(n + shift, dtype=dtype, device="cuda")[shift:]
    g = torch.full((n + shift,), 0.1, dtype=dtype, device="cuda")[shift:]
    st = ops.adamw8_state(p)
    bad = {3: float("nan"), 700: float("inf"), n - 1: -float("inf")}
    for i, x in bad.items():
        g[i] = x
    ops.adamw8_step([p], [g], *[[x] for x in st], step=1, **HYPER)
    assert [e == 255 for e in st[1].tolist()] == [b in (0, 2, 5) for b in range(6)]
    assert [e == 255 for e in st[3].tolist()] == [b in (0, 2, 5) for b in range(6)]
    assert torch.isnan(p).nonzero().view(-1).tolist() == sorted(bad)
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    p = torch.ones(n + shift, dtype=dtype, device="cuda")[shift:]
    ops.adamw_step([p], [g], [m], [v], step=1, **HYPER)
    assert torch.isnan(p).nonzero().view(-1).tolist() == sorted(bad)
    assert (~torch.isfinite(m)).nonzero().view(-1).tolist() == sorted(bad)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), 0.0])
def test_grad_scales_that_are_not_ordinary(scale):
    """NaN and infinity reach every parameter (0 times infinity is NaN, and the first
    step of an infinite average is infinity over infinity), zero none."""
    c = torch.tensor(scale, device="cuda")
    p, g = torch.ones(600, device="cuda"), torch.full((600,), 0.1, device="cuda")
    g[5] = 0
    m, v = torch.zeros(600, device="cuda"), torch.zeros(600, device="cuda")
    ops.adamw_step([p], [g], [m], [v], step=1, grad_scale=c, **HYPER)
    q = torch.ones(600, device="cuda")
    st = ops.adamw8_state(q)
    ops.adamw8_step([q], [g], *[[x] for x in st], step=1, grad_scale=c, **HYPER)
    if scale == 0.0:
        assert not m.any() and not v.any() and not st[0].any() and not st[2].any()
        assert torch.equal(p, q) and torch.isfinite(p).all()
    else:
        assert torch.isnan(p).all() and torch.isnan(q).all()
        assert (st[1] == 255).all() and (st[3] == 255).all()


def test_a_closure_runs_with_gradients_and_gives_the_loss():
    p = torch.ones(5, device="cuda", requires_grad=True)
    opt = manbo.AdamW([p], lr=0.1, weight_decay=0.0)

    def closure():
        opt.zero_grad()
        loss = (p * p).sum()
        loss.backward()
        return loss
    assert float(opt.step(closure).detach()) == 5.0
    # the first step moves by lr against the gradient's sign; eps and roundings: 1e-6
    assert float((p.detach() - 0.9).abs().max()) < 1e-6


def test_float32_tensors_of_many_chunks_a_cta():
    """60 M float32 elements: four and more blocks a warp, without the prefetch
    that 16-bit parameters have; windows against the restatement."""
    n = 60_000_077
    gen = torch.Generator(device="cuda").manual_seed(n)
    p = torch.randn(n, device="cuda", generator=gen) * 0.3
    g = torch.randn(n, device="cuda", generator=gen) * 1e-2
    st = ops.adamw8_state(p)
    ops.adamw8_step([p], [g], *[[x] for x in st], step=1, seed=3, **HYPER)
    blocks, chunks = -(-n // 256), -(-n // 1024)
    starts = {0, blocks - 3, blocks // 2}
    for per in (2, 4, 8, 16, 32):
        stride = -(-chunks // per) * 4
        starts |= {b for b in (stride - 2, stride * (per - 1) - 1) if 0 <= b < blocks - 3}
    for b in sorted(starts):
        at, end = b * 256, min(n, (b + 3) * 256)
        zeros, scales = np.zeros(end - at, np.uint8), np.zeros(-(-(end - at) // 256), np.uint8)
        new = oa.step8(g[at:end].cpu().numpy(), zeros, scales, zeros, scales, step=1,
                       betas=HYPER["betas"], seed=3, first_block=b)
        for got, want in zip((st[0][at:end], st[1][b:b + 3], st[2][at:end], st[3][b:b + 3]),
                             new[2:]):
            np.testing.assert_array_equal(got.cpu().numpy(), want)
    assert int((st[0] == 0).sum()) < n // 1000 and not (st[1] == 0).any()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("capturable", [False, True])
def test_empty_parameters_are_counted_and_nothing_else(bits, capturable):
    ps = [torch.zeros(n, device="cuda", requires_grad=True) for n in (0, 5, 0)]
    opt = manbo.AdamW(ps, state_bits=bits, capturable=capturable, max_grad_norm=1.0)
    for t in (1, 2, 3):
        for p in ps:
            p.grad = torch.ones_like(p)
        if t == 3:
            ps[1].grad = None  # nothing to move at all
        opt.step()
    assert [int(opt.state[p]["step"]) for p in ps] == [3, 2, 3]
    assert float(opt.grad_norm) == 0.0 and bool((ps[1] < 0).all())


def test_counted_8_bit_steps_of_many_parameters_round_as_the_restatement():
    """More tensors than a table and than a launch of counters take."""
    ps, gen = params_of([1 + (i * 7) % 600 for i in range(900)], seed=15)
    opt = manbo.AdamW(ps, state_bits=8, capturable=True, seed=21)
    state = [(np.zeros(p.numel(), np.uint8), np.zeros(-(-p.numel() // 256), np.uint8)) * 2
             for p in ps]
    for t in (1, 2):
        for i, p in enumerate(ps):
            p.grad = make(p.numel(), F32, gen)
            state[i] = oa.step8(p.grad.cpu().numpy(), *state[i], step=t, seed=21, place=i)[2:]
        opt.step()
    for p, want in zip(ps, state):
        st = opt.state[p]
        for k, w in zip(("exp_avg", "exp_avg_scales", "exp_avg_sq", "exp_avg_sq_scales"), want):
            np.testing.assert_array_equal(st[k].cpu().numpy(), w)
