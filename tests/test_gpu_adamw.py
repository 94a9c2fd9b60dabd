"""The AdamW operators on the GPU against float64 and, for the 8-bit moments'
bytes, against the float32 restatement bit for bit (oracle/adamw.py).

Tolerances: a float32 result is within the error bounds that oracle.adamw64
derives; a 16-bit parameter adds half a step of its type (2^-8 relative to the
value for bfloat16, 2^-11 for float16, and 2^-25 for float16's smallest
numbers).  The norm is summed in double and rounded once: 2^-24."""
import numpy as np
import pytest
import torch

import manbo
from manbo import ops
from oracle import adamw as oa

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_STEP = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
LEAST = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -25}
# one element, around a scale block, around a CTA's chunk, several chunks
SIZES = [1, 31, 255, 256, 257, 2047, 2048, 2049, 5003, 70001]
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)


def n64(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def storage_order(t):
    """A dense tensor's elements as they lie in memory."""
    return t.detach().as_strided((t.numel(),), (1,))


def make(n, dtype, gen, scale=1e-2):
    return (torch.randn(n, generator=gen) * scale).to(dtype).cuda()


def moments32(p, gen, dead=True):
    m = torch.randn(p.numel(), generator=gen) * 1e-3
    v = (torch.randn(p.numel(), generator=gen) * 1e-2).square()
    if dead:
        m[::7] = 0
        v[::7] = 0
    def like(x):
        out = torch.empty_like(p, dtype=F32)
        storage_order(out).copy_(x)
        return out
    return like(m), like(v)


def check_param(p, dtype, p1, bound):
    got = n64(p)
    tol = bound + (np.abs(p1) + bound) * HALF_STEP[dtype] + LEAST[dtype]
    assert (np.abs(got - p1) <= tol).all(), np.abs(got - p1).max()


# --- gradient norm ----------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16, F16, "mixed"])
@pytest.mark.parametrize("count", [1, 5, 200, 1500])
def test_grad_norm_matches_float64(dtype, count):
    gen = torch.Generator().manual_seed(count)
    kinds = [F32, BF16, F16] if dtype == "mixed" else [dtype]
    grads = [make([0, 1, 17, 300][i % 4] if count > 20 else SIZES[i % len(SIZES)] * 3,
                  kinds[i % len(kinds)], gen) for i in range(count)]
    for max_norm in (0.0, 1e-3, 1e6):
        norm, scale = ops.grad_norm(grads, max_norm=max_norm)
        want, c = oa.norm64([n64(g) for g in grads], max_norm)
        assert norm.dtype == F32 and norm.dim() == 0 and scale.dim() == 0
        assert abs(float(norm) - want) <= 6.1e-8 * want
        assert abs(float(scale) - c) <= 6.1e-8 * c


def test_grad_norm_of_large_and_small_values():
    for x in (1e30, 1e-30, 3e38):
        g = torch.full((1000,), x, device="cuda")
        norm, scale = ops.grad_norm([g], max_norm=1.0)
        want = float(torch.tensor(x, dtype=F32).double()) * 1000 ** 0.5
        if want > 3.4e38:
            assert torch.isinf(norm) and float(scale) > 0
        else:
            assert abs(float(norm) - want) <= 6.1e-8 * want
            c = min(1.0, 1.0 / (want + 1e-6))
            assert abs(float(scale) - c) <= 6.1e-8 * c


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_grad_norm_of_every_16_bit_value(dtype):
    """All finite bit patterns (subnormal ones and zeros among them), alone in
    their own tensors by magnitude, aligned and not; then each infinity and NaN."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).cuda()
    every = bits.view(dtype)
    finite = every[torch.isfinite(every)]
    size = finite.float().abs()
    small = torch.finfo(dtype).tiny
    for g in (finite, finite[size < small], finite[size == 0], finite[size >= small][1:],
              finite[size < small][3:]):
        want, _ = oa.norm64([n64(g)])
        norm, _ = ops.grad_norm([g])
        if want > np.finfo(np.float32).max:  # rounds to infinity
            assert torch.isinf(norm)
            continue
        # a norm below float32's normal range is rounded to its subnormal spacing
        assert abs(float(norm) - want) <= 6.1e-8 * want + 2.0 ** -150
    for at in (0, 1, 4099):
        for bad in every[~torch.isfinite(every)][:: 9 if dtype == F16 else 1].tolist():
            g = torch.ones(4100, dtype=dtype, device="cuda")
            g[at] = bad
            norm, _ = ops.grad_norm([g])
            assert torch.isnan(norm) if bad != bad else torch.isinf(norm)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_grad_norm_of_full_chunks_of_every_size(dtype):
    """Long aligned tensors: ordinary values, zeros, zeros with signs, and values
    whose squares float32 does not hold, alone and among ordinary ones."""
    gen = torch.Generator().manual_seed(2)
    n = 1 << 18
    ordinary = make(n, dtype, gen)
    kinds = [ordinary, torch.zeros(n, dtype=dtype, device="cuda"),
             -torch.zeros(n, dtype=dtype, device="cuda")]
    for size in ((1e-6, 6e4) if dtype == F16 else (1e-39, 1e-25, 1e-16, 1e16, 1e25)):
        some = ordinary.clone()
        some[::1000] = size
        kinds += [some, torch.full((n,), size, dtype=dtype, device="cuda"),
                  torch.cat([ordinary[:n // 2], torch.full((n // 2,), size, dtype=dtype,
                                                           device="cuda")])]
    for g in kinds:
        want, _ = oa.norm64([n64(g)])
        norm, _ = ops.grad_norm([g, ordinary[:5]])
        want = (want ** 2 + float((n64(ordinary[:5]) ** 2).sum())) ** 0.5
        assert abs(float(norm) - want) <= 6.1e-8 * want
    for at in (0, n - 1):
        for bad in (float("nan"), float("inf"), -float("inf")):
            g = ordinary.clone()
            g[at] = bad
            norm, _ = ops.grad_norm([g])
            assert torch.isnan(norm) if bad != bad else torch.isinf(norm)


def test_grad_norm_of_nan_inf_and_nothing():
    g = torch.ones(300, device="cuda")
    g[299] = float("nan")
    norm, scale = ops.grad_norm([g], max_norm=1.0)
    assert torch.isnan(norm) and torch.isnan(scale)
    g[299] = float("inf")
    norm, scale = ops.grad_norm([g], max_norm=1.0)
    assert torch.isinf(norm) and float(scale) == 0.0
    norm, scale = ops.grad_norm([torch.empty(0, device="cuda")], max_norm=1.0)
    assert float(norm) == 0.0 and float(scale) == 1.0


def test_grad_norm_of_views():
    base = torch.randn(64, 33, device="cuda")
    for g in (base[:, ::2], base.t(), base.view(-1)[1:], base[3:5, 4:7], base[:1, :1].expand(9, 9),
              base.view(-1).to(BF16)[3:1000], torch.randn(2, 3, 5, 7, device="cuda")
              .contiguous(memory_format=torch.channels_last)):
        norm, _ = ops.grad_norm([g])
        want, _ = oa.norm64([n64(g)])
        assert abs(float(norm) - want) <= 6.1e-8 * want


def test_grad_norm_is_the_same_every_time():
    g = [torch.randn(n, device="cuda") for n in (1_000_003, 77, 5)]
    a = ops.grad_norm(g, max_norm=1.0)
    for _ in range(3):
        b = ops.grad_norm(g, max_norm=1.0)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# --- 32-bit step ------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n", SIZES)
def test_adamw_step_matches_float64(n, dtype):
    gen = torch.Generator().manual_seed(n)
    p, g = make(n, dtype, gen, 0.3), make(n, dtype, gen)
    g[::7] = 0
    m, v = moments32(p, gen)
    for step, scale in ((1, None), (2, 0.37), (5000, 1.0)):
        c = None if scale is None else torch.tensor(scale, device="cuda")
        want = oa.adamw64(n64(p), n64(g), n64(m), n64(v), step,
                          scale=1.0 if c is None else float(c), **HYPER)
        ops.adamw_step([p], [g], [m], [v], step=step, grad_scale=c, **HYPER)
        assert (np.abs(n64(m) - want[1]) <= want[3][1]).all()
        assert (np.abs(n64(v) - want[2]) <= want[3][2]).all()
        check_param(p, dtype, want[0], want[3][0])


def _mixed(count, seed, least=1):
    gen = torch.Generator().manual_seed(seed)
    kinds = [F32, BF16, F16]
    sizes = torch.randint(least, 900, (count,), generator=gen).tolist()
    params = [make(n, kinds[i % 3], gen, 0.3) for i, n in enumerate(sizes)]
    grads = [make(n, kinds[i % 3], gen) for i, n in enumerate(sizes)]
    return gen, params, grads


@pytest.mark.parametrize("count", [1, 36, 37, 40, 41, 561, 1300])
def test_adamw_step_of_many_tensors(count):
    """Table borders of both sizes, empty tensors among them, mixed types."""
    gen, params, grads = _mixed(count, count, least=0)
    ms, vs = zip(*[moments32(p, gen) for p in params])
    want = [oa.adamw64(n64(p), n64(g), n64(m), n64(v), 3, **HYPER)
            for p, g, m, v in zip(params, grads, ms, vs)]
    ops.adamw_step(params, grads, ms, vs, step=3, **HYPER)
    for p, m, v, w in zip(params, ms, vs, want):
        assert (np.abs(n64(m) - w[1]) <= w[3][1]).all()
        assert (np.abs(n64(v) - w[2]) <= w[3][2]).all()
        check_param(p, p.dtype, w[0], w[3][0])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift", [1, 2, 3, 4, 5, 8])
def test_adamw_step_of_views_leaves_their_surroundings(shift, dtype):
    gen = torch.Generator().manual_seed(shift)
    n = 4099
    flat, gflat = make(n + 40, dtype, gen, 0.3), make(n + 40, dtype, gen)
    mflat, vflat = moments32(flat, gen)
    before = [x.clone() for x in (flat, mflat, vflat)]
    p, g, m, v = (x[shift:shift + n] for x in (flat, gflat, mflat, vflat))
    want = oa.adamw64(n64(p), n64(g), n64(m), n64(v), 7, **HYPER)
    ops.adamw_step([p], [g], [m], [v], step=7, **HYPER)
    check_param(p, dtype, want[0], want[3][0])
    assert (np.abs(n64(m) - want[1]) <= want[3][1]).all()
    for x, old in zip((flat, mflat, vflat), before):
        assert torch.equal(x[:shift], old[:shift]) and torch.equal(x[shift + n:], old[shift + n:])


def test_adamw_step_of_other_layouts():
    """Dense tensors in any dimension order; a gradient in another order is
    matched by index, not by place."""
    gen = torch.Generator().manual_seed(5)
    shape = (4, 6, 5, 7)
    p = make(840, F32, gen).view(shape).contiguous(memory_format=torch.channels_last)
    m, v = moments32(p, gen)
    for g in (make(840, F32, gen).view(shape), make(1680, F32, gen).view(4, 6, 5, 14)[..., ::2],
              make(1, F32, gen).expand(shape), torch._neg_view(p.clone(
                  memory_format=torch.preserve_format))):
        want = oa.adamw64(n64(p), n64(g), n64(m), n64(v), 7, **HYPER)
        ops.adamw_step([p], [g], [m], [v], step=7, **HYPER)
        check_param(p, F32, want[0], want[3][0])
        assert (np.abs(n64(m) - want[1]) <= want[3][1]).all()
    t = make(12, F32, gen).view(3, 4).t()
    m, v = moments32(t, gen)
    g = make(12, F32, gen).view(4, 3)
    want = oa.adamw64(n64(t), n64(g), n64(m), n64(v), 7, **HYPER)
    ops.adamw_step([t], [g], [m], [v], step=7, **HYPER)
    check_param(t, F32, want[0], want[3][0])
    s = make(1, F32, gen).view(())
    m, v = moments32(s, gen, dead=False)
    want = oa.adamw64(n64(s), n64(s), n64(m), n64(v), 7, **HYPER)
    ops.adamw_step([s], [s.clone()], [m], [v], step=7, **HYPER)
    check_param(s, F32, want[0], want[3][0])


def test_device_counter_and_learning_rate_equal_host_ones():
    gen, params, grads = _mixed(9, 4)
    ms, vs = zip(*[moments32(p, gen) for p in params])
    copies = [[x.clone() for x in xs] for xs in (params, ms, vs)]
    count = torch.tensor(6, device="cuda")
    lr = torch.tensor(HYPER["lr"], device="cuda")
    ops.adamw_step(params, grads, ms, vs, step=7, **HYPER)
    ops.adamw_step(copies[0], grads, copies[1], copies[2], step=count, **{**HYPER, "lr": lr})
    assert int(count) == 7
    for a, b in zip((params, ms, vs), copies):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_non_finite_gradients_stay_where_they_are():
    p, g = torch.ones(600, device="cuda"), torch.full((600,), 0.1, device="cuda")
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    g[3], g[400] = float("nan"), float("inf")
    ops.adamw_step([p], [g], [m], [v], step=1, **HYPER)
    bad = torch.zeros(600, dtype=torch.bool)
    bad[[3, 400]] = True
    assert torch.equal(torch.isnan(p).cpu(), bad)
    assert torch.isnan(m[3]) and torch.isinf(m[400]) and torch.isfinite(m).sum() == 598


# --- 8-bit step -------------------------------------------------------------

def bytes_of(st):
    return [storage_order(x).cpu().numpy() if x.dim() else x.cpu().numpy().reshape(1) for x in st]


def step8_and_check(params, grads, states, step, scale=None, seed=0):
    """Runs one step and compares bytes with the restatement, parameters with
    float64 from the same bytes."""
    c = None if scale is None else torch.tensor(scale, device="cuda")
    want = []
    for i, (p, g, st) in enumerate(zip(params, grads, states)):
        gs = storage_order(g).float().cpu().numpy()
        mc, me, vc, ve = bytes_of(st)
        new = oa.step8(gs, mc, me, vc, ve, step=step, betas=HYPER["betas"],
                       scale=None if c is None else float(c), seed=seed, place=i)
        ref = oa.adamw64(storage_order(p).double().cpu().numpy(), gs, oa.decode_m(mc, me),
                         oa.decode_v(vc, ve), step, scale=1.0 if c is None else float(c), **HYPER)
        want.append((new, ref))
    cols = list(zip(*states))
    ops.adamw8_step(params, grads, *cols, step=step, grad_scale=c, seed=seed, **HYPER)
    for p, st, (new, ref) in zip(params, states, want):
        mc, me, vc, ve = bytes_of(st)
        np.testing.assert_array_equal(me, new[3])
        np.testing.assert_array_equal(ve, new[5])
        np.testing.assert_array_equal(mc, new[2])
        np.testing.assert_array_equal(vc, new[4])
        # twice the bound of IEEE operations: the square root and the quotient may be the
        # hardware's approximations, each within 2^-22 (4 u)
        check_param(storage_order(p), p.dtype, ref[0], 2 * ref[3][0])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n", SIZES)
def test_adamw8_step_matches_bytes_and_float64(n, dtype):
    gen = torch.Generator().manual_seed(n)
    p = make(n, dtype, gen, 0.3)
    st = ops.adamw8_state(p)
    for step, scale in ((1, None), (2, 0.37), (3, 1.0), (4, 2.5)):
        g = make(n, dtype, gen)
        g[::7] = 0
        step8_and_check([p], [g], [st], step, scale, seed=step * 1000 + 5)


@pytest.mark.parametrize("count", [36, 37, 421, 900])
def test_adamw8_step_of_many_tensors(count):
    gen, params, grads = _mixed(count, count, least=0)
    states = [ops.adamw8_state(p) for p in params]
    for step in (1, 2):
        step8_and_check(params, grads, states, step, seed=0xFFFFFFFF)


@pytest.mark.parametrize("size", [1e-12, 1e-6, 1e4, 1e15])
def test_adamw8_step_of_small_and_large_gradients(size):
    """Below the smallest scale, and squares near the float32 range's ends."""
    gen = torch.Generator().manual_seed(1)
    p = make(1000, F32, gen, 0.3)
    st = ops.adamw8_state(p)
    for step in (1, 2, 3):
        step8_and_check([p], [make(1000, F32, gen, size)], [st], step)


def test_adamw8_step_of_blocks_with_every_size_of_gradient():
    """Magnitudes from 1e-21 (whose square is subnormal) to 1e17 in one block,
    between blocks that hold a part of them: scales above and below the ranges
    that one power of two covers, v too small for its block's scale, zeros."""
    gen = torch.Generator().manual_seed(8)
    n = 256 * 24 + 5
    p = make(n, F32, gen, 0.3)
    st = ops.adamw8_state(p)
    for step in (1, 2, 3, 4):
        top = torch.randint(-21, 18, (n // 256 + 1,), generator=gen).repeat_interleave(256)[:n]
        low = torch.rand(n, generator=gen) * 38 - 21
        g = 10.0 ** torch.minimum(low, top.float()) * torch.sign(torch.randn(n, generator=gen))
        g[::11] = 0
        step8_and_check([p], [g.cuda()], [st], step)


def test_a_learning_rate_of_zero_moves_nothing():
    gen = torch.Generator().manual_seed(8)
    for dtype in (F32, BF16):
        p, g = make(3000, dtype, gen, 0.3), make(3000, dtype, gen)
        p[::5] = 0
        g[::3] = 0
        old = p.clone()
        st = ops.adamw8_state(p)
        ops.adamw8_step([p], [g], *[[x] for x in st], step=1, lr=0.0)
        m, v = moments32(p, gen)
        ops.adamw_step([p], [g], [m], [v], step=1, lr=0.0)
        assert torch.equal(p, old) and st[0].any()


@pytest.mark.parametrize("shift", [1, 3, 4, 8])
def test_adamw8_step_of_views_leaves_their_surroundings(shift):
    gen = torch.Generator().manual_seed(shift)
    n = 4099
    flat, gflat = make(n + 40, BF16, gen, 0.3), make(n + 40, BF16, gen)
    codes = [torch.full((n + 40,), 77, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.full((17 + 4,), 99, dtype=torch.uint8, device="cuda") for _ in range(2)]
    before = [x.clone() for x in (flat, *codes, *scales)]
    st = (codes[0][shift:shift + n], scales[0][shift % 4:][:17], codes[1][shift:shift + n],
          scales[1][shift % 4:][:17])
    step8_and_check([flat[shift:shift + n]], [gflat[shift:shift + n]], [st], 9)
    for x, old, at, k in zip((flat, *codes, *scales), before,
                             (shift,) * 3 + (shift % 4,) * 2, (n,) * 3 + (17,) * 2):
        assert torch.equal(x[:at], old[:at]) and torch.equal(x[at + k:], old[at + k:])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shift", [1, 2, 7])
@pytest.mark.parametrize("n", [255, 256, 1025, 5003])
def test_unaligned_parameters_with_moments_of_their_own(n, shift, dtype):
    """Views into a flat parameter buffer and a gradient bucket (only one of them
    off its border, too), moments as an allocator gives them."""
    gen = torch.Generator().manual_seed(n + shift)
    flat, gflat = make(n + 16, dtype, gen, 0.3), make(n + 16, dtype, gen)
    for at, gat in ((shift, shift), (0, shift), (shift, 8)):
        p, g = flat[at:at + n], gflat[gat:gat + n]
        old = flat.clone()
        m, v = moments32(p, gen)
        want = oa.adamw64(n64(p), n64(g), n64(m), n64(v), 7, **HYPER)
        ops.adamw_step([p], [g], [m], [v], step=7, **HYPER)
        check_param(p, dtype, want[0], want[3][0])
        assert (np.abs(n64(m) - want[1]) <= want[3][1]).all()
        assert (np.abs(n64(v) - want[2]) <= want[3][2]).all()
        st = ops.adamw8_state(p)
        for step in (1, 2):
            step8_and_check([p], [g], [st], step, 0.7)
        assert torch.equal(flat[:at], old[:at]) and torch.equal(flat[at + n:], old[at + n:])


def test_adamw8_step_of_other_layouts():
    gen = torch.Generator().manual_seed(5)
    p = make(840, F32, gen).view(4, 6, 5, 7).contiguous(memory_format=torch.channels_last)
    g = make(840, F32, gen).view(4, 6, 5, 7).contiguous(memory_format=torch.channels_last)
    st = ops.adamw8_state(p)
    assert st[0].stride() == p.stride()
    step8_and_check([p], [g], [st], 1)
    q = p.clone(memory_format=torch.preserve_format)
    other = [x.clone(memory_format=torch.preserve_format) for x in st]
    ops.adamw8_step([p], [g.contiguous()], *[[x] for x in st], step=2, **HYPER)
    ops.adamw8_step([q], [g], *[[x] for x in other], step=2, **HYPER)
    assert torch.equal(p, q) and all(torch.equal(a, b) for a, b in zip(st, other))


def test_adamw8_marks_blocks_that_are_not_finite():
    p, g = torch.ones(1000, device="cuda"), torch.full((1000,), 0.1, device="cuda")
    st = ops.adamw8_state(p)
    g[300] = float("nan")
    g[999] = float("inf")
    ops.adamw8_step([p], [g], *[[x] for x in st], step=1, **HYPER)
    assert st[1].tolist()[1] == 255 and st[1].tolist()[3] == 255
    assert st[1].tolist()[0] != 255 and st[1].tolist()[2] != 255
    m, v = ops.adamw8_moments(*[[x] for x in st])
    want = torch.zeros(1000, dtype=torch.bool)
    want[256:512] = True
    want[768:] = True
    assert torch.equal(torch.isnan(m[0]).cpu(), want) and torch.equal(torch.isnan(v[0]).cpu(), want)
    assert torch.isnan(p).sum() == 2  # this step's parameters: the two elements alone


def test_adamw8_moments_of_every_code():
    for n in (256, 300, 70000):
        codes = (torch.arange(n) % 256).to(torch.uint8).cuda()
        blocks = -(-n // 256)
        for e in (0, 40, 120, 253, 255):
            s = torch.full((blocks,), e, dtype=torch.uint8, device="cuda")
            m, v = ops.adamw8_moments([codes], [s], [codes], [s])
            hs = s.cpu().numpy()
            np.testing.assert_array_equal(m[0].cpu().numpy(), oa.decode_m(codes.cpu().numpy(), hs))
            np.testing.assert_array_equal(v[0].cpu().numpy(), oa.decode_v(codes.cpu().numpy(), hs))
    many = [(torch.arange(n) % 256).to(torch.uint8).cuda() for n in range(0, 900, 2)]
    s = [torch.full((-(-c.numel() // 256),), 99, dtype=torch.uint8, device="cuda") for c in many]
    m, v = ops.adamw8_moments(many, s, many, s)
    for c, x, a, b in zip(many, s, m, v):
        np.testing.assert_array_equal(a.cpu().numpy(), oa.decode_m(c.cpu().numpy(), x.cpu().numpy()))
        np.testing.assert_array_equal(b.cpu().numpy(), oa.decode_v(c.cpu().numpy(), x.cpu().numpy()))


def test_offsets_past_32_bits():
    """More than 2^31 elements of two bytes: the last blocks match a step of
    their own elements (the random bits of a block go by its number)."""
    n, tail = (1 << 31) + 700, 700 + 256
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free device memory")
    start = n - tail
    assert start % 256 == 0 and start < 1 << 31
    gen = torch.Generator().manual_seed(2)
    p = torch.zeros(n, dtype=BF16, device="cuda")
    g = torch.zeros(n, dtype=BF16, device="cuda")
    p[start:] = make(tail, BF16, gen, 0.3)
    g[start:] = make(tail, BF16, gen)
    old = n64(p[start:])
    ref = oa.adamw64(old, n64(g[start:]), 0 * old, 0 * old, 1, **HYPER)
    norm, _ = ops.grad_norm([g])
    want, _ = oa.norm64([n64(g[start:])])
    assert abs(float(norm) - want) <= 6.1e-8 * want
    st = ops.adamw8_state(p)
    ops.adamw8_step([p], [g], *[[x] for x in st], step=1, seed=3, **HYPER)
    check_param(p[start:], BF16, ref[0], 2 * ref[3][0])
    m, v = ops.adamw8_moments([st[0]], [st[1]], [st[2]], [st[3]])
    np.testing.assert_array_equal(
        m[0][start:].cpu().numpy(),
        oa.decode_m(st[0][start:].cpu().numpy(), st[1][start // 256:].cpu().numpy()))
    zeros, scales = np.zeros(tail, np.uint8), np.zeros(4, np.uint8)
    new = oa.step8(g[start:].float().cpu().numpy(), zeros, scales, zeros, scales, step=1,
                   betas=HYPER["betas"], seed=3, first_block=start // 256)
    for got, want in zip((st[0][start:], st[1][start // 256:], st[2][start:], st[3][start // 256:]),
                         new[2:]):
        np.testing.assert_array_equal(got.cpu().numpy(), want)
    del st
    m[0].zero_()
    v[0].zero_()
    p[start:] = torch.from_numpy(old).to(BF16).cuda()
    ops.adamw_step([p], [g], m, v, step=1, **HYPER)
    check_param(p[start:], BF16, ref[0], ref[3][0])
    assert (np.abs(n64(m[0][start:]) - ref[1]) <= ref[3][1]).all()
    assert not m[0][:start].any() and not p[:start].any()


@pytest.mark.parametrize("dtype,n", [(F32, 5_000_077), (BF16, 20_000_300), (F16, 160_000_077)])
@pytest.mark.parametrize("shift", [0, 1])
def test_large_tensors_take_several_chunks_a_cta(shift, dtype, n):
    """Sizes at which a CTA takes several chunks (up to 32), aligned and not, beside a
    short tensor: windows of blocks at the start, around the CTAs' strides, in the
    middle and at the cut end, against the restatement."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    p = (torch.randn(n + shift, device="cuda", generator=gen) * 0.3).to(dtype)[shift:]
    g = (torch.randn(n + shift, device="cuda", generator=gen) * 1e-2).to(dtype)[shift:]
    small = torch.zeros(70, device="cuda")
    st, st2 = ops.adamw8_state(p), ops.adamw8_state(small)
    ops.adamw8_step([small, p], [small + 1, g], *zip(st2, st), step=1, seed=3, **HYPER)
    chunks = -(-n // 1024)  # four scale blocks
    blocks = -(-n // 256)
    starts = {0, blocks - 3, blocks // 2}
    for per in (2, 4, 8, 16, 32):
        stride = -(-chunks // per) * 4
        starts |= {b for b in (stride - 2, stride * (per - 1) - 1) if 0 <= b < blocks - 3}
    for b in sorted(starts):
        at, end = b * 256, min(n, (b + 3) * 256)
        zeros, scales = np.zeros(end - at, np.uint8), np.zeros(-(-(end - at) // 256), np.uint8)
        gs = g[at:end].float().cpu().numpy()
        new = oa.step8(gs, zeros, scales, zeros, scales, step=1, betas=HYPER["betas"], seed=3,
                       place=1, first_block=b)
        for got, want in zip((st[0][at:end], st[1][b:b + 3], st[2][at:end], st[3][b:b + 3]),
                             new[2:]):
            np.testing.assert_array_equal(got.cpu().numpy(), want)
    # what is left of the whole: no element was skipped or moved twice
    assert int((st[0] == 0).sum()) < n // 1000 and not (st[1] == 0).any()
    m, v = moments_zero(p), moments_zero(p)
    q = p.clone()
    p2 = torch.empty(n + shift, dtype=dtype, device="cuda")[shift:]
    p2.copy_(p)
    ops.adamw_step([q], [g.clone()], [m], [v], step=1, **HYPER)
    m2, v2 = moments_zero(p), moments_zero(p)
    ops.adamw_step([small, p2], [small, g], [moments_zero(small), m2], [moments_zero(small), v2],
                   step=1, **HYPER)
    assert torch.equal(q, p2) and torch.equal(m, m2) and torch.equal(v, v2)
    err = (m.double() - 0.1 * g.double()).abs() - 1e-6 * g.double().abs()
    assert bool((err <= 1e-44).all())


def moments_zero(p):
    return torch.zeros(p.numel(), dtype=F32, device="cuda")


def test_scalars_inference_tensors_and_tuples():
    gen = torch.Generator().manual_seed(8)
    s = make(1, F32, gen).view(())
    st = ops.adamw8_state(s)
    step8_and_check([s], [s.clone()], [st], 1)
    with torch.inference_mode():
        p, g = make(700, F32, gen), make(700, F32, gen)
        m, v = moments32(p, gen)
        want = oa.adamw64(n64(p), n64(g), n64(m), n64(v), 2, **HYPER)
        norm, scale = ops.grad_norm((g,))
        ops.adamw_step((p,), (g,), (m,), (v,), step=2, **HYPER)
        check_param(p, F32, want[0], want[3][0])


# --- refusals ---------------------------------------------------------------

def test_refusals():
    def t(n=8, dtype=F32):
        return torch.zeros(n, dtype=dtype, device="cuda")
    p, g, m, v = t(), t(), t(), t()
    cases = [
        (([p], [t(8, BF16)], [m], [v]), "grads\\[0\\] must have its parameter's shape and type"),
        (([p], [t(7)], [m], [v]), "grads\\[0\\] must have its parameter's shape and type"),
        (([p], [g], [t(8, F16)], [v]), "exp_avgs\\[0\\] must be Float, got Half"),
        (([p], [g], [m], [t(9)]), "exp_avg_sqs\\[0\\] must have its parameter's shape"),
        (([t(8, torch.float64)], [t(8, torch.float64)], [m], [v]), "params\\[0\\] must be float32"),
        (([t(16)[::2]], [g], [m], [v]), "params\\[0\\] must be non-overlapping and dense"),
        (([p], [torch.zeros(8)], [m], [v]), "grads\\[0\\] must be a CUDA tensor"),
        (([p], [g.to_sparse()], [m], [v]), "grads\\[0\\] must be a dense tensor"),
        (([p, p], [g, g], [m, t()], [v, t()]), "params\\[1\\] is given twice"),
        (([p, t()], [g, g], [m, m], [v, t()]), "exp_avgs\\[1\\] is given twice"),
        (([p], [g], [m], [m]), "exp_avg_sqs\\[0\\] is given twice"),
    ]
    for args, msg in cases:
        with pytest.raises(ValueError, match=msg):
            ops.adamw_step(*args, step=1)
    a = t(12).view(3, 4)
    with pytest.raises(ValueError, match="shape and strides"):
        ops.adamw_step([a], [a.clone()], [t(12).view(4, 3).t()], [t(12).view(3, 4)], step=1)
    for scale in (torch.ones(2, device="cuda"), torch.ones((), device="cuda", dtype=BF16),
                  torch.ones(())):
        with pytest.raises(ValueError, match="grad_scale must be one float32 value"):
            ops.adamw_step([p], [g], [m], [v], step=1, grad_scale=scale)
    with pytest.raises(ValueError, match="step must be an int"):
        ops.adamw_step([p], [g], [m], [v], step=torch.ones((), device="cuda"))
    c, s = t(8, torch.uint8), t(1, torch.uint8)
    for args, msg in (
            (([p], [g], [m], [s], [c], [t(1, torch.uint8)]), "exp_avgs\\[0\\] must be Byte"),
            (([p], [g], [c], [t(2, torch.uint8)], [t(8, torch.uint8)], [s]),
             "exp_avg_scales\\[0\\] must be 1 contiguous uint8 scales"),
            (([p], [g], [c], [s], [t(8, torch.uint8)], [s]), "exp_avg_sq_scales\\[0\\] is given twice"),
            (([p], [g], [c], [s], [c], [t(1, torch.uint8)]), "exp_avg_sqs\\[0\\] is given twice")):
        with pytest.raises(ValueError, match=msg):
            ops.adamw8_step(*args, step=1)
    with pytest.raises(ValueError, match="params\\[0\\] must not be a lazily negated view"):
        ops.adamw_step([torch._neg_view(p)], [g], [m], [v], step=1)
    with pytest.raises(ValueError, match="exp_avgs\\[0\\] must not be a lazily negated view"):
        ops.adamw_step([p], [g], [torch._neg_view(m)], [v], step=1)
    with pytest.raises(ValueError, match="out\\[0\\]\\[0\\] must be Float"):
        ops.adamw8_moments([c], [s], [c], [s], out=([c], [t()]))
    assert not p.any() and not m.any() and not v.any() and not c.any() and not s.any()
    assert p._version == 0  # a refused call has changed nothing


# --- optimiser --------------------------------------------------------------

def _fit(params, opt, grads, steps):
    for t in range(steps):
        for p, g in zip(params, grads(t)):
            p.grad = g
        opt.step()


@pytest.mark.parametrize("capturable", [False, True])
def test_optimizer_matches_float64_with_groups_and_clipping(capturable):
    """Two groups, one parameter without a gradient at first, clipped; every step
    is compared from the state before it."""
    gen = torch.Generator().manual_seed(0)
    ps = [make(n, F32, gen, 0.3).requires_grad_() for n in (12288, 1536, 700)]
    opt = manbo.AdamW([{"params": ps[:1], "lr": 0.5}, {"params": ps[1:], "weight_decay": 0.0}],
                      lr=0.01, max_grad_norm=0.5, capturable=capturable)
    for t in range(1, 5):
        for i, p in enumerate(ps):
            p.grad = make(p.numel(), F32, gen) if i < 2 or t > 2 else None
        before = [(n64(p), *((n64(x) for x in opt.moments(p)) if opt.state[p] else
                             (np.zeros(p.numel()),) * 2)) for p in ps]
        norm, c = oa.norm64([n64(p.grad) for p in ps if p.grad is not None], 0.5)
        c = float(np.float32(c))
        opt.step()
        assert abs(float(opt.grad_norm) - norm) <= 6.1e-8 * norm
        for i, (p, b) in enumerate(zip(ps, before)):
            if p.grad is None:
                assert not opt.state[p]
                continue
            step = t if i < 2 else t - 2
            assert int(opt.state[p]["step"]) == step
            # the clip factor itself is one rounding (2^-24) off: g' and so m and v's terms
            want = oa.adamw64(b[0], n64(p.grad), b[1], b[2], step, lr=0.5 if i == 0 else 0.01,
                              weight_decay=0.01 if i == 0 else 0.0, scale=c)
            m, v = opt.moments(p)
            assert (np.abs(n64(m) - want[1]) <= want[3][1] * 2).all()
            assert (np.abs(n64(v) - want[2]) <= want[3][2] * 2).all()
            assert (np.abs(n64(p) - want[0]) <= want[3][0] * 2).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_equal_eager_ones(bits):
    """A step captured once and replayed, gradients refilled between replays,
    against an eager optimiser; a schedule writes the learning rate."""
    def build():
        gen = torch.Generator().manual_seed(1)
        ps = [make(n, F32, gen, 0.3).requires_grad_() for n in (3000, 257, 1)]
        lr = torch.tensor(0.02, device="cuda")
        opt = manbo.AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 0.1}], lr=lr,
                          state_bits=bits, max_grad_norm=1.0, capturable=True, seed=5)
        for p in ps:
            p.grad = torch.zeros_like(p)
        return ps, opt, lr

    def fill(ps, t):
        gen = torch.Generator().manual_seed(100 + t)
        for p in ps:
            p.grad.copy_(make(p.numel(), F32, gen))

    runs = []
    for captured in (False, True):
        ps, opt, lr = build()
        fill(ps, 0)
        opt.step()
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
        norms = []
        for t in range(1, 5):
            fill(ps, t)
            lr.fill_(0.02 / t)
            graph.replay() if captured else opt.step()
            norms.append(opt.grad_norm.clone())
        runs.append((ps, [x for p in ps for x in opt.moments(p)], norms,
                     [opt.state[p]["step"] for p in ps]))
    a, b = runs
    assert [int(x) for x in a[3]] == [5, 5, 5] == [int(x) for x in b[3]]
    for x, y in zip((*a[0], *a[1], *a[2]), (*b[0], *b[1], *b[2])):
        assert torch.equal(x, y)


def test_capture_needs_a_capturable_optimiser_with_state():
    p = torch.zeros(10, device="cuda", requires_grad=True)
    p.grad = torch.ones_like(p)
    for opt, msg in ((manbo.AdamW([p]), "capturable=True"),
                     (manbo.AdamW([p], capturable=True), "one step before capturing")):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match=msg):
            with torch.cuda.graph(graph):
                p.grad.mul_(1.0)
                opt.step()
        assert not opt.state[p]
    assert not p.any()


def test_two_captured_optimisers_on_two_streams():
    """Each captured step owns its workspaces: replays on two streams at once
    give what replays one after the other give."""
    def build():
        out = []
        for seed in (1, 2):
            gen = torch.Generator().manual_seed(seed)
            ps = [make(200_000, F32, gen, 0.3).requires_grad_() for _ in range(3)]
            opt = manbo.AdamW(ps, max_grad_norm=0.1, state_bits=8, capturable=True)
            for p in ps:
                p.grad = make(p.numel(), F32, gen)
            opt.step()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
            out.append((ps, opt, graph))
        return out

    one, two = build(), build()
    for _, _, graph in one:
        for _ in range(20):
            graph.replay()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for s, (_, _, graph) in zip(streams, two):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (pa, oa_, _), (pb, ob, _) in zip(one, two):
        assert torch.equal(oa_.grad_norm, ob.grad_norm)
        assert all(torch.equal(x, y) for x, y in zip(pa, pb))


def test_steps_on_a_side_stream():
    gen, params, grads = _mixed(30, 8)
    ms, vs = zip(*[moments32(p, gen) for p in params])
    copies = [[x.clone() for x in xs] for xs in (params, ms, vs)]
    norm, scale = ops.grad_norm(grads, max_norm=0.01)
    ops.adamw_step(params, grads, ms, vs, step=2, grad_scale=scale, **HYPER)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        norm, scale = ops.grad_norm(grads, max_norm=0.01)
        ops.adamw_step(*(copies[0], grads, copies[1], copies[2]), step=2, grad_scale=scale, **HYPER)
    side.synchronize()
    for a, b in zip((params, ms, vs), copies):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_step_invalidates_saved_parameters():
    """The parameters are versioned: a backward through a graph that saved them
    before the step is refused, as with any in-place change."""
    p = torch.ones(5, device="cuda", requires_grad=True)
    y = (p * p).sum()
    p.grad = torch.ones_like(p)
    manbo.AdamW([p]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("capturable", [False, True])
def test_state_dict_round_trip(bits, capturable):
    gen = torch.Generator().manual_seed(3)
    ps = [make(n, d, gen, 0.3).requires_grad_() for n, d in ((5000, BF16), (300, F32))]
    grads = [[make(p.numel(), p.dtype, gen) for p in ps] for _ in range(6)]
    opt = manbo.AdamW(ps, state_bits=bits, capturable=capturable, seed=9)
    _fit(ps, opt, lambda t: grads[t], 3)
    saved = opt.state_dict()
    qs = [p.detach().clone().requires_grad_() for p in ps]
    other = manbo.AdamW(qs, state_bits=bits, capturable=capturable)
    other.load_state_dict(saved)
    _fit(ps, opt, lambda t: grads[3 + t], 3)
    _fit(qs, other, lambda t: grads[3 + t], 3)
    for p, q in zip(ps, qs):
        assert torch.equal(p, q) and int(other.state[q]["step"]) == 6
        for a, b in zip(opt.moments(p), other.moments(q)):
            assert a.dtype == F32 and torch.equal(a, b)
    if bits == 8:
        assert other.state[qs[0]]["exp_avg"].dtype == torch.uint8
        with pytest.raises(ValueError, match="state_bits"):
            other.param_groups[0]["state_bits"] = 32
            other.step()


def test_many_groups_of_every_kind_in_one_optimiser():
    """More groups than a launch takes, 32- and 8-bit ones, own seeds, betas and
    rates: the same as an optimiser for each group (8-bit: whose places in a list
    are then others, so only one group of that kind for each seed)."""
    def build():
        gen = torch.Generator().manual_seed(2)
        return [make(200 + 13 * i, [F32, BF16, F16][i % 3], gen, 0.3).requires_grad_()
                for i in range(40)], gen

    def options(i):
        o = dict(lr=1e-3 * (i + 1), betas=(0.5 + 0.01 * i, 0.9), eps=1e-8 * (i + 1),
                 weight_decay=0.01 * i)
        return {**o, "state_bits": 8, "seed": i} if i % 10 == 7 else o
    together, gen = build()
    apart, _ = build()
    opt = manbo.AdamW([{"params": [p], **options(i)} for i, p in enumerate(together)])
    each = [manbo.AdamW([p], **options(i)) for i, p in enumerate(apart)]
    for _ in range(3):
        for p, q in zip(together, apart):
            p.grad = make(p.numel(), p.dtype, gen)
            q.grad = p.grad.clone()
        opt.step()
        for o in each:
            o.step()
    for p, q, o in zip(together, apart, each):
        assert torch.equal(p, q)
        assert all(torch.equal(a, b) for a, b in zip(opt.moments(p), o.moments(q)))


def test_state_of_torch_adamw_loads_and_continues():
    """Two steps of torch's AdamW, then one here from its state, against float64
    from that state; what this class does not compute is refused."""
    gen = torch.Generator().manual_seed(3)
    p = make(1000, F32, gen, 0.3).requires_grad_()
    kw = dict(lr=1e-2, betas=(0.8, 0.99), weight_decay=0.1)
    old = torch.optim.AdamW([p], **kw)
    for _ in range(2):
        p.grad = make(1000, F32, gen)
        old.step()
    opt = manbo.AdamW([p])
    opt.load_state_dict(old.state_dict())
    m, v = opt.moments(p)
    p.grad = make(1000, F32, gen)
    want = oa.adamw64(n64(p), n64(p.grad), n64(m), n64(v), 3, **kw)
    opt.step()
    check_param(p, F32, want[0], want[3][0])
    assert opt.state[p]["step"] == 3
    for other in (torch.optim.AdamW([p], amsgrad=True), torch.optim.AdamW([p], maximize=True),
                  torch.optim.Adam([p])):
        with pytest.raises(ValueError, match="does not support"):
            opt.load_state_dict(other.state_dict())


@pytest.mark.parametrize("bits", [8, 32])
def test_fit_of_a_scene_runs_with_adamw(bits):
    """Renderer, loss, backward, clipping and step together: three steps of a
    small fill scene, each step's update checked against float64 from the
    renderer's own gradients."""
    from repo_b200 import scenes
    sc = scenes.small_fill_scene(1234, h=48, w=64, paths=6)
    cn = sc.cubics_norm().cuda().requires_grad_(True)
    col = sc.colors.cuda().requires_grad_(True)
    fixed = [x.cuda() for x in (sc.seg_offsets(), sc.opacities, sc.depths, sc.background)]
    opt = manbo.AdamW([{"params": [cn], "lr": 1e-3}, {"params": [col], "lr": 1e-2}],
                      weight_decay=0.0, max_grad_norm=0.05, state_bits=bits)
    target = torch.rand(48, 64, 3, generator=torch.Generator().manual_seed(1)).cuda()
    for t in range(1, 4):
        opt.zero_grad(set_to_none=t % 2 == 0)
        out = manbo.ops.render_cubic_fill_splat_tilelang(
            cn, fixed[0], col, fixed[1], fixed[2], 48, 64, 16, 16, fixed[3],
            fill_rules=sc.fill_rules.cuda(), aa_widths=sc.aa_widths.cuda(),
            distance_samples=sc.samples)
        manbo.mse_loss_tilelang(out, target).backward()
        before = [(n64(p), *((n64(x) for x in opt.moments(p)) if opt.state[p] else
                             (np.zeros(p.numel()),) * 2)) for p in (cn, col)]
        _, c = oa.norm64([n64(cn.grad), n64(col.grad)], 0.05)
        opt.step()
        for p, b, lr in ((cn, before[0], 1e-3), (col, before[1], 1e-2)):
            want = oa.adamw64(b[0], n64(p.grad), b[1], b[2], t, lr=lr, weight_decay=0.0,
                              scale=float(np.float32(c)))
            assert (np.abs(n64(p) - want[0]) <= 2 * want[3][0]).all()
