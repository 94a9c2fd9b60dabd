"""The CPU restatement of the 8-bit moments: format, rounding, random bits."""
import numpy as np
import pytest

from oracle import adamw as oa


def _grid(signed):
    """Every value a code stands for in units of the scale, from its definition."""
    out = []
    for c in range(256):
        k = c & 127 if signed else c
        top = 15 if signed else 31
        x = (k & 7) / 8 * 2.0 ** (1 - top) if k < 8 else (1 + (k & 7) / 8) * 2.0 ** ((k >> 3) - top)
        out.append(-x if signed and c > 127 else x)
    return np.array(out)


@pytest.mark.parametrize("e", [40, 100, 127, 200, 253])
def test_every_code_decodes_to_its_definition_and_encodes_back(e):
    codes = np.arange(256, dtype=np.uint8)
    for signed, dec, enc in ((True, oa.decode_m, oa.encode_m), (False, oa.decode_v, oa.encode_v)):
        x = dec(codes, np.array([e]))
        np.testing.assert_array_equal(x.astype(np.float64), _grid(signed) * 2.0 ** (e - 127))
        for r in (0, 0x8000, 0xFFFF):  # a value on the grid stays, whatever the random bits
            c, s = enc(x, np.full(256, r))
            assert s[0] == e
            np.testing.assert_array_equal(c, codes)


def test_zeroed_bytes_and_marked_blocks():
    z = np.zeros(300, np.uint8)
    assert (oa.decode_m(z, np.zeros(2, np.uint8)) == 0).all()
    assert (oa.decode_v(z, np.zeros(2, np.uint8)) == 0).all()
    x = np.ones(600, np.float32)
    x[300] = np.nan
    x[599] = 2.0 ** 127
    assert oa.scale_bytes(x).tolist() == [127, 255, 255]
    c, s = oa.encode_m(x, np.zeros(600))
    y = oa.decode_m(c, s)
    assert (y[:256] == 1).all() and np.isnan(y[256:]).all()


def test_scale_is_the_smallest_power_that_holds_the_largest():
    for x, e in ((1.875, 127), (np.nextafter(np.float32(1.875), np.float32(2)), 128), (1.0, 127),
                 (0.0, 40), (1e-38, 40), (-3.0, 128), (1.8e38, 255), (-np.inf, 255)):
        assert oa.scale_bytes(np.array([x, 0], np.float32)).tolist() == [e], x


@pytest.mark.parametrize("signed", [True, False])
def test_rounding_goes_to_a_neighbour_and_is_unbiased(signed):
    """Over all 2^16 random values the mean of the rounding is the value, to
    2^-16 of the gap (the bits below the random ones are cut)."""
    rng = np.random.default_rng(1)
    grid = np.sort(np.unique(_grid(signed)))
    enc, dec = (oa.encode_m, oa.decode_m) if signed else (oa.encode_v, oa.decode_v)
    for x in np.concatenate([rng.uniform(0, 1.8, 6), 2.0 ** rng.uniform(-13, 0, 6)]):
        x = np.float32(-x if signed and rng.random() < 0.5 else x)
        col = np.full(1 << 16, x, np.float32)
        col[::256] = 1.0  # the block's largest keeps the scale at 2^0
        r = np.arange(1 << 16)
        c, s = enc(col, r)
        assert (s == (128 if abs(x) > 1.875 else 127)).all()
        y = dec(c, s).astype(np.float64)
        keep = np.arange(1 << 16) % 256 != 0
        lo = grid[np.searchsorted(grid, x, "right") - 1]
        hi = grid[np.searchsorted(grid, x, "left")]
        assert set(np.unique(y[keep])) <= {lo, hi}
        # the removed columns (1/256 of the random values, spread evenly) move the mean by < gap/256
        assert abs(y[keep].mean() - x) <= (hi - lo) * (2.0 ** -16 + 1 / 256)


def test_a_positive_v_never_becomes_zero():
    x = np.zeros(256, np.float32)
    x[0], x[1], x[2] = 1.0, 1e-30, 1e-45
    for r in (0, 0xFFFF):
        c, s = oa.encode_v(x, np.full(256, r))
        assert c[1] >= 1 and c[2] >= 1 and (c[3:] == 0).all() if r == 0 else c[1] >= 1


def test_random_bits_are_even_and_differ():
    """Means, bit counts and correlations of 2^20 hashes within 6 standard
    deviations of independent fair bits."""
    n = 1 << 20
    a = oa.random_bits(7, 100, 3, n)
    for other in (oa.random_bits(8, 100, 3, n), oa.random_bits(7, 101, 3, n),
                  oa.random_bits(7, 100, 4, n), np.roll(a, 1), np.roll(a, 256)):
        agree = np.unpackbits((a ^ other).view(np.uint8)).mean()
        assert abs(agree - 0.5) < 6 * 0.5 / np.sqrt(32 * n)
    for half in (a & 0xFFFF, a >> 16):
        assert abs(half.mean() - 32767.5) < 6 * 65536 / np.sqrt(12 * n)
        counts = np.bincount(half >> 8, minlength=256)
        assert abs(counts - n / 256).max() < 6 * np.sqrt(n / 256)
    lo, hi = (a & 0xFFFF).astype(float), (a >> 16).astype(float)
    assert abs(np.corrcoef(lo, hi)[0, 1]) < 6 / np.sqrt(n)


def test_eight_bit_averages_follow_the_32_bit_ones():
    """400 steps of constant-variance gradients: the block means of the 8-bit
    averages follow the float64 ones; by rounding to nearest v would stay where
    it is.  A mean over 256 elements of a rounding noise below one code's gap
    (1/8 of the value) that the average forgets at rate 1 - beta: its variance
    is at most gap * |drift| / (2 (1 - beta)), the drift at most (1 - beta)
    times the distance to the target, so a standard deviation below 40% an
    element and 2.5% a block; five of them."""
    rng = np.random.default_rng(3)
    n, blocks = 256 * 16, 16
    mc = np.zeros(n, np.uint8)
    vc = np.zeros(n, np.uint8)
    me = np.zeros(blocks, np.uint8)
    ve = np.zeros(blocks, np.uint8)
    v = np.zeros(n)
    size = np.exp(rng.standard_normal(n) * 0.5)
    for t in range(1, 401):
        g = (rng.standard_normal(n) * size * (0.3 if t > 200 else 1.0)).astype(np.float32)
        _, _, mc, me, vc, ve = oa.step8(g, mc, me, vc, ve, step=t, seed=11)
        v = 0.999 * v + 0.001 * g.astype(np.float64) ** 2
    got = oa.decode_v(vc, ve).astype(np.float64).reshape(blocks, 256).mean(axis=1)
    want = v.reshape(blocks, 256).mean(axis=1)
    assert np.abs(got / want - 1).max() < 0.125


def test_norm_and_step_in_64_bits_against_a_hand_worked_case():
    n, c = oa.norm64([[3.0, 0.0], [4.0]], max_norm=2.5, eps=0.0)
    assert n == 5.0 and c == 0.5
    assert oa.norm64([[3.0]], max_norm=5.0)[1] == 1.0
    p, m, v, _ = oa.adamw64([1.0], [2.0], [0.0], [0.0], 1, lr=0.1, weight_decay=0.5, eps=0.0)
    # the first step moves by lr times the gradient's sign after the decay
    assert abs(m[0] - 0.2) < 1e-15 and abs(v[0] - 0.004) < 1e-15 and abs(p[0] - (0.95 - 0.1)) < 1e-12
