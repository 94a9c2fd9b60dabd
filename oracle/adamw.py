"""CPU restatement of the AdamW operators (test infrastructure only).

``adamw64`` and ``norm64`` are the definitions in float64.  The 8-bit moments
are restated in numpy float32 and uint32, operation by operation, so that the
kernels' bytes can be compared for equality: a block of 256 elements has a scale
byte E (2^(E - 127), at least E = 40, 255 for a block that is not finite), an
element of m is a sign, 4 exponent and 3 fraction bits in units of the scale, an
element of v 5 exponent and 3 fraction bits, both with gradual underflow and
rounded stochastically by 16 hashed bits.
"""
import numpy as np

BLOCK = 256
U32 = np.uint32
F32 = np.float32


def norm64(grads, max_norm=0.0, eps=1e-6):
    n = np.sqrt(sum(float(np.sum(np.asarray(g, np.float64) ** 2)) for g in grads))
    if max_norm <= 0:
        return n, 1.0
    with np.errstate(invalid="ignore"):
        q = np.float64(max_norm) / (n + eps)
    return n, (1.0 if q > 1.0 else q)


def adamw64(p, g, m, v, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
            scale=1.0):
    """(p, m, v, bounds): the step in float64, with how far a float32 evaluation
    of each may be off, before a 16-bit parameter's own rounding.

    With u = 2^-24, one rounding an operation and float32 constants: m sums
    b1 m (3 roundings: b1, product, sum) and (1-b1) g' (4: g', 1-b1, product,
    sum); v sums non-negative terms of 3 and 6 roundings (g' counts twice);
    p (1 - lr wd) has the decay's rounding and lr's and wd's (both times
    lr wd << 1), the product's and the difference's (4 in all); the update has
    lr, 1/(1-b1^t) and their product (3), sqrt(v): half of v's 6 and its own
    (4), 1/sqrt(1-b2^t), product, eps, sum (4), division, product and
    difference (3), 14 in all, and m's error over the denominator.
    """
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    b1, b2 = betas
    g = g * scale
    m1 = b1 * m + (1 - b1) * g
    v1 = b2 * v + (1 - b2) * g * g
    denom = np.sqrt(v1) / np.sqrt(1 - b2 ** step) + eps
    size = lr / (1 - b1 ** step)
    with np.errstate(invalid="ignore"):
        update = size * m1 / denom
        p1 = p * (1 - lr * weight_decay) - update
        u = 2.0 ** -24
        bm = 4.1 * u * (np.abs(b1 * m) + np.abs((1 - b1) * g)) + 1e-44
        bv = 6.1 * u * v1 + 1e-44
        bp = u * (4.1 * np.abs(p) + 16 * np.abs(update)) + size * bm / denom + 1e-44
    return p1, m1, v1, (bp, bm, bv)


# --- 8-bit moments ----------------------------------------------------------

def mix(h):
    """32-bit multiply-xorshift hash."""
    h = np.asarray(h, np.uint64) & 0xFFFFFFFF
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(0x6A09E667)) & 0xFFFFFFFF
    h = ((h ^ (h >> np.uint64(15))) * np.uint64(0xBB67AE85)) & 0xFFFFFFFF
    return h ^ (h >> np.uint64(16))


def random_bits(seed, step, place, numel, first_block=0):
    """The 32 bits of every element from a block on, as uint32 [numel]."""
    key = int(mix((seed + (step & 0xFFFFFFFF) * 0x9E3779B1) & 0xFFFFFFFF))
    block = np.arange(-(-numel // BLOCK), dtype=np.uint64) + np.uint64(first_block)
    start = (key + place * 0x3C6EF373) & 0xFFFFFFFF
    b = mix((start + block * np.uint64(0xA54FF53B)) & 0xFFFFFFFF)
    h = (b[:, None] + np.arange(BLOCK, dtype=np.uint64) * np.uint64(0x9E3779B1)) & 0xFFFFFFFF
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(0x6A09E667)) & 0xFFFFFFFF
    return (h ^ (h >> np.uint64(15))).astype(U32).reshape(-1)[:numel]


def _rows(x):
    x = np.asarray(x).reshape(-1)
    return np.pad(x, (0, -x.size % BLOCK)).reshape(-1, BLOCK)


def scale_bytes(x):
    """The scale byte of every block of float32 values."""
    bits = (_rows(np.asarray(x, F32)).view(U32) & U32(0x7FFFFFFF)).max(axis=1).astype(np.int64)
    e = np.maximum((bits + 0xFFFFF) >> 23, 40)
    return np.where(e >= 254, 255, e).astype(np.uint8)


def _encode(x, rand16, power, signed):
    x = np.asarray(x, F32).reshape(-1)
    e = scale_bytes(x)
    inverse = np.where(e == 255, F32(0), np.ldexp(F32(1), 127 - e.astype(np.int64)).astype(F32))
    inverse = np.repeat(inverse, BLOCK)[:x.size]
    with np.errstate(all="ignore"):
        y = ((x * inverse).astype(F32) * F32(2.0 ** -power)).astype(F32)
    bits = y.view(U32).astype(np.int64)
    code = ((bits & 0x7FFFFFFF) + (np.asarray(rand16, np.int64) << 4)) >> 20
    if signed:
        return ((code & 127) | ((bits >> 24) & 128)).astype(np.uint8), e
    return (np.maximum(code, x > 0) & 255).astype(np.uint8), e


def encode_m(x, rand16):
    return _encode(x, rand16, 112, True)


def encode_v(x, rand16):
    return _encode(x, rand16, 96, False)


def _decode(code, scales, power, signed):
    code = np.asarray(code, np.uint8).reshape(-1).astype(U32)
    e = np.repeat(np.asarray(scales, np.int64), BLOCK)[:code.size]
    unit = np.where(e == 255, F32(np.nan),
                    np.where(e == 0, F32(0), np.ldexp(F32(1), np.minimum(e, 254) - 127)))
    size = (code & U32(127) if signed else code) << U32(20)
    with np.errstate(all="ignore"):
        x = (size.view(F32) * F32(2.0 ** power)).astype(F32) * unit.astype(F32)
    return np.where(code > 127, -x, x).astype(F32) if signed else x.astype(F32)


def decode_m(code, scales):
    return _decode(code, scales, 112, True)


def decode_v(code, scales):
    return _decode(code, scales, 96, False)


def step8(g, m_codes, m_scales, v_codes, v_scales, *, step, betas=(0.9, 0.999), scale=None,
          seed=0, place=0, first_block=0):
    """The moments' part of an 8-bit step: (m, v, m codes, m scales, v codes, v
    scales), m and v the float32 averages before rounding, everything flat."""
    b1, b2 = betas
    g = np.asarray(g, F32).reshape(-1)
    with np.errstate(all="ignore"):
        if scale is not None:
            g = (g * F32(scale)).astype(F32)
        m = (decode_m(m_codes, m_scales) * F32(b1)).astype(F32) + (g * F32(1 - b1)).astype(F32)
        v = (decode_v(v_codes, v_scales) * F32(b2)).astype(F32) \
            + ((g * g).astype(F32) * F32(1 - b2)).astype(F32)
    bits = random_bits(seed, step, place, g.size, first_block)
    mc, me = encode_m(m, bits & U32(0xFFFF))
    vc, ve = encode_v(v, bits >> U32(16))
    return m.astype(F32), v.astype(F32), mc, me, vc, ve
