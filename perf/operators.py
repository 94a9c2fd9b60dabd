"""Cases of the optimiser operators: the global gradient norm and the AdamW step
over many tensors at once, with its moments in 32 bits or in 8.

Formulas (t the step, c the gradient scale, 1 where none is given):

  norm    n = sqrt(sum of g^2 over every gradient),
          c = min(1, max_norm / (n + 1e-6)), or 1 where max_norm is 0
  adamw   g' = c g,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2,
          p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
  adamw8  the same step, with m and v held as one byte an element and one scale
          byte for each block of 256 elements of a tensor (in storage order)

The 8-bit format.  A block's scale byte E stands for 2^(E - 127), the smallest
power of two (E at least 40) with max |x| <= 1.875 2^(E - 127); a block whose
largest magnitude needs E >= 254, or is not a number, gets 255 and stands for
NaN.  An element of m is a sign, 4 exponent and 3 fraction bits, an element of
v is 5 exponent and 3 fraction bits, both with gradual underflow, in units of
the scale.  That is the top of a float32's bits after scaling the block to the
bottom of the float32 range (2^-112 for m, 2^-96 for v): 20 low bits go.  They
go by stochastic rounding, without which an average that moves by 0.1% a step
would not move at all: 16 random bits, shifted by 4, are added to the float's
bits before the cut.  A v above zero never becomes zero.  The random bits come
from the seed, the step, the tensor's place in the list, the block and the
element by the integer hash in _random_bits.  The step's arithmetic on m and v
is float32, one rounding an operation, so the bytes are defined bit for bit.
"""
import math
import random

import torch

own = False

BLOCK = 256
M32 = 0xFFFFFFFF
HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
MAX_NORM = 1.0
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
MOST = 404_000_000  # elements of the largest listed case


def listed():
    return [
        # a fit of 512 closed paths: its ring points, colours, opacities and
        # widths, the smallest call, where only latency counts
        {"name": "norm-curves-512", "op": "norm", "layout": "curves", "paths": 512, "segs": 4, "dtype": "fp32"},
        # the gradients of a network with many small and odd tensors of every type
        {"name": "norm-ragged-mixed", "op": "norm", "layout": "ragged", "count": 240, "least": 1, "most": 400_000, "shapes": 1,
         "dtype": "mixed", "packed": False},
        # two wide layers in bf16: the norm is one read of every gradient
        {"name": "norm-layers-bf16", "op": "norm", "layout": "layers", "layers": 2, "width": 4096, "hidden": 16384, "dtype": "bf16"},
        # the same fit's step
        {"name": "adamw-curves-512", "op": "adamw", "layout": "curves", "paths": 512, "segs": 4, "dtype": "fp32", "step": 1, "clip": False},
        # the largest path count of the sweep, clipped: norm and step together
        {"name": "adamw-curves-16384-clip", "op": "adamw", "layout": "curves", "paths": 16384, "segs": 4, "dtype": "fp32", "step": 50,
         "clip": True},
        # many odd tensors packed end to end in one buffer, so hardly any is aligned
        {"name": "adamw-ragged-packed", "op": "adamw", "layout": "ragged", "count": 300, "least": 1, "most": 300_000, "shapes": 2,
         "dtype": "mixed", "packed": True, "step": 700, "clip": True},
        # a whole training step's update of wide layers, in float32 and in bf16
        {"name": "adamw-layers-fp32", "op": "adamw", "layout": "layers", "layers": 5, "width": 2048, "hidden": 8192, "dtype": "fp32",
         "step": 3000, "clip": False},
        {"name": "adamw-layers-bf16", "op": "adamw", "layout": "layers", "layers": 2, "width": 4096, "hidden": 16384, "dtype": "bf16",
         "step": 3000, "clip": False},
        # the fit's step with 8-bit moments
        {"name": "adamw8-curves-512", "op": "adamw8", "layout": "curves", "paths": 512, "segs": 4, "dtype": "fp32", "step": 1, "clip": False},
        # odd tensors of every type, aligned as an allocator gives them
        {"name": "adamw8-ragged-mixed", "op": "adamw8", "layout": "ragged", "count": 300, "least": 1, "most": 300_000, "shapes": 3,
         "dtype": "mixed", "packed": False, "step": 700, "clip": True},
        # wide layers whose moments would not fit otherwise
        {"name": "adamw8-layers-fp32", "op": "adamw8", "layout": "layers", "layers": 5, "width": 2048, "hidden": 8192, "dtype": "fp32",
         "step": 3000, "clip": False},
        {"name": "adamw8-layers-bf16", "op": "adamw8", "layout": "layers", "layers": 2, "width": 4096, "hidden": 16384, "dtype": "bf16",
         "step": 3000, "clip": True},
    ]


def _log(rng, least, most):
    return int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))


def draw(rng):
    case = {"op": rng.choice(["norm", "adamw", "adamw", "adamw8", "adamw8"])}
    case["layout"] = rng.choice(["curves", "ragged", "layers"])
    if case["layout"] == "curves":
        case.update(paths=_log(rng, 16, 20000), segs=rng.randint(1, 9), dtype="fp32")
    elif case["layout"] == "ragged":
        case.update(count=_log(rng, 2, 400), least=_log(rng, 1, 300), most=_log(rng, 2000, 900_000), shapes=rng.randrange(1 << 20),
                    dtype=rng.choice(["fp32", "bf16", "fp16", "mixed"]), packed=rng.random() < 0.4)
    else:
        width = _log(rng, 64, 4096)
        hidden = rng.choice([4 * width, _log(rng, 128, 16384)])
        each = 4 * width * width + 2 * width * hidden + 2 * width
        case.update(layers=_log(rng, 1, max(1, min(48, MOST // each))), width=width, hidden=hidden, dtype=rng.choice(["fp32", "bf16", "fp16"]))
    if case["op"] != "norm":
        case.update(step=_log(rng, 1, 100_000), clip=rng.random() < 0.5)
    return case


def _shapes(case):
    """The tensors of a case: (shape, type) each."""
    if case["layout"] == "curves":
        p, s = case["paths"], case["segs"]
        shapes = [(p, 3 * s, 2), (p, 3), (p,), (p,)]
    elif case["layout"] == "layers":
        h, f = case["width"], case["hidden"]
        shapes = [(h, h), (h, h), (h, h), (h, h), (h, f), (f, h), (h,), (h,)] * case["layers"]
    else:
        rng = random.Random(case["shapes"])
        shapes = [(_log(rng, case["least"], case["most"]),) for _ in range(case["count"])]
    kinds = list(DTYPES) if case["dtype"] == "mixed" else [case["dtype"]]
    return [(s, kinds[i % len(kinds)]) for i, s in enumerate(shapes)]


def _sizes(case):
    return [(math.prod(s), k) for s, k in _shapes(case)]


def work(case):
    """Each input read once and each output written once: parameters, gradients
    and moments (for adamw8 also the moments' values, which run() returns)."""
    sizes = _sizes(case)
    n = sum(k for k, _ in sizes)
    grads = sum(k * BYTES[d] for k, d in sizes)
    if case["op"] == "norm":
        return {"bytes": grads + 8, "flops": 2 * n}
    clip = 2 * n if case["clip"] else 0
    if case["op"] == "adamw":
        return {"bytes": 3 * grads + 16 * n, "flops": 14 * n + clip}
    blocks = sum(-(-k // BLOCK) for k, _ in sizes)
    return {"bytes": 3 * grads + 4 * n + 4 * blocks + 8 * n, "flops": 24 * n + clip}


def _views(flat, offsets, shapes):
    return [flat[o:o + math.prod(s)].view(s) for o, s in zip(offsets, shapes)]


def _offsets(counts, unit):
    at, found = 0, []
    for n in counts:
        found.append(at)
        at += -(-n // unit) * unit
    return found, at


def prepare(case, seed):
    """Every kind of tensor lives in one buffer for each type (a flat parameter
    buffer, a gradient bucket, a moment arena), as views on 512-byte borders, or
    end to end for the parameters and gradients of a packed case."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shapes = _shapes(case)
    only = [s for s, _ in shapes]
    counts = [math.prod(s) for s in only]
    state = {"case": case, "params": [None] * len(only), "grads": [None] * len(only), "flat_params": {}}

    def normal(n):
        return torch.randn(n, device="cuda", generator=gen)

    def gradients(n):
        # layers and rows differ in scale, and some rows get no gradient
        rows = -(-n // BLOCK)
        scale = torch.exp(normal(rows)) * 1e-3 * (torch.rand(rows, device="cuda", generator=gen) > 0.05)
        return (normal(rows * BLOCK).view(rows, BLOCK) * scale[:, None]).view(-1)[:n]

    for kind, dtype in DTYPES.items():
        mine = [i for i, (_, k) in enumerate(shapes) if k == kind]
        unit = 1 if case.get("packed") else 512 // BYTES[kind]
        offsets, total = _offsets([counts[i] for i in mine], unit)
        if not mine:
            continue
        grads = gradients(total).to(dtype)
        params = (normal(total) * 0.05).to(dtype)
        state["flat_params"][kind] = params
        for i, g, p in zip(mine, _views(grads, offsets, [only[i] for i in mine]), _views(params, offsets, [only[i] for i in mine])):
            state["grads"][i], state["params"][i] = g, p
    if case["op"] == "norm":
        return state
    state["step"], state["seed"] = case["step"], seed & M32
    state["grad_scale"] = None if case["clip"] else torch.tensor(0.5 + (seed % 97) / 194, device="cuda")
    offsets, total = _offsets(counts, 128)
    late = 1.0 - 0.9 ** (case["step"] - 1), 1.0 - 0.999 ** (case["step"] - 1)
    spread = torch.exp(normal(-(-total // BLOCK))).repeat_interleave(BLOCK)[:total] * 1e-3
    m = normal(total) * spread * (0.3 * late[0])
    v = (spread * torch.exp(0.5 * normal(total))).square() * late[1]
    if case["op"] == "adamw":
        state["flat_m"], state["flat_v"] = m, v
        state["exp_avgs"], state["exp_avg_sqs"] = _views(m, offsets, only), _views(v, offsets, only)
        return state
    state["flat_m"], state["flat_v"] = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    state["out"] = (_views(state["flat_m"], offsets, only), _views(state["flat_v"], offsets, only))
    half = torch.full((1, BLOCK), 0x8000, dtype=torch.int64, device="cuda")  # prepared states are rounded to nearest
    for name, flat, put in (("exp_avg", m, _to_m), ("exp_avg_sq", v, _to_v)):
        codes = torch.zeros(total, dtype=torch.uint8, device="cuda")
        state[name + "s"], state[name + "_scales"] = _views(codes, offsets, only), []
        for values, code in zip(_views(flat, offsets, only), state[name + "s"]):
            c, e = put(_blocks(values.reshape(-1)), half)
            code.view(-1).copy_(c.view(-1)[:code.numel()])
            state[name + "_scales"].append(e)
    return state


# --- the plain form ---------------------------------------------------------

def _blocks(x):
    """A flat tensor as rows of one block, the last one filled up with zeros."""
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _scale_bytes(x):
    bits = x.abs().amax(dim=1).view(torch.int32).to(torch.int64)
    e = ((bits + 0xFFFFF) >> 23).clamp(min=40)
    return torch.where(e >= 254, 255, e)


def _two_to(exponent):
    """2^exponent as float32, for whole exponents from -126 to 127 (0 below)."""
    return ((exponent + 127).clamp(min=0) << 23).to(torch.int32).view(torch.float32)


def _to_m(x, rand16):
    e = _scale_bytes(x)
    y = (x * _two_to(127 - e)[:, None]) * 2.0 ** -112
    bits = y.abs().view(torch.int32).to(torch.int64)
    code = ((bits + (rand16 << 4)) >> 20) & 127
    code = torch.where(torch.signbit(y), code + 128, code)
    return code.to(torch.uint8), e.to(torch.uint8)


def _to_v(x, rand16):
    e = _scale_bytes(x)
    y = (x * _two_to(127 - e)[:, None]) * 2.0 ** -96
    bits = y.abs().view(torch.int32).to(torch.int64)
    code = torch.maximum((bits + (rand16 << 4)) >> 20, (x > 0).to(torch.int64))
    return (code & 255).to(torch.uint8), e.to(torch.uint8)


def _unit(scale_bytes):
    e = scale_bytes.to(torch.int64)
    return torch.where(e == 255, math.nan, _two_to(e - 127))[:, None]


def _from_m(code, scale_bytes):
    c = code.to(torch.int32)
    size = ((c & 127) << 20).view(torch.float32) * 2.0 ** 112 * _unit(scale_bytes)
    return torch.where(c > 127, -size, size)


def _from_v(code, scale_bytes):
    return (code.to(torch.int32) << 20).view(torch.float32) * 2.0 ** 96 * _unit(scale_bytes)


def _mix(h):
    """A 32-bit integer hash, of whole numbers or tensors of them."""
    h = ((h ^ (h >> 16)) * 0x6A09E667) & M32
    h = ((h ^ (h >> 15)) * 0xBB67AE85) & M32
    return h ^ (h >> 16)


def _random_bits(seed, step, place, blocks, device):
    """32 random bits for every element of a tensor, [blocks, 256]."""
    key = _mix((seed + step * 0x9E3779B1) & M32)
    block = torch.arange(blocks, device=device, dtype=torch.int64)
    at = torch.arange(BLOCK, device=device, dtype=torch.int64)
    h = (_mix((key + place * 0x3C6EF373 + block * 0xA54FF53B) & M32)[:, None] + at * 0x9E3779B1) & M32
    h = ((h ^ (h >> 16)) * 0x6A09E667) & M32
    return h ^ (h >> 15)


def _moved(p, m, v, step, lr, betas, eps, weight_decay):
    step_size, root = lr / (1.0 - betas[0] ** step), 1.0 / math.sqrt(1.0 - betas[1] ** step)
    return p * (1.0 - lr * weight_decay) - step_size * (m / (v.sqrt() * root + eps))


def _plain_norm(grads, max_norm):
    n = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    c = torch.clamp(max_norm / (n + 1e-6), max=1.0) if max_norm > 0 else torch.ones_like(n)
    return n.float(), c.float()


def _plain_adamw(p, g, m, v, scale, step):
    b1, b2 = HYPER["betas"]
    g = g.float() if scale is None else g.float() * scale
    m.copy_(m * b1 + g * (1.0 - b1))
    v.copy_(v * b2 + (g * g) * (1.0 - b2))
    p.copy_(_moved(p.float(), m, v, step, **HYPER))


def _plain_adamw8(place, p, g, mc, me, vc, ve, out_m, out_v, scale, step, seed):
    b1, b2 = HYPER["betas"]
    n = p.numel()
    g = g.float().view(-1) if scale is None else g.float().view(-1) * scale
    g = _blocks(g)
    m = _from_m(_blocks(mc.view(-1)), me) * b1 + g * (1.0 - b1)
    v = _from_v(_blocks(vc.view(-1)), ve) * b2 + (g * g) * (1.0 - b2)
    p.copy_(_moved(p.float(), m.view(-1)[:n].view(p.shape), v.view(-1)[:n].view(p.shape), step, **HYPER))
    bits = _random_bits(seed, step, place, m.shape[0], p.device)
    m_codes, m_scales = _to_m(_blocks(m.view(-1)[:n]), bits & 0xFFFF)
    v_codes, v_scales = _to_v(_blocks(v.view(-1)[:n]), bits >> 16)
    mc.view(-1).copy_(m_codes.view(-1)[:n])
    vc.view(-1).copy_(v_codes.view(-1)[:n])
    me.copy_(m_scales)
    ve.copy_(v_scales)
    out_m.view(-1).copy_(_from_m(m_codes, m_scales).view(-1)[:n])
    out_v.view(-1).copy_(_from_v(v_codes, v_scales).view(-1)[:n])


def run(state):
    """norm: (norm, scale).  adamw, adamw8: the parameters, the moments as
    values and, where the step clips, the norm."""
    case, s = state["case"], state
    if own:
        from manbo import ops
        if case["op"] == "norm":
            return ops.grad_norm(s["grads"], max_norm=MAX_NORM)
        norm, scale = ops.grad_norm(s["grads"], max_norm=MAX_NORM) if case["clip"] else (None, s["grad_scale"])
        if case["op"] == "adamw":
            ops.adamw_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], step=s["step"], grad_scale=scale, **HYPER)
        else:
            ops.adamw8_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_scales"], s["exp_avg_sqs"], s["exp_avg_sq_scales"],
                            step=s["step"], seed=s["seed"], grad_scale=scale, **HYPER)
            ops.adamw8_moments(s["exp_avgs"], s["exp_avg_scales"], s["exp_avg_sqs"], s["exp_avg_sq_scales"], out=s["out"])
    else:
        if case["op"] == "norm":
            return _plain_norm(s["grads"], MAX_NORM)
        norm, scale = _plain_norm(s["grads"], MAX_NORM) if case["clip"] else (None, s["grad_scale"])
        if case["op"] == "adamw":
            [_plain_adamw(*x, scale, s["step"]) for x in zip(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"])]
        else:
            [_plain_adamw8(i, *x, scale, s["step"], s["seed"])
             for i, x in enumerate(zip(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_scales"], s["exp_avg_sqs"],
                                       s["exp_avg_sq_scales"], *s["out"]))]
    return {"params": s["flat_params"], "exp_avg": s["flat_m"], "exp_avg_sq": s["flat_v"], "norm": norm}


# --- 64 bits ----------------------------------------------------------------

def exact(case, seed):
    """The definition in float64.  The moments of adamw8 after their rounding
    have no value there: next to a border of the rounding the float32 average
    decides, so they are None."""
    s = prepare(case, seed)
    norm = torch.zeros((), dtype=torch.float64, device="cuda")
    for g in s["grads"]:
        norm = norm + torch.linalg.vector_norm(g.reshape(-1).to(torch.float64)) ** 2
    norm = norm ** 0.5
    clip = min(1.0, MAX_NORM / (float(norm) + 1e-6))
    if case["op"] == "norm":
        return norm, clip
    c = clip if case["clip"] else float(s["grad_scale"])
    (b1, b2), lr, t = HYPER["betas"], HYPER["lr"], case["step"]
    big = {k: f.to(torch.float64) for k, f in s["flat_params"].items()}
    flat = {k: f.data_ptr() for k, f in s["flat_params"].items()}
    kinds = [k for _, k in _shapes(case)]
    eight = case["op"] == "adamw8"
    out_m, out_v = (None, None) if eight else (s["flat_m"].to(torch.float64), s["flat_v"].to(torch.float64))
    for i, (p, g) in enumerate(zip(s["params"], s["grads"])):
        n, k = p.numel(), kinds[i]
        if eight:
            m0, v0 = (_exact_moment(s[x + "s"][i], s[x + "_scales"][i], x == "exp_avg") for x in ("exp_avg", "exp_avg_sq"))
        else:
            m0, v0 = s["exp_avgs"][i].reshape(-1).double(), s["exp_avg_sqs"][i].reshape(-1).double()
        x = g.reshape(-1).double() * c
        m1 = m0 + (x - m0) * (1.0 - b1)
        v1 = v0 + (x ** 2 - v0) * (1.0 - b2)
        old = p.reshape(-1).double()
        change = (m1 / (1.0 - b1 ** t)) / ((v1 / (1.0 - b2 ** t)) ** 0.5 + HYPER["eps"])
        at = (p.data_ptr() - flat[k]) // BYTES[k]
        big[k][at:at + n] = old - lr * HYPER["weight_decay"] * old - lr * change
        if not eight:
            at = s["exp_avgs"][i].storage_offset()
            out_m[at:at + n], out_v[at:at + n] = m1, v1
    return {"params": big, "exp_avg": out_m, "exp_avg_sq": out_v, "norm": norm if case["clip"] else None}


def _exact_moment(codes, scale_bytes, signed):
    """The value of every code from a table of all 256, times its block's power of two."""
    table = []
    for c in range(256):
        size = c & 127 if signed else c
        top = 15 if signed else 31
        value = (size & 7) / 8 * 2.0 ** (1 - top) if size < 8 else (1 + (size & 7) / 8) * 2.0 ** ((size >> 3) - top)
        table.append(-value if signed and c > 127 else value)
    table = torch.tensor(table, dtype=torch.float64, device=codes.device)
    unit = 2.0 ** (scale_bytes.double() - 127)
    return table[codes.reshape(-1).long()] * unit.repeat_interleave(BLOCK)[:codes.numel()]
