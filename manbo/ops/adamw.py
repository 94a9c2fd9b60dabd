"""AdamW over many tensors at once, on the B200 kernels.

``grad_norm`` is the global 2-norm of a list of gradients with its clip factor,
both left on the device; ``adamw_step`` moves a list of parameters, several
hundred a launch, ``adamw8_step`` does so with moments of one byte an element, and
``adamw8_moments`` gives the values those bytes stand for.  The reference has
none of them: its optimisers are Adan (``adan_step_from_grad_tilelang``) and
torch's Adam, one parameter at a time, with the clip factor read on the host.

Tensors are float32, bfloat16 or float16 CUDA tensors of one device, mixed
freely; each is non-overlapping and dense in any dimension order.  A gradient
has its parameter's type; one with other strides is copied first.  No tensor
that is written may share memory with another one of the call.  All work is
enqueued on the current stream and nothing is read back, so the calls can be
captured in CUDA graphs.
"""
from __future__ import annotations

from typing import List, Sequence, Tuple

import torch

from repo_b200 import _ext

ADAMW8_BLOCK = 256  # elements, in storage order, that share a scale byte


def grad_norm(grads: Sequence[torch.Tensor], *, max_norm: float = 0.0,
              eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(norm, scale) of a list of gradients, two 0-dim float32 device tensors:
    norm is the 2-norm over all of them, summed in double, and scale is
    min(1, max_norm / (norm + eps)), or 1 where max_norm is 0."""
    return _ext.load().grad_norm(grads, max_norm, eps)


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor],
               exp_avgs: Sequence[torch.Tensor], exp_avg_sqs: Sequence[torch.Tensor], *, step,
               lr=1e-3, betas: tuple = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, grad_scale: torch.Tensor | None = None) -> None:
    """One AdamW step in place, several hundred tensors a launch.

    With g' = grad_scale g: m = b1 m + (1 - b1) g', v = b2 v + (1 - b2) g'^2,
    p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps).
    The moments are float32 in the parameter's layout.  ``step`` is t (an int
    from 1) or an int64 device counter, which the call advances and then uses (an
    empty list moves nothing and counts nothing);
    ``lr`` a float or a float32 device scalar; ``grad_scale`` a float32 device
    scalar such as ``grad_norm`` returns.  A 16-bit parameter is rounded to the
    nearest value once, at the end.
    """
    _ext.load().adamw_step(params, grads, exp_avgs, exp_avg_sqs,
                           [(len(params), lr, betas[0], betas[1], eps, weight_decay, step)],
                           grad_scale)


def adamw8_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor],
                exp_avgs: Sequence[torch.Tensor], exp_avg_scales: Sequence[torch.Tensor],
                exp_avg_sqs: Sequence[torch.Tensor], exp_avg_sq_scales: Sequence[torch.Tensor], *,
                step, lr=1e-3, betas: tuple = (0.9, 0.999), eps: float = 1e-8,
                weight_decay: float = 1e-2, grad_scale: torch.Tensor | None = None,
                seed: int = 0) -> None:
    """``adamw_step`` with moments held as uint8 codes in the parameter's layout
    and one uint8 scale for each started block of 256 elements (see
    ``adamw8_state``).

    A scale E stands for 2^(E - 127).  A code of m is a sign, 4 exponent and 3
    fraction bits, one of v 5 exponent and 3 fraction bits, both with gradual
    underflow, so a moment keeps 3 to 4 significant bits down to 2^-14 (m) or
    2^-30 (v) of its block's largest.  They are rounded stochastically, by a
    hash of ``seed``, the step, the tensor's place in the list and the element,
    so an average moves by less than a code's width without being lost, and a
    call is reproducible.  The step itself uses the moments before rounding, the
    hardware's approximate square root and reciprocal (2^-22 each), and 2^-60, the
    root of the smallest v, for a smaller ``eps``.  A block with a moment that is
    not finite (or above 1.5e38) turns NaN.
    """
    _ext.load().adamw8_step(params, grads, exp_avgs, exp_avg_scales, exp_avg_sqs,
                            exp_avg_sq_scales,
                            [(len(params), lr, betas[0], betas[1], eps, weight_decay, step)],
                            seed & 0xFFFFFFFF, grad_scale)


def adamw8_state(param: torch.Tensor) -> Tuple[torch.Tensor, ...]:
    """Zero 8-bit moments of a parameter: (exp_avg, exp_avg_scales, exp_avg_sq,
    exp_avg_sq_scales)."""
    blocks = -(-param.numel() // ADAMW8_BLOCK)

    def codes():
        return torch.zeros_like(param, dtype=torch.uint8, memory_format=torch.preserve_format)

    def scales():
        return torch.zeros(blocks, dtype=torch.uint8, device=param.device)
    return codes(), scales(), codes(), scales()


def adamw8_moments(exp_avgs: Sequence[torch.Tensor], exp_avg_scales: Sequence[torch.Tensor],
                   exp_avg_sqs: Sequence[torch.Tensor],
                   exp_avg_sq_scales: Sequence[torch.Tensor], *,
                   out=None) -> Tuple[List[torch.Tensor], List[torch.Tensor]]:
    """The values of 8-bit moments as float32 tensors in the codes' layout, as
    two lists; ``out`` gives the two lists to write into."""
    if out is None:
        out = tuple([torch.empty_like(c, dtype=torch.float32) for c in x]
                    for x in (exp_avgs, exp_avg_sqs))
    _ext.load().adamw8_moments(exp_avgs, exp_avg_scales, exp_avg_sqs, exp_avg_sq_scales, out[0],
                               out[1])
    return out


__all__ = ["ADAMW8_BLOCK", "grad_norm", "adamw_step", "adamw8_step", "adamw8_state",
           "adamw8_moments"]
