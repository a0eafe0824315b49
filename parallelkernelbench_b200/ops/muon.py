"""Orthogonalised updates (kernels: csrc/kernels/muon.cu): Newton-Schulz products on the tensor cores, and the optimiser step around them.

The step stands beside :func:`~parallelkernelbench_b200.ops.elementwise.adam_step`: it is for the matrices of a model (embeddings, heads, gains
and biases keep Adam).
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from .. import _native as nv

_P, _I, _LL, _F, _D = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_double
_ARGS = [_P, _I, _P, _F, _I, _LL, _I, _I, _P, _I, _D, _P, _P, _F, _F, _P, _P, _P]
_DT = {torch.bfloat16: 0, torch.float32: 1}

#: Coefficients (a, b, c) of a step s -> a s + b s^3 + c s^5 that lift small singular values fast and leave them within about 0.7 .. 1.2.
FAST = (3.4445, -4.7750, 2.0315)


@functools.lru_cache(maxsize=64)
def _coefficients(coefficients, steps: int, longer: int):
    """The steps' coefficients as a C array. The products run in fp16: what the singular values (at most 1 at the start), the Gram matrix and
    the polynomial can reach has to stay inside its range. At the other end a matrix of many small singular values has entries of 1 / sqrt(shorter
    side) after the scaling; fp16 holds them to 11 bits down to 2^-14. So that 16384 rows (2^-7) keep these, small singular values, which a step
    multiplies by ``a``, may not shrink below 2^-6 of themselves on the way."""
    per_step = coefficients if isinstance(coefficients[0], tuple) else (coefficients,) * steps
    if len(per_step) != steps or any(len(c) != 3 for c in per_step):
        raise ValueError("coefficients are one (a, b, c) or one per step")
    top = small = 1.0
    k = 2.0 ** round(math.log2(longer) / 2)
    for a, b, c in per_step:
        if not all(math.isfinite(v) for v in (a, b, c)):
            raise ValueError("coefficients must be finite")
        small *= abs(a)
        if small < 2.0 ** -6:
            raise ValueError("coefficients whose linear terms shrink small singular values to less than 1/64 leave the range of fp16")
        inner = abs(b) * top ** 2 + abs(c) * top ** 4
        top = 1.01 * max(abs(a * s + b * s ** 3 + c * s ** 5) for s in (top * i / 512 for i in range(513)))
        if not max(inner, top * top, top * k) <= 3e4:
            raise ValueError("these coefficients can leave the range of fp16")
    flat = [v for c in per_step for v in c]
    return (ctypes.c_float * len(flat))(*flat)


def _check(g, steps, coefficients, eps):
    """The coefficients as a C array (None for empty matrices); refuses what the kernels do not take."""
    if isinstance(coefficients, list) or (len(coefficients) and isinstance(coefficients[0], list)):
        coefficients = tuple(tuple(c) if isinstance(c, list) else c for c in coefficients)
    if not steps >= 1 or not eps >= 0:
        raise ValueError("at least one step, and eps >= 0")
    if not len(coefficients):
        raise ValueError("coefficients are one (a, b, c) or one per step")
    rows, cols = g.shape[-2:]
    if not g.numel():
        return None
    if g.numel() // (rows * cols) > 65535:
        raise ValueError("at most 65535 matrices at once")
    if max(rows, cols) >= 1 << 24:
        raise ValueError("sides of at most 2^24 - 1")
    return _coefficients(coefficients, int(steps), max(rows, cols))


def _launch(g, m, momentum, nesterov, steps, coeff, eps, out, p, decay, scale, p_bf16) -> None:
    rows, cols = g.shape[-2:]
    batch = g.numel() // (rows * cols)
    g = g.contiguous()
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    launches = _I()
    nbytes = nv.bound("pkb_newton_schulz_scratch", [_LL, _I, _I, _I, _P], _LL)(batch, rows, cols, steps, ctypes.addressof(launches))
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=g.device) if nbytes else None
    nv.launch("pkb_newton_schulz", _ARGS, g, g.data_ptr(), _DT[g.dtype], ptr(m), momentum, int(nesterov), batch, rows, cols, coeff, steps, eps, ptr(out),
              ptr(p), decay, scale, ptr(p_bf16), ptr(scratch), launches=launches.value)


def newton_schulz(g: torch.Tensor, *, steps: int = 5, coefficients=FAST, eps: float = 1e-7) -> torch.Tensor:
    """Orthogonalises the matrices ``g`` (bf16 or fp32 ``[..., rows, cols]``, any sides): ``X = g / (|g|_F + eps)``, then ``steps`` times
    ``X <- a X + (b A + c A^2) X`` with ``A = X X^T``. ``coefficients`` is one ``(a, b, c)`` or a sequence of one per step; they must keep the
    singular values within what fp16 products hold (refused otherwise: growth beyond 3e4, and linear terms whose product falls under 1/64).
    Returns bf16 of the same shape (at most 65535 matrices).

    The iterate is held in fp32 and multiplied in fp16 with fp32 sums: against 64 bits five steps are 1.1e-3 to
    2.1e-3 off (2-norm) for noise and 3e-4 to 9e-4 for matrices of few directions, before the rounding to bf16 adds its 1.7e-3. Up to 128 x 4096 the
    polynomial keeps 22 bits (1.1e-3 to 1.6e-3), in larger matrices 11 (1.1e-3 to 2.1e-3, the most where the sides differ most).

    A matrix of zeros stays zero; one with a value that is not finite comes back as NaN, alone. The same call gives the same bits; alone a matrix may
    be split over the GPU in another way than in a batch."""
    if g.dtype not in _DT:
        raise TypeError(f"newton_schulz takes bf16 or fp32, got {g.dtype}")
    if g.dim() < 2:
        raise ValueError("newton_schulz takes matrices [..., rows, cols]")
    coeff = _check(g, steps, coefficients, eps)
    nv.same_cuda_device(g)
    out = g.new_empty(g.shape, dtype=torch.bfloat16)
    if g.numel():
        _launch(g, None, 0.0, False, steps, coeff, eps, out, None, 0.0, 0.0, None)
    return out


def _check_apart(p, m, g, p_bf16) -> None:
    """No byte of what a step writes in place belongs to another of its tensors (all but ``g`` are contiguous)."""
    n, at_p, at_m, at_g = p.numel(), p.data_ptr(), m.data_ptr(), g.data_ptr()
    of_g = (n if g.is_contiguous() else sum((k - 1) * s for k, s in zip(g.shape, g.stride())) + 1) * g.element_size()
    apart = (at_p + 4 * n <= at_m or at_m + 4 * n <= at_p) and (at_p + 4 * n <= at_g or at_g + of_g <= at_p) and (at_m + 4 * n <= at_g or at_g + of_g <= at_m)
    if apart and p_bf16 is not None:
        at = p_bf16.data_ptr()
        apart = all(at + 2 * n <= other or other + size <= at for other, size in ((at_p, 4 * n), (at_m, 4 * n), (at_g, of_g)))
    if not apart:
        raise ValueError("p, m, g and p_bf16 must be different tensors that do not overlap")


def muon_step(p: torch.Tensor, m: torch.Tensor, g: torch.Tensor, *, lr: float, momentum: float = 0.95, nesterov: bool = True,
              weight_decay: float = 0.0, scale: float | None = None, steps: int = 5, coefficients=FAST, eps: float = 1e-7,
              p_bf16: torch.Tensor | None = None) -> None:
    """One step on fp32 matrices ``p [..., rows, cols]`` with the momentum ``m`` (fp32) and the gradient ``g`` (bf16 or fp32), in place::

        m <- momentum * m + g;   u = g + momentum * m (nesterov) or m
        p <- p * (1 - lr * weight_decay) - lr * scale * newton_schulz(u)

    ``scale`` defaults to ``0.2 * sqrt(max(rows, cols))``: an update of about Adam's root mean square, so that its learning rate and decay carry
    over. ``p_bf16`` receives a bf16 copy. Leading dimensions are matrices of their own (the experts of a MoE layer). None of the tensors may overlap
    another. The products' error (:func:`newton_schulz`) enters as ``lr * scale`` times it: a step of 3e-4 moves weights of standard deviation
    0.02 to within 2e-6 to 5e-6 (2-norm) of a computation in 64 bits."""
    for name, t in (("p", p), ("m", m)):
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise TypeError(f"{name} must be contiguous fp32")
    if g.dtype not in _DT:
        raise TypeError(f"g must be bf16 or fp32, got {g.dtype}")
    if p.dim() < 2 or m.shape != p.shape or g.shape != p.shape:
        raise ValueError("p, m and g must be matrices [..., rows, cols] of one shape")
    if p_bf16 is not None and (p_bf16.dtype != torch.bfloat16 or p_bf16.shape != p.shape or not p_bf16.is_contiguous()):
        raise ValueError("p_bf16 must be contiguous bf16 of the shape of p")
    coeff = _check(g, steps, coefficients, eps)
    if p.numel():
        _check_apart(p, m, g, p_bf16)
    nv.same_cuda_device(p, m=m, g=g, p_bf16=p_bf16)
    if not p.numel():
        return
    if scale is None:
        scale = 0.2 * math.sqrt(max(p.shape[-2:]))
    _launch(g, m, momentum, nesterov, steps, coeff, eps, None, p, 1.0 - lr * weight_decay, lr * scale, p_bf16)
