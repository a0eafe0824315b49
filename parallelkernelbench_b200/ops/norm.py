"""RMSNorm (csrc/kernels/norm.cu) and layer norm (csrc/kernels/layernorm.cu) kernels.

``sum_rmsnorm`` is the consumer end of a reduce-scatter: it adds the per-source partial buffers in
a fixed order, scales, and normalises, so the reduced tensor is never stored un-normalised
(reference behaviour: reference/45_reducescatter_fused_rmsnorm.py:23-29,
reference/18_tp_rms_norm.py:9-19).
"""
from __future__ import annotations

import functools

import torch

from .. import _native as nv


def rmsnorm(x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
    if x.dtype != torch.bfloat16 or gamma.dtype != torch.bfloat16:
        raise TypeError("rmsnorm expects bf16 input and gain")
    cols = x.shape[-1]
    x2 = x.contiguous().view(-1, cols)
    if out is None:
        out = torch.empty_like(x2)
    nv.check(nv.cuda_lib().pkb_rmsnorm_bf16(nv.ptr(x2), nv.ptr(gamma), nv.ptr(out), x2.shape[0], cols,
                                            nv.c_float(eps), nv.current_stream()), "pkb_rmsnorm_bf16")
    nv.count_launch()
    return out.view(x.shape)


def sum_rmsnorm(parts: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-6, scale: float = 1.0,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """``parts`` is ``[nsrc, rows, cols]`` (bf16 or fp32, contiguous); returns bf16 ``[rows, cols]``."""
    if parts.dim() != 3 or not parts.is_contiguous():
        raise ValueError("parts must be a contiguous [nsrc, rows, cols] tensor")
    nsrc, rows, cols = parts.shape
    if out is None:
        out = torch.empty((rows, cols), dtype=torch.bfloat16, device=parts.device)
    nv.check(nv.cuda_lib().pkb_sum_rmsnorm(nv.ptr(parts), nv.c_ll(rows * cols), nsrc,
                                           1 if parts.dtype == torch.float32 else 0, nv.ptr(gamma), nv.ptr(out),
                                           rows, cols, nv.c_float(scale), nv.c_float(eps), nv.current_stream()),
             "pkb_sum_rmsnorm")
    nv.count_launch()
    return out


# ------------------------------------------------------------------------------------------------ layer norm
_P, _I, _LL, _F = nv.c_void_p, nv.c_int, nv.c_ll, nv.c_float
_LN_FWD = [_P, _LL, _P, _P, _I, _P, _P, _P, _LL, _I, _F, _I, _P]
_LN_BWD = [_P, _LL, _P, _LL, _P, _I, _P, _P, _P, _P, _P, _P, _LL, _I, _I, _P]
_DT = {torch.bfloat16: 0, torch.float32: 1}
_MAX_COLS = 1 << 30       # the kernels count columns in 32 bits


def _rows_of(t: torch.Tensor, cols: int) -> torch.Tensor:
    """``[rows, cols]`` with unit inner stride; a view wherever the strides allow one (rows may lie apart, repeat or overlap)."""
    t = t.reshape(-1, cols) if t.dim() != 2 else t
    return t if t.stride(1) == 1 or cols == 1 else t.contiguous()


def _ln_param(name: str, p: torch.Tensor, x: torch.Tensor, cols: int) -> None:
    if p.dtype not in _DT or p.numel() != cols or not p.is_contiguous():
        raise ValueError(f"{name} must be contiguous bf16 or fp32 with {cols} values")
    if p.get_device() != x.get_device():
        raise ValueError(f"{name} is on {p.device}, not on {x.device}")


def _ln_check(x: torch.Tensor, gamma, beta=None) -> int:
    if x.dtype not in _DT:
        raise TypeError(f"layer norm takes bf16 or fp32 rows, got {x.dtype}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _MAX_COLS:
        raise ValueError("layer norm needs at least one column, and at most 2^30")
    cols = x.shape[-1]
    if gamma is not None:
        _ln_param("gamma", gamma, x, cols)
    if beta is not None:
        _ln_param("beta", beta, x, cols)
        if gamma is not None and beta.dtype != gamma.dtype:
            raise TypeError("gamma and beta must have the same dtype")
    return cols


def _ln_forward(x, gamma, beta, eps, stats: bool):
    cols = _ln_check(x, gamma, beta)
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    if not x.is_cuda:
        raise ValueError("expected CUDA tensors")
    x2 = _rows_of(x, cols)
    rows = x2.shape[0]
    y = nv.contiguous_like(x)
    mean = rstd = None
    if stats:
        mean = x.new_empty(rows, dtype=torch.float32) if x.dim() == 2 else x.new_empty(x.shape[:-1], dtype=torch.float32)
        rstd = torch.empty_like(mean)
    if rows:
        param = gamma if gamma is not None else beta
        nv.launch("pkb_layer_norm_fwd", _LN_FWD, x, x2.data_ptr(), x2.stride(0), 0 if gamma is None else gamma.data_ptr(),
                  0 if beta is None else beta.data_ptr(), 0 if param is None else _DT[param.dtype], y.data_ptr(),
                  mean.data_ptr() if stats else 0, rstd.data_ptr() if stats else 0, rows, cols, eps, _DT[x.dtype])
    return y, mean, rstd


def layer_norm(x: torch.Tensor, gamma: torch.Tensor | None = None, beta: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) * rsqrt(var + eps) * gamma + beta`` over the last dimension. ``x`` is bf16 or fp32 ``[..., cols]`` (any row pitch,
    any width), ``gamma`` and ``beta`` bf16 or fp32 ``[cols]`` or None (1 and 0); fp32 inside, one rounding to the type of ``x``. A constant row
    comes out as ``beta``, as long as its sum fits fp32."""
    return _ln_forward(x, gamma, beta, eps, False)[0]


def layer_norm_fwd(x: torch.Tensor, gamma: torch.Tensor | None = None, beta: torch.Tensor | None = None, eps: float = 1e-5):
    """:func:`layer_norm` with what its backward needs: ``(y, mean, rstd)``, the statistics fp32 of shape ``x.shape[:-1]``."""
    return _ln_forward(x, gamma, beta, eps, True)


@functools.lru_cache(maxsize=256)
def _ln_plan(rows: int, cols: int, dtype: int, device: int) -> tuple[int, int, int]:
    """Blocks that write partial sums (at most), and launches where everything lies on 16 bytes and where it does not."""
    launches = nv.bound("pkb_layer_norm_bwd_launches", [_LL, _I, _I, _I, _I])
    with torch.cuda.device(device):
        return (nv.bound("pkb_layer_norm_bwd_partials", [_LL, _I, _I])(rows, cols, dtype), launches(rows, cols, dtype, 1, 0),
                launches(rows, cols, dtype, 0, 0))


def _on_16_bytes(gamma, dx, *rows) -> bool:
    """Base, pitch and width of ``rows``, and the addresses of ``gamma`` and ``dx``, as the backward's 16-byte accesses want them."""
    size = dx.element_size()
    bits = dx.data_ptr() | (0 if gamma is None else gamma.data_ptr()) | rows[0].shape[1] * size
    for t in rows:
        bits |= t.data_ptr() | t.stride(0) * size
    return bits % 16 == 0


def layer_norm_bwd(x: torch.Tensor, gamma: torch.Tensor | None, dy: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor):
    """Backward of :func:`layer_norm_fwd`: ``(dx, dgamma, dbeta)``, ``dx`` in the type of ``x``, the weight gradients fp32 ``[cols]``
    (what a gain of 1 or a bias of 0 would get where there is none). Sums run in a fixed order: the same inputs give the same bits."""
    cols = _ln_check(x, gamma)
    if dy.dtype != x.dtype or dy.shape != x.shape:
        raise ValueError("dy must have the shape and dtype of x")
    for name, s in (("mean", mean), ("rstd", rstd)):
        if s.dtype != torch.float32 or s.numel() * cols != x.numel() or not s.is_contiguous():
            raise ValueError(f"{name} must be contiguous fp32 with one value per row")
    nv.same_cuda_device(x, dy=dy, mean=mean, rstd=rstd)
    x2, dy2 = _rows_of(x, cols), _rows_of(dy, cols)
    rows = x2.shape[0]
    dx = nv.contiguous_like(x)
    if not rows:
        return dx, x.new_zeros(cols, dtype=torch.float32), x.new_zeros(cols, dtype=torch.float32)
    dgamma = torch.empty_like(gamma) if gamma is not None and gamma.dtype == torch.float32 and gamma.dim() == 1 else x.new_empty(cols, dtype=torch.float32)
    dbeta = torch.empty_like(dgamma)
    blocks, launches, launches_off = _ln_plan(rows, cols, _DT[x.dtype], x.get_device())
    if launches != launches_off and not _on_16_bytes(gamma, dx, x2, dy2):
        launches = launches_off
    part = x.new_empty(blocks * 2 * cols, dtype=torch.float32) if blocks else None
    nv.launch("pkb_layer_norm_bwd", _LN_BWD, x, x2.data_ptr(), x2.stride(0), dy2.data_ptr(), dy2.stride(0), 0 if gamma is None else gamma.data_ptr(),
              0 if gamma is None else _DT[gamma.dtype], mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), dgamma.data_ptr(), dbeta.data_ptr(),
              part.data_ptr() if blocks else 0, rows, cols, _DT[x.dtype], launches=launches)
    return dx, dgamma, dbeta
