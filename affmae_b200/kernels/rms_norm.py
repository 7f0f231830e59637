"""Root-mean-square norm with the residual's addition, and its 8-bit output.

* ``fused_rms_norm(x, weight, eps, delta, row_scale, out_dtype)``:
  ``s = x + row_scale * delta`` (the residual stream, in x's dtype) and
  ``y = s * rsqrt(mean(s^2) + eps) * weight`` in one pass, with the backward
  in one pass over the gradients of both;
* ``rms_norm_e4m3``: the same with y as e4m3 rows and one fp32 scale per row,
  the operand of ``linear_e4m3`` (forward only);
* ``FusedRMSNorm``: the module.

Statistics are fp32, taken of the sum before it is rounded to x's dtype; the
backward forms a 16-bit stream's sum again from x and delta (in fp32 it reads
the sum).
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _native as nat

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_CODE = nat._DTYPE_CODE


def _check(x, weight, delta, row_scale):
    xs, d = x.shape, x.get_device()
    # the common case in a few comparisons; whatever else is looked at in order below
    if d >= 0 and row_scale is None and xs and xs[-1] and weight.dim() == 1 and weight.shape[0] == xs[-1] \
            and weight.get_device() == d and x.dtype in _FLOATS and weight.dtype in _FLOATS \
            and (delta is None or (delta.get_device() == d and delta.dtype in _FLOATS and delta.shape == xs)):
        return
    nat.require_cuda(x, weight, delta, row_scale)
    if x.dim() < 1 or tuple(weight.shape) != (x.shape[-1],) or x.shape[-1] < 1:
        raise RuntimeError(f"rms_norm: weight {tuple(weight.shape)} does not match the rows of {tuple(x.shape)}")
    for t in (x, weight) + ((delta,) if delta is not None else ()):
        if t.dtype not in _FLOATS:
            raise RuntimeError(f"rms_norm: unsupported dtype {t.dtype}; expected float32, float16 or bfloat16")
    if delta is not None and delta.shape != x.shape:
        raise RuntimeError(f"rms_norm: delta {tuple(delta.shape)} does not have the shape {tuple(x.shape)} of x")
    if row_scale is not None:
        if delta is None:
            raise RuntimeError("rms_norm: row_scale scales delta, which is missing")
        rows = x.numel() // x.shape[-1]
        if row_scale.dim() != 1 or row_scale.numel() < 1 or rows % row_scale.numel():
            raise RuntimeError(f"rms_norm: row_scale [{row_scale.numel()}] does not divide {rows} rows")
    for t in (weight, delta, row_scale):
        if t is not None and t.device != x.device:
            raise RuntimeError("rms_norm: tensors are on different devices")


def _launch(x, delta, row_scale, weight, eps, out_dtype, keep):
    """One forward pass: (x, row_scale, weight as the kernel read them, s, rstd,
    y, q, scale).  out_dtype None writes e4m3 rows and scales; rstd only with
    `keep`, s only with delta."""
    C = x.shape[-1]
    R = x.numel() // C
    xc = nat.dense(x)
    w = nat.dense(weight.detach().float() if weight.requires_grad or weight.dtype != torch.float32 else weight)
    s = rs = rstd = y = q = scale = None
    dptr = sptr = rptr = kptr = yptr = qptr = cptr = None
    ddt = ydt = groups = 0
    if delta is not None:
        delta = nat.dense(delta)
        s = torch.empty_like(xc)
        dptr, ddt, sptr = delta.data_ptr(), _CODE[delta.dtype], s.data_ptr()
    if row_scale is not None:
        rs = row_scale.float().contiguous()
        rptr, groups = rs.data_ptr(), rs.numel()
    if keep:
        rstd = xc.new_empty(R, dtype=torch.float32)
        kptr = rstd.data_ptr()
    if out_dtype is None:
        q = torch.empty_like(xc, dtype=torch.float8_e4m3fn)
        scale = xc.new_empty(x.shape[:-1], dtype=torch.float32)
        qptr, cptr = q.data_ptr(), scale.data_ptr()
    else:
        y = torch.empty_like(xc, dtype=out_dtype)
        yptr, ydt = y.data_ptr(), _CODE[out_dtype]
    nat.call_on(x.get_device(), "affb_rms_norm_fwd", xc.data_ptr(), _CODE[xc.dtype], dptr, ddt, rptr, groups, w.data_ptr(),
                float(eps), R, C, sptr, kptr, yptr, ydt, qptr, cptr)
    return xc, rs, w, s, rstd, y, q, scale


def rms_norm_bwd(dy, ds, s, rstd, weight, row_scale, need_x: bool, need_w: bool, delta_dtype, delta=None):
    """(dx, dw, ddelta), None where not needed (`delta_dtype` None: no
    ddelta); weight, row_scale, dw fp32; dy or ds may be None.  With `delta`,
    s is x and the sum is formed again."""
    C = s.shape[-1]
    R = s.numel() // C
    index = s.get_device()
    dx = torch.empty_like(s) if need_x else None
    dd = torch.empty_like(s, dtype=delta_dtype) if delta_dtype is not None else None
    dw = s.new_empty(C, dtype=torch.float32) if need_w else None
    ws = nat.workspace(index, "affb_rms_norm_bwd_workspace_bytes", s, R, C) if need_w else None
    nat.call_on(index, "affb_rms_norm_bwd", nat.ptr(dy), nat.dcode(dy) if dy is not None else 0, nat.ptr(ds), nat.ptr(s),
                nat.dcode(s), nat.ptr(delta), nat.ptr(rstd), nat.ptr(weight), nat.ptr(row_scale),
                row_scale.numel() if row_scale is not None else 0, R, C, nat.ptr(dx), nat.ptr(dd),
                nat.dcode(dd if dd is not None else delta) if dd is not None or delta is not None else 0, nat.ptr(dw),
                nat.ptr(ws), ws.numel() if ws is not None else 0)
    return dx, dw, dd


class FusedRMSNormFunction(Function):
    @staticmethod
    def forward(ctx, x, weight, delta, row_scale, eps, out_dtype):
        ctx.set_materialize_grads(False)
        keep = any(ctx.needs_input_grad[:3])
        xc, rs, w, s, rstd, y, _, _ = _launch(x, delta, row_scale, weight, eps, out_dtype, keep)
        if keep:
            again = s is not None and x.dtype != torch.float32
            ctx.save_for_backward(xc if s is None or again else s, rstd, w, rs, nat.dense(delta) if again else None)
            ctx.meta = (weight.dtype, delta.dtype if delta is not None else None)
        return y if s is None else (s, y)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        s, rstd, w, rs, delta = ctx.saved_tensors
        wdt, ddt = ctx.meta
        ds, dy = grads if ddt is not None else (None, grads[0])
        need_x, need_w, need_d = ctx.needs_input_grad[:3]
        dx, dw, dd = rms_norm_bwd(nat.dense(dy) if dy is not None else None, nat.dense(ds) if ds is not None else None,
                                  s, rstd, w, rs, need_x, need_w, ddt if need_d else None, delta)
        return dx, dw.to(wdt) if need_w else None, dd, None, None, None


def fused_rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, delta: torch.Tensor | None = None,
                   row_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None):
    """y, or (s, y) when ``delta`` is given: ``s = x + row_scale * delta`` in
    x's dtype and ``y = s * rsqrt(mean(s^2) + eps) * weight`` in ``out_dtype``
    (x's by default).

    x [..., C] and delta of the same shape, each fp32 / fp16 / bf16;
    row_scale [G]: one factor per G-th of the rows (stochastic depth per
    sample), no gradient.  Differentiable once in x, weight and delta."""
    _check(x, weight, delta, row_scale)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in _FLOATS:
        raise RuntimeError(f"rms_norm: unsupported output dtype {out_dtype}")
    if not nat.differentiates(x, weight, delta):
        _, _, _, s, _, y, _, _ = _launch(x, delta, row_scale, weight, eps, out_dtype, False)
        return y if s is None else (s, y)
    return FusedRMSNormFunction.apply(x, weight, delta, row_scale, eps, out_dtype)


def rms_norm_e4m3(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, delta: torch.Tensor | None = None,
                  row_scale: torch.Tensor | None = None):
    """(q, scale), or (s, q, scale) when ``delta`` is given: the norm with its
    output as e4m3 rows, ``y ~ q * scale``, ``scale = max|y| / 448`` of each
    row (1 for a zero row).  A gradient through it, that of s included, is
    refused."""
    _check(x, weight, delta, row_scale)
    if nat.differentiates(x, weight, delta):
        return nat.forward_only("rms_norm_e4m3", lambda: _rms_e4m3(x, weight, eps, delta, row_scale), x, weight, delta)
    return _rms_e4m3(x, weight, eps, delta, row_scale)


def _rms_e4m3(x, weight, eps, delta, row_scale):
    _, _, _, s, _, _, q, scale = _launch(x, delta, row_scale, weight, eps, None, False)
    return (q, scale) if delta is None else (s, q, scale)


class FusedRMSNorm(nn.Module):
    """``forward(x)`` -> y; ``forward(x, delta, row_scale)`` -> (s, y)."""

    def __init__(self, dim: int, eps: float = 1e-6, device=None, dtype=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))

    def forward(self, x, delta=None, row_scale=None, out_dtype=None):
        return fused_rms_norm(x, self.weight, self.eps, delta, row_scale, out_dtype)

    def quantized(self, x, delta=None, row_scale=None):
        """(q, scale) or (s, q, scale): ``rms_norm_e4m3`` with this weight."""
        return rms_norm_e4m3(x, self.weight, self.eps, delta, row_scale)
