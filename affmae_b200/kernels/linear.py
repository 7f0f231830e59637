"""Matrix product with bias, activation and residual in its epilogue.

* ``fused_linear(x, weight, bias, act, residual)`` computes
  ``act(x W^T + bias) + residual`` in one kernel (tensor cores for fp16, bf16
  and, as three bf16 parts, fp32; a streaming kernel for up to 8 rows), with
  its backward;
* ``FusedLinear`` is the ``nn.Linear`` of it, in the autocast dtype under CUDA
  autocast;
* ``linear_e4m3`` is the forward for 8-bit operands with one fp32 scale per
  row (``quantize_e4m3`` makes them, as does ``rms_norm_e4m3``), and
  ``LinearE4M3`` a layer that keeps its weight so.

Sums are fp32.  Everything runs on the current stream; the gradients do not
depend on timing.  In fp32, from 9 rows on, finite operands whose product is
far beyond the type's range may give NaN in the place of an infinity.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _native as nat

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_CODE = nat._DTYPE_CODE


def _act_code(act: str) -> int:
    try:
        return ACTIVATIONS[act]
    except KeyError:
        raise RuntimeError(f"unknown activation {act!r}; expected one of {sorted(ACTIVATIONS)}")


def _check(x, weight, bias, residual):
    """Shapes, devices and the bias's type (refuses in the order a caller would
    want to know).  The accepted case is decided by a few comparisons: a
    one-token call takes as long as its checks."""
    xs, ws, d = x.shape, weight.shape, x.get_device()
    if d >= 0 and len(ws) == 2 and xs and xs[-1] == ws[1] and ws[0] and ws[1] and weight.get_device() == d \
            and (bias is None or (bias.get_device() == d and bias.dim() == 1 and bias.shape[0] == ws[0]
                                  and bias.dtype in _FLOATS)) \
            and (residual is None or (residual.get_device() == d and residual.dim() == len(xs)
                                      and residual.shape[-1] == ws[0] and residual.shape[:-1] == xs[:-1])):
        return
    nat.require_cuda(x, weight, bias, residual)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise RuntimeError(f"linear: input {tuple(x.shape)} does not match weight {tuple(weight.shape)} [out, in]")
    if bias is not None and (tuple(bias.shape) != (weight.shape[0],) or bias.dtype not in _FLOATS):
        raise RuntimeError(f"linear: bias must be a float vector of {weight.shape[0]} values")
    out_shape = (*x.shape[:-1], weight.shape[0])
    if residual is not None and tuple(residual.shape) != out_shape:
        raise RuntimeError(f"linear: residual {tuple(residual.shape)} does not have the output's shape {out_shape}")
    raise RuntimeError("linear: tensors are on different devices")


def _check_operands(x, weight, bias, residual):
    _check(x, weight, bias, residual)
    dt = x.dtype
    if dt not in _FLOATS or weight.dtype != dt:
        raise RuntimeError(f"linear: input ({x.dtype}) and weight ({weight.dtype}) must share one of fp32, fp16, bf16")
    if residual is not None and residual.dtype != dt and residual.dtype != torch.float32:
        raise RuntimeError(f"linear: residual must be {x.dtype} or float32, got {residual.dtype}")


def linear_fwd(x, weight, bias, residual, act: int, save: bool):
    """(out, z): the product and, where `save` asks for them and the output
    does not serve (``linear_saves``), the pre-activation sums, else None.
    x and weight dense."""
    N, K = weight.shape
    M = x.numel() // K
    index = x.get_device()
    dt = _CODE[x.dtype]
    bptr = rptr = zptr = wptr = None
    bdt = wbytes = 0
    if bias is not None:
        if not bias.is_contiguous():
            bias = bias.contiguous()
        bptr, bdt = bias.data_ptr(), _CODE[bias.dtype]
    if residual is None:
        out, rdt = x.new_empty((*x.shape[:-1], N)), dt
    else:
        if not residual.is_contiguous():
            residual = residual.contiguous()
        out, rptr, rdt = torch.empty_like(residual), residual.data_ptr(), _CODE[residual.dtype]
    z = None
    if save and linear_saves(act, residual):
        z = x.new_empty(out.shape, dtype=z_dtype(x.dtype, act))
        zptr = z.data_ptr()
    ws = nat.workspace(index, "affb_linear_fwd_workspace_bytes", x, dt, M, N, K)
    if ws is not None:
        wptr, wbytes = ws.data_ptr(), ws.numel()
    nat.call_on(index, "affb_linear_fwd", x.data_ptr(), weight.data_ptr(), bptr, bdt, rptr, rdt, act, dt, M, N, K,
                out.data_ptr(), rdt, zptr, wptr, wbytes)
    return out, z


def linear_saves(act: int, residual) -> bool:
    """Whether the backward needs the pre-activation sums: not without an
    activation, and the sign of ReLU's output serves as well as theirs."""
    return act != 0 and not (act == ACTIVATIONS["relu"] and residual is None)


def z_dtype(dtype: torch.dtype, act: int) -> torch.dtype:
    """Type of the pre-activation sums kept for the backward: fp16 instead of
    bf16 for GELU and SiLU, whose gradients want their absolute accuracy."""
    return torch.float16 if dtype == torch.bfloat16 and act >= ACTIVATIONS["gelu"] else dtype


def linear_bwd(dout, z, x, weight, act: int, need_x: bool, need_w: bool, bias_dtype):
    """(dx, dw, db), None where not needed (`bias_dtype` None: no db).  dout,
    x and weight dense; z as saved (the output itself for ReLU without a
    residual)."""
    N, K = weight.shape
    M = x.numel() // K
    index = x.get_device()
    dx = torch.empty_like(x) if need_x else None
    dw = torch.empty_like(weight) if need_w else None
    db = x.new_empty(N, dtype=bias_dtype) if bias_dtype is not None else None
    if need_x or need_w or db is not None:
        dt = nat.dcode(x)
        ws = nat.workspace(index, "affb_linear_bwd_workspace_bytes", x, dt, M, N, K)
        nat.call_on(index, "affb_linear_bwd", nat.ptr(dout), nat.dcode(dout), nat.ptr(z), nat.ptr(x), nat.ptr(weight), act,
                    dt, M, N, K, nat.ptr(dx), nat.ptr(dw), nat.ptr(db), nat.dcode(db) if db is not None else 0,
                    nat.ptr(ws), ws.numel() if ws is not None else 0)
    return dx, dw, db


class FusedLinearFunction(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        save = any(ctx.needs_input_grad[:3])
        xc, wc = nat.dense(x), nat.dense(weight)
        out, z = linear_fwd(xc, wc, bias, residual, act, save)
        if save:
            ctx.save_for_backward(xc, wc, z if linear_saves(act, residual) else out if act else None)
            ctx.meta = (act, bias.dtype if bias is not None else None)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        dx = dw = db = None
        if need_x or need_w or need_b:
            xc, wc, z = ctx.saved_tensors
            act, bdt = ctx.meta
            dx, dw, db = linear_bwd(nat.dense(dout), z, xc, wc, act, need_x, need_w, bdt if need_b else None)
        return dx, dw, db, dout if need_r else None, None


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, act: str = "none",
                 residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``.

    x [..., K] and weight [N, K] in one of fp32 / fp16 / bf16; bias [N] of any
    of these; residual [..., N] in x's dtype or fp32.  The output has the
    residual's dtype, else x's.  act: "none", "relu", "gelu" (exact) or
    "silu".  Differentiable once in x, weight, bias and residual."""
    code = ACTIVATIONS[act] if act in ACTIVATIONS else _act_code(act)
    _check_operands(x, weight, bias, residual)
    if not nat.differentiates(x, weight, bias, residual):
        return linear_fwd(nat.dense(x), nat.dense(weight), bias, residual, code, False)[0]
    return FusedLinearFunction.apply(x, weight, bias, residual, code)


class FusedLinear(nn.Linear):
    """nn.Linear with an activation and a residual in the kernel's epilogue.
    Under CUDA autocast the operands are in the autocast dtype; a residual
    keeps its own dtype when that is fp32."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, act: str = "none", device=None,
                 dtype=None):
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        _act_code(act)
        self.act = act

    def forward(self, x, residual=None):
        w, b = self.weight, self.bias
        if torch.is_autocast_enabled("cuda"):
            dt = torch.get_autocast_dtype("cuda")
            x, w = x.to(dt), w.to(dt)
            if residual is not None and residual.dtype not in (dt, torch.float32):
                residual = residual.to(dt)
        return fused_linear(x, w, b, self.act, residual)


# ----------------------------------------------------------- 8-bit operands --

def quantize_e4m3(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of x [..., C] as e4m3 values and the fp32 scale [...] of each row:
    x ~ q * scale, scale = max|row| / 448 (1 for a zero row).  A gradient
    through it is refused."""
    nat.require_cuda(x)
    if x.dim() < 1 or x.shape[-1] < 1 or x.dtype not in _FLOATS:
        raise RuntimeError("quantize_e4m3: needs fp32, fp16 or bf16 rows of at least one value")
    if nat.differentiates(x):
        return nat.forward_only("quantize_e4m3", lambda: _quantize(x), x)
    return _quantize(x)


def _quantize(x):
    xc = nat.dense(x.detach())
    C = x.shape[-1]
    q = torch.empty(x.shape, device=x.device, dtype=torch.float8_e4m3fn)
    scale = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    nat.call_on(x.get_device(), "affb_quantize_e4m3", nat.ptr(xc), nat.dcode(xc), xc.numel() // C, C, nat.ptr(q),
                nat.ptr(scale))
    return q, scale


def linear_e4m3(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: torch.Tensor | None = None, act: str = "none", residual: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``act((x * x_scale) @ (weight * weight_scale).T + bias) + residual`` for
    e4m3 x [..., K] and weight [N, K] with fp32 scales per row ([...] and
    [N]); bias fp32; residual of any float dtype.  A gradient through it is
    refused."""
    code = _act_code(act)
    _check(x, weight, bias, residual)
    if x.dtype != torch.float8_e4m3fn or weight.dtype != torch.float8_e4m3fn:
        raise RuntimeError("linear_e4m3: input and weight must be float8_e4m3fn")
    if out_dtype not in _FLOATS or (residual is not None and residual.dtype not in _FLOATS):
        raise RuntimeError("linear_e4m3: output and residual must be fp32, fp16 or bf16")
    index = x.get_device()
    if x_scale.shape != x.shape[:-1] or weight_scale.shape != weight.shape[:1]:
        raise RuntimeError("linear_e4m3: scales must have one value per row")
    if x_scale.get_device() != index or weight_scale.get_device() != index:
        raise RuntimeError("linear_e4m3: scales must be on the operands' device")
    if nat.differentiates(x, x_scale, weight, weight_scale, bias, residual):
        return nat.forward_only("linear_e4m3",
                                lambda: _linear_e4m3(x, x_scale, weight, weight_scale, bias, code, residual, out_dtype),
                                x, x_scale, weight, weight_scale, bias, residual)
    return _linear_e4m3(x, x_scale, weight, weight_scale, bias, code, residual, out_dtype)


def _linear_e4m3(x, x_scale, weight, weight_scale, bias, code, residual, out_dtype):
    N, K = weight.shape
    index = x.get_device()
    M = x.numel() // K
    x, weight = nat.dense(x), nat.dense(weight)
    x_scale, weight_scale = _f32(x_scale), _f32(weight_scale)
    bptr = rptr = wptr = None
    rdt = wbytes = 0
    if bias is not None:
        bias = _f32(bias)
        bptr = bias.data_ptr()
    if residual is not None:
        residual = residual if residual.is_contiguous() else residual.contiguous()
        rptr, rdt = residual.data_ptr(), _CODE[residual.dtype]
    out = x.new_empty((*x.shape[:-1], N), dtype=out_dtype)
    ws = nat.workspace(index, "affb_linear_e4m3_workspace_bytes", x, M, N, K)
    if ws is not None:
        wptr, wbytes = ws.data_ptr(), ws.numel()
    nat.call_on(index, "affb_linear_e4m3", x.data_ptr(), x_scale.data_ptr(), weight.data_ptr(), weight_scale.data_ptr(),
                bptr, rptr, rdt, code, M, N, K, out.data_ptr(), _CODE[out_dtype], wptr, wbytes)
    return out


def _f32(t):
    """`t` as a dense fp32 vector (itself where it is one)."""
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.to(torch.float32).contiguous()


class LinearE4M3(nn.Module):
    """A trained Linear kept as e4m3 rows for inference (``from_linear``);
    forward takes the e4m3 rows and scales that ``rms_norm_e4m3`` writes."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None, act: str = "none"):
        super().__init__()
        _act_code(act)
        q, scale = quantize_e4m3(weight.detach())
        self.act = act
        self.register_buffer("weight", q)
        self.register_buffer("weight_scale", scale)
        self.register_buffer("bias", bias.detach().float() if bias is not None else None)

    @classmethod
    def from_linear(cls, linear: nn.Linear, act: str | None = None) -> "LinearE4M3":
        return cls(linear.weight, linear.bias, act if act is not None else getattr(linear, "act", "none"))

    def forward(self, q, q_scale, residual=None, out_dtype=torch.bfloat16):
        return linear_e4m3(q, q_scale, self.weight, self.weight_scale, self.bias, self.act, residual, out_dtype)


def linear_status() -> bool:
    """True unless a product or norm on the current device gave up a bounded wait
    (which leaves its output incomplete) that no call has reported yet: the
    next product or norm called after that raises RuntimeError, once.  Waits
    for the device."""
    import ctypes
    failed = ctypes.c_int(0)
    nat.call("affb_linear_status", ctypes.addressof(failed))
    return failed.value == 0
