"""The hot-path operators registered with the PyTorch dispatcher (namespace
``affb200``), on top of the same C ABI the ``kernels`` package calls.

The reference's operators are plain Python functions around Triton launches,
invisible to the dispatcher.  Registering them as custom ops gives every
operator a schema (``torch.ops.affb200.<name>``), a fake (meta) implementation
for shape propagation under FakeTensor / ``torch.compile`` tracing, and, for
the differentiable ones, an autograd formula that calls the backward op:

  knn                     knn(query, ref, k) -> int64 [B,M,k]  (src/layers/kernels/knn.py:1615)
  nbhd_attn_fwd / _bwd    FlashLocalAttentionFunction (local_attn.py:843-936)
  weighted_features_fwd / _bwd
                          WeightedFeaturesFunction (weighted_features.py:401-429)
  deform_cross_fwd / _bwd FusedKNNDeformCrossAttnFunction (fused_deform_attn.py:4020-4056)

Optional tensors are passed as ``None``; optional gradients come back as
empty tensors (a custom op returns tensors only).
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.library import custom_op

from . import _native as _nat
from .kernels import bucket_bias as _bb
from .kernels import fused_deform_attn as _fd
from .kernels import knn as _knn
from .kernels import linear as _li
from .kernels import local_attn as _la
from .kernels import rms_norm as _rn
from .kernels import weighted_features as _wf

_EMPTY = (0,)


def _none_if_empty(t: Optional[Tensor]) -> Optional[Tensor]:
    return None if t is None or t.numel() == 0 else t


# ------------------------------------------------------------------- KNN --
@custom_op("affb200::knn", mutates_args=())
def knn(query: Tensor, ref: Tensor, k: int) -> Tensor:
    D = query.shape[-1]
    _knn._check(query, ref, k, D)
    return _knn._knn_int64(query, ref, k, D)


@knn.register_fake
def _(query, ref, k):
    return query.new_empty((query.shape[0], query.shape[1], k), dtype=torch.int64)


# ------------------------------------------------ neighbourhood attention --
@custom_op("affb200::nbhd_attn_fwd", mutates_args=())
def nbhd_attn_fwd(q: Tensor, k: Tensor, v: Tensor, member_idx: Tensor, bias: Optional[Tensor],
                  mask: Optional[Tensor], blank_k: Optional[Tensor], blank_v: Optional[Tensor],
                  scale: float) -> tuple[Tensor, Tensor]:
    return _la.launch_flash_nbhood_attn_fwd(q, k, v, member_idx, scale, bias=bias, mask=mask, blank_k=blank_k,
                                            blank_v=blank_v)


@nbhd_attn_fwd.register_fake
def _(q, k, v, member_idx, bias, mask, blank_k, blank_v, scale):
    B, H, N, _ = q.shape
    return torch.empty_like(q), q.new_empty((B, H, N), dtype=torch.float32)


@custom_op("affb200::nbhd_attn_bwd", mutates_args=())
def nbhd_attn_bwd(q: Tensor, k: Tensor, v: Tensor, member_idx: Tensor, scale: float, o: Tensor, lse: Tensor,
                  dout: Tensor, bias: Optional[Tensor], mask: Optional[Tensor], blank_k: Optional[Tensor],
                  blank_v: Optional[Tensor]) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    dq, dk, dv, dbias, dbk, dbv = _la.launch_flash_nbhood_attn_bwd(
        q, k, v, member_idx, scale, o, lse, dout, bias=bias, mask=mask, blank_k=blank_k, blank_v=blank_v)
    e = q.new_empty(_EMPTY)
    return dq, dk, dv, (dbias if dbias is not None else e), (dbk if dbk is not None else e), \
        (dbv if dbv is not None else e)


@nbhd_attn_bwd.register_fake
def _(q, k, v, member_idx, scale, o, lse, dout, bias, mask, blank_k, blank_v):
    e = q.new_empty(_EMPTY)
    return (torch.empty_like(q), torch.empty_like(q), torch.empty_like(q),
            torch.empty_like(bias) if bias is not None else e,
            torch.empty_like(blank_k) if blank_k is not None else e,
            torch.empty_like(blank_v) if blank_v is not None else e)


def _attn_setup(ctx, inputs, output):
    q, k, v, member_idx, bias, mask, blank_k, blank_v, scale = inputs
    o, lse = output
    ctx.save_for_backward(q, k, v, member_idx, bias, mask, blank_k, blank_v, o, lse)
    ctx.scale = scale


def _attn_backward(ctx, grad_o, grad_lse):
    q, k, v, member_idx, bias, mask, blank_k, blank_v, o, lse = ctx.saved_tensors
    dq, dk, dv, dbias, dbk, dbv = nbhd_attn_bwd(q, k, v, member_idx, ctx.scale, o, lse, grad_o.contiguous(),
                                                bias, mask, blank_k, blank_v)
    return dq, dk, dv, None, _none_if_empty(dbias), None, _none_if_empty(dbk), _none_if_empty(dbv), None


nbhd_attn_fwd.register_autograd(_attn_backward, setup_context=_attn_setup)


# ------------------------------------------------------ weighted features --
@custom_op("affb200::weighted_features_fwd", mutates_args=())
def weighted_features_fwd(weights: Tensor, feat: Tensor, nbhd_idx: Tensor) -> Tensor:
    return _wf.weighted_features_fwd(weights, feat, nbhd_idx)


@weighted_features_fwd.register_fake
def _(weights, feat, nbhd_idx):
    B, No, _, IC = weights.shape
    return feat.new_empty((B, No, IC, feat.shape[-1]))


@custom_op("affb200::weighted_features_bwd", mutates_args=())
def weighted_features_bwd(dout: Tensor, weights: Tensor, feat: Tensor, nbhd_idx: Tensor) -> tuple[Tensor, Tensor]:
    return _wf.weighted_features_bwd(dout, weights, feat, nbhd_idx)


@weighted_features_bwd.register_fake
def _(dout, weights, feat, nbhd_idx):
    return weights.new_empty(weights.shape, dtype=feat.dtype), torch.empty_like(feat)


def _wf_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _wf_backward(ctx, grad):
    weights, feat, nbhd_idx = ctx.saved_tensors
    dw, dfeat = weighted_features_bwd(grad.contiguous(), weights, feat, nbhd_idx)
    return dw.to(weights.dtype), dfeat.to(feat.dtype), None


weighted_features_fwd.register_autograd(_wf_backward, setup_context=_wf_setup)


# ----------------------------------------- fused KNN deformable attention --
@custom_op("affb200::deform_cross_fwd", mutates_args=())
def deform_cross_fwd(query_pos: Tensor, kv_pos: Tensor, offsets: Tensor, attn_weights: Tensor, values: Tensor,
                     power: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    return _fd.fused_knn_deform_cross_attn_forward_save(query_pos, kv_pos, offsets, attn_weights, values, power)


@deform_cross_fwd.register_fake
def _(query_pos, kv_pos, offsets, attn_weights, values, power):
    B, Nq, H, K, _ = offsets.shape
    return (values.new_empty((B, Nq, H, values.shape[-1])),
            offsets.new_empty((B, Nq, H, K, 4), dtype=torch.int32),
            offsets.new_empty((B, Nq, H, K, 4), dtype=torch.float32))


@custom_op("affb200::deform_cross_bwd", mutates_args=())
def deform_cross_bwd(dout: Tensor, query_pos: Tensor, kv_pos: Tensor, offsets: Tensor, attn_weights: Tensor,
                     values: Tensor, power: Tensor, knn_idx: Tensor, knn_d2: Tensor
                     ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    dq, dkv, doff, daw, dval, dpow = _fd.fused_knn_deform_cross_attn_backward(
        dout, query_pos, kv_pos, offsets, attn_weights, values, power, knn_idx, knn_d2)
    return dq, dkv, doff, daw, dval, dpow.reshape(power.shape).to(power.dtype)


@deform_cross_bwd.register_fake
def _(dout, query_pos, kv_pos, offsets, attn_weights, values, power, knn_idx, knn_d2):
    return (torch.empty_like(query_pos), torch.empty_like(kv_pos), torch.empty_like(offsets),
            torch.empty_like(attn_weights), torch.empty_like(values), torch.empty_like(power))


def _deform_setup(ctx, inputs, output):
    _, knn_idx, knn_d2 = output
    ctx.save_for_backward(*inputs, knn_idx, knn_d2)


def _deform_backward(ctx, grad_out, grad_idx, grad_d2):
    query_pos, kv_pos, offsets, attn_weights, values, power, knn_idx, knn_d2 = ctx.saved_tensors
    return deform_cross_bwd(grad_out.contiguous(), query_pos, kv_pos, offsets, attn_weights, values, power,
                            knn_idx, knn_d2)


deform_cross_fwd.register_autograd(_deform_backward, setup_context=_deform_setup)


# --------------------------------------------------------- matrix product --
@custom_op("affb200::linear_fwd", mutates_args=())
def linear_fwd(x: Tensor, weight: Tensor, bias: Optional[Tensor], act: str, residual: Optional[Tensor],
               save: bool = True) -> tuple[Tensor, Tensor]:
    """(out, z): z holds the pre-activation sums, empty where the backward needs none, or without `save`
    (inference), which saves their writing."""
    code = _li._act_code(act)
    _li._check_operands(x, weight, bias, residual)
    _nat.refuse_tangents("affb200::linear_fwd", x, weight, bias, residual)
    out, z = _li.linear_fwd(_nat.dense(x), _nat.dense(weight), bias, residual, code, save)
    return out, (z if z is not None else x.new_empty(_EMPTY))


@linear_fwd.register_fake
def _(x, weight, bias, act, residual, save=True):
    shape = (*x.shape[:-1], weight.shape[0])
    saves = save and _li.linear_saves(_li._act_code(act), residual)
    return (x.new_empty(shape, dtype=x.dtype if residual is None else residual.dtype),
            x.new_empty(shape if saves else _EMPTY,
                        dtype=_li.z_dtype(x.dtype, _li._act_code(act)) if saves else x.dtype))


@custom_op("affb200::linear_bwd", mutates_args=())
def linear_bwd(dout: Tensor, z: Tensor, x: Tensor, weight: Tensor, bias: Optional[Tensor], act: str,
               need_x: bool = True, need_w: bool = True) -> tuple[Tensor, Tensor, Tensor]:
    """(dx, dweight, dbias), empty where not needed (dbias: without `bias`)."""
    dx, dw, db = _li.linear_bwd(_nat.dense(dout), _none_if_empty(z), _nat.dense(x), _nat.dense(weight),
                                _li._act_code(act), need_x, need_w, bias.dtype if bias is not None else None)
    return tuple(t if t is not None else x.new_empty(_EMPTY) for t in (dx, dw, db))


@linear_bwd.register_fake
def _(dout, z, x, weight, bias, act, need_x=True, need_w=True):
    return (x.new_empty(x.shape if need_x else _EMPTY), weight.new_empty(weight.shape if need_w else _EMPTY),
            bias.new_empty(bias.shape) if bias is not None else x.new_empty(_EMPTY))


def _linear_setup(ctx, inputs, output):
    x, weight, bias, act, residual, save = inputs
    out, z = output
    code = _li._act_code(act)
    ctx.save_for_backward(x, weight, bias, z if _li.linear_saves(code, residual) or not code else out)
    ctx.act, ctx.residual = act, residual is not None
    ctx.lacks_sums = not save and _li.linear_saves(code, residual)
    ctx.set_materialize_grads(False)


def _refuse_gradient(grad, name):
    if grad is not None:
        raise RuntimeError(f"{name} is kept for the backward and has no gradient of its own")


def _linear_backward(ctx, grad_out, grad_z):
    _refuse_gradient(grad_z, "affb200::linear_fwd: z")
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    dx = dw = db = None
    if need_x or need_w or need_b:
        if ctx.lacks_sums:
            raise RuntimeError("affb200::linear_fwd: called without save, it has no gradient")
        x, weight, bias, z = ctx.saved_tensors
        got = linear_bwd(grad_out.contiguous(), z, x, weight, bias if need_b else None, ctx.act, need_x, need_w)
        dx, dw, db = (t if need else None for t, need in zip(got, (need_x, need_w, need_b)))
    return dx, dw, db, None, grad_out if ctx.residual else None, None


linear_fwd.register_autograd(_linear_backward, setup_context=_linear_setup)


@custom_op("affb200::linear_e4m3", mutates_args=())
def linear_e4m3(x: Tensor, x_scale: Tensor, weight: Tensor, weight_scale: Tensor, bias: Optional[Tensor], act: str,
                residual: Optional[Tensor], out_dtype: torch.dtype) -> Tensor:
    _nat.refuse_tangents("affb200::linear_e4m3", x_scale, weight_scale, bias, residual)
    return _li.linear_e4m3(x, x_scale, weight, weight_scale, bias, act, residual, out_dtype)


@linear_e4m3.register_fake
def _(x, x_scale, weight, weight_scale, bias, act, residual, out_dtype):
    return x.new_empty((*x.shape[:-1], weight.shape[0]), dtype=out_dtype)


# ---------------------------------------------------------------- RMS norm --
@custom_op("affb200::rms_norm_fwd", mutates_args=())
def rms_norm_fwd(x: Tensor, weight: Tensor, eps: float, delta: Optional[Tensor], row_scale: Optional[Tensor],
                 out_dtype: torch.dtype) -> tuple[Tensor, Tensor, Tensor]:
    """(s, y, rstd): s is empty without delta."""
    _rn._check(x, weight, delta, row_scale)
    _nat.refuse_tangents("affb200::rms_norm_fwd", x, weight, delta)
    _, _, _, s, rstd, y, _, _ = _rn._launch(x, delta, row_scale, weight, eps, out_dtype, True)
    return (s if s is not None else x.new_empty(_EMPTY)), y, rstd


@rms_norm_fwd.register_fake
def _(x, weight, eps, delta, row_scale, out_dtype):
    return (x.new_empty(x.shape if delta is not None else _EMPTY), x.new_empty(x.shape, dtype=out_dtype),
            x.new_empty((x.numel() // x.shape[-1],), dtype=torch.float32))


@custom_op("affb200::rms_norm_bwd", mutates_args=())
def rms_norm_bwd(dy: Optional[Tensor], ds: Optional[Tensor], s: Tensor, rstd: Tensor, weight: Tensor,
                 row_scale: Optional[Tensor], delta: Optional[Tensor], need_x: bool = True, need_w: bool = True,
                 need_delta: bool = True) -> tuple[Tensor, Tensor, Tensor]:
    """(dx, dweight, ddelta), empty where not needed.  s: the forward's sum in fp32; x itself in 16 bits or without
    delta."""
    dx, dw, dd = _rn.rms_norm_bwd(_nat.dense(dy) if dy is not None else None,
                                  _nat.dense(ds) if ds is not None else None, _nat.dense(s), rstd,
                                  _nat.dense(weight.float()),
                                  row_scale.float().contiguous() if row_scale is not None else None, need_x, need_w,
                                  delta.dtype if delta is not None and need_delta else None,
                                  _nat.dense(delta) if delta is not None and s.dtype != torch.float32 else None)
    return (dx if dx is not None else s.new_empty(_EMPTY),
            dw.to(weight.dtype) if dw is not None else weight.new_empty(_EMPTY),
            dd if dd is not None else s.new_empty(_EMPTY, dtype=delta.dtype if delta is not None else s.dtype))


@rms_norm_bwd.register_fake
def _(dy, ds, s, rstd, weight, row_scale, delta, need_x=True, need_w=True, need_delta=True):
    return s.new_empty(s.shape if need_x else _EMPTY), weight.new_empty(weight.shape if need_w else _EMPTY), \
        (delta.new_empty(delta.shape if need_delta else _EMPTY) if delta is not None else s.new_empty(_EMPTY))


def _rms_setup(ctx, inputs, output):
    x, weight, eps, delta, row_scale, out_dtype = inputs
    s, y, rstd = output
    ctx.save_for_backward(s if delta is not None and x.dtype == torch.float32 else x, rstd, weight, row_scale, delta)
    ctx.set_materialize_grads(False)


def _rms_backward(ctx, grad_s, grad_y, grad_rstd):
    _refuse_gradient(grad_rstd, "affb200::rms_norm_fwd: rstd")
    s, rstd, weight, row_scale, delta = ctx.saved_tensors
    need_x, need_w, _, need_d = ctx.needs_input_grad[:4]
    got = rms_norm_bwd(grad_y, grad_s if delta is not None else None, s, rstd, weight, row_scale, delta, need_x, need_w,
                       need_d)
    dx, dw, dd = (t if need else None for t, need in zip(got, (need_x, need_w, need_d)))
    return dx, dw, None, dd, None, None


rms_norm_fwd.register_autograd(_rms_backward, setup_context=_rms_setup)


@custom_op("affb200::rms_norm_e4m3", mutates_args=())
def rms_norm_e4m3(x: Tensor, weight: Tensor, eps: float, delta: Optional[Tensor], row_scale: Optional[Tensor]
                  ) -> tuple[Tensor, Tensor, Tensor]:
    """(s, q, scale): s is empty without delta."""
    _nat.refuse_tangents("affb200::rms_norm_e4m3", x, weight, delta)
    got = _rn.rms_norm_e4m3(x, weight, eps, delta, row_scale)
    return got if delta is not None else (x.new_empty(_EMPTY), *got)


@rms_norm_e4m3.register_fake
def _(x, weight, eps, delta, row_scale):
    return (x.new_empty(x.shape if delta is not None else _EMPTY),
            x.new_empty(x.shape, dtype=torch.float8_e4m3fn), x.new_empty(x.shape[:-1], dtype=torch.float32))


# ------------------------------------------------------------- bucket bias --
@custom_op("affb200::bucket_bias_fwd", mutates_args=())
def bucket_bias_fwd(table: Tensor, edges: list[int], q_pos: Tensor, k_pos: Tensor, member_idx: Optional[Tensor],
                    one_sided: bool, dtype: torch.dtype) -> Tensor:
    edges = _bb._check(table, edges, q_pos, k_pos, member_idx, one_sided, dtype)
    _nat.refuse_tangents("affb200::bucket_bias_fwd", table)
    return _bb.bucket_bias_fwd(table.contiguous(), edges, _nat.dense(q_pos), _nat.dense(k_pos),
                               _bb._members(member_idx), one_sided, dtype)


@bucket_bias_fwd.register_fake
def _(table, edges, q_pos, k_pos, member_idx, one_sided, dtype):
    M = member_idx.shape[2] if member_idx is not None else k_pos.shape[1]
    return table.new_empty((q_pos.shape[0], table.shape[1], q_pos.shape[1], M), dtype=dtype)


@custom_op("affb200::bucket_bias_bwd", mutates_args=())
def bucket_bias_bwd(dout: Tensor, edges: list[int], q_pos: Tensor, k_pos: Tensor, member_idx: Optional[Tensor],
                    one_sided: bool, dtype: torch.dtype) -> Tensor:
    return _bb.bucket_bias_bwd(_nat.dense(dout), tuple(edges), _nat.dense(q_pos), _nat.dense(k_pos),
                               _bb._members(member_idx), one_sided, dtype)


@bucket_bias_bwd.register_fake
def _(dout, edges, q_pos, k_pos, member_idx, one_sided, dtype):
    return dout.new_empty((_bb.bucket_count(edges, q_pos.shape[2], one_sided), dout.shape[1]), dtype=dtype)


def _bias_setup(ctx, inputs, output):
    table, edges, q_pos, k_pos, member_idx, one_sided, _ = inputs
    ctx.save_for_backward(q_pos, k_pos, member_idx)
    ctx.meta = (edges, one_sided, table.dtype)


def _bias_backward(ctx, grad):
    q_pos, k_pos, member_idx = ctx.saved_tensors
    edges, one_sided, dt = ctx.meta
    return bucket_bias_bwd(grad.contiguous(), edges, q_pos, k_pos, member_idx, one_sided, dt), None, None, None, \
        None, None, None


bucket_bias_fwd.register_autograd(_bias_backward, setup_context=_bias_setup)
