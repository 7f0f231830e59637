"""Learned relative-position bias by buckets.

``bucket_bias(table, edges, q_pos, k_pos, member_idx)`` gives the additive
bias [B, H, Nq, M] of attention (the ``bias`` of
``FlashLocalAttentionFunction``, or a dense attention mask) from a table with
one row per bucket and one column per head, straight from the token positions:
no index array and no table of offsets is formed.  Its backward sums the
gradients of each bucket without atomics whose order could matter.

``edges`` e_1 < e_2 < ... are the distances where a new bucket begins
(``log_edges`` makes the usual ones: single steps, then geometric).  With
c(n) the number of edges <= n, an offset d = round(k_pos - q_pos) along one
axis has the index ``len(edges) + sign(d) c(|d|)``, or, with ``one_sided``
(causal: a key's distance in the past), ``c(max(-d, 0))``.  Two axes combine
as ``index(y) * n + index(x)`` of ``n = bucket_count(edges, 1, one_sided)``.
"""
from __future__ import annotations

import ctypes
import functools

import torch
import torch.nn as nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _native as nat

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_POS = {torch.float32: 0, torch.int32: 1, torch.int64: 2}


def log_edges(count: int, reach: int) -> tuple[int, ...]:
    """`count` ascending distances: 1, 2, ... for the first half, then
    geometric up to `reach`."""
    if count < 1 or reach < 1:
        raise RuntimeError("log_edges: needs count >= 1 and reach >= 1")
    half = (count + 1) // 2
    e = list(range(1, half + 1))
    for j in range(1, count - half + 1):
        e.append(max(e[-1] + 1, round(half * (max(reach, half) / half) ** (j / (count - half)))))
    return tuple(e)


def bucket_count(edges, axes: int = 1, one_sided: bool = False) -> int:
    """Rows of the table."""
    return (len(edges) + 1 if one_sided else 2 * len(edges) + 1) ** axes


def _check_edges(edges) -> tuple[int, ...]:
    edges = tuple(edges)
    if set(map(type, edges)) != {int}:  # tensors, say, whose values may change while they stay the same keys
        return _checked.__wrapped__(edges)
    return _checked(edges)


@functools.lru_cache(maxsize=256)
def _checked(edges) -> tuple[int, ...]:
    if not 1 <= len(edges) <= 64 or any(int(e) != e or not 1 <= e <= 1 << 30 for e in edges) \
            or any(a >= b for a, b in zip(edges, edges[1:])):
        raise RuntimeError("bucket_bias: edges must be 1 to 64 ascending integers in [1, 2^30]")
    return tuple(int(e) for e in edges)


@functools.lru_cache(maxsize=256)
def _edge_array(edges):
    return (ctypes.c_int32 * len(edges))(*edges)


def _check(table, edges, q_pos, k_pos, member_idx, one_sided, dtype) -> tuple[int, ...]:
    edges = _check_edges(edges)
    qs, ks, d, pt = q_pos.shape, k_pos.shape, table.get_device(), q_pos.dtype
    # the common case in a few comparisons; whatever else is looked at in order below
    if d >= 0 and q_pos.get_device() == d and k_pos.get_device() == d and len(qs) == 3 and len(ks) == 3 \
            and (qs[2] == 1 or (qs[2] == 2 and len(edges) <= 32)) and qs[2] == ks[2] and qs[0] == ks[0] and pt in _POS \
            and k_pos.dtype == pt and len(table.shape) == 2 and table.shape[0] == bucket_count(edges, qs[2], one_sided) \
            and table.dtype in _FLOATS and dtype in _FLOATS and member_idx is None:
        return edges
    nat.require_cuda(table, q_pos, k_pos, member_idx)
    if q_pos.dim() != 3 or k_pos.dim() != 3 or q_pos.shape[2] not in (1, 2) or q_pos.shape[2] != k_pos.shape[2] \
            or q_pos.shape[0] != k_pos.shape[0]:
        raise RuntimeError(f"bucket_bias: positions {tuple(q_pos.shape)} and {tuple(k_pos.shape)} are not "
                           "[B, Nq, axes] and [B, Nk, axes] with 1 or 2 axes")
    axes = q_pos.shape[2]
    if axes == 2 and len(edges) > 32:
        raise RuntimeError("bucket_bias: at most 32 edges with two axes")
    if q_pos.dtype not in _POS or k_pos.dtype != q_pos.dtype:
        raise RuntimeError("bucket_bias: positions must share one of float32, int32, int64")
    if table.dim() != 2 or table.shape[0] != bucket_count(edges, axes, one_sided) or table.dtype not in _FLOATS:
        raise RuntimeError(f"bucket_bias: table must be a float array of {bucket_count(edges, axes, one_sided)} rows, "
                           f"got {tuple(table.shape)} {table.dtype}")
    if member_idx is not None and (member_idx.dim() != 3 or member_idx.shape[:2] != q_pos.shape[:2]
                                   or member_idx.dtype not in (torch.int32, torch.int64)):
        raise RuntimeError(f"bucket_bias: member_idx must be an int32 or int64 array [B, Nq, M], got "
                           f"{tuple(member_idx.shape)} {member_idx.dtype}")
    if dtype not in _FLOATS:
        raise RuntimeError(f"bucket_bias: unsupported output dtype {dtype}")
    for t in (q_pos, k_pos, member_idx):
        if t is not None and t.device != table.device:
            raise RuntimeError("bucket_bias: tensors are on different devices")
    return edges


def _members(member_idx):
    if member_idx is None:
        return None
    if member_idx.dtype == torch.int64:  # an index beyond 32 bits stays out of range
        member_idx = member_idx.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    return nat.dense(member_idx)


def bucket_bias_fwd(table, edges, q_pos, k_pos, member_idx, one_sided, dtype):
    """bias [B,H,Nq,M]; dense inputs, int32 members."""
    arr = _edge_array(edges)
    B, Nq, axes = q_pos.shape
    Nk, H = k_pos.shape[1], table.shape[1]
    M = member_idx.shape[2] if member_idx is not None else Nk
    out = table.new_empty((B, H, Nq, M), dtype=dtype)
    nat.call_on(table.get_device(), "affb_bucket_bias_fwd", nat.ptr(table), nat.dcode(table), ctypes.addressof(arr), len(edges),
                int(one_sided), nat.ptr(q_pos), nat.ptr(k_pos), _POS[q_pos.dtype], axes, nat.ptr(member_idx), B, H, Nq,
                Nk, M, nat.ptr(out), nat.dcode(out))
    return out


def bucket_bias_bwd(dout, edges, q_pos, k_pos, member_idx, one_sided, dtype):
    """The table's gradient in `dtype`; dense inputs, int32 members."""
    arr = _edge_array(edges)
    B, Nq, axes = q_pos.shape
    _, H, _, M = dout.shape
    index = dout.get_device()
    dtable = dout.new_empty((bucket_count(edges, axes, one_sided), H), dtype=dtype)
    ws = nat.workspace(index, "affb_bucket_bias_bwd_workspace_bytes", dout, len(edges), int(one_sided), axes, B, H, Nq, M)
    nat.call_on(index, "affb_bucket_bias_bwd", nat.ptr(dout), nat.dcode(dout), ctypes.addressof(arr), len(edges),
                int(one_sided), nat.ptr(q_pos), nat.ptr(k_pos), _POS[q_pos.dtype], axes, nat.ptr(member_idx), B, H, Nq,
                k_pos.shape[1], M, nat.ptr(dtable), nat.dcode(dtable), nat.ptr(ws), ws.numel() if ws is not None else 0)
    return dtable


class BucketBiasFunction(Function):
    @staticmethod
    def forward(ctx, table, edges, q_pos, k_pos, member_idx, one_sided, dtype):
        qp, kp, mem = nat.dense(q_pos), nat.dense(k_pos), _members(member_idx)
        out = bucket_bias_fwd(table.contiguous(), edges, qp, kp, mem, one_sided, dtype)
        ctx.save_for_backward(qp, kp, mem)
        ctx.meta = (edges, bool(one_sided), table.dtype)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qp, kp, mem = ctx.saved_tensors
        edges, one_sided, dt = ctx.meta
        dtable = bucket_bias_bwd(nat.dense(dout), edges, qp, kp, mem, one_sided, dt)
        return dtable, None, None, None, None, None, None


def bucket_bias(table: torch.Tensor, edges, q_pos: torch.Tensor, k_pos: torch.Tensor,
                member_idx: torch.Tensor | None = None, one_sided: bool = False,
                dtype: torch.dtype | None = None) -> torch.Tensor:
    """bias [B, H, Nq, M] in ``dtype`` (the table's by default).

    table [bucket_count(edges, axes, one_sided), H] fp32 / fp16 / bf16;
    q_pos [B, Nq, axes] and k_pos [B, Nk, axes] in fp32, int32 or int64 with 1
    or 2 axes (x, y); member_idx [B, Nq, M]: the keys of each query (an index
    outside [0, Nk) gives a bias of 0), or None: all keys, M = Nk.
    Differentiable once in the table."""
    dtype = table.dtype if dtype is None else dtype
    edges = _check(table, edges, q_pos, k_pos, member_idx, one_sided, dtype)
    if not nat.differentiates(table):
        return bucket_bias_fwd(table.contiguous(), edges, nat.dense(q_pos), nat.dense(k_pos), _members(member_idx),
                               one_sided, dtype)
    return BucketBiasFunction.apply(table, edges, q_pos, k_pos, member_idx, one_sided, dtype)


class BucketBias(nn.Module):
    """The learned table: ``forward(q_pos, k_pos, member_idx, dtype)``."""

    def __init__(self, heads: int, edges, axes: int = 2, one_sided: bool = False):
        super().__init__()
        self.edges = _check_edges(edges)
        self.one_sided = one_sided
        self.table = nn.Parameter(torch.zeros(bucket_count(self.edges, axes, one_sided), heads))

    def forward(self, q_pos, k_pos, member_idx=None, dtype=None):
        return bucket_bias(self.table, self.edges, q_pos, k_pos, member_idx, self.one_sided, dtype)
