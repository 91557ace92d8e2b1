"""The norms before and after a block, with its gate, its residual and the next product's quantisation in
one pass, over libmq (the reference's rmsnorm and rmsnorm_pack kernels, qwen3/kernels/qwen3k.mojo:17-57,
run the norm alone).
"""
import torch

from ._lib import MQError, lib
from .int8 import MQ_S8, _rows, int8_rows
from .kernels import MQ_F32, _need, _p, _stream
from .pack import _DT

__all__ = ["pre_norm", "pre_norm_s8", "post_norm", "post_norm_s8"]


def pre_norm(x, w, eps=1e-6, h=None, dtype=None):
    """h = x / sqrt(mean(x^2) + eps) * w per row: x [.., cols], w [cols], each fp32 / fp16 / bf16; h like x, of
    `dtype` (default x's) if None."""
    rows, cols, ldx = _rows(x, "x", _DT)
    _need(w, "w", tuple(_DT), cols)
    h = torch.empty(x.shape, dtype=dtype or x.dtype, device=x.device) if h is None else h
    ldh = _rows(h, "h", _DT, cols, rows)[2]
    lib.call("mq_pre_norm", _p(x), _DT[x.dtype], ldx, _p(w), _DT[w.dtype], eps, _p(h), _DT[h.dtype], ldh, None, rows, cols,
             _stream())
    return h


def pre_norm_s8(x, w, eps=1e-6, q=None, s=None):
    """pre_norm quantised per row as quantize_s8 does: (q int8 [rows, cols], s fp32 [rows])."""
    rows, cols, ldx = _rows(x, "x", _DT)
    _need(w, "w", tuple(_DT), cols)
    q = int8_rows(rows, cols, x.device) if q is None else q
    s = torch.empty(rows, dtype=torch.float32, device=x.device) if s is None else s
    ldq = _rows(q, "q", (torch.int8,), cols, rows)[2]
    _need(s, "s", (torch.float32,), rows)
    lib.call("mq_pre_norm", _p(x), _DT[x.dtype], ldx, _p(w), _DT[w.dtype], eps, _p(q), MQ_S8, ldq, _p(s), rows, cols,
             _stream())
    return q, s


def _post(y, w, residual, gate, scale, eps, out, next_w, next_eps, h, h_dt, ldh, hs, rows, cols, ldy):
    ldr = _rows(residual, "residual", _DT, cols, rows)[2]
    ldo = _rows(out, "out", (residual.dtype,), cols, rows)[2]
    if w is not None:
        _need(w, "w", tuple(_DT), cols)
    if next_w is not None:
        _need(next_w, "next_w", tuple(_DT), cols)
    ldg = per = 1
    if gate is not None:
        groups, _, ldg = _rows(gate, "gate", _DT, cols)
        if groups == 0 or rows % groups:
            raise MQError(-1, f"gate: {groups} rows do not divide {rows}")
        per = max(1, rows // groups)
    lib.call("mq_post_norm", _p(y), _DT[y.dtype], ldy, None if w is None else _p(w), MQ_F32 if w is None else _DT[w.dtype],
             eps, _p(residual), _DT[residual.dtype], ldr, None if gate is None else _p(gate),
             MQ_F32 if gate is None else _DT[gate.dtype], ldg, per, scale, _p(out), ldo,
             None if next_w is None else _p(next_w), MQ_F32 if next_w is None else _DT[next_w.dtype], next_eps,
             None if h is None else _p(h), h_dt, ldh, None if hs is None else _p(hs), rows, cols, _stream())


def post_norm(y, w, residual, next_w=None, gate=None, scale=1.0, eps=1e-6, next_eps=None, out=None, h=None, dtype=None):
    """out = residual + scale * gate * norm(y; w) and, with next_w, h = norm(out; next_w) of the sum before it
    is rounded: y, residual [.., cols]; w, next_w [cols]; each fp32 / fp16 / bf16. w None: y itself. gate
    None, [cols], or [groups, cols] with a row per rows / groups consecutive rows. out (may be residual):
    residual's type, made if None; h of `dtype` (default y's) if None. Returns (out, h); h None without next_w."""
    rows, cols, ldy = _rows(y, "y", _DT)
    out = torch.empty(residual.shape, dtype=residual.dtype, device=y.device) if out is None else out
    ldh = cols
    if next_w is not None:
        h = torch.empty(y.shape, dtype=dtype or y.dtype, device=y.device) if h is None else h
        ldh = _rows(h, "h", _DT, cols, rows)[2]
    elif h is not None:
        raise MQError(-1, "h: needs next_w")
    _post(y, w, residual, gate, scale, eps, out, next_w, eps if next_eps is None else next_eps, h,
          MQ_F32 if h is None else _DT[h.dtype], ldh, None, rows, cols, ldy)
    return out, h


def post_norm_s8(y, w, residual, next_w, gate=None, scale=1.0, eps=1e-6, next_eps=None, out=None, q=None, s=None):
    """post_norm with the next norm quantised per row as quantize_s8 does: (out, q int8 [rows, cols], s fp32 [rows])."""
    rows, cols, ldy = _rows(y, "y", _DT)
    out = torch.empty(residual.shape, dtype=residual.dtype, device=y.device) if out is None else out
    q = int8_rows(rows, cols, y.device) if q is None else q
    s = torch.empty(rows, dtype=torch.float32, device=y.device) if s is None else s
    ldq = _rows(q, "q", (torch.int8,), cols, rows)[2]
    _need(s, "s", (torch.float32,), rows)
    if next_w is None:
        raise MQError(-1, "next_w: expected a torch.Tensor")
    _post(y, w, residual, gate, scale, eps, out, next_w, eps if next_eps is None else next_eps, q, MQ_S8, ldq, s, rows,
          cols, ldy)
    return out, q, s
