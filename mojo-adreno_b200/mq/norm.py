"""The norms before and after a block, with its gate, its residual and the next product's quantisation in
one pass, over libmq (the reference's rmsnorm and rmsnorm_pack kernels, qwen3/kernels/qwen3k.mojo:17-57,
run the norm alone).
"""
import torch

from ._lib import MQError, lib
from .int8 import MQ_S8, _F32, _S8, _flat, _rows, _stream, int8_rows
from .kernels import MQ_F32
from .pack import _DT

__all__ = ["pre_norm", "pre_norm_s8", "post_norm", "post_norm_s8"]


def pre_norm(x, w, eps=1e-6, h=None, dtype=None):
    """h = x / sqrt(mean(x^2) + eps) * w per row: x [.., cols], w [cols], each fp32 / fp16 / bf16; h like x, of
    `dtype` (default x's) if None."""
    rows, cols, ldx = _rows(x, "x", _DT)
    h = torch.empty(x.shape, dtype=dtype or x.dtype, device=x.device) if h is None else h
    ldh = _rows(h, "h", _DT, cols, rows)[2]
    lib.call("mq_pre_norm", x.data_ptr(), _DT[x.dtype], ldx, _flat(w, "w", _DT, cols), _DT[w.dtype], eps, h.data_ptr(),
             _DT[h.dtype], ldh, None, rows, cols, _stream())
    return h


def pre_norm_s8(x, w, eps=1e-6, q=None, s=None):
    """pre_norm quantised per row as quantize_s8 does: (q int8 [rows, cols], s fp32 [rows])."""
    rows, cols, ldx = _rows(x, "x", _DT)
    q = int8_rows(rows, cols, x.device) if q is None else q
    s = torch.empty(rows, dtype=torch.float32, device=x.device) if s is None else s
    ldq = _rows(q, "q", _S8, cols, rows)[2]
    lib.call("mq_pre_norm", x.data_ptr(), _DT[x.dtype], ldx, _flat(w, "w", _DT, cols), _DT[w.dtype], eps, q.data_ptr(),
             MQ_S8, ldq, _flat(s, "s", _F32, rows), rows, cols, _stream())
    return q, s


def _post(y, w, residual, gate, scale, eps, out, next_w, next_eps, h, h_dt, ldh, hs, rows, cols, ldy):
    ldr = _rows(residual, "residual", _DT, cols, rows)[2]
    ldo = ldr if out is residual else _rows(out, "out", (residual.dtype,), cols, rows)[2]
    w_p = w_dt = nw_p = nw_dt = gate_p = g_dt = 0
    ldg = per = 1
    if w is not None:
        w_p, w_dt = _flat(w, "w", _DT, cols), _DT[w.dtype]
    if next_w is not None:
        nw_p, nw_dt = _flat(next_w, "next_w", _DT, cols), _DT[next_w.dtype]
    if gate is not None:
        groups, _, ldg = _rows(gate, "gate", _DT, cols)
        if groups == 0 or rows % groups:
            raise MQError(-1, f"gate: {groups} rows do not divide {rows}")
        per = rows // groups or 1
        gate_p, g_dt = gate.data_ptr(), _DT[gate.dtype]
    lib.call("mq_post_norm", y.data_ptr(), _DT[y.dtype], ldy, w_p, w_dt, eps, residual.data_ptr(), _DT[residual.dtype], ldr,
             gate_p, g_dt, ldg, per, scale, out.data_ptr(), ldo, nw_p, nw_dt, next_eps,
             None if h is None else h.data_ptr(), h_dt, ldh, hs, rows, cols, _stream())


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
    ldq = _rows(q, "q", _S8, cols, rows)[2]
    if next_w is None:
        raise MQError(-1, "next_w: expected a torch.Tensor")
    _post(y, w, residual, gate, scale, eps, out, next_w, eps if next_eps is None else next_eps, q, MQ_S8, ldq,
          _flat(s, "s", _F32, rows), rows, cols, ldy)
    return out, q, s
