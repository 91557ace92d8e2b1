"""int8 products with a scale per token and per output channel, over libmq.

The reference has no kernel of this kind on its hot path (its weights have at most 4 bits). An int8
matrix is a [rows, k] int8 tensor whose rows start 16 bytes aligned (`int8_rows` allocates one; k may be any
number), with one fp32 scale per row; quantize_s8 makes both, of tokens and, once, of weights.
"""
import torch

from ._lib import MQError, lib
from .kernels import _need, _raw_stream
from .kernels import _stream as _any_stream
from .pack import _DT

__all__ = ["MQ_S8", "int8_rows", "quantize_s8", "gemm_w8a8", "gate_up_w8a8"]

MQ_S8 = 3


_device = getattr(torch._C, "_cuda_getDevice", None)


def _stream():
    """The current device's current stream, behind a check of a CUDA tensor (so CUDA is initialised)."""
    return _any_stream() if _device is None or _raw_stream is None else _raw_stream(_device())


def _rows(t, name, dtypes, cols=None, rows=None):
    """(rows, cols, row stride in elements) of a CUDA tensor [.., cols] whose rows are contiguous: two
    dimensions with any row stride, or any number of dimensions without gaps."""
    if not isinstance(t, torch.Tensor):
        raise MQError(-1, f"{name}: expected a torch.Tensor")
    if not t.is_cuda:
        raise MQError(-1, f"{name}: must be a CUDA tensor (there is no CPU path)")
    if t.dtype not in dtypes:
        raise MQError(-1, f"{name}: dtype {t.dtype} not in {tuple(dtypes)}")
    shape = t.shape
    if len(shape) == 2:
        r, c = shape
        ld, step = t.stride()
        if step != 1 and c > 1:
            raise MQError(-1, f"{name}: the last dimension must be contiguous")
        if r <= 1:
            ld = c or 1
    else:
        if not shape or not t.is_contiguous():
            raise MQError(-1, f"{name}: must be two-dimensional or contiguous")
        c = shape[-1]
        r = t.numel() // c if c else 0
        ld = c or 1
    if cols is not None and c != cols:
        raise MQError(-1, f"{name}: has rows of {c} elements, expected {cols}")
    if rows is not None and r != rows:
        raise MQError(-1, f"{name}: has {r} rows, expected {rows}")
    return r, c, ld


def _flat(t, name, dtypes, numel):
    """The data pointer of a contiguous CUDA tensor of numel elements."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in dtypes or t.numel() != numel or \
            not t.is_contiguous():
        _need(t, name, tuple(dtypes), numel)
    return t.data_ptr()


_F32 = frozenset((torch.float32,))
_S8 = frozenset((torch.int8,))


def _rows8(t, name, cols=None, rows=None):
    """_rows of an int8 matrix; the stride of a single row is never used and is rounded up to 16."""
    r, c, ld = _rows(t, name, _S8, cols, rows)
    return r, c, -(-ld // 16) * 16 if r <= 1 else ld


def int8_rows(rows, cols, device=None):
    """An uninitialised int8 [rows, cols] matrix with 16-byte aligned rows."""
    return torch.empty(rows, -(-cols // 16) * 16, dtype=torch.int8, device=device or "cuda")[:, :cols]


def quantize_s8(x, q=None, s=None):
    """(q, s) with q = rint(x * (127 / a)) and s = a / 127, a the largest |x| of each row: x fp32 / fp16 / bf16
    [.., cols] -> int8 [rows, cols] and fp32 [rows]. For tokens, and once for weights."""
    rows, cols, ldx = _rows(x, "x", _DT)
    q = int8_rows(rows, cols, x.device) if q is None else q
    s = torch.empty(rows, dtype=torch.float32, device=x.device) if s is None else s
    ldq = _rows(q, "q", _S8, cols, rows)[2]
    lib.call("mq_quantize_s8", x.data_ptr(), _DT[x.dtype], ldx, q.data_ptr(), ldq, _flat(s, "s", _F32, rows), rows, cols,
             _stream())
    return q, s


def gemm_w8a8(xq, xs, wq, ws, y=None, bias=None, add=False, dtype=torch.float16):
    """y[t, r] (+)= xs[t] * ws[r] * sum_k xq[t, k] wq[r, k] + bias[r]: xq int8 [m, k], wq int8 [n, k] (rows 16-byte
    aligned), xs fp32 [m], ws fp32 [n], bias fp32 [n]; y fp32 / fp16 / bf16 [m, n] (made of `dtype` if None)."""
    m, k, ldx = _rows8(xq, "xq")
    n, _, ldw = _rows8(wq, "wq", k)
    if y is None:
        if add:
            raise MQError(-1, "y: add needs the tensor to add into")
        y = torch.empty(m, n, dtype=dtype, device=xq.device)
    ldy = _rows(y, "y", _DT, n, m)[2]
    lib.call("mq_gemm_w8a8", xq.data_ptr(), ldx, _flat(xs, "xs", _F32, m), wq.data_ptr(), ldw, _flat(ws, "ws", _F32, n),
             None if bias is None else _flat(bias, "bias", _F32, n), y.data_ptr(), _DT[y.dtype], ldy, m, n, k,
             1 if add else 0, _stream())
    return y


def gate_up_w8a8(xq, xs, wq, ws, a=None, dtype=torch.float16):
    """a[t, j] = silu(g) * u, g and u the products of rows j and f + j of the fused gate|up matrix wq int8
    [2f, k] (ws fp32 [2f]); a fp32 / fp16 / bf16 [m, f]."""
    m, k, ldx = _rows8(xq, "xq")
    n, _, ldw = _rows8(wq, "wq", k)
    if n % 2:
        raise MQError(-1, f"wq: {n} rows are not gate and up rows")
    a = torch.empty(m, n // 2, dtype=dtype, device=xq.device) if a is None else a
    lda = _rows(a, "a", _DT, n // 2, m)[2]
    lib.call("mq_gate_up_w8a8", xq.data_ptr(), ldx, _flat(xs, "xs", _F32, m), wq.data_ptr(), ldw, _flat(ws, "ws", _F32, n),
             a.data_ptr(), _DT[a.dtype], lda, m, n // 2, k, _stream())
    return a
