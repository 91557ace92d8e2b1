"""A paged cache of keys and values, and the attention of new tokens over it, over libmq.

The reference's attention reads one contiguous cache of one sequence. Here a cache is a pool of pages that sequences
share: sequence b keeps position p in page table[b, p // page], row p % page. The operators take a batch's
new tokens (a prompt, a chunk of one, drafted tokens, one token each) behind one another: sequence b has rows
starts[b] .. starts[b + 1], and lengths[b] positions in the cache with them, so that its row i of n is position
lengths[b] - n + i, n = starts[b + 1] - starts[b]. Starts that pass the rows are reported (device_status() 27) and those that
are there keep their positions. Table, lengths and starts are int32 on the device and are never read on the host.
"""
import ctypes

import torch

from ._lib import MQError, lib
from .int8 import MQ_S8, _current_device, _flat, _stream
from .pack import _DT

__all__ = ["PagedCache", "paged_cache", "kv_store", "kv_load", "paged_attention", "paged_attention_workspace"]

_I32 = frozenset((torch.int32,))
_CACHE = {torch.float16: _DT[torch.float16], torch.bfloat16: _DT[torch.bfloat16], torch.int8: MQ_S8}
_BITS16 = frozenset((torch.float16, torch.bfloat16))
_Three = ctypes.c_int64 * 3


class _Pages(ctypes.Structure):  # mq_kv_pages
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
                ("k_stride", _Three), ("v_stride", _Three), ("ks_stride", _Three), ("vs_stride", _Three),
                ("pages", ctypes.c_int64), ("dtype", ctypes.c_int32), ("heads", ctypes.c_int32), ("page", ctypes.c_int32),
                ("dim", ctypes.c_int32)]


class PagedCache:
    """A layer's pool: k and v [pages, kv_heads, page, dim], fp16, bf16 or int8, in any order of the first three
    dimensions (rows 16-byte aligned); int8 with k_scale and v_scale fp32 [pages, kv_heads, page]. page: 16, 32, 64, 128 or
    256; dim: a multiple of 16 up to 128. The cache keeps the tensors; it owns nothing else."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        for t, name in ((k, "k"), (v, "v")):
            if not isinstance(t, torch.Tensor) or not t.is_cuda:
                raise MQError(-1, f"{name}: must be a CUDA tensor (there is no CPU path)")
            if t.dtype not in _CACHE or t.dtype != k.dtype:
                raise MQError(-1, f"{name}: dtype {t.dtype} is not the fp16, bf16 or int8 of both")
            if t.dim() != 4 or t.shape != k.shape:
                raise MQError(-1, f"{name}: expected [pages, kv_heads, page, dim], the same for keys and values")
            if t.shape[3] > 1 and t.stride(3) != 1:
                raise MQError(-1, f"{name}: the last dimension must be contiguous")
            if t.device != k.device:
                raise MQError(-1, f"{name}: keys and values are on different devices")
        scales = (k_scale, v_scale)
        if k.dtype == torch.int8:
            for t, name in zip(scales, ("k_scale", "v_scale")):
                if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != k.shape[:3] or t.device != k.device:
                    raise MQError(-1, f"{name}: an int8 cache needs fp32 [pages, kv_heads, page] on its device")
        elif k_scale is not None or v_scale is not None:
            raise MQError(-1, "k_scale, v_scale: only an int8 cache has scales")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device_index = k.device.index
        p = self._pages = _Pages(k=k.data_ptr(), v=v.data_ptr(), k_stride=_Three(*k.stride()[:3]), v_stride=_Three(*v.stride()[:3]),
                                 pages=k.shape[0], dtype=_CACHE[k.dtype], heads=k.shape[1], page=k.shape[2], dim=k.shape[3])
        if k.dtype == torch.int8:
            p.k_scale, p.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
            p.ks_stride, p.vs_stride = _Three(*k_scale.stride()), _Three(*v_scale.stride())
        self._address = ctypes.addressof(p)

    @property
    def kv_heads(self):
        return self._pages.heads

    @property
    def page(self):
        return self._pages.page

    @property
    def dim(self):
        return self._pages.dim


def paged_cache(pages, kv_heads, page, dim, dtype=torch.float16, device=None):
    """A PagedCache of new tensors, zeroed."""
    device = device or "cuda"
    k, v = (torch.zeros(pages, kv_heads, page, dim, dtype=dtype, device=device) for _ in range(2))
    if dtype != torch.int8:
        return PagedCache(k, v)
    return PagedCache(k, v, *(torch.zeros(pages, kv_heads, page, device=device) for _ in range(2)))


def _here(cache):
    if not isinstance(cache, PagedCache):
        raise MQError(-1, "cache: expected a PagedCache")
    device = cache.device_index
    if device != _current_device():
        raise MQError(-1, f"cache: is on device {device}, not on the current one")
    return device


def _where(table, lengths, starts, tokens, device):
    """The arguments that say which positions the rows are."""
    if not isinstance(table, torch.Tensor) or table.dtype != torch.int32 or table.dim() != 2 or table.get_device() != device:
        raise MQError(-1, "table: expected int32 [batch, width] on the cache's device")
    batch, width = table.shape
    ldt, step = table.stride()
    if step != 1 and width > 1:
        raise MQError(-1, "table: the last dimension must be contiguous")
    lengths_p = _flat(lengths, "lengths", _I32, batch)
    if starts is None:
        if tokens != batch:
            raise MQError(-1, f"starts: {tokens} tokens of {batch} sequences need starts")
        starts_p = None
    else:
        starts_p = _flat(starts, "starts", _I32, batch + 1)
        if starts.get_device() != device:
            raise MQError(-1, "starts: is not on the cache's device")
    if lengths.get_device() != device:
        raise MQError(-1, "lengths: is not on the cache's device")
    return table.data_ptr(), ldt, width, lengths_p, starts_p, batch


def _rows3(t, name, dtypes, heads, dim, device):
    """(tokens, heads, token stride, head stride) of a tensor [tokens, heads, dim]."""
    if not isinstance(t, torch.Tensor) or t.get_device() != device or t.dtype not in dtypes:
        raise MQError(-1, f"{name}: expected a CUDA tensor on the cache's device, of a type in {tuple(dtypes)}")
    if t.dim() != 3:
        raise MQError(-1, f"{name}: expected [tokens, heads, dim]")
    tokens, h, d = t.shape
    if d != dim or (heads and h != heads):
        raise MQError(-1, f"{name}: shape {tuple(t.shape)} does not go with a cache of {heads or 'any'} heads of {dim}")
    st, sh, se = t.stride()
    if se != 1:
        raise MQError(-1, f"{name}: the last dimension must be contiguous")
    # (the stride of one token or one head is never used)
    return tokens, h, st if tokens > 1 else h * dim, sh if h > 1 else dim


def kv_store(k, v, cache, table, lengths, starts=None):
    """Writes the new tokens' keys and values into their pages, rounded to the cache's type or, int8, quantised row by
    row as quantize_s8 does. k, v: fp32, fp16 or bf16 [tokens, kv_heads, dim], rows 16-byte aligned. A table entry
    outside the pool is skipped and reported (device_status() 19), and so are positions beyond the table (20). k and v must not lie in
    the pages. Returns the cache."""
    device = _here(cache)
    p = cache._pages
    tokens, _, kt, kh = _rows3(k, "k", _DT, p.heads, p.dim, device)
    if not isinstance(v, torch.Tensor) or v.dtype != k.dtype or v.shape != k.shape:
        raise MQError(-1, "v: expected k's type and shape")
    _, _, vt, vh = _rows3(v, "v", _DT, p.heads, p.dim, device)
    lib.call("mq_kv_store", k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, _DT[k.dtype], cache._address,
             *_where(table, lengths, starts, tokens, device), tokens, _stream())
    return cache


def kv_load(cache, table, lengths, starts=None, k=None, v=None, tokens=None, dtype=torch.float16):
    """(k, v) [tokens, kv_heads, dim]: what the pages hold of the positions that kv_store would write. k, v: fp32, fp16 or
    bf16, made of `dtype` if None, with as many rows as `tokens` (None: one per sequence, and with starts, whose end is on the
    device, to be said)."""
    device = _here(cache)
    p = cache._pages
    if k is None or v is None:
        if tokens is None:
            have = k if k is not None else v
            if have is None and starts is not None:
                raise MQError(-1, "tokens: with starts, say how many rows there are (or give k or v)")
            if not isinstance(table if have is None else have, torch.Tensor):
                raise MQError(-1, "table, k, v: expected a torch.Tensor")
            tokens = (table if have is None else have).shape[0]
        shape = (tokens, p.heads, p.dim)
        kind = k.dtype if k is not None else v.dtype if v is not None else dtype
        k = torch.empty(shape, dtype=kind, device=cache.k.device) if k is None else k
        v = torch.empty(shape, dtype=kind, device=cache.k.device) if v is None else v
    n, _, kt, kh = _rows3(k, "k", _DT, p.heads, p.dim, device)
    if not isinstance(v, torch.Tensor) or v.dtype != k.dtype or v.shape != k.shape:
        raise MQError(-1, "v: expected k's type and shape")
    if tokens is not None and n != tokens:
        raise MQError(-1, f"k: has {n} rows, expected {tokens}")
    _, _, vt, vh = _rows3(v, "v", _DT, p.heads, p.dim, device)
    lib.call("mq_kv_load", cache._address, *_where(table, lengths, starts, n, device), n, k.data_ptr(), kt, kh, v.data_ptr(), vt,
             vh, _DT[k.dtype], _stream())
    return k, v


def paged_attention_workspace(cache, heads, batch, tokens, max_new=0):
    """The bytes of a workspace for paged_attention; enough for fewer sequences or tokens, and a smaller max_new, too."""
    _here(cache)
    return max(lib.mq_paged_attention_workspace_size(cache._address, heads, batch, tokens, max_new), 16)


def paged_attention(q, cache, table, lengths, starts=None, out=None, scale=None, window=0, max_new=0, workspace=None):
    """Attention of the new tokens over what their sequences have in the cache, themselves included: out[t, h] =
    softmax(scale * q[t, h] . k_j) v_j over the positions j up to the token's own, the last `window` of them if that is
    not 0. q fp16 or bf16 (a 16-bit cache's type) [tokens, heads, dim], heads a multiple of the cache's (query head h
    uses kv head h // (heads // kv_heads)); out likewise, made if None, may be q
    (but not share memory with it in another way). scale: dim ** -0.5 if None. A row that sees
    nothing gives zeros; positions that a row does not see do not matter, whatever they hold. max_new: no sequence has
    more new tokens than this (0: unknown); said, it spares a launch where all have few. Calls that may overlap in time
    need a workspace each."""
    device = _here(cache)
    p = cache._pages
    tokens, heads, qt, qh = _rows3(q, "q", _BITS16, 0, p.dim, device)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif not isinstance(out, torch.Tensor) or out.dtype != q.dtype or out.shape != q.shape:
        raise MQError(-1, "out: expected q's type and shape")
    _, _, ot, oh = _rows3(out, "out", _BITS16, 0, p.dim, device)
    where = _where(table, lengths, starts, tokens, device)
    if workspace is None:
        nbytes = lib.mq_paged_attention_workspace_size(cache._address, heads, where[5], tokens, max_new)
        workspace = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=q.device)
    elif not isinstance(workspace, torch.Tensor) or workspace.dtype != torch.uint8 or not workspace.is_contiguous() or \
            workspace.get_device() != device:
        raise MQError(-1, "workspace: expected a contiguous uint8 tensor on the cache's device")
    lib.call("mq_paged_attention", q.data_ptr(), _DT[q.dtype], qt, qh, cache._address, *where, tokens, heads,
             p.dim ** -0.5 if scale is None else scale, window, max_new, out.data_ptr(), ot, oh, workspace.data_ptr(),
             workspace.numel(), _stream())
    return out
