"""The refusals of the paged cache, the attention over it and the verification of drafted tokens, without a GPU: arguments are
checked before a device is touched."""
import ctypes

import pytest

P = ctypes.c_void_p
OK = 1 << 20  # never dereferenced: validation fails first


def pages(**kw):
    from mq.paged import _Pages, _Three

    p = _Pages(k=OK, v=OK, k_scale=OK, v_scale=OK, k_stride=_Three(2 * 16 * 64, 16 * 64, 64), v_stride=_Three(2 * 16 * 64, 16 * 64, 64),
               ks_stride=_Three(32, 16, 1), vs_stride=_Three(32, 16, 1), pages=8, dtype=1, heads=2, page=16, dim=64)
    for name, value in kw.items():
        setattr(p, name, _Three(*value) if isinstance(value, tuple) else value)
    return p


def status(name, *args):
    from mq._lib import lib

    rc = getattr(lib, name)(*args)
    return rc, lib.mq_last_error().decode()


def without_device():
    """For calls that the checks let pass: with a device they would go on to addresses that are none."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("needs a machine without a GPU")


def attention(cache=None, **kw):
    a = dict(q=OK, q_dtype=1, q_token=512, q_head=64, table=OK, ldt=4, width=4, lengths=OK, starts=OK, batch=2, tokens=5, heads=8,
             scale=0.125, window=0, max_new=0, out=OK, o_token=512, o_head=64, workspace=OK, size=16)
    a.update(kw)
    c = pages() if cache is None else cache
    return status("mq_paged_attention", a["q"], a["q_dtype"], a["q_token"], a["q_head"], ctypes.addressof(c), a["table"], a["ldt"],
                  a["width"], a["lengths"], a["starts"], a["batch"], a["tokens"], a["heads"], a["scale"], a["window"], a["max_new"],
                  a["out"], a["o_token"], a["o_head"], a["workspace"], a["size"], None)


@pytest.mark.parametrize("cache,code,match", [
    (dict(k=None), -1, "null"), (dict(dtype=0), -1, "type"), (dict(dtype=4), -1, "type"), (dict(pages=0), -1, "pages"),
    (dict(heads=0), -1, "heads"), (dict(page=8), -4, "page"), (dict(page=48), -4, "page"), (dict(page=512), -4, "page"),
    (dict(dim=8), -4, "dim"), (dict(dim=72), -4, "dim"), (dict(dim=144), -4, "dim"), (dict(k=OK + 8), -2, "aligned"),
    (dict(v_stride=(2 * 16 * 64, 16 * 64, 68)), -2, "aligned"), (dict(k_stride=(2 * 16 * 64, 16 * 64, 56)), -1, "overlap"),
    (dict(k_stride=(0, 16 * 64, 64)), -1, "overlap"), (dict(k_stride=(-2048, 16 * 64, 64)), -1, "overlap"),
    (dict(k_stride=(1 << 40, 16 * 64, 64)), -1, "overlap"), (dict(dtype=3, v_scale=None), -1, "scales"),
    (dict(dtype=3, ks_stride=(32, 16, 0)), -1, "overlap"), (dict(dtype=3, k_scale=OK + 2), -2, "aligned"),
])
def test_caches(cache, code, match):
    c = pages(**cache)
    for rc, msg in (attention(c), status("mq_kv_store", OK, 128, 64, OK, 128, 64, 1, ctypes.addressof(c), OK, 4, 4, OK, OK, 2, 5, None),
                    status("mq_kv_load", ctypes.addressof(c), OK, 4, 4, OK, OK, 2, 5, OK, 128, 64, OK, 128, 64, 1, None)):
        assert rc == code and match in msg


@pytest.mark.parametrize("args,code,match", [
    (dict(batch=-1), -1, "shape"), (dict(tokens=-1), -1, "shape"), (dict(width=-1), -1, "shape"), (dict(batch=1 << 22), -4, "too many"),
    (dict(tokens=1 << 30), -4, "too many"), (dict(width=1 << 40), -4, "positions"), (dict(width=1 << 27, ldt=1 << 27), -4, "positions"),
    (dict(starts=None), -1, "one row"), (dict(lengths=None), -1, "null"), (dict(table=None), -1, "null"),
    (dict(lengths=OK + 2), -2, "aligned"), (dict(ldt=3), -1, "stride"), (dict(heads=0), -1, "multiple"), (dict(heads=7), -1, "multiple"),
    (dict(heads=1 << 17), -4, "heads"), (dict(q_dtype=0), -1, "q must"), (dict(q_dtype=2), -1, "16-bit cache"), (dict(scale=0.0), -1, "scale"),
    (dict(scale=-1.0), -1, "scale"), (dict(scale=float("inf")), -1, "scale"), (dict(scale=float("nan")), -1, "scale"),
    (dict(window=-1), -1, "window"), (dict(window=1 << 31), -4, "window"), (dict(max_new=-1), -1, "new tokens"), (dict(q=None), -1, "null"),
    (dict(q=OK + 2), -2, "q must start"), (dict(q_token=500), -2, "q must start"), (dict(q_head=-64), -1, "negative"),
    (dict(out=None), -1, "null"), (dict(out=OK + 8), -2, "out must start"), (dict(o_token=448), -1, "overlap"), (dict(o_head=0), -1, "overlap"),
])
def test_attention(args, code, match):
    rc, msg = attention(**args)
    assert rc == code and match in msg, msg


def test_attention_of_nothing():
    assert attention(tokens=0)[0] == 0 and attention(batch=0, tokens=0, starts=None)[0] == 0


@pytest.mark.parametrize("args,code,match", [(dict(dtype=3), -1, "rows must"), (dict(k=None), -1, "null"), (dict(k=OK + 4), -2, "k must start"),
                                           (dict(vt=100), -2, "v must start"), (dict(kh=-64), -1, "negative")])
def test_copies(args, code, match):
    a = dict(k=OK, kt=128, kh=64, v=OK, vt=128, vh=64, dtype=1)
    a.update(args)
    c = pages()
    rows = (a["k"], a["kt"], a["kh"], a["v"], a["vt"], a["vh"])
    where = (ctypes.addressof(c), OK, 4, 4, OK, OK, 2, 5)
    for rc, msg in (status("mq_kv_store", *rows, a["dtype"], *where, None), status("mq_kv_load", *where, *rows, a["dtype"], None)):
        assert rc == code and match in msg, msg


@pytest.mark.parametrize("shift,refused", [(0, True), (128, True), (64 * 2 * 16 * 2 - 16, True), (64 * 2 * 16 * 2 * 8, False), (-64 * 2 * 16 * 2 * 8, False)])
def test_store_where_keys_and_values_share_memory(shift, refused):
    """v `shift` bytes behind k, both of 8 pages of 2 x 16 rows of 128 bytes."""
    c = pages(v=OK + shift)
    rc, msg = status("mq_kv_store", OK, 128, 64, OK, 128, 64, 1, ctypes.addressof(c), OK, 4, 4, OK, OK, 2, 5, None)
    assert ("share memory" in msg and rc == -1) if refused else rc != -1  # (without a device the call ends behind the checks)


def test_store_of_interleaved_pages_is_not_refused():
    """One tensor [pages, 2, heads, page, dim]: keys and values lie between one another's pages."""
    stride = (2 * 2 * 16 * 64, 16 * 64, 64)
    c = pages(k_stride=stride, v_stride=stride, v=OK + 2 * 16 * 64 * 2)
    rc, msg = status("mq_kv_store", OK, 128, 64, OK, 128, 64, 1, ctypes.addressof(c), OK, 4, 4, OK, OK, 2, 5, None)
    assert rc != -1, msg


def test_load_into_rows_that_overlap():
    rc, msg = status("mq_kv_load", ctypes.addressof(pages()), OK, 4, 4, OK, OK, 2, 5, OK, 64, 64, OK, 128, 64, 1, None)
    assert rc == -1 and "overlap" in msg


@pytest.mark.parametrize("args,code,match", [
    (dict(batch=-1), -1, "shape"), (dict(vocab=0), -1, "shape"), (dict(drafts=-1), -1, "shape"), (dict(drafts=33), -4, "drafts above"),
    (dict(batch=1 << 21), -4, "batch"), (dict(vocab=1 << 31, ld=1 << 31), -4, "vocab"), (dict(dtype=3), -1, "type"), (dict(ld=99), -1, "stride"),
    (dict(ld_draft=99), -1, "stride"), (dict(target=None), -1, "null"), (dict(drafted=None), -1, "null"), (dict(uniform=None), -1, "null"),
    (dict(tokens=None), -1, "null"), (dict(target=OK + 2), -2, "aligned"), (dict(workspace=OK + 8), -2, "aligned"), (dict(size=16), -1, "too small"),
])
def test_verify(args, code, match):
    a = dict(target=OK, ld=100, draft=OK, ld_draft=100, dtype=0, drafted=OK, counts=None, uniform=OK, temperature=None, tokens=OK, accepted=OK,
             logprobs=OK, batch=2, drafts=3, vocab=100, workspace=OK, size=1 << 20)
    a.update(args)
    rc, msg = status("mq_verify_drafts", *a.values(), None)
    assert rc == code and match in msg, msg
    assert status("mq_verify_drafts", *{**a, **dict(batch=0, drafts=3, vocab=100, dtype=0, ld=100, ld_draft=100)}.values(), None)[0] == 0


def test_workspace_sizes_of_what_is_refused():
    from mq._lib import lib

    assert lib.mq_verify_workspace_size(1 << 21, 3, 100) == 0 and lib.mq_verify_workspace_size(2, 33, 100) == 0
    assert lib.mq_verify_workspace_size(2, 3, 100) > 0
    assert lib.mq_paged_attention_workspace_size(ctypes.addressof(pages(dim=8)), 8, 2, 5, 0) == 0
    assert lib.mq_paged_attention_workspace_size(ctypes.addressof(pages()), 7, 2, 5, 0) == 0


def test_python_operators_refuse_cpu_tensors():
    import torch

    import mq

    x = torch.zeros(2, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(mq.MQError, match="CUDA"):
        mq.PagedCache(x, x)
    with pytest.raises(mq.MQError, match="CUDA"):
        mq.verify_drafts(torch.zeros(4, 10), torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, 4))
    with pytest.raises(mq.MQError, match="PagedCache"):
        mq.kv_store(x[0], x[0], None, None, None)


def test_verify_workspace_of_a_larger_call_is_enough():
    """Sizes never fall when a call has more requests, drafts or tokens, and hold a pair of fp32 for each CTA of the scan: as many per
    row as let eight run on each of 148 SMs, 64 at most, and one step of 16 KB of fp32 each."""
    from mq._lib import lib

    def needs(rows, vocab):
        return 8 * rows * max(1, min(64, 148 * 8 // rows, -(-vocab * 4 // (256 * 4 * 16))))

    for vocab in (1, 100, 4096, 32000, 128256, 151669, 262144, 1 << 20):
        for drafts in (0, 1, 2, 4, 8, 32):
            largest = 0
            for batch in list(range(1, 140)) + [250, 591, 592, 593, 1183, 1184, 1185, 5000, 1 << 20]:
                size = lib.mq_verify_workspace_size(batch, drafts, vocab)
                assert size >= largest and size >= needs(batch * (2 * drafts + 1), vocab) and size >= needs(batch * (drafts + 1), vocab)
                assert size >= lib.mq_verify_workspace_size(batch, max(drafts - 1, 0), vocab)
                assert size >= lib.mq_verify_workspace_size(batch, drafts, max(vocab // 3, 1))
                largest = size


@pytest.mark.parametrize("shift,stride,refused", [(0, (32, 16, 1), True), (4, (32, 16, 1), True), (4 * 255, (32, 16, 1), True), (4 * 256, (32, 16, 1), False),
                                                  (-4 * 255, (32, 16, 1), True), (-4 * 256, (32, 16, 1), False), (64, (64, 32, 1), False),
                                                  (68, (64, 32, 1), True), (4, (64, 32, 2), False), (8, (64, 32, 2), True), (0, (1, 8, 16), True)])
def test_store_where_scales_share_memory(shift, stride, refused):
    """v_scale `shift` bytes behind k_scale, both of 8 pages of 2 x 16 fp32: side by side or between one another they may lie."""
    without_device()

    def store(dtype):
        c = pages(v=OK + (1 << 16), dtype=dtype, k_scale=OK << 2, v_scale=(OK << 2) + shift, ks_stride=stride, vs_stride=stride)
        return status("mq_kv_store", OK, 128, 64, OK, 128, 64, 1, ctypes.addressof(c), OK, 4, 4, OK, OK, 2, 5, None)

    rc, msg = store(3)
    assert ("share memory" in msg and rc == -1) if refused else rc != -1, msg
    assert store(1)[0] != -1  # (a 16-bit cache has none)


# ---- calls that overlap: the pages of `pages()` are 8 x 2 x 16 rows of 128 bytes, 32768 in all --------------------

FAR = OK + (1 << 24)


def apart(**kw):
    return pages(**{**dict(k=OK, v=OK + 32768, k_scale=OK + 65536, v_scale=OK + 65536 + 1024), **kw})


@pytest.mark.parametrize("args,refused", [
    (dict(out=FAR), None), (dict(out=FAR, o_head=128, o_token=1024), "q"), (dict(out=FAR + 16), "q"), (dict(out=FAR + 512), "q"),
    (dict(out=FAR + 5 * 1024), None), (dict(out=FAR - 5 * 1024), None), (dict(out=FAR - 5 * 1024 + 16), "q"),
    # A fused projection's buffer: q's 8 of 12 heads, out in the 4 (of 4 heads of 64, 2 kv heads) behind them or over q's last.
    (dict(q_token=768, out=FAR + 1024, o_token=768, heads=4), None), (dict(q_token=768, out=FAR + 256, o_token=768, heads=4), "q"),
    (dict(q_token=768, out=FAR + 1024, o_token=760, heads=4), None), (dict(q_token=768, out=FAR + 1024, o_token=776, heads=4), "q"), (dict(q_token=768, out=FAR + 512, o_token=760, heads=4), "q"),
    # Heads behind one another instead of tokens: the same bytes in another order.
    (dict(out=FAR, o_token=64, o_head=5 * 64), "q"), (dict(q=FAR, q_token=0, q_head=0, out=FAR + 128), None), (dict(q_token=0, q_head=0, out=FAR), "q"),
    (dict(out=OK), "pages"), (dict(out=OK + 32768 + 32752), "pages"), (dict(out=OK + 65536), None), (dict(out=OK - 5 * 1024), None),
])
def test_attention_into_memory_that_is_read(args, refused):
    without_device()
    rc, msg = attention(apart(), **{**dict(q=FAR), **args})
    if refused:
        assert rc == -1 and "shares memory with " + ("q" if refused == "q" else "the pages") in msg, msg
    else:
        assert rc not in (-1, 0) and "memory" not in msg, msg


def test_attention_into_scales():
    without_device()
    for at, refused in ((65536, True), (65536 + 2047 // 16 * 16, True), (65536 + 2048, False)):
        rc, msg = attention(apart(dtype=3), q=FAR, out=OK + at)
        assert (rc == -1 and "with the pages" in msg) if refused else rc not in (-1, 0), msg


@pytest.mark.parametrize("k,kt,v,vt,match", [
    (FAR, 128, FAR, 128, "k and v"), (FAR, 128, FAR + 1280, 128, None), (FAR, 128, FAR + 1280 - 16, 128, "k and v"), (FAR, 256, FAR + 256, 256, None),
    (FAR, 256, FAR + 240, 256, "k and v"), (FAR, 256, FAR + 256, 384, "k and v"), (OK, 128, FAR, 128, "pages"), (FAR, 128, OK + 65536 - 16, 128, "pages"),
    (FAR, 128, OK + 65536, 128, None)])
def test_load_into_memory_that_is_read(k, kt, v, vt, match):
    without_device()
    c = apart()
    rc, msg = status("mq_kv_load", ctypes.addressof(c), OK, 4, 4, OK, OK, 2, 5, k, kt, 64, v, vt, 64, 1, None)
    assert (rc == -1 and match in msg and "memory" in msg) if match else rc not in (-1, 0), msg


@pytest.mark.parametrize("cache,refused", [
    (dict(), False), (dict(v=OK), True), (dict(v=OK + 32768 - 16), True),
    # Pages of keys head by head and of values position by position, one behind the other in each block of 8192 bytes.
    (dict(k_stride=(4096, 1024, 64), v=OK + 4096, v_stride=(4096, 64, 128)), False),
    (dict(k_stride=(4096, 1024, 64), v=OK + 4096 - 128, v_stride=(4096, 64, 128)), True),
    # Keys, values and scales of a page in one block of 8448 bytes.
    (dict(dtype=3, k_stride=(8448, 1024, 64), v=OK + 2048, v_stride=(8448, 1024, 64), k_scale=OK + 4096, v_scale=OK + 4224, ks_stride=(2112, 16, 1),
          vs_stride=(2112, 16, 1)), False),
    (dict(dtype=3, k_stride=(8448, 1024, 64), v=OK + 2048, v_stride=(8448, 1024, 64), k_scale=OK + 4092, v_scale=OK + 4224, ks_stride=(2112, 16, 1),
          vs_stride=(2112, 16, 1)), True),
    (dict(dtype=3, k_stride=(8448, 1024, 64), v=OK + 2048, v_stride=(8448, 1024, 64), k_scale=OK + 4096, v_scale=OK + 4096, ks_stride=(2112, 32, 2),
          vs_stride=(2112, 32, 1)), True),
])
def test_store_into_caches_of_two_layouts(cache, refused):
    without_device()
    c = apart(**cache)
    rc, msg = status("mq_kv_store", FAR, 128, 64, FAR, 128, 64, 1, ctypes.addressof(c), OK, 4, 4, OK, OK, 2, 5, None)
    assert (rc == -1 and "share memory" in msg) if refused else rc not in (-1, 0), msg


def test_verify_into_memory_that_is_read():
    without_device()
    n, rows = 2 * 4 * 4, 2 * 4 * 100 * 4
    inputs = dict(target=OK, draft=OK + rows, drafted=FAR, counts=FAR + 64, uniform=FAR + 128, temperature=FAR + 192)
    outputs = dict(tokens=FAR + 256, accepted=FAR + 320, logprobs=FAR + 384, workspace=FAR + 448)
    size = dict(target=rows, draft=rows * 3 // 4, drafted=24, counts=8, uniform=n, temperature=8, tokens=n, accepted=8, logprobs=n, workspace=9472)

    def verify(**kw):
        a = dict(target=0, ld=100, draft=0, ld_draft=100, dtype=0, drafted=0, counts=0, uniform=0, temperature=0, tokens=0, accepted=0,
                 logprobs=0, batch=2, drafts=3, vocab=100, workspace=0, size=1 << 20)
        a.update(**inputs, **outputs)
        a.update(kw)
        return status("mq_verify_drafts", *a.values(), None)

    assert verify()[0] not in (-1, 0), verify()
    assert verify(draft=None, counts=None, temperature=None)[0] not in (-1, 0)
    for out in outputs:
        for other in [*inputs, *outputs]:
            if other == out:
                continue
            at = {**inputs, **outputs}[other]
            for shift in (0, size[other] // 16 * 16 - 16):  # its first and one of its last bytes
                if shift >= 0:
                    rc, msg = verify(**{out: at + shift})
                    assert rc == -1 and ("shares memory" in msg or "share memory" in msg), (out, other, msg)
