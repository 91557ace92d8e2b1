"""The norms around a block against a 64-bit plain form. fp32 error: a row's sum of squares takes at most 64
additions in a thread and 10 across threads, half of which (a square root) reaches the result, then the
root and the products: below 60 roundings of 2^-24, and the output type's own."""
import numpy as np
import pytest
import torch

from oracle import serving

import mq

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROUND = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
TYPES = list(ROUND)
COLS = [1, 7, 8, 100, 256, 264, 1000, 2048, 4095, 4096, 8192, 12288, 20000, 32768]


def np64(t):
    return None if t is None else t.detach().cpu().to(torch.float64).numpy()


def rand(rng, rows, cols, dtype, cuda, pad=0):
    x = rng.standard_normal((rows, cols + pad)).astype(np.float32)
    x[:, :: max(1, cols // 5)] *= 12
    return torch.from_numpy(x).to(cuda).to(dtype)[:, pad:]


def within(got, ref, bound, dtype):
    err = np.abs(np64(got) - ref)
    limit = bound + ROUND[dtype] * (np.abs(ref) + bound) + TINY[dtype]
    assert (err <= limit).all(), f"{(err / limit).max()} of the bound"


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype,out", [(torch.float32, torch.float16), (torch.float16, torch.float32),
                                       (torch.bfloat16, torch.bfloat16)])
def test_pre_norm(cuda, cols, dtype, out):
    rng = np.random.default_rng(cols)
    for rows, pad in ((1, 0), (5, 0), (9, 3)):
        x, w = rand(rng, rows, cols, dtype, cuda, pad), rand(rng, 1, cols, dtype, cuda)[0]
        ref = serving.rms_norm(np64(x), np64(w), 1e-5)
        h = mq.pre_norm(x, w.contiguous(), 1e-5, dtype=out)
        within(h, ref, 60 * U * np.abs(ref), out)


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", TYPES)
def test_pre_norm_s8(cuda, cols, dtype):
    rng = np.random.default_rng(cols)
    x, w = rand(rng, 6, cols, dtype, cuda), rand(rng, 1, cols, torch.float32, cuda)[0].contiguous()
    if cols > 8:
        x[1] = 0
        x[2, 3] = float("nan")
        x[3, 5] = float("-inf")
    q, s = mq.pre_norm_s8(x, w, 1e-6)
    v = x.float().cpu().numpy() * w.cpu().numpy()
    with np.errstate(all="ignore"):
        rq, rs = serving.quantize_s8(v)
        inv = 1 / np.sqrt((np64(x) ** 2).mean(-1) + 1e-6)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)  # the statistics cancel from the integers
    np.testing.assert_allclose(s.cpu().numpy(), rs * inv, rtol=60 * U)


CASES = [(1, 4096, 1, True), (13, 1000, 13, True), (12, 264, 4, True), (6, 2048, None, True), (6, 2048, 1, False),
         (3, 7, 3, True), (4, 20000, 2, True), (130, 100, 130, False), (2, 1, 1, True)]


@pytest.mark.parametrize("rows,cols,gates,normed", CASES)
@pytest.mark.parametrize("y_t,r_t,h_t", [(torch.bfloat16, torch.bfloat16, torch.bfloat16),
                                         (torch.float16, torch.float32, torch.float16),
                                         (torch.float32, torch.bfloat16, torch.float32)])
def test_post_norm(cuda, rows, cols, gates, normed, y_t, r_t, h_t):
    rng = np.random.default_rng(rows + cols)
    y, res = rand(rng, rows, cols, y_t, cuda, 1 if rows == 13 else 0), rand(rng, rows, cols, r_t, cuda)
    w = rand(rng, 1, cols, y_t, cuda)[0].contiguous() if normed else None
    nw = rand(rng, 1, cols, torch.float32, cuda)[0].contiguous()
    gate = rand(rng, gates, cols, h_t, cuda) if gates else None
    ref, added = serving.post_norm(np64(y), np64(w), np64(res), np64(gate), 0.3, 1e-6)
    err = 60 * U * added + U * np.abs(ref)  # of the sum, before it is stored
    h_ref = serving.rms_norm(ref, np64(nw), 1e-5)
    inv = 1 / np.sqrt((ref * ref).mean(-1, keepdims=True) + 1e-5)
    # the sum's error through the norm: its own, and the row's through the root
    share = np.sqrt((err * err).sum(-1, keepdims=True) / np.maximum((ref * ref).sum(-1, keepdims=True), 1e-30))
    h_err = np.abs(np64(nw)) * inv * err + np.abs(h_ref) * (60 * U + share)
    kept = res.clone()
    out, h = mq.post_norm(y, w, res, nw, gate=gate, scale=0.3, eps=1e-6, next_eps=1e-5, dtype=h_t)
    within(out, ref, err, r_t)
    within(h, h_ref, h_err, h_t)
    assert torch.equal(res, kept)
    # in place on the residual, without the norm that follows, and quantised
    same, none = mq.post_norm(y, w, res, gate=gate, scale=0.3, eps=1e-6, out=res)
    assert same is res and none is None and torch.equal(res, out)
    out8, q, s = mq.post_norm_s8(y, w, kept, nw, gate=gate, scale=0.3, eps=1e-6, next_eps=1e-5)
    assert torch.equal(out8, out)
    got, step = np64(q) * np64(s)[:, None], np64(s)[:, None]
    assert (np.abs(got - h_ref) <= step * (0.5 + 1e-4) + h_err + 128 * 60 * U * step).all()


MANY = [(601, 256, 0), (1500, 264, 0), (700, 777, 0), (700, 1000, 0), (3001, 1001, 0), (640, 2048, 8), (1200, 4096, 0),
        (600, 4096, 1), (640, 5003, 0), (600, 8191, 3), (620, 8192, 0), (600, 8200, 0)]


@pytest.mark.parametrize("rows,cols,pad", MANY)
@pytest.mark.parametrize("y_t,r_t,w_t,h_t", [(torch.bfloat16, torch.bfloat16, torch.bfloat16, torch.bfloat16),
                                             (torch.float16, torch.float32, torch.float32, torch.float16),
                                             (torch.float32, torch.float32, torch.float32, torch.bfloat16),
                                             (torch.bfloat16, torch.float16, torch.float32, torch.float32)])
def test_many_rows(cuda, rows, cols, pad, y_t, r_t, w_t, h_t):
    """Row counts at which the rows stream through persistent CTAs, aligned and not, all outputs."""
    rng = np.random.default_rng(rows + cols)
    y, res = rand(rng, rows, cols, y_t, cuda, pad), rand(rng, rows, cols, r_t, cuda, pad)
    w, nw = rand(rng, 1, cols, w_t, cuda)[0].contiguous(), rand(rng, 1, cols, w_t, cuda)[0].contiguous()
    h_ref = serving.rms_norm(np64(y), np64(nw), 1e-6)
    within(mq.pre_norm(y, nw, 1e-6, dtype=h_t), h_ref, 60 * U * np.abs(h_ref), h_t)
    v = y.float().cpu().numpy() * nw.float().cpu().numpy()
    q, s = mq.pre_norm_s8(y, nw, 1e-6)
    np.testing.assert_array_equal(q.cpu().numpy(), serving.quantize_s8(v)[0])
    q, s = mq.quantize_s8(y)
    rq, rs = serving.quantize_s8(y.float().cpu().numpy())
    np.testing.assert_array_equal(q.cpu().numpy(), rq)
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    groups = next(g for g in (7, 5, 3, 2, 1) if rows % g == 0)
    gate = rand(rng, groups, cols, w_t, cuda)
    ref, added = serving.post_norm(np64(y), np64(w), np64(res), np64(gate), 0.3, 1e-6)
    err = 60 * U * added + U * np.abs(ref)
    h_ref = serving.rms_norm(ref, np64(nw), 1e-6)
    inv = 1 / np.sqrt((ref * ref).mean(-1, keepdims=True) + 1e-6)
    share = np.sqrt((err * err).sum(-1, keepdims=True) / (ref * ref).sum(-1, keepdims=True))
    h_err = np.abs(np64(nw)) * inv * err + np.abs(h_ref) * (60 * U + share)
    out, h = mq.post_norm(y, w, res, nw, gate=gate, scale=0.3, eps=1e-6, dtype=h_t)
    within(out, ref, err, r_t)
    within(h, h_ref, h_err, h_t)
    out8, q, s = mq.post_norm_s8(y, w, res, nw, gate=gate, scale=0.3, eps=1e-6)
    assert torch.equal(out8, out)
    got, step = np64(q) * np64(s)[:, None], np64(s)[:, None]
    assert (np.abs(got - h_ref) <= step * (0.5 + 1e-4) + h_err + 128 * 60 * U * step).all()
    same, _ = mq.post_norm(y, w, res, gate=gate, scale=0.3, eps=1e-6, out=res)  # in place, nothing behind it
    assert same is res and torch.equal(res, out)
    assert mq.device_status() == 0


@pytest.mark.parametrize("rows,cols", [(5, 264), (640, 2048), (640, 1001)])
def test_post_norm_without_h_has_no_use_for_next_w(cuda, rows, cols):
    """The C entry with h NULL writes the same, a next_w given or not, whatever type is said of it."""
    y, r = torch.randn(rows, cols, device=cuda).bfloat16(), torch.randn(rows, cols, device=cuda).bfloat16()
    w, next_w = torch.rand(cols, device=cuda).bfloat16(), torch.full((cols,), float("nan"), device=cuda)

    def call(next_w, next_dtype):
        out = torch.empty_like(r)
        mq.lib.call("mq_post_norm", y.data_ptr(), 2, cols, w.data_ptr(), 2, 1e-6, r.data_ptr(), 2, cols, None, 0, cols, 1,
                    0.7, out.data_ptr(), cols, next_w, next_dtype, 1e-6, None, 0, cols, None, rows, cols,
                    torch.cuda.current_stream().cuda_stream)
        return out

    want = call(None, 0)
    assert torch.equal(call(next_w.data_ptr(), 0), want) and torch.equal(call(next_w.data_ptr(), 77), want)
    assert torch.equal(mq.post_norm(y, w, r, scale=0.7)[0], want) and mq.device_status() == 0


def test_many_rows_propagate_nan_in_its_row_alone(cuda):
    for cols in (1001, 4096):
        x, w = torch.randn(900, cols, device=cuda), torch.ones(cols, device=cuda)
        x[700, cols - 1] = float("nan")
        x[3, 0] = float("inf")
        bad = torch.zeros(900, dtype=torch.bool, device=cuda)
        bad[[3, 700]] = True
        q, s = mq.pre_norm_s8(x, w)
        assert s[bad].isnan().all() and s[~bad].isfinite().all() and (q[bad] == 0).all()
        h = mq.pre_norm(x, w)
        assert h[700].isnan().all() and h[~bad].isfinite().all()


def test_post_norm_gate_of_one_row_is_a_vector(cuda):
    y, r, w = torch.randn(4, 64, device=cuda), torch.randn(4, 64, device=cuda), torch.rand(64, device=cuda)
    g = torch.randn(64, device=cuda)
    a, b = mq.post_norm(y, w, r, w, gate=g), mq.post_norm(y, w, r, w, gate=g.expand(4, 64).contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_norms_propagate_nan_in_its_row_alone(cuda):
    x, w = torch.randn(5, 512, device=cuda), torch.ones(512, device=cuda)
    x[2, 100] = float("nan")
    h = mq.pre_norm(x, w)
    out, hh = mq.post_norm(x, w, torch.zeros_like(x), w)
    for t in (h, out, hh):
        assert t[2].isnan().all() and t[[0, 1, 3, 4]].isfinite().all()


def test_norms_of_no_rows_and_three_dimensions(cuda):
    w = torch.ones(64, device=cuda)
    assert mq.pre_norm(torch.empty(0, 64, device=cuda), w).shape == (0, 64)
    x = torch.randn(2, 3, 64, device=cuda)
    assert torch.equal(mq.pre_norm(x, w).view(6, 64), mq.pre_norm(x.view(6, 64), w))
    z = torch.zeros(1, 64, device=cuda)
    assert (mq.pre_norm(z, w) == 0).all()


def test_norm_refusals(cuda):
    x, w = torch.randn(4, 64, device=cuda), torch.ones(64, device=cuda)
    with pytest.raises(mq.MQError, match="w: has"):
        mq.pre_norm(x, w[:63])
    with pytest.raises(mq.MQError, match="contiguous"):
        mq.pre_norm(x.T, w[:4])
    with pytest.raises(mq.MQError, match="do not divide"):
        mq.post_norm(x, w, x, gate=torch.ones(3, 64, device=cuda))
    with pytest.raises(mq.MQError, match="dtype"):
        mq.post_norm(x, w, x, out=torch.empty(4, 64, device=cuda, dtype=torch.float16))
    with pytest.raises(mq.MQError, match="next_w"):
        mq.post_norm(x, w, x, h=torch.empty(4, 64, device=cuda))
    with pytest.raises(mq.MQError, match="above 32768"):
        mq.pre_norm(torch.randn(1, 32769, device=cuda), torch.ones(32769, device=cuda))
