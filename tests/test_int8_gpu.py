"""The int8 products and the per-row quantiser against a 64-bit plain form. The quantiser's integers are
exact; a product's int32 sums are exact, so what is left is fp32 roundings (one of the sum, one per
scale, one per addition) and the output type's."""
import numpy as np
import pytest
import torch

from oracle import serving

import mq

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INF = float("inf")
# half an ulp relative, and half of the smallest step
ROUND = {torch.float32: (U, 2.0 ** -150), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 2.0 ** -134)}
TYPES = list(ROUND)


def np64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def matrix(rng, rows, cols, cuda, ld=None, full=False):
    """An int8 matrix in rows of ld bytes, the bytes between the rows not zero."""
    ld = ld or -(-cols // 16) * 16
    q = rng.integers(-128, 128, size=(rows, ld), dtype=np.int8)
    if full:
        q[:] = -128
    return q[:, :cols], torch.from_numpy(q).to(cuda)[:, :cols]


def scales(rng, n, cuda):
    s = rng.uniform(1e-3, 1e-2, n).astype(np.float32)
    return s, torch.from_numpy(s).to(cuda)


def close(y, ref, size, dtype):
    """|y - ref| within 5 fp32 roundings of `size` (the magnitudes that were added) and one of the output type."""
    rel, tiny = ROUND[dtype]
    err = np.abs(np64(y) - ref)
    bound = 5 * U * size + rel * (np.abs(ref) + 5 * U * size) + tiny
    assert (err <= bound).all(), f"{(err - bound).max()} over at {np.unravel_index((err - bound).argmax(), err.shape)}"


SIZES = [(1, 1, 1), (1, 128, 128), (1, 2048, 2048), (2, 129, 100), (5, 4099, 2048), (16, 640, 1000), (17, 127, 33),
         (31, 300, 4100), (64, 1024, 512), (65, 257, 777), (129, 200, 260), (255, 130, 128), (256, 256, 256),
         (257, 513, 129), (431, 2048, 8192), (700, 260, 640), (1031, 515, 384)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(cuda, m, n, k):
    rng = np.random.default_rng(m * 7 + n + k)
    (xq, dx), (wq, dw) = matrix(rng, m, k, cuda), matrix(rng, n, k, cuda)
    (xs, dxs), (ws, dws) = scales(rng, m, cuda), scales(rng, n, cuda)
    ref = serving.product(xq, xs, wq, ws)
    for dtype in TYPES:
        close(mq.gemm_w8a8(dx, dxs, dw, dws, dtype=dtype), ref, np.abs(ref), dtype)
    assert mq.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 300, 200), (3, 2048, 512), (70, 131, 384), (300, 700, 300), (513, 256, 1024)])
def test_product_bias_add_and_strides(cuda, m, n, k, dtype):
    rng = np.random.default_rng(n)
    (xq, dx), (wq, dw) = matrix(rng, m, k, cuda, ld=(k + 31) // 16 * 16), matrix(rng, n, k, cuda, ld=(k + 63) // 16 * 16)
    (xs, dxs), (ws, dws) = scales(rng, m, cuda), scales(rng, n, cuda)
    bias = rng.standard_normal(n).astype(np.float32)
    wide = torch.randn(m, n + 5, device=cuda).to(dtype)
    before = np64(wide)
    y = wide[:, 2:n + 2]
    mq.gemm_w8a8(dx, dxs, dw, dws, y, bias=torch.from_numpy(bias).to(cuda), add=True)
    prod = serving.product(xq, xs, wq, ws)
    ref = prod + bias + before[:, 2:n + 2]
    close(y, ref, np.abs(prod) + np.abs(bias) + np.abs(before[:, 2:n + 2]), dtype)
    after = np64(wide)
    np.testing.assert_array_equal(after[:, :2], before[:, :2])  # nothing outside y is written
    np.testing.assert_array_equal(after[:, n + 2:], before[:, n + 2:])


@pytest.mark.parametrize("m,f,k", [(1, 1, 64), (1, 8192, 2048), (4, 130, 96), (64, 1000, 512), (100, 64, 2048), (129, 257, 100),
                                   (431, 768, 2048), (600, 1300, 256)])
def test_gate_up(cuda, m, f, k):
    rng = np.random.default_rng(m + f)
    (xq, dx), (wq, dw) = matrix(rng, m, k, cuda), matrix(rng, 2 * f, k, cuda)
    (xs, dxs), (ws, dws) = scales(rng, m, cuda), scales(rng, 2 * f, cuda)
    y = serving.product(xq, xs, wq, ws)
    ref = serving.silu_mul(y)
    for dtype in TYPES:
        a = mq.gate_up_w8a8(dx, dxs, dw, dws, dtype=dtype)
        # a relative error e of g moves silu by at most (1 + |g|) e; exp, the sum and the division add a few ulp
        close(a, ref, np.abs(ref) * (3 + np.abs(y[:, :f])), dtype)
    assert mq.device_status() == 0


@pytest.mark.parametrize("m", [1, 40, 2000])
def test_gate_up_keeps_its_bits_at_large_gates(cuda, m):
    """fp32 outputs with gates from -104 to 90: within six steps of 2^-23 (2^t two, the reciprocal one, the sum and the
    products one half each), however large the gate; below -87.3, where e^g is no normal number, between 0 and the value."""
    f, k = 777, 32
    gate = np.linspace(-104, 90, f).astype(np.float32)
    xq, wq = np.zeros((m, k), np.int8), np.zeros((2 * f, k), np.int8)
    xq[:, 3], wq[:, 3] = 1, 1
    ws = np.concatenate([gate, np.full(f, 1, np.float32)])
    a = mq.gate_up_w8a8(*(torch.from_numpy(v).to(cuda) for v in (xq, np.ones(m, np.float32), wq, ws)), dtype=torch.float32)
    ref = serving.silu_mul(ws.astype(np.float64))
    high, low = gate >= -87.3, np64(a)[:, gate < -87.3]
    ratio = np.abs(np64(a) - ref)[:, high] / np.maximum(6 * 2.0 ** -23 * np.abs(ref), 1e-300)[high]
    assert ratio.max() <= 1, f"{ratio.max()} of the bound at a gate of {gate[high][ratio.max(0).argmax()]}"
    assert (low <= 0).all() and (low >= 1.001 * ref[gate < -87.3]).all()


def test_gate_up_of_infinite_gates(cuda):
    """silu(+inf) u = inf u, silu(-inf) is 0 times infinity: NaN, as the formula; its neighbours stay."""
    q = torch.ones(1, 16, dtype=torch.int8, device=cuda)
    w = torch.ones(6, 16, dtype=torch.int8, device=cuda)
    ws = torch.tensor([INF, 1e37, -1e37, 2, 2, 2], device=cuda)
    for dtype in (torch.float32, torch.bfloat16):
        a = mq.gate_up_w8a8(q, torch.ones(1, device=cuda), w, ws, dtype=dtype)
        assert a[0].tolist() == [INF, INF, 0], a
    ws[0] = -INF
    assert mq.gate_up_w8a8(q, torch.ones(1, device=cuda), w, ws)[0, 0].isnan()


def test_largest_sums(cuda):
    """k at the limit of the int32 sums with every product at its largest."""
    rng = np.random.default_rng(0)
    k = 131071
    (xq, dx), (wq, dw) = matrix(rng, 2, k, cuda, full=True), matrix(rng, 130, k, cuda, full=True)
    y = mq.gemm_w8a8(dx, torch.ones(2, device=cuda), dw, torch.ones(130, device=cuda), dtype=torch.float32)
    assert (np64(y) == float(np.float32(128 * 128 * k))).all()


def test_products_repeat_exactly_and_follow_their_stream(cuda):
    rng = np.random.default_rng(1)
    (_, dx), (_, dw) = matrix(rng, 37, 4096, cuda), matrix(rng, 2048, 4096, cuda)
    (_, dxs), (_, dws) = scales(rng, 37, cuda), scales(rng, 2048, cuda)
    first = mq.gemm_w8a8(dx, dxs, dw, dws, dtype=torch.float32)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q = torch.zeros_like(dx)
        q.copy_(dx)
        again = [mq.gemm_w8a8(q, dxs, dw, dws, dtype=torch.float32) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(a, first) for a in again)


def test_product_of_a_nan_token_is_nan_there_alone(cuda):
    x = torch.randn(3, 256, device=cuda)
    x[1, 7] = float("inf")
    q, s = mq.quantize_s8(x)
    w, ws = mq.quantize_s8(torch.randn(40, 256, device=cuda))
    y = mq.gemm_w8a8(q, s, w, ws)
    assert y[1].isnan().all() and y[[0, 2]].isfinite().all()


def test_no_tokens(cuda):
    w, ws = mq.quantize_s8(torch.randn(40, 256, device=cuda))
    q, s = mq.quantize_s8(torch.empty(0, 256, device=cuda))
    assert mq.gemm_w8a8(q, s, w, ws).shape == (0, 40) and mq.gate_up_w8a8(q, s, w, ws).shape == (0, 20)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (2, 256), (5, 1000), (4, 2048), (1, 12288), (3, 16385), (2, 32768)])
def test_quantize(cuda, rows, cols, dtype):
    rng = np.random.default_rng(cols)
    x = torch.from_numpy((rng.standard_normal((rows, cols)) * np.exp(rng.uniform(-5, 5, (rows, 1)))).astype(np.float32)).to(cuda).to(dtype)
    if rows > 2:
        x[0] = 0
        x[1, 0] = float("nan")
    q, s = mq.quantize_s8(x)
    rq, rs = serving.quantize_s8(x.float().cpu().numpy())
    np.testing.assert_array_equal(q.cpu().numpy(), rq)
    np.testing.assert_array_equal(s.cpu().numpy(), rs)


def test_quantize_tiny_and_huge_rows_and_strides(cuda):
    x = torch.randn(6, 40, device=cuda)
    x[0] *= 1e-38
    x[1] *= 1e-44  # subnormal
    x[2] *= 1e38 / x[2].abs().max()
    wide = torch.zeros(6, 51, device=cuda)
    wide[:, 3:43] = x
    q, s = mq.quantize_s8(wide[:, 3:43])
    rq, rs = serving.quantize_s8(x.cpu().numpy())
    np.testing.assert_array_equal(q.cpu().numpy(), rq)
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    assert (q.abs().max(-1).values[[0, 2, 3]] == 127).all()


def test_refusals(cuda):
    w, ws = mq.quantize_s8(torch.randn(40, 256, device=cuda))
    q, s = mq.quantize_s8(torch.randn(3, 256, device=cuda))
    with pytest.raises(mq.MQError, match="dtype"):
        mq.gemm_w8a8(q.float(), s, w, ws)
    with pytest.raises(mq.MQError, match="rows of 256"):
        mq.gemm_w8a8(q[:, :255].contiguous()[:, :240], s, w, ws)
    with pytest.raises(mq.MQError, match="ws: has"):
        mq.gemm_w8a8(q, s, w, ws[:-1])
    with pytest.raises(mq.MQError, match="16"):
        mq.gemm_w8a8(q[:, :250].contiguous(), s, w[:, :250], ws)
    with pytest.raises(mq.MQError, match="gate and up"):
        mq.gate_up_w8a8(q, s, w[:39], ws[:39])
    with pytest.raises(mq.MQError, match="add"):
        mq.gemm_w8a8(q, s, w, ws, add=True)
    with pytest.raises(mq.MQError, match="contiguous"):
        mq.quantize_s8(torch.randn(8, 6, device=cuda).T)
