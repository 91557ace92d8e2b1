"""The int8 products where a CTA (or a pair) works on several tiles, where pairs share a tile's k, and where pairs
add into y: sizes at which the cost rule takes those kernels by a clear margin. The reference is formed on the GPU
in fp64, in which the sums are exact; what is left is roundings, counted as in the other product tests."""
import pytest
import torch

import mq

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROUND = {torch.float32: (U, 2.0 ** -150), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 2.0 ** -134)}


def operands(m, rows, k, cuda, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)

    def matrix(r):
        q = mq.int8_rows(r, k, cuda)
        q.copy_(torch.randint(-128, 128, (r, k), generator=g, device=cuda, dtype=torch.int8))
        return q

    def scales(n, size):
        return (torch.rand(n, generator=g, device=cuda) + 0.5) * size

    # sums of some 74^2 sqrt(k): gates of a usual size
    return matrix(m), scales(m, 1e-3), matrix(rows), scales(rows, 3e-1 / k ** 0.5), scales(rows, 1.0) - 1


def product(xq, xs, wq, ws):
    return (xq.double() @ wq.double().T) * xs.double()[:, None] * ws.double()


def close(y, ref, error):
    rel, tiny = ROUND[y.dtype]
    over = (y.double() - ref).abs() - (error + rel * (ref.abs() + error) + tiny)
    at = divmod(int(over.argmax()), y.shape[1])
    assert float(over.max()) <= 0, f"{float(over.max())} over at {at}"


def output(m, n, dtype, aligned, cuda):
    """y, and the tensor around it that must keep its zeros."""
    wide = torch.zeros(m, n + 21, dtype=dtype, device=cuda)
    if aligned:
        wide = torch.zeros(m, (n + 31) // 16 * 16, dtype=dtype, device=cuda)
    y = wide[:, :n] if aligned else wide[:, 3:n + 3]
    return y, wide


def check_around(wide, y):
    y.zero_()
    assert not wide.any() and mq.device_status() == 0


@pytest.mark.parametrize("m,n,k,dtype,aligned", [
    (3, 40007, 300, torch.float32, True), (3, 40007, 300, torch.float16, False),       # streaming, 313 tiles
    (70, 40007, 300, torch.bfloat16, True), (70, 40007, 300, torch.float32, False),
    (2500, 3000, 260, torch.float16, True), (2500, 3001, 260, torch.bfloat16, False),  # pairs, 120 tiles, two bands
    (2500, 5000, 516, torch.float32, True), (2500, 5000, 516, torch.float16, False),   # 200 tiles
    (1024, 2048, 16385, torch.float32, True), (1024, 2048, 16385, torch.bfloat16, True)])  # pairs that share k
@pytest.mark.parametrize("bias", [False, True])
def test_product_tiles(cuda, m, n, k, dtype, aligned, bias):
    xq, xs, wq, ws, b = operands(m, n, k, cuda, n + k)
    y, wide = output(m, n, dtype, aligned, cuda)
    ref = product(xq, xs, wq, ws)
    size = ref.abs() + (b.double().abs() if bias else 0)
    mq.gemm_w8a8(xq, xs, wq, ws, y, bias=b if bias else None)
    close(y, ref + b.double() if bias else ref, 5 * U * size)
    check_around(wide, y)


@pytest.mark.parametrize("m,f,k,dtype,aligned", [
    (3, 30000, 300, torch.float16, True), (70, 30000, 300, torch.float32, False),      # streaming, 235 and 470 tiles
    (2500, 3000, 900, torch.bfloat16, True), (2500, 3000, 4100, torch.float32, True),  # pairs, 240 tiles
    (2500, 3001, 4100, torch.float16, False),
    (1024, 1024, 16384, torch.float16, True), (1024, 1024, 16384, torch.float32, True),  # pairs that share k
    (1024, 1024, 131071, torch.bfloat16, False)])
def test_gate_up_tiles(cuda, m, f, k, dtype, aligned):
    xq, xs, wq, ws, _ = operands(m, 2 * f, k, cuda, f + k)
    a, wide = output(m, f, dtype, aligned, cuda)
    g, u = product(xq, xs, wq, ws).split(f, 1)
    ref = g * torch.sigmoid(g) * u
    mq.gate_up_w8a8(xq, xs, wq, ws, a)
    # silu's 6 * 2^-23; three roundings each of g, which moves silu by at most 1 + |g| times as much, and of u
    close(a, ref, ref.abs() * U * (12 + 3 * (1 + g.abs()) + 3))
    check_around(wide, a)


@pytest.mark.parametrize("m,n,k,dtype", [(2500, 3001, 260, torch.float16), (2500, 3001, 260, torch.bfloat16),
                                         (2560, 18944, 8192, torch.float32)])
def test_add_of_pairs(cuda, m, n, k, dtype):
    xq, xs, wq, ws, b = operands(m, n, k, cuda, k)
    y, wide = output(m, n, dtype, False, cuda)
    y.copy_(torch.randn(m, n, device=cuda))
    before = y.double()
    mq.gemm_w8a8(xq, xs, wq, ws, y, bias=b, add=True)
    ref = product(xq, xs, wq, ws)
    close(y, ref + b.double() + before, 5 * U * (ref.abs() + b.double().abs() + before.abs()))
    check_around(wide, y)
