"""Plain 64-bit forms of the int8 products, the norms around a block and the beam-search step (numpy)."""
import numpy as np

F32, F64 = np.float32, np.float64


def quantize_s8(x):
    """(q, s) of fp32 rows with the operator's own fp32 operations, so the integers are to be equal: a the
    largest |x|, q = rint(x * (127 / a)), s = a / 127; a row that is not finite gives 0 and NaN."""
    x = np.asarray(x, F32)
    a = np.abs(x).max(-1)
    bad = ~np.isfinite(x).all(-1)
    with np.errstate(all="ignore"):
        lift = np.where(a < F32(1e-30), F32(2.0 ** 80), F32(1))
        f = np.where((a == 0) | bad, F32(0), F32(127) / (a * lift))
        q = np.rint((x * lift[..., None]) * f[..., None])
    q[bad] = 0
    return q.astype(np.int8), np.where(bad, F32(np.nan), a / F32(127))


def product(xq, xs, wq, ws, bias=None):
    """xs * ws * (xq . wq^T) + bias in fp64 (the sums of int8 products are exact there)."""
    y = xq.astype(F64) @ wq.astype(F64).T * xs.astype(F64)[:, None] * ws.astype(F64)
    return y if bias is None else y + bias.astype(F64)


def silu_mul(y):
    g, u = np.split(y, 2, -1)
    return g / (1 + np.exp(-g)) * u


def rms_norm(x, w, eps):
    x = np.asarray(x, F64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, F64)


def post_norm(y, w, residual, gate, scale, eps):
    """residual + scale * gate * norm(y; w), and the size of the added term (for the error bound)."""
    n = np.asarray(y, F64) if w is None else rms_norm(y, w, eps)
    if gate is not None:
        n = n * np.repeat(np.asarray(gate, F64), n.shape[0] // gate.shape[0], 0)
    return np.asarray(residual, F64) + scale * n, np.abs(scale * n)


def beam_scores(logits, scores, finished, eos):
    """The score of every candidate in fp64: [batch, beams, vocab]."""
    z, c = np.asarray(logits, F64), np.asarray(scores, F64)
    z = z.reshape(*c.shape, -1)
    with np.errstate(all="ignore"):
        top = z.max(-1, keepdims=True)
        lse = top + np.log(np.exp(z - top).sum(-1, keepdims=True))
        out = c[..., None] + (z - lse)
    out[~np.isfinite(lse[..., 0]) | ~(c > -np.inf)] = -np.inf
    if finished is not None:
        done = np.asarray(finished, bool)
        out[done] = -np.inf
        out[done, eos] = c[done]
    return out


def beam_select(cand):
    """(scores, parents, tokens): the `beams` best of each request, the lowest flat index among equals."""
    batch, beams, vocab = cand.shape
    flat = cand.reshape(batch, -1)
    order = np.argsort(-flat, -1, kind="stable")[:, :beams]
    return np.take_along_axis(flat, order, -1), order // vocab, order % vocab
