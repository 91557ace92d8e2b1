"""The paged cache and the attention over it, against the oracle in 64 bits.

Bound of an output, from the roundings on its way (u = eps / 2 of a type): the output's own, u |o|; the weights', u of the
cache's type (int8: fp16) each, in the sum over the values and in the sum of weights, 2 u sum_j p_j |v_j|; the scores', whose
absolute error e in the exponent changes a weight by a factor 1 + e, in both sums: e <= (dim + 16) 2^-23 times the
largest scale sum_d |q_d k_jd| (fp32 products and sums in any order, and the scaling), and int8's q, exact down to 2^-25 of its
largest, 2^-25 max|q| scale sum_d |k_jd|; 2^-19 for the exponentials, the rescaling and the division.
A weight of an fp16 product below 2^-14 is subnormal there: its error is up to 2^-25 absolute, not relative to it. The largest
weight is 1 or more there, so in units of the sums that is 2^-25 max_j p_j times each |v_j|; int8's weights are p_j t_j, with t_j the
value's scale, and meet the integers v_j / t_j: 2^-25 max_j (p_j t_j) sum_j |v_j| / t_j. It counts where the keys that have the weight
have values near 0.
bf16 rows of more than 16 per kv head meet an int8 cache as fp16 operands, integer * (scale / the largest of 32 keys): the ratio
and the product are rounded, 2^-11 each, so scores carry 2^-10 (times 1 + 2^-12) of scale sum_d |q_d k_jd| more and values 2^-10 of
themselves; a ratio below 2^-14 is off by up to 2^-25, an integer times it by 127 times that and 2^-25 of its own product, below
2^-17 of the largest scale: 2^-17 kmax scale sum_d |q_d| in a score, 2^-17 vmax in a value."""
import numpy as np
import pytest
import torch

from oracle import paged, serving

import mq

pytestmark = pytest.mark.gpu
F16, BF16, S8, F32 = torch.float16, torch.bfloat16, torch.int8, torch.float32
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}


def host(t):
    return t.double().cpu().numpy()


class Batch:
    """Sequences of (new tokens, length), their table and starts. The pool's other positions hold NaN (int8: NaN scales),
    the table's other entries nonsense; order "position" lays a page's rows out position by position."""

    def __init__(self, cuda, sizes, kv_heads, page, dim, dtype, order="head", seed=0, spare=2, gap=0, scale_v=1.0):
        self.g = torch.Generator(device=cuda).manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.sizes, self.cuda, self.dtype = sizes, cuda, dtype
        need = [-(-max(length, 0) // page) for _, length in sizes]
        pages = sum(need) + spare
        shape = (pages, kv_heads, page, dim) if order == "head" else (pages, page, kv_heads, dim)
        self.ints = dtype == S8

        def pool():
            if self.ints:
                t = torch.randint(-128, 128, shape, generator=self.g, device=cuda, dtype=torch.int32).to(S8)
            else:
                t = torch.full(shape, float("nan"), device=cuda, dtype=dtype)
            return t if order == "head" else t.transpose(1, 2)

        self.k, self.v = pool(), pool()
        self.scales = [torch.full((pages, kv_heads, page), float("nan"), device=cuda) for _ in range(2)] if self.ints else [None, None]
        ids = rng.permutation(pages)
        table = np.full((len(sizes), max(max(need), 1) + 1), -7, np.int32)
        table[:, -1] = 1 << 30
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = ids[at:at + n]
            at += n
        self.np_table = table
        self.table = torch.from_numpy(table).to(cuda)
        self.lengths = torch.tensor([length for _, length in sizes], dtype=torch.int32, device=cuda)
        starts = [gap]
        for n, _ in sizes:
            starts.append(starts[-1] + n)
        self.np_starts, self.tokens = starts, starts[-1] + gap
        self.starts = torch.tensor(starts, dtype=torch.int32, device=cuda)
        self.page, self.kv_heads, self.dim = page, kv_heads, dim
        for b, (_, length) in enumerate(sizes):
            if length <= 0:
                continue
            j = torch.arange(length, device=cuda)
            of, row = self.table[b][j // page].long(), j % page
            for t, sc in zip((self.k, self.v), self.scales):
                x = torch.randn(length, kv_heads, dim, generator=self.g, device=cuda)
                if self.ints:
                    t[of, :, row] = (x * 40).round().clamp(-127, 127).to(S8)
                    sc[of, :, row] = torch.rand(length, kv_heads, generator=self.g, device=cuda) * 0.05 + 0.001
                else:
                    t[of, :, row] = x.to(dtype)
        if self.ints:
            self.scales[1] *= scale_v

    def cache(self):
        return mq.PagedCache(self.k, self.v, *self.scales)

    def where(self):
        return self.table, self.lengths, self.starts

    def held(self, b, length):
        """keys, values [kv_heads, length, dim] in 64 bits, and their scales [kv_heads, length] (None: 16-bit)."""
        out, steps = [], []
        for t, sc in zip((self.k, self.v), self.scales):
            j = torch.arange(max(length, 0), device=self.cuda)
            of, row = self.table[b][j // self.page].long(), j % self.page
            x = t[of, :, row].double()
            if self.ints:
                x = x * sc[of, :, row].double()[..., None]
                steps.append(host(sc[of, :, row].transpose(0, 1)))
            out.append(host(x.transpose(0, 1)))
        return *out, steps or None

    def check(self, out, q, scale, window=0):
        got, qh = host(out), host(q)
        unit, unit_w = UNIT[q.dtype], UNIT[F16 if self.ints else self.dtype]
        for b, (n, length) in enumerate(self.sizes):
            if n == 0:
                continue
            s0 = self.np_starts[b]
            keys, values, steps = self.held(b, length)
            rows = qh[s0:s0 + n]
            ref, size, tiny = paged.attention(rows, keys, values, range(length - n, length), scale, window, steps and steps[1])
            group = rows.shape[1] // self.kv_heads
            if keys.shape[1]:
                big = scale * np.einsum("thd,hjd->thj", np.abs(rows), np.repeat(np.abs(keys), group, 0)).max(-1)
                small = 2.0 ** -25 * scale * np.abs(rows).max(-1) * np.repeat(np.abs(keys).sum(-1).max(-1), group)[None] if self.ints else 0
            else:
                big = small = np.zeros(rows.shape[:2])
            e = (self.dim + 16) * 2.0 ** -23 * big + small
            folded = 0
            if self.ints and q.dtype == BF16 and n * group > 16 and keys.shape[1]:
                kmax, vmax = (np.repeat(s.max(-1), group)[None] for s in steps)
                e = e + 1.01 * 2.0 ** -10 * big + 2.0 ** -17 * kmax * scale * np.abs(rows).sum(-1)
                folded = 1.01 * 2.0 ** -10 * size + 2.0 ** -17 * vmax[..., None]
            bound = unit * np.abs(ref) + (2 * unit_w + 2 * e + 2.0 ** -19)[..., None] * size + 2.0 ** -24 * (q.dtype == F16) + \
                2.0 ** -25 * tiny * (self.dtype != BF16) + folded
            bad = ~(np.abs(got[s0:s0 + n] - ref) <= bound)
            assert not bad.any(), (b, n, length, int(bad.sum()), np.argwhere(bad)[:3], np.nanmax(np.abs(got[s0:s0 + n] - ref) / bound))


def attend(batch, heads, dtype, scale=None, window=0, max_new=0, **kw):
    q = (torch.randn(batch.tokens, heads, batch.dim, generator=batch.g, device=batch.cuda) * 2).to(dtype)
    out = torch.full_like(q, 7.0)
    mq.device_status()
    got = mq.paged_attention(q, batch.cache(), *batch.where(), out=out, scale=scale, window=window, max_new=max_new, **kw)
    assert mq.device_status() == 0
    assert got is out
    lo, hi = batch.np_starts[0], batch.np_starts[-1]
    assert (out[:lo] == 7).all() and (out[hi:] == 7).all(), "rows of no sequence are left as they are"
    batch.check(out, q, batch.dim ** -0.5 if scale is None else scale, window)
    return q, out


CACHES = [(F16, F16), (BF16, BF16), (S8, F16), (S8, BF16)]
ONE = [(1, 1), (1, 2), (1, 63), (1, 64), (1, 65), (1, 333)]


@pytest.mark.parametrize("cache,x", CACHES)
@pytest.mark.parametrize("kv_heads,group,page,dim,order", [(1, 1, 16, 64, "head"), (2, 4, 16, 128, "position"), (3, 5, 64, 96, "head"),
                                                         (8, 8, 128, 64, "position"), (1, 16, 256, 128, "head"), (2, 3, 32, 16, "head")])
def test_one_token_each(cuda, cache, x, kv_heads, group, page, dim, order):
    attend(Batch(cuda, ONE, kv_heads, page, dim, cache, order, gap=2), kv_heads * group, x)


@pytest.mark.parametrize("cache,x", CACHES)
def test_one_token_each_without_starts(cuda, cache, x):
    batch = Batch(cuda, ONE, 2, 16, 64, cache)
    q = torch.randn(len(ONE), 8, 64, generator=batch.g, device=cuda).to(x)
    out = mq.paged_attention(q, batch.cache(), batch.table, batch.lengths)
    batch.check(out, q, 64 ** -0.5)


FEW = [(5, 5), (1, 300), (0, 40), (3, 64), (7, 65), (4, 2), (1, 0), (6, 200)]


@pytest.mark.parametrize("cache,x", CACHES)
@pytest.mark.parametrize("kv_heads,group,page,dim,max_new", [(2, 2, 16, 128, 7), (1, 4, 32, 128, 7), (2, 8, 64, 64, 7), (2, 1, 16, 112, 0),
                                                           (1, 9, 16, 128, 7)])
def test_few_tokens(cuda, cache, x, kv_heads, group, page, dim, max_new):
    attend(Batch(cuda, FEW, kv_heads, page, dim, cache, gap=1), kv_heads * group, x, max_new=max_new)


@pytest.mark.parametrize("cache,x", CACHES)
@pytest.mark.parametrize("window", [1, 2, 64, 100])
def test_window(cuda, cache, x, window):
    attend(Batch(cuda, FEW + [(40, 400), (129, 129)], 2, 16, 64, cache), 8, x, window=window)


MANY = [(65, 65), (1, 77), (128, 128), (129, 700), (0, 9), (300, 300), (17, 17)]


@pytest.mark.parametrize("cache,x", CACHES)
@pytest.mark.parametrize("kv_heads,group,page,dim,order", [(1, 1, 16, 64, "head"), (2, 4, 32, 128, "position"), (2, 3, 128, 96, "head"),
                                                         (1, 8, 256, 128, "head"), (2, 5, 64, 32, "position")])
def test_many_tokens(cuda, cache, x, kv_heads, group, page, dim, order):
    attend(Batch(cuda, MANY, kv_heads, page, dim, cache, order, gap=3), kv_heads * group, x)


@pytest.mark.parametrize("cache,x", CACHES)
def test_more_heads_than_a_tile_of_rows(cuda, cache, x):
    attend(Batch(cuda, [(1, 70), (3, 90)], 1, 16, 64, cache), 71, x)


@pytest.mark.parametrize("cache,x", CACHES)
@pytest.mark.parametrize("dim", [64, 128])
def test_long_context_split_over_the_gpu(cuda, cache, x, dim):
    attend(Batch(cuda, [(1, 20011)], 1, 64, dim, cache), 4, x)
    attend(Batch(cuda, [(3, 5000), (1, 3), (2, 9001)], 1, 16, dim, cache), 8, x, max_new=3)
    attend(Batch(cuda, [(40, 6011)], 1, 64, dim, cache), 4, x)


@pytest.mark.parametrize("cache,x", CACHES)
def test_more_positions_than_new_tokens_and_fewer(cuda, cache, x):
    """Rows at positions below 0 see nothing and give zeros."""
    sizes = [(4, 2), (100, 37), (3, 0), (90, 0)]
    batch = Batch(cuda, sizes, 2, 16, 64, cache)
    _, out = attend(batch, 8, x)
    assert (out[:2] == 0).all() and (out[2:4] != 0).any()
    assert (out[4:67] == 0).all() and (out[104:] == 0).all()


@pytest.mark.parametrize("cache", [F16, BF16])
@pytest.mark.parametrize("n,length", [(6, 70), (200, 260)])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_what_a_row_does_not_see_does_not_matter(cuda, cache, n, length, which, value):
    """A value that is no number at a new position, and one at an old position behind the window."""
    batch = Batch(cuda, [(n, length), (1, 40)], 2, 16, 64, cache)
    q = torch.randn(batch.tokens, 8, 64, generator=batch.g, device=cuda).to(cache)
    window = 50
    clean = mq.paged_attention(q, batch.cache(), *batch.where(), window=window)
    at = length - n // 2
    pool = batch.k if which == "k" else batch.v
    for j in (at, 3):
        pool[batch.table[0, j // 16].long(), :, j % 16, 5] = value
    got = mq.paged_attention(q, batch.cache(), *batch.where(), window=window)
    pos = torch.arange(length - n, length)
    sees = torch.zeros(n, dtype=torch.bool)
    for j in (at, 3):
        sees |= (pos >= j) & (pos - window < j)
    assert torch.equal(got[:n][~sees].nan_to_num(9.0), clean[:n][~sees])
    assert torch.equal(got[n:], clean[n:])
    if value != value or which == "v":
        assert not got[:n][sees][..., 5].isfinite().any()


def test_int8_scales_that_are_no_numbers(cuda):
    batch = Batch(cuda, [(6, 70), (200, 260)], 2, 16, 64, S8)
    q = torch.randn(batch.tokens, 8, 64, generator=batch.g, device=cuda).bfloat16()
    clean = mq.paged_attention(q, batch.cache(), *batch.where())
    for b, (n, length) in enumerate(batch.sizes):
        j = length - 3
        batch.scales[1][batch.table[b, j // 16].long(), :, j % 16] = float("nan")
    got = mq.paged_attention(q, batch.cache(), *batch.where())
    for first, n in ((0, 6), (6, 200)):
        assert torch.equal(got[first:first + n - 3], clean[first:first + n - 3])
        assert got[first + n - 3:first + n].isnan().all()


@pytest.mark.parametrize("scale_v", [1e-12, 1e-3, 1e4])
def test_int8_value_scales_of_any_size(cuda, scale_v):
    attend(Batch(cuda, [(1, 200), (5, 80), (100, 200)], 2, 16, 64, S8, scale_v=scale_v), 8, BF16)


def test_int8_values_of_zero(cuda):
    """Rows that were quantised from zeros have scale 0: they count with their weight and add nothing."""
    batch = Batch(cuda, [(1, 200), (100, 200)], 2, 16, 64, S8)
    for b, (n, length) in enumerate(batch.sizes):
        for j in range(0, length, 2):
            batch.v[batch.table[b, j // 16].long(), :, j % 16] = 0
            batch.scales[1][batch.table[b, j // 16].long(), :, j % 16] = 0
    attend(batch, 8, F16)


def test_int8_queries_of_any_size(cuda):
    batch = Batch(cuda, [(2, 100), (90, 150)], 1, 16, 64, S8)
    q = (torch.randn(batch.tokens, 4, 64, generator=batch.g, device=cuda) * 10.0 ** torch.linspace(-6, 6, batch.tokens, device=cuda)[:, None, None])
    q = q.bfloat16()
    out = mq.paged_attention(q, batch.cache(), *batch.where(), scale=1e-5)
    batch.check(out, q, 1e-5)


@pytest.mark.parametrize("cache", [F16, BF16])
def test_peaked_and_growing_scores(cuda, cache):
    """Scores that grow along the sequence, so that the maximum keeps moving, and large ones."""
    for n, length in ((1, 700), (130, 700)):
        batch = Batch(cuda, [(n, length)], 1, 16, 64, cache)
        j = torch.arange(length, device=cuda)
        of, row = batch.table[0][j // 16].long(), j % 16
        batch.k[of, :, row] = (batch.k[of, :, row].float() * (j / 30.0)[:, None, None]).to(cache)
        attend(batch, 4, cache, scale=0.5)


def test_strided_rows_and_in_place(cuda):
    """q as a slice of a fused projection, out its own buffer; tables with a stride."""
    batch = Batch(cuda, MANY, 2, 32, 64, BF16)
    fused = torch.randn(batch.tokens, 12, 64, generator=batch.g, device=cuda).bfloat16()
    q = fused[:, :8]
    keep = fused.clone()
    wide = torch.full((len(MANY), batch.table.shape[1] + 5), 99999, dtype=torch.int32, device=cuda)
    wide[:, 2:2 + batch.table.shape[1]] = batch.table
    table = wide[:, 2:2 + batch.table.shape[1]]
    plain = mq.paged_attention(q.contiguous(), batch.cache(), *batch.where())
    out = mq.paged_attention(q, batch.cache(), table, batch.lengths, batch.starts, out=q)
    assert torch.equal(out, plain)
    assert torch.equal(fused[:, 8:], keep[:, 8:])
    heads_first = keep[:, :8].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(mq.paged_attention(heads_first, batch.cache(), *batch.where()), plain)


def test_results_do_not_vary(cuda):
    batch = Batch(cuda, [(1, 3000), (5, 700), (300, 2000)], 2, 16, 128, BF16)
    q = torch.randn(batch.tokens, 8, 128, generator=batch.g, device=cuda).bfloat16()
    first = mq.paged_attention(q, batch.cache(), *batch.where())
    for _ in range(5):
        assert torch.equal(mq.paged_attention(q, batch.cache(), *batch.where()), first)


def test_bad_pages_are_reported_and_read_as_zeros(cuda):
    for n in (1, 90):
        batch = Batch(cuda, [(n, 100), (1, 30)], 2, 16, 64, F16)
        zero = Batch(cuda, [(n, 100), (1, 30)], 2, 16, 64, F16)
        bad = zero.table[0, 2].long()
        zero.k[bad] = 0
        zero.v[bad] = 0
        q = torch.randn(batch.tokens, 8, 64, generator=batch.g, device=cuda).half()
        want = mq.paged_attention(q, zero.cache(), *zero.where())
        mq.device_status()
        for entry in (-1, batch.k.shape[0], 2 ** 31 - 1, -2 ** 31):
            batch.table[0, 2] = entry
            got = mq.paged_attention(q, batch.cache(), *batch.where())
            assert mq.device_status() == 19
            assert torch.equal(got, want)


def test_bad_lengths_starts_and_counts_are_cut(cuda):
    batch = Batch(cuda, [(2, 48), (70, 96)], 2, 16, 64, F16)
    q = torch.randn(batch.tokens, 8, 64, generator=batch.g, device=cuda).half()
    table = batch.table[:, :3].contiguous()
    mq.device_status()
    got = mq.paged_attention(q, batch.cache(), table, batch.lengths, batch.starts)
    assert mq.device_status() == 20
    shorter = batch.lengths.clamp(max=48)
    assert torch.equal(got, mq.paged_attention(q, batch.cache(), table, shorter, batch.starts))
    batch.lengths[0] = -5
    got = mq.paged_attention(q, batch.cache(), *batch.where())
    assert mq.device_status() == 20 and (got[:2] == 0).all()
    batch.lengths[0] = 48
    out = torch.full_like(q, 7.0)
    mq.paged_attention(q, batch.cache(), *batch.where(), out=out, max_new=16)
    assert mq.device_status() == 26 and (out[2:] == 7).all() and (out[:2] != 7).any()
    starts = torch.tensor([-9, 2, 10 ** 6], dtype=torch.int32, device=cuda)
    got = mq.paged_attention(q, batch.cache(), batch.table, batch.lengths, starts)
    assert torch.equal(got, mq.paged_attention(q, batch.cache(), *batch.where()))
    starts = torch.tensor([5, 3, 1], dtype=torch.int32, device=cuda)
    mq.paged_attention(q, batch.cache(), batch.table, batch.lengths, starts)  # (no sequence has a row)
    assert mq.device_status() == 0


def test_nothing_to_do(cuda):
    cache = mq.paged_cache(4, 2, 16, 64)
    empty = torch.empty(0, 8, 64, device=cuda, dtype=F16)
    table = torch.empty(0, 3, dtype=torch.int32, device=cuda)
    none = torch.empty(0, dtype=torch.int32, device=cuda)
    assert mq.paged_attention(empty, cache, table, none).shape == (0, 8, 64)
    kv = torch.empty(0, 2, 64, device=cuda, dtype=F16)
    mq.kv_store(kv, kv, cache, table, none)
    mq.kv_load(cache, table, none)
    # A table without entries, sequences of length 0.
    table, lengths = torch.empty(3, 0, dtype=torch.int32, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda)
    q = torch.randn(3, 8, 64, device=cuda).half()
    assert (mq.paged_attention(q, cache, table, lengths) == 0).all()


# ---- the cache's rows -------------------------------------------------------------------------------------

STORED = [(5, 5), (1, 300), (0, 40), (31, 64), (7, 65), (4, 2), (1, 0), (60, 200)]


def sources(batch, dtype):
    k, v = (torch.randn(batch.tokens, batch.kv_heads, batch.dim, generator=batch.g, device=batch.cuda) for _ in range(2))
    v[3::7] = 0
    k *= 10.0 ** torch.randint(-3, 4, k.shape[:2], generator=batch.g, device=batch.cuda)[..., None]
    if dtype == F32:
        k[::5] *= 1e-35  # (rows below 1e-30 are quantised through a power of two)
    return k.to(dtype), v.to(dtype)


@pytest.mark.parametrize("x", [F32, F16, BF16])
@pytest.mark.parametrize("cache", [F16, BF16, S8])
@pytest.mark.parametrize("kv_heads,page,dim,order", [(1, 16, 64, "head"), (8, 16, 128, "position"), (3, 64, 96, "head"), (2, 256, 16, "position"),
                                                   (40, 32, 48, "head")])
def test_store_and_load(cuda, x, cache, kv_heads, page, dim, order):
    batch = Batch(cuda, STORED, kv_heads, page, dim, cache, order, gap=2)
    k, v = sources(batch, x)
    before = [t.clone() for t in (batch.k, batch.v, *[s for s in batch.scales if s is not None])]
    mq.device_status()
    assert mq.kv_store(k, v, batch.cache(), *batch.where()).k is batch.k
    assert mq.device_status() == 0
    places = paged.places(batch.np_starts, batch.lengths.tolist(), batch.tokens)
    after = (batch.k, batch.v, *[s for s in batch.scales if s is not None])
    want = [t.clone() for t in before]
    for i, t in enumerate((k, v)):
        rows, scales = (torch.from_numpy(a).to(cuda) for a in serving.quantize_s8(t.float().cpu().numpy())) if cache == S8 else (t.to(cache), None)
        for token, (b, p) in enumerate(places):
            if b >= 0 and p >= 0:
                of = int(batch.np_table[b, p // page])
                want[i][of, :, p % page] = rows[token]
                if cache == S8:
                    want[2 + i][of, :, p % page] = scales[token]
    for a, w in zip(after, want):
        assert torch.equal(a.nan_to_num(nan=123.0) if a.is_floating_point() else a, w.nan_to_num(nan=123.0) if w.is_floating_point() else w)

    for out in (F32, F16, BF16):
        got = [torch.full((batch.tokens, kv_heads, dim), 7.0, device=cuda, dtype=out) for _ in range(2)]
        mq.kv_load(batch.cache(), *batch.where(), k=got[0], v=got[1])
        assert mq.device_status() == 0
        for i, t in enumerate(got):
            ref = torch.full_like(t, 7.0)
            for token, (b, p) in enumerate(places):
                if b >= 0:
                    ref[token] = 0
                    if p >= 0:
                        of = int(batch.np_table[b, p // page])
                        row = after[i][of, :, p % page].float()
                        ref[token] = (row * after[2 + i][of, :, p % page][:, None] if cache == S8 else row).to(out)
            assert torch.equal(t, ref)


def test_store_not_numbers(cuda):
    for cache in (S8, F16):
        batch = Batch(cuda, [(9, 20)], 2, 16, 64, cache)
        k, v = sources(batch, F32)
        k[2, 1, 3], k[4, 0, 0], v[5, 1, 63] = float("nan"), float("inf"), float("-inf")
        mq.kv_store(k, v, batch.cache(), *batch.where())
        lk, lv = mq.kv_load(batch.cache(), *batch.where(), tokens=9, dtype=F32)
        if cache == S8:
            assert lk[2, 1].isnan().all() and lk[4, 0].isnan().all() and lv[5, 1].isnan().all()
            assert lk[2, 0].isfinite().all() and lk[4, 1].isfinite().all()
        else:
            assert torch.equal(lk.isfinite(), k.half().isfinite()) and torch.equal(lv.isfinite(), v.half().isfinite())


def test_store_strided_sources(cuda):
    batch, same = (Batch(cuda, STORED, 2, 16, 64, S8) for _ in range(2))
    fused = torch.randn(batch.tokens, 8 + 2 + 2, 64, generator=batch.g, device=cuda).bfloat16()
    mq.kv_store(fused[:, 8:10], fused[:, 10:], batch.cache(), *batch.where())
    mq.kv_store(fused[:, 8:10].contiguous(), fused[:, 10:].contiguous(), same.cache(), *same.where())
    assert torch.equal(batch.k, same.k) and torch.equal(batch.v, same.v)
    assert torch.equal(batch.scales[0].nan_to_num(), same.scales[0].nan_to_num())


def test_store_and_load_bad_pages(cuda):
    batch = Batch(cuda, [(40, 40), (3, 3)], 2, 16, 64, F16)
    k, v = sources(batch, F16)
    before = batch.k.clone()
    missing = int(batch.table[0, 1])
    mq.device_status()
    for entry in (-1, batch.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        batch.table[0, 1] = entry
        mq.kv_store(k, v, batch.cache(), *batch.where())
        assert mq.device_status() == 19
        assert torch.equal(batch.k[missing].nan_to_num(), before[missing].nan_to_num())
        lk, lv = mq.kv_load(batch.cache(), *batch.where(), tokens=43)
        assert mq.device_status() == 19
        assert (lk[16:32] == 0).all() and torch.equal(lk[:16], k[:16]) and torch.equal(lk[32:], k[32:]) and torch.equal(lv[40:], v[40:])


def test_store_then_attend_as_used(cuda):
    """Prompt, chunk, single tokens: the int8 cache is written and read step by step, and the outputs are those of the
    whole sequence at once."""
    heads, kv_heads, dim, page = 8, 2, 64, 16
    g = torch.Generator(device=cuda).manual_seed(5)
    total = 150
    q, k, v = (torch.randn(total, h, dim, generator=g, device=cuda).bfloat16() for h in (heads, kv_heads, kv_heads))
    for dtype in (S8, BF16):
        cache = mq.paged_cache(total // page + 2, kv_heads, page, dim, dtype)
        table = torch.arange(total // page + 1, -1, -1, dtype=torch.int32, device=cuda)[None, :total // page + 1].contiguous()
        outs, at = [], 0
        for n in (100, 30, 5, 1, 1, 13):
            lengths = torch.tensor([at + n], dtype=torch.int32, device=cuda)
            starts = torch.tensor([0, n], dtype=torch.int32, device=cuda)
            mq.kv_store(k[at:at + n], v[at:at + n], cache, table, lengths, starts)
            outs.append(mq.paged_attention(q[at:at + n], cache, table, lengths, starts))
            at += n
        starts = torch.tensor([0, total], dtype=torch.int32, device=cuda)
        whole = mq.paged_attention(q, cache, table, lengths, starts)
        unit = UNIT[BF16]
        size = 8 * unit * v.float().abs().max()  # (two results, each within half of this of the exact one)
        assert (torch.cat(outs).float() - whole.float()).abs().max() <= size
        assert mq.device_status() == 0


class Drafted(Batch):
    """Steps with drafted tokens, as they are used: qkv product, kv_store, paged_attention, head product, verify_drafts, and the
    lengths that follow from what was accepted, all on the device. Three requests, one of them greedy, one that begins empty."""

    heads, kv_heads, dim, page, drafts, vocab = 8, 2, 64, 16, 3, 203
    temperatures, before = [1.0, 0.0, 0.7], [0, 5, 33]

    def __init__(self, cuda, dtype, x):
        g = torch.Generator(device=cuda).manual_seed(9)
        self.g, self.cuda, self.dtype, self.x, self.ints = g, cuda, dtype, x, dtype == S8
        wide, self.n, b = self.heads * self.dim, self.drafts + 1, 3
        self.np_starts = [self.n * i for i in range(b + 1)]
        self.tokens, self.starts = self.n * b, torch.tensor(self.np_starts, dtype=torch.int32, device=cuda)
        self.table = torch.randperm(6 * b, generator=g, device=cuda).int().view(b, 6).contiguous()
        self.pool = mq.paged_cache(6 * b, self.kv_heads, self.page, self.dim, dtype)
        self.k, self.v, self.scales = self.pool.k, self.pool.v, [self.pool.k_scale, self.pool.v_scale]
        self.qkv = mq.quantize_s8(torch.randn(wide + 2 * self.kv_heads * self.dim, wide, generator=g, device=cuda) * wide ** -0.5)
        self.head = mq.quantize_s8(torch.randn(self.vocab, wide, generator=g, device=cuda) * 3 * wide ** -0.5)
        self.temperature = torch.tensor(self.temperatures, device=cuda)
        self.h = torch.empty(self.tokens, wide, dtype=F16, device=cuda)
        self.draft = torch.empty(b * self.drafts, self.vocab, device=cuda)
        self.drafted = torch.empty(b, self.drafts, dtype=torch.int32, device=cuda)
        self.uniform = torch.empty(b, self.n, device=cuda)
        self.lengths = torch.empty(b, dtype=torch.int32, device=cuda)
        self.work = torch.empty(mq.paged_attention_workspace(self.pool, self.heads, b, self.tokens, self.n), dtype=torch.uint8, device=cuda)
        self.verify_work = torch.empty(mq.verify_workspace(b, self.drafts, self.vocab), dtype=torch.uint8, device=cuda)
        self.past = [[torch.randn(m, self.kv_heads, self.dim, generator=g, device=cuda).to(x) for _ in range(2)] for m in self.before]
        self.inputs = [self.draw() for _ in range(6)]

    def draw(self):
        draft = torch.randn(self.draft.shape, generator=self.g, device=self.cuda)
        drafted = torch.multinomial(draft.softmax(-1), 1, generator=self.g).int().view(self.drafted.shape)
        return (torch.randn(self.h.shape, generator=self.g, device=self.cuda).half(), draft, drafted,
                torch.rand(self.uniform.shape, generator=self.g, device=self.cuda))

    def begin(self):
        for b, (k, v) in enumerate(self.past):
            if len(k):
                m = torch.tensor([len(k)], dtype=torch.int32, device=self.cuda)
                mq.kv_store(k, v, self.pool, self.table[b:b + 1], m, torch.tensor([0, len(k)], dtype=torch.int32, device=self.cuda))
        self.lengths.copy_(torch.tensor(self.before, device=self.cuda) + self.n)

    def feed(self, i):
        for t, new in zip((self.h, self.draft, self.drafted, self.uniform), self.inputs[i]):
            t.copy_(new)

    def step(self):
        at = self.lengths.clone()
        wide, kv = self.heads * self.dim, self.kv_heads * self.dim
        y = mq.gemm_w8a8(*mq.quantize_s8(self.h), *self.qkv, dtype=self.x)
        q, k, v = (p.view(self.tokens, -1, self.dim) for p in y.split([wide, kv, kv], 1))
        mq.kv_store(k, v, self.pool, self.table, self.lengths, self.starts)
        o = mq.paged_attention(q, self.pool, self.table, self.lengths, self.starts, max_new=self.n, workspace=self.work)
        logits = mq.gemm_w8a8(*mq.quantize_s8(o.view(self.tokens, -1)), *self.head, dtype=F32)
        got = mq.verify_drafts(logits, self.drafted, self.uniform, draft=self.draft, temperature=self.temperature, workspace=self.verify_work)
        self.lengths.add_(got[1] + 1)
        return [at, q, k, v, o, logits, *got, self.lengths]


@pytest.mark.parametrize("dtype,x", CACHES)
def test_drafted_steps_as_used(cuda, dtype, x):
    """Each operator against the oracle on what it was given, step after step as the lengths follow from the tokens that were
    accepted; then the same steps as one captured graph, with the same bits."""
    d = Drafted(cuda, dtype, x)
    d.begin()
    want, seen = [], set()
    for i in range(len(d.inputs)):
        d.feed(i)
        at, q, k, v, o, logits, tokens, accepted, logprobs, after = got = d.step()
        assert mq.device_status() == 0
        d.sizes = [(d.n, length) for length in at.tolist()]
        if dtype != S8:
            held = mq.kv_load(d.pool, d.table, at, d.starts, tokens=d.tokens, dtype=x)
            assert torch.equal(held[0], k) and torch.equal(held[1], v)
        d.check(o, q, d.dim ** -0.5)
        for b, t in enumerate(d.temperatures):
            rows, theirs = host(logits.view(3, d.n, -1)[b]), host(d.draft.view(3, d.drafts, -1)[b])
            # (temperatures as the device holds them)
            ref = paged.verify(rows, host(d.drafted[b]), host(d.uniform[b]), theirs, float(d.temperature[b]))
            assert tokens[b].tolist() == ref[0] and int(accepted[b]) == ref[1]
            unit = 2.0 ** -24 * (2 * (np.log2(d.vocab) + 2) + 4 + d.vocab / 256 + 24)  # as the verification's own tests derive it
            assert (np.abs(host(logprobs[b]) - ref[2]) <= unit + 2.0 ** -24 * np.abs(ref[2])).all()
            seen.add(ref[1])
        assert torch.equal(after, at + accepted + 1)
        want.append([t.clone() for t in got])
    assert 0 in seen and len(seen) > 1, "the steps keep different numbers of drafted tokens"
    d.begin()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = d.step()
    for i in range(len(d.inputs)):
        d.feed(i)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want[i])), i
    assert mq.device_status() == 0


# ---- streams, graphs, refusals ----------------------------------------------------------------------------------


def test_two_streams_at_once(cuda):
    sizes = [(1, 900), (80, 300)]
    batches = [Batch(cuda, sizes, 2, 16, 128, d, seed=i) for i, d in enumerate((BF16, S8))]
    qs = [torch.randn(81, 8, 128, generator=b.g, device=cuda).bfloat16() for b in batches]
    want = [mq.paged_attention(q, b.cache(), *b.where()) for q, b in zip(qs, batches)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for s, q, b in zip(streams, qs, batches):
            with torch.cuda.stream(s):
                got.append(mq.paged_attention(q, b.cache(), *b.where()))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 2])


def test_captured_step(cuda):
    """Store and attention in one graph, replayed as the lengths grow on the device."""
    heads, kv_heads, dim, page, most = 8, 2, 64, 16, 64
    g = torch.Generator(device=cuda).manual_seed(1)
    for dtype in (F16, S8):
        cache = mq.paged_cache(2 * most // page, kv_heads, page, dim, dtype)
        table = torch.randperm(2 * most // page, generator=g, device=cuda).int().view(2, -1).contiguous()
        lengths = torch.zeros(2, dtype=torch.int32, device=cuda)
        q, k, v = (torch.empty(2, h, dim, device=cuda, dtype=F16) for h in (heads, kv_heads, kv_heads))
        out = torch.empty_like(q)
        work = torch.empty(mq.paged_attention_workspace(cache, heads, 2, 2, 1), dtype=torch.uint8, device=cuda)

        def step():
            lengths.add_(1)
            mq.kv_store(k, v, cache, table, lengths)
            mq.paged_attention(q, cache, table, lengths, out=out, workspace=work)

        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        lengths.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        lengths.zero_()
        ks, vs = [], []
        for i in range(20):
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=g, device=cuda))
            ks.append(k.clone())
            vs.append(v.clone())
            graph.replay()
            want = mq.paged_attention(q, cache, table, lengths)
            assert torch.equal(out, want)
            if dtype == F16:
                lk, lv = mq.kv_load(cache, table, lengths)
                assert torch.equal(lk, k) and torch.equal(lv, v)
                z = torch.einsum("bkgd,lbkd->bkgl", q.double().view(2, kv_heads, -1, dim), torch.stack(ks).double()) * dim ** -0.5
                ref = torch.einsum("bkgl,lbkd->bkgd", z.softmax(-1), torch.stack(vs).double()).reshape(2, heads, dim)
                # (fp16 output and weights: 3 units of the largest value; scores below 2^-17)
                assert (out.double() - ref).abs().max() <= (3 * 2.0 ** -11 + 2.0 ** -16) * torch.stack(vs).abs().max()
        assert mq.device_status() == 0


@pytest.mark.parametrize("cache,x", [(S8, BF16), (F16, F16)])
def test_pages_beyond_32_bits(cuda, cache, x):
    """A pool of more than 2^32 bytes (fp16: 2^32 elements): the pages in use are its first and its last ones."""
    page, kv_heads, dim = 64, 8, 128
    pages = 2 ** 32 // (page * kv_heads * dim) + 9
    k, v = (torch.empty(pages, kv_heads, page, dim, dtype=cache, device=cuda) for _ in range(2))
    scales = [torch.zeros(pages, kv_heads, page, device=cuda) for _ in range(2)] if cache == S8 else []
    pool = mq.PagedCache(k, v, *scales)
    ids = [pages - 1, 0, pages - 3, pages // 2 + 1, 2, pages - 2]
    small = mq.paged_cache(len(ids), kv_heads, page, dim, cache)
    g = torch.Generator(device=cuda).manual_seed(2)
    table = torch.tensor([ids[:3], ids[3:]], dtype=torch.int32, device=cuda)
    near = torch.arange(6, dtype=torch.int32, device=cuda).view(2, 3)
    lengths = torch.tensor([180, 130], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, 180, 310], dtype=torch.int32, device=cuda)
    rows = [torch.randn(310, kv_heads, dim, generator=g, device=cuda).to(x) for _ in range(2)]
    q = torch.randn(310, 16, dim, generator=g, device=cuda).to(x)
    for c, t in ((pool, table), (small, near)):
        mq.kv_store(*rows, c, t, lengths, starts)
    for a, b in zip(mq.kv_load(pool, table, lengths, starts, tokens=310, dtype=x), mq.kv_load(small, near, lengths, starts, tokens=310, dtype=x)):
        assert torch.equal(a, b)
    assert torch.equal(mq.paged_attention(q, pool, table, lengths, starts), mq.paged_attention(q, small, near, lengths, starts))
    assert torch.equal(mq.paged_attention(q[:2], pool, table, lengths), mq.paged_attention(q[:2], small, near, lengths))
    assert mq.device_status() == 0


def test_workspace_of_a_larger_call_is_enough(cuda):
    """Sizes never fall when a call has more sequences, tokens or new tokens."""
    for dim, dtype in ((64, F16), (128, S8)):
        cache = mq.paged_cache(2, 2, 16, dim, dtype)
        for heads in (2, 8, 16, 64):
            size = {}
            for batch in (1, 2, 4, 9):
                for tokens in (1, 2, 4, 9, 40):
                    for most in (1, 2, 5, 40):
                        size[batch, tokens, most] = mq.paged_attention_workspace(cache, heads, batch, tokens, most)
            for a, sa in size.items():
                for b, sb in size.items():
                    if all(i <= j for i, j in zip(a, b)):
                        assert sa <= sb, (heads, a, b)


def test_workspace_serves_smaller_calls(cuda):
    batch = Batch(cuda, [(1, 900), (80, 300)], 2, 16, 128, BF16)
    cache = batch.cache()
    work = torch.empty(mq.paged_attention_workspace(cache, 8, 8, 4096), dtype=torch.uint8, device=cuda)
    attend(batch, 8, BF16, workspace=work)
    attend(Batch(cuda, ONE, 2, 16, 128, BF16), 8, BF16, workspace=work, max_new=1)


def test_refusals(cuda):
    cache = mq.paged_cache(4, 2, 16, 64)
    table = torch.zeros(1, 4, dtype=torch.int32, device=cuda)
    lengths = torch.ones(1, dtype=torch.int32, device=cuda)
    q = torch.zeros(1, 8, 64, device=cuda, dtype=F16)
    kv = torch.zeros(1, 2, 64, device=cuda, dtype=F16)

    def refuses(match, call):
        with pytest.raises(mq.MQError, match=match):
            call()

    refuses("type in", lambda: mq.paged_attention(q.float(), cache, table, lengths))
    refuses("16-bit cache", lambda: mq.paged_attention(q.bfloat16(), cache, table, lengths))
    refuses("multiple of the cache", lambda: mq.paged_attention(q[:, :3], cache, table, lengths))
    refuses("does not go with", lambda: mq.paged_attention(q[..., :32].contiguous(), cache, table, lengths))
    refuses("scale must be positive", lambda: mq.paged_attention(q, cache, table, lengths, scale=0.0))
    refuses("scale must be positive", lambda: mq.paged_attention(q, cache, table, lengths, scale=float("nan")))
    refuses("bad window", lambda: mq.paged_attention(q, cache, table, lengths, window=-1))
    refuses("need starts", lambda: mq.paged_attention(q.expand(2, 8, 64).contiguous(), cache, table, lengths))
    refuses("overlap", lambda: mq.paged_attention(q.expand(2, 8, 64).contiguous(), cache, table, lengths, torch.tensor([0, 2], dtype=torch.int32, device=cuda),
                                                  out=torch.empty(1, 8, 64, device=cuda, dtype=F16).expand(2, 8, 64)))
    refuses("workspace is too small", lambda: mq.paged_attention(q, cache, table, lengths, workspace=torch.empty(64, dtype=torch.uint8, device=cuda)))
    refuses("16-byte aligned", lambda: mq.paged_attention(torch.zeros(1 * 8 * 64 + 4, device=cuda, dtype=F16)[4:].view(1, 8, 64), cache, table, lengths))
    refuses("int32", lambda: mq.paged_attention(q, cache, table.long(), lengths))
    refuses("lengths", lambda: mq.paged_attention(q, cache, table, lengths.long()))
    refuses("lengths", lambda: mq.paged_attention(q, cache, table, lengths.expand(2).contiguous()))
    refuses("starts", lambda: mq.paged_attention(q, cache, table, lengths, lengths))
    refuses("CUDA|device", lambda: mq.paged_attention(q.cpu(), cache, table, lengths))
    refuses("device", lambda: mq.paged_attention(q, cache, table.cpu(), lengths))
    refuses("does not go with", lambda: mq.kv_store(kv[:, :1], kv[:, :1], cache, table, lengths))
    refuses("k's type", lambda: mq.kv_store(kv, kv.float(), cache, table, lengths))
    refuses("rows", lambda: mq.kv_load(cache, table, lengths, k=kv, v=kv, tokens=2))
    refuses("PagedCache", lambda: mq.kv_store(kv, kv, None, table, lengths))
    refuses("scales", lambda: mq.PagedCache(cache.k, cache.v, lengths, lengths))
    refuses("int8 cache needs", lambda: mq.PagedCache(cache.k.to(S8), cache.v.to(S8)))
    refuses("the same for keys", lambda: mq.PagedCache(cache.k, cache.v[:2]))
    refuses("positions", lambda: mq.kv_store(kv, kv, mq.paged_cache(4, 2, 24, 64), table, lengths))
    refuses("multiple of 16", lambda: mq.paged_attention(q[..., :40].contiguous(), mq.paged_cache(4, 2, 16, 40), table, lengths))
    refuses("multiple of 16", lambda: mq.paged_attention(torch.zeros(1, 8, 256, device=cuda, dtype=F16), mq.paged_cache(4, 2, 16, 256), table, lengths))
    wide = torch.zeros(4, 2, 16, 68, device=cuda, dtype=F16)[..., :64]
    refuses("16-byte", lambda: mq.kv_store(kv, kv, mq.PagedCache(wide, wide.clone()), table, lengths))
    flat = torch.zeros(1, 2, 16, 64, device=cuda, dtype=F16).expand(4, 2, 16, 64)
    refuses("overlap", lambda: mq.kv_store(kv, kv, mq.PagedCache(flat, cache.v), table, lengths))


@pytest.mark.parametrize("x", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_int8_narrow_and_wide_items_in_turn(cuda, x, dim):
    """Items of at most 128 rows and items of more, of one block each, several in turn for every CTA: the rows' factors (which
    differ from row to row) change while the accumulators are not equally far."""
    sizes = [(n, n + extra) for n, extra in ((9, 40), (40, 60), (64, 0), (30, 98), (64, 64), (33, 0))] * 60
    batch = Batch(cuda, sizes, 2, 16, dim, S8)
    q = torch.randn(batch.tokens, 8, dim, generator=batch.g, device=cuda) * 2.0 ** torch.randint(-6, 3, (batch.tokens, 8, 1), generator=batch.g, device=cuda)
    q = q.to(x)
    mq.device_status()
    out = mq.paged_attention(q, batch.cache(), *batch.where(), max_new=64)
    for _ in range(20):
        assert torch.equal(mq.paged_attention(q, batch.cache(), *batch.where(), max_new=64), out)
    assert mq.device_status() == 0
    batch.check(out, q, dim ** -0.5)


@pytest.mark.parametrize("cache,x", CACHES)
@pytest.mark.parametrize("batch,new", [(161, 1), (320, 1), (321, 3), (512, 6), (513, 40), (1025, 9)])
def test_more_sequences_than_threads_that_find_the_shares(cuda, cache, x, batch, new):
    """Shares are found by 160 threads (few rows) or 512 (tiles), which go through the sequences in turns, and twice through more
    of them than threads; what they leave in shared memory is where a CTA's first keys come to lie."""
    rng = np.random.default_rng(batch)
    sizes = [(n, n + int(rng.integers(0, 90))) for n in (int(rng.integers(0, new + 1)) for _ in range(batch))]
    sizes[0], sizes[batch // 2], sizes[-1] = (new, new + 700), (0, 50), (new, new + 900)
    attend(Batch(cuda, sizes, 2, 16, 64, cache), 8, x, max_new=new)


@pytest.mark.parametrize("cache,x", CACHES)
@pytest.mark.parametrize("held,rows", [([(3, 10)], 2), ([(1, 5), (4, 40), (3, 9)], 7), ([(2, 7), (5, 60), (4, 8), (1, 3)], 4),
                                       ([(150, 200), (40, 300)], 170), ([(90, 80), (300, 295)], 100), ([(4, 6), (9, 9)], 4)])
def test_starts_that_pass_the_rows(cuda, cache, x, held, rows):
    """The rows that are there keep their positions; the others are left out, and the status says so."""
    batch = Batch(cuda, held, 2, 16, 64, cache)
    full = [torch.randn(batch.tokens, 2, 64, generator=batch.g, device=cuda).to(x) for _ in range(2)]
    q = torch.randn(batch.tokens, 8, 64, generator=batch.g, device=cuda).to(x)
    before = [t.clone() for t in (batch.k, batch.v)]
    mq.device_status()
    got = mq.paged_attention(q[:rows].clone(), batch.cache(), *batch.where())
    assert mq.device_status() == 27
    want = mq.paged_attention(q, batch.cache(), *batch.where())
    batch.check(want, q, 64 ** -0.5)
    short = Batch.__new__(Batch)  # the rows that are there, by the oracle: each sequence's, at positions counted from its whole end
    short.__dict__.update(batch.__dict__)
    for b, (n, length) in enumerate(held):
        s0, s1 = batch.np_starts[b], min(batch.np_starts[b + 1], rows)
        if s1 > s0:
            # (a sequence that is cut to the positions of its rows holds the same for them)
            short.sizes, short.np_starts = [(s1 - s0, length - n + s1 - s0)], [s0, s1]
            short.held = lambda _, upto, b=b: batch.held(b, upto)
            if length - n + s1 - s0 > 0:
                short.check(got, q[:rows], 64 ** -0.5)
            else:
                assert (got[s0:s1] == 0).all()
    lk, lv = mq.kv_load(batch.cache(), *batch.where(), tokens=rows, dtype=x)
    assert mq.device_status() == 27
    ak, av = mq.kv_load(batch.cache(), *batch.where(), tokens=batch.tokens, dtype=x)
    assert torch.equal(lk, ak[:rows]) and torch.equal(lv, av[:rows])
    mq.kv_store(full[0][:rows], full[1][:rows], batch.cache(), *batch.where())
    assert mq.device_status() == 27
    lk, lv = mq.kv_load(batch.cache(), *batch.where(), tokens=batch.tokens, dtype=x)
    assert mq.device_status() == 0
    places = paged.places(batch.np_starts, [length for _, length in held], batch.tokens)
    real = torch.tensor([p >= 0 for _, p in places], device=cuda)
    if cache != S8:
        assert torch.equal(lk[:rows][real[:rows]], full[0][:rows][real[:rows]]) and torch.equal(lv[:rows][real[:rows]], full[1][:rows][real[:rows]])
    else:  # (half a step of the row's largest over 127, and the rounding to x)
        for a, b in ((lk, full[0]), (lv, full[1])):
            b = b[:rows][real[:rows]].double()
            tol = b.abs().amax(-1, keepdim=True) / 254 * 1.001 + UNIT[x] * b.abs().amax(-1, keepdim=True)
            assert ((a[:rows][real[:rows]].double() - b).abs() <= tol).all()
    assert torch.equal(lk[rows:], ak[rows:]) and torch.equal(lv[rows:], av[rows:])
    # All that no row belongs to is as it was.
    for t, old in zip((batch.k, batch.v), before):
        for (b, p), there in zip(places, range(batch.tokens)):
            if there < rows and p >= 0:
                page = int(batch.np_table[b, p // 16])
                old[page, :, p % 16] = t[page, :, p % 16]
        assert torch.equal(t.view(torch.uint8) if cache == S8 else t.view(torch.int16), old.view(torch.uint8) if cache == S8 else old.view(torch.int16))


def test_starts_far_behind_the_rows(cuda):
    """An end that can be none (more rows than the table has positions, none of those that are there at one) is the rows' end to the
    attention; the copies leave such rows out, and say so. One that can be makes rows without positions, which see nothing."""
    batch = Batch(cuda, [(3, 40), (5, 60)], 2, 16, 64, F16)
    q = torch.randn(batch.tokens, 8, 64, generator=batch.g, device=cuda).half()
    for end in (3 + 5 * 16 + 1, 10 ** 6, 2 ** 31 - 1):
        starts = torch.tensor([-2 ** 31, 3, end], dtype=torch.int32, device=cuda)
        mq.device_status()
        want = mq.paged_attention(q, batch.cache(), *batch.where())
        assert torch.equal(mq.paged_attention(q, batch.cache(), batch.table, batch.lengths, starts), want)
        assert mq.device_status() == 0
        before = [batch.k.clone(), batch.v.clone()]
        kv = torch.randn(8, 2, 64, generator=batch.g, device=cuda)
        mq.kv_store(kv, kv, batch.cache(), batch.table, batch.lengths, starts)
        assert mq.device_status() == 27
        k, v = mq.kv_load(batch.cache(), batch.table, batch.lengths, starts, tokens=8)
        assert mq.device_status() == 27
        assert torch.equal(k[:3], kv[:3].half()) and torch.equal(v[:3], kv[:3].half()) and (k[3:] == 0).all() and (v[3:] == 0).all()
        for j in range(40, 60):
            page = int(batch.np_table[1, j // 16])
            assert torch.equal(batch.k[page, :, j % 16], before[0][page, :, j % 16])
    want = mq.paged_attention(q, batch.cache(), *batch.where())
    for end in (8 + 60, 3 + 5 * 16):
        starts = torch.tensor([0, 3, end], dtype=torch.int32, device=cuda)
        got = mq.paged_attention(q, batch.cache(), batch.table, batch.lengths, starts)
        assert mq.device_status() == 27 and (got[3:] == 0).all() and torch.equal(got[:3], want[:3])
    starts = torch.tensor([0, 3, 8 + 59], dtype=torch.int32, device=cuda)  # the last row's position is 0
    got = mq.paged_attention(q, batch.cache(), batch.table, batch.lengths, starts)
    assert mq.device_status() == 27
    first = batch.v[int(batch.np_table[1, 0]), :, 0].repeat_interleave(4, 0)
    assert (got[3:7] == 0).all() and torch.equal(got[7], first)


def test_load_with_starts_needs_the_number_of_rows(cuda):
    """Without it there was one row per sequence, of positions that the starts do not mean."""
    batch = Batch(cuda, [(3, 10), (2, 20)], 2, 16, 64, F16)
    with pytest.raises(mq.MQError, match="tokens"):
        mq.kv_load(batch.cache(), *batch.where())
    with pytest.raises(mq.MQError, match="table"):
        mq.kv_load(batch.cache(), None, batch.lengths)
    want = mq.kv_load(batch.cache(), *batch.where(), tokens=5)
    for kw in (dict(k=torch.empty_like(want[0])), dict(v=torch.empty_like(want[1])), dict(k=torch.empty_like(want[0]), v=torch.empty_like(want[1]))):
        got = mq.kv_load(batch.cache(), *batch.where(), **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    k, v = mq.kv_load(batch.cache(), batch.table, batch.lengths)  # each one's last position
    assert torch.equal(k, want[0][[2, 4]]) and torch.equal(v, want[1][[2, 4]])


def test_int8_operands_are_the_integers(cuda):
    """Scores of many terms of one sign, where an error that a key's terms share would show (bf16 rows, most blocks seen by every row).
    Weights are rounded to fp16, u = 2^-11 at most, u / sqrt(3) in the mean; a score is off by dim 2^-24 of itself, for the fp32
    sums; an output by those of its terms p_j v_j, root of the sum of squares, within six standard deviations, and by 2^-8 of itself."""
    n, length, dim, heads = 64, 1000, 128, 8
    batch = Batch(cuda, [(n, length)], 2, 16, dim, S8)
    batch.k.copy_(torch.randint(32, 128, batch.k.shape, generator=batch.g, device=cuda, dtype=torch.int32).to(S8))
    batch.scales[0].uniform_(0.00097, 0.001, generator=batch.g)
    batch.scales[1].uniform_(0.01, 0.02, generator=batch.g)
    q = (torch.rand(n, heads, dim, generator=batch.g, device=cuda) + 0.5).bfloat16()
    scale = 6.0  # scores of 60 or so
    out = mq.paged_attention(q, batch.cache(), *batch.where(), scale=scale)
    keys, values, _ = batch.held(0, length)
    got, rows, u = host(out), host(q), 2.0 ** -11
    for h in range(heads):
        k, v = keys[h // 4], values[h // 4]
        z = scale * rows[:, h] @ k.T
        assert 40 < z.mean() < 80
        e2 = (dim * 2.0 ** -24 * z) ** 2
        z[np.arange(length) > np.arange(length - n, length)[:, None]] = -np.inf
        p = np.exp(z - z.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        ref = p @ v
        # (the sum of weights carries the scores' errors as well)
        sigma = np.sqrt((p ** 2 * (e2 + u * u / 3)) @ v ** 2 + (p ** 2 * e2).sum(1, keepdims=True) * ref ** 2)
        bad = np.abs(got[:, h] - ref) > 6 * sigma + 2.0 ** -8 * np.abs(ref)
        assert not bad.any(), (h, int(bad.sum()), float((np.abs(got[:, h] - ref) / sigma).max()))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("spike", [4096.0, 2.0 ** 20])
@pytest.mark.parametrize("which", ["k", "v", "kv"])
def test_int8_one_scale_far_above_its_neighbours(cuda, dim, spike, which):
    """One key of 32 has a scale `spike` times the others', and (its row being against q) no weight: what the others give must not
    suffer from it. bf16 rows; the bound is that of an int8 cache at the head of this file, q's conversion being exact here."""
    n, length, heads = 64, 500, 8
    batch = Batch(cuda, [(n, length)], 2, 16, dim, S8)
    q = (torch.rand(n, heads, dim, generator=batch.g, device=cuda) + 0.5).bfloat16()
    for j in range(5, length, 32):
        of, row = batch.table[0, j // 16].long(), j % 16
        batch.k[of, :, row] = -100
        batch.scales[0][of, :, row] = 0.05 * (spike if "k" in which else 40)
        if "v" in which:
            batch.scales[1][of, :, row] = 0.05 * spike
    scale = dim ** -0.5
    mq.device_status()
    got = host(mq.paged_attention(q, batch.cache(), *batch.where()))
    assert mq.device_status() == 0
    keys, values, steps = batch.held(0, length)
    rows = host(q)
    ref, size, tiny = paged.attention(rows, keys, values, range(length - n, length), scale, 0, steps[1])
    near = np.ones(length, bool)
    near[5::32] = False
    big = scale * np.einsum("thd,hjd->thj", np.abs(rows), np.repeat(np.abs(keys[:, near]), 4, 0)).max(-1)
    e = (dim + 16) * 2.0 ** -23 * big
    bound = 2.0 ** -8 * np.abs(ref) + (2 * 2.0 ** -11 + 2 * e + 2.0 ** -19)[..., None] * size + 2.0 ** -25 * tiny
    assert (np.abs(got - ref) <= bound).all(), float((np.abs(got - ref) / bound).max())


@pytest.mark.parametrize("x", [F16, BF16])
@pytest.mark.parametrize("which", ["k", "v"])
def test_int8_scales_of_zero(cuda, x, which):
    """Rows that were quantised from zeros, alone and 64 in a row, in blocks that every row sees and in others."""
    batch = Batch(cuda, [(1, 400), (100, 400), (7, 300)], 2, 16, 64, S8)
    for b, (n, length) in enumerate(batch.sizes):
        for j in sorted({*range(1, length, 7), *range(128, 192)}):
            of = batch.table[b, j // 16].long()
            (batch.k if which == "k" else batch.v)[of, :, j % 16] = 0
            batch.scales["kv".index(which)][of, :, j % 16] = 0
    attend(batch, 8, x)


@pytest.mark.parametrize("x", [F16, BF16])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("at", [5, 200, -3])
def test_int8_scales_that_are_no_numbers_anywhere(cuda, x, which, value, at):
    """In blocks that every row sees and in others: the rows that see such a scale are no numbers, the others as without it."""
    batch = Batch(cuda, [(6, 400), (1, 400), (100, 400), (40, 500)], 2, 16, 64, S8)
    q = torch.randn(batch.tokens, 8, 64, generator=batch.g, device=cuda).to(x)
    clean = mq.paged_attention(q, batch.cache(), *batch.where())
    for b, (n, length) in enumerate(batch.sizes):
        j = at % length
        batch.scales["kv".index(which)][batch.table[b, j // 16].long(), :, j % 16] = value
    got = mq.paged_attention(q, batch.cache(), *batch.where())
    for b, (n, length) in enumerate(batch.sizes):
        first, sees = batch.np_starts[b], torch.arange(length - n, length) >= at % length
        assert torch.equal(got[first:first + n][~sees], clean[first:first + n][~sees])
        assert not got[first:first + n][sees].isfinite().any(), b


@pytest.mark.parametrize("cache", [F16, S8])
def test_positions_beyond_the_table_are_not_copied(cuda, cache):
    """They were stored over the last positions that the table names."""
    batch = Batch(cuda, [(2, 30), (5, 32), (1, 32)], 2, 16, 64, cache)
    table = batch.table[:, :2].contiguous()
    lengths = torch.tensor([33, 35, 2 ** 31 - 1], dtype=torch.int32, device=cuda)  # 31 and 32; 30 .. 34; 2^31 - 2
    kv = torch.randn(8, 2, 64, generator=batch.g, device=cuda).half()
    before = [batch.k.clone(), batch.v.clone()]
    mq.device_status()
    mq.kv_store(kv, kv, batch.cache(), table, lengths, batch.starts)
    assert mq.device_status() == 20
    for t, old in zip((batch.k, batch.v), before):
        changed = {(int(p), int(r)) for p, _, r, _ in (t.view(torch.uint8) != old.view(torch.uint8)).nonzero()}
        assert changed == {(int(table[0, 1]), 15), (int(table[1, 1]), 14), (int(table[1, 1]), 15)}
    k, v = mq.kv_load(batch.cache(), table, lengths, batch.starts, tokens=8)
    assert mq.device_status() == 20
    there = torch.tensor([True, False, True, True, False, False, False, False], device=cuda)
    assert (k[~there] == 0).all() and (v[~there] == 0).all()
    k2, v2 = mq.kv_load(batch.cache(), table, torch.tensor([32, 32, 32], dtype=torch.int32, device=cuda),
                        torch.tensor([0, 1, 3, 3], dtype=torch.int32, device=cuda), tokens=3)
    assert mq.device_status() == 0
    assert torch.equal(k[there], k2) and torch.equal(v[there], v2)
    if cache == F16:
        assert torch.equal(k[there], kv[there])
    mq.kv_store(kv[:3], kv[:3], batch.cache(), table, lengths)  # without starts: positions 32, 34, 2^31 - 2
    assert mq.device_status() == 20
    k, v = mq.kv_load(batch.cache(), table, torch.full_like(lengths, 32))
    assert torch.equal(k[:2], k2[[0, 2]]) and torch.equal(v[:2], v2[[0, 2]])


@pytest.mark.parametrize("batch,new,group", [(300, 1, 1), (520, 5, 4)])
def test_shares_of_more_units_than_32_bits_divide(cuda, batch, new, group):
    """Sequences of 131072 positions or so that share one table's pages: more than 2^21 units (a block of 64 keys for few rows, of 128
    for more, and two for each item), whose shares take 64-bit products. A sample of the sequences against the formula."""
    page, kv_heads, dim, most = 256, 4, 16, 131072
    cache = mq.paged_cache(most // page, kv_heads, page, dim, F16)
    g = torch.Generator(device=cuda).manual_seed(batch)
    for t in (cache.k, cache.v):
        t.normal_(generator=g)
    table = torch.randperm(most // page, generator=g, device=cuda).int().repeat(batch, 1)
    lengths = most - 3 * torch.arange(batch, dtype=torch.int32, device=cuda).flip(0).contiguous()
    assert batch * kv_heads * (2 + (most - 3 * batch) // (64 if new * group <= 16 else 128)) > 2 ** 21
    starts = torch.arange(0, (batch + 1) * new, new, dtype=torch.int32, device=cuda)
    q = (torch.randn(batch * new, kv_heads * group, dim, generator=g, device=cuda) * 4).half()
    mq.device_status()
    out = mq.paged_attention(q, cache, table, lengths, starts, max_new=new)
    assert mq.device_status() == 0
    k, v = (t[table[0].long()].transpose(0, 1).reshape(kv_heads, most, dim).double() for t in (cache.k, cache.v))
    for b in {0, 1, batch // 3, batch // 2, batch - 2, batch - 1}:
        rows = q[b * new:(b + 1) * new].double().view(new, kv_heads, group, dim)
        z = torch.einsum("tkgd,kld->tkgl", rows, k) * dim ** -0.5
        end = int(lengths[b])
        z = z.masked_fill(torch.arange(most, device=cuda) > torch.arange(end - new, end, device=cuda)[:, None, None, None], -float("inf"))
        p = z.softmax(-1)
        ref, size = torch.einsum("tkgl,kld->tkgd", p, v), torch.einsum("tkgl,kld->tkgd", p, v.abs())
        big = dim ** -0.5 * torch.einsum("tkgd,kd->tkg", rows.abs(), k.abs().amax(1))
        bound = 2.0 ** -11 * ref.abs() + (2 * 2.0 ** -11 + 2 * (dim + 16) * 2.0 ** -23 * big + 2.0 ** -19)[..., None] * size + 2.0 ** -24 + \
            2.0 ** -25 * p.amax(-1)[..., None] * v.abs().sum(1)[:, None]
        err = (out[b * new:(b + 1) * new].double().view_as(ref) - ref).abs()
        assert (err <= bound).all(), (b, float((err / bound).max()))


@pytest.mark.parametrize("cache,x", CACHES)
@pytest.mark.parametrize("batch", [16, 17, 40])
@pytest.mark.parametrize("new", [(5,), (13, 1, 1, 1), (8, 1), (8, 7, 6, 5), (1, 2, 3, 4, 5, 6, 7, 8)])
def test_drafted_and_single_tokens_in_one_batch(cuda, cache, x, batch, new):
    """Mixes for which the plan takes one launch or two."""
    rng = np.random.default_rng(batch)
    sizes = [(new[b % len(new)], new[b % len(new)] + int(rng.integers(0, 300))) for b in range(batch)]
    attend(Batch(cuda, sizes, 2, 16, 64, cache), 16, x, max_new=max(new))


def test_workspace_that_shares_memory(cuda):
    cache = mq.paged_cache(4, 2, 16, 64)
    table = torch.zeros(1, 4, dtype=torch.int32, device=cuda)
    lengths = torch.ones(1, dtype=torch.int32, device=cuda)
    nbytes = mq.paged_attention_workspace(cache, 8, 1, 1)
    buf = torch.zeros(nbytes + 2048, dtype=torch.uint8, device=cuda)
    inside, behind = (buf[at:at + 1024].view(F16).view(1, 8, 64) for at in (nbytes // 2 // 16 * 16, (nbytes + 15) // 16 * 16))
    clear = torch.zeros(1, 8, 64, device=cuda, dtype=F16)
    for q, out in ((inside, clear), (clear, inside), (inside, inside)):
        with pytest.raises(mq.MQError, match="workspace shares memory"):
            mq.paged_attention(q, cache, table, lengths, out=out, workspace=buf)
    pool = buf[:4 * 2 * 16 * 64 * 2].view(F16).view(4, 2, 16, 64)
    with pytest.raises(mq.MQError, match="workspace shares memory"):
        mq.paged_attention(clear, mq.PagedCache(pool, cache.v), table, lengths, workspace=buf)
    mq.device_status()
    assert (mq.paged_attention(behind, cache, table, lengths, workspace=buf[:nbytes]) == 0).all() and mq.device_status() == 0
