"""Beam search's selection and the reordering of states. Scores are fp32: each of the two operations rounds
once and lse carries a few roundings of its own, so |error| <= 8 * 2^-24 * (|score| + |logit| + |lse|);
indices are equal wherever no two candidates of different beams are that near (stated per test)."""
import numpy as np
import pytest
import torch

from oracle import serving

import mq

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INF = float("inf")


def t(a, cuda, dtype=None):
    x = torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    return x if dtype is None else x.to(dtype)


def select(logits, scores, cuda, finished=None, eos=-1, dtype=torch.float32, pad=0):
    rows, vocab = logits.shape
    wide = torch.full((rows, vocab + pad), 1e4, device=cuda, dtype=dtype)
    wide[:, pad:] = t(logits, cuda, dtype)
    args = dict(finished=None if finished is None else t(finished.astype(np.uint8), cuda), eos=eos)
    got = mq.beam_select(wide[:, pad:], t(scores.astype(np.float32), cuda), **args)
    z = wide[:, pad:].double().cpu().numpy()
    return [g.cpu().numpy() for g in got], serving.beam_scores(z, scores.astype(np.float32), finished, eos)


def grid(rng, batch, beams, vocab, steps=64):
    """Logits in steps of 1/8 (many equal ones, exact in every type) and scores whose fractions keep the
    beams apart: no two candidates of different beams come within 1e-3 of one another unless equal."""
    z = rng.integers(-steps, steps, (batch * beams, vocab)) / 8.0
    return z.astype(np.float32), (-20 - np.sort(rng.permutation(batch * beams * 4)[:batch * beams].reshape(batch, beams), -1) / 7.0).astype(np.float32)


def check(got, cand, beams, size=None):
    """size: the largest |score| + |logit| + |lse| where it is above the 3 |score| of the other tests."""
    scores, tokens, parents, _ = got
    ref, rp, rt = serving.beam_select(cand)
    fin = np.isfinite(ref)
    np.testing.assert_array_equal(fin, np.isfinite(scores))
    # |logit|, |lse| <= 16 here (steps of 1/8 up to 8, vocabularies below e^8 times that)
    np.testing.assert_allclose(scores[fin], ref[fin], atol=8 * U * size if size else 0, rtol=8 * U * (1 + 40 / 20))
    flat = cand.reshape(cand.shape[0], -1)
    for b in range(flat.shape[0]):  # the precondition: the best candidates of different beams are apart
        top = np.argsort(-flat[b], kind="stable")[:beams + 1]
        for x, y in zip(top, top[1:]):
            assert x // cand.shape[2] == y // cand.shape[2] or not np.isfinite(flat[b][y]) or flat[b][x] - flat[b][y] > 1e-4
    np.testing.assert_array_equal(parents, rp)
    np.testing.assert_array_equal(tokens, rt)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,beams,vocab,pad,seed", [(1, 1, 1, 0, 0), (1, 4, 1, 0, 0), (2, 3, 2, 0, 0), (3, 4, 5, 1, 0),
                                                       (2, 2, 255, 0, 0), (1, 4, 4095, 0, 0), (1, 4, 4097, 3, 0),
                                                       (5, 8, 1000, 0, 0), (1, 32, 3001, 0, 0), (2, 5, 20011, 0, 0),
                                                       (40, 6, 517, 0, 0), (1, 2, 151669, 0, 0)])
def test_select(cuda, batch, beams, vocab, pad, seed, dtype):
    rng = np.random.default_rng([seed, batch, beams, vocab])
    # few steps in bf16's 8 bits; distinct tops per row keep the beams apart
    z, scores = grid(rng, batch, beams, vocab, 16)
    got, cand = select(z, scores, cuda, dtype=dtype, pad=pad)
    flat = np.sort(cand.reshape(batch, -1), -1)[:, ::-1][:, :beams + 1]
    gaps = flat[:, :-1] - flat[:, 1:]
    if np.any((gaps > 0) & (gaps < 1e-4)):
        pytest.fail("the inputs do not keep the beams apart: choose another seed")
    check(got, cand, beams)
    assert mq.device_status() == 0


@pytest.mark.parametrize("kind", ["rising", "falling", "equal", "masked", "one"])
@pytest.mark.parametrize("vocab", [3, 700, 9000, 40000])
def test_select_orders_and_masks(cuda, kind, vocab):
    beams = 4
    z = np.zeros((2 * beams, vocab), np.float32)
    ramp = (np.arange(vocab) % 30000 / 4096).astype(np.float32)
    if kind in ("rising", "falling"):
        z[:] = ramp if kind == "rising" else ramp[::-1]
    if kind == "masked":
        z[:] = -INF
        z[:, vocab // 2] = 1.0
        z[3] = -INF  # a row that its mask leaves empty
    if kind == "one":
        z[:] = -INF
        z[0, vocab - 1] = 3
    scores = np.array([[-1, -1.37, -2.71, -3.05]] * 2, np.float32)
    scores[1, 1:] = -INF  # a first step: one beam in use
    got, cand = select(z, scores, cuda)
    check(got, cand, beams)
    assert mq.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [3, 5000, 33000])
def test_select_masks_of_the_lowest_value(cuda, dtype, vocab):
    """Masks of the type's lowest finite value: they count as what they are, in a row that has nothing else too."""
    rng = np.random.default_rng(vocab)
    low = float(torch.finfo(dtype).min)
    z = np.full((4, vocab), low)
    z[0, rng.integers(0, vocab, 7)] = 1.5
    z[1, : vocab // 2] = rng.integers(-16, 16, vocab // 2) / 8.0
    z[2, vocab - 1] = low / 2  # (rows 2 and 3: nothing of a usual size)
    for b, scores in enumerate(([-1, -2.37], [-3, -5.71], [-15.71, -3])):  # the third: row 3, all masked, is the best
        rows = z[2 * min(b, 1):][:2].astype(np.float32)
        scores = np.array([scores], np.float32)
        got, _ = select(rows, scores, cuda, dtype=dtype)
        # fp16's lowest value leaves lse some last bits; the others' swallows everything beside it
        check(got, serving.beam_scores(rows, scores, None, -1), 2, 3 * abs(low) if b and dtype == torch.float16 else None)
    assert mq.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [3, 5000, 33000])
@pytest.mark.parametrize("size", [1e5, 3e6, 1e9, 1e10, 1e30, 3e37])
def test_select_rows_of_one_huge_magnitude(cuda, size, vocab, dtype):
    """A row all of whose logits are far from zero, as masks of -1e9 or -1e30 make one, is a row like any other; so
    is one where such values stand beside usual ones."""
    rng = np.random.default_rng(vocab)
    usual = (rng.integers(-16, 16, vocab) / 8.0).astype(np.float32)
    for mask in (-size, size):
        z = np.stack([usual, np.full(vocab, mask, np.float32)])
        z[1] = t(z[1:], cuda, dtype).float().cpu().numpy()
        # lse swallows what is beside it, so such a token scores between scores[1] - log(vocab) and scores[1]: best of all
        got, cand = select(z, np.array([[-40, -3]], np.float32), cuda, dtype=dtype)
        check(got, cand, 2, 3 * size)
    z[1, : vocab // 2 + 1] = -abs(z[1, 0])  # a part that is masked, the rest is usual
    z[1, vocab // 2 + 1:] = usual[vocab // 2 + 1:]
    got, cand = select(z, np.array([[-40, -3.37]], np.float32), cuda, dtype=dtype)
    check(got, cand, 2)
    assert mq.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("vocab", [1000, 40000])
def test_select_takes_equal_scores_of_dropped_tokens(cuda, vocab, dtype):
    """Tokens 100 and 101 are one step of the type above tokens 10 and 20. Where the step is lost in the scores'
    rounding the lower two win, else the upper two; one of each is never right. The logits start at one of eight
    neighbouring values per request, so that the rounding falls differently."""
    base, score = (5.0, -25.0) if dtype == torch.float32 else (0.2, -3000.0)
    one = torch.tensor(base, dtype=dtype)
    bits = one.view(torch.int32 if dtype == torch.float32 else torch.int16)
    ladder = torch.stack([(bits + j).view(dtype) for j in range(9)]).float().numpy()
    for upper in ((100, 101), (vocab - 2, vocab - 1)):
        z = np.full((8, 3, vocab), -2, np.float32)
        z[:, 0, vocab // 2] = 8  # the best one, and most of lse
        for j in range(8):
            z[j, 0, [10, 20]] = ladder[j]
            z[j, 0, list(upper)] = ladder[j + 1]
        scores = np.full((8, 3), -INF, np.float32)
        scores[:, 0] = score
        (_, tokens, parents, _), _ = select(z.reshape(24, vocab), scores, cuda, dtype=dtype)
        assert (tokens[:, 0] == vocab // 2).all() and (parents == 0).all()
        pairs = [tuple(row) for row in tokens[:, 1:]]
        assert set(pairs) == {(10, 20), upper}, pairs


def test_select_takes_equal_scores_by_index(cuda):
    """Unequal logits far below the score's last bit: every token of the beam scores the same, so the first
    tokens win, wherever the largest logits are."""
    rng = np.random.default_rng(0)
    z = (rng.standard_normal((4, 10007)) * 1e-8).astype(np.float32)
    scores = np.array([[-25, -26, -27, -28]], np.float32)
    (s, tokens, parents, _), _ = select(z, scores, cuda)
    np.testing.assert_array_equal(tokens, [[0, 1, 2, 3]])
    np.testing.assert_array_equal(parents, [[0, 0, 0, 0]])
    z[0, 5000] = 0.5  # one above the ties: first, then the ties from the start
    (s, tokens, parents, _), _ = select(z, scores, cuda)
    np.testing.assert_array_equal(tokens, [[5000, 0, 1, 2]])


def test_select_finished_beams(cuda):
    rng = np.random.default_rng(3)
    z, scores = grid(rng, 6, 4, 333, 16)
    finished = rng.random((6, 4)) < 0.5
    finished[0], finished[1] = True, [True, False, False, False]
    scores[1, 1:] = -INF
    got, cand = select(z, scores, cuda, finished, eos=7)
    check(got, cand, 4)
    ended = np.take_along_axis(finished, got[2], -1) | (got[1] == 7)
    np.testing.assert_array_equal(got[3].astype(bool), ended)
    np.testing.assert_array_equal(np.sort(got[0][0])[::-1], np.sort(scores[0])[::-1])  # unchanged


@pytest.mark.parametrize("value", [float("nan"), INF])
def test_select_drops_and_reports_a_beam_that_is_not_finite(cuda, value):
    rng = np.random.default_rng(4)
    z, scores = grid(rng, 2, 3, 5000, 16)
    z[1, 4321] = value
    mq.device_status()
    (s, tokens, parents, _), _ = select(z, scores, cuda)
    assert mq.device_status() == 15
    z[1] = -INF
    cand = serving.beam_scores(z, scores, None, -1)
    check((s, tokens, parents, None), cand, 3)


def test_select_in_place_and_no_requests(cuda):
    rng = np.random.default_rng(5)
    z, scores = grid(rng, 3, 4, 1000, 16)
    dz, ds = t(z, cuda), t(scores, cuda)
    want = mq.beam_select(dz, ds, finished=torch.zeros(3, 4, dtype=torch.bool, device=cuda), eos=3)
    flags = torch.zeros(3, 4, dtype=torch.uint8, device=cuda)
    got = mq.beam_select(dz, ds, finished=flags, eos=3, next_scores=ds, next_finished=flags)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and got[0] is ds
    empty = mq.beam_select(torch.empty(0, 10, device=cuda), torch.empty(0, 4, device=cuda))
    assert empty[0].shape == (0, 4)


def test_select_random_logits_are_the_best(cuda):
    """Continuous logits: the chosen are the best up to the scores' error, in order, without repetition."""
    rng = np.random.default_rng(6)
    batch, beams, vocab = 3, 8, 50257
    z = (rng.standard_normal((batch * beams, vocab)) * 2.5).astype(np.float32)
    z[rng.random(z.shape) < 0.05] = -INF
    scores = -np.sort(rng.uniform(20, 30, (batch, beams)), -1).astype(np.float32)
    (s, tokens, parents, _), cand = select(z, scores, cuda)
    tol = 8 * U * 80
    for b in range(batch):
        flat = parents[b].astype(np.int64) * vocab + tokens[b]
        assert len(set(flat)) == beams and (np.diff(s[b]) <= 0).all()
        exact = cand[b].reshape(-1)
        assert np.abs(exact[flat] - s[b]).max() <= tol
        rest = np.delete(exact, flat)
        assert rest.max() <= exact[flat].min() + 2 * tol


def test_select_refusals(cuda):
    z, s = torch.randn(8, 100, device=cuda), torch.zeros(2, 4, device=cuda)
    f = torch.zeros(2, 4, dtype=torch.uint8, device=cuda)
    for bad, match in (((z[:7], s), "rows"), ((z, s[0]), "batch, beams"), ((z.double(), s), "dtype"),
                       ((z.T.contiguous().T, s), "contiguous")):
        with pytest.raises(mq.MQError, match=match):
            mq.beam_select(*bad)
    with pytest.raises(mq.MQError, match="eos"):
        mq.beam_select(z, s, finished=f)
    with pytest.raises(mq.MQError, match="eos"):
        mq.beam_select(z, s, eos=100)
    with pytest.raises(mq.MQError, match="beams is above 32"):
        mq.beam_select(torch.randn(33, 100, device=cuda), torch.zeros(1, 33, device=cuda))
    with pytest.raises(mq.MQError, match="workspace"):
        mq.beam_select(z, s, workspace=torch.empty(16, dtype=torch.uint8, device=cuda))


def reordered(x, parents):
    batch, beams = parents.shape
    base = (torch.arange(batch, device=x.device) * beams)[:, None]
    return x[(base + parents).view(-1)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, torch.uint8, torch.int64])
@pytest.mark.parametrize("batch,beams,shape", [(1, 1, (5,)), (1, 4, (1,)), (3, 2, (7,)), (2, 5, (3, 33)), (1, 16, (4, 10, 8)),
                                               (4, 32, (64,)), (70, 3, (2, 3, 128))])
def test_reorder(cuda, batch, beams, shape, dtype):
    g = torch.Generator(device=cuda).manual_seed(batch + beams)
    x = [torch.randint(0, 200, (batch * beams, *shape), generator=g, device=cuda).to(dtype) for _ in range(3)]
    parents = torch.randint(0, beams, (batch, beams), generator=g, device=cuda, dtype=torch.int32)
    want = [reordered(a, parents.long()) for a in x]
    mq.beam_reorder(x, parents)
    assert all(torch.equal(a, b) for a, b in zip(x, want))
    assert mq.device_status() == 0


@pytest.mark.parametrize("perm", [(0, 1, 2, 3), (0, 2, 1, 3), (1, 0, 2, 3), (2, 0, 3, 1), (1, 2, 0, 3)])
@pytest.mark.parametrize("cut", [(slice(None),) * 3, (slice(None), slice(0, 5), slice(None)), (slice(1, 3), slice(2, 7), slice(1, 9)),
                                 (slice(0, 0),) * 3])
def test_reorder_views(cuda, perm, cut):
    """Caches in any order of their dimensions, and slices of them; what lies outside a slice stays."""
    g = torch.Generator(device=cuda).manual_seed(1)
    sizes = (12, 4, 9, 16)
    full = torch.randn([sizes[i] for i in perm], generator=g, device=cuda).half()
    state = full.permute([perm.index(i) for i in range(4)])  # [rows, heads, length, dim]
    part = state[(slice(None), *cut)]
    parents = torch.randint(0, 4, (3, 4), generator=g, device=cuda, dtype=torch.int32)
    want = state.clone()
    want[(slice(None), *cut)] = reordered(part, parents.long())
    mq.beam_reorder(part, parents)
    assert torch.equal(state, want)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.uint8])
def test_reorder_of_one_number_per_beam(cuda, dtype):
    """States [batch * beams]: lengths, positions, flags; also a column of a table."""
    parents = torch.tensor([[1, 1, 0, 2], [3, 0, 0, 0]], dtype=torch.int32, device=cuda)
    x, table = torch.arange(8, device=cuda).to(dtype), torch.arange(24, device=cuda).to(dtype).view(8, 3)
    want, column = reordered(x, parents.long()), reordered(table[:, 1], parents.long())
    others = table[:, [0, 2]]
    mq.beam_reorder([x, table[:, 1]], parents)
    assert torch.equal(x, want) and torch.equal(table[:, 1], column) and torch.equal(table[:, [0, 2]], others)
    with pytest.raises(mq.MQError, match="shape"):
        mq.beam_reorder(x.sum(), parents)


def test_reorder_of_states_beside_and_inside_one_another(cuda):
    """Keys and values of all layers in one tensor are moved together; a tensor given twice is refused and stays."""
    parents = torch.tensor([[1, 1, 0, 2], [3, 0, 0, 0]], dtype=torch.int32, device=cuda)
    cache = torch.randn(8, 3, 2, 10, 4, 16, device=cuda)  # [rows, layers, keys and values, length, heads, dim]
    want = cache.clone()
    want[:, :, :, :7] = reordered(cache, parents.long())[:, :, :, :7]
    mq.beam_reorder([cache[:, i, j, :7] for i in range(3) for j in range(2)], parents)
    assert torch.equal(cache, want)
    for pair in ([cache, cache], [cache[:, 0, 0, :7], cache[:, 1, 0, :7], cache[:, 0, 0, 2:9]]):
        with pytest.raises(mq.MQError, match="one another"):
            mq.beam_reorder(pair, parents)
    assert torch.equal(cache, want) and mq.device_status() == 0


def test_reorder_past_32_bits_and_many_tensors(cuda):
    """A request's state more than 4 GiB from the first one's, and more tensors than one launch takes."""
    big = torch.empty(4, 1400 << 20, dtype=torch.uint8, device=cuda)
    for i in range(4):
        big[i] = i + 1
    mq.beam_reorder(big[:, (1400 << 20) - 100000:], torch.tensor([[1, 0], [1, 1]], dtype=torch.int32, device=cuda))
    assert [int(big[i, -1]) for i in range(4)] == [2, 1, 4, 4] and [int(big[i, 0]) for i in range(4)] == [1, 2, 3, 4]
    del big
    many = [torch.full((2, 24), float(i), device=cuda) for i in range(130)]
    for x in many:
        x[1] += 0.5
    mq.beam_reorder(many, torch.tensor([[1, 1]], dtype=torch.int32, device=cuda))
    assert all((x == i + 0.5).all() for i, x in enumerate(many))


def test_reorder_reports_a_bad_parent_and_keeps_its_beam(cuda):
    x = torch.arange(12, device=cuda).view(3, 4).float()
    want = x[[1, 1, 0]]
    want[1] = x[1]
    mq.device_status()
    mq.beam_reorder(x, torch.tensor([[1, 7, 0]], dtype=torch.int32, device=cuda))
    assert mq.device_status() == 16 and torch.equal(x, want)


def test_reorder_refuses_before_it_moves_anything(cuda):
    good, bad = torch.randn(8, 16, device=cuda), torch.randn(7, 16, device=cuda)
    kept = good.clone()
    with pytest.raises(mq.MQError, match="shape"):
        mq.beam_reorder([good, bad], torch.tensor([[1, 0, 0, 0], [3, 3, 3, 3]], dtype=torch.int32, device=cuda))
    assert torch.equal(good, kept)


@pytest.mark.parametrize("bad", ["expanded", "overlapping", "twice"])
def test_reorder_moves_all_layouts_or_none(cuda, bad):
    """A state of a second layout that only the library refuses: the first layout's states stay too."""
    good, x = torch.randn(8, 16, device=cuda), torch.randn(9, 32, device=cuda)
    second = {"expanded": [x[0].expand(8, 32)], "overlapping": [x.as_strided((8, 24), (16, 1))], "twice": [x[:8], x[:8]]}[bad]
    kept, parents = (good.clone(), x.clone()), torch.tensor([[1, 0, 0, 0], [3, 3, 3, 3]], dtype=torch.int32, device=cuda)
    with pytest.raises(mq.MQError, match="overlap"):
        mq.beam_reorder([good, *second], parents)
    assert torch.equal(good, kept[0]) and torch.equal(x, kept[1])


def test_reorder_refusals(cuda):
    x, p = torch.randn(8, 16, device=cuda), torch.zeros(2, 4, dtype=torch.int32, device=cuda)
    with pytest.raises(mq.MQError, match="shape"):
        mq.beam_reorder(x[:7], p)
    with pytest.raises(mq.MQError, match="dtype"):
        mq.beam_reorder(x, p.long())
    with pytest.raises(mq.MQError, match="overlap"):
        mq.beam_reorder(x.view(-1).as_strided((8, 16), (8, 1)), p)
    with pytest.raises(mq.MQError, match="overlap"):
        mq.beam_reorder(x[:1].expand(8, 16), p)
    with pytest.raises(mq.MQError, match="beams is above 32"):
        mq.beam_reorder(torch.randn(40, 16, device=cuda), torch.zeros(1, 40, dtype=torch.int32, device=cuda))
