"""The verification of drafted tokens, against the oracle in 64 bits.

Tokens and counts are equal: the drawn token comes from 64-bit sums, and a comparison of u q with p in fp32 decides otherwise only
where they are within 1e-6 of one another, which the tests that look at it keep apart by construction and the random
ones meet with odds of 1e-6 a token. Log-probabilities: z / T - log(sum) where the sum's terms 2^y carry 2 roundings of y (2^-24 |y| each,
and the weighted mean of |y| is below log2(vocab) + 2) and 2^-22 of the exponential, and up to vocab / 256 + 24 roundings of
additions: (2 (log2(vocab) + 2) + 4 + vocab / 256 + 24) 2^-24, and one more of the result."""
import math

import numpy as np
import pytest
import torch

from oracle import paged

import mq

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF = float("inf")


class Case:
    def __init__(self, cuda, batch, drafts, vocab, dtype, draft=True, temperature=None, seed=0, pad=0, spread=2.5, masked=0.1):
        g = torch.Generator(device=cuda).manual_seed(seed)

        def logits(x):  # rows `pad` elements further apart than they are long, not 16-byte aligned then
            wide = torch.full((x.shape[0] * x.shape[1], vocab + pad), 1e4, device=cuda).to(dtype)
            wide[:, pad:] = x.reshape(-1, vocab).to(dtype)
            return wide[:, pad:]

        z = torch.randn(batch, drafts + 1, vocab, generator=g, device=cuda) * spread
        z[torch.rand(z.shape, generator=g, device=cuda) < masked] = -INF
        z[..., vocab // 2] = 0  # no row is masked whole
        y = z[:, :drafts] * 0.9 + torch.randn(batch, drafts, vocab, generator=g, device=cuda)
        self.target, self.draft = logits(z), logits(y) if draft and drafts else None
        t = torch.ones(batch) if temperature is None else torch.tensor([temperature[b % len(temperature)] for b in range(batch)])
        self.temperature = None if temperature is None else t.to(cuda)
        hot = t.to(cuda).view(batch, 1, 1)
        noise = -torch.log(-torch.log(torch.rand(batch, drafts, vocab, generator=g, device=cuda).clamp(1e-7, 1 - 1e-7)))
        self.drafted = (y.to(dtype).float() + noise * hot).argmax(-1).int() if drafts else torch.empty(batch, 0, dtype=torch.int32, device=cuda)
        self.uniform = torch.rand(batch, drafts + 1, generator=g, device=cuda)
        self.counts = None
        self.batch, self.drafts, self.vocab = batch, drafts, vocab

    def call(self, **kw):
        return mq.verify_drafts(self.target, self.drafted, self.uniform, draft=self.draft, temperature=self.temperature,
                                counts=self.counts, **kw)

    def check(self, got):
        tokens, accepted, logprobs = (t.cpu().numpy() for t in got)
        z = self.target.double().cpu().numpy().reshape(self.batch, self.drafts + 1, self.vocab)
        y = None if self.draft is None else self.draft.double().cpu().numpy().reshape(self.batch, self.drafts, self.vocab)
        d, u = self.drafted.cpu().numpy(), self.uniform.cpu().numpy()
        for b in range(self.batch):
            t = 1.0 if self.temperature is None else float(self.temperature[b])
            want, n, logp = paged.verify(z[b], d[b], u[b], None if y is None else y[b], t,
                                         None if self.counts is None else int(self.counts[b]))
            assert accepted[b] == n and tokens[b].tolist() == want, (b, accepted[b], n, tokens[b], want)
            unit = 2.0 ** -24 * (2 * (math.log2(self.vocab) + 2) + 4 + self.vocab / 256 + 24)
            np.testing.assert_array_less(np.abs(logprobs[b] - logp), unit + 2.0 ** -24 * np.abs(logp) + 1e-30)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch,drafts,vocab,pad", [(1, 1, 1, 0), (1, 4, 2, 0), (3, 2, 5, 1), (2, 3, 31, 0), (5, 4, 1000, 0), (2, 8, 4099, 3),
                                                  (40, 3, 517, 0), (1, 32, 3001, 0), (2, 4, 20011, 0), (1, 4, 151669, 0), (3, 0, 999, 1)])
@pytest.mark.parametrize("draft", [True, False])
def test_verify(cuda, dtype, batch, drafts, vocab, pad, draft):
    for seed in range(3):
        case = Case(cuda, batch, drafts, vocab, dtype, draft, [1.0, 0.7, 0.0, 1.7, 1e-6], seed, pad)
        mq.device_status()
        got = case.call()
        assert mq.device_status() == 0
        case.check(got)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch", [12, 13, 37, 38])
def test_batches_where_the_draw_is_split_otherwise(cuda, dtype, batch):
    case = Case(cuda, batch, 2, 1501, dtype, True, [1.0, 0.0, 0.7], batch)
    case.check(case.call())


@pytest.mark.parametrize("draft", [True, False])
def test_without_temperature_and_given_outputs(cuda, draft):
    case = Case(cuda, 6, 3, 2003, F32, draft)
    out = dict(tokens=torch.full((6, 4), 7, dtype=torch.int32, device=cuda), accepted=torch.full((6,), 7, dtype=torch.int32, device=cuda),
               logprobs=torch.full((6, 4), 7.0, device=cuda), workspace=torch.empty(mq.verify_workspace(6, 3, 2003), dtype=torch.uint8, device=cuda))
    got = case.call(**out)
    assert all(a is b for a, b in zip(got, out.values()))
    case.check(got)


@pytest.mark.parametrize("u", [0.0, 1 - 2.0 ** -24, 0.5])
def test_uniforms_at_the_ends(cuda, u):
    for seed in range(4):
        case = Case(cuda, 8, 3, 1003, F32, seed % 2 == 0, [1.0, 0.5], seed)
        case.uniform.fill_(u)
        case.check(case.call())


def test_draws_from_every_place(cuda):
    """One request per place of the uniform, a few kinds of rows: the first and the last token, runs of masked ones."""
    batch, vocab = 256, 777
    case = Case(cuda, batch, 1, vocab, F32, False, masked=0.0, spread=0.3)
    case.target[:, :40] = -INF
    case.target[:, 300:600] = -INF
    case.target[:, 770:] = -INF
    case.drafted.fill_(50)
    case.uniform[:, 0] = torch.linspace(0, 1 - 2.0 ** -24, batch, device=cuda)
    case.uniform[:, 1] = torch.linspace(0, 1 - 2.0 ** -24, batch, device=cuda)
    case.check(case.call())
    case.counts = torch.zeros(batch, dtype=torch.int32, device=cuda)  # drawn from p itself
    case.check(case.call())


def test_counts(cuda):
    case = Case(cuda, 9, 4, 601, BF16, True, [1.0, 0.0])
    case.counts = torch.tensor([0, 1, 2, 3, 4, 4, 0, 2, 1], dtype=torch.int32, device=cuda)
    case.target[4 + 5 * 0 + 0:5] = case.target[4:5]
    case.check(case.call())
    mq.device_status()
    case.counts[2] = 99
    case.counts[3] = -1
    got = case.call()
    assert mq.device_status() == 25
    case.check(got)


def test_temperatures_at_the_ends(cuda):
    """An infinite temperature: all tokens that are not masked alike; one that is no number: greedy."""
    case = Case(cuda, 4, 2, 301, F32, True, [1.0])
    case.temperature[:] = torch.tensor([float("inf"), 1e38, float("nan"), -1.0], device=cuda)
    mq.device_status()
    tokens, accepted, logprobs = case.call()
    assert mq.device_status() == 0
    z = case.target.view(4, 3, 301)
    for b in range(2):  # 1 / (tokens that are not masked) each
        for i in range(int(accepted[b]) + 1):
            assert abs(float(logprobs[b, i]) + math.log(int(z[b, i].isfinite().sum()))) < 1e-4
            assert z[b, i, tokens[b, i]].isfinite()
    for b in range(2, 4):
        assert tokens[b, 0] == z[b, 0].argmax()


def test_identical_distributions_keep_all(cuda):
    """Draft and target the same: every token that the draft gives any weight is kept."""
    case = Case(cuda, 16, 5, 3001, F32, True)
    case.draft = case.target.view(16, 6, 3001)[:, :5].reshape(80, 3001).contiguous()
    case.drafted = case.draft.view(16, 5, 3001).argmax(-1).int()
    case.uniform[:, :5] *= 0.999
    got = case.call()
    assert (got[1] == 5).all()
    case.check(got)


def test_greedy_takes_the_lowest_of_equal_logits(cuda):
    case = Case(cuda, 4, 2, 5003, F32, True, [0.0])
    z = case.target.view(4, 3, 5003)
    z[:, :, [4900, 17, 3000, 18]] = 50.0
    case.drafted[:] = 17
    case.drafted[1, 0] = 18
    case.drafted[2, 1] = 3000
    got = case.call()
    assert got[0].tolist() == [[17, 17, 17], [17, -1, -1], [17, 17, -1], [17, 17, 17]]
    assert got[1].tolist() == [2, 0, 1, 2] and (got[2] == 0).all()
    # The first element of an unaligned row is not in its vectors.
    case = Case(cuda, 2, 1, 5003, F16, True, [0.0], pad=3)
    case.target[:, 0] = 60.0
    case.target[:, 5002] = 60.0
    case.drafted.fill_(0)
    assert case.call()[0].tolist() == [[0, 0], [0, 0]]


@pytest.mark.parametrize("offset", [-1e4, 3e4, 1e10, -1e30, 3e38])
def test_logits_of_any_size(cuda, offset):
    """A large common offset, and masks of the type's lowest value."""
    case = Case(cuda, 4, 2, 4001, F32, True, [1.0, 0.5])
    for x in (case.target, case.draft):
        if abs(offset) < 1e6:
            x += offset
        else:  # all but a few tokens masked by a huge finite number, or a few far above the others
            rows = torch.arange(x.shape[0], device=cuda)
            if offset < 0:
                x[:, 100:] = offset
            else:
                x[rows, (rows * 37) % 4001] = offset
    for row in range(8):
        case.drafted.view(-1)[row] = int(case.draft[row].argmax())
    got = case.call()
    assert mq.device_status() == 0
    case.check(got)
    case = Case(cuda, 3, 2, 3001, BF16, True)
    lowest = torch.finfo(BF16).min
    for x in (case.target, case.draft):
        x[:, ::3] = lowest
    case.drafted.clamp_(1, 1)
    case.check(case.call())


@pytest.mark.parametrize("value", [float("nan"), INF, "masked"])
@pytest.mark.parametrize("greedy", [False, True])
def test_rows_that_are_no_distribution(cuda, value, greedy):
    for row in range(3):  # of the target
        case = Case(cuda, 3, 2, 2003, F32, True, [0.0] if greedy else None)
        z = case.target.view(3, 3, 2003)
        if value == "masked":
            z[1, row] = -INF
        else:
            z[1, row, 1999] = value
        case.drafted[:] = z[:, :2].nan_to_num(0, 0, -1e9).argmax(-1)
        case.uniform[:, :2] = 0
        mq.device_status()
        got = case.call()
        case.check(got)
        assert mq.device_status() == 24 and got[1][1] == row and (got[0][1, row:] == -1).all()
    if not greedy:
        case = Case(cuda, 3, 2, 2003, F32, True)
        y = case.draft.view(3, 2, 2003)
        if value == "masked":
            y[1, 0] = -INF
        else:
            y[1, 0, 5] = value
        got = case.call()
        case.check(got)
        assert mq.device_status() == 24 and got[1][1] == 0 and got[0][1, 0] >= 0


def test_drafted_tokens_out_of_range(cuda):
    for draft in (True, False):
        for token in (-1, 2003, 2 ** 31 - 1, -2 ** 31):
            case = Case(cuda, 3, 2, 2003, F32, draft, [1.0, 0.0])
            case.drafted[0, 0] = token
            case.drafted[1, 0] = token
            mq.device_status()
            got = case.call()
            assert mq.device_status() == 25
            case.check(got)


def test_the_only_token_rejected(cuda):
    """Without draft logits, p all on the drafted token and a uniform of 1: nothing is left to draw from."""
    case = Case(cuda, 2, 1, 100, F32, False)
    case.target.fill_(-INF)
    case.target[:, 7] = 3.0
    case.drafted.fill_(7)
    case.uniform.fill_(1.0)
    got = case.call()
    assert got[0].tolist() == [[-1, -1]] * 2 and got[1].tolist() == [0, 0]


def test_captured_and_on_another_stream(cuda):
    case = Case(cuda, 8, 4, 20011, F32, True, [1.0, 0.0])
    want = [t.clone() for t in case.call()]
    out = [torch.empty_like(t) for t in want]
    work = torch.empty(mq.verify_workspace(8, 4, 20011), dtype=torch.uint8, device=cuda)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        case.call(tokens=out[0], accepted=out[1], logprobs=out[2], workspace=work)
    for _ in range(3):
        for t in out:
            t.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = case.call()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_follows_the_target(cuda):
    """Over many requests with the same rows, the first emitted token is distributed as the target's, whatever the
    drafter: 60000 draws over 6 tokens, each frequency within 6 standard deviations."""
    n, vocab = 60000, 6
    g = torch.Generator(device=cuda).manual_seed(3)
    z, y = torch.randn(2, vocab, generator=g, device=cuda)
    q = y.softmax(-1)
    case = Case(cuda, n, 1, vocab, F32, True)
    case.target[:], case.draft[:] = z, y
    case.drafted = torch.multinomial(q, n, replacement=True, generator=g).int().view(n, 1)
    tokens = case.call()[0][:, 0]
    p = z.double().softmax(-1).cpu().numpy()
    seen = np.bincount(tokens.cpu().numpy(), minlength=vocab) / n
    np.testing.assert_array_less(np.abs(seen - p), 6 * np.sqrt(p * (1 - p) / n))


def test_refusals(cuda):
    case = Case(cuda, 2, 3, 100, F32, True)

    def refuses(match, **kw):
        args = dict(target=case.target, drafted=case.drafted, uniform=case.uniform, draft=case.draft)
        args.update(kw)
        with pytest.raises(mq.MQError, match=match):
            mq.verify_drafts(**args)

    refuses("drafted", drafted=case.drafted.long())
    refuses("drafted", drafted=case.drafted.view(-1))
    refuses("target", target=case.target[:5])
    refuses("draft", draft=case.draft.half())
    refuses("draft", draft=case.draft[:, :50])
    refuses("uniform", uniform=case.uniform[:, :2])
    refuses("uniform", uniform=case.uniform.cpu())
    refuses("temperature", temperature=torch.ones(3, device=cuda))
    refuses("counts", counts=torch.ones(2, device=cuda))
    refuses("workspace is too small", workspace=torch.empty(8, dtype=torch.uint8, device=cuda))
    refuses("drafts above", drafted=torch.zeros(2, 33, dtype=torch.int32, device=cuda), uniform=torch.zeros(2, 34, device=cuda),
            target=torch.zeros(68, 100, device=cuda), draft=None)
    with pytest.raises(mq.MQError, match="CUDA"):
        mq.verify_drafts(case.target.cpu(), case.drafted, case.uniform)


@pytest.mark.parametrize("draft", [True, False])
def test_workspace_of_a_larger_batch_serves(cuda, draft):
    """A server has one of its largest batch. What the call leaves alone behind it stays as it was."""
    work = torch.empty(mq.verify_workspace(64, 4, 40009) + 64, dtype=torch.uint8, device=cuda)
    for batch in (1, 5, 7, 8, 9, 10, 11, 13, 18, 21, 64):
        case = Case(cuda, batch, 4, 40009, F16, draft, [1.0, 0.0], seed=batch)
        work.fill_(0x5a)
        case.check(case.call(workspace=work[:-64]))
        assert (work[-64:] == 0x5a).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch", [2, 20, 40])
@pytest.mark.parametrize("shift", [0.0, 64.0, -32.0])
def test_equal_distributions_draw_from_the_target(cuda, dtype, batch, shift):
    """A token that neither can give is drafted, so it is not kept, and nothing is left of p - q: the draw is from p. The logits are whole
    numbers, and the draft's a constant above them (the same probabilities)."""
    vocab = 20000
    case = Case(cuda, batch, 2, vocab, dtype, True, [1.0, 0.7], seed=batch)
    z = case.target.view(batch, 3, vocab)
    z.copy_((z.float() * 2).round().clamp(-INF, 12))
    z[..., 3] = -INF
    case.draft = (z[:, :2].float() + shift).to(dtype).reshape(batch * 2, vocab).contiguous()
    case.drafted[:, 0] = 3
    got = case.call()
    assert (got[1] == 0).all()
    case.check(got)


def test_equal_distributions_and_a_uniform_of_one(cuda):
    case = Case(cuda, 8, 1, 4000, F32, True)
    case.draft = case.target.view(8, 2, 4000)[:, 0].contiguous()
    case.uniform[:, 0] = 1.0
    got = case.call()
    assert (got[1] == 0).all()
    case.check(got)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("batch", [1, 6, 7, 12, 13])
@pytest.mark.parametrize("vocab", [99999, 100003])
def test_long_rows_where_the_draw_is_split_otherwise(cuda, dtype, batch, vocab):
    case = Case(cuda, batch, 1, vocab, dtype, True, [1.0, 0.0, 0.7], batch)
    case.check(case.call())
