"""The int8 decode loop end to end: each hypothesis that beam search returns scores the same when it is decoded
alone, so products, norms, selection, parents and the caches that follow their beams fit together."""
import importlib.util
import os

import pytest
import torch

from conftest import PKG

import mq

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("int8_beam_decode", os.path.join(PKG, "examples", "int8_beam_decode.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("batch,beams,steps,vocab,d,f", [(1, 1, 3, 50, 64, 96), (2, 4, 12, 2000, 256, 512), (5, 8, 6, 777, 200, 333)])
def test_hypotheses_score_the_same_alone(cuda, example, batch, beams, steps, vocab, d, f):
    model = example.Decoder(vocab=vocab, d=d, f=f, layers=2)
    start = torch.arange(5, 5 + batch, device=cuda)
    sequences, scores = example.decode(model, start, beams, steps)
    alone = example.score(model, start, sequences)
    # a row of a product does not depend on the other rows, so only the sums of log-probabilities differ: two
    # fp32 roundings of numbers below 256 per step
    assert (scores.double() - alone).abs().max().item() <= 2 * steps * 256 * 2.0 ** -24
    assert (scores[:, :-1] >= scores[:, 1:]).all()
    flat = sequences.view(batch, beams, -1)
    assert all(len({tuple(s) for s in flat[b].tolist()}) == beams for b in range(batch))
    assert mq.device_status() == 0
