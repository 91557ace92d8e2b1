"""One decode step of the int8, norm and beam operators with int4 products between them, as a CUDA graph and on
another stream: the same bits as eagerly on the first stream."""
import numpy as np
import pytest
import torch

import mq
from mq import synth

pytestmark = pytest.mark.gpu


class Step:
    def __init__(self, cuda, rows=8, d=512, f=768, vocab=5003):
        rng = np.random.default_rng(0)
        g = torch.Generator(device=cuda).manual_seed(0)
        wq, ws = synth.q4_matrix(rng, d, d, 32)
        self.q4 = torch.from_numpy(wq.view(np.int32)).to(cuda), torch.from_numpy(ws).to(cuda)
        self.x = torch.randn(rows, d, generator=g, device=cuda)
        self.w = [torch.rand(d, generator=g, device=cuda) + 0.5 for _ in range(3)]
        self.gate = torch.randn(2, d, generator=g, device=cuda)
        self.gate_up = mq.quantize_s8(torch.randn(2 * f, d, generator=g, device=cuda) * d ** -0.5)
        self.down = mq.quantize_s8(torch.randn(d, f, generator=g, device=cuda) * f ** -0.5)
        self.head = mq.quantize_s8(torch.randn(vocab, d, generator=g, device=cuda) * 3 * d ** -0.5)
        self.scores = torch.arange(rows, device=cuda).view(2, -1) * -0.37
        self.state = torch.randn(rows, 2, 33, 64, generator=g, device=cuda)
        self.lengths = torch.arange(rows, device=cuda)
        self.d = d
        n = mq.lib.mq_beam_workspace_size(2, rows // 2, vocab)
        self.workspace = torch.empty(n, dtype=torch.uint8, device=cuda)

    def __call__(self):
        d, state, lengths = self.d, self.state.clone(), self.lengths.clone()
        mixed = [torch.empty(4, d, device=self.x.device) for _ in range(2)]
        for i, y in enumerate(mixed):  # int4 products, whose weights are copied early where the kernel before lets them
            mq.gemv_q4(*self.q4, self.x[4 * i:4 * i + 4], y, d, group=32)
        x = torch.cat(mixed)
        q, s = mq.pre_norm_s8(x, self.w[0])
        a = mq.gate_up_w8a8(q, s, *self.gate_up, dtype=torch.float32)
        y = mq.gemm_w8a8(*mq.quantize_s8(a), *self.down, dtype=torch.float32)
        out, h = mq.post_norm(y, self.w[1], x, self.w[2], gate=self.gate, scale=0.5)
        again = torch.empty(4, d, device=self.x.device)
        mq.gemv_q4(*self.q4, h[:4], again, d, group=32)  # right behind a norm that lets it start early
        y[:4] += again
        out, q, s = mq.post_norm_s8(y, None, out, self.w[0])
        logits = mq.gemm_w8a8(q, s, *self.head, dtype=torch.float16)
        picked = mq.beam_select(logits, self.scores, workspace=self.workspace)
        after = torch.empty(4, d, device=self.x.device)
        mq.gemv_q4(*self.q4, out[:4], after, d, group=32)  # right behind the selection
        mq.beam_reorder([state, lengths], picked[2])
        return [x, a, out, h, again, logits, after, *picked, state, lengths]


def test_step_as_a_graph_and_on_another_stream(cuda):
    step = Step(cuda)
    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    assert mq.device_status() == 0
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, captured))
    assert mq.device_status() == 0
