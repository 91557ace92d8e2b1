"""Beam search through a small int8 decoder: the int8 products, the norms around a block and the beam-search
step as one decode loop.

    python mojo-adreno_b200/examples/int8_beam_decode.py [--batch 2 --beams 4 --steps 12]

Each layer is a SwiGLU block with a norm before and one after it, a gate per channel and a residual scale; in
the place of attention a token sees a decayed sum of its hypothesis' earlier block outputs, kept per layer in
a cache that has to follow its beam. Weights are random, quantised once. A layer's launches:

    gate_up_w8a8 -> quantize_s8 -> gemm_w8a8 -> post_norm_s8   (the next layer's norm and quantisation in it)

and after the last layer the vocabulary head (gemm_w8a8), beam_select and beam_reorder.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import mq  # noqa: E402

EOS = 0


class Decoder:
    def __init__(self, vocab=2000, d=256, f=512, layers=3, most=64, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape, scale=1.0):
            return torch.randn(*shape, generator=g, device="cuda") * scale

        self.vocab, self.d, self.layers, self.most, self.scale = vocab, d, layers, most, 0.5
        self.embedding = normal(vocab, d).bfloat16()
        self.head = mq.quantize_s8(normal(vocab, d, scale=3 / d ** 0.5))
        self.gate_up = [mq.quantize_s8(normal(2 * f, d, scale=d ** -0.5)) for _ in range(layers)]
        self.down = [mq.quantize_s8(normal(d, f, scale=f ** -0.5)) for _ in range(layers)]
        self.gate = [1 + normal(d, scale=0.1) for _ in range(layers)]
        self.norms = [1 + normal(d, scale=0.1) for _ in range(layers + 1)]  # before each layer, and before the head
        self.post = [1 + normal(d, scale=0.1) for _ in range(layers)]

    def caches(self, rows):
        return [torch.zeros(rows, self.most, self.d, dtype=torch.bfloat16, device="cuda") for _ in range(self.layers)]

    def step(self, tokens, caches, at):
        """Logits fp32 [rows, vocab] of the token after `tokens` [rows], which are at position `at`."""
        x = self.embedding[tokens.view(-1).long()]
        decay = 0.8 ** torch.arange(at, 0, -1, device="cuda")
        q, s = mq.pre_norm_s8(x, self.norms[0])
        for i in range(self.layers):
            a = mq.gate_up_w8a8(q, s, *self.gate_up[i], dtype=torch.bfloat16)
            y = mq.gemm_w8a8(*mq.quantize_s8(a), *self.down[i], dtype=torch.bfloat16)
            caches[i][:, at] = y
            y = y + (caches[i][:, :at].float() * decay[:, None]).sum(1).bfloat16()
            x, q, s = mq.post_norm_s8(y, self.post[i], x, self.norms[i + 1], gate=self.gate[i], scale=self.scale, out=x)
        return mq.gemm_w8a8(q, s, *self.head, dtype=torch.float32)


def decode(model, start, beams, steps):
    """(sequences int64 [batch, beams, steps], scores [batch, beams]) of beam search from the tokens start [batch]."""
    batch = start.numel()
    tokens = start.view(batch, 1).expand(batch, beams).contiguous()
    scores = torch.full((batch, beams), float("-inf"), device="cuda")
    scores[:, 0] = 0  # the beams are the same at the start: one of them counts
    finished = torch.zeros(batch, beams, dtype=torch.uint8, device="cuda")
    caches = model.caches(batch * beams)
    history = torch.zeros(batch * beams, steps, dtype=torch.int32, device="cuda")
    for at in range(steps):
        logits = model.step(tokens, caches, at)
        scores, tokens, parents, finished = mq.beam_select(logits, scores, finished=finished, eos=EOS)
        mq.beam_reorder([c[:, :at + 1] for c in caches], parents)  # only what is filled
        mq.beam_reorder(history, parents)
        history[:, at] = tokens.view(-1)
    return history.view(batch, beams, steps).long(), scores


def score(model, start, sequences):
    """The score of each hypothesis when it is decoded alone, without selection or reordering."""
    batch, beams, steps = sequences.shape
    tokens = start.view(batch, 1).expand(batch, beams).reshape(-1)
    total = torch.zeros(batch * beams, dtype=torch.float64, device="cuda")
    open_ = torch.ones(batch * beams, dtype=torch.bool, device="cuda")
    caches = model.caches(batch * beams)
    for at in range(steps):
        chosen = sequences.reshape(batch * beams, steps)[:, at]
        logp = torch.log_softmax(model.step(tokens, caches, at).double(), -1)
        total += torch.where(open_, logp.gather(1, chosen[:, None])[:, 0], torch.zeros_like(total))
        open_ &= chosen != EOS
        tokens = chosen
    return total.view(batch, beams)


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--batch", type=int, default=2)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--steps", type=int, default=12)
    a = ap.parse_args()
    model = Decoder()
    start = torch.arange(5, 5 + a.batch, device="cuda")
    sequences, scores = decode(model, start, a.beams, a.steps)
    alone = score(model, start, sequences)
    for b in range(a.batch):
        for i in range(a.beams):
            print(f"request {b} beam {i}: {scores[b, i].item():9.4f} (alone {alone[b, i].item():9.4f}) {sequences[b, i].tolist()}")
    assert mq.device_status() == 0


if __name__ == "__main__":
    main()
