"""Beam search over libmq: the selection over beams and vocabulary, and the states that follow their beams
(head_argmax's place when more than one hypothesis is kept).
"""
import ctypes

import torch

from ._lib import MQError, lib
from .int8 import _F32, _flat, _rows, _stream
from .kernels import _need
from .pack import _DT

__all__ = ["beam_select", "beam_reorder"]

_FLAGS = frozenset((torch.uint8, torch.bool))
_I32 = frozenset((torch.int32,))


def beam_select(logits, scores, finished=None, eos=-1, next_scores=None, tokens=None, parents=None, next_finished=None,
                workspace=None):
    """The `beams` best continuations of each request by scores[b, i] + log_softmax(logits[b, i])[v], the lowest
    i * vocab + v among equal ones. logits fp32 / fp16 / bf16 [batch * beams, vocab] (-inf masks a token);
    scores fp32 [batch, beams] (-inf: a beam not in use); finished uint8 / bool [batch, beams]: such a beam
    goes on with `eos` alone, its score unchanged. Returns (next_scores, tokens, parents, next_finished), fp32, int32,
    int32 and uint8 [batch, beams]; the parent is the beam's index within its request. A beam whose logits
    hold a NaN or +inf is dropped and reported by device_status() (15)."""
    if not isinstance(scores, torch.Tensor) or scores.dim() != 2:
        raise MQError(-1, "scores: expected a [batch, beams] tensor")
    batch, beams = scores.shape
    n = batch * beams
    _, vocab, ld = _rows(logits, "logits", _DT, None, n)
    if next_scores is None:
        next_scores = torch.empty_like(scores)
    if tokens is None:
        tokens = torch.empty(batch, beams, dtype=torch.int32, device=logits.device)
    if parents is None:
        parents = torch.empty(batch, beams, dtype=torch.int32, device=logits.device)
    if next_finished is None:
        next_finished = torch.empty(batch, beams, dtype=torch.uint8, device=logits.device)
    if workspace is None:
        workspace = torch.empty(max(lib.mq_beam_workspace_size(batch, beams, vocab), 16), dtype=torch.uint8,
                                device=logits.device)
    else:
        _need(workspace, "workspace", (torch.uint8,))
    lib.call("mq_beam_select", logits.data_ptr(), _DT[logits.dtype], ld, _flat(scores, "scores", _F32, n),
             None if finished is None else _flat(finished, "finished", _FLAGS, n), eos,
             _flat(next_scores, "next_scores", _F32, n), _flat(tokens, "tokens", _I32, n), _flat(parents, "parents", _I32, n),
             _flat(next_finished, "next_finished", _FLAGS, n), batch, beams, vocab, workspace.data_ptr(), workspace.numel(),
             _stream())
    return next_scores, tokens, parents, next_finished


_Three = ctypes.c_int64 * 3


def _layout(t):
    """(row stride, outer sizes, outer strides, inner bytes) of a state [rows, ..] in bytes: its dimensions
    after the first, those without a gap between them merged, the innermost one contiguous."""
    size = t.element_size()
    inner, outer = size, []  # outer: (size, stride), fastest first
    for n, st in sorted(zip(t.shape[1:], t.stride()[1:]), key=lambda d: d[1]):
        st *= size
        if n == 1:
            continue
        if not outer and st == inner:
            inner *= n
        elif outer and st == outer[-1][0] * outer[-1][1]:
            outer[-1] = (outer[-1][0] * n, outer[-1][1])
        else:
            outer.append((n, st))
    if len(outer) > 3:
        raise MQError(-1, "states: at most three gaps between a state's dimensions")
    outer = [(1, 0)] * (3 - len(outer)) + outer[::-1]
    return t.stride(0) * size, [n for n, _ in outer], [st for _, st in outer], inner


def beam_reorder(states, parents):
    """state[b * beams + i] <- state[b * beams + parents[b, i]] in place for each tensor of `states` (one tensor or
    a list, e.g. every layer's keys and values): [batch * beams, ..] of any type, their other dimensions
    in any order, sliced or not (a cache's filled part: cache[:, :, :length]). parents int32 [batch,
    beams], as beam_select gives them. Only beams that change their parent are copied. No two states may share memory
    (refused where they have one layout). Returns states."""
    each = [states] if isinstance(states, torch.Tensor) else list(states)
    if not isinstance(parents, torch.Tensor) or parents.dim() != 2:
        raise MQError(-1, "parents: expected a [batch, beams] tensor")
    batch, beams = parents.shape
    parents_p = _flat(parents, "parents", _I32, batch * beams)
    calls = []  # one for all states of one layout, none before all are checked
    while each:
        first = each[0]
        if not isinstance(first, torch.Tensor):
            raise MQError(-1, "states: expected CUDA tensors (there is no CPU path)")
        shape, stride, dtype = first.shape, first.stride(), first.dtype
        same, rest = [], []
        for t in each:
            if not isinstance(t, torch.Tensor) or not t.is_cuda:
                raise MQError(-1, "states: expected CUDA tensors (there is no CPU path)")
            if t.shape == shape and t.stride() == stride and t.dtype == dtype:
                same.append(t.data_ptr())
            else:
                rest.append(t)
        each = rest
        if not shape or shape[0] != batch * beams:
            raise MQError(-1, f"states: shape {tuple(shape)} is not [{batch * beams}, ..]")
        if 0 not in shape:
            row, outer, strides, inner = _layout(first)
            n = len(same)
            calls.append(((ctypes.c_void_p * n)(*same), n, parents_p, batch, beams, row, _Three(*outer), _Three(*strides), inner))
    if len(calls) > 1:
        for args in calls:
            lib.call("mq_beam_reorder_check", *args)
    stream = _stream()
    for args in calls:
        lib.call("mq_beam_reorder", *args, stream)
    return states
