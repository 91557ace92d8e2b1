"""Verification of drafted tokens over libmq (beam_select's and head_argmax's place where a drafter proposes several
tokens at once).
"""
import torch

from ._lib import MQError, lib
from .int8 import _F32, _current_device, _flat, _rows, _stream
from .pack import _DT

__all__ = ["verify_drafts", "verify_workspace"]

_I32 = frozenset((torch.int32,))


def verify_workspace(batch, drafts, vocab):
    """The bytes of a workspace for verify_drafts; enough for fewer requests, drafts or tokens too."""
    return max(lib.mq_verify_workspace_size(batch, drafts, vocab), 16)


def verify_drafts(target, drafted, uniform, draft=None, temperature=None, counts=None, tokens=None, accepted=None, logprobs=None,
                  workspace=None):
    """Which drafted tokens stay, so that the tokens are distributed as the target's own samples. target: logits fp32 /
    fp16 / bf16 [batch * (drafts + 1), vocab]; drafted int32 [batch, drafts]; uniform fp32 [batch, drafts + 1] in [0, 1);
    draft: the drafter's logits [batch * drafts, vocab] of target's type (None: its tokens came without a distribution);
    temperature fp32 [batch] (None: 1; 0: greedy); counts int32 [batch]: how many drafts each request has (None: all).
    Token i is kept while uniform * q(token) < p(token), with p and q the softmax of the logits / temperature; at the
    first that is not, one is drawn from max(p - q, 0), from p where all are kept or the two are the same, with the last uniform. Returns (tokens
    int32 [batch, drafts + 1]: the kept ones, the drawn one, then -1; accepted int32 [batch]; logprobs fp32 [batch,
    drafts + 1]: the target's log-probability of each, 0 behind). Outputs and workspace may not share memory with the inputs."""
    if not isinstance(drafted, torch.Tensor) or drafted.dim() != 2:
        raise MQError(-1, "drafted: expected a [batch, drafts] tensor")
    batch, drafts = drafted.shape
    _, vocab, ld = _rows(target, "target", _DT, None, batch * (drafts + 1))
    if draft is None:
        draft_p, ld_draft = None, 0
    else:
        if not isinstance(draft, torch.Tensor) or draft.dtype != target.dtype:
            raise MQError(-1, "draft: expected a tensor of target's type")
        ld_draft = _rows(draft, "draft", _DT, vocab, batch * drafts)[2]
        draft_p = draft.data_ptr()
    device = target.get_device()
    if tokens is None:
        tokens = torch.empty(batch, drafts + 1, dtype=torch.int32, device=target.device)
    if accepted is None:
        accepted = torch.empty(batch, dtype=torch.int32, device=target.device)
    if logprobs is None:
        logprobs = torch.empty(batch, drafts + 1, dtype=torch.float32, device=target.device)
    if workspace is None:
        workspace = torch.empty(verify_workspace(batch, drafts, vocab), dtype=torch.uint8, device=target.device)
    for t, name in ((drafted, "drafted"), (uniform, "uniform"), (draft, "draft"), (temperature, "temperature"), (counts, "counts"),
                    (tokens, "tokens"), (accepted, "accepted"), (logprobs, "logprobs"), (workspace, "workspace")):
        if t is not None and (not isinstance(t, torch.Tensor) or t.get_device() != device):
            raise MQError(-1, f"{name}: is not on target's device")
    if device != _current_device():
        raise MQError(-1, f"target: is on device {device}, not on the current one")
    n = batch * (drafts + 1)
    lib.call("mq_verify_drafts", target.data_ptr(), ld, draft_p, ld_draft, _DT[target.dtype], _flat(drafted, "drafted", _I32, batch * drafts),
             None if counts is None else _flat(counts, "counts", _I32, batch), _flat(uniform, "uniform", _F32, n),
             None if temperature is None else _flat(temperature, "temperature", _F32, batch), _flat(tokens, "tokens", _I32, n),
             _flat(accepted, "accepted", _I32, batch), _flat(logprobs, "logprobs", _F32, n), batch, drafts, vocab,
             _flat(workspace, "workspace", (torch.uint8,), workspace.numel()), workspace.numel(), _stream())
    return tokens, accepted, logprobs
