"""Log probabilities of given tokens, with the entropy and the most likely alternatives.

What a server reports beside its tokens, what a verification step picks from, and what a trainer scores its samples by,
in one pass over the logits.  No counterpart in the reference (its decoder takes the argmax, tiny_model.py:142-157).  A
row's bits depend on that row alone.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

from detkernels_b200 import _lib

MAX_TOP_K = 32


class TokenLogprobs(NamedTuple):
    """The fields that were not asked for are None."""
    logprobs: Optional[object]       # f32 [...]: of the given tokens
    entropy: Optional[object]        # f32 [...]: -sum p log p, in nats
    top_ids: Optional[object]        # int64 [..., top_k]: most likely first, equal logits by their index
    top_logprobs: Optional[object]   # f32 [..., top_k]


def token_logprobs_reference(logits, tokens=None, *, top_k: int = 0, entropy: bool = True):
    """Plain PyTorch form, f32 (f64 stays f64), on any device."""
    import torch

    x = logits if logits.dtype == torch.float64 else logits.float()
    lp = torch.log_softmax(x, dim=-1)
    given = ent = ids = top = None
    if tokens is not None:
        given = lp.gather(-1, tokens.clamp(min=0)[..., None])[..., 0].masked_fill(tokens == -1, 0.0)
    if entropy:
        p = lp.exp()
        ent = -torch.where(p == 0, 0.0, p * lp).sum(-1)
    if top_k:
        # -0 and 0 are equal, and stays in the order of the indices what is
        ids = torch.sort(x + 0.0, dim=-1, descending=True, stable=True).indices[..., :top_k]
        top = lp.gather(-1, ids)
    return TokenLogprobs(given, ent, ids, top)


def token_logprobs(logits, tokens=None, *, top_k: int = 0, entropy: bool = True) -> TokenLogprobs:
    """Log softmax of logits [..., V] at tokens [...], its entropy and the top_k most likely tokens.

    logits: f32, f16 or bf16 CUDA tensor, unit stride along V; other strides are free.  tokens: int64 [...] (None: not
    asked for); -1 asks for nothing there and gives 0, any other token outside [0, V) sets the device status and gives NaN.
    top_k: 0 to 32 alternatives, the largest logit first, equal ones by their index (NaN above all, -0 equal to 0).
    A logit of -infinity has probability 0 and adds nothing to the entropy; a row that holds NaN, +infinity or nothing
    but -infinity has NaN log probabilities and entropy.  f32 arithmetic and outputs; no gradient."""
    import torch

    assert logits.is_cuda, "token_logprobs requires CUDA tensors"
    dev, shape = logits.device, logits.shape
    if logits.dim() < 1 or shape[-1] < 1:
        raise ValueError("token_logprobs: logits must have at least one entry a row")
    V, lead = shape[-1], shape[:-1]
    if V >= 2 ** 31:
        raise ValueError("token_logprobs: %d logits a row" % V)
    top_k = int(top_k)
    if top_k < 0 or top_k > V:
        raise ValueError("token_logprobs: top_k %d outside [0, %d]" % (top_k, V))
    if top_k > MAX_TOP_K:
        raise NotImplementedError("token_logprobs: top_k %d, at most %d are built" % (top_k, MAX_TOP_K))
    code = _lib.dtype_code(logits.dtype)
    if tokens is not None:
        assert tokens.dtype == torch.int64 and tokens.get_device() == dev.index and tokens.shape == lead, \
            "token_logprobs: tokens must be int64 on the logits' device, one a row"
        tokens = tokens.contiguous()
    x = logits.detach() if logits.requires_grad else logits
    if V > 1 and x.stride(-1) != 1:
        x = x.contiguous()
    if x.dim() != 2:
        x = x.reshape(-1, V)   # a view where the leading strides allow it
    R = x.shape[0]
    # (a tensor made after one of its type and device costs a third less than one from scratch)
    lp = ent = ids = top = some = None
    if tokens is not None:
        lp = some = torch.empty(lead, dtype=torch.float32, device=dev)
    if entropy:
        ent = some = torch.empty(lead, dtype=torch.float32, device=dev) if some is None else torch.empty_like(some)
    if top_k:
        shape = (*lead, top_k)
        top = torch.empty(shape, dtype=torch.float32, device=dev) if some is None else some.new_empty(shape)
        ids = torch.empty(shape, dtype=torch.int64, device=dev) if tokens is None else tokens.new_empty(shape)
    if R and not (lp is None and ent is None and ids is None):
        with _lib.on_device(dev):
            rc = _lib.load().dk_token_logprobs(
                x.data_ptr(), x.stride(0), R, V, code, None if lp is None else tokens.data_ptr(),
                None if lp is None else lp.data_ptr(), None if ent is None else ent.data_ptr(), top_k,
                None if ids is None else ids.data_ptr(), None if ids is None else top.data_ptr(), _lib.stream_ptr(dev))
        _lib.check(rc, "token_logprobs")
        _lib.count_launch()
    return TokenLogprobs(lp, ent, ids, top)
