"""Trees of drafted tokens: their masks, and the path that the model accepts.

A verification step gives each request a tree of drafted tokens, node 0 being its last sampled token, runs the model
over all nodes at once (``attention.attention_tree``) and keeps the path along which the model agrees.  ``tree_accept``
finds it on the device; ``paging.paged_compact`` then keeps its keys and values.  No counterpart in the reference (its
decoder takes one token a step, tiny_model.py:142-157).
"""
from __future__ import annotations

from typing import NamedTuple

from detkernels_b200 import _lib


class TreeAccept(NamedTuple):
    keep: object          # int32 [B, max_keep]: the path's nodes, ascending, -1 behind them
    n_keep: object        # int32 [B]
    next_tokens: object   # int64 [B]: the pick after the path's last node, -1 without nodes


def tree_mask(parents, cu_rows, words: int = 1, max_rows=None):
    """The mask of ``attention_tree``: bit j of row i's words (int64 [R, words], 64 nodes a word) says that node j of the
    row's sequence is the row's node or one of its ancestors.

    parents: int32 [R], the parent's index among the sequence's nodes (smaller than the node's own), -1 for none;
    cu_rows: int32 [B + 1], ascending.  Elementary torch operations, on any device, without a host round trip, three for each
    binary digit of max_rows, a bound on a sequence's nodes (all rows if not given).  Nodes from 64 * words on have no bit,
    and rows behind the last sequence no bits at all."""
    import torch

    assert parents.dim() == 1 and cu_rows.dim() == 1 and words >= 1
    R, dev = parents.numel(), parents.device
    row = torch.arange(R, device=dev)
    cu = cu_rows.long()
    seq = torch.searchsorted(cu, row, right=True) - 1
    start = cu[seq.clamp(0, cu.numel() - 1)]
    at = row - start
    live = (seq >= 0) & (row < cu[-1])
    word = torch.arange(words, device=dev)
    own = torch.ones_like(at) << (at & 63)
    mask = torch.where(live[:, None] & (word[None, :] == (at >> 6)[:, None]), own[:, None], 0)
    parent = parents.long()
    up = torch.where(live & (parent >= 0) & (parent < at), start + parent, row)
    deep = R if max_rows is None else min(R, int(max_rows))
    for _ in range(max(deep - 1, 0).bit_length()):   # ancestors twice as far each time
        mask = mask | mask[up]
        up = up[up]
    return mask


def tree_accept_reference(parents, tokens, picked, cu_rows, *, max_keep):
    """Plain Python form on host sequences; the fields of TreeAccept as lists."""
    keep, n_keep, nxt = [], [], []
    for a, b in zip(cu_rows[:-1], cu_rows[1:]):
        path = [0] if b > a else []
        while path and len(path) < max_keep:
            cur = path[-1]
            kids = [i for i in range(cur + 1, b - a) if parents[a + i] == cur and tokens[a + i] == picked[a + cur]]
            if not kids:
                break
            path.append(kids[0])
        keep.append(path + [-1] * (max_keep - len(path)))
        n_keep.append(len(path))
        nxt.append(picked[a + path[-1]] if path else -1)
    return TreeAccept(keep, n_keep, nxt)


def tree_accept(parents, tokens, picked, cu_rows, *, max_keep: int) -> TreeAccept:
    """The accepted path of each sequence's tree.

    Sequence b's nodes are the rows cu_rows[b] to cu_rows[b + 1] (int32 CUDA [B + 1]).  parents (int32 CUDA [R]): the
    parent's index among the sequence's nodes, smaller than the node's own; -1 for node 0 and for nodes that nothing
    reaches (padding).  tokens (int64 CUDA [R]): the nodes' tokens; picked (int64 CUDA [R]): the model's token after each
    node, the largest logit or a sample.  From node 0 the path goes on to the first child whose token is the pick after
    the current node, for at most max_keep nodes.

    A sequence without nodes keeps none.  Offsets that do not ascend inside the rows set the device status, and that
    sequence keeps none; rows behind the last sequence are not read."""
    import torch

    dev, i32, i64 = parents.device, torch.int32, torch.int64
    index = dev.index
    assert parents.is_cuda and tokens.get_device() == index and picked.get_device() == index \
        and cu_rows.get_device() == index, "tree_accept requires CUDA tensors on one device"
    assert parents.dtype == i32 and cu_rows.dtype == i32, "parents and cu_rows must be int32"
    assert tokens.dtype == i64 and picked.dtype == i64, "tokens and picked must be int64"
    R, B = parents.numel(), cu_rows.numel() - 1
    assert parents.shape == tokens.shape == picked.shape == (R,) and cu_rows.dim() == 1 and B >= 0, \
        "tree_accept: one parent, token and pick a row, and B + 1 offsets"
    if not 1 <= max_keep < 2 ** 31 or max(R, B) >= 2 ** 31:
        raise ValueError("tree_accept: max_keep must be positive, and sizes below 2^31")
    with _lib.on_device(dev):
        parents, tokens, picked, cu_rows = parents.contiguous(), tokens.contiguous(), picked.contiguous(), cu_rows.contiguous()
        r = TreeAccept(parents.new_empty(B, max_keep), parents.new_empty(B), tokens.new_empty(B))
        if B == 0:
            return r
        rc = _lib.load().dk_tree_accept(parents.data_ptr(), tokens.data_ptr(), picked.data_ptr(), cu_rows.data_ptr(), B, R,
                                        int(max_keep), r.keep.data_ptr(), r.n_keep.data_ptr(), r.next_tokens.data_ptr(),
                                        _lib.stream_ptr(dev))
    _lib.check(rc, "tree_accept")
    _lib.count_launch()
    return r
