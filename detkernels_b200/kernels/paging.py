"""Page plan of a serving step, built on the GPU from the requests' lengths.

The device counterpart of ``tiny_model.BlockAllocator`` and of the host side of
``DecodeEngine.plan``: block-table growth from a free list, the slot of every
new token in the paged cache, its sequence, position and attention length, and
the attention kernels' row tiles, in one launch (small steps) or two, without a host round trip.
No counterpart in the reference (its cache is one tensor grown by
``torch.cat``, tiny_model.py:119-125).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

from detkernels_b200 import _lib


class PagedPlan(NamedTuple):
    """One step's plan; the fields that were not asked for are None."""
    block_table: object            # int32 [B, blocks_per_seq] (the caller's tensor, grown in place)
    cursor: Optional[object]       # int32 [1]: free blocks handed out, this step's included
    cu_rows: object                # int32 [B + 1]: first row of each sequence, and the total
    row_seq: Optional[object]      # int32 [n_rows]
    row_pos: Optional[object]      # int32 [n_rows]
    slots: Optional[object]        # int64 [n_rows]: block * page_size + token in the block
    q_lens: Optional[object]       # int32 [n_rows]: row_pos + 1
    row_tiles: Optional[object]    # int32 [n_tiles, 3]: (first row, rows, sequence)


_NOTHING = PagedPlan(*[None] * len(PagedPlan._fields))


def paged_plan_reference(block_table, kv_lens, new_lens, page_size, *, free_blocks=None, cursor=0, rows_per_tile=0):
    """Plain Python plan of one step on host sequences; block_table is a list of lists.  Returns the
    fields of PagedPlan as Python lists (block_table a grown copy)."""
    table = [list(row) for row in block_table]
    cu, seq, pos, slots, tiles = [0], [], [], [], []
    for b, (kv, new) in enumerate(zip(kv_lens, new_lens)):
        if free_blocks is not None:
            for pg in range(-(-kv // page_size), -(-(kv + new) // page_size)):
                table[b][pg] = free_blocks[cursor]
                cursor += 1
        for t in range(kv, kv + new):
            seq.append(b)
            pos.append(t)
            slots.append(table[b][t // page_size] * page_size + t % page_size)
        if rows_per_tile:
            tiles += [(cu[-1] + i, min(rows_per_tile, new - i), b) for i in range(0, new, rows_per_tile)]
        cu.append(cu[-1] + new)
    return PagedPlan(table, cursor, cu, seq, pos, slots, [t + 1 for t in pos], tiles)


def _apart(lens, plan):
    """lens, or a copy if a row or tile output lies over it (the kernels read lengths while they write rows)."""
    begin = lens.data_ptr()
    end = begin + 4 * lens.numel()
    for t in plan[2:]:
        if t is not None and t.data_ptr() < end and begin < t.data_ptr() + t.numel() * t.element_size():
            return lens.clone()
    return lens


def paged_plan(block_table, kv_lens, new_lens, page_size: int, *, free_blocks=None, cursor=None,
               n_rows: Optional[int] = None, rows_per_tile: int = 0, n_tiles: Optional[int] = None,
               out: Optional[PagedPlan] = None, pad: bool = False) -> PagedPlan:
    """Plan one step in which sequence b, holding kv_lens[b] tokens, gets new_lens[b] more.

    block_table: int32 CUDA [>= B, blocks_per_seq]; kv_lens, new_lens: int32 CUDA [B].
    free_blocks (int32 CUDA [F]) and cursor (int32 CUDA [1], how many of them are already handed out):
    the table entries of the pages that the new tokens open become the next free blocks, in sequence
    order; without them the table must already cover every sequence.  Other entries, and rows of the
    table past B, stay as they are.
    n_rows: how many new tokens there are (the sum of new_lens, or a bound on it): asks for row_seq,
    row_pos, slots and q_lens.  rows_per_tile and n_tiles (the sum of ceil(new_lens / rows_per_tile), or
    a bound) ask for row_tiles.
    out: a PagedPlan of an earlier call whose tensors take the results (its cursor may be ``cursor``, its
    q_lens kv_lens: a decode step's lengths are the next one's).
    pad: what lies past the step's own totals in the tensors of ``out`` becomes neutral: row_seq, row_pos
    and q_lens 0, slots -1 (``qk_norm_rope`` stores nothing there), tiles of 0 rows (attention skips them).
    A captured step that serves smaller ones needs it: without it those entries, an earlier step's slots and
    tiles, stay as they are.  New tensors are always padded.  (The matmul's fused store of K and V goes by
    row_seq and row_pos and has no neutral rows: give it exact sizes.)

    A negative length, a sequence longer than its table row, an exhausted free list or more rows or tiles
    than announced sets the device status (``_lib.raise_on_device_error``) and leaves the table and all
    outputs but cu_rows as they were; where entries are padded all of them become neutral, so that the rest
    of the step stores nothing."""
    import torch

    dev, i32 = block_table.device, torch.int32
    B, index = kv_lens.numel(), dev.index
    assert block_table.is_cuda and kv_lens.get_device() == index and new_lens.get_device() == index, \
        "paged_plan requires CUDA tensors on one device"
    shape, stride = block_table.shape, block_table.stride()
    assert block_table.dtype == i32 and len(shape) == 2 and shape[0] >= B
    assert shape[1] <= 1 or stride[1] == 1, "block_table: unit stride along a row"
    assert kv_lens.dtype == i32 and new_lens.dtype == i32 and kv_lens.dim() == 1 and new_lens.shape == (B,), \
        "lengths must be int32 [B]"
    if not 1 <= page_size < 2 ** 31:
        raise ValueError("paged_plan: page_size must be positive and below 2^31")
    if (free_blocks is None) != (cursor is None):
        raise ValueError("paged_plan: free_blocks and cursor go together")
    if free_blocks is not None:
        assert free_blocks.dtype == i32 and free_blocks.get_device() == index and free_blocks.is_contiguous()
        assert cursor.dtype == i32 and cursor.get_device() == index and cursor.numel() == 1
    if rows_per_tile < 0 or (rows_per_tile > 0 and n_tiles is None) or (rows_per_tile == 0 and n_tiles):
        raise ValueError("paged_plan: rows_per_tile and n_tiles go together")
    rows_per_tile = min(rows_per_tile, 2 ** 31 - 1)   # no sequence has more rows
    if (n_rows is not None and n_rows < 0) or (n_tiles is not None and n_tiles < 0):
        raise ValueError("paged_plan: n_rows and n_tiles must not be negative")

    def take(t, *shape, dtype=i32, neutral=None):
        """The tensor of an earlier plan, or a new one."""
        if t is None:
            t = kv_lens.new_empty(*shape) if dtype == i32 else kv_lens.new_empty(shape, dtype=dtype)
            return t if neutral is None or padded else t.fill_(neutral)
        assert t.dtype == dtype and t.get_device() == index and t.shape == shape and t.is_contiguous(), \
            "paged_plan: a tensor of out does not fit"
        return t

    old = out if out is not None else _NOTHING
    # the kernel pads all outputs or none; new tensors beside given ones that stay as they are get it beforehand
    padded = pad or out is None or (old.row_seq is None and old.row_pos is None and old.slots is None
                                    and old.q_lens is None and old.row_tiles is None)
    with _lib.on_device(dev):
        kv_lens, new_lens = kv_lens.contiguous(), new_lens.contiguous()
        cu = take(old.cu_rows, B + 1)
        cur = take(old.cursor, 1) if cursor is not None else None
        row_seq = row_pos = slots = q_lens = tiles = None
        if n_rows is not None:
            row_seq, row_pos = take(old.row_seq, n_rows, neutral=0), take(old.row_pos, n_rows, neutral=0)
            q_lens = take(old.q_lens, n_rows, neutral=0)
            slots = take(old.slots, n_rows, dtype=torch.int64, neutral=-1)
        if rows_per_tile > 0:
            tiles = take(old.row_tiles, n_tiles, 3, neutral=0)
        plan = PagedPlan(block_table, cur, cu, row_seq, row_pos, slots, q_lens, tiles)
        if out is not None:
            kv_lens, new_lens = _apart(kv_lens, plan), _apart(new_lens, plan)
        if B == 0:
            cu.zero_()
            if cur is not None and cur.data_ptr() != cursor.data_ptr():
                cur.copy_(cursor.view(1))
            if padded:
                for t, neutral in ((row_seq, 0), (row_pos, 0), (slots, -1), (q_lens, 0), (tiles, 0)):
                    if t is not None:
                        t.fill_(neutral)
            return plan
        lib = _lib.load()
        ws = kv_lens.new_empty(-(-lib.dk_paged_plan_workspace_size(B) // 4))
        ws_ptr = ws.data_ptr()

        def ptr(t):
            # an output of no entries is still asked for: its pointer is never followed
            return None if t is None else (t.data_ptr() or ws_ptr)

        rc = (lib.dk_paged_plan_padded if padded else lib.dk_paged_plan)(
            block_table.data_ptr(), stride[0] if shape[0] > 1 else shape[1], shape[1], kv_lens.data_ptr(), new_lens.data_ptr(), B,
            int(page_size), ptr(free_blocks), 0 if free_blocks is None else free_blocks.numel(), ptr(cursor), ptr(cur),
            cu.data_ptr(), ptr(row_seq), ptr(row_pos), ptr(slots), ptr(q_lens), n_rows or 0, ptr(tiles),
            int(rows_per_tile), n_tiles or 0, ws_ptr, 4 * ws.numel(), _lib.stream_ptr(dev))
    _lib.check(rc, "paged_plan")
    _lib.count_launch()   # at least: large steps take a second
    return plan
