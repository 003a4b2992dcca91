"""Page plan of a serving step, built on the GPU from the requests' lengths; pages forked, compacted and freed.

The device counterpart of ``tiny_model.BlockAllocator`` and of the host side of
``DecodeEngine.plan``: block-table growth from a free list, the slot of every
new token in the paged cache, its sequence, position and attention length, and
the attention kernels' row tiles, in one launch (small steps) or two, without a host round trip.
``paged_fork`` and ``paged_compact`` keep the same table and free list for sequences that are copied,
thinned out or ended.
No counterpart in the reference (its cache is one tensor grown by
``torch.cat``, tiny_model.py:119-125).
"""
from __future__ import annotations

from array import array
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


class PagedCompact(NamedTuple):
    lens: object                 # int32 [B]: tokens each sequence holds now
    cursor: Optional[object]     # int32 [1]: free blocks handed out, without those that came back


def paged_fork_reference(block_table, kv_lens, src, dst, page_size, *, free_blocks, cursor=0, shares=None):
    """Plain Python form on host sequences (block_table a list of lists).  Returns (table, kv_lens, cursor, shares,
    copies), copied lists, copies the (source block, new block, tokens) to copy in every pool."""
    table, kv = [list(r) for r in block_table], list(kv_lens)
    shares = None if shares is None else list(shares)
    copies = []
    for s, d in zip(src, dst):
        for j in range(-(-kv[s] // page_size)):
            if shares is not None and (j + 1) * page_size <= kv[s]:
                table[d][j] = table[s][j]
                shares[table[s][j]] += 1
            else:
                table[d][j] = free_blocks[cursor]
                cursor += 1
                copies.append((table[s][j], table[d][j], min(page_size, kv[s] - j * page_size)))
        kv[d] = kv[s]
    return table, kv, cursor, shares, copies


def paged_compact_reference(block_table, kv_lens, new_lens, n_keep, page_size, *, keep=None, free_blocks=None, cursor=0,
                            shares=None):
    """Plain Python form on host sequences.  Returns (lens, cursor, free_blocks, shares, moves), copied lists, moves the
    (block, token, new block, new token) of the tokens to move in every pool, to be done in order."""
    free = None if free_blocks is None else list(free_blocks)
    shares = None if shares is None else list(shares)
    lens, moves, given = [], [], []
    for b, (kv, new, nk) in enumerate(zip(kv_lens, new_lens, n_keep)):
        for j in range(nk):
            s, d = kv + (j if keep is None else keep[b][j]), kv + j
            if s != d:
                moves.append((block_table[b][s // page_size], s % page_size, block_table[b][d // page_size], d % page_size))
        given += [block_table[b][j] for j in range(-(-(kv + nk) // page_size), -(-(kv + new) // page_size))]
        lens.append(kv + nk)
    if free is not None:
        if shares is not None:
            for x in given:
                shares[x] -= 1
            # a page without a holder goes back where the last one gave it up
            given = [x for i, x in enumerate(given) if shares[x] < 0 and x not in given[i + 1:]]
            for x in given:
                shares[x] = 0
        cursor -= len(given)
        free[cursor:cursor + len(given)] = given
    return lens, cursor, free, shares, moves


def _check_pools(pools, dev, page_size, what):
    """(their addresses, number, element strides by block, head and token, blocks, heads, head_dim, element size)."""
    pools = list(pools)
    if not pools:
        return array("Q"), 0, (0, 0, 0), 0, 0, 0, 1
    first = pools[0]
    shape, stride, dtype = first.shape, first.stride(), first.dtype
    index = dev.index
    for t in pools:
        assert t.get_device() == index, "%s requires CUDA tensors on one device" % what
        if t.stride() != stride or t.shape != shape or t.dtype is not dtype:
            raise ValueError("%s: the pools must share shape, strides and dtype" % what)
    at = array("Q", [t.data_ptr() for t in pools])
    assert len(shape) == 4 and shape[2] == page_size, "%s: pools must be [n_blocks, heads, page_size, head_dim]" % what
    if shape[3] > 1 and stride[3] != 1:
        raise ValueError("%s: unit stride along head_dim required" % what)
    if len(set(at)) != len(at):
        raise ValueError("%s: a pool is named twice" % what)
    return at, len(pools), stride[:3], shape[0], shape[1], shape[3], first.element_size()


def _check_books(block_table, kv_lens, page_size, free_blocks, cursor, shares, n_blocks, what):
    """The table, the free list and the holders: (table stride, blocks that ids may name)."""
    import torch
    dev, i32 = block_table.device, torch.int32
    assert block_table.is_cuda and kv_lens.get_device() == dev.index, "%s requires CUDA tensors on one device" % what
    assert block_table.dtype == i32 and block_table.dim() == 2
    assert block_table.shape[1] <= 1 or block_table.stride(1) == 1, "block_table: unit stride along a row"
    assert kv_lens.dtype == i32 and kv_lens.dim() == 1, "%s: lengths must be int32 vectors" % what
    if not 1 <= page_size < 2 ** 31:
        raise ValueError("%s: page_size must be positive and below 2^31" % what)
    if max(*block_table.shape, kv_lens.shape[0]) >= 2 ** 31:
        raise ValueError("%s: a table of 2^31 rows or columns" % what)
    if (free_blocks is None) != (cursor is None):
        raise ValueError("%s: free_blocks and cursor go together" % what)
    if free_blocks is not None:
        assert free_blocks.dtype == i32 and free_blocks.get_device() == dev.index and free_blocks.is_contiguous()
        assert free_blocks.dim() == 1 and cursor.dtype == i32 and cursor.get_device() == dev.index and cursor.numel() == 1
    if shares is not None:
        assert shares.dtype == i32 and shares.get_device() == dev.index and shares.is_contiguous() and shares.dim() == 1
        if shares.numel() < max(n_blocks, 1):   # (no entries bound no id: they would be looked up all the same)
            raise ValueError("%s: shares must have an entry a block" % what)
        n_blocks = n_blocks or shares.numel()
    return block_table.stride(0) if block_table.shape[0] > 1 else block_table.shape[1], n_blocks or 2 ** 31 - 1


def paged_fork(block_table, kv_lens, src, dst, page_size: int, *, free_blocks, cursor, pools=(), shares=None):
    """Sequence dst[i] becomes a copy of sequence src[i]: several samples of one prompt, or the beams of a search.

    block_table (int32 CUDA [n, blocks_per_seq]) and kv_lens (int32 CUDA [n], the tokens each row holds) are updated in
    place; src, dst: int32 CUDA [F].  A source may be named several times, a destination once and not as a source; the
    blocks that a destination held are not given back (``paged_compact`` does that).
    shares (int32 CUDA [n_blocks]): how many further sequences hold a block beyond the first.  With it whole pages are
    shared (shares[block] += 1), and only the last, open page gets a block of its own; without it every page does.  New
    blocks are the next of free_blocks from cursor on (as for ``paged_plan``), in the order of the forks; returns the
    new cursor (int32 CUDA [1]).
    pools: the K and V pools of all layers ([n_blocks, heads, page_size, head_dim], any dtype, same strides, none over
    another), in which the tokens of the new blocks are copied; what lies behind a sequence's last token is left as it was.

    Rows outside the table or misnamed, a length outside its row, a block id outside the pools or too few free blocks set
    the device status (``_lib.raise_on_device_error``), and nothing changes."""
    import torch

    what = "paged_fork"
    dev = block_table.device
    at, n_pools, st, n_blocks, heads, dim, size = _check_pools(pools, dev, page_size, what)
    if free_blocks is None or cursor is None:
        raise ValueError("paged_fork: free_blocks and cursor are needed")
    stride, n_blocks = _check_books(block_table, kv_lens, page_size, free_blocks, cursor, shares, n_blocks, what)
    assert kv_lens.shape == (block_table.shape[0],) and kv_lens.is_contiguous(), "paged_fork: one length a table row"
    assert src.dtype == torch.int32 and dst.dtype == torch.int32 and src.shape == dst.shape and src.dim() == 1
    if src.shape[0] >= 2 ** 31:
        raise ValueError("paged_fork: 2^31 forks or more")
    assert src.get_device() == dev.index and dst.get_device() == dev.index, "paged_fork requires CUDA tensors on one device"
    with _lib.on_device(dev):
        src, dst = src.contiguous(), dst.contiguous()
        if src.numel() == 0 or block_table.shape[0] == 0:
            if src.numel():
                raise ValueError("paged_fork: the table has no rows")
            return cursor.clone()
        out = torch.empty_like(cursor)
        lib = _lib.load()
        ws = src.new_empty(-(-lib.dk_paged_fork_workspace_size(block_table.shape[0]) // 4))
        rc = lib.dk_paged_fork(
            block_table.data_ptr(), stride, block_table.shape[0], block_table.shape[1], kv_lens.data_ptr(), src.data_ptr(),
            dst.data_ptr(), src.numel(), int(page_size), free_blocks.data_ptr() or ws.data_ptr(), free_blocks.numel(),
            cursor.data_ptr(), out.data_ptr(), None if shares is None else shares.data_ptr(), n_blocks, at.buffer_info()[0],
            n_pools, *st, heads, dim, size, ws.data_ptr(), 4 * ws.numel(), _lib.stream_ptr(dev))
    _lib.check(rc, what)
    _lib.count_launch(2 if n_pools else 1)
    return out


def paged_compact(block_table, kv_lens, new_lens, n_keep, page_size: int, *, keep=None, pools=(), free_blocks=None,
                  cursor=None, shares=None) -> PagedCompact:
    """Keep some of each sequence's last tokens, and give the pages back that then hold nothing.

    Sequence b (row b of block_table, int32 CUDA [>= B, blocks_per_seq]) holds kv_lens[b] tokens and new_lens[b] behind
    them, of which n_keep[b] stay (all int32 CUDA [B]): those at kv_lens[b] + keep[b, j], ascending (keep: int32 CUDA
    [B, K], K at least the largest n_keep; what lies behind a row's n_keep is not read), or the first ones without
    ``keep``.  They are moved to kv_lens[b] + j in all ``pools`` (as in ``paged_fork``): the accepted path of a tree
    (``drafts.tree_accept``), or a cache thinned out.  kv_lens = 0 and n_keep = 0 free a sequence.
    free_blocks (updated in place) and cursor: the pages behind a sequence's tokens go back before the cursor, in the order
    of sequences and pages, and the new cursor, from which ``paged_plan`` and ``paged_fork`` take them again, is returned.
    With shares (as in ``paged_fork``) a page with further holders loses one instead, and one given up by all its holders
    goes back once; without, a page must be one sequence's alone.  Table entries stay as they are.  Tokens are not moved
    into a page that another sequence shares (free that one first, in a call before); ``paged_fork`` leaves each sequence its
    open page to itself.  A sequence that a call leaves ending inside a shared page must not take new tokens there: its fork
    may, which has a copy of that page.

    A negative length, more kept than held, a sequence beyond its table row, a ``keep`` that does not ascend inside the
    new tokens, a block id outside the pools, more pages than were handed out, a page given up by more sequences than hold
    it or a token to move into a shared page set the device status; then lens are kv_lens, the cursor stays, and nothing
    changes."""
    import torch

    what = "paged_compact"
    dev = block_table.device
    at, n_pools, st, n_blocks, heads, dim, size = _check_pools(pools, dev, page_size, what)
    stride, n_blocks = _check_books(block_table, kv_lens, page_size, free_blocks, cursor, shares, n_blocks, what)
    if shares is not None and free_blocks is None:
        raise ValueError("paged_compact: shares need a free list")
    B = kv_lens.numel()
    assert block_table.shape[0] >= B and new_lens.shape == (B,) and n_keep.shape == (B,), "paged_compact: [B] lengths"
    for t in (new_lens, n_keep):
        assert t.dtype == torch.int32 and t.get_device() == dev.index, "paged_compact: lengths must be int32 on one device"
    if keep is not None:
        assert keep.dtype == torch.int32 and keep.get_device() == dev.index and keep.dim() == 2 and keep.shape[0] == B
        if keep.shape[1] >= 2 ** 31:
            raise ValueError("paged_compact: keep of 2^31 columns or more")
        if keep.shape[1] > 1 and keep.stride(1) != 1:
            keep = keep.contiguous()
    with _lib.on_device(dev):
        kv_lens, new_lens, n_keep = kv_lens.contiguous(), new_lens.contiguous(), n_keep.contiguous()
        lens = torch.empty_like(kv_lens)
        out = None if cursor is None else torch.empty_like(cursor)
        if B == 0:
            return PagedCompact(lens, None if cursor is None else cursor.clone())
        lib = _lib.load()
        ws = kv_lens.new_empty(-(-lib.dk_paged_compact_workspace_size() // 4))

        def ptr(t):
            # without entries nothing is followed, but it was given
            return None if t is None else (t.data_ptr() or ws.data_ptr())

        rc = lib.dk_paged_compact(
            block_table.data_ptr(), stride, block_table.shape[1], kv_lens.data_ptr(), new_lens.data_ptr(),
            n_keep.data_ptr(), ptr(keep), 0 if keep is None else keep.stride(0), 0 if keep is None else keep.shape[1], B,
            int(page_size), lens.data_ptr(), ptr(free_blocks), 0 if free_blocks is None else free_blocks.numel(),
            ptr(cursor), ptr(out), ptr(shares), n_blocks, at.buffer_info()[0], n_pools, *st, heads, dim, size,
            ws.data_ptr(), 4 * ws.numel(), _lib.stream_ptr(dev))
    _lib.check(rc, what)
    _lib.count_launch(2 if n_pools and keep is not None else 1)
    return PagedCompact(lens, out)
