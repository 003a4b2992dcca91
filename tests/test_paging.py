"""The page plan of a step on the GPU: block-table growth, slot map and row tiles against the plain form."""
import numpy as np
import pytest


def _i32(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype=np.int32))).to(dev)


def _case(rng, B, kv_hi, new_hi, page, width_extra=1, table_rows=None):
    kv = rng.integers(0, kv_hi + 1, size=B)
    new = rng.integers(0, new_hi + 1, size=B)
    width = int(-(-(kv + new).max() // page)) + width_extra if B else 1
    table = rng.integers(0, 1000, size=(table_rows or B, max(width, 1)))
    need = int((-(-(kv + new) // page) - -(-kv // page)).sum())
    free = 1000 + rng.permutation(need + 5)
    return kv, new, table, free, need


def _check(dev, kv, new, table, free, page, rpt, spare_rows=0, cursor=2):
    import torch

    from detkernels_b200.kernels.paging import paged_plan, paged_plan_reference
    B = len(kv)
    want = paged_plan_reference(table.tolist(), kv.tolist(), new.tolist(), page,
                                free_blocks=None if free is None else free.tolist(), cursor=cursor, rows_per_tile=rpt)
    n, nt = len(want.row_seq), len(want.row_tiles)
    t = _i32(table, dev)
    got = paged_plan(t, _i32(kv, dev), _i32(new, dev), page, free_blocks=None if free is None else _i32(free, dev),
                     cursor=None if free is None else _i32([cursor], dev), n_rows=n + spare_rows, rows_per_tile=rpt,
                     n_tiles=nt + spare_rows if rpt else None)
    assert got.block_table is t and t.tolist() == [list(map(int, r)) for r in want.block_table]
    assert got.cu_rows.tolist() == want.cu_rows
    assert got.row_seq[:n].tolist() == want.row_seq and got.row_pos[:n].tolist() == want.row_pos
    assert got.slots.dtype == torch.int64 and got.slots[:n].tolist() == want.slots
    assert got.q_lens[:n].tolist() == want.q_lens
    if free is not None:
        assert got.cursor.tolist() == [want.cursor]
    if rpt:
        assert [tuple(x) for x in got.row_tiles[:nt].tolist()] == want.row_tiles
    return got


def test_reference_on_a_small_step():
    from detkernels_b200.kernels.paging import paged_plan_reference
    p = paged_plan_reference([[7, 0, 0], [9, 0, 0]], [3, 4], [2, 1], 4, free_blocks=[5, 6, 8], cursor=1, rows_per_tile=2)
    assert p.block_table == [[7, 6, 0], [9, 8, 0]] and p.cursor == 3
    assert p.cu_rows == [0, 2, 3] and p.row_seq == [0, 0, 1] and p.row_pos == [3, 4, 4]
    assert p.slots == [31, 24, 32] and p.q_lens == [4, 5, 5] and p.row_tiles == [(0, 2, 0), (2, 1, 1)]


def test_entry_point_refuses_on_the_host():
    """The C entry rejects bad arguments before it touches a device pointer."""
    from detkernels_b200 import _lib
    lib = _lib.load()

    def call(n_seqs=2, page=64, width=4, stride=4, free=None, cursor=None, row_seq=None, rpt=0, tiles=None, ws=0,
             n_rows=4):
        return lib.dk_paged_plan(16, stride, width, 16, 16, n_seqs, page, free, 8, cursor, cursor, 16, row_seq, row_seq,
                                 row_seq, row_seq, n_rows, tiles, rpt, 4, 16, ws, None)
    assert call(n_seqs=0) == _lib.DK_OK
    assert call(page=0) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(n_rows=-1) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(stride=3) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(width=1 << 20, stride=1 << 20, page=1 << 14) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(free=16) == _lib.DK_ERR_INVALID_ARGUMENT and "cursor" in _lib.last_error()
    assert call(tiles=16) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(ws=0) == _lib.DK_ERR_WORKSPACE
    assert lib.dk_paged_plan_workspace_size(3) >= 4 * (2 + 2 * 4)


def test_wrapper_refuses_cpu_tensors():
    import torch

    from detkernels_b200.kernels.paging import paged_plan
    with pytest.raises(AssertionError):
        paged_plan(torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                   torch.ones(2, dtype=torch.int32), 64)


@pytest.mark.gpu
@pytest.mark.parametrize("B,kv_hi,new_hi,page,rpt", [
    (1, 0, 1, 64, 1), (1, 5000, 3000, 64, 16), (7, 1500, 1, 64, 0), (33, 40, 40, 16, 3), (256, 0, 512, 64, 16),
    (1023, 300, 30, 1, 2), (1024, 300, 30, 7, 5), (1025, 3, 2, 128, 16), (2500, 200, 60, 64, 8), (3, 0, 0, 64, 4),
    (9000, 100, 9, 32, 4)])
def test_plan_equals_the_plain_form(dev, B, kv_hi, new_hi, page, rpt):
    rng = np.random.default_rng(B * 7 + page)
    kv, new, table, free, _ = _case(rng, B, kv_hi, new_hi, page)
    _check(dev, kv, new, table, free, page, rpt)
    _check(dev, kv, new, table, None, page, rpt)      # the table already covers everything


@pytest.mark.gpu
def test_empty_sequences_at_the_ends_and_between(dev):
    kv = np.array([0, 0, 64, 0, 63, 128, 0])
    new = np.array([0, 0, 1, 0, 2, 0, 0])
    table = np.arange(7 * 4).reshape(7, 4)
    _check(dev, kv, new, table, np.array([90, 91, 92, 93, 94]), 64, 4)


@pytest.mark.gpu
def test_entries_and_rows_behind_the_last_stay_as_they_were(dev):
    import torch

    from detkernels_b200.kernels.paging import PagedPlan, paged_plan
    table = torch.full((5, 4), -7, dtype=torch.int32, device=dev)
    old = PagedPlan(None, torch.tensor([0], dtype=torch.int32, device=dev),
                    torch.full((4,), -5, dtype=torch.int32, device=dev),
                    *(torch.full((9,), -5, dtype=d, device=dev)
                      for d in (torch.int32, torch.int32, torch.int64, torch.int32)),
                    torch.full((6, 3), -5, dtype=torch.int32, device=dev))
    free = _i32([10, 11, 12, 13], dev)
    got = paged_plan(table, _i32([0, 64, 3], dev), _i32([2, 1, 0], dev), 64, free_blocks=free, cursor=old.cursor,
                     n_rows=9, rows_per_tile=2, n_tiles=6, out=old)
    assert got.cursor.data_ptr() == old.cursor.data_ptr() and got.cursor.tolist() == [2]   # advanced in place
    assert table.tolist() == [[10, -7, -7, -7], [-7, 11, -7, -7]] + [[-7] * 4] * 3
    assert got.row_seq.tolist() == [0, 0, 1] + [-5] * 6 and got.slots.tolist()[3:] == [-5] * 6
    assert got.row_tiles.tolist()[:2] == [[0, 2, 0], [2, 1, 1]] and got.row_tiles.tolist()[2:] == [[-5] * 3] * 4


@pytest.mark.gpu
def test_large_block_ids_give_64_bit_slots(dev):
    from detkernels_b200.kernels.paging import paged_plan
    got = paged_plan(_i32([[2 ** 30]], dev), _i32([255], dev), _i32([1], dev), 256, n_rows=1)
    assert got.slots.tolist() == [2 ** 38 + 255]


@pytest.mark.gpu
@pytest.mark.parametrize("kv,new,n_rows,free,detail", [
    ([-1, 3], [1, 1], 2, 8, 0x600), ([0, 3], [1, -1], 2, 8, 0x600), ([0, 250], [1, 10], 11, 8, 0x600),
    ([0, 0], [64, 65], 129, 2, 0x601), ([0, 0], [3, 3], 5, 8, 0x602),
    ([2 ** 31 - 1, 0], [2 ** 31 - 1, 1], 2, 8, 0x600)])
def test_bad_lengths_are_reported_and_nothing_is_written(dev, kv, new, n_rows, free, detail):
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.paging import PagedPlan, paged_plan
    table = torch.full((2, 4), -7, dtype=torch.int32, device=dev)
    outs = [torch.full((n_rows,), -5, dtype=d, device=dev) for d in (torch.int32, torch.int32, torch.int64, torch.int32)]
    out = PagedPlan(None, None, None, *outs, None)
    got = paged_plan(table, _i32(kv, dev), _i32(new, dev), 64, free_blocks=_i32(np.arange(free), dev),
                     cursor=_i32([0], dev), n_rows=n_rows, out=out)
    assert _lib.device_status(dev.index) == (_lib.DK_ERR_DEVICE_CHECK, detail)
    assert (table == -7).all() and got.cursor.tolist() == [0]
    assert all((t == -5).all() for t in outs)


@pytest.mark.gpu
def test_plan_replayed_in_a_graph_advances_the_pool(dev):
    """A captured decode step: each replay plans one token a sequence, in place."""
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.paging import PagedPlan, paged_plan, paged_plan_reference
    page, B, steps = 4, 5, 11
    kv0 = np.array([0, 3, 4, 7, 1])
    table0 = np.zeros((B, 6), np.int64)
    table0[:, :2] = np.arange(10).reshape(5, 2)
    free = np.arange(100, 130)
    table, kv, one, fr = _i32(table0, dev), _i32(kv0, dev), _i32(np.ones(B), dev), _i32(free, dev)
    cursor = _i32([0], dev)
    out = PagedPlan(None, cursor, None, None, None, None, None, None)
    paged_plan(table.clone(), kv, one, page, free_blocks=fr, cursor=cursor.clone(), n_rows=B)    # load the library
    g = torch.cuda.CUDAGraph()
    with _lib.graph_capture(g):
        plan = paged_plan(table, kv, one, page, free_blocks=fr, cursor=cursor, n_rows=B, out=out)
        kv.add_(one)
    want_t, want_c, want_kv = table0.tolist(), 0, kv0.tolist()
    for _ in range(steps):
        g.replay()
        w = paged_plan_reference(want_t, want_kv, [1] * B, page, free_blocks=free.tolist(), cursor=want_c)
        want_t, want_c, want_kv = w.block_table, w.cursor, w.q_lens
        assert plan.slots.tolist() == w.slots and table.tolist() == want_t and cursor.tolist() == [want_c]


@pytest.mark.gpu
def test_equals_the_host_allocator(dev):
    """From an empty cache, with the host allocator's block order as the free list: its table."""
    import torch

    from detkernels_b200.kernels.paging import paged_plan
    from detkernels_b200.kernels.tiny_model import BlockAllocator
    rng = np.random.default_rng(4)
    tokens = rng.integers(1, 600, size=40)
    al = BlockAllocator(500, 50, 10, seed=3)
    want = al.assign(tokens.tolist(), 64)
    table = torch.zeros(50, 10, dtype=torch.int32, device=dev)
    paged_plan(table, _i32(np.zeros(40), dev), _i32(tokens, dev), 64, free_blocks=_i32(al.order, dev),
               cursor=_i32([0], dev))
    assert np.array_equal(table.cpu().numpy(), want)


@pytest.mark.gpu
def test_rows_of_a_table_that_overlap_are_refused(dev):
    """An expanded table has one row in memory: no call may take it for B."""
    import torch

    from detkernels_b200.kernels.attention import attention_shared_prefix
    from detkernels_b200.kernels.paging import paged_plan
    one = torch.zeros(1, 4, dtype=torch.int32, device=dev)
    ln = torch.ones(3, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        paged_plan(one.expand(3, 4), ln, ln, 64, n_rows=3)
    q = torch.zeros(3, 2, 64, device=dev, dtype=torch.bfloat16)
    pool = torch.zeros(2, 2, 64, 64, device=dev, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        attention_shared_prefix(q, pool[0], pool[0], pool, pool, ln, block_table=one.expand(3, 4))
    # one row of a wider table, and a single sequence, are fine with any stride
    wide = torch.zeros(3, 8, dtype=torch.int32, device=dev)
    plan = paged_plan(wide[:, :4], ln, ln, 64, n_rows=3)
    assert plan.slots.tolist() == [1, 1, 1]
    assert paged_plan(one, ln[:1], ln[:1], 64, n_rows=1).slots.tolist() == [1]
