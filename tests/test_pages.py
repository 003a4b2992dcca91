"""Forking, compacting and freeing the pages of a cache: against the plain forms, refusals that change nothing."""
import numpy as np
import pytest


def _i32(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype=np.int32))).to(dev)


def _pools(dev, n_blocks, Hkv, page, D, dt, n, layout="plain", seed=0):
    import torch
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = getattr(torch, dt)

    def make(*s):
        if dt == torch.uint8:
            return torch.randint(0, 256, s, device=dev, generator=g, dtype=dt)
        return torch.randn(*s, device=dev, generator=g).to(dt)
    if layout == "plain":
        return [make(n_blocks, Hkv, page, D) for _ in range(n)]
    if layout == "paired":      # K and V of a block side by side
        both = make(n_blocks, n, Hkv, page, D)
        return [both[:, i] for i in range(n)]
    if layout == "tokens":      # [block, page, head, D] in memory
        return [make(n_blocks, page, Hkv, D).transpose(1, 2) for _ in range(n)]
    if layout == "odd":         # heads off 16 bytes
        return [make(n_blocks, Hkv, page, D + 3)[..., 1:D + 1] for _ in range(n)]
    raise AssertionError(layout)


def _table(rng, lens, page, rows, extra):
    need = [-(-int(n) // page) for n in lens]
    n_blocks = sum(need) + extra
    order = rng.permutation(n_blocks)
    width = max(1, max(need, default=1)) + 1
    table = rng.integers(0, n_blocks, size=(rows, width))
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    return table, n_blocks, order[at:]


def test_references():
    from detkernels_b200.kernels.paging import paged_compact_reference, paged_fork_reference
    table, kv, cursor, shares, copies = paged_fork_reference([[3, 4], [0, 0], [0, 0]], [5, 0, 0], [0, 0], [2, 1], 4,
                                                             free_blocks=[9, 7, 8], cursor=1, shares=[0] * 10)
    assert table == [[3, 4], [3, 8], [3, 7]] and kv == [5, 5, 5] and cursor == 3 and shares[3] == 2
    assert copies == [(4, 7, 1), (4, 8, 1)]
    lens, cursor, free, shares, moves = paged_compact_reference([[3, 4], [3, 5]], [2, 0], [4, 6], [2, 0], 4,
                                                                keep=[[1, 3], [0, 0]], free_blocks=[1, 2, 0, 0], cursor=4,
                                                                shares=[0, 0, 0, 1, 0, 0])
    assert lens == [4, 0] and moves == [(3, 3, 3, 2), (4, 1, 3, 3)] and cursor == 2 and free == [1, 2, 4, 5]
    assert shares == [0] * 6
    # a page that all of its holders give up goes back once, where the last one did
    assert paged_compact_reference([[3], [5], [3]], [0] * 3, [1] * 3, [0] * 3, 4, free_blocks=[0] * 4, cursor=4,
                                   shares=[0, 0, 0, 1, 0, 0])[1:4] == (2, [0, 0, 5, 3], [0] * 6)


def test_entry_points_refuse_on_the_host():
    import ctypes

    from detkernels_b200 import _lib
    lib = _lib.load()
    one = (ctypes.c_void_p * 1)(16)
    none = (ctypes.c_void_p * 1)(None)

    def fork(rows=4, width=4, stride=4, n=2, page=8, free=16, cursor=16, shares=None, n_blocks=9, pools=one, size=2,
             dim=8, ws=1 << 16, heads=1, st=(64, 64, 8)):
        return lib.dk_paged_fork(16, stride, rows, width, 16, 16, 16, n, page, free, 5, cursor, cursor, shares, n_blocks,
                                 pools, 1, *st, heads, dim, size, 16, ws, None)
    bad = _lib.DK_ERR_INVALID_ARGUMENT
    assert fork(n=0) == _lib.DK_OK
    assert fork(n=-1) == bad and fork(page=0) == bad and fork(stride=3) == bad and fork(free=None) == bad
    assert fork(cursor=None) == bad and fork(n_blocks=0) == bad and fork(pools=None) == bad and fork(pools=none) == bad
    assert fork(width=1 << 20, stride=1 << 20, page=1 << 14) == bad
    assert fork(size=3) == _lib.DK_ERR_UNSUPPORTED and fork(dim=0) == bad
    # elements of one place, and more tokens than a launch takes
    assert fork(st=(0, 64, 8)) == bad and fork(st=(64, 0, 8), heads=2) == bad and fork(st=(64, 64, 0)) == bad
    assert fork(n=1 << 28, heads=1 << 12) == bad
    assert fork(ws=lib.dk_paged_fork_workspace_size(4) - 1) == _lib.DK_ERR_WORKSPACE

    def compact(n=2, width=4, stride=4, page=8, out=32, free=16, cursor=16, shares=None, n_blocks=9, keep_width=3, ws=1 << 16):
        return lib.dk_paged_compact(16, stride, width, 16, 16, 16, 16, 3, keep_width, n, page, out, free, 5, cursor, cursor,
                                    shares, n_blocks, one, 1, 64, 64, 8, 1, 8, 2, 16, ws, None)
    assert compact(n=0) == _lib.DK_OK
    assert compact(n=-1) == bad and compact(page=0) == bad and compact(stride=3) == bad and compact(out=16) == bad
    assert compact(keep_width=-1) == bad and compact(cursor=None) == bad and compact(free=None, shares=16) == bad
    assert compact(n=1 << 20, width=1 << 12, stride=1 << 12, shares=16) == bad
    assert compact(ws=lib.dk_paged_compact_workspace_size() - 1) == _lib.DK_ERR_WORKSPACE


def test_wrappers_refuse_cpu_tensors():
    import torch

    from detkernels_b200.kernels.paging import paged_compact, paged_fork
    t, i = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(AssertionError):
        paged_fork(t, i, i, i, 8, free_blocks=i, cursor=i[:1])
    with pytest.raises(AssertionError):
        paged_compact(t, i, i, i, 8)


POOLS = [("bfloat16", 2, 64, "plain"), ("float16", 3, 80, "paired"), ("float32", 1, 32, "tokens"), ("float16", 2, 20, "plain"),
         ("uint8", 2, 48, "plain"), ("bfloat16", 2, 64, "odd"), ("float64", 1, 1, "odd"), ("uint8", 1, 5, "plain")]


@pytest.mark.gpu
@pytest.mark.parametrize("dt,Hkv,D,layout", POOLS)
@pytest.mark.parametrize("page,shares", [(1, True), (3, False), (16, True), (64, True), (64, False)])
def test_fork(dev, dt, Hkv, D, layout, page, shares):
    import torch

    from detkernels_b200.kernels.paging import paged_fork, paged_fork_reference
    rng = np.random.default_rng(page)
    B = 6
    lens = np.array([0, 1, page, page + 1, 5 * page - 1, 130])
    src = rng.integers(0, B, size=9)
    dst = B + rng.permutation(12)[:9]
    table, n_blocks, free = _table(rng, lens, page, B + 12, 9 * (130 // page + 6))
    kv = np.concatenate([lens, rng.integers(0, 9, size=12)])
    sh = rng.integers(0, 4, size=n_blocks) if shares else None
    w_table, w_kv, w_cur, w_sh, copies = paged_fork_reference(table.tolist(), kv.tolist(), src.tolist(), dst.tolist(), page,
                                                              free_blocks=[0, 0] + free.tolist(), cursor=2,
                                                              shares=None if sh is None else sh.tolist())
    pools = _pools(dev, n_blocks, Hkv, page, D, dt, 3, layout)
    want = [p.clone() for p in pools]
    for s, d, n in copies:
        for p in want:
            p[d, :, :n] = p[s, :, :n]
    t, k, s = _i32(table, dev), _i32(kv, dev), None if sh is None else _i32(sh, dev)
    cur = _i32([2], dev)
    got = paged_fork(t, k, _i32(src, dev), _i32(dst, dev), page, free_blocks=_i32([0, 0] + free.tolist(), dev), cursor=cur,
                     pools=pools, shares=s)
    assert got.tolist() == [w_cur] and cur.tolist() == [2]
    assert t.tolist() == [list(map(int, r)) for r in w_table] and k.tolist() == list(map(int, w_kv))
    if shares:
        assert s.tolist() == list(map(int, w_sh))
    for a, b in zip(pools, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_fork_of_many(dev):
    """More forks than the plan has warps, and more pools than a launch takes."""
    import torch

    from detkernels_b200.kernels.paging import paged_fork, paged_fork_reference
    rng = np.random.default_rng(5)
    B, F, page = 300, 1500, 4
    lens = rng.integers(0, 40, size=B)
    src, dst = rng.integers(0, B, size=F), B + rng.permutation(F)
    table, n_blocks, free = _table(rng, lens, page, B + F, F + 5)
    w = paged_fork_reference(table.tolist(), lens.tolist() + [0] * F, src.tolist(), dst.tolist(), page,
                             free_blocks=free.tolist(), cursor=0, shares=[0] * n_blocks)
    pools = _pools(dev, n_blocks, 1, page, 8, "bfloat16", 131)
    want = [p.clone() for p in pools]
    s, d, n = (torch.tensor(x, device=dev) for x in zip(*w[4]))
    live = torch.arange(page, device=dev)[None] < n[:, None]
    for p in want:
        p[d] = torch.where(live[:, None, :, None], p[s], p[d])
    t, k, sh = _i32(table, dev), _i32(np.concatenate([lens, np.zeros(F)]), dev), _i32(np.zeros(n_blocks), dev)
    got = paged_fork(t, k, _i32(src, dev), _i32(dst, dev), page, free_blocks=_i32(free, dev), cursor=_i32([0], dev), pools=pools,
                     shares=sh)
    assert got.tolist() == [w[2]] and t.tolist() == [list(map(int, r)) for r in w[0]] and sh.tolist() == w[3]
    for a, b in zip(pools, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["src", "dst", "same", "twice", "both", "len", "negative", "block", "free_block", "free"])
@pytest.mark.parametrize("shares", [True, False])
def test_refused_fork_changes_nothing(dev, what, shares):
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.paging import paged_fork
    page = 4
    table = np.array([[3, 4, 5], [6, 7, 8], [0, 0, 0], [0, 0, 0], [0, 0, 0]])
    kv, src, dst, free, detail = [9, 6, 0, 0, 0], [0, 1, 0], [2, 3, 4], [9, 10, 11, 12, 13, 14, 15, 16], 0x640
    if what == "src":
        src[1] = 5
    elif what == "dst":
        dst[2] = -1
    elif what == "same":
        dst[1] = 1
    elif what == "twice":
        dst[2] = 2
    elif what == "both":
        src[2] = 3
    elif what in ("len", "negative"):
        kv[1], detail = (13 if what == "len" else -1), 0x641
    elif what == "block":
        table[0, 1], detail = 17, 0x642
    elif what == "free_block":
        free[2], detail = -1, 0x642
    elif what == "free":
        free, detail = free[:2], 0x643
    pools = _pools(dev, 17, 2, page, 8, "float16", 2)
    want = [p.clone() for p in pools]
    t, k, s, f = _i32(table, dev), _i32(kv, dev), _i32(np.zeros(17), dev), _i32(free, dev)
    got = paged_fork(t, k, _i32(src, dev), _i32(dst, dev), page, free_blocks=f, cursor=_i32([0], dev), pools=pools,
                     shares=s if shares else None)
    code, det = _lib.device_status(dev.index)
    assert code == _lib.DK_ERR_DEVICE_CHECK and det == detail
    assert got.tolist() == [0] and t.tolist() == table.tolist() and k.tolist() == kv and not s.any()
    for a, b in zip(pools, want):
        assert torch.equal(a, b)


def _compact_case(rng, B, page, kv_hi, new_hi, full=False):
    kv, new = rng.integers(0, kv_hi + 1, size=B), rng.integers(0, new_hi + 1, size=B)
    nk = new.copy() if full else np.array([rng.integers(0, n + 1) for n in new])
    keep = np.full((B, max(1, int(nk.max(initial=0)))), -7)
    for b in range(B):
        keep[b, :nk[b]] = np.sort(rng.permutation(int(new[b]))[:nk[b]])
    table, n_blocks, _ = _table(rng, kv + new, page, B, 3)
    return kv, new, nk, keep, table, n_blocks


@pytest.mark.gpu
@pytest.mark.parametrize("dt,Hkv,D,layout", POOLS)
@pytest.mark.parametrize("page,B,kv_hi,new_hi", [(1, 5, 3, 7), (3, 9, 20, 40), (16, 4, 50, 700), (64, 33, 200, 24)])
def test_compact(dev, dt, Hkv, D, layout, page, B, kv_hi, new_hi):
    import torch

    from detkernels_b200.kernels.paging import paged_compact, paged_compact_reference
    rng = np.random.default_rng(B)
    kv, new, nk, keep, table, n_blocks = _compact_case(rng, B, page, kv_hi, new_hi)
    handed = int((-(-(kv + new) // page)).sum())
    free = np.zeros(handed + 2, int)
    w_lens, w_cur, w_free, _, moves = paged_compact_reference(table.tolist(), kv.tolist(), new.tolist(), nk.tolist(), page,
                                                              keep=keep.tolist(), free_blocks=free.tolist(), cursor=handed)
    pools = _pools(dev, n_blocks, Hkv, page, D, dt, 2, layout)
    want = [p.clone() for p in pools]
    if moves:
        src = torch.tensor([(a, b) for a, b, _, _ in moves], device=dev).T
        dst = torch.tensor([(c, d) for _, _, c, d in moves], device=dev).T
        for p in want:      # every token is read before any is overwritten by a later one's move: sources ascend
            p[dst[0], :, dst[1]] = p[src[0], :, src[1]].clone()
    f, cur = _i32(free, dev), _i32([handed], dev)
    got = paged_compact(_i32(table, dev), _i32(kv, dev), _i32(new, dev), _i32(nk, dev), page, keep=_i32(keep, dev),
                        pools=pools, free_blocks=f, cursor=cur)
    assert got.lens.tolist() == list(map(int, w_lens)) and got.cursor.tolist() == [w_cur] and f.tolist() == w_free
    assert cur.tolist() == [handed]
    for a, b in zip(pools, want):
        assert torch.equal(a, b)
    # nothing kept moves, nothing comes back without a list
    got = paged_compact(_i32(table, dev), _i32(kv, dev), _i32(new, dev), _i32(nk, dev), page, pools=pools)
    assert got.lens.tolist() == list(map(int, w_lens)) and got.cursor is None
    for a, b in zip(pools, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 7, 300])
def test_shared_pages_come_back_once(dev, B):
    """Sequences that share pages give them up in one call and in several."""
    from detkernels_b200.kernels.paging import paged_compact, paged_compact_reference
    rng = np.random.default_rng(B)
    page, width, n_blocks = 4, 6, 40 + 3 * B
    lens = rng.integers(0, page * width + 1, size=B)
    order = rng.permutation(n_blocks)
    common, own = order[:12], list(order[12:])
    table, shares = np.zeros((B, width), int), np.full(n_blocks, -1)
    for b in range(B):
        for j in range(-(-lens[b] // page)):
            table[b, j] = common[rng.integers(0, 12)] if rng.random() < 0.7 or not own else own.pop()
    for b in range(B):      # a block twice in one row counts twice
        for j in range(-(-lens[b] // page)):
            shares[table[b, j]] += 1
    held = int((shares >= 0).sum())
    shares = np.maximum(shares, 0)
    left = rng.integers(0, lens + 1)
    t, free, cursor = _i32(table, dev), _i32(np.zeros(held), dev), held
    plain = (np.zeros(held, int).tolist(), shares.tolist())
    s = _i32(shares, dev)
    for kv, new in ((left, lens - left), (np.zeros(B, int), left)):
        zero = np.zeros(B, int)
        w = paged_compact_reference(table.tolist(), kv.tolist(), new.tolist(), zero.tolist(), page, free_blocks=plain[0],
                                    cursor=cursor, shares=plain[1])
        got = paged_compact(t, _i32(kv, dev), _i32(new, dev), _i32(zero, dev), page, free_blocks=free,
                            cursor=_i32([cursor], dev), shares=s)
        plain, cursor = (w[2], w[3]), w[1]
        assert got.cursor.tolist() == [cursor] and free.tolist() == list(map(int, w[2])) and s.tolist() == w[3]
        assert got.lens.tolist() == kv.tolist()
    assert cursor == 0 and not s.any()


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["kv", "new", "n_keep", "more", "width", "past", "order", "equal", "outside", "block", "handed",
                                  "holders"])
@pytest.mark.parametrize("shares", [True, False])
def test_refused_compaction_changes_nothing(dev, what, shares):
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.paging import paged_compact
    page = 4
    table = np.array([[3, 4, 5], [6, 7, 8], [9, 10, 11]])
    kv, new, nk, keep, cursor, detail = [2, 5, 0], [6, 6, 9], [2, 3, 2], [[1, 3, 0], [0, 4, 5], [2, 8, 0]], 9, 0x644
    sh = np.zeros(12, int)
    if what == "kv":
        kv[0] = -1
    elif what == "new":
        new[2] = -1
    elif what == "n_keep":
        nk[1] = -1
    elif what == "more":
        nk[0], new[0] = 3, 2
    elif what == "width":
        nk[2] = 4
    elif what == "past":
        new[1] = 8
    elif what in ("order", "equal", "outside"):
        keep[1], detail = {"order": [0, 5, 4], "equal": [0, 4, 4], "outside": [0, 4, 6]}[what], 0x645
    elif what == "block":
        table[0, 1], detail = 12, 0x642
    elif what == "handed":
        cursor, detail = 2, 0x643
    elif what == "holders":
        if not shares:
            pytest.skip("holders are counted in shares")
        table[2, 2], detail = 8, 0x646
        sh[4] = 1
    pools = _pools(dev, 12, 2, page, 8, "float16", 2)
    want = [p.clone() for p in pools]
    free, s = _i32(np.arange(9), dev), _i32(sh, dev)
    got = paged_compact(_i32(table, dev), _i32(kv, dev), _i32(new, dev), _i32(nk, dev), page, keep=_i32(keep, dev), pools=pools,
                        free_blocks=free, cursor=_i32([cursor], dev), shares=s if shares else None)
    code, det = _lib.device_status(dev.index)
    assert code == _lib.DK_ERR_DEVICE_CHECK and det == detail, (code, hex(det))
    assert got.lens.tolist() == kv and got.cursor.tolist() == [cursor] and free.tolist() == list(range(9))
    assert s.tolist() == sh.tolist()
    for a, b in zip(pools, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("wrong", [None, 0, 1, 31, 32, 33, 255, 256, 257, 511, 512, 998])
def test_long_rows_of_kept_tokens(dev, wrong):
    """An entry that does not ascend is found wherever it stands, and only inside a row's n_keep."""
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.paging import paged_compact
    keep = np.sort(np.stack([np.random.default_rng(b).permutation(1500)[:1003] for b in range(3)]), axis=1)
    n_keep = [1003, 999, 0]
    keep[1, 999] = -5                      # behind the row's last
    if wrong is not None:
        keep[1, wrong] = keep[1, wrong - 1] if wrong else -1
    table = _i32(np.arange(3 * 30).reshape(3, 30), dev)
    got = paged_compact(table, _i32([5, 0, 9], dev), _i32([1500] * 3, dev), _i32(n_keep, dev), 64, keep=_i32(keep, dev),
                        pools=[torch.zeros(90, 1, 64, 8, device=dev)])
    code, det = _lib.device_status(dev.index)
    if wrong is None:
        assert code == _lib.DK_OK and got.lens.tolist() == [1008, 999, 9]
    else:
        assert (code, det) == (_lib.DK_ERR_DEVICE_CHECK, 0x645) and got.lens.tolist() == [5, 0, 9]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 128, 300])
@pytest.mark.parametrize("captured", [False, True])
def test_a_life_of_pages(dev, n, captured):
    """Two forks of a prompt, one token of two drafts kept in each, all freed: in the pools of many layers."""
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.paging import paged_compact, paged_fork
    page = 4
    pools = [torch.randn(9, 1, page, 8, device=dev, generator=torch.Generator(device=dev).manual_seed(i)) for i in range(n)]
    start = [p.clone() for p in pools]
    books = [_i32([[0, 1, 2], [0, 0, 0], [0, 0, 0]], dev), _i32([10, 0, 0], dev), _i32(np.zeros(9), dev),
             _i32([0, 1, 2, 4, 5, 6, 7, 8], dev)]
    table, kv, shares, free = books
    was = [t.clone() for t in books]
    cursor, src, dst = _i32([3], dev), _i32([0, 0], dev), _i32([1, 2], dev)
    eight, two, one, none, nine = (_i32([x] * 3, dev) for x in (8, 2, 1, 0, 9))
    keep = _i32([[1]] * 3, dev)

    def step():
        at = paged_fork(table, kv, src, dst, page, free_blocks=free, cursor=cursor, shares=shares, pools=pools)
        a = paged_compact(table, eight, two, one, page, keep=keep, pools=pools, free_blocks=free, cursor=at, shares=shares)
        held = shares.clone()
        return a, held, paged_compact(table, none, nine, none, page, free_blocks=free, cursor=a.cursor, shares=shares)
    if captured:
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream(dev)
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            a, held, b = step()
        graph.replay()
        torch.cuda.synchronize()
        for p, s in zip(pools, start):
            p.copy_(s)
        for t, s in zip(books, was):
            t.copy_(s)
        graph.replay()
    else:
        a, held, b = step()
    torch.cuda.synchronize()
    _lib.raise_on_device_error(torch.cuda.current_device())
    assert a.lens.tolist() == [9] * 3 and a.cursor.tolist() == [5] and kv.tolist() == [10] * 3
    assert held.tolist() == [2, 2] + [0] * 7 and shares.tolist() == [0] * 9
    assert table.tolist() == [[0, 1, 2], [0, 1, 4], [0, 1, 5]]
    assert b.lens.tolist() == [0] * 3 and b.cursor.tolist() == [0] and free.tolist() == [2, 4, 0, 1, 5, 6, 7, 8]
    for p, s in zip(pools, start):
        for block in (2, 4, 5):      # token 9 is token 8 now
            s[block, :, :2] = s[2, :, 1:2]
        assert torch.equal(p, s)


@pytest.mark.gpu
def test_wrappers_refuse_on_the_gpu(dev):
    import torch

    from detkernels_b200.kernels.paging import paged_compact, paged_fork
    t, i, c = _i32(np.zeros((2, 2)), dev), _i32([0, 0], dev), _i32([0], dev)
    pool = torch.zeros(4, 1, 8, 8, device=dev)
    with pytest.raises(ValueError):
        paged_fork(t, i, i, i, 8, free_blocks=None, cursor=None)
    with pytest.raises(ValueError):
        paged_fork(t, i, i, i, 8, free_blocks=i, cursor=c, pools=[pool, pool])
    with pytest.raises(ValueError):
        paged_fork(t, i, i, i, 8, free_blocks=i, cursor=c, pools=[pool, torch.zeros(5, 1, 8, 8, device=dev)])
    with pytest.raises(ValueError):
        paged_fork(t, i, i, i, 8, free_blocks=i, cursor=c, pools=[pool], shares=i)
    with pytest.raises(ValueError):
        paged_fork(t, i, i, i, 8, free_blocks=i, cursor=c, pools=[pool[:1].expand(4, 1, 8, 8)])
    with pytest.raises(AssertionError):
        paged_fork(t, i, i, i, 16, free_blocks=i, cursor=c, pools=[pool])
    with pytest.raises(AssertionError):
        paged_fork(t, i[:1], i, i, 8, free_blocks=i, cursor=c)
    with pytest.raises(ValueError):
        paged_compact(t, i, i, i, 0)
    with pytest.raises(ValueError):
        paged_compact(t, i, i, i, 8, shares=i)
    with pytest.raises(ValueError):
        paged_compact(t, i, i, i, 8, free_blocks=i)
    with pytest.raises(AssertionError):
        paged_compact(t, i, i.long(), i, 8)
    with pytest.raises(AssertionError):
        paged_compact(t, i, i, i, 8, keep=i[:1, None])
    e = _i32([], dev)
    assert paged_compact(t, e, e, e, 8).lens.shape == (0,)
    assert paged_fork(t, i, e, e, 8, free_blocks=i, cursor=c).tolist() == [0]


def test_shares_without_entries_are_refused():
    """They would bound no block id, with pools or without.  (Tensors without memory, so that it runs anywhere.)"""
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode

    from detkernels_b200.kernels.paging import paged_compact, paged_fork
    with FakeTensorMode():
        dev = torch.device("cuda", 0)
        t, i, c = (torch.zeros(*s, dtype=torch.int32, device=dev) for s in ((2, 2), (2,), (1,)))
        none = torch.zeros(0, dtype=torch.int32, device=dev)
        with pytest.raises(ValueError, match="an entry a block"):
            paged_fork(t, i, i, i, 8, free_blocks=i, cursor=c, shares=none)
        with pytest.raises(ValueError, match="an entry a block"):
            paged_compact(t, i, i, i, 8, free_blocks=i, cursor=c, shares=none)
        with pytest.raises(ValueError, match="an entry a block"):
            paged_compact(t, i, i, i, 8, keep=t, free_blocks=i, cursor=c, shares=none)


@pytest.mark.gpu
@pytest.mark.parametrize("row,col", [(1, 1), (1, 2), (0, 0), (2, 2)])
@pytest.mark.parametrize("bad", [-1, 12, 2 ** 31 - 1])
@pytest.mark.parametrize("listed,shares", [(True, True), (True, False), (False, False)])
def test_a_bad_block_under_kept_tokens_changes_nothing(dev, row, col, bad, listed, shares):
    """Where moved tokens come from or go to, whether pages come back or not."""
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.paging import paged_compact
    page = 4
    table = np.array([[3, 4, 5], [6, 7, 8], [9, 10, 11]])
    table[row, col] = bad
    kv, new, nk, keep = [2, 5, 0], [6, 6, 9], [2, 3, 2], [[1, 3, 0], [0, 4, 5], [2, 8, 0]]
    pools = _pools(dev, 12, 2, page, 8, "float16", 2)
    want = [p.clone() for p in pools]
    free, cursor, s = _i32(np.arange(9), dev), _i32([9], dev), _i32(np.zeros(12), dev)
    got = paged_compact(_i32(table, dev), _i32(kv, dev), _i32(new, dev), _i32(nk, dev), page, keep=_i32(keep, dev), pools=pools,
                        free_blocks=free if listed else None, cursor=cursor if listed else None, shares=s if shares else None)
    code, det = _lib.device_status(dev.index)
    assert (code, det) == (_lib.DK_ERR_DEVICE_CHECK, 0x642), (code, hex(det))
    assert got.lens.tolist() == kv and free.tolist() == list(range(9)) and not s.any()
    assert got.cursor.tolist() == [9] if listed else got.cursor is None
    for a, b in zip(pools, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_blocks_that_no_kept_token_needs_are_not_asked_for(dev):
    """Without a free list: a page between kept tokens, the tokens that stay where they are, and a call that moves nothing."""
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.paging import paged_compact
    page = 4
    table = np.array([[3, 4, 5], [-1, 7, 8], [9, -1, 11]])
    kv, new, nk, keep = [2, 0, 0], [6, 10, 9], [2, 6, 2], [[1, 3, 0, 0, 0, 0], [0, 1, 2, 3, 5, 8], [2, 8, 0, 0, 0, 0]]
    pools = _pools(dev, 12, 2, page, 8, "float16", 2)
    want = [p.clone() for p in pools]
    for p in want:
        p[3, :, 2:] = torch.stack([p[3, :, 3], p[4, :, 1]], 1)
        p[7, :, :2] = torch.stack([p[7, :, 1], p[8, :, 0]], 1)
        p[9, :, :2] = torch.stack([p[9, :, 2], p[11, :, 0]], 1)
    args = _i32(table, dev), _i32(kv, dev), _i32(new, dev), _i32(nk, dev), page
    got = paged_compact(*args, keep=_i32(keep, dev), pools=pools)
    assert _lib.device_status(dev.index)[0] == _lib.DK_OK and got.lens.tolist() == [4, 6, 2]
    for a, b in zip(pools, want):
        assert torch.equal(a, b)
    assert paged_compact(_i32(table * 0 - 1, dev), *args[1:], keep=_i32(keep, dev)).lens.tolist() == [4, 6, 2]


@pytest.mark.gpu
@pytest.mark.parametrize("at", [0, 31, 250, 997])
def test_a_bad_block_far_into_a_long_row(dev, at):
    """Long rows are checked by many warps: entry `at` of 999 is the only one that needs the block."""
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.paging import paged_compact
    keep = np.arange(999) + 1
    table = np.arange(2 * 1002).reshape(2, 1002)
    table[1, 3 + at + 1] = -9           # pages of one token: entry at's source, entry at + 1's destination
    pool = torch.randn(2004, 1, 1, 8, device=dev)
    want = pool.clone()
    free = _i32(np.arange(2004), dev)
    got = paged_compact(_i32(table, dev), _i32([2, 3], dev), _i32([999, 999], dev), _i32([0, 998], dev), 1,
                        keep=_i32(np.stack([keep, keep]), dev), pools=[pool], free_blocks=free, cursor=_i32([2003], dev))
    code, det = _lib.device_status(dev.index)
    assert (code, det) == (_lib.DK_ERR_DEVICE_CHECK, 0x642)
    assert got.lens.tolist() == [2, 3] and got.cursor.tolist() == [2003] and free.tolist() == list(range(2004))
    assert torch.equal(pool, want)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["thinned", "both", "given_up", "last_page"])
def test_tokens_are_not_moved_into_a_shared_page(dev, what):
    """Two sequences share the blocks 0 and 1 of four tokens: thinning one out would change the other's."""
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.paging import paged_compact
    page = 4
    table, shares = np.array([[0, 1, 2], [0, 1, 3]]), [1, 1, 0, 0, 0]
    kv, new, nk = [0, 0], [11, 10], [11, 5]
    keep = [list(range(11)), [0, 2, 3, 5, 9] + [0] * 6]
    if what == "both":              # in the same way: their moves would meet
        nk[0], keep[0] = 5, keep[1]
    elif what == "given_up":        # by the other one in the same call
        nk[0] = 0
    elif what == "last_page":       # only the last kept token's page is shared still
        shares, nk[1], keep[1] = [0, 1, 0, 0, 0], 6, [0, 2, 3, 5, 8, 9] + [0] * 5
    pools = _pools(dev, 5, 2, page, 8, "float16", 2)
    want = [p.clone() for p in pools]
    free, cursor, s = _i32([0, 1, 2, 3, 4], dev), _i32([4], dev), _i32(shares, dev)
    got = paged_compact(_i32(table, dev), _i32(kv, dev), _i32(new, dev), _i32(nk, dev), page, keep=_i32(keep, dev), pools=pools,
                        free_blocks=free, cursor=cursor, shares=s)
    code, det = _lib.device_status(dev.index)
    assert (code, det) == (_lib.DK_ERR_DEVICE_CHECK, 0x647), (code, hex(det))
    assert got.lens.tolist() == kv and got.cursor.tolist() == [4] and free.tolist() == list(range(5)) and s.tolist() == shares
    for a, b in zip(pools, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_shared_pages_before_the_first_moved_token(dev):
    """They stay as they are, are read from and given up; once the other sequence is freed, tokens move in them, too."""
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.paging import paged_compact
    page = 4
    pools = _pools(dev, 6, 2, page, 8, "float16", 2)
    want = [p.clone() for p in pools]
    free, s = _i32([0] * 6, dev), _i32([1, 0, 0, 1, 0, 0], dev)
    t, kv = _i32([[0, 1, 3], [0, 2, 3]], dev), _i32([0, 0], dev)
    # sequence 1 keeps its first five tokens and the two behind them in block 3, which it gives up
    keep = _i32([list(range(12)), [0, 1, 2, 3, 4, 8, 10] + [0] * 5], dev)
    a = paged_compact(t, kv, _i32([12, 12], dev), _i32([12, 7], dev), page, keep=keep, pools=pools, free_blocks=free,
                      cursor=_i32([5], dev), shares=s)
    assert _lib.device_status(dev.index)[0] == _lib.DK_OK
    assert a.lens.tolist() == [12, 7] and a.cursor.tolist() == [5] and s.tolist() == [1, 0, 0, 0, 0, 0]
    for p in want:
        p[2, :, 1:3] = p[3, :, 0:3:2]
    for x, y in zip(pools, want):
        assert torch.equal(x, y)
    b = paged_compact(t, kv, _i32([12, 0], dev), _i32([0, 0], dev), page, free_blocks=free, cursor=a.cursor, shares=s)
    assert b.cursor.tolist() == [3] and free.tolist()[3:5] == [1, 3] and not s.any()
    c = paged_compact(t, kv, _i32([0, 7], dev), _i32([0, 2], dev), page, keep=_i32([[0, 0], [1, 6]], dev), pools=pools,
                      free_blocks=free, cursor=b.cursor, shares=s)
    assert _lib.device_status(dev.index)[0] == _lib.DK_OK
    assert c.lens.tolist() == [0, 2] and c.cursor.tolist() == [2] and free.tolist()[2:5] == [2, 1, 3]
    for p in want:
        p[0, :, 0], p[0, :, 1] = p[0, :, 1].clone(), p[2, :, 2]
    for x, y in zip(pools, want):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_calls_of_nothing_hand_the_cursor_on(dev):
    """Through the C entries, whose callers chain the cursors themselves."""
    import torch

    from detkernels_b200 import _lib
    lib = _lib.load()
    books, cursor, out = _i32(np.zeros(8), dev), _i32([5], dev), _i32([-1, -1], dev)
    at, st = books.data_ptr(), _lib.stream_ptr(dev)
    assert lib.dk_paged_fork(at, 2, 4, 2, at, None, None, 0, 8, at, 8, cursor.data_ptr(), out.data_ptr(), None, 9, None, 0,
                             0, 0, 0, 0, 0, 2, None, 0, st) == _lib.DK_OK

    def compact(free, to):
        return lib.dk_paged_compact(at, 2, 2, None, None, None, None, 0, 0, 0, 8, None, free, 8, cursor.data_ptr(), to, None, 9,
                                    None, 0, 0, 0, 0, 0, 0, 2, None, 0, st)
    assert compact(at, out[1:].data_ptr()) == _lib.DK_OK and out.tolist() == [5, 5]
    assert compact(at, cursor.data_ptr()) == _lib.DK_OK and cursor.tolist() == [5]
    assert compact(None, None) == _lib.DK_OK      # without a free list there is no cursor
    torch.cuda.synchronize(dev)
