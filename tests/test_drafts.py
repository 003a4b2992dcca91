"""Trees of drafted tokens: masks and accepted paths against the plain forms."""
import numpy as np
import pytest


def _trees(rng, sizes, reach=8):
    """Parents of each tree's nodes, node 0 the root."""
    out = []
    for n in sizes:
        out += [-1 if i == 0 else int(rng.integers(max(0, i - reach), i)) for i in range(n)]
    return np.array(out, np.int32)


def _cu(sizes):
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)


def _plain_mask(parents, cu, words):
    want = np.zeros((len(parents), 64 * words), bool)
    for a, b in zip(cu[:-1], cu[1:]):
        for i in range(b - a):
            j = i
            while j >= 0:
                if j < 64 * words:
                    want[a + i, j] = True
                j = parents[a + j]
    return want


def _bits(mask):
    return np.unpackbits(np.ascontiguousarray(mask.cpu().numpy()).view(np.uint8), axis=1, bitorder="little").astype(bool)


def test_tree_mask():
    import torch

    from detkernels_b200.kernels.drafts import tree_mask
    rng = np.random.default_rng(0)
    for sizes, words in (([1, 5, 0, 64, 3], 1), ([0, 130, 7, 0], 3), ([], 2), ([90], 1)):
        parents, cu = _trees(rng, sizes, reach=3), _cu(sizes)
        mask = tree_mask(torch.from_numpy(parents), torch.from_numpy(cu), words)
        assert mask.dtype == torch.int64 and mask.shape == (len(parents), words)
        assert (_bits(mask) == _plain_mask(parents, cu, words)).all()
    # nodes beyond the words have no bit, and their rows those of all their ancestors; a bound on the nodes changes nothing
    parents, cu = _trees(rng, [7, 200, 31], reach=1), _cu([7, 200, 31])
    for words, bound in ((1, None), (1, 200), (2, 1000), (4, 200)):
        mask = tree_mask(torch.from_numpy(parents), torch.from_numpy(cu), words, max_rows=bound)
        assert (_bits(mask) == _plain_mask(parents, cu, words)).all()
    # a chain is as deep as it is long; rows behind the last sequence have no bits
    chain = torch.arange(-1, 127, dtype=torch.int32)
    mask = tree_mask(torch.cat([chain, chain[:3]]), torch.tensor([0, 128], dtype=torch.int32), 2)
    assert (_bits(mask)[:128] == np.tril(np.ones((128, 128), bool))).all() and not _bits(mask)[128:].any()


def test_accept_reference():
    from detkernels_b200.kernels.drafts import tree_accept_reference
    # 0 -> {1: 5, 2: 6}, 2 -> {3: 7}
    r = tree_accept_reference([-1, 0, 0, 2], [4, 5, 6, 7], [6, 1, 7, 9], [0, 4, 4], max_keep=5)
    assert r.keep == [[0, 2, 3, -1, -1], [-1] * 5] and r.n_keep == [3, 0] and r.next_tokens == [9, -1]
    assert tree_accept_reference([-1, 0, 0, 2], [4, 5, 6, 7], [6, 1, 7, 9], [0, 4], max_keep=2).next_tokens == [7]


def test_entry_point_refuses_on_the_host():
    from detkernels_b200 import _lib
    lib = _lib.load()

    def call(n_seqs=2, n_rows=4, max_keep=3, cu=16, par=16):
        return lib.dk_tree_accept(par, 16, 16, cu, n_seqs, n_rows, max_keep, 16, 16, 16, None)
    assert call(n_seqs=0) == _lib.DK_OK
    assert call(n_seqs=-1) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(n_rows=-1) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(max_keep=0) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(cu=None) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(par=None) == _lib.DK_ERR_INVALID_ARGUMENT


def test_wrapper_refuses():
    import torch

    from detkernels_b200.kernels.drafts import tree_accept
    i, t = torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(AssertionError):
        tree_accept(i, t, t, i, max_keep=2)


def _dev(dev, a, dt=np.int32):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a).astype(dt)).to(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,reach", [([1], 1), ([0], 1), ([0, 3, 0, 0, 2], 2), (list(range(40)), 4), ([64, 65, 128, 129, 300], 3),
                                         ([1000, 1], 60), ([33] * 777, 8)])
@pytest.mark.parametrize("max_keep", [1, 5, 33, 400])
def test_accept(dev, sizes, reach, max_keep):
    from detkernels_b200.kernels.drafts import tree_accept, tree_accept_reference
    rng = np.random.default_rng(len(sizes) + max_keep)
    parents, cu = _trees(rng, sizes, reach), _cu(sizes)
    n = len(parents)
    at = np.arange(n) - np.repeat(cu[:-1], sizes)
    tokens, picked = rng.integers(0, 4, size=n), rng.integers(0, 4, size=n)     # few tokens: siblings agree too
    deep = np.nonzero((parents >= 0) & (rng.random(n) < 0.7))[0]
    picked[deep - at[deep] + parents[deep]] = tokens[deep]
    big = rng.random() < 0.5
    if big:
        tokens, picked = tokens + 2 ** 33, picked + 2 ** 33
    want = tree_accept_reference(parents.tolist(), tokens.tolist(), picked.tolist(), cu.tolist(), max_keep=max_keep)
    # rows behind the last sequence are not read
    pad = 3
    got = tree_accept(_dev(dev, np.concatenate([parents, np.zeros(pad)])), _dev(dev, np.concatenate([tokens, [0] * pad]), np.int64),
                      _dev(dev, np.concatenate([picked, [0] * pad]), np.int64), _dev(dev, cu), max_keep=max_keep)
    assert got.keep.tolist() == want.keep and got.n_keep.tolist() == want.n_keep
    assert got.next_tokens.tolist() == want.next_tokens


@pytest.mark.gpu
def test_bad_offsets_set_the_status(dev):
    from detkernels_b200 import _lib
    from detkernels_b200.kernels.drafts import tree_accept
    par, tok = _dev(dev, [-1, 0, -1, 0]), _dev(dev, [1, 2, 3, 4], np.int64)
    for cu in ([0, 2, 5], [0, 2, 1], [-1, 2, 4]):
        r = tree_accept(par, tok, _dev(dev, [2, 0, 4, 0], np.int64), _dev(dev, cu), max_keep=3)
        code, detail = _lib.device_status(dev.index)
        assert code == _lib.DK_ERR_DEVICE_CHECK and detail == 0x660
        bad = [not 0 <= a <= b <= 4 for a, b in zip(cu, cu[1:])]
        for b in range(2):
            assert (r.n_keep[b].item() == 0 and r.next_tokens[b].item() == -1) if bad[b] else r.n_keep[b].item() > 0


@pytest.mark.gpu
def test_accept_refuses_on_the_gpu(dev):
    import torch

    from detkernels_b200.kernels.drafts import tree_accept
    i, t = _dev(dev, [0, 2]), _dev(dev, [0, 2], np.int64)
    with pytest.raises(ValueError):
        tree_accept(i, t, t, i, max_keep=0)
    with pytest.raises(AssertionError):
        tree_accept(i, t, t[:1], i, max_keep=2)
    with pytest.raises(AssertionError):
        tree_accept(i, i, t, i, max_keep=2)
    r = tree_accept(i, t, t, i[:1], max_keep=2)
    assert r.keep.shape == (0, 2) and torch.numel(r.next_tokens) == 0
