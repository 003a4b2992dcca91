"""Shared-prefix attention of batches large enough that a run of the prefix is a whole group of chunks, joined on chip:
the bits of small batches, whose chunks are joined through memory, and the definition's values."""
import numpy as np
import pytest

from test_shared_prefix import _call, _dt, _make, _tol_check


def _runs(R, H, Hkv, D, P):
    """Runs of the prefix, from the states that the workspace of a call without own tokens holds a row."""
    from detkernels_b200 import _lib
    n = _lib.load().dk_attention_shared_prefix_workspace_size(R, R, H, Hkv, D, P, 0)
    return n // (R * H * (D + 2) * 4)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,R,H,Hkv,D,P,page,most", [
    # head_dim 128: groups of 4 chunks; the last group and its last chunk are short
    ("bf16", 1000, 16, 1, 128, 4500, 0, 90),      # 5 chunks; several warps a row of own tokens
    ("f16", 1010, 16, 2, 128, 5000, 64, 90),      # 5 chunks; one warp a row
    ("bf16", 705, 16, 2, 128, 9100, 128, 200),    # 9 chunks; the last pair of row tiles has one
    ("f16", 300, 32, 4, 128, 9990, 0, 1),         # 10 chunks
    ("f16", 512, 32, 4, 128, 8191, 0, 127),       # two whole groups
    ("bf16", 1000, 32, 4, 128, 2048, 0, 70),      # one group of 4 chunks of 512
    ("bf16", 1300, 32, 8, 128, 7990, 64, 20),     # 336 items, several a CTA; the last pair of row tiles has one
    # up to head_dim 64: groups of 8
    ("f16", 2001, 32, 8, 64, 2048, 0, 30),        # 256 items
    ("bf16", 1184, 16, 1, 64, 14500, 0, 64),      # 15 chunks in two groups
    ("f16", 1184, 16, 1, 32, 14337, 64, 40),      # 15, the last of one token
    ("f16", 1005, 32, 4, 64, 5100, 256, 130),     # 5 chunks in one group
    ("bf16", 1000, 32, 4, 32, 1500, 0, 10)])      # 3 chunks of 512
def test_whole_groups_give_the_bits_of_chunks(dev, dt, R, H, Hkv, D, P, page, most):
    import torch
    small = ((0, 1), (R // 2, R // 2 + 9), (R - 1, R))
    chunks, runs = _runs(1, H, Hkv, D, P), _runs(R, H, Hkv, D, P)
    group = 8 if D <= 64 else 4
    # both schedules are taken, or this test shows nothing
    assert 1 < chunks == max(_runs(hi - lo, H, Hkv, D, P) for lo, hi in small) and runs == -(-chunks // group) < chunks
    rng = np.random.default_rng(R)
    lens = [int(x) for x in rng.integers(0, most + 1, size=R)]
    q, kp, vp, own, kw = _make(dev, _dt(dt), R, H, Hkv, D, P, lens, page, seed=D + P)
    full = _call(q, kw, lens)
    assert torch.equal(_call(q, kw, lens), full)
    for lo, hi in small:
        part = dict(kw, kwargs=dict(kw["kwargs"]))
        if page:
            part["kwargs"]["block_table"] = kw["kwargs"]["block_table"][lo:hi]
        else:
            part["kv"] = tuple(x[lo:hi] for x in kw["kv"])
        assert torch.equal(_call(q[lo:hi], part, lens[lo:hi]), full[lo:hi])
    some = [0, R // 3, R - 1]
    _tol_check(full[some], q[some], kp, vp, [own[i][0] for i in some], [own[i][1] for i in some], D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("D,P,R,H,Hkv", [(128, 4500, 1000, 16, 2), (64, 5100, 1005, 32, 4)])
def test_rising_and_peaked_scores_in_whole_groups(dev, D, P, R, H, Hkv):
    """Maxima that rise from chunk to chunk, fall, or sit in the last one alone: the joins' weights run from 0 to 1 both
    ways, and an accumulator that is joined in two places stays one row's."""
    import torch
    assert _runs(R, H, Hkv, D, P) < _runs(1, H, Hkv, D, P)
    lens = [3] * R
    q, kp, vp, own, kw = _make(dev, torch.bfloat16, R, H, Hkv, D, P, lens, seed=7)
    t = torch.arange(P, device=dev).float()
    for ramp in (t / P - 0.5, 0.5 - t / P, (t >= P - 5).float(), (t // 700 % 2)):
        kp2 = (kp.float() * 0.3 + ramp[None, :, None]).to(kp.dtype)
        q2 = (q.float() * 0.2 + torch.where(torch.arange(R, device=dev) % 2 == 0, 1.0, -1.0)[:, None, None]).to(q.dtype)
        kw2 = dict(kw, prefix=(kp2, vp))
        full = _call(q2, kw2, lens)
        for lo, hi in ((0, 2), (R - 3, R)):
            part = dict(kw2, kv=tuple(x[lo:hi] for x in kw["kv"]))
            assert torch.equal(_call(q2[lo:hi], part, lens[lo:hi]), full[lo:hi])
        some = [0, R - 1]
        _tol_check(full[some], q2[some], kp2, vp, [own[i][0] for i in some], [own[i][1] for i in some], D ** -0.5)
