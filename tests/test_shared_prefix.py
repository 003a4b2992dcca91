"""Attention over a shared prefix: against the definition in 64 bits, bitwise batch invariance, refusals, and a
decode step of plan, norm with rotation and attention together."""
import math

import numpy as np
import pytest


def _dt(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16}[name]


def _tol_check(got, q, kp, vp, ks, vs, scale):
    """Row by row against f64.  With A = sum p |v| / sum p and half a step h = eps / 2 of the type: the
    rounded weights move the result by at most 2 h A (h in the sums of products, and h in the own tokens'
    sum of weights), a score's f32 dot product of D terms is off by at most D 2^-24 sum |q k| scale =: E,
    which moves weights and their sum by E each, the f32 sums of a chunk by 2 (1024 or a sixteenth of the prefix, + 64) 2^-24 A, and the
    store rounds once.  (ks, vs: a row's own tokens [H_kv, n, D], n may be 0.)"""
    import torch
    R, H, D = got.shape
    eps = torch.finfo(got.dtype).eps
    for r in range(R):
        k = torch.cat([kp, ks[r]], 1).double().repeat_interleave(H // kp.shape[0], 0)
        v = torch.cat([vp, vs[r]], 1).double().repeat_interleave(H // kp.shape[0], 0)
        qr = q[r].double()[:, None]
        s = (qr @ k.transpose(1, 2))[:, 0] * scale
        E = (qr.abs() @ k.abs().transpose(1, 2)).amax() * abs(scale) * D * 2.0 ** -24
        p = torch.softmax(s, -1)
        want = (p[:, None] @ v)[:, 0]
        A = (p[:, None] @ v.abs())[:, 0]
        chunk = max(1024, kp.shape[1] // 16 + 128)
        tol = eps / 2 * want.abs() + A * (eps + 2 * E + 2 * (chunk + 64) * 2.0 ** -24)
        if got.dtype == torch.float16:
            tol = tol + 2.0 ** -25 + v.abs().amax() * 2.0 ** -24    # subnormal weights and results
        bad = ((got[r].double() - want).abs() - tol).max().item()
        assert bad <= 0, (r, bad)


def _make(dev, dt, R, H, Hkv, D, P, lens, page=0, seed=0, scale_q=1.0):
    """q, prefix and own tokens; paged: the prefix and the rows' tokens share scattered blocks of one pool."""
    import torch
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)

    def randn(*s):
        return torch.randn(*s, device=dev, generator=g).to(dt)
    q = (randn(R, H, D).float() * scale_q).to(dt)
    kp, vp = randn(Hkv, P, D), randn(Hkv, P, D)
    cap = -(-max(1, max(lens)) // 64) * 64
    k, v = randn(len(lens), Hkv, cap, D), randn(len(lens), Hkv, cap, D)
    own = [(k[i, :, :n], v[i, :, :n]) for i, n in enumerate(lens)]
    kw = dict(kv=(k, v), prefix=(kp, vp), kwargs={})
    if page:
        per = -(-cap // page)
        npre = -(-P // page)
        n_blocks = len(lens) * per + npre + 2
        order = rng.permutation(n_blocks)
        pool = [torch.full((n_blocks, Hkv, page, D), float("nan"), device=dev, dtype=dt) for _ in range(2)]
        table = order[:len(lens) * per].reshape(len(lens), per)
        pre = order[len(lens) * per:len(lens) * per + npre]
        for x, (src, psrc) in zip(pool, ((k, kp), (v, vp))):
            for i, n in enumerate(lens):
                for t0 in range(0, n, page):
                    m = min(page, n - t0)
                    x[table[i, t0 // page], :, :m] = src[i, :, t0:t0 + m]
            for t0 in range(0, P, page):
                m = min(page, P - t0)
                x[pre[t0 // page], :, :m] = psrc[:, t0:t0 + m]
        i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a.astype(np.int32))).to(dev)
        kw["kv"] = kw["prefix"] = tuple(pool)
        kw["kwargs"] = dict(prefix_len=P, prefix_blocks=i32(pre), block_table=i32(table))
    return q, kp, vp, own, kw


def _call(q, kw, lens, **extra):
    import torch

    from detkernels_b200.kernels.attention import attention_shared_prefix
    ln = lens if isinstance(lens, (int, torch.Tensor)) else torch.tensor(lens, dtype=torch.int32, device=q.device)
    return attention_shared_prefix(q, *kw["prefix"], *kw["kv"], ln, **kw["kwargs"], **extra)


def test_refusals_on_the_host():
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.attention import attention_shared_prefix
    z = torch.zeros(1, 2, 64)
    with pytest.raises(AssertionError):
        attention_shared_prefix(z, z, z, z[None], z[None], 1)
    lib = _lib.load()

    def call(dtype=_lib.DK_BF16, D=64, H=4, Hkv=2, P=10, pb=None, pool=0, pg=0, qs=512, q=16, max_len=0, pst=64,
             cst=64, n_seq=3, table=None, page=0, width=1):
        return lib.dk_attention_shared_prefix(
            q, qs, D, 16, 16, 0, 640, pst, P, pb, pool, pg, 16, 16, 0, 0, cst, n_seq, 64, table, width, width, 4, page,
            16, qs, D, 16, None, 0, 3, H, Hkv, D, max_len, 0.1, dtype, 16, 0, None)
    assert call(dtype=_lib.DK_F32) == _lib.DK_ERR_UNSUPPORTED
    assert call(D=96) == _lib.DK_ERR_UNSUPPORTED and call(H=34) == _lib.DK_ERR_UNSUPPORTED
    assert call(H=5) == _lib.DK_ERR_INVALID_ARGUMENT and call(P=0) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(max_len=-1) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(q=8) == _lib.DK_ERR_INVALID_ARGUMENT and call(qs=260) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(pst=68) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(pb=16, pool=4, pg=96) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(max_len=9, cst=4) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(max_len=9, n_seq=2) == _lib.DK_ERR_INVALID_ARGUMENT and "fewer KV sequences" in _lib.last_error()
    assert call(max_len=9, table=16, page=32) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call() == _lib.DK_ERR_WORKSPACE and "bytes needed" in _lib.last_error()
    # room for the chunk states of every (row, head) and for the rows' own tokens
    assert lib.dk_attention_shared_prefix_workspace_size(3, 3, 4, 2, 64, 1025, 600) >= (3 + 3) * 3 * 4 * (64 + 2) * 4


def test_reference_joins_prefix_and_own_tokens():
    import torch

    from detkernels_b200.kernels.attention import attention_reference, attention_shared_prefix_reference
    g = torch.Generator().manual_seed(0)
    q, kp, vp = torch.randn(2, 4, 8, generator=g), torch.randn(2, 5, 8, generator=g), torch.randn(2, 5, 8, generator=g)
    k, v = torch.randn(2, 2, 3, 8, generator=g), torch.randn(2, 2, 3, 8, generator=g)
    got = attention_shared_prefix_reference(q, kp, vp, k, v, [3, 0])
    want = attention_reference(q[:1], torch.cat([kp, k[0]], 1)[None], torch.cat([vp, v[0]], 1)[None])
    assert torch.equal(got[:1], want)
    assert torch.equal(got[1:], attention_reference(q[1:], kp[None], vp[None]))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("R,H,Hkv,D,P,page", [
    (1, 1, 1, 64, 1, 0), (1, 4, 4, 128, 15, 0), (3, 4, 2, 32, 63, 64), (2, 8, 1, 64, 64, 64), (5, 6, 2, 128, 65, 128),
    (4, 8, 8, 64, 500, 0), (9, 16, 1, 128, 127, 64), (130, 2, 2, 64, 129, 0), (129, 2, 1, 128, 513, 64),
    (33, 20, 4, 32, 1025, 0), (17, 30, 2, 128, 1111, 256), (300, 3, 3, 32, 640, 64), (40, 8, 2, 128, 4500, 64),
    (12, 4, 1, 64, 17000, 0)])
def test_against_the_definition(dev, dt, R, H, Hkv, D, P, page):
    rng = np.random.default_rng(R + P)
    lens = [int(x) for x in rng.integers(0, 90, size=R)]
    lens[0] = 0
    q, kp, vp, own, kw = _make(dev, _dt(dt), R, H, Hkv, D, P, lens, page, seed=P)
    out = _call(q, kw, lens)
    some = sorted({0, 1, R // 2, R - 1} & set(range(R)))
    _tol_check(out[some], q[some], kp, vp, [own[i][0] for i in some], [own[i][1] for i in some], D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("scale_q,scale", [(6.0, None), (1.0, -0.2), (1.0, 0.0), (30.0, 0.125)])
def test_peaked_scores_and_scales(dev, scale_q, scale):
    """Large scores raise the running maximum again and again; a negative or zero scale is as valid."""
    import torch
    lens = [70, 0, 300, 5, 1, 64]
    for D in (64, 128):
        q, kp, vp, own, kw = _make(dev, torch.bfloat16, 6, 4, 2, D, 2000, lens, 64, seed=3, scale_q=scale_q)
        out = _call(q, kw, lens, scale=scale)
        _tol_check(out, q, kp, vp, [o[0] for o in own], [o[1] for o in own], D ** -0.5 if scale is None else scale)


@pytest.mark.gpu
def test_rising_scores_rescale_every_block(dev):
    """Keys ordered so that each 128-token block's maximum is far above the last: the accumulator is
    rescaled at every block, and the early tokens fall out."""
    import torch
    D, P = 64, 1300
    q = torch.ones(2, 2, D, device=dev, dtype=torch.bfloat16)
    ramp = (torch.arange(P, device=dev) // 100 - 6).float()[None, :, None].expand(1, P, D)
    kp = (ramp * 0.25).to(torch.bfloat16).contiguous()
    g = torch.Generator(device=dev).manual_seed(1)
    vp = torch.randn(1, P, D, device=dev, generator=g).to(torch.bfloat16)
    k = torch.zeros(2, 1, 64, D, device=dev, dtype=torch.bfloat16)
    for sgn in (1.0, -1.0):
        out = _call(q, dict(prefix=(kp, vp), kv=(k, k), kwargs={}), 0, scale=sgn)
        e = torch.zeros(1, 0, D, device=dev, dtype=torch.bfloat16)
        _tol_check(out, q, kp, vp, [e, e], [e, e], sgn)


def _tiles(lens, rpt):
    tiles, at = [], 0
    for s, n in enumerate(lens):
        tiles += [(at + i, min(rpt, n - i), s) for i in range(0, n, rpt)]
        at += n
    return np.array(tiles, np.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,D,page", [(4, 2, 64, 64), (16, 1, 128, 0), (3, 3, 32, 128)])
def test_prefill_rows_of_ragged_sequences(dev, H, Hkv, D, page):
    """Several rows a sequence through row tiles, row i seeing i + 1 own tokens: the bits of single rows."""
    import torch
    lens = [5, 1, 40, 17]
    q0, kp, vp, own, kw = _make(dev, torch.bfloat16, 4, H, Hkv, D, 700, lens, page, seed=2)
    rows = sum(lens)
    q = torch.randn(rows, H, D, device=dev, generator=torch.Generator(device=dev).manual_seed(8)).to(torch.bfloat16)
    q_lens = [i + 1 for n in lens for i in range(n)]
    seq = [s for s, n in enumerate(lens) for _ in range(n)]
    tiles = torch.from_numpy(_tiles(lens, 16 // (H // Hkv))).to(dev)
    out = _call(q, kw, q_lens, row_tiles=tiles)
    some = [0, 5, 6, 30, rows - 1]
    _tol_check(out[some], q[some], kp, vp, [own[seq[r]][0][:, :q_lens[r]] for r in some],
               [own[seq[r]][1][:, :q_lens[r]] for r in some], D ** -0.5)
    one = torch.tensor([[0, 1, seq[30]]], dtype=torch.int32, device=dev)
    assert torch.equal(_call(q[30:31], kw, [q_lens[30]], row_tiles=one)[0], out[30])


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,D,n_seq", [(4, 2, 64, 3), (4, 2, 64, 700), (16, 1, 128, 5), (2, 2, 32, 40)])
def test_rows_that_no_tile_covers_are_left(dev, H, Hkv, D, n_seq):
    """A batch padded behind its last sequence, and a gap in its middle: those rows keep what out held, whether
    one warp owns a row (many tiles) or several do; the covered rows' bits are those of a batch without them."""
    import torch
    rng = np.random.default_rng(n_seq)
    lens = [int(x) for x in rng.integers(1, 6, size=n_seq)]
    q0, kp, vp, own, kw = _make(dev, torch.bfloat16, n_seq, H, Hkv, D, 300, lens, seed=4)
    gap, pad = 3, 9
    first = np.cumsum([0] + lens)[:-1] + gap * (np.arange(n_seq) >= n_seq // 2)
    rows = int(first[-1] + lens[-1] + pad)
    tiles = np.array([(f, n, s) for s, (f, n) in enumerate(zip(first, lens)) if n * (H // Hkv) <= 16]
                     + [(f + i, 1, s) for s, (f, n) in enumerate(zip(first, lens)) if n * (H // Hkv) > 16
                        for i in range(n)], np.int32)
    rng.shuffle(tiles)
    q = torch.randn(rows, H, D, device=dev, generator=torch.Generator(device=dev).manual_seed(8)).to(torch.bfloat16)
    q_lens = np.zeros(rows, np.int32)
    for f, n in zip(first, lens):
        q_lens[f:f + n] = np.arange(1, n + 1)
    covered = torch.from_numpy(q_lens > 0).to(dev)
    q_lens[q_lens == 0] = 5   # a length of a row that is not there
    out = torch.full_like(q, 7.0)
    ln, tl = torch.from_numpy(q_lens).to(dev), torch.from_numpy(tiles).to(dev)
    _call(q, kw, ln, row_tiles=tl, out=out)
    assert (out[~covered] == 7.0).all() and int((~covered).sum()) == gap + pad
    tight = torch.from_numpy(_tiles(lens, 16 // (H // Hkv))).to(dev)
    assert torch.equal(out[covered], _call(q[covered], kw, ln[covered], row_tiles=tight))


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,D,P", [(8, 2, 64, 1500), (8, 8, 128, 700), (16, 2, 128, 5000), (24, 8, 128, 5000),
                                       (4, 1, 32, 20000)])
def test_a_row_does_not_depend_on_its_batch(dev, H, Hkv, D, P):
    """The same rows alone, in small batches and in one that takes whole groups a run: the same bits."""
    import torch
    rng = np.random.default_rng(0)
    R = 800
    lens = [int(x) for x in rng.integers(0, 300, size=R)]
    q, kp, vp, own, kw = _make(dev, torch.bfloat16, R, H, Hkv, D, P, lens, seed=1)
    full = _call(q, kw, lens)
    for lo, hi in ((0, 1), (3, 4), (10, 75), (100, 356), (799, 800)):
        part = dict(kw, kv=tuple(x[lo:hi] for x in kw["kv"]))
        assert torch.equal(_call(q[lo:hi], part, lens[lo:hi]), full[lo:hi])
    again = _call(q, kw, lens)
    assert torch.equal(again, full)
    some = [0, 399, 799]
    _tol_check(full[some], q[some], kp, vp, [own[i][0] for i in some], [own[i][1] for i in some], D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D,page", [("bf16", 64, 64), ("f16", 128, 0), ("bf16", 32, 128)])
def test_values_behind_a_rows_end_never_reach_it(dev, dt, D, page):
    """Prefill rows whose later tokens hold infinities and NaN, and cache rows with NaN behind the end: each
    row's bits are those of a call that only has its own tokens."""
    import torch
    lens, H, Hkv = [37, 5], 4, 2
    q0, kp, vp, own, kw = _make(dev, _dt(dt), 2, H, Hkv, D, 150, lens, page, seed=6)
    rows = sum(lens)
    q = torch.randn(rows, H, D, device=dev, generator=torch.Generator(device=dev).manual_seed(8)).to(_dt(dt))
    q_lens = [i + 1 for n in lens for i in range(n)]
    tiles = torch.from_numpy(_tiles(lens, 16 // (H // Hkv))).to(dev)
    want = _call(q, kw, q_lens, row_tiles=tiles)
    kc, vc = (x.clone() for x in kw["kv"])
    for t, bad in ((20, float("inf")), (21, float("nan")), (30, -float("inf"))):
        if page:
            b = int(kw["kwargs"]["block_table"][0, t // page])
            vc[b, :, t % page, 3], kc[b, :, t % page, 1] = bad, float("nan")
        else:
            vc[0, :, t, 3], kc[0, :, t, 1] = bad, float("nan")
            vc[:, :, 37:], kc[:, :, 37:] = float("nan"), float("nan")
    kw2 = dict(kw, kv=(kc, vc))
    if page:
        kw2["prefix"] = kw["prefix"]
    got = _call(q, kw2, q_lens, row_tiles=tiles)
    fine = [r for r in range(rows) if r < 20 or r >= 37]
    assert torch.equal(got[fine], want[fine]) and torch.isfinite(got[fine].float()).all()
    assert torch.isnan(got[21:37].float()).any(-1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("R,H,Hkv,D,page", [(2, 4, 1, 64, 64), (3, 2, 2, 128, 0), (1, 16, 1, 128, 256), (700, 2, 1, 32, 0),
                                               (700, 6, 3, 32, 0)])
def test_long_own_sequences(dev, R, H, Hkv, D, page):
    """Own tokens over many splits, by one warp (many rows) or many (few rows): one definition, the same bits."""
    import torch
    rng = np.random.default_rng(R)
    lens = [int(x) for x in rng.integers(0, 1300 if R > 100 else 5000, size=R)]
    lens[0] = 1025
    q, kp, vp, own, kw = _make(dev, torch.bfloat16, R, H, Hkv, D, 77, lens, page, seed=R)
    out = _call(q, kw, lens)
    some = list(range(min(R, 3)))
    _tol_check(out[some], q[some], kp, vp, [own[i][0] for i in some], [own[i][1] for i in some], D ** -0.5)
    if R > 100:
        part = dict(kw, kv=tuple(x[:2] for x in kw["kv"]))
        assert torch.equal(_call(q[:2], part, lens[:2]), out[:2])


@pytest.mark.gpu
def test_no_own_tokens_no_prefix_and_no_rows(dev):
    import torch

    from detkernels_b200.kernels.attention import attention_decode, attention_shared_prefix
    lens = [33, 0, 64]
    q, kp, vp, own, kw = _make(dev, torch.float16, 3, 4, 2, 64, 200, lens)
    e = torch.zeros(2, 0, 64, device=dev, dtype=q.dtype)
    none = _call(q, kw, 0)
    _tol_check(none, q, kp, vp, [e] * 3, [e] * 3, 0.125)
    assert torch.equal(none, _call(q, kw, [0, 0, 0]))
    assert torch.equal(none[1], _call(q, kw, lens)[1])
    ln = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = attention_shared_prefix(q, kp, vp, *kw["kv"], ln, prefix_len=0)
    assert torch.equal(got, attention_decode(q, *kw["kv"], ln)) and (got[1] == 0).all()
    assert _call(q[:0], kw, []).shape == (0, 4, 64)
    # a shorter prefix than the buffer holds; what lies behind it may be anything
    kp2, vp2 = kp.clone(), vp.clone()
    kp2[:, 131:], vp2[:, 131:] = float("nan"), float("inf")
    got = attention_shared_prefix(q, kp2, vp2, *kw["kv"], ln, prefix_len=131)
    want = attention_shared_prefix(q, kp[:, :131].contiguous(), vp[:, :131].contiguous(), *kw["kv"], ln)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_strides_streams_and_out(dev):
    """Prefix views inside larger tensors, a strided q and out, another stream: the same bits."""
    import torch

    from detkernels_b200.kernels.attention import attention_shared_prefix
    lens = [9, 30, 2, 0, 64]
    q, kp, vp, own, kw = _make(dev, torch.bfloat16, 5, 6, 3, 64, 333, lens)
    ln = torch.tensor(lens, dtype=torch.int32, device=dev)
    want = attention_shared_prefix(q, kp, vp, *kw["kv"], ln)
    both = torch.stack([kp, vp], 0).permute(2, 1, 0, 3).contiguous()     # [P, H_kv, 2, D]
    kview, vview = both[:, :, 0].transpose(0, 1), both[:, :, 1].transpose(0, 1)
    assert torch.equal(attention_shared_prefix(q, kview, vview, *kw["kv"], ln), want)
    wide = torch.zeros(5, 6, 72, device=dev, dtype=q.dtype)
    wide[..., :64] = q
    odd = torch.zeros(5, 6, 67, device=dev, dtype=q.dtype)
    odd[..., 3:] = q
    outs = torch.zeros(5, 6, 80, device=dev, dtype=q.dtype)
    attention_shared_prefix(wide[..., :64], kp, vp, *kw["kv"], ln, out=outs[..., 7:71])
    assert torch.equal(outs[..., 7:71], want) and (outs[..., :7] == 0).all() and (outs[..., 71:] == 0).all()
    assert torch.equal(attention_shared_prefix(odd[..., 3:], kp, vp, *kw["kv"], ln), want)
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        got = attention_shared_prefix(q, kp, vp, *kw["kv"], ln)
    torch.cuda.current_stream(dev).wait_stream(s)
    assert torch.equal(got, want)
    with pytest.raises(ValueError):
        attention_shared_prefix(q, kp, vp, *kw["kv"], ln, prefix_len=334)
    with pytest.raises(TypeError):
        attention_shared_prefix(q, kp.half(), vp.half(), *kw["kv"], ln)
    with pytest.raises(ValueError):
        attention_shared_prefix(q, torch.zeros(3, 10, 65, device=dev, dtype=q.dtype)[..., 1:],
                                torch.zeros(3, 10, 65, device=dev, dtype=q.dtype)[..., 1:], *kw["kv"], ln)


@pytest.mark.gpu
def test_two_graphs_and_eager_calls_share_nothing(dev):
    """Two captured calls of different sizes, replayed in turn with eager calls between."""
    import torch

    from detkernels_b200 import _lib
    cases = []
    for R, P, seed in ((3, 600, 1), (40, 2100, 2)):
        lens = [int(x) for x in np.random.default_rng(seed).integers(0, 900, size=R)]
        q, kp, vp, own, kw = _make(dev, torch.bfloat16, R, 8, 4, 64, P, lens, seed=seed)
        ln = torch.tensor(lens, dtype=torch.int32, device=dev)
        want = _call(q, kw, ln)
        g = torch.cuda.CUDAGraph()
        with _lib.graph_capture(g):
            out = _call(q, kw, ln)
        cases.append((g, out, want, q, kw, ln))
    for _ in range(3):
        for g, out, want, q, kw, ln in cases:
            out.zero_()
            g.replay()
            assert torch.equal(_call(q, kw, ln), want)
            assert torch.equal(out, want)


@pytest.mark.gpu
def test_a_prefix_block_outside_the_pool_is_reported(dev):
    import torch

    from detkernels_b200 import _lib
    q, kp, vp, own, kw = _make(dev, torch.bfloat16, 2, 2, 1, 64, 100, [3, 4], 64)
    for bad in (-1, kw["kv"][0].shape[0]):
        kw["kwargs"]["prefix_blocks"][1] = bad
        _call(q, kw, [3, 4])
        assert _lib.device_status(dev.index) == (_lib.DK_ERR_DEVICE_CHECK, 0x62a)


@pytest.mark.gpu
def test_lengths_beyond_the_announced_maximum_are_reported(dev):
    import torch

    from detkernels_b200 import _lib
    q, kp, vp, own, kw = _make(dev, torch.bfloat16, 2, 2, 1, 64, 100, [3, 64])
    _call(q, kw, [3, 65], max_kv_len=64)
    assert _lib.device_status(dev.index) == (_lib.DK_ERR_DEVICE_CHECK, 0x210)


@pytest.mark.gpu
@pytest.mark.parametrize("D,page", [(64, 64), (128, 128)])
def test_a_decode_step_of_plan_norm_and_attention(dev, D, page):
    """Three steps of a small batch as a server runs them: the plan opens pages, the norm stores rotated keys
    at its slots, attention reads the shared prefix and each request's pages; against f64 from the same caches."""
    import torch

    from detkernels_b200.kernels.attention import attention_shared_prefix
    from detkernels_b200.kernels.paging import paged_plan
    from detkernels_b200.kernels.rope import qk_norm_rope, qk_norm_rope_reference, rope_table
    H, Hkv, P, B = 8, 2, 300, 5
    g = torch.Generator(device=dev).manual_seed(D)
    dt = torch.bfloat16

    def randn(*s):
        return torch.randn(*s, device=dev, generator=g).to(dt)
    n_pre = -(-P // page)
    kc, vc = (torch.full((n_pre + 20, Hkv, page, D), float("nan"), device=dev, dtype=dt) for _ in range(2))
    order = torch.randperm(n_pre + 20, device=dev, generator=g).to(torch.int32)
    pre, free = order[:n_pre].contiguous(), order[n_pre:].contiguous()
    kp, vp = randn(Hkv, P, D), randn(Hkv, P, D)
    for t in range(P):
        kc[pre[t // page], :, t % page], vc[pre[t // page], :, t % page] = kp[:, t], vp[:, t]
    table = torch.zeros(B, 4, dtype=torch.int32, device=dev)
    cursor = torch.zeros(1, dtype=torch.int32, device=dev)
    kv = torch.zeros(B, dtype=torch.int32, device=dev)
    rope = rope_table(1024, D, device=dev)
    qw, kw = (1 + 0.1 * randn(D).float()).to(dt), (1 + 0.1 * randn(D).float()).to(dt)
    hist_k, hist_v = [[] for _ in range(B)], [[] for _ in range(B)]
    for new in ([3, 70, 1, 20, 64], [1] * 5, [1] * 5):
        n = sum(new)
        qkv = randn(n, (H + 2 * Hkv) * D)
        q = qkv[:, :H * D].view(n, H, D)
        k = qkv[:, H * D:(H + Hkv) * D].view(n, Hkv, D)
        v = qkv[:, (H + Hkv) * D:].view(n, Hkv, D)
        nw = torch.tensor(new, dtype=torch.int32, device=dev)
        rpt = 16 // (H // Hkv)
        plan = paged_plan(table, kv, nw, page, free_blocks=free, cursor=cursor, n_rows=n, rows_per_tile=rpt,
                          n_tiles=sum(-(-x // rpt) for x in new))
        cursor = plan.cursor
        qr, _ = qk_norm_rope(q, k, plan.row_pos + P, qw, kw, rope, v=v, k_cache=kc, v_cache=vc, slots=plan.slots)
        out = attention_shared_prefix(qr, kc, vc, kc, vc, plan.q_lens, prefix_len=P, prefix_blocks=pre,
                                      block_table=table, row_tiles=plan.row_tiles)
        kv = kv + nw
        _, k_ref = qk_norm_rope_reference(q, k, plan.row_pos + P, qw, kw, rope)
        at, rows_k, rows_v, some = 0, [], [], []
        for b, m in enumerate(new):
            # the cache's own bits are attention's input; they are the reference's up to one step of the type
            for i in range(m):
                s = int(plan.slots[at + i])
                kk = kc[s // page, :, s % page]
                assert ((kk.float() - k_ref[at + i].float()).abs() <= 2.0 ** -7 * k_ref[at + i].float().abs() + 1e-6).all()
                hist_k[b].append(kk)
                hist_v[b].append(v[at + i])
            some.append(at + m - 1)
            rows_k.append(torch.stack(hist_k[b], 1))
            rows_v.append(torch.stack(hist_v[b], 1))
            at += m
        _tol_check(out[some], qr[some], kp, vp, rows_k, rows_v, D ** -0.5)
    assert math.isfinite(float(out.float().sum()))


def _step_state(dev, B, H, Hkv, D, P, page, seed):
    import torch

    from detkernels_b200.kernels.rope import rope_table
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, device=dev, generator=g).to(torch.bfloat16)
    n_pre = -(-P // page)
    st = dict(kc=randn(n_pre + 4 * B, Hkv, page, D), vc=randn(n_pre + 4 * B, Hkv, page, D), qkv=randn(B, (H + 2 * Hkv) * D),
              qw=randn(D), kw=randn(D), rope=rope_table(2048, D, device=dev), kv=torch.full((B,), 60, dtype=torch.int32, device=dev),
              nw=torch.ones(B, dtype=torch.int32, device=dev), cursor=torch.full((1,), B, dtype=torch.int32, device=dev))
    order = torch.randperm(n_pre + 4 * B, device=dev, generator=g).to(torch.int32)
    st["pre"], st["free"] = order[:n_pre].contiguous(), order[n_pre:].contiguous()
    st["table"] = torch.zeros(B, 4, dtype=torch.int32, device=dev)
    st["table"][:, 0] = st["free"][:B]     # 60 tokens each
    return st


def _step(st, H, Hkv, D, P, page, out=None):
    """One decode step in place: plan, norm into the cache, attention, lengths."""
    from detkernels_b200.kernels.attention import attention_shared_prefix
    from detkernels_b200.kernels.paging import paged_plan
    from detkernels_b200.kernels.rope import qk_norm_rope
    B = st["qkv"].shape[0]
    q, k, v = (x.view(B, -1, D) for x in st["qkv"].split([H * D, Hkv * D, Hkv * D], 1))
    plan = paged_plan(st["table"], st["kv"], st["nw"], page, free_blocks=st["free"], cursor=st["cursor"], n_rows=B, out=out)
    if plan.cursor is not st["cursor"]:
        st["cursor"].copy_(plan.cursor)
    qr, _ = qk_norm_rope(q, k, plan.row_pos, st["qw"], st["kw"], st["rope"], v=v, k_cache=st["kc"], v_cache=st["vc"],
                         slots=plan.slots)
    o = attention_shared_prefix(qr, st["kc"], st["vc"], st["kc"], st["vc"], plan.q_lens, prefix_len=P,
                                prefix_blocks=st["pre"], block_table=st["table"])
    st["kv"] += st["nw"]
    return o, plan


@pytest.mark.gpu
def test_a_captured_step_replays_as_eager_steps(dev):
    """A whole step captured once, its plan in the tensors of an earlier call, replayed over a page's end."""
    import torch

    from detkernels_b200 import _lib
    dims = (8, 4, 64, 130, 64)
    a, b = (_step_state(dev, 6, *dims, seed=5) for _ in range(2))
    o, plan = _step(a, *dims)
    plan = plan._replace(cursor=a["cursor"])
    want, _ = _step(b, *dims)
    assert torch.equal(o, want)
    g = torch.cuda.CUDAGraph()
    keep = {k: v.clone() for k, v in a.items()}
    with _lib.graph_capture(g):
        o, _ = _step(a, *dims, out=plan)
    for k, v in keep.items():
        assert torch.equal(a[k], v), k            # a capture runs nothing
    for _ in range(9):
        g.replay()
        want, _ = _step(b, *dims)
        assert torch.equal(o, want)
        for k in ("table", "cursor", "kv", "kc", "vc"):
            assert torch.equal(a[k], b[k]), k
    assert int(a["cursor"]) == 12 and int(a["kv"][0]) == 70


@pytest.mark.gpu
def test_steps_on_two_streams_at_once(dev):
    """Two servers' steps side by side on two streams, against the same steps one after the other."""
    import torch
    dims = [(8, 4, 64, 130, 64), (16, 2, 128, 1500, 128)]
    make = lambda: [_step_state(dev, n, *d, seed=s) for s, (n, d) in enumerate(zip((6, 90), dims))]
    alone, both = make(), make()
    want = [[_step(st, *d)[0] for _ in range(20)] for st, d in zip(alone, dims)]
    torch.cuda.synchronize(dev)
    streams = [torch.cuda.Stream(device=dev) for _ in dims]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_step(both[i], *dims[i])[0])
    torch.cuda.synchronize(dev)
    for w, g in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(w, g))
