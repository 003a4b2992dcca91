"""Attention of drafted tokens: against the definition in 64 bits, bitwise invariance, masks and values that go wrong,
refusals, and a verification step of all operators together."""
import math

import numpy as np
import pytest


def _dt(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16}[name]


def _i32(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype=np.int32))).to(dev)


def _masks(rng, sizes, words, kind):
    """int64 [rows, words]: trees, chains, any set, or nothing."""
    rows = []
    for n in sizes:
        seen = []
        for i in range(n):
            if kind == "tree":
                up = int(rng.integers(max(0, i - 6), i)) if i else -1
                bits = (seen[up] if up >= 0 else 0) | 1 << i
            elif kind == "chain":
                bits = (1 << (i + 1)) - 1
            elif kind == "any":
                bits = int.from_bytes(rng.bytes(8 * words), "little")      # its own and later drafts, or neither
            else:
                bits = 0
            seen.append(bits)
            rows.append([(bits >> (64 * w)) & (2 ** 64 - 1) for w in range(words)])
    return np.array(rows, dtype=np.uint64).reshape(len(rows), words).view(np.int64)


def _case(dev, dt, sizes, kvs, H, Hkv, D, page=0, words=1, kind="tree", seed=0, fill=float("nan"), scale_q=1.0):
    """q, caches (what no row may see is `fill`), masks and keyword arguments; and each sequence's keys and values."""
    import torch
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)

    def randn(*s):
        return torch.randn(*s, device=dev, generator=g).to(dt)
    B, R = len(sizes), sum(sizes)
    q = (randn(R, H, D).float() * scale_q).to(dt)
    total = [a + b for a, b in zip(kvs, sizes)]
    own = [(randn(Hkv, n, D), randn(Hkv, n, D)) for n in total]
    kw = {}
    if page:
        need = [-(-n // page) for n in total]
        order = rng.permutation(sum(need) + 2)
        table = np.full((B, max(need + [1]) + 1), -1)
        caches = [torch.full((sum(need) + 2, Hkv, page, D), fill, device=dev, dtype=dt) for _ in range(2)]
        at = 0
        for b in range(B):
            table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
            for j in range(need[b]):
                n = min(page, total[b] - j * page)
                for c in range(2):
                    caches[c][int(table[b, j]), :, :n] = own[b][c][:, j * page:j * page + n]
        kw["block_table"] = _i32(table, dev)
    else:
        cap = -(-max(total + [1]) // 8) * 8 + 8
        caches = [torch.full((B, Hkv, cap, D), fill, device=dev, dtype=dt) for _ in range(2)]
        for b in range(B):
            for c in range(2):
                caches[c][b, :, :total[b]] = own[b][c]
    mask = torch.from_numpy(_masks(rng, sizes, words, kind)).to(dev) if R else torch.zeros(0, words, dtype=torch.int64, device=dev)
    args = (q, caches[0], caches[1], _i32(kvs, dev), _i32(np.concatenate([[0], np.cumsum(sizes)]), dev), mask)
    return args, kw, own


def _sees(mask_row, kv, t):
    bits = np.unpackbits(mask_row.view(np.uint8), bitorder="little")[:t].astype(bool)
    bits = np.concatenate([bits, np.zeros(t - len(bits), bool)])
    return np.concatenate([np.ones(kv, bool), bits])


def _check(got, args, own, scale, D):
    """Row by row against f64.  With A = sum p |v| / sum p and half a step h = eps / 2 of the type: the rounded weights move
    the result by at most h A, a score's f32 dot product of D terms is off by at most D 2^-24 sum |q k| scale =: E, which
    moves weights and their sum by E each, the f32 sums of the tokens of a chunk and the joins by 2 (n + 64) 2^-24 A, and
    the store rounds once.  Weights below f16's normal range are off by up to 2^-25 each, which counts for the largest |v|."""
    import torch
    q, _, _, kv, cu, mask = args
    eps = torch.finfo(got.dtype).eps
    kv, cu, bits = kv.tolist(), cu.tolist(), mask.cpu().numpy()
    G = q.shape[1] // own[0][0].shape[0]
    for b in range(len(kv)):
        t = cu[b + 1] - cu[b]
        if not t:
            continue
        k, v = (x.double().repeat_interleave(G, 0) for x in own[b])
        for r in range(cu[b], cu[b + 1]):
            sees = torch.from_numpy(_sees(bits[r], kv[b], t)).to(q.device)
            if not bool(sees.any()):
                assert not got[r].any(), r
                continue
            ks, vs = k[:, sees], v[:, sees]
            qr = q[r].double()[:, None]
            s = (qr @ ks.transpose(1, 2))[:, 0] * scale
            E = (qr.abs() @ ks.abs().transpose(1, 2)).amax() * abs(scale) * D * 2.0 ** -24
            p = torch.softmax(s, -1)
            want = (p[:, None] @ vs)[:, 0]
            A = (p[:, None] @ vs.abs())[:, 0]
            tol = eps / 2 * want.abs() + A * (eps / 2 + 2 * E + 2 * (ks.shape[1] + 64) * 2.0 ** -24)
            if got.dtype == torch.float16:
                tol = tol + 2.0 ** -25 + vs.abs().amax() * ks.shape[1] * 2.0 ** -25 / max(1.0, (p / p.amax(-1, keepdim=True)).sum(-1).min().item())
            bad = ((got[r].double() - want).abs() - tol).max().item()
            assert bad <= 0, (b, r, bad)


def test_reference_form():
    import torch

    from detkernels_b200.kernels.attention import attention_reference, attention_tree_reference
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(*s, generator=g) for s in ((3, 4, 8), (2, 2, 6, 8), (2, 2, 6, 8)))
    mask = torch.tensor([[1], [2], [0]])
    out = attention_tree_reference(q, k, v, [3, 0], [0, 2, 3], mask)
    want = attention_reference(q[:1], k[:1, :, :4], v[:1, :, :4])
    assert torch.allclose(out[:1], want, atol=1e-6) and not out[2].any()
    sel = [0, 1, 2, 4]
    assert torch.allclose(out[1:2], attention_reference(q[1:2], k[:1, :, sel], v[:1, :, sel]), atol=1e-6)


def test_entry_point_refuses_on_the_host():
    from detkernels_b200 import _lib
    lib = _lib.load()
    bad = _lib.DK_ERR_INVALID_ARGUMENT

    def call(rows=8, seqs=2, H=8, Hkv=4, D=64, words=1, max_rows=8, max_kv=700, dtype=_lib.DK_BF16, table=None, stride=4, page=64,
             n_seq=2, cap=1024, q=16, mask=16, q_sr=512, ws=0):
        return lib.dk_attention_tree(q, q_sr, 64, 16, 16, 65536, 16384, 64, n_seq, cap, table, stride, 4, 9, page, 16, 512, 64,
                                     16, 16, mask, words, words, seqs, rows, max_rows, H, Hkv, D, max_kv, 0.1, dtype, 16,
                                     ws, None)
    assert call(rows=0) == _lib.DK_OK and call(seqs=0) == _lib.DK_OK
    assert call(dtype=_lib.DK_F32) == _lib.DK_ERR_UNSUPPORTED and call(D=96) == _lib.DK_ERR_UNSUPPORTED
    assert call(H=7) == bad and call(Hkv=0) == bad and call(rows=-1) == bad and call(H=129, Hkv=1) == _lib.DK_ERR_UNSUPPORTED
    assert call(words=0) == bad and call(max_rows=0) == bad and call(max_kv=0) == bad
    assert call(q=8) == bad and call(q_sr=511) == bad and call(mask=None) == bad and call(n_seq=1) == bad and call(cap=0) == bad
    assert call(table=16, page=48) == bad and call(table=16, stride=3) == bad
    assert call(max_kv=1000, ws=100) == _lib.DK_ERR_WORKSPACE
    size = lib.dk_attention_tree_workspace_size
    assert size(2, 8, 8, 8, 4, 64, 768) == 0 and size(2, 8, 8, 8, 4, 64, 769) >= 2 * 64 * 66 * 4
    assert size(200, 200, 1, 8, 4, 64, 100) >= 4 * (4 + 4 * 200)      # more items than SMs: their order
    # a chunk's number never exceeds what the workspace was sized for
    for D in (64, 128):
        for kv in (0, 511, 768, 2049, 4096, 4097, 8192, 8193, 9000, 16384, 16385, 20000, 32768, 32769, 70001, 1000003):
            for t in (1, 64, 700, 5000):
                chunk = (768 if kv <= 4096 else 1024 if kv <= 8192 else 1536 if kv <= 16384 else 2048 if kv <= 32768 else
                         -(-(-(-kv // 16)) // 128) * 128)
                n = -(-(kv + t) // chunk)
                assert n == 1 or size(1, t, t, 1, 1, D, kv + t) >= t * n * (D + 2) * 4, (D, kv, t)
                assert n == 1 or size(1, 2 * t, 2 * t, 1, 1, D, 2 * (kv + t)) >= 2 * t * n * (D + 2) * 4, (D, kv, t)


def test_wrapper_refuses_cpu_tensors():
    import torch

    from detkernels_b200.kernels.attention import attention_tree
    q, c, i = torch.zeros(2, 2, 64), torch.zeros(1, 2, 64, 64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(AssertionError):
        attention_tree(q, c, c, i[:1], i, torch.zeros(2, 1, dtype=torch.int64))


CASES = [
    # sizes, kvs, H, Hkv, D, page, words, kind
    ([1], [0], 1, 1, 64, 0, 1, "tree"),
    ([3], [5], 2, 1, 64, 0, 1, "tree"),
    ([1, 7, 0, 33, 64], [0, 63, 9, 64, 500], 8, 8, 64, 0, 1, "tree"),
    ([5, 12, 30], [510, 1, 2047], 8, 2, 128, 64, 1, "tree"),
    ([17, 1, 64], [129, 700, 1], 6, 3, 32, 128, 1, "tree"),
    ([64, 20], [1500, 2100], 16, 2, 128, 64, 1, "tree"),        # several tiles of rows
    ([64, 33, 2], [100, 3000, 40], 32, 4, 64, 256, 1, "any"),
    ([130, 70, 200], [600, 0, 1000], 4, 2, 64, 0, 4, "tree"),     # more drafts than a word
    ([100, 90], [64, 130], 3, 1, 128, 64, 1, "any"),            # more drafts than the words hold
    ([10, 10], [0, 0], 4, 4, 64, 0, 1, "none"),                 # rows that see nothing
    ([10, 40], [0, 3], 4, 4, 128, 0, 1, "none"),
    ([600], [0], 2, 1, 64, 0, 10, "chain"),                     # a prompt
    ([9, 9, 9], [17000, 5000, 9000], 8, 4, 128, 64, 1, "tree"),   # chunks that grow with the length
    ([4], [40000], 2, 2, 64, 0, 1, "tree"),
    ([2], [50], 128, 1, 64, 0, 1, "tree"),                      # as many heads a KV head as a tile has rows
    ([16] * 40, [int(x) for x in np.arange(40) * 37], 4, 1, 64, 64, 1, "tree"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=range(len(CASES)))
def test_against_64_bits(dev, dt, case):
    from detkernels_b200.kernels.attention import attention_tree
    sizes, kvs, H, Hkv, D, page, words, kind = case
    args, kw, own = _case(dev, _dt(dt), sizes, kvs, H, Hkv, D, page, words, kind, seed=len(sizes) + D)
    got = attention_tree(*args, max_rows=max(sizes), **kw)
    _check(got, args, own, D ** -0.5, D)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.3, 0.0, 4.0])
def test_scales(dev, scale):
    import torch

    from detkernels_b200.kernels.attention import attention_tree
    args, kw, own = _case(dev, torch.float16, [9, 20], [700, 30], 8, 2, 64, 64)
    _check(attention_tree(*args, scale=scale, **kw), args, own, scale, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [0, 64])
def test_a_row_is_itself_in_any_batch(dev, D, page):
    """Bit for bit: alone or in a batch, whatever the bounds, beside other drafts, paged or not, strided or not."""
    import torch

    from detkernels_b200.kernels.attention import attention_tree
    sizes, kvs = [5, 64, 20, 33], [530, 900, 2500, 0]
    args, kw, own = _case(dev, torch.bfloat16, sizes, kvs, 16, 4, D, page, fill=0.5)
    want = attention_tree(*args, **kw)
    q, kc, vc, kv, cu, mask = args
    assert torch.equal(want, attention_tree(*args, max_rows=64, max_kv_len=2600, **kw))
    for b in range(4):
        r0, r1 = int(cu[b]), int(cu[b + 1])
        sub = dict(block_table=kw["block_table"][b:b + 1]) if page else {}
        cs = (kc, vc) if page else (kc[b:b + 1], vc[b:b + 1])
        one = attention_tree(q[r0:r1], *cs, kv[b:b + 1], cu[b:b + 2] - r0, mask[r0:r1], **sub)
        assert torch.equal(one, want[r0:r1]), b
        # a row whose mask lies behind the others': the same bits with fewer rows, where it sees the same tokens
        few = max(1, (r1 - r0) // 2)
        some = attention_tree(q[r0:r0 + few], *cs, kv[b:b + 1], _i32([0, few], dev), mask[r0:r0 + few], **sub)
        assert torch.equal(some, want[r0:r0 + few]), b
    # other masks and other queries around it change nothing for row 7 of sequence 1
    r = int(cu[1]) + 7
    m2, q2 = torch.randint(-2 ** 62, 2 ** 62, mask.shape, device=dev), torch.randn_like(q)
    m2[r], q2[r] = mask[r], q[r]
    assert torch.equal(attention_tree(q2, kc, vc, kv, cu, m2, **kw)[r], want[r])
    # strides: q and out inside wider tensors, masks with a row stride, caches [.., token, head, D] in memory
    wide = torch.zeros(q.shape[0], 16, 3 * D, device=dev, dtype=q.dtype)
    wide[..., D:2 * D] = q
    out = torch.zeros(q.shape[0], 18, D + 1, device=dev, dtype=q.dtype)[:, 1:17, :D]
    mw = torch.full((q.shape[0], 3), -1, device=dev)
    mw[:, 1:2] = mask
    turned = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kc, vc)]
    got = attention_tree(wide[..., D:2 * D], *turned, kv, cu, mw[:, 1:2], out=out, **kw)
    assert got is out and torch.equal(out, want)
    odd = torch.zeros(q.shape[0], 16, D + 1, device=dev, dtype=q.dtype)[..., :D]      # rows off 16 bytes are copied
    odd.copy_(q)
    assert torch.equal(attention_tree(odd, kc, vc, kv, cu, mask, **kw), want)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Hkv,G", [(3, 4), (2, 8), (1, 5)])
def test_many_items_a_cta(dev, D, Hkv, G):
    """Several items a CTA, of one tile and of two, of one KV head and of two, of one block and of many: the same bits each time
    and alone, and right."""
    import torch

    from detkernels_b200.kernels.attention import attention_tree
    rng = np.random.default_rng(D + Hkv)
    B = 130
    sizes = [int(x) for x in rng.choice([1, 3, 16, 20, 33, 40, 64, 0], size=B)]
    kvs = [int(x) for x in rng.choice([0, 5, 64, 300, 511, 900, 2100, 3000], size=B)]
    args, kw, own = _case(dev, torch.bfloat16, sizes, kvs, Hkv * G, Hkv, D, 64, seed=B)
    q, kc, vc, kv, cu, mask = args
    want = attention_tree(*args, **kw)
    for _ in range(8):
        assert torch.equal(attention_tree(*args, **kw), want)
    ends = cu.tolist()
    for b in range(0, B, 9):
        r0, r1 = ends[b], ends[b + 1]
        if r0 == r1:
            continue
        sub = (q[r0:r1], kc, vc, kv[b:b + 1], _i32([0, r1 - r0], dev), mask[r0:r1])
        one = attention_tree(*sub, block_table=kw["block_table"][b:b + 1])
        assert torch.equal(one, want[r0:r1]), b
        _check(one, sub, own[b:b + 1], D ** -0.5, D)


@pytest.mark.gpu
@pytest.mark.parametrize("D,long", [(128, 270000), (32, 9000)])
def test_an_order_of_many_sequences(dev, D, long):
    """More sequences than the order's threads, and a chunk that costs more than it tells apart."""
    import torch

    from detkernels_b200.kernels.attention import attention_tree
    rng = np.random.default_rng(D)
    B = 700
    sizes = [int(x) for x in rng.choice([1, 4, 0, 70], size=B)]
    kvs = [int(x) for x in rng.choice([0, 3, 64, 800, 1700], size=B)]
    sizes[333], kvs[333] = 6, long
    args, kw, own = _case(dev, torch.float16, sizes, kvs, 2, 1, D, 64, words=2, seed=D)
    q, kc, vc, kv, cu, mask = args
    want = attention_tree(*args, **kw)
    assert torch.equal(attention_tree(*args, **kw), want)
    ends = cu.tolist()
    for b in list(range(0, B, 37)) + [333]:
        r0, r1 = ends[b], ends[b + 1]
        if r0 == r1:
            continue
        sub = (q[r0:r1], kc, vc, kv[b:b + 1], _i32([0, r1 - r0], dev), mask[r0:r1])
        one = attention_tree(*sub, block_table=kw["block_table"][b:b + 1])
        assert torch.equal(one, want[r0:r1]), b
        _check(one, sub, own[b:b + 1], D ** -0.5, D)


@pytest.mark.gpu
def test_a_chain_is_decode_attention(dev):
    """Drafts that each see all before them are a causal continuation: the rows of attention_decode, up to rounding."""
    import torch

    from detkernels_b200.kernels.attention import attention_decode, attention_tree
    args, kw, own = _case(dev, torch.bfloat16, [8, 8], [300, 77], 8, 2, 64, 64, kind="chain")
    q, kc, vc, kv, cu, mask = args
    got = attention_tree(*args, **kw)
    seq = torch.arange(2, device=dev).repeat_interleave(8)
    lens = (kv[seq] + torch.arange(8, device=dev).repeat(2) + 1).int()
    want = attention_decode(q, kc, vc, lens, block_table=kw["block_table"][seq].contiguous())
    assert (got.float() - want.float()).abs().max().item() <= 2.0 ** -6
    # a chain of one row a sequence, for every length around a block, a chunk and a page
    for n in (1, 2, 63, 64, 65, 127, 128, 129, 511, 512, 513, 767, 768, 769, 1535, 1536, 1537):
        args, kw, own = _case(dev, torch.float16, [1], [n - 1], 4, 2, 128, 64, seed=n)
        _check(attention_tree(*args, **kw), args, own, 128 ** -0.5, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("kv,t,G", [(0, 40, 1), (61, 40, 8), (500, 64, 2), (700, 30, 4)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_drafts_that_are_not_finite(dev, D, kv, t, G, bad):
    """A draft with non-finite keys or values changes the rows that see it, as the definition says, and no other row."""
    import torch

    from detkernels_b200.kernels.attention import attention_tree
    H = 3 * G
    args, kw, own = _case(dev, torch.bfloat16, [t, 5], [kv, 9], H, 3, D, 64, kind="tree", seed=kv + t)
    q, kc, vc, kv_t, cu, mask = args
    clean = attention_tree(*args, **kw)
    j = t // 3
    pos = kv + j
    blk, off = int(kw["block_table"][0, pos // 64]), pos % 64
    sees = (mask[:t, 0] >> j) & 1 == 1
    assert bool(sees.any()) and not bool(sees.all())
    # values: one element of one KV head
    v2 = vc.clone()
    v2[blk, 1, off, 5] = bad
    got = attention_tree(q, kc, v2, kv_t, cu, mask, **kw)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[:t][sees, G:2 * G, 5] = True
    assert torch.equal(got[~hit], clean[~hit])
    assert bool((got[hit].isnan() if math.isnan(bad) else got[hit] == bad).all())
    # keys of a draft that nobody else's mask names: its rows are NaN (or, for a score of -inf, without it), others stay
    k2 = kc.clone()
    k2[blk, :, off] = bad
    got = attention_tree(q, k2, vc, kv_t, cu, mask, **kw)
    assert torch.equal(got[:t][~sees], clean[:t][~sees]) and torch.equal(got[t:], clean[t:])
    assert bool(got[:t][sees].isnan().any())


@pytest.mark.gpu
def test_padded_rows_and_out(dev):
    """Rows behind the last sequence, and sequences without rows, keep what out holds; bounds may be wide."""
    import torch

    from detkernels_b200.kernels.attention import attention_tree
    args, kw, own = _case(dev, torch.float16, [4, 0, 30], [600, 77, 5], 4, 2, 64, 64)
    q, kc, vc, kv, cu, mask = args
    want = attention_tree(*args, **kw)
    q2, m2 = torch.cat([q, q[:7]]), torch.cat([mask, mask[:7]])
    out = torch.full_like(q2, 7.0)
    got = attention_tree(q2, kc, vc, kv, cu, m2, out=out, max_rows=1000, max_kv_len=10 ** 9, **kw)
    assert torch.equal(got[:34], want) and bool((got[34:] == 7).all())
    assert attention_tree(q[:0], kc, vc, kv, cu, mask[:0], **kw).shape == (0, 4, 64)
    out.fill_(3.0)
    zero = torch.zeros_like(cu)
    assert bool((attention_tree(q2, kc, vc, kv, zero, m2, out=out, **kw) == 3).all())


@pytest.mark.gpu
@pytest.mark.parametrize("page", [0, 64])
@pytest.mark.parametrize("D,kvs", [(64, [100, 0, 200]), (128, [900, 2000, 5]), (32, [70, 1600, 300])])
def test_layouts(dev, D, kvs, page):
    """Queries inside a fused projection, caches by tokens, outputs inside a wider tensor, aligned and not, masks inside one."""
    import torch

    from detkernels_b200.kernels.attention import attention_tree
    H, Hkv = 6, 2
    args, kw, own = _case(dev, torch.float16, [5, 40, 2], kvs, H, Hkv, D, page, fill=0.5)
    q, kc, vc, kv, cu, mask = args
    want = attention_tree(*args, **kw)
    R = q.shape[0]
    for pad, off in ((2 * Hkv * D, 0), (24, 8), (5, 1)):
        wide = torch.full((R, H * D + pad), 9.0, device=dev, dtype=q.dtype)
        q2 = wide[:, off:off + H * D].view(R, H, D)
        q2.copy_(q)
        out_wide = torch.full((R, H * D + pad), 3.0, device=dev, dtype=q.dtype)
        out = out_wide[:, off:off + H * D].view(R, H, D)
        assert attention_tree(q2, kc, vc, kv, cu, mask, out=out, **kw) is out
        assert torch.equal(out, want)
        assert bool((out_wide[:, :off] == 3).all()) and bool((out_wide[:, off + H * D:] == 3).all())
    k2, v2 = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kc, vc))
    assert torch.equal(attention_tree(q, k2, v2, kv, cu, mask, **kw), want)
    both = torch.stack([kc, vc], dim=2)     # K and V of a head side by side
    assert torch.equal(attention_tree(q, both[:, :, 0], both[:, :, 1], kv, cu, mask, **kw), want)
    m2 = torch.full((R, 3), -1, device=dev, dtype=torch.int64)
    m2[:, 1:2] = mask
    assert torch.equal(attention_tree(q, kc, vc, kv, cu, m2[:, 1:2], **kw), want)
    if page:
        t2 = torch.full((3, kw["block_table"].shape[1] + 5), -1, device=dev, dtype=torch.int32)
        t2[:, 2:-3] = kw["block_table"]
        assert torch.equal(attention_tree(q, kc, vc, kv, cu, mask, block_table=t2[:, 2:-3]), want)


@pytest.mark.gpu
@pytest.mark.parametrize("kvs", [[100, 0, 200], [900, 2000, 5]])
def test_broadcast_inputs(dev, kvs):
    """Queries, caches and masks that take one place in memory for several rows, heads or sequences; out in q's place."""
    import torch

    from detkernels_b200.kernels.attention import attention_tree
    args, kw, own = _case(dev, torch.bfloat16, [5, 5, 5], kvs, 8, 2, 64, fill=0.5)
    q, kc, vc, kv, cu, mask = args

    def same(q, kc, vc, mask):
        want = attention_tree(q.contiguous(), kc.contiguous(), vc.contiguous(), kv, cu, mask.contiguous(), **kw)
        assert torch.equal(attention_tree(q, kc, vc, kv, cu, mask, **kw), want)
    same(q[:1].expand_as(q), kc, vc, mask)
    same(q[:, :1].expand_as(q), kc, vc, mask)
    same(q, kc[:1].expand_as(kc), vc[:1].expand_as(vc), mask)
    same(q, kc[:, :1].expand_as(kc), vc[:, :1].expand_as(vc), mask)
    same(q, kc, vc, mask[:1].expand_as(mask))
    want, out = attention_tree(*args, **kw), q.clone()
    assert attention_tree(out, kc, vc, kv, cu, mask, out=out, **kw) is out and torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["cu_past", "cu_descends", "cu_negative", "rows", "kv_negative", "kv_long", "block"])
def test_bad_extents_set_the_status(dev, what):
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.attention import attention_tree
    args, kw, own = _case(dev, torch.float16, [4, 6, 5], [600, 77, 1030], 4, 2, 64, 64, fill=1.0)
    q, kc, vc, kv, cu, mask = args
    want = attention_tree(*args, **kw)
    kv, cu, bt, keep, detail = kv.clone(), cu.clone(), kw["block_table"].clone(), [1], 0x67d
    max_rows = None
    if what == "cu_past":
        cu[3], keep = 16, [2]
    elif what == "cu_descends":
        cu[2], keep = 2, [1, 2]      # sequence 2 then has more rows than its bound
        max_rows = 6
    elif what == "cu_negative":
        cu[0], keep = -1, [0]
    elif what == "rows":
        max_rows, keep = 5, [1]
    elif what == "kv_negative":
        kv[1] = -1
    elif what == "kv_long":
        kv[1] = 64 * bt.shape[1] - 5
    elif what == "block":
        bt[1, 0], keep, detail = kc.shape[0], [], 0x67a
    out = torch.full_like(q, 9.0)
    got = attention_tree(q, kc, vc, kv, cu, mask, out=out, max_rows=max_rows, block_table=bt)
    code, det = _lib.device_status(dev.index)
    assert code == _lib.DK_ERR_DEVICE_CHECK and det == detail, (code, hex(det))
    rows = [(0, 4), (4, 10), (10, 15)]
    for b, (a, z) in enumerate(rows):
        if b in keep:
            assert bool((got[a:z] == 9).all())
        elif detail == 0x67d:
            assert torch.equal(got[a:z], want[a:z])


@pytest.mark.gpu
def test_wrapper_refuses_on_the_gpu(dev):
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.attention import attention_tree
    args, kw, own = _case(dev, torch.float16, [4, 6], [900, 77], 4, 2, 64, 64)
    q, kc, vc, kv, cu, mask = args
    with pytest.raises(TypeError):
        attention_tree(q.bfloat16(), kc, vc, kv, cu, mask, **kw)
    with pytest.raises(NotImplementedError):
        attention_tree(q.float(), kc.float(), vc.float(), kv, cu, mask, **kw)
    with pytest.raises(AssertionError):
        attention_tree(q, kc, vc, kv, cu[:-1], mask, **kw)
    with pytest.raises(AssertionError):
        attention_tree(q, kc, vc, kv, cu, mask.int(), **kw)
    with pytest.raises(AssertionError):
        attention_tree(q, kc, vc, kv, cu, mask[:-1], **kw)
    with pytest.raises(ValueError):
        attention_tree(q, kc, vc, kv, cu, mask, max_rows=-1, **kw)
    with pytest.raises(ValueError):      # pages of 32
        attention_tree(q, kc[:, :, :32], vc[:, :, :32], kv, cu, mask, block_table=kw["block_table"].repeat(1, 2))
    with pytest.raises(_lib.DetKernelsError):
        attention_tree(q, kc, vc, kv, cu, mask, workspace=torch.zeros(16, dtype=torch.uint8, device=dev), **kw)
    with pytest.raises(ValueError):      # keys off 16 bytes
        odd = torch.zeros(*kc.shape[:3], 65, device=dev, dtype=kc.dtype)[..., 1:]
        attention_tree(q, odd, odd, kv, cu, mask, **kw)


@pytest.mark.gpu
def test_streams_and_graphs(dev):
    import torch

    from detkernels_b200.kernels.attention import attention_tree
    args, kw, own = _case(dev, torch.bfloat16, [30, 20, 64], [900, 2000, 60], 8, 2, 128, 64, fill=0.0)
    other, kw2, _ = _case(dev, torch.bfloat16, [30, 20, 64], [900, 2000, 60], 8, 2, 128, 64, fill=0.0, seed=5)
    want, want2 = attention_tree(*args, **kw), attention_tree(*other, **kw2)
    a, b = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    for s in (a, b):
        s.wait_stream(torch.cuda.current_stream(dev))
    graphs = []
    for s, (x, k) in ((a, (args, kw)), (b, (other, kw2))):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = attention_tree(*x, **k)
        graphs.append((g, y))
    for _ in range(5):      # both at once
        for s, (g, _) in zip((a, b), graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize(dev)
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want2)
    # a captured call serves other lengths and trees
    args[3].copy_(_i32([800, 1990, 20], dev))
    args[4].copy_(_i32([0, 10, 30, 90], dev))
    with torch.cuda.stream(a):
        graphs[0][0].replay()
    torch.cuda.synchronize(dev)
    assert torch.equal(graphs[0][1][:90], attention_tree(*args, **kw)[:90])


@pytest.mark.gpu
def test_offsets_beyond_32_bits(dev):
    """A pool whose last blocks lie more than 2^32 bytes and 2^31 elements from its start."""
    import torch

    from detkernels_b200.kernels.attention import attention_tree
    args, kw, own = _case(dev, torch.bfloat16, [5, 3], [100, 64], 4, 2, 128, 64, fill=0.0)
    want = attention_tree(*args, **kw)
    n = 2 ** 31 // (2 * 64 * 128) + 8
    big = [torch.empty(n, 2, 64, 128, device=dev, dtype=torch.bfloat16) for _ in range(2)]
    bt = kw["block_table"]
    moved = torch.where(bt >= 0, bt + n - args[1].shape[0], bt)
    for x, y in zip(big, args[1:3]):
        x[n - y.shape[0]:] = y
    assert torch.equal(attention_tree(args[0], *big, *args[3:], block_table=moved.int()), want)


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_a_verification_step(dev, captured):
    """Plan, rotation into the cache, attention, logits, picks, accepted paths and compaction, as a server runs them, against
    the same steps on the host; the next step's plan takes the pages that came back."""
    import torch

    from detkernels_b200.kernels.attention import attention_tree
    from detkernels_b200.kernels.drafts import tree_accept, tree_accept_reference, tree_mask
    from detkernels_b200.kernels.logprobs import token_logprobs
    from detkernels_b200.kernels.paging import paged_compact, paged_fork, paged_plan
    from detkernels_b200.kernels.rope import qk_norm_rope, rope_table
    g = torch.Generator(device=dev).manual_seed(7)
    rng = np.random.default_rng(7)
    B, H, Hkv, D, V, page, n_blocks, width, top = 5, 8, 2, 64, 50, 64, 60, 8, 6

    def randn(*s):
        return torch.randn(*s, device=dev, generator=g).bfloat16()
    pools = [randn(n_blocks, Hkv, page, D) for _ in range(2)]
    free = torch.from_numpy(rng.permutation(np.arange(1, n_blocks)).astype(np.int32)).to(dev)
    cursor, table = _i32([0], dev), torch.zeros(B, width, dtype=torch.int32, device=dev)
    shares = torch.zeros(n_blocks, dtype=torch.int32, device=dev)
    kv = torch.zeros(B, dtype=torch.int32, device=dev)
    lens0 = [130, 64, 1, 200]
    # prompts of four requests; the fifth is another sample of the first
    plan = paged_plan(table, kv[:4].contiguous(), _i32(lens0, dev), page, free_blocks=free, cursor=cursor)
    kv[:4] = _i32(lens0, dev)
    cursor = paged_fork(table, kv, _i32([0], dev), _i32([4], dev), page, free_blocks=free, cursor=plan.cursor, pools=pools,
                        shares=shares)
    assert kv.tolist() == lens0 + [130] and int(shares.sum()) == 2
    sizes = [9, 1, 20, 62, 7]
    parents = np.concatenate([[-1] + [int(rng.integers(max(0, i - 3), i)) for i in range(1, n)] for n in sizes]).astype(np.int32)
    cu = np.concatenate([[0], np.cumsum(sizes)])
    depth = np.zeros(len(parents), int)
    for b in range(B):
        for i in range(1, sizes[b]):
            depth[cu[b] + i] = depth[cu[b] + parents[cu[b] + i]] + 1
    R = len(parents)
    q, k, v, head, ones = randn(R, H, D), randn(R, Hkv, D), randn(R, Hkv, D), randn(H * D, V), torch.ones(D, device=dev).bfloat16()
    tokens = torch.from_numpy(rng.integers(0, V, size=R)).to(dev)
    angles = rope_table(1000, D, device=dev)
    par, new = torch.from_numpy(parents).to(dev), _i32(sizes, dev)
    deep = torch.from_numpy(depth.astype(np.int32)).to(dev)

    def step():
        plan = paged_plan(table, kv, new, page, free_blocks=free, cursor=cursor, n_rows=R)
        pos = (kv[plan.row_seq.long()] + deep).int()
        qr, _ = qk_norm_rope(q, k, pos, ones, ones, angles, v=v, k_cache=pools[0], v_cache=pools[1], slots=plan.slots)
        mask = tree_mask(par, plan.cu_rows)
        o = attention_tree(qr, pools[0], pools[1], kv, plan.cu_rows, mask, block_table=table, max_rows=64, max_kv_len=300)
        logits = o.flatten(1) @ head
        lp = token_logprobs(logits, tokens, top_k=1)
        # here most drafts are what the model picks: a drafter that is often right
        picked = torch.where(agree, want_pick, lp.top_ids[:, 0])
        acc = tree_accept(par, tokens, picked, plan.cu_rows, max_keep=top)
        done = paged_compact(table, kv, new, acc.n_keep, page, keep=acc.keep, pools=pools, free_blocks=free, cursor=plan.cursor,
                             shares=shares)
        return plan, qr, mask, o, lp, picked, acc, done
    agree = torch.zeros(R, dtype=torch.bool, device=dev)
    want_pick = torch.zeros(R, dtype=torch.int64, device=dev)
    for r in range(R):
        if parents[r] >= 0 and rng.random() < 0.8:
            up = cu[np.searchsorted(cu, r, side="right") - 1] + parents[r]
            agree[up], want_pick[up] = True, tokens[r]
    start = [x.clone() for x in (table, free, shares, *pools)]
    if captured:
        keep_state = [x.clone() for x in (table, free, shares, *pools)]
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream(dev).wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step()
        for x, y in zip((table, free, shares, *pools), keep_state):
            x.copy_(y)
        graph.replay()
    else:
        res = step()
    plan, qr, mask, o, lp, picked, acc, done = res
    # attention against 64 bits over the cache as it was
    bt, lens = table.tolist(), kv.tolist()
    before = [x.clone() for x in start[3:]]
    slots = plan.slots.tolist()
    stored = qk_norm_rope(q, k, (kv[plan.row_seq.long()] + deep).int(), ones, ones, angles)[1]
    for r, sl in enumerate(slots):
        before[0][sl // page, :, sl % page] = stored[r]
        before[1][sl // page, :, sl % page] = v[r]
    own = [tuple(torch.cat([x[bt[b][j]] for j in range(-(-(lens[b] + sizes[b]) // page))], 1)[:, :lens[b] + sizes[b]] for x in before)
           for b in range(B)]
    _check(o, (qr, None, None, kv, plan.cu_rows, mask), own, D ** -0.5, D)
    want = tree_accept_reference(parents.tolist(), tokens.tolist(), picked.tolist(), cu.tolist(), max_keep=top)
    assert acc.keep.tolist() == want.keep and acc.n_keep.tolist() == want.n_keep and acc.next_tokens.tolist() == want.next_tokens
    assert max(want.n_keep) > 2
    # the kept tokens lie behind the old ones, and the last pages are free again
    for b in range(B):
        n = lens[b] + want.n_keep[b]
        sel = list(range(lens[b])) + [lens[b] + j for j in want.keep[b][:want.n_keep[b]]]
        for c in range(2):
            now = torch.cat([pools[c][bt[b][j]] for j in range(-(-n // page))], 1)[:, :n]
            assert torch.equal(now, own[b][c][:, sel])
    back = int(plan.cursor) - int(done.cursor)
    given = [bt[b][j] for b in range(B)
             for j in range(-(-int(done.lens[b]) // page), -(-(lens[b] + sizes[b]) // page))]
    assert back == len(given) and free[int(done.cursor):int(done.cursor) + back].tolist() == given
    assert done.lens.tolist() == [a + n for a, n in zip(lens, want.n_keep)]
    # all requests end: every page comes back once, the shared ones with their last holder
    zero = torch.zeros_like(kv)
    end = paged_compact(table, zero, done.lens, zero, page, free_blocks=free, cursor=done.cursor, shares=shares)
    assert end.cursor.tolist() == [0] and sorted(free.tolist()) == list(range(1, n_blocks)) and not shares.any()
