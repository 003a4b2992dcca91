"""Log probabilities of given tokens, entropy and alternatives: against 64 bits, bitwise invariance, refusals."""
import math

import pytest

DTYPES = ["bf16", "f16", "f32"]


def _dt(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def _check(x, tokens, k, got):
    """Against f64.  u = 2^-24 is half a step of f32.  A logit's distance d from the maximum is a difference and a product
    with a constant that is off by less than u / 2: 2.5 u |d|; its exponential is off by that and 4 u (2^-22, the
    instruction).  Sums of 32 a chain of a thread, five, seven and seven joins of threads, warps and parts, three
    roundings each: less than 100 u of the sum of magnitudes.  So S is off by (104 + 2.5 E|d|) u relatively, T by the
    same of its terms' magnitudes E|d| and by 2.5 E d^2, each with its share of the roundings of the last step (a
    logarithm of 2 u, products and differences)."""
    import torch
    u = 2.0 ** -24
    x64 = x.double()
    lp = torch.log_softmax(x64, -1)
    p = lp.exp()
    d = torch.where(p == 0, 0.0, (x64 - x64.amax(-1, keepdim=True)).abs())
    ed, ed2 = (p * d).sum(-1), (p * d * d).sum(-1)
    logs = -lp.amax(-1)                                     # log S with the maximum as the reference
    ts = u * (104 + 3 * ed + 4 * logs)
    plain = torch.isfinite(lp).any(-1) & ~torch.isnan(lp).any(-1)
    if tokens is not None:
        want = lp.gather(-1, tokens.clamp(min=0)[:, None])[:, 0]
        dist = (x64.gather(-1, tokens.clamp(min=0)[:, None])[:, 0] - x64.amax(-1)).abs()
        want = torch.where(tokens == -1, 0.0, want)
        tol = ts + u * (4 * dist + 4 * want.abs())
        same = (got.logprobs.double() == want) | (got.logprobs.isnan() & want.isnan())
        assert bool((same | ((got.logprobs.double() - want).abs() <= tol)).all()), (got.logprobs, want)
    if got.entropy is not None:
        ent = -torch.where(p == 0, 0.0, p * lp).sum(-1)
        tol = ts + u * (220 * ed + 3 * ed2 + 3 * ed * ed + 4 * ent.abs())
        same = got.entropy.isnan() & ~plain
        assert bool((same | ((got.entropy.double() - ent).abs() <= tol)).all()), (got.entropy, ent)
    if k:
        ids = torch.sort(x.float() + 0.0, dim=-1, descending=True, stable=True).indices[:, :k]
        assert got.top_ids.dtype == torch.int64 and torch.equal(got.top_ids, ids)
        want = lp.gather(-1, ids)
        dist = (x64.gather(-1, ids) - x64.amax(-1, keepdim=True)).abs()
        tol = ts[:, None] + u * (4 * dist + 4 * want.abs())
        same = (got.top_logprobs.double() == want) | (got.top_logprobs.isnan() & want.isnan())
        assert bool((same | ((got.top_logprobs.double() - want).abs() <= tol)).all())


def test_reference_form():
    import torch

    from detkernels_b200.kernels.logprobs import token_logprobs_reference
    x = torch.tensor([[0.0, -0.0, 1.0, -math.inf]])
    r = token_logprobs_reference(x, torch.tensor([2]), top_k=3)
    z = math.log(2 + math.e)
    assert r.logprobs.item() == pytest.approx(1 - z, abs=1e-6)
    assert r.entropy.item() == pytest.approx(z - math.e / (2 + math.e), abs=1e-6)
    assert r.top_ids.tolist() == [[2, 0, 1]]
    assert token_logprobs_reference(x, torch.tensor([-1])).logprobs.item() == 0


def test_entry_point_refuses_on_the_host():
    from detkernels_b200 import _lib
    lib = _lib.load()

    def call(rows=2, vocab=100, dtype=_lib.DK_BF16, tokens=16, lp=16, ent=16, k=0, ids=16, top=16, x=16):
        return lib.dk_token_logprobs(x, vocab, rows, vocab, dtype, tokens, lp, ent, k, ids, top, None)
    assert call(rows=0) == _lib.DK_OK
    assert call(dtype=9) == _lib.DK_ERR_UNSUPPORTED
    assert call(rows=-1) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(vocab=0) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(k=101) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(k=33) == _lib.DK_ERR_UNSUPPORTED and "32" in _lib.last_error()
    assert call(lp=None) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(k=3, ids=None) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(x=17) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(rows=2 ** 31, vocab=32) == _lib.DK_ERR_INVALID_ARGUMENT


def test_wrapper_refuses():
    import torch

    from detkernels_b200.kernels.logprobs import token_logprobs
    with pytest.raises(AssertionError):
        token_logprobs(torch.zeros(2, 8))


@pytest.mark.gpu
def test_wrapper_refuses_on_the_gpu(dev):
    import torch

    from detkernels_b200.kernels.logprobs import token_logprobs
    x = torch.zeros(2, 40, device=dev)
    with pytest.raises(ValueError):
        token_logprobs(x, top_k=41)
    with pytest.raises(ValueError):
        token_logprobs(x, top_k=-1)
    with pytest.raises(NotImplementedError):
        token_logprobs(x, top_k=33)
    with pytest.raises(NotImplementedError):
        token_logprobs(x.double())
    with pytest.raises(AssertionError):
        token_logprobs(x, torch.zeros(3, dtype=torch.int64, device=dev))
    with pytest.raises(AssertionError):
        token_logprobs(x, torch.zeros(2, dtype=torch.int32, device=dev))
    r = token_logprobs(x[:0], torch.zeros(0, dtype=torch.int64, device=dev), top_k=3)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 3)
    assert token_logprobs(x, entropy=False) == (None, None, None, None)


SHAPES = [(1, 1, 1), (3, 7, 7), (2, 31, 31), (2, 33, 32), (4, 255, 20), (3, 257, 5), (2, 500, 32), (2, 600, 32), (3, 2049, 20),
          (5, 5000, 32), (2, 16384, 5), (2, 16385, 5), (3, 50001, 20), (1, 131072, 32), (2, 131073, 1), (1, 300001, 32),
          (301, 1003, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("R,V,k", SHAPES)
def test_against_64_bits(dev, dt, R, V, k):
    import torch

    from detkernels_b200.kernels.logprobs import token_logprobs
    g = torch.Generator(device=dev).manual_seed(V)
    x = (torch.randn(R, V, device=dev, generator=g) * 4).to(_dt(dt))
    tok = torch.randint(0, V, (R,), device=dev, generator=g)
    tok[0] = V - 1
    if R > 1:
        tok[1] = -1
    _check(x, tok, k, token_logprobs(x, tok, top_k=k))
    _check(x, tok, 0, token_logprobs(x, tok, entropy=False))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("kind", ["equal", "zeros", "sorted", "reversed", "allowed", "one", "peaked", "columns", "far", "all_masked",
                                  "nan", "nans", "inf", "lowest", "all_lowest", "huge"])
@pytest.mark.parametrize("V", [700, 16384, 40000])
def test_rows_that_go_wrong(dev, dt, kind, V):
    """Ties, bounds that say nothing, excluded and non-finite logits."""
    import torch

    from detkernels_b200.kernels.logprobs import token_logprobs
    g = torch.Generator(device=dev).manual_seed(1)
    k = 32
    x = torch.randn(3, V, device=dev, generator=g)
    if kind == "equal":
        x[:] = 1.5
    elif kind == "zeros":
        x = torch.where(x > 0, 0.0, -0.0)
    elif kind in ("sorted", "reversed"):
        x = torch.sort(x, dim=1, descending=kind == "sorted").values
    elif kind == "allowed":      # three tokens a row may be taken
        keep = torch.randint(0, V, (3, 3), device=dev, generator=g)
        x = torch.full_like(x, -math.inf).scatter(1, keep, x[:, :3])
    elif kind == "one":
        x[:] = -math.inf
        x[:, V - 1] = -3.0
    elif kind == "peaked":
        x[:, 77] = 40.0
    elif kind == "columns":      # the largest logits all belong to 31 of the 256 threads
        x[:, (torch.arange(V, device=dev) // 8) % 256 < 31] += 20
    elif kind == "far":          # f16 ends at 65504
        x = x * 8 + 6e4
    elif kind == "all_masked":
        x[:] = -math.inf
    elif kind == "nan":
        x[:, V // 2] = math.nan
    elif kind == "nans":
        x[:, ::3] = math.nan
    elif kind == "inf":
        x[:, 5] = math.inf
    elif kind == "lowest":
        x[:, ::2] = torch.finfo(_dt(dt)).min
    elif kind == "all_lowest":   # a row that an additive mask has left nothing of is uniform
        x[:] = torch.finfo(_dt(dt)).min
    elif kind == "huge":
        x = torch.where(x > 1, torch.finfo(_dt(dt)).max / 2, torch.where(x < -1, torch.finfo(_dt(dt)).min / 2, x))
    x = x.to(_dt(dt))
    tok = torch.tensor([0, 77, V - 1], device=dev)
    _check(x, tok, k, token_logprobs(x, tok, top_k=k))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("kind", ["crests", "plateau", "stairs"])
@pytest.mark.parametrize("k", [1, 5, 32])
def test_a_later_pass_is_far_above(dev, dt, kind, k):
    """Many rows, a CTA each, whose later passes lie all above the alternatives so far: as many larger maxima as there are
    alternatives and no more, equal ones, and ever larger ones."""
    import torch

    from detkernels_b200.kernels.logprobs import token_logprobs
    V = 5 * 4096 + 100 if dt == "f32" else 5 * 8192 + 100
    at = torch.arange(V, device=dev)
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.rand(200, V, device=dev, generator=g)
    x[:, V // 2:] = 2.0
    if kind == "crests":
        x[:, V - 90 * 8::8] = 10.0 + (torch.arange(90, device=dev) * 37 % 90).float()
    elif kind == "plateau":
        x[:, V // 2 + 9::11] = 7.0
    else:
        x[:] = (at * 16 // V).float()
    x = x.to(_dt(dt))
    tok = torch.randint(0, V, (200,), device=dev, generator=g)
    _check(x, tok, k, token_logprobs(x, tok, top_k=k))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V", [37, 999, 20011, 140000])
def test_a_row_is_itself_wherever_it_lies(dev, dt, V):
    """Bit for bit: alone, in a batch, at every alignment, behind a row stride, with more dimensions."""
    import torch

    from detkernels_b200.kernels.logprobs import token_logprobs
    g = torch.Generator(device=dev).manual_seed(2)
    k = 9
    row = (torch.randn(V, device=dev, generator=g) * 3).to(_dt(dt))
    tok = torch.tensor([V // 3], device=dev)
    want = token_logprobs(row[None], tok, top_k=k)

    def same(got, at=0):
        for a, b in zip(want, got):
            assert torch.equal(a[0], b[at])
    for off in range(9):
        buf = torch.full((2, V + off + 3), 100.0, device=dev).to(_dt(dt))    # what lies around a row does not reach it
        buf[1, off:off + V] = row
        same(token_logprobs(buf[:, off:off + V], tok.expand(2), top_k=k), 1)
    batch = torch.randn(70, V, device=dev, generator=g).to(_dt(dt))
    batch[63] = row
    same(token_logprobs(batch, tok.expand(70), top_k=k), 63)
    got = token_logprobs(batch.view(7, 10, V), tok.expand(7, 10), top_k=k)
    assert got.top_ids.shape == (7, 10, k) and got.entropy.shape == (7, 10)
    same([t.flatten(0, 1) for t in got], 63)
    same(token_logprobs(batch.t().contiguous().t(), tok.expand(70), top_k=k), 63)
    one = token_logprobs(row, tok[0], top_k=k)
    assert one.logprobs.shape == () and torch.equal(one.logprobs, want.logprobs[0])


@pytest.mark.gpu
def test_bad_token_sets_the_status(dev):
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.logprobs import token_logprobs
    x = torch.zeros(3, 16, device=dev)
    r = token_logprobs(x, torch.tensor([16, 3, -2], device=dev))
    assert r.logprobs.isnan().tolist() == [True, False, True]
    code, detail = _lib.device_status(dev.index)
    assert code == _lib.DK_ERR_DEVICE_CHECK and detail == 0x650


@pytest.mark.gpu
def test_captured_and_on_another_stream(dev):
    import torch

    from detkernels_b200.kernels.logprobs import token_logprobs
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(9, 33000, device=dev, generator=g).bfloat16()
    tok = torch.randint(0, 33000, (9,), device=dev, generator=g)
    want = token_logprobs(x, tok, top_k=4)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        other = token_logprobs(x, tok, top_k=4)
    torch.cuda.current_stream(dev).wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = token_logprobs(x, tok, top_k=4)
    y = x.clone()
    x.zero_()
    graph.replay()
    assert got.top_ids.tolist() == [[0, 1, 2, 3]] * 9
    x.copy_(y)
    graph.replay()
    for a, b, c in zip(want, got, other):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.gpu
def test_the_pick_is_the_matmuls(dev):
    """The most likely token is the one that the fused greedy step of the LM head takes."""
    import torch

    from detkernels_b200.kernels.logprobs import token_logprobs
    from detkernels_b200.kernels.matmul import argmax_finish, matmul_fused
    g = torch.Generator(device=dev).manual_seed(4)
    a = torch.randn(13, 256, device=dev, generator=g).bfloat16()
    w = (torch.randn(256, 1000, device=dev, generator=g) * 0.02).bfloat16()   # coarse: ties are common
    logits = torch.empty(13, 1000, device=dev, dtype=torch.bfloat16)
    keys = torch.zeros(13, dtype=torch.int64, device=dev)
    matmul_fused(a, w, epilogue="argmax", argmax_keys=keys, out=logits)
    tok = argmax_finish(keys, torch.empty(13, dtype=torch.int64, device=dev))
    assert torch.equal(token_logprobs(logits, top_k=1).top_ids[:, 0], tok)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("V", [40, 700, 40000])
def test_maxima_of_any_size(dev, dt, sign, V):
    """A row a maximum, from 2^20 on: neighbours of the type, so that every rounding of their products with log2 e occurs
    (next to 1.5e9 that of a product is off by up to 128, which is a weight of 2^-128)."""
    import torch

    from detkernels_b200.kernels.logprobs import token_logprobs
    first = [2.0 ** e for e in range(20, 40)] + [1.4885e9, 1.48853e9, 1.4886e9, 2.9e9]
    at = torch.tensor(first, device=dev).to(_dt(dt))
    ints = at.view(torch.int16 if dt == "bf16" else torch.int32)
    m = torch.cat([(ints + i).view(_dt(dt)) for i in range(24)]).float() * sign
    g = torch.Generator(device=dev).manual_seed(V)
    # the maximum, its neighbours below, and logits far away
    x = torch.where(m[:, None] > 0, 0.0, m[:, None] * 2).expand(-1, V).clone()
    near = torch.rand(len(m), V, device=dev, generator=g) < 0.3
    step = 2.0 ** (-8 if dt == "bf16" else -23)
    below = m[:, None] * (1 - sign * step * torch.randint(0, 3, x.shape, device=dev, generator=g))
    x = torch.where(near, below, x)
    x[:, V // 3] = m
    x = x.to(_dt(dt))
    tok = torch.full((len(m),), V // 3, device=dev)
    _check(x, tok, 5, token_logprobs(x, tok, top_k=5))
    y = x[:, V // 3:V // 3 + 1].expand(-1, V).contiguous()      # nothing but the maximum
    _check(y, tok, 5, token_logprobs(y, tok, top_k=5))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("R", [3, 200])
@pytest.mark.parametrize("passes", [(0,), (1,), (0, 1, 3), (2, 3)])
def test_fewer_threads_than_alternatives_hold_the_largest(dev, dt, R, passes):
    """All logits of 31 threads of a warp above all others, with 32 alternatives: the most that a bound from the threads'
    maxima lets through, alone, behind alternatives of an earlier pass, and pass after pass ever larger ones.  Few rows
    are split, many are not."""
    import torch

    from detkernels_b200.kernels.logprobs import token_logprobs
    t = _dt(dt)
    vec = 16 // torch.empty(0, dtype=t).element_size()   # logits a thread takes side by side; a warp 128 times as many a pass
    span = 8 * 128 * vec                                 # a pass
    V = 4 * span + 77
    g = torch.Generator(device=dev).manual_seed(R)
    x = torch.randn(R, V, device=dev, generator=g).to(t)
    at = torch.arange(span, device=dev) // vec
    bits = torch.int32 if dt == "f32" else torch.int16
    for n, j in enumerate(passes):
        for warp in (0, 5) if R == 3 else (5,):
            hot = j * span + torch.nonzero((at // 128 == warp) & (at % 32 < 31))[:, 0]
            # neighbours of the type from 8 (and then 2048) on, in any order: no two alike
            base = torch.tensor(8.0 if n == 0 else 2048.0, device=dev).to(t).view(bits)
            order = torch.randperm(len(hot), device=dev, generator=g)
            x[:, hot] = (base + order.to(bits)).view(t) if n < 2 else x[:, hot] + 100
    tok = torch.randint(0, V, (R,), device=dev, generator=g)
    _check(x, tok, 32, token_logprobs(x, tok, top_k=32))
