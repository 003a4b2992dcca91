"""Head norm with rotation: against the definition in 64 bits, through strides, caches and refusals."""
import numpy as np
import pytest


def _exact(x, w, pos, table, inter, eps):
    """(value, magnitude) of norm + rotation in f64; magnitude = |a cos| + |b sin| bounds what f32 can lose."""
    import torch
    x, w = x.double(), w.double()
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
    rd = table.shape[1]
    cs = table[pos.long()].double()[:, None, :]
    c, s = cs[..., :rd // 2], cs[..., rd // 2:]
    r = y[..., :rd]
    a, b = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., :rd // 2], r[..., rd // 2:])
    val, mag = (a * c - b * s, a * s + b * c), ((a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs())
    def join(p):
        return torch.stack(p, -1).flatten(-2) if inter else torch.cat(p, -1)
    return torch.cat([join(val), y[..., rd:]], -1), torch.cat([join(mag), y[..., rd:].abs()], -1)


def _close(got, x, w, pos, table, inter, eps=1e-6):
    """One rounding of the result, and the f32 steps before it: a sum of squares of at most 32 terms a
    lane and 5 joins (its relative error halved by the root), then mean, eps, root, two products and the
    rotation's two: 28 units of 2^-24 of the terms' magnitude."""
    import torch
    want, mag = _exact(x, w, pos, table, inter, eps)
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + 28 * 2.0 ** -24 * mag
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25       # half a step of the subnormals
    bad = (got.double() - want).abs() - tol * 1.0001
    assert bad.max().item() <= 0, bad.max().item()


def _inputs(dev, dt, T, H, Hkv, D, rd, max_pos=700, seed=0, wdt=None):
    import torch

    from detkernels_b200.kernels.rope import rope_table
    g = torch.Generator(device=dev).manual_seed(seed)
    qkv = torch.randn(T, (H + 2 * Hkv) * D, device=dev, generator=g).to(dt)
    q = qkv[:, :H * D].view(T, H, D)
    k = qkv[:, H * D:(H + Hkv) * D].view(T, Hkv, D)
    v = qkv[:, (H + Hkv) * D:].view(T, Hkv, D)
    w = [(1 + 0.2 * torch.randn(D, device=dev, generator=g)).to(wdt or dt) for _ in range(2)]
    pos = torch.randint(0, max_pos, (T,), device=dev, generator=g)
    return q, k, v, w[0], w[1], pos, rope_table(max_pos, rd, device=dev)


def _dt(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def test_table_holds_far_angles():
    """Angles of far positions come from 64-bit products (a 32-bit product loses whole radians there)."""
    from detkernels_b200.kernels.rope import rope_table
    t = rope_table(1 << 20, 8, theta=10000.0)
    p = (1 << 20) - 1
    for i in range(4):
        a = p * 10000.0 ** (-2 * i / 8)
        assert abs(float(t[p, i]) - np.cos(a)) < 1e-6 and abs(float(t[p, 4 + i]) - np.sin(a)) < 1e-6
    with pytest.raises(ValueError):
        rope_table(4, 7)
    with pytest.raises(ValueError):
        rope_table(0, 8)


def test_reference_matches_the_definition():
    import torch

    from detkernels_b200.kernels.rope import qk_norm_rope_reference
    for inter in (False, True):
        q, k, _, qw, kw, pos, table = _inputs("cpu", torch.float32, 9, 4, 2, 16, 8)
        got = qk_norm_rope_reference(q, k, pos, qw, kw, table, interleaved=inter)
        _close(got[0], q, qw, pos, table, inter)
        _close(got[1], k, kw, pos, table, inter)


def test_refusals_on_the_host():
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.rope import qk_norm_rope
    q, k, _, qw, kw, pos, table = _inputs("cpu", torch.float32, 3, 2, 1, 16, 8)
    with pytest.raises(AssertionError):
        qk_norm_rope(q, k, pos, qw, kw, table)
    lib = _lib.load()

    def call(dtype=_lib.DK_BF16, D=64, rd=64, k_out=16, cache=None, slots=None, v=None, slabs=1, cap=1, H=2, wd=0):
        return lib.dk_qk_norm_rope(16, 1, 1, 16, 1, 1, v, 1, 1, 16, 1, 1, k_out, 1, 1, cache, cache, 1, 1, 1, slabs, cap,
                                   slots, 16, 0, 16, 16, wd, 16, 8, 4, H, 1, D, rd, 0, 1e-6, dtype, None)
    assert call(dtype=9) == _lib.DK_ERR_UNSUPPORTED and call(wd=5) == _lib.DK_ERR_UNSUPPORTED
    assert call(D=513) == _lib.DK_ERR_UNSUPPORTED
    assert call(rd=63) == _lib.DK_ERR_INVALID_ARGUMENT and call(rd=66) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(k_out=None) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(cache=16) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(cache=16, slots=16, v=16, slabs=0) == _lib.DK_ERR_INVALID_ARGUMENT
    assert call(H=70000) == _lib.DK_ERR_INVALID_ARGUMENT


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,rd,inter", [(64, 64, False), (128, 128, False), (128, 64, False), (128, 128, True),
                                        (32, 32, False), (80, 80, False), (96, 48, True), (96, 64, False),
                                        (256, 256, False), (256, 64, False), (50, 20, True), (33, 32, False),
                                        (512, 512, False), (8, 2, True)])
def test_against_the_definition(dev, dt, D, rd, inter):
    from detkernels_b200.kernels.rope import qk_norm_rope
    for T, H, Hkv in ((1, 1, 1), (5, 6, 2), (67, 16, 4)):
        q, k, _, qw, kw, pos, table = _inputs(dev, _dt(dt), T, H, Hkv, D, rd, seed=T)
        qo, ko = qk_norm_rope(q, k, pos, qw, kw, table, interleaved=inter)
        _close(qo, q, qw, pos, table, inter)
        _close(ko, k, kw, pos, table, inter)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,wdt", [("bf16", "f32"), ("f16", "bf16"), ("f32", "f16")])
def test_weight_types_and_int32_positions(dev, dt, wdt):
    import torch

    from detkernels_b200.kernels.rope import qk_norm_rope
    q, k, _, qw, kw, pos, table = _inputs(dev, _dt(dt), 31, 8, 2, 64, 64, wdt=_dt(wdt))
    qo, ko = qk_norm_rope(q, k, pos.to(torch.int32), qw, kw, table)
    _close(qo, q, qw, pos, table, False)
    _close(ko, k, kw, pos, table, False)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 37, 2500])
@pytest.mark.parametrize("D,dt,paged", [(64, "bf16", True), (128, "f16", False), (96, "bf16", True), (36, "f32", False)])
def test_keys_and_values_reach_their_slots(dev, T, D, dt, paged):
    """Rows go to scattered slots; every other cache element, and rows of negative slots, stay."""
    import torch

    from detkernels_b200.kernels.rope import qk_norm_rope
    H, Hkv = 6, 3
    q, k, v, qw, kw, pos, table = _inputs(dev, _dt(dt), T, H, Hkv, D, D - D % 4)
    n, cap = (-(-T // 64) + 3, 64) if paged else (3, T)
    g = torch.Generator(device=dev).manual_seed(5)
    kc, vc = (torch.randn(n, Hkv, cap, D, device=dev, generator=g).to(q.dtype) for _ in range(2))
    k0, v0 = kc.clone(), vc.clone()
    slots = torch.randperm(n * cap, device=dev, generator=g)[:T]
    if T > 2:
        slots[1] = -1
    qo, ko = qk_norm_rope(q, k, pos, qw, kw, table, v=v, k_cache=kc, v_cache=vc, slots=slots)
    assert ko is None
    _close(qo, q, qw, pos, table, False)
    ids = slots[slots >= 0]
    rows = torch.nonzero(slots >= 0)[:, 0]
    _close(kc[ids // cap, :, ids % cap], k[rows], kw, pos[rows], table, False)
    assert torch.equal(vc[ids // cap, :, ids % cap], v[rows])
    rest = torch.ones(n * cap, dtype=torch.bool, device=dev)
    rest[ids] = False
    rest = torch.nonzero(rest)[:, 0]
    assert torch.equal(kc[rest // cap, :, rest % cap], k0[rest // cap, :, rest % cap])
    assert torch.equal(vc[rest // cap, :, rest % cap], v0[rest // cap, :, rest % cap])
    # with k_out as well: the same bits in both places
    ko = torch.empty_like(k, memory_format=torch.contiguous_format)
    qk_norm_rope(q, k, pos, qw, kw, table, v=v, k_cache=k0, v_cache=v0, slots=slots, k_out=ko)
    assert torch.equal(k0, kc) and torch.equal(ko[rows], kc[ids // cap, :, ids % cap])


@pytest.mark.gpu
def test_in_place_and_odd_strides_give_the_same_bits(dev):
    import torch

    from detkernels_b200.kernels.rope import qk_norm_rope
    for D, rd in ((64, 64), (48, 20)):
        q, k, _, qw, kw, pos, table = _inputs(dev, torch.bfloat16, 40, 4, 2, D, rd)
        want = qk_norm_rope(q, k, pos, qw, kw, table)
        pad = torch.zeros(40, 4, D + 8, device=dev, dtype=q.dtype)
        pad[..., :D] = q
        kt = k.transpose(0, 1).contiguous().transpose(0, 1)      # head-major
        got = qk_norm_rope(pad[..., :D], kt, pos, qw, kw, table)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        nonunit = q.transpose(1, 2).contiguous().transpose(1, 2)
        got = qk_norm_rope(nonunit, k, pos, qw, kw, table)
        assert torch.equal(got[0], want[0])
        qi, ki = q.clone(), k.clone()
        qk_norm_rope(qi, ki, pos, qw, kw, table, q_out=qi, k_out=ki)
        assert torch.equal(qi, want[0]) and torch.equal(ki, want[1])


@pytest.mark.gpu
def test_a_row_does_not_depend_on_its_batch(dev):
    import torch

    from detkernels_b200.kernels.rope import qk_norm_rope
    q, k, _, qw, kw, pos, table = _inputs(dev, torch.bfloat16, 5000, 16, 8, 64, 64)
    want = qk_norm_rope(q, k, pos, qw, kw, table)
    for lo, hi in ((0, 1), (4999, 5000), (17, 90), (0, 2400)):
        got = qk_norm_rope(q[lo:hi], k[lo:hi], pos[lo:hi], qw, kw, table)
        assert torch.equal(got[0], want[0][lo:hi]) and torch.equal(got[1], want[1][lo:hi])


@pytest.mark.gpu
def test_zero_rows_and_large_values(dev):
    """A zero vector stays zero (eps keeps the root finite); values whose squares leave 16 bits do not overflow."""
    import torch

    from detkernels_b200.kernels.rope import qk_norm_rope
    q, k, _, qw, kw, pos, table = _inputs(dev, torch.float16, 4, 2, 1, 64, 64)
    q, k = q.clone(), k.clone()
    q[0] = 0
    q[1] = 60000.0
    k[2] = 6e-8
    qo, ko = qk_norm_rope(q, k, pos, qw, kw, table)
    assert (qo[0] == 0).all()
    _close(qo, q, qw, pos, table, False)
    _close(ko, k, kw, pos, table, False)
    empty = qk_norm_rope(q[:0], k[:0], pos[:0], qw, kw, table)
    assert empty[0].shape == (0, 2, 64) and empty[1].shape == (0, 1, 64)


@pytest.mark.gpu
def test_positions_and_slots_outside_are_reported_and_skipped(dev):
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.rope import qk_norm_rope
    for D in (64, 36):
        q, k, v, qw, kw, pos, table = _inputs(dev, torch.bfloat16, 4, 2, 1, D, 32)
        kc, vc = (torch.full((2, 1, 4, D), 3.0, device=dev, dtype=q.dtype) for _ in range(2))
        for bad_pos in (-1, table.shape[0]):
            p2 = pos.clone()
            p2[1] = bad_pos
            qo = torch.full((4, 2, D), 9.0, device=dev, dtype=q.dtype)
            qk_norm_rope(q, k, p2, qw, kw, table, v=v, k_cache=kc, v_cache=vc,
                         slots=torch.tensor([0, 1, 2, 7], device=dev), q_out=qo)
            assert _lib.device_status(dev.index) == (_lib.DK_ERR_DEVICE_CHECK, 0x610)
            assert (qo[1] == 9.0).all() and (kc[0, :, 1] == 3.0).all() and not (qo[0] == 9.0).all()
        vc.fill_(3.0)
        qk_norm_rope(q, k, pos, qw, kw, table, v=v, k_cache=kc, v_cache=vc,
                     slots=torch.tensor([0, 8, 2 ** 40, 3], device=dev))
        assert _lib.device_status(dev.index) == (_lib.DK_ERR_DEVICE_CHECK, 0x611)
        assert torch.equal(vc[0, :, 3], v[3]) and (vc[0, :, 1:3] == 3.0).all() and (vc[1] == 3.0).all()


@pytest.mark.gpu
def test_wrapper_refusals(dev):
    import torch

    from detkernels_b200.kernels.rope import qk_norm_rope
    q, k, v, qw, kw, pos, table = _inputs(dev, torch.bfloat16, 4, 2, 1, 64, 64)
    with pytest.raises(TypeError):
        qk_norm_rope(q, k.half(), pos, qw, kw, table)
    with pytest.raises(ValueError):
        qk_norm_rope(q, k, pos, qw, kw, table, v=v)
    with pytest.raises(ValueError):
        qk_norm_rope(q[..., :32], k[..., :32], pos, qw[:32], kw[:32], table)
    with pytest.raises(AssertionError):
        qk_norm_rope(q, k, pos.float(), qw, kw, table)
    with pytest.raises(AssertionError):
        qk_norm_rope(q, k, pos, qw[:32], kw, table)
    with pytest.raises(NotImplementedError):
        big = torch.zeros(1, 1, 520, device=dev, dtype=q.dtype)
        qk_norm_rope(big, big, pos[:1], big[0, 0], big[0, 0], table)
