"""Calls at the edges of the serving operators' ranges: bounds larger than a step, refused plans, bad lengths and
tiles, captured and shared scratch, sizes that leave 32 bits."""
import numpy as np
import pytest


def _i32(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype=np.int32))).to(dev)


def _attn_inputs(dev, R, H, Hkv, D, P, cap, n_seq, seed=0, dt=None):
    import torch
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, device=dev, generator=g).to(dt or torch.bfloat16)
    return randn(R, H, D), randn(Hkv, P, D), randn(Hkv, P, D), randn(n_seq, Hkv, cap, D), randn(n_seq, Hkv, cap, D)


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [0, 100])
@pytest.mark.parametrize("tile", [(2 ** 31 - 1, 1, 0), (2 ** 31 - 8, 8, 0), (4, 1, 0), (-1, 1, 0), (0, 1, 3), (0, 9, 0),
                                  (0, -1, 0), (0, -2 ** 31, 0)])
def test_a_tile_outside_the_batch_is_reported_and_skipped(dev, prefix, tile):
    """Rows near 2^31 included, where first row + rows leaves 32 bits; the other tile's rows are as without it."""
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.attention import attention_shared_prefix
    q, kp, vp, k, v = _attn_inputs(dev, 4, 4, 2, 64, 100, 64, 3)
    ln = _i32([5, 6, 7, 8], dev)
    out = torch.full_like(q, 7.0)
    attention_shared_prefix(q, kp, vp, k, v, ln, prefix_len=prefix, row_tiles=_i32([tile, (2, 2, 1)], dev), out=out)
    assert _lib.device_status(dev.index) == (_lib.DK_ERR_DEVICE_CHECK, 0x211)
    want = attention_shared_prefix(q, kp, vp, k, v, ln, prefix_len=prefix, row_tiles=_i32([(2, 2, 1)], dev))
    assert torch.equal(out[2:], want[2:]) and (out[:2] == 7.0).all()


def test_divisions_are_exact_over_all_32_bits(tmp_path):
    """The kernels' division by the heads a group, the page size and the tile rows, compiled for the host: around
    multiples near every power of two (2^28 rows and up among them) and at the ends."""
    import os
    import subprocess
    src = tmp_path / "divide.cpp"
    src.write_text(r"""
#include <initializer_list>
#include <stdio.h>
#include "dk_divide.cuh"
int main() {
  const uint32_t odd[] = {24, 64, 96, 127, 128, 1000, 4097, 65535, 65536, 65537, 1u << 28, (1u << 31) - 1, 1u << 31, 0xffffffffu};
  unsigned long long bad = 0, n = 0;
  for (uint32_t i = 1; i <= 16 + sizeof(odd) / sizeof(odd[0]); ++i) {
    const uint32_t d = i <= 16 ? i : odd[i - 17];
    const dk::Divisor v = dk::divisor(d);
    const dk::Divisor31 w = dk::divisor31(d);
    for (int e = 0; e < 32; ++e)
      for (uint32_t k = 0; k < 64; ++k)
        for (int s = -1; s <= 1; ++s) {
          const uint32_t near = ((1u << e) / d + k) * d + s, at = (1u << e) + k + s, end = 0xffffffffu - k;
          bad += dk::div_by(near, v) != near / d;
          bad += dk::div_by(at, v) != at / d;
          bad += dk::div_by(end, v) != end / d;
          for (uint32_t x : {near & 0x7fffffffu, at & 0x7fffffffu, end & 0x7fffffffu}) bad += dk::div_by(x, w) != x / d;
          bad += dk::ceil_div32(at, v) != at / d + (at % d != 0);
          n += 7;
        }
  }
  printf("%llu wrong of %llu\n", bad, n);
  return bad != 0;
}
""")
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "detkernels_b200", "csrc")
    exe = tmp_path / "divide"
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", csrc, "-o", str(exe), str(src)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout


@pytest.mark.gpu
def test_more_than_2_to_28_rows(dev):
    """One narrow head of 2^28 + 300 rows (17 GB of queries): each row is its own, bit for bit that of a small call."""
    import torch

    from detkernels_b200.kernels.attention import attention_shared_prefix
    if torch.cuda.mem_get_info(dev)[0] < 100 << 30:
        pytest.skip("needs 100 GB of free device memory")
    R = 2 ** 28 + 300
    g = torch.Generator(device=dev).manual_seed(3)
    kp, vp = (torch.randn(1, 70, 32, device=dev, generator=g).to(torch.bfloat16) for _ in range(2))
    some = torch.tensor([0, 1, 255, 2 ** 27, 2 ** 28 - 1, 2 ** 28, 2 ** 28 + 1, 2 ** 28 + 44, R - 1], device=dev)
    q = torch.zeros(R, 1, 32, dtype=torch.bfloat16, device=dev)
    q[some] = torch.randn(len(some), 1, 32, device=dev, generator=g).to(torch.bfloat16)
    k = torch.zeros(1, 1, 64, 32, dtype=torch.bfloat16, device=dev)
    out = attention_shared_prefix(q, kp, vp, k, k, 0)
    assert torch.equal(out[some], attention_shared_prefix(q[some], kp, vp, k, k, 0))
    flat = attention_shared_prefix(q[2:3], kp, vp, k, k, 0)
    assert torch.equal(out[2], flat[0]) and torch.equal(out[2 ** 28 + 2], flat[0])
    del q, out
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,rd,inter", [(96, 48, True), (64, 32, True), (128, 128, True), (128, 64, False), (50, 20, True)])
def test_an_infinite_element_reaches_only_its_own_pair(dev, dt, D, rd, inter):
    """1 / root is 0 then: by the definition the element itself (and, if rotated, its partner) is NaN, everything else
    a zero, which behind the rotated part has the sign of its element times its weight."""
    import torch

    from detkernels_b200.kernels.rope import qk_norm_rope, rope_table
    t = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[dt]
    g = torch.Generator(device=dev).manual_seed(D)
    T = D
    q = torch.randn(T, 2, D, device=dev, generator=g).to(t)
    k = torch.randn(T, 1, D, device=dev, generator=g).to(t)
    q[torch.arange(T), 0, torch.arange(T)] = float("inf")      # row i: element i of head 0
    w = torch.randn(D, device=dev, generator=g).to(t)
    pos = torch.arange(1, T + 1, device=dev)
    qo, _ = qk_norm_rope(q, k, pos, w, w, rope_table(T + 2, rd, device=dev), interleaved=inter)
    want = torch.zeros(T, D, dtype=torch.bool, device=dev)
    for i in range(T):
        want[i, i] = True
        if i < rd:
            want[i, i ^ 1 if inter else (i + rd // 2) % rd] = True
    assert torch.equal(torch.isnan(qo[:, 0]), want)
    assert torch.isfinite(qo[:, 1]).all() and (qo[:, 0][~want] == 0).all()
    rest = ~want[:, rd:]
    sign = torch.signbit(q[:, 0, rd:]) ^ torch.signbit(w[rd:])
    assert torch.equal(torch.signbit(qo[:, 0, rd:])[rest], sign[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("R", [24, 3000])
@pytest.mark.parametrize("tiled", [False, True])
@pytest.mark.parametrize("bad", [-1, 641, 2 ** 31 - 1])
def test_rows_of_a_bad_length_are_left(dev, D, R, tiled, bad):
    """Whether several warps share a row (few rows) or one owns it: a length outside the announced maximum is reported,
    its row, or every row of its tile, keeps what out held, and all others are as in a call without it."""
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.attention import attention_shared_prefix
    per = 4 if tiled else 1                      # rows a sequence
    q, kp, vp, k, v = _attn_inputs(dev, R, 4, 2, D, 200, 704, R // per, seed=R)
    rng = np.random.default_rng(R)
    lens = rng.integers(0, 641, size=R)
    kw = dict(max_kv_len=640)
    if tiled:
        kw["row_tiles"] = _i32([(4 * s, 4, s) for s in range(R // 4)], dev)
    want = attention_shared_prefix(q, kp, vp, k, v, _i32(lens, dev), **kw)
    at = [0, 9, R - 1]
    lens[at] = bad
    left = np.zeros(R, bool)
    for r in at:
        left[r // per * per:r // per * per + per] = True
    out = torch.full_like(q, 7.0)
    torch.cuda.synchronize(dev)
    attention_shared_prefix(q, kp, vp, k, v, _i32(lens, dev), out=out, **kw)
    assert _lib.device_status(dev.index) == (_lib.DK_ERR_DEVICE_CHECK, 0x210)
    left = torch.from_numpy(left).to(dev)
    assert (out[left] == 7.0).all() and torch.equal(out[~left], want[~left])


@pytest.mark.gpu
@pytest.mark.parametrize("n_seq", [3, 900])
@pytest.mark.parametrize("prefix", [0, 100])
def test_tiles_of_no_rows_are_padding(dev, n_seq, prefix):
    """Tiles of 0 rows, whatever else they hold, between and behind the others: nothing is reported, the covered rows'
    bits are those of a list without them and the rest of out stays."""
    import torch

    from detkernels_b200.kernels.attention import attention_shared_prefix
    R = 4 * n_seq + 5
    q, kp, vp, k, v = _attn_inputs(dev, R, 4, 2, 64, 100, 640, n_seq)
    rng = np.random.default_rng(n_seq)
    ln = _i32(rng.integers(0, 641, size=R), dev)
    tiles = [(4 * s, 4, s) for s in range(n_seq)]
    padded = [(0, 0, 0), (-1, 0, -5)] + [x for t in tiles for x in (t, (2 ** 31 - 1, 0, 2 ** 31 - 1))] + [(0, 0, 0)] * 7
    outs = []
    for t in (tiles, padded):
        out = torch.full_like(q, 7.0)
        attention_shared_prefix(q, kp, vp, k, v, ln, prefix_len=prefix, row_tiles=_i32(t, dev), out=out)
        outs.append(out)
    assert torch.equal(*outs) and (outs[1][4 * n_seq:] == 7.0).all() and not (outs[1][:4 * n_seq] == 7.0).all(-1).any()


NEUTRAL = dict(row_seq=0, row_pos=0, slots=-1, q_lens=0, row_tiles=0)


def _plan_outputs(dev, B, n_rows, n_tiles, fill):
    """A plan whose tensors hold an earlier step's values."""
    import torch

    from detkernels_b200.kernels.paging import PagedPlan
    full = lambda *s, d=torch.int32: torch.full(s, fill, dtype=d, device=dev)
    return PagedPlan(None, None, None, full(n_rows), full(n_rows), full(n_rows, d=torch.int64), full(n_rows),
                     full(n_tiles, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("B,new_hi,spare", [(1, 1, 3), (7, 5, 1), (40, 30, 700), (40, 300, 9), (2500, 40, 5), (64, 64, 70000)])
def test_entries_behind_a_plan_are_neutral(dev, B, new_hi, spare):
    """Bounds larger than the step, in one launch and in two: new tensors, and with pad those of an earlier step, hold
    the plan and neutral entries behind it; rows alone and tiles alone too."""
    import torch

    from detkernels_b200.kernels.paging import paged_plan, paged_plan_reference
    rng = np.random.default_rng(B + spare)
    kv, new = rng.integers(0, 200, size=B), rng.integers(0, new_hi + 1, size=B)
    width = int(-(-(kv + new).max() // 16))
    table = rng.permutation(B * width).reshape(B, width)
    want = paged_plan_reference(table.tolist(), kv.tolist(), new.tolist(), 16, rows_per_tile=4)
    n, nt = len(want.row_seq), len(want.row_tiles)
    args = (_i32(table, dev), _i32(kv, dev), _i32(new, dev), 16)
    rows, tiles = dict(n_rows=n + spare), dict(rows_per_tile=4, n_tiles=nt + spare)
    old = lambda: _plan_outputs(dev, B, n + spare, nt + spare, 12345)
    mixed = old()._replace(slots=None, row_tiles=None)     # some tensors of an earlier step, which stay; the rest new
    for kw, out, pad in (({**rows, **tiles}, None, False), ({**rows, **tiles}, old(), True), (rows, None, False),
                         (rows, old(), True), (tiles, None, False), (tiles, old(), True), ({**rows, **tiles}, mixed, False)):
        got = paged_plan(*args, **kw, out=out, pad=pad)
        for name, m in (("row_seq", n), ("row_pos", n), ("slots", n), ("q_lens", n), ("row_tiles", nt)):
            t, w = getattr(got, name), getattr(want, name)
            if (name == "row_tiles" and "n_tiles" not in kw) or (name != "row_tiles" and "n_rows" not in kw):
                assert t is None
                continue
            w = np.asarray(w, np.int64).reshape(m, *t.shape[1:])
            assert np.array_equal(t[:m].cpu().numpy(), w), name
            rest = 12345 if out is mixed and getattr(mixed, name) is not None else NEUTRAL[name]
            assert t.shape[0] == m + spare and (t[m:] == rest).all(), name
    none = paged_plan(_i32(np.zeros((2, 1)), dev), _i32([], dev), _i32([], dev), 16, n_rows=5, rows_per_tile=4, n_tiles=2)
    assert all((getattr(none, k) == v).all() for k, v in NEUTRAL.items())


@pytest.mark.gpu
@pytest.mark.parametrize("B", [2, 3000])
@pytest.mark.parametrize("why", ["length", "pool", "rows"])
def test_a_refused_plan_leaves_nothing_to_do(dev, B, why):
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.paging import paged_plan
    new = np.full(B, 3)
    new[-1] = -1 if why == "length" else 3
    n = 3 * B - (why == "rows")
    free = _i32(np.arange(B - (why == "pool")), dev)
    for out in (None, _plan_outputs(dev, B, n, B, 7)):
        table = torch.full((B, 1), -9, dtype=torch.int32, device=dev)
        got = paged_plan(table, _i32(np.zeros(B), dev), _i32(new, dev), 64, free_blocks=free, cursor=_i32([0], dev),
                         n_rows=n, rows_per_tile=3, n_tiles=B, out=out, pad=True)
        code = {"length": 0x600, "pool": 0x601, "rows": 0x602}[why]
        assert _lib.device_status(dev.index) == (_lib.DK_ERR_DEVICE_CHECK, code)
        assert (table == -9).all() and got.cursor.tolist() == [0]
        for k, v in NEUTRAL.items():
            assert (getattr(got, k) == v).all(), k


@pytest.mark.gpu
def test_a_step_captured_at_its_largest_serves_smaller_ones(dev):
    """Plan, norm into the cache and attention captured once for 40 rows and 16 tiles, then replayed for ragged steps of
    fewer, the last one refused: caches, tables and covered rows as in eager steps of the exact sizes, everything else
    as it was."""
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.attention import attention_shared_prefix
    from detkernels_b200.kernels.paging import paged_plan
    from detkernels_b200.kernels.rope import qk_norm_rope, rope_table
    B, H, Hkv, D, P, page, rows, tiles = 6, 8, 2, 64, 130, 64, 40, 16
    g = torch.Generator(device=dev).manual_seed(2)
    randn = lambda *s: torch.randn(*s, device=dev, generator=g).to(torch.bfloat16)
    rope, qw, kw = rope_table(1024, D, device=dev), randn(D), randn(D)
    n_pre = -(-P // page)
    kc0, vc0 = randn(n_pre + 14, Hkv, page, D), randn(n_pre + 14, Hkv, page, D)
    order = torch.randperm(n_pre + 14, device=dev, generator=g).to(torch.int32)
    pre, free = order[:n_pre].contiguous(), order[n_pre:].contiguous()

    def state():
        z = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)
        return dict(kc=kc0.clone(), vc=vc0.clone(), table=z(B, 5), cursor=z(1), kv=z(B), nw=z(B),
                    qkv=torch.zeros(rows, (H + 2 * Hkv) * D, dtype=torch.bfloat16, device=dev),
                    out=torch.full((rows, H, D), 7.0, dtype=torch.bfloat16, device=dev))

    def step(s, n_rows, n_tiles, plan=None, pad=False):
        q, k, v = (x.view(n_rows, -1, D) for x in s["qkv"][:n_rows].split([H * D, Hkv * D, Hkv * D], 1))
        plan = paged_plan(s["table"], s["kv"], s["nw"], page, free_blocks=free, cursor=s["cursor"], n_rows=n_rows,
                          rows_per_tile=4, n_tiles=n_tiles, out=plan, pad=pad)
        s["cursor"].copy_(plan.cursor)
        q, _ = qk_norm_rope(q, k, plan.row_pos + P, qw, kw, rope, v=v, k_cache=s["kc"], v_cache=s["vc"], slots=plan.slots)
        attention_shared_prefix(q, s["kc"], s["vc"], s["kc"], s["vc"], plan.q_lens, prefix_len=P, prefix_blocks=pre,
                                block_table=s["table"], row_tiles=plan.row_tiles, out=s["out"][:n_rows], max_kv_len=320)
        return plan

    a, b = state(), state()
    plan = step(a, rows, tiles)          # an empty step: loads the library and makes the plan's tensors
    for k in ("kc", "vc", "table", "kv"):
        assert torch.equal(a[k], b[k])
    graph = torch.cuda.CUDAGraph()
    with _lib.graph_capture(graph):
        step(a, rows, tiles, plan=plan, pad=True)
    for i, new in enumerate(([8, 8, 8, 8, 4, 4], [1, 0, 3, 1, 0, 9], [0] * 6, [1] * 6, [0, 0, 33, 1, 0, 0], [1, 1, 0, 0, 0, 1])):
        a["nw"].copy_(_i32(new, dev))
        a["qkv"].copy_(randn(*a["qkv"].shape))
        a["out"].fill_(7.0)
        for k in ("nw", "qkv", "out"):
            b[k].copy_(a[k])
        graph.replay()
        n = sum(new)
        if n:
            step(b, n, sum(-(-x // 4) for x in new))
        for k in ("kc", "vc", "table", "cursor", "out"):
            assert torch.equal(a[k], b[k]), (i, k)
        a["kv"] += a["nw"]
        b["kv"] += b["nw"]
    keep = {k: v.clone() for k, v in a.items()}
    a["nw"].fill_(64)                    # more rows than the step was captured for
    graph.replay()
    assert _lib.device_status(dev.index) == (_lib.DK_ERR_DEVICE_CHECK, 0x602)
    for k in ("kc", "vc", "table", "cursor", "out"):
        assert torch.equal(a[k], keep[k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("R,n_tiles", [(9, 1), (700, 300)])
@pytest.mark.parametrize("prefix", [0, 100])
def test_rows_without_tokens_of_their_own_keep_to_the_tiles(dev, R, n_tiles, prefix):
    """max_kv_len = 0: lengths are not read, rows that a tile covers are those of a call without tiles, the others stay,
    and a malformed tile is reported."""
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.attention import attention_shared_prefix
    q, kp, vp, k, v = _attn_inputs(dev, R, 6, 2, 64, 100, 64, R)
    ln = torch.full((R,), 5, dtype=torch.int32, device=dev)
    kw = dict(prefix_len=prefix, max_kv_len=0)
    want = attention_shared_prefix(q, kp, vp, k, v, ln, **kw)
    assert prefix or (want == 0).all()
    tiles = [(2 * i + 1, 1 + i % 2, i) for i in range(n_tiles)] + [(0, 0, 0)]
    covered = np.zeros(R, bool)
    for a, n, _ in tiles:
        covered[a:a + n] = True
    covered = torch.from_numpy(covered).to(dev)
    for extra in ([], [(R, 1, 0)]):
        out = torch.full_like(q, 7.0)
        attention_shared_prefix(q, kp, vp, k, v, ln, row_tiles=_i32(tiles + extra, dev), out=out, **kw)
        assert _lib.device_status(dev.index) == ((_lib.DK_ERR_DEVICE_CHECK, 0x211) if extra else (0, 0))
        assert torch.equal(out[covered], want[covered]) and (out[~covered] == 7.0).all() and not covered.all()


@pytest.mark.gpu
def test_calls_without_a_prefix_share_no_scratch(dev, monkeypatch):
    """prefix_len = 0 with rows of several splits: the bits of attention_decode, from scratch of the call's own; two
    captured calls replayed at once on two streams."""
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.attention import attention_decode, attention_shared_prefix
    cases = []
    for R, seed in ((3, 1), (40, 2)):
        q, kp, vp, k, v = _attn_inputs(dev, R, 8, 4, 64, 1, 2048, R, seed)
        ln = _i32(np.random.default_rng(seed).integers(0, 2049, size=R), dev)
        cases.append((q, kp, vp, k, v, ln, attention_decode(q, k, v, ln)))

    def shared(nbytes, *_):
        assert nbytes == 0, "a workspace that other calls use"
    monkeypatch.setattr(_lib, "workspace", shared)
    graphs = []
    for q, kp, vp, k, v, ln, want in cases:
        assert torch.equal(attention_shared_prefix(q, kp, vp, k, v, ln, prefix_len=0), want)
        g = torch.cuda.CUDAGraph()
        with _lib.graph_capture(g):
            out = attention_shared_prefix(q, kp, vp, k, v, ln, prefix_len=0)
        graphs.append((g, out, want, torch.cuda.Stream(device=dev)))
    for _ in range(20):
        for g, out, _, s in graphs:
            with torch.cuda.stream(s):
                out.zero_()
                g.replay()
        torch.cuda.synchronize(dev)
        assert all(torch.equal(out, want) for _, out, want, _ in graphs)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [5, 900, 6000])
def test_a_plan_over_its_own_lengths(dev, B):
    """kv_lens and new_lens inside the outputs that the plan writes: the plan of copies of them."""
    import torch

    from detkernels_b200.kernels.paging import paged_plan
    rng = np.random.default_rng(B)
    kv, new = rng.integers(1, 60, size=B), rng.integers(0, 4, size=B)
    table = _i32(rng.permutation(B * 64).reshape(B, 64), dev)
    n, nt = int(new.sum()), int((-(-new // 2)).sum())
    kw = dict(n_rows=n, rows_per_tile=2, n_tiles=nt)
    want = paged_plan(table, _i32(kv, dev), _i32(new, dev), 1, **kw)
    for lens, name, at in ((kv, "q_lens", n - B), (kv, "q_lens", 0), (new, "row_seq", n - B), (new, "row_tiles", 0), (kv, "cu_rows", 1)):
        old = paged_plan(table, _i32(kv, dev), _i32(new, dev), 1, **kw)
        over = getattr(old, name).view(-1)[at:at + B]
        over.copy_(_i32(lens, dev))
        a, b = (over, _i32(new, dev)) if lens is kv else (_i32(kv, dev), over)
        got = paged_plan(table, a, b, 1, out=old, **kw)
        for x, y in zip(got, want):
            assert (x is None and y is None) or torch.equal(x, y), name


def test_the_longest_caches_on_the_host():
    """Whole splits of 64 stay inside 32 bits: a capacity of 2^31 - 64 tokens gets as far as its workspace."""
    from detkernels_b200 import _lib
    lib = _lib.load()

    def call(cap, max_len):
        return lib.dk_attention_shared_prefix(16, 128, 64, 16, 16, 0, 640, 64, 10, None, 0, 0, 16, 16, 64, 64, 64, 3, cap,
                                              None, 0, 0, 0, 0, 16, 128, 64, 16, None, 0, 3, 2, 2, 64, max_len, 0.1,
                                              _lib.DK_BF16, 16, 0, None)
    assert call(2 ** 31 - 64, 2 ** 31 - 1) == _lib.DK_ERR_WORKSPACE
    assert call(2 ** 31 - 63, 100) == _lib.DK_ERR_INVALID_ARGUMENT and "KV extents" in _lib.last_error()


@pytest.mark.gpu
def test_sizes_that_leave_32_bits(dev):
    """Refused, not cut to their low half; a maximum beyond the cache is the cache's."""
    import torch

    from detkernels_b200.kernels.attention import attention_shared_prefix
    from detkernels_b200.kernels.paging import paged_plan
    one, none = _i32([1], dev), _i32([0], dev)
    table = _i32([[0]], dev)
    with pytest.raises(ValueError):
        paged_plan(table, none, one, 2 ** 32 + 64, n_rows=1)
    got = paged_plan(table, none, one, 64, n_rows=1, rows_per_tile=2 ** 32 + 1, n_tiles=1)
    assert got.row_tiles.tolist() == [[0, 1, 0]]
    q, kp, vp, k, v = _attn_inputs(dev, 3, 2, 1, 32, 10, 64, 3)
    ln = _i32([5, 0, 64], dev)
    want = attention_shared_prefix(q, kp, vp, k, v, ln)
    for most in (65, 2 ** 31 - 1, 2 ** 32, 2 ** 40 + 1):
        assert torch.equal(attention_shared_prefix(q, kp, vp, k, v, ln, max_kv_len=most), want)
    pool = torch.zeros(1, 1, 4096, 32, dtype=q.dtype, device=dev)
    wide = torch.zeros(3, 2 ** 20, dtype=torch.int32, device=dev)      # 2^32 tokens a row
    with pytest.raises(ValueError):
        attention_shared_prefix(q, kp, vp, pool, pool, ln, block_table=wide)
    with pytest.raises(ValueError):
        attention_shared_prefix(q, pool, pool, k, v, ln, prefix_blocks=wide[0].repeat(2)[:2 ** 20 + 1])


@pytest.mark.gpu
def test_a_workspace_of_the_callers(dev):
    """Its contents do not matter, too small a one is refused, and so is anything that is not bytes on the device."""
    import torch

    from detkernels_b200 import _lib
    from detkernels_b200.kernels.attention import attention_shared_prefix
    q, kp, vp, k, v = _attn_inputs(dev, 3, 4, 2, 64, 700, 640, 3)
    ln = _i32([5, 0, 640], dev)
    want = attention_shared_prefix(q, kp, vp, k, v, ln)
    n = _lib.load().dk_attention_shared_prefix_workspace_size(3, 3, 4, 2, 64, 700, 640)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=dev)
    assert torch.equal(attention_shared_prefix(q, kp, vp, k, v, ln, workspace=ws), want)
    with pytest.raises(_lib.DetKernelsError):
        attention_shared_prefix(q, kp, vp, k, v, ln, workspace=ws[:n - 16])
    for bad in (ws.cpu(), ws[:n // 4 * 4].view(torch.int32), ws[::2]):
        with pytest.raises(AssertionError):
            attention_shared_prefix(q, kp, vp, k, v, ln, workspace=bad)


@pytest.mark.gpu
def test_a_small_plan_counts_the_one_launch_it_takes(dev):
    from detkernels_b200 import _lib
    from detkernels_b200.kernels.paging import paged_plan
    n0 = _lib.launch_count()
    paged_plan(_i32([[0]], dev), _i32([0], dev), _i32([1], dev), 64, n_rows=1)
    assert _lib.launch_count() - n0 == 1


@pytest.mark.gpu
@pytest.mark.parametrize("paged", [True, False])
def test_caches_beyond_32_bit_offsets(dev, paged):
    """Slots, pages, prefix blocks and whole sequences whose element offsets pass 2^32: the norm's stores, the own tokens'
    and the prefix's reads are those of a small cache with the same contents."""
    import torch

    from detkernels_b200.kernels.attention import attention_shared_prefix
    from detkernels_b200.kernels.rope import qk_norm_rope, rope_table
    if torch.cuda.mem_get_info(dev)[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    H, Hkv, D, page = 8, 4, 128, 64
    T = 3
    n = 2 ** 32 // (Hkv * page * D) + 9
    small = 12
    g = torch.Generator(device=dev).manual_seed(1)
    randn = lambda *s: torch.randn(*s, device=dev, generator=g).to(torch.bfloat16)
    ks, vs = randn(small, Hkv, page, D), randn(small, Hkv, page, D)
    kb, vb = (torch.empty(n, Hkv, page, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    far = torch.tensor([n - 1 - i * (n // 13) for i in range(small)], device=dev)   # where block i of the small one lies
    kb[far], vb[far] = ks, vs
    qkv = randn(T, (H + 2 * Hkv) * D)
    q, k, v = (x.view(T, -1, D) for x in qkv.split([H * D, Hkv * D, Hkv * D], 1))
    w, table, pos = randn(D), rope_table(300, D, device=dev), torch.arange(200, 200 + T, device=dev)
    own = torch.tensor([0, 1, 2], device=dev)            # a block a row, its last token new
    outs = []
    for kc, vc, where in ((ks, vs, torch.arange(small, device=dev)), (kb, vb, far)):
        slots = where[own] * page + page - 1
        qr, _ = qk_norm_rope(q, k, pos, w, w, table, v=v, k_cache=kc, v_cache=vc, slots=slots)
        ln = torch.full((T,), page, dtype=torch.int32, device=dev)
        i32 = lambda x: x.to(torch.int32)
        if paged:
            outs.append(attention_shared_prefix(qr, kc, vc, kc, vc, ln, prefix_len=page * 9 - 5, prefix_blocks=i32(where[3:]),
                                                block_table=i32(where[own][:, None])))
        else:
            kp, vp = (x.permute(1, 0, 2, 3)[:, where[3:]].reshape(Hkv, -1, D) for x in (kc, vc))
            tiles = torch.stack([own, torch.ones_like(own), where[own]], 1).to(torch.int32)
            outs.append(attention_shared_prefix(qr, kp, vp, kc, vc, ln, row_tiles=tiles))
    assert torch.equal(kb[far], ks) and torch.equal(vb[far], vs)
    assert torch.equal(*outs) and torch.isfinite(outs[0].float()).all()
    del kb, vb
    torch.cuda.empty_cache()
