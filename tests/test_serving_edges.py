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
