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
