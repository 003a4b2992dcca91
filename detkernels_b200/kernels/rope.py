"""Per-head RMSNorm of queries and keys with the position rotation in the same pass.

Stands beside ``rmsnorm.py`` (the whole-row norm): every query and key head is
normalised over its own head_dim, its first rotary_dim elements are rotated by
the row's position, and, with a KV cache, the key and the value go straight to
their slot.  f32 math with one rounding at the store; a row's bits depend on
that row alone, and on which of two kernels the call's layout takes (their sums
of squares differ in order).  No counterpart in the reference (its decoder has neither,
tiny_model.py:99-140).
"""
from __future__ import annotations

from detkernels_b200 import _lib

MAX_HEAD_DIM = 512


def rope_table(max_pos: int, rotary_dim: int, theta: float = 10000.0, device=None):
    """f32 [max_pos, rotary_dim]: cos then sin of pos * theta^(-2i / rotary_dim), i < rotary_dim / 2,
    from angles in 64 bits (in 32 the angles of far positions lose their last turns)."""
    import torch

    if max_pos < 1 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rope_table: max_pos must be positive and rotary_dim even")
    inv = float(theta) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    ang = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * inv[None, :]
    return torch.cat([ang.cos(), ang.sin()], dim=1).to(torch.float32)


def qk_norm_rope_reference(q, k, positions, q_weight, k_weight, table, eps: float = 1e-6, *, interleaved=False):
    """Plain PyTorch form, f32: returns (q_out, k_out) in q's and k's dtype."""
    import torch

    rd = table.shape[1]
    cs = table[positions.long()].to(torch.float32)[:, None, :]
    cos, sin = cs[..., :rd // 2], cs[..., rd // 2:]
    outs = []
    for x, w in ((q, q_weight), (k, k_weight)):
        x32 = x.to(torch.float32)
        y = x32 * torch.rsqrt(x32.pow(2).mean(dim=-1, keepdim=True) + eps) * w.to(torch.float32)
        r, rest = y[..., :rd], y[..., rd:]
        a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rd // 2], r[..., rd // 2:])
        a, b = a * cos - b * sin, a * sin + b * cos
        r = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
        outs.append(torch.cat([r, rest], dim=-1).to(x.dtype))
    return tuple(outs)


def qk_norm_rope(q, k, positions, q_weight, k_weight, table, eps: float = 1e-6, *, interleaved: bool = False, v=None,
                 k_cache=None, v_cache=None, slots=None, q_out=None, k_out=None):
    """RMSNorm of each query and key head, then the rotation of its first table.shape[1] elements.

    q [T, H, D], k [T, H_kv, D] (any row and head strides, e.g. views of one QKV matmul's output);
    positions int32 or int64 CUDA [T]; q_weight, k_weight [D]; table f32 [max_pos, rotary_dim] of
    ``rope_table`` (cos, then sin).  Pairs are (i, i + rotary_dim / 2), or (2i, 2i + 1) when interleaved.
    q_out / k_out may be q / k.

    With k_cache, v_cache ([n, H_kv, capacity, D]: one slab per sequence, or a block pool), v [T, H_kv, D]
    and slots (int64 CUDA [T], slab * capacity + token, e.g. ``paged_plan(...).slots``), the key and the
    value of each row are stored at its slot; a negative slot stores nothing.  k_out is then only written
    if given.  A position outside the table or a slot outside the cache sets the device status, and that
    row (or its K and V) is not written.  Rows of one call must not share a slot.

    Two kernels, either batch invariant: vectors of 16 bytes where every tensor's rows and heads start on 16
    bytes and the rotated half is a half or a quarter of the head in whole vectors (neighbouring pairs: any
    rotary_dim of whole vectors); elements otherwise, for all of the call, also where only one tensor is
    laid out so, and for some f32 heads beyond 256 elements.  Their results may differ in the last bit.

    Returns (q_out, k_out); k_out is None when the keys went to the cache only."""
    import torch

    dev, dt = q.device, q.dtype
    assert q.is_cuda, "qk_norm_rope requires CUDA tensors"
    T, H, D = q.shape
    kv_shape = k.shape
    assert len(kv_shape) == 3 and kv_shape[0] == T and kv_shape[2] == D, "q/k shape mismatch"
    Hkv = kv_shape[1]
    if k.dtype != dt or q_weight.dtype != k_weight.dtype:
        raise TypeError("qk_norm_rope: q and k, and the two weights, must share a dtype")
    assert q_weight.numel() == D and k_weight.numel() == D, "qk_norm_rope: weights must have head_dim elements"
    assert positions.dtype in (torch.int32, torch.int64) and positions.shape == (T,), \
        "positions must be int32 or int64 [T]"
    assert table.dtype == torch.float32 and table.dim() == 2 and table.is_contiguous(), "table must be f32, contiguous"
    if D > MAX_HEAD_DIM:
        raise NotImplementedError("qk_norm_rope: head_dim %d > %d" % (D, MAX_HEAD_DIM))
    max_pos, rd = table.shape
    if rd < 2 or rd % 2 or rd > D or max_pos < 1:
        raise ValueError("qk_norm_rope: a table of an even rotary_dim in [2, head_dim] required")
    n_cache = (v is not None) + (k_cache is not None) + (v_cache is not None) + (slots is not None)
    if n_cache not in (0, 4):
        raise ValueError("qk_norm_rope: v, k_cache, v_cache and slots go together")
    tensors = [k, positions, q_weight, k_weight, table]
    cs, n_slabs, cap = (0, 0, 0, 1), 0, 0
    if n_cache:
        tensors += [v, k_cache, v_cache, slots]
        assert v.shape == kv_shape and v.dtype == dt, "k/v shape mismatch"
        c_shape, cs = k_cache.shape, k_cache.stride()
        assert k_cache.dtype == dt and v_cache.dtype == dt and c_shape == v_cache.shape
        assert len(c_shape) == 4 and c_shape[1] == Hkv and c_shape[3] == D, "cache shape mismatch"
        assert cs == v_cache.stride() and (D <= 1 or cs[3] == 1), \
            "k and v caches must share strides, with a unit stride along head_dim"
        assert slots.dtype == torch.int64 and slots.shape == (T,), "slots must be int64 [T]"
        n_slabs, cap = c_shape[0], c_shape[2]
    elif k_out is None:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        assert q_out.shape == q.shape and q_out.dtype == dt
        tensors.append(q_out)
    qo_st, ko_st = q_out.stride(), (0, 0, 1)
    if k_out is not None:
        assert k_out.shape == kv_shape and k_out.dtype == dt
        tensors.append(k_out)
        ko_st = k_out.stride()
    assert D <= 1 or (qo_st[2] == 1 and ko_st[2] == 1), "outputs must have a unit stride along head_dim"
    index = dev.index
    for t in tensors:
        assert t.get_device() == index, "qk_norm_rope: all tensors must be on q's device"
    if T == 0:
        return q_out, k_out

    def unit(t):
        """t and its strides, with a unit stride along head_dim."""
        st = t.stride()
        if D <= 1 or st[2] == 1:
            return t, st
        t = t.contiguous()
        return t, t.stride()

    with _lib.on_device(dev):
        (q2, q_st), (k2, k_st) = unit(q), unit(k)
        v2, v_st = unit(v) if n_cache else (None, (0, 0))
        qw = q_weight if q_weight.is_contiguous() else q_weight.reshape(-1).contiguous()
        kw = k_weight if k_weight.is_contiguous() else k_weight.reshape(-1).contiguous()
        pos = positions.contiguous()
        slots = slots.contiguous() if n_cache else None
        rc = _lib.load().dk_qk_norm_rope(
            q2.data_ptr(), q_st[0], q_st[1], k2.data_ptr(), k_st[0], k_st[1], v2.data_ptr() if n_cache else None,
            v_st[0], v_st[1], q_out.data_ptr(), qo_st[0], qo_st[1], k_out.data_ptr() if k_out is not None else None,
            ko_st[0], ko_st[1], k_cache.data_ptr() if n_cache else None, v_cache.data_ptr() if n_cache else None,
            cs[0], cs[1], cs[2], n_slabs, cap, slots.data_ptr() if n_cache else None, pos.data_ptr(),
            1 if pos.dtype == torch.int64 else 0, qw.data_ptr(), kw.data_ptr(), _lib.dtype_code(qw.dtype),
            table.data_ptr(), max_pos, T, H, Hkv, D, rd, 1 if interleaved else 0, float(eps),
            _lib.dtype_code(dt), _lib.stream_ptr(dev))
    _lib.check(rc, "qk_norm_rope")
    _lib.count_launch()
    return q_out, k_out
