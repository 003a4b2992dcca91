"""Batch-invariant single-query (decode-step) attention.

Drop-in for the reference's ``kernels/attention.py``:

* ``attention_reference`` (attention.py:49-71): einsum scores, softmax, einsum
  with V, all f32.  Extended (keyword-only) with GQA -- k/v may carry fewer
  heads than q, query head h reading kv head h // (H / H_kv) -- and per-row KV
  lengths ``kv_lens``.
* ``attention_batch_invariant`` (attention.py:289-298): split-KV decode
  attention with a fixed split SIZE of 256 tokens, a fixed in-split order and a
  fixed-order combine, so a row's output bits depend only on its own q, KV and
  length.  ``block_s`` is accepted for signature compatibility.
* ``attention_batch_variant`` (attention.py:301-348): the deliberately variant
  twin -- a fixed split COUNT with f32 atomics when B*H < split_bh_threshold.
* ``attention_shared_prefix`` (no counterpart in the reference): decode
  attention of rows that share a prefix, whose part is computed once for the
  whole batch on the tensor cores; ``attention_shared_prefix_reference`` is its
  plain form.
* ``attention_tree`` (no counterpart either): the rows of a sequence are drafted
  tokens, a tree of them or any other set given by masks, behind its cached tokens;
  ``attention_tree_reference`` is its plain form.

Shapes: q [B, H, D]; k, v [B, H_kv, S, D]; out like q.
"""
from __future__ import annotations

from detkernels_b200 import _lib

KV_SPLIT = _lib.ATTN_KV_SPLIT
_I32_MAX = 2 ** 31 - 1


def attention_reference(q, k, v, scale: float | None = None, *, kv_lens=None):
    """Plain PyTorch eager decode-step attention, f32 (reference attention.py:49-71).

    q: (B, H, D); k, v: (B, H_kv, S, D) with H % H_kv == 0; kv_lens: optional
    per-row valid lengths (row b attends to k[b, :, :kv_lens[b]])."""
    import torch

    orig_dtype = q.dtype
    d = q.shape[-1]
    if scale is None:
        scale = 1.0 / (d ** 0.5)
    q32 = q.to(torch.float32)
    H, Hkv = q.shape[1], k.shape[1]
    if kv_lens is None:
        k32 = k.to(torch.float32)
        v32 = v.to(torch.float32)
        if Hkv != H:
            k32 = k32.repeat_interleave(H // Hkv, dim=1)
            v32 = v32.repeat_interleave(H // Hkv, dim=1)
        scores = torch.einsum("bhd,bhsd->bhs", q32, k32) * scale
        probs = torch.softmax(scores, dim=-1)
        out = torch.einsum("bhs,bhsd->bhd", probs, v32)
        return out.to(orig_dtype)
    # ragged rows: each row's own prefix of the cache, converted and expanded alone (the padding
    # beyond a row's length is never touched)
    outs = []
    for b in range(q.shape[0]):
        L = int(kv_lens[b])
        if L == 0:
            outs.append(torch.zeros_like(q32[b]))
            continue
        kb = k[b, :, :L].to(torch.float32)
        vb = v[b, :, :L].to(torch.float32)
        if Hkv != H:
            kb = kb.repeat_interleave(H // Hkv, dim=0)
            vb = vb.repeat_interleave(H // Hkv, dim=0)
        s = torch.einsum("hd,hsd->hs", q32[b], kb) * scale
        outs.append(torch.einsum("hs,hsd->hd", torch.softmax(s, dim=-1), vb))
    return torch.stack(outs).to(orig_dtype)


def attention_decode(q, k_cache, v_cache, kv_lens, *, scale=None, row_tiles=None, max_kv_len=None, out=None,
                     workspace=None, block_table=None):
    """General entry: q [R, H, D] rows over a KV cache [N_seq, H_kv, capacity, D].

    kv_lens: int32 CUDA tensor [R] (or an int for every row).  row_tiles:
    optional int32 CUDA tensor [T, 3] (first row, row count, sequence) grouping
    consecutive rows of one sequence; without it row r reads sequence r.  A tile of 0 rows is skipped
    (padding), and rows that no tile covers keep what ``out`` holds.
    max_kv_len: host-side bound on every kv_len (defaults to the capacity).
    block_table: optional int32 CUDA tensor [N_seq, blocks_per_seq] for a paged cache: k_cache /
    v_cache are then block pools [n_blocks, H_kv, page, D] (page a multiple of 64) and token t of
    sequence s lives at block_table[s, t // page], token t % page.  Same bits as a contiguous cache.
    """
    import torch

    assert q.is_cuda and k_cache.is_cuda and v_cache.is_cuda, "attention requires CUDA tensors"
    R, H, D = q.shape
    n_seq, Hkv, cap, D2 = k_cache.shape
    if block_table is not None:
        assert block_table.dtype == torch.int32 and block_table.is_cuda and block_table.dim() == 2
        assert block_table.stride(1) == 1
        n_blocks, page = n_seq, cap
        n_seq, cap = block_table.shape[0], block_table.shape[1] * page
    assert D2 == D and v_cache.shape == k_cache.shape, "q/k/v shape mismatch"
    assert k_cache.stride() == v_cache.stride(), "k and v caches must share strides"
    assert k_cache.stride(3) == 1 and q.stride(2) == 1, "unit stride along head_dim required"
    if q.dtype != k_cache.dtype or v_cache.dtype != k_cache.dtype:
        raise TypeError("attention: q, k, v must share a dtype")
    if scale is None:
        scale = 1.0 / (D ** 0.5)
    if out is None:
        out = torch.empty((R, H, D), dtype=q.dtype, device=q.device)
    if R == 0:
        return out
    if max_kv_len is None:
        max_kv_len = cap
    lens_ptr, uniform = None, 0
    if isinstance(kv_lens, int):
        uniform = kv_lens
    else:
        assert kv_lens.dtype == torch.int32 and kv_lens.is_cuda and kv_lens.numel() == R
        lens_ptr = kv_lens.data_ptr()
    tiles_ptr, n_tiles, rows_per_tile = None, R, 1
    if row_tiles is not None:
        assert row_tiles.dtype == torch.int32 and row_tiles.is_cuda and row_tiles.is_contiguous()
        tiles_ptr, n_tiles, rows_per_tile = row_tiles.data_ptr(), row_tiles.shape[0], 2
    lib = _lib.load()
    stream = _lib.stream_ptr(q.device)
    if workspace is None:
        nbytes = lib.dk_attention_workspace_size(n_tiles, rows_per_tile, H, Hkv, D, int(max_kv_len))
        workspace = _lib.workspace(nbytes, q.device, stream)
    if block_table is not None:
        rc = lib.dk_attention_paged_batch_invariant(
            q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0),
            k_cache.stride(1), k_cache.stride(2), n_blocks, page, block_table.data_ptr(), block_table.stride(0),
            n_seq, block_table.shape[1], out.data_ptr(), out.stride(0), out.stride(1), lens_ptr, int(uniform),
            tiles_ptr, int(n_tiles), R, H, Hkv, D, int(max_kv_len), float(scale), _lib.dtype_code(q.dtype),
            workspace.data_ptr() if workspace is not None else None,
            workspace.numel() if workspace is not None else 0, stream)
        _lib.check(rc, "attention_paged_batch_invariant")
        _lib.count_launch()
        return out
    rc = lib.dk_attention_batch_invariant(
        q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0),
        k_cache.stride(1), k_cache.stride(2), n_seq, cap, out.data_ptr(), out.stride(0), out.stride(1),
        lens_ptr, int(uniform), tiles_ptr, int(n_tiles), R, H, Hkv, D, int(max_kv_len), float(scale),
        _lib.dtype_code(q.dtype), workspace.data_ptr() if workspace is not None else None,
        workspace.numel() if workspace is not None else 0, stream)
    _lib.check(rc, "attention_batch_invariant")
    _lib.count_launch()
    return out


def _kv_ready(t):
    # TMA needs a unit stride along D and 16-byte aligned strides elsewhere
    if t.stride(3) == 1 and all((s * t.element_size()) % 16 == 0 for s in t.stride()[:3]) \
            and t.data_ptr() % 16 == 0:
        return t
    return t.contiguous()


def attention_batch_invariant(q, k, v, scale: float | None = None, block_s: int = 64, *, kv_lens=None):
    """Batch-invariant decode-step attention (fixed split size, fixed-order combine)."""
    import torch

    assert q.is_cuda and k.is_cuda and v.is_cuda, "attention_batch_invariant requires CUDA tensors"
    B, H, D = q.shape
    Bk, Hkv, S, Dk = k.shape
    assert Bk == B and Dk == D and v.shape == k.shape, "q/k/v shape mismatch"
    assert H % Hkv == 0, "query heads must be a multiple of kv heads"
    q2 = q if q.stride(2) == 1 and q.stride(0) % 2 == 0 and q.stride(1) % 2 == 0 else q.contiguous()
    k2, v2 = _kv_ready(k), _kv_ready(v)
    if k2.stride() != v2.stride():
        k2, v2 = k2.contiguous(), v2.contiguous()
    if kv_lens is None:
        lens = S
    else:
        lens = torch.as_tensor(kv_lens, device=q.device).to(torch.int32).contiguous()
    out = torch.empty((B, H, D), dtype=q.dtype, device=q.device)
    return attention_decode(q2, k2, v2, lens, scale=scale, max_kv_len=S, out=out)


def attention_batch_variant(q, k, v, scale: float | None = None, split_bh_threshold: int = 32, split_s: int = 4,
                            block_s: int = 64):
    """Deliberately batch-variant decode attention (reference attention.py:301-348): a fixed split COUNT
    combined with f32 atomics when B * H < split_bh_threshold, else the invariant kernel."""
    import torch

    assert q.is_cuda and k.is_cuda and v.is_cuda, "attention_batch_variant requires CUDA tensors"
    B, H, D = q.shape
    if scale is None:
        scale = 1.0 / (D ** 0.5)
    if B * H >= split_bh_threshold:
        return attention_batch_invariant(q, k, v, scale)
    S = k.shape[2]
    if k.shape[1] != H:
        k = k.repeat_interleave(H // k.shape[1], dim=1)
        v = v.repeat_interleave(H // v.shape[1], dim=1)
    if k.stride(3) != 1 or k.stride() != v.stride():
        k, v = k.contiguous(), v.contiguous()
    q2 = q if q.stride(2) == 1 else q.contiguous()
    out = torch.empty((B, H, D), dtype=q.dtype, device=q.device)
    lib = _lib.load()
    stream = _lib.stream_ptr(q.device)
    ws = _lib.workspace(lib.dk_attention_variant_workspace_size(B, H, D), q.device, stream)
    rc = lib.dk_attention_batch_variant(
        q2.data_ptr(), q2.stride(0), q2.stride(1), k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1),
        k.stride(2), out.data_ptr(), out.stride(0), out.stride(1), B, H, S, D, float(scale), int(split_s),
        _lib.dtype_code(q.dtype), ws.data_ptr(), ws.numel(), stream)
    _lib.check(rc, "attention_batch_variant")
    return out


def attention_shared_prefix_reference(q, k_prefix, v_prefix, k, v, kv_lens, scale: float | None = None):
    """Plain PyTorch attention of rows behind a shared prefix, f32.

    q: (R, H, D); k_prefix, v_prefix: (H_kv, P, D); k, v: (R, H_kv, S, D), row r's own tokens, of which
    it reads the first kv_lens[r] after the prefix.  A row that reads nothing is zero."""
    import torch

    outs = []
    for r in range(q.shape[0]):
        n = int(kv_lens[r])
        kr = torch.cat([k_prefix, k[r, :, :n].to(k_prefix.dtype)], dim=1)[None]
        vr = torch.cat([v_prefix, v[r, :, :n].to(v_prefix.dtype)], dim=1)[None]
        outs.append(attention_reference(q[r:r + 1], kr, vr, scale) if kr.shape[2] else torch.zeros_like(q[r:r + 1]))
    return torch.cat(outs) if outs else torch.empty_like(q)


def _tma_strides(t, name):
    """Element strides of a 16-bit cache tensor as the kernels need them (unit along D, the others
    multiples of 8 elements, 16-byte aligned base); a dimension of one element takes any stride."""
    st = t.stride()
    if min(t.shape) <= 1:
        st, nat = list(st), 1
        for i in range(t.dim() - 1, -1, -1):
            if t.shape[i] <= 1:
                st[i] = nat
            nat = max(nat, st[i] * max(1, t.shape[i]))
        st = tuple(st)
    if st[-1] != 1 or any([s % 8 for s in st[:-1]]) or t.data_ptr() % 16:
        raise ValueError("%s: unit stride along head_dim, strides that are multiples of 8 elements and a 16-byte "
                         "aligned start required" % name)
    return st


def _shared_strides(k, v, what):
    """The strides of a pair of equal shape, which must share them."""
    st = _tma_strides(k, "k_" + what)
    if v.stride() != k.stride() or v.data_ptr() % 16:
        assert _tma_strides(v, "v_" + what) == st, "k and v %s must share strides" % what
    return st


def attention_shared_prefix(q, k_prefix, v_prefix, k_cache, v_cache, kv_lens, *, prefix_len=None, prefix_blocks=None,
                            block_table=None, row_tiles=None, max_kv_len=None, scale=None, out=None, workspace=None):
    """Batch-invariant decode attention of rows that share a prefix.

    q [R, H, D]; row r attends to the first ``prefix_len`` tokens of the prefix and then to the first
    kv_lens[r] tokens of its own KV sequence (row r reads sequence r, or ``row_tiles`` as in
    ``attention_decode``).  The prefix part is computed once for all rows.

    k_prefix, v_prefix: [H_kv, P, D]; or, with ``prefix_blocks`` (int32 CUDA [ceil(prefix_len / page)]),
    block pools [n_blocks, H_kv, page, D] (page a multiple of 64) whose block prefix_blocks[t // page]
    holds prefix token t.  prefix_len defaults to all of it; 0 is plain ``attention_decode``.
    k_cache, v_cache, kv_lens, block_table, max_kv_len: as in ``attention_decode`` (kv_lens and
    max_kv_len count the rows' own tokens only; the workspace of a small batch grows with max_kv_len, so
    give it where the cache is much longer than the rows).  bf16 or f16; head_dim 32, 64 or 128; at most 16 query
    heads per KV head.  workspace: uint8 CUDA tensor of at least
    ``dk_attention_shared_prefix_workspace_size`` bytes (a new one if not given, and without a prefix; its
    contents do not matter, and calls that may overlap need separate ones).

    A row that row_tiles leaves out keeps what ``out`` holds (rows of a padded batch); with max_kv_len = 0
    no row has tokens of its own, and kv_lens are not read.  A length outside [0, max_kv_len] or the cache, or a
    malformed tile, sets the device status; the rows of that tile keep what ``out`` holds too.
    A row's bits depend on its q, the prefix, its own tokens and nothing else of the batch."""
    import torch

    dev, dt = q.device, q.dtype
    index = dev.index
    for t in (q, k_prefix, v_prefix, k_cache, v_cache):
        assert t.is_cuda and t.get_device() == index, "attention_shared_prefix requires CUDA tensors on one device"
        if t.dtype != dt:
            raise TypeError("attention_shared_prefix: q, the prefix and the caches must share a dtype")
    R, H, D = q_shape = q.shape
    p_shape, c_shape = k_prefix.shape, k_cache.shape
    assert v_prefix.shape == p_shape and v_cache.shape == c_shape, "q/k/v shape mismatch"
    n_seq, Hkv, cap, Dk = c_shape
    assert Dk == D and H % Hkv == 0, "q/k/v shape mismatch"
    n_pool = page_p = 0
    if prefix_blocks is None:
        assert len(p_shape) == 3 and p_shape[0] == Hkv and p_shape[2] == D, "prefix shape mismatch"
        p_cap = p_shape[1]
    else:
        assert prefix_blocks.dtype == torch.int32 and prefix_blocks.get_device() == index and prefix_blocks.dim() == 1
        assert prefix_blocks.numel() <= 1 or prefix_blocks.stride(0) == 1
        assert len(p_shape) == 4 and p_shape[1] == Hkv and p_shape[3] == D, "prefix shape mismatch"
        n_pool, page_p = p_shape[0], p_shape[2]
        p_cap = prefix_blocks.numel() * page_p
    P = p_cap if prefix_len is None else int(prefix_len)
    if P < 0 or P > min(p_cap, _I32_MAX):
        raise ValueError("attention_shared_prefix: prefix_len %d outside [0, %d]" % (P, min(p_cap, _I32_MAX)))
    uniform = isinstance(kv_lens, int)
    if not uniform:
        assert kv_lens.dtype == torch.int32 and kv_lens.get_device() == index and kv_lens.numel() == R
        kv_lens = kv_lens.contiguous()
    n_blocks = page = width = bt_stride = 0
    if block_table is not None:
        assert block_table.dtype == torch.int32 and block_table.get_device() == index and block_table.dim() == 2
        assert block_table.shape[1] <= 1 or block_table.stride(1) == 1
        n_blocks, page = n_seq, cap
        n_seq, width = block_table.shape
        # a single row has any stride; the rows of a larger table must not overlap (the C entry refuses them)
        cap, bt_stride = width * page, block_table.stride(0) if n_seq > 1 else width
    if max_kv_len is None:
        max_kv_len = kv_lens if uniform else cap
    max_kv_len = int(max_kv_len)
    if max_kv_len < 0 or (max_kv_len and not cap):
        raise ValueError("attention_shared_prefix: max_kv_len %d outside the cache" % max_kv_len)
    max_kv_len = min(max_kv_len, cap)   # a bound beyond the cache bounds nothing, but sizes the work
    if max_kv_len > _I32_MAX:
        raise ValueError("attention_shared_prefix: max_kv_len %d exceeds 2^31 - 1" % max_kv_len)
    if uniform and not 0 <= kv_lens <= max_kv_len:
        raise ValueError("attention_shared_prefix: kv_lens %d outside [0, %d]" % (kv_lens, max_kv_len))
    if scale is None:
        scale = 1.0 / (D ** 0.5)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    o_st = out.stride()
    assert out.shape == q_shape and out.dtype == dt and out.get_device() == index and o_st[2] == 1
    if row_tiles is not None:
        assert row_tiles.dtype == torch.int32 and row_tiles.get_device() == index and row_tiles.is_contiguous()
        assert row_tiles.dim() == 2 and row_tiles.shape[1] == 3
    if workspace is not None:
        assert workspace.dtype == torch.uint8 and workspace.get_device() == index and workspace.is_contiguous(), \
            "workspace must be a contiguous uint8 CUDA tensor on q's device"
    if R == 0:
        return out
    q_st = q.stride()
    if q.data_ptr() % 16 or q_st[2] != 1 or q_st[0] % 8 or q_st[1] % 8:
        q = q.clone(memory_format=torch.contiguous_format)
        q_st = q.stride()
    with _lib.on_device(dev):
        if P == 0:
            # scratch of this call alone, its counters zeroed: the shared one of attention_decode would be raced for
            # by two captured calls replayed at once
            n_tiles, per = (R, 1) if row_tiles is None else (row_tiles.shape[0], 2)
            nbytes = _lib.load().dk_attention_workspace_size(n_tiles, per, H, Hkv, D, max_kv_len)
            ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
            if nbytes:
                ws[:_lib.WORKSPACE_COUNTER_BYTES].zero_()
            return attention_decode(q, k_cache, v_cache, kv_lens if max_kv_len else 0, scale=scale, workspace=ws,
                                    row_tiles=row_tiles, max_kv_len=max_kv_len, out=out, block_table=block_table)
        ps = _shared_strides(k_prefix, v_prefix, "prefix")
        cs = [0, 0, 0, 1]
        n_tiles = R if row_tiles is None else row_tiles.shape[0]
        if max_kv_len:
            cs = _shared_strides(k_cache, v_cache, "cache")
            if uniform:
                kv_lens = torch.full((R,), kv_lens, dtype=torch.int32, device=q.device)
        lib = _lib.load()
        nbytes = lib.dk_attention_shared_prefix_workspace_size(R, n_tiles, H, Hkv, D, P, max_kv_len)
        if workspace is None:
            workspace = q.new_empty(max(nbytes, 16), dtype=torch.uint8)
        rc = lib.dk_attention_shared_prefix(
            q.data_ptr(), q_st[0], q_st[1], k_prefix.data_ptr(), v_prefix.data_ptr(),
            ps[0] if prefix_blocks is not None else 0, ps[-3], ps[-2], P,
            prefix_blocks.data_ptr() if prefix_blocks is not None else None, n_pool, page_p, k_cache.data_ptr(),
            v_cache.data_ptr(), cs[0], cs[1], cs[2], n_seq, cap,
            block_table.data_ptr() if block_table is not None else None, bt_stride, width, n_blocks, page,
            out.data_ptr(), o_st[0], o_st[1], None if uniform and not max_kv_len else kv_lens.data_ptr(),
            row_tiles.data_ptr() if row_tiles is not None else None, n_tiles, R, H, Hkv, D, max_kv_len, float(scale),
            _lib.dtype_code(dt), workspace.data_ptr(), workspace.numel(), _lib.stream_ptr(dev))
    _lib.check(rc, "attention_shared_prefix")
    _lib.count_launch(2)   # at least: rows split over several warps take a third
    return out


def attention_tree_reference(q, k, v, kv_lens, cu_rows, tree_mask, scale: float | None = None):
    """Plain PyTorch attention of drafted tokens, f32.

    q: (R, H, D); k, v: (B, H_kv, S, D); rows cu_rows[b] to cu_rows[b + 1] are sequence b's drafts, whose keys and values
    lie behind its first kv_lens[b] tokens; tree_mask: int64 (R, W), bit j of a row's words: it sees draft j.  A row that
    sees nothing is zero, and so are rows behind the last sequence."""
    import torch

    out = torch.zeros_like(q)
    scale = 1.0 / (q.shape[-1] ** 0.5) if scale is None else scale
    G = q.shape[1] // k.shape[1]
    for b in range(len(cu_rows) - 1):
        r0, n, t = int(cu_rows[b]), int(kv_lens[b]), int(cu_rows[b + 1]) - int(cu_rows[b])
        for i in range(t):
            sees = list(range(n)) + [n + j for j in range(min(t, 64 * tree_mask.shape[1]))
                                     if int(tree_mask[r0 + i, j // 64]) >> (j % 64) & 1]
            if sees:
                ks, vs = (x[b][:, sees].float().repeat_interleave(G, 0) for x in (k, v))
                p = torch.softmax((ks * q[r0 + i].float()[:, None]).sum(-1) * scale, -1)
                out[r0 + i] = (p[..., None] * vs).sum(1).to(q.dtype)
    return out


def attention_tree(q, k_cache, v_cache, kv_lens, cu_rows, tree_mask, *, block_table=None, max_kv_len=None, max_rows=None,
                   scale=None, out=None, workspace=None):
    """Batch-invariant attention of drafted tokens over a cache that holds them.

    q [R, H, D]; rows cu_rows[b] to cu_rows[b + 1] (int32 CUDA [B + 1]) are the drafts of sequence b, which holds kv_lens[b]
    tokens (int32 CUDA [B]) and the drafts' keys and values behind them (``paged_plan`` gives their slots, and cu_rows).
    A row attends to all of the kv_lens[b] tokens and to the drafts that its mask names: bit j of tree_mask[row]
    (int64 CUDA [R, W], 64 drafts a word) stands for draft j of its sequence; ``drafts.tree_mask`` makes it from a tree.
    Bits from the sequence's row count on are ignored, drafts past the words are not seen, and a row that sees nothing is 0.

    k_cache, v_cache: [>= B, H_kv, S, D], or with ``block_table`` (int32 CUDA [>= B, blocks]) block pools [n_blocks, H_kv,
    page, D], page a multiple of 64.  bf16 or f16; head_dim 32, 64 or 128; at most 128 query heads per KV head.
    max_rows: a bound on a sequence's rows (64 W if not given); max_kv_len: one on its tokens, drafts included (the cache's
    capacity if not given).  They size the work and the workspace: uint8 CUDA of at least
    ``dk_attention_tree_workspace_size`` bytes (a new one if not given; its contents do not matter, and calls that may
    overlap need separate ones).

    Rows behind the last sequence keep what ``out`` (which may be q) holds.  Offsets that do not ascend inside the rows, more than max_rows
    rows a sequence, a negative length or more than max_kv_len tokens set the device status; that sequence's rows keep what
    ``out`` holds too.  A row's bits depend on its q and the tokens that it sees, and nothing else of the batch."""
    import torch

    dev, dt = q.device, q.dtype
    index = dev.index
    for t in (q, k_cache, v_cache):
        assert t.is_cuda and t.get_device() == index, "attention_tree requires CUDA tensors on one device"
        if t.dtype != dt:
            raise TypeError("attention_tree: q and the caches must share a dtype")
    R, H, D = q_shape = q.shape
    c_shape = k_cache.shape
    assert v_cache.shape == c_shape, "q/k/v shape mismatch"
    n_seq, Hkv, cap, Dk = c_shape
    assert Dk == D and H % Hkv == 0, "q/k/v shape mismatch"
    assert kv_lens.dtype == torch.int32 and kv_lens.get_device() == index and kv_lens.dim() == 1
    B = kv_lens.numel()
    assert cu_rows.dtype == torch.int32 and cu_rows.get_device() == index and cu_rows.shape == (B + 1,)
    assert tree_mask.dtype == torch.int64 and tree_mask.get_device() == index and tree_mask.dim() == 2
    W = tree_mask.shape[1]
    assert tree_mask.shape[0] == R and W >= 1, "attention_tree: one mask a row"
    n_blocks = page = width = bt_stride = 0
    if block_table is not None:
        assert block_table.dtype == torch.int32 and block_table.get_device() == index and block_table.dim() == 2
        assert block_table.shape[1] <= 1 or block_table.stride(1) == 1
        n_blocks, page = n_seq, cap
        n_seq, width = block_table.shape
        cap, bt_stride = width * page, block_table.stride(0) if n_seq > 1 else width
    assert n_seq >= B, "attention_tree: fewer KV sequences than lengths"
    max_kv_len = min(cap, _I32_MAX) if max_kv_len is None else int(max_kv_len)
    max_rows = 64 * W if max_rows is None else int(max_rows)
    if max_rows < 0 or max_kv_len < 0:
        raise ValueError("attention_tree: max_rows and max_kv_len must not be negative")
    if max(R, B, width) > _I32_MAX:
        raise ValueError("attention_tree: too many rows or sequences")
    max_kv_len = min(max_kv_len, cap, _I32_MAX)   # bounds beyond the cache or the batch bound nothing, but size the work
    max_rows = min(max_rows, R, max_kv_len)
    if scale is None:
        scale = 1.0 / (D ** 0.5)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    o_st = out.stride()
    assert out.shape == q_shape and out.dtype == dt and out.get_device() == index and o_st[2] == 1
    if workspace is not None:
        assert workspace.dtype == torch.uint8 and workspace.get_device() == index and workspace.is_contiguous(), \
            "workspace must be a contiguous uint8 CUDA tensor on q's device"
    if R == 0 or B == 0:
        return out
    with _lib.on_device(dev):
        kv_lens, cu_rows = kv_lens.contiguous(), cu_rows.contiguous()
        if W > 1 and tree_mask.stride(1) != 1:
            tree_mask = tree_mask.contiguous()
        q_st = q.stride()
        if q.data_ptr() % 16 or q_st[2] != 1 or q_st[0] % 8 or q_st[1] % 8:
            q = q.clone(memory_format=torch.contiguous_format)
            q_st = q.stride()
        cs = _shared_strides(k_cache, v_cache, "cache")
        lib = _lib.load()
        nbytes = lib.dk_attention_tree_workspace_size(B, R, max_rows, H, Hkv, D, max_kv_len)
        if workspace is None and nbytes:
            workspace = q.new_empty(nbytes, dtype=torch.uint8)
        rc = lib.dk_attention_tree(
            q.data_ptr(), q_st[0], q_st[1], k_cache.data_ptr(), v_cache.data_ptr(), cs[0], cs[1], cs[2], n_seq, cap,
            block_table.data_ptr() if block_table is not None else None, bt_stride, width, n_blocks, page, out.data_ptr(),
            o_st[0], o_st[1], kv_lens.data_ptr(), cu_rows.data_ptr(), tree_mask.data_ptr(), tree_mask.stride(0), W, B, R,
            max_rows, H, Hkv, D, max_kv_len, float(scale), _lib.dtype_code(dt),
            workspace.data_ptr() if workspace is not None else None, workspace.numel() if workspace is not None else 0,
            _lib.stream_ptr(dev))
    _lib.check(rc, "attention_tree")
    _lib.count_launch(2 if nbytes else 1)
    return out
