"""What is measured of the serving operators: the page plan of a step, the per-head norm with the
position rotation into a KV cache, and attention over a shared prefix.

``run`` computes each operator with elementary torch operations in 32 bits, or, where ``own`` is
true, through the package's entry points.  ``exact`` gives the same outputs from the definitions in
64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


# --------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------
def listed():
    return [
        # --- page plan: block table, slot map and attention tiles of one step ---
        # a decode step of a small batch: one new token for each of 7 requests
        dict(name="plan_decode_7", op="plan", B=7, kv_lo=1, kv_hi=1500, new_lo=1, new_hi=1, page=64, rpt=0),
        # the prefill of 256 ragged prompts of up to 512 tokens (the benchmark's batch)
        dict(name="plan_prefill_256", op="plan", B=256, kv_lo=0, kv_hi=0, new_lo=1, new_hi=512, page=64, rpt=16),
        # a large step: 4099 requests, each extended by a ragged chunk of up to 1024 tokens
        dict(name="plan_chunked_4099", op="plan", B=4099, kv_lo=0, kv_hi=3000, new_lo=0, new_hi=1024, page=128, rpt=8),
        # --- head norm + rotation, K and V stored into the cache ---
        # one decode step of 8 requests into a contiguous cache (the smallest: latency)
        dict(name="rope_decode_8", op="rope", dt="f16", B=8, lo=1, hi=1, H=8, Hkv=8, D=64, rd=64, inter=False,
             page=0, max_pos=2048),
        # one decode step of 256 requests at far positions into a paged cache, grouped heads
        dict(name="rope_decode_256_far", op="rope", dt="bf16", B=256, lo=1, hi=1, H=32, Hkv=8, D=128, rd=128,
             inter=False, page=64, max_pos=131072),
        # a prefill like the benchmark's: 256 ragged prompts of up to 512 tokens, heads of 64, grouped
        dict(name="rope_prefill_256", op="rope", dt="bf16", B=256, lo=1, hi=512, H=16, Hkv=8, D=64, rd=64,
             inter=False, page=64, max_pos=2048),
        # neighbouring pairs rotated, half of each head only, odd token counts, 32-bit, no cache
        dict(name="rope_partial_f32", op="rope", dt="f32", B=3, lo=100, hi=1001, H=12, Hkv=3, D=96, rd=48,
             inter=True, page=-1, max_pos=1024),
        # --- attention over a shared prefix and each request's own tokens ---
        # a few requests behind a short system prompt (the smallest: latency)
        dict(name="attn_decode_4", op="attn", dt="f16", B=4, H=8, Hkv=8, D=64, P=500, lo=1, hi=60, rows=0, page=0),
        # the benchmark's batch and heads behind a 2048-token prompt, paged
        dict(name="attn_decode_256", op="attn", dt="bf16", B=256, H=16, Hkv=16, D=64, P=2048, lo=1, hi=639, rows=0,
             page=64),
        # a long document asked about by 32 requests: the prefix is the traffic
        dict(name="attn_decode_long", op="attn", dt="bf16", B=32, H=32, Hkv=8, D=128, P=32768, lo=0, hi=511, rows=0,
             page=256),
        # many requests with 8 query heads a KV head and a prefix of odd length: the products bound it
        dict(name="attn_decode_512_wide", op="attn", dt="f16", B=512, H=32, Hkv=4, D=128, P=8191, lo=1, hi=127,
             rows=0, page=0),
        # the prompts' own tokens prefilled behind the shared prompt, as rows of ragged sequences
        dict(name="attn_prefill_rows", op="attn", dt="bf16", B=48, H=16, Hkv=8, D=64, P=4096, lo=1, hi=255, rows=1,
             page=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15


def draw(rng):
    largest = {}
    for c in listed():
        largest[c["op"]] = max(largest.get(c["op"], 0.0), _cost(c))
    while True:
        op = rng.choice(["plan", "rope", "attn", "attn"])
        if op == "plan":
            prefill = rng.random() < 0.6
            c = dict(op=op, B=_log_int(rng, 1, 5000), kv_lo=0, kv_hi=_log_int(rng, 1, 4000), new_lo=0 if prefill else 1,
                     new_hi=_log_int(rng, 2, 1024) if prefill else 1, page=rng.choice([16, 64, 128, 256]),
                     rpt=rng.choice([0, 1, 2, 3, 8, 16]))
        elif op == "rope":
            D = rng.choice([32, 64, 80, 96, 128, 256])
            hkv = rng.choice([1, 2, 3, 4, 8, 16])
            c = dict(op=op, dt=rng.choice(["bf16", "f16", "f32"]), B=_log_int(rng, 1, 300), lo=1,
                     hi=rng.choice([1, 1, 7, 100, 500]), H=hkv * rng.choice([1, 2, 3, 4, 5, 8]), Hkv=hkv, D=D,
                     rd=rng.choice([D, D, D // 2]), inter=rng.random() < 0.4, page=rng.choice([-1, 0, 64, 128]),
                     max_pos=_log_int(rng, 600, 200000))
        else:
            hkv = rng.choice([1, 2, 3, 4, 8, 16])
            rows = 1 if rng.random() < 0.3 else 0
            c = dict(op=op, dt=rng.choice(["bf16", "f16"]), B=_log_int(rng, 1, 600) if not rows else _log_int(rng, 1, 60),
                     H=hkv * rng.choice([1, 2, 3, 4, 5, 8, 16]), Hkv=hkv, D=rng.choice([32, 64, 64, 128, 128]),
                     P=_log_int(rng, 1, 40000), lo=rng.choice([0, 1]) if not rows else 1, hi=_log_int(rng, 1, 700),
                     rows=rows, page=rng.choice([0, 0, 64, 128, 256]))
            if c["rows"] and c["hi"] > 255:
                c["hi"] = 255
        if _cost(c) > largest[op]:
            continue
        if op == "attn":
            # the plain form keeps every score of the batch in 32 bits
            rows = sum(_lens(c, 0)) if c["rows"] else c["B"]
            if rows * c["H"] * (c["P"] + c["hi"]) > 6e8 or c["B"] * c["Hkv"] * c["hi"] * c["D"] > 3e8:
                continue
        return c


def _spread(n, lo, hi, salt):
    """n whole numbers of [lo, hi], the same ones for every seed (their order is the seed's)."""
    r = np.random.default_rng([n, lo, hi, salt])
    return r.integers(lo, hi + 1, size=n)


def _lens(case, seed):
    key = ("new_lo", "new_hi") if case["op"] == "plan" else ("lo", "hi")
    v = _spread(case["B"], case[key[0]], case[key[1]], 1)
    return np.random.default_rng(seed + 1).permutation(v)


def work(case):
    op = case["op"]
    lens = _lens(case, 0).astype(np.int64)
    if op == "plan":
        rows = int(lens.sum())
        blocks = rows / case["page"]
        tiles = int(sum(-(-int(x) // case["rpt"]) for x in lens)) if case["rpt"] else 0
        # two lengths in, the row offsets out; a table entry a new page (id in, entry out); per row its
        # sequence, position, slot and length; three numbers a tile
        return {"bytes": case["B"] * 12 + blocks * 8 + rows * 20 + tiles * 12, "flops": rows * 4}
    e = 4 if case["dt"] == "f32" else 2
    if op == "rope":
        T = int(lens.sum())
        H, Hkv, D, rd = case["H"], case["Hkv"], case["D"], case["rd"]
        vh = Hkv if case["page"] >= 0 else 0
        # a row's table entry is shared by its heads; far-apart positions each read their own
        return {"bytes": T * (2 * (H + Hkv + vh) * D * e + rd * 4 + 4 + (8 if vh else 0)) + 2 * D * e,
                "flops": T * (H + Hkv) * D * 8}
    B, H, Hkv, D, P = case["B"], case["H"], case["Hkv"], case["D"], case["P"]
    if case["rows"]:
        rows, pairs = int(lens.sum()), int((lens * (lens + 1) // 2).sum())
    else:
        rows, pairs = B, int(lens.sum())
    kv = (P + int(lens.sum())) * Hkv * D * 2 * e
    table = 4 * int(sum(-(-int(x) // case["page"]) for x in lens) + -(-P // case["page"])) if case["page"] else 0
    return {"bytes": kv + 2 * rows * H * D * e + rows * 4 + table, "flops": 4 * H * D * (rows * P + pairs)}


# --------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


def _randn(g, *shape, dtype):
    return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32).to(dtype)


def _pages(lens, page, rng, extra=3):
    """Scattered blocks for sequences of these lengths: (table, number of blocks of the pool)."""
    need = [-(-int(x) // page) for x in lens]
    n_blocks = 1 + sum(need) + extra
    order = rng.permutation(np.arange(1, n_blocks))
    table = np.zeros((len(lens), max(1, max(need))), np.int64)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, n_blocks, order[at:]


def prepare(case, seed):
    op = case["op"]
    rng = np.random.default_rng(seed)
    lens = _lens(case, seed).astype(np.int64)
    st = {"case": case}
    if op == "plan":
        B, page = case["B"], case["page"]
        kv = rng.integers(case["kv_lo"], case["kv_hi"] + 1, size=B)
        width = -(-(case["kv_hi"] + case["new_hi"]) // page) + 1
        table, n_blocks, _ = _pages(kv, page, rng)
        bt = np.zeros((B, width), np.int64)
        bt[:, :table.shape[1]] = table[:, :width]
        total = int(lens.sum())
        free = n_blocks + rng.permutation(np.arange(total // page + B + 8))
        st.update(table=_i32(bt), kv_lens=_i32(kv), new_lens=_i32(lens), free=_i32(free), cursor=_i32(np.array([3])),
                  n_rows=total,
                  n_tiles=int(sum(-(-int(x) // case["rpt"]) for x in lens)) if case["rpt"] else 0)
        return st
    g = _gen(seed)
    dt = DTYPES[case["dt"]]
    if op == "rope":
        H, Hkv, D, rd = case["H"], case["Hkv"], case["D"], case["rd"]
        T = int(lens.sum())
        qkv = _randn(g, T, (H + 2 * Hkv) * D, dtype=dt)
        inv = 10000.0 ** (-torch.arange(0, rd, 2, device="cuda", dtype=torch.float64) / rd)
        ang = torch.arange(case["max_pos"], device="cuda", dtype=torch.float64)[:, None] * inv[None, :]
        st["table"] = torch.cat([ang.cos(), ang.sin()], dim=1).float()
        if case["hi"] == 1:     # a decode step: each request at its own position
            pos = rng.integers(0, case["max_pos"], size=T)
        else:
            pos = np.concatenate([np.arange(n) for n in lens]) % case["max_pos"]
        st.update(q=qkv[:, :H * D].view(T, H, D), k=qkv[:, H * D:(H + Hkv) * D].view(T, Hkv, D),
                  v=qkv[:, (H + Hkv) * D:].view(T, Hkv, D), pos=_i32(pos),
                  qw=(1 + 0.1 * _randn(g, D, dtype=torch.float32)).to(dt),
                  kw=(1 + 0.1 * _randn(g, D, dtype=torch.float32)).to(dt))
        if case["page"] >= 0:
            within = np.concatenate([np.arange(n) for n in lens])
            seqs = np.repeat(np.arange(len(lens)), lens)
            if case["page"] == 0:
                cap = max(64, int(lens.max()))
                n, slots = len(lens), seqs * cap + within
            else:
                cap = case["page"]
                bt, n, _ = _pages(lens, cap, rng)
                slots = bt[seqs, within // cap] * cap + within % cap
            st.update(slots=torch.from_numpy(slots.astype(np.int64)).cuda(),
                      kc=_randn(g, n, Hkv, cap, D, dtype=dt), vc=_randn(g, n, Hkv, cap, D, dtype=dt))
        return st
    B, H, Hkv, D, P, page = case["B"], case["H"], case["Hkv"], case["D"], case["P"], case["page"]
    rows = int(lens.sum()) if case["rows"] else B
    st["q"] = _randn(g, rows, H, D, dtype=dt)
    if page:
        table, n_blocks, rest = _pages(lens, page, rng, extra=-(-P // page) + 2)
        kc, vc = (_randn(g, n_blocks, Hkv, page, D, dtype=dt) for _ in range(2))
        st.update(kc=kc, vc=vc, kp=kc, vp=vc, bt=_i32(table), pblocks=_i32(rest[:-(-P // page)]))
    else:
        cap = -(-max(1, int(lens.max())) // 64) * 64
        st.update(kc=_randn(g, B, Hkv, cap, D, dtype=dt), vc=_randn(g, B, Hkv, cap, D, dtype=dt),
                  kp=_randn(g, Hkv, P, D, dtype=dt), vp=_randn(g, Hkv, P, D, dtype=dt), bt=None, pblocks=None)
    if case["rows"]:
        starts = np.cumsum(lens) - lens
        rpt = 16 // (H // Hkv)
        tiles = [(starts[s] + i, min(rpt, lens[s] - i), s) for s in range(B) for i in range(0, int(lens[s]), rpt)]
        st["tiles"] = _i32(np.array(tiles))
        st["lens"] = _i32(np.concatenate([np.arange(1, n + 1) for n in lens]))
        st["seq_lens"] = [int(x) for x in lens]
    else:
        st["tiles"] = None
        st["lens"] = _i32(lens)
    st["max_len"] = int(lens.max())
    return st


# --------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------
def run(state):
    return {"plan": _run_plan, "rope": _run_rope, "attn": _run_attn}[state["case"]["op"]](state)


def _run_plan(st):
    c = st["case"]
    page, rpt = c["page"], c["rpt"]
    if own:
        from detkernels_b200.kernels.paging import paged_plan
        p = paged_plan(st["table"], st["kv_lens"], st["new_lens"], page, free_blocks=st["free"], cursor=st["cursor"],
                       n_rows=st["n_rows"], rows_per_tile=rpt, n_tiles=st["n_tiles"])
        out = [p.block_table, p.cursor, p.cu_rows, p.row_seq, p.row_pos, p.slots, p.q_lens]
        return out + [p.row_tiles] if rpt else out
    table, kv, new = st["table"], st["kv_lens"].long(), st["new_lens"].long()
    dev, B = table.device, table.shape[0]
    have = (kv + page - 1) // page
    need = (kv + new + page - 1) // page
    take = need - have
    first = st["cursor"].long() + torch.cumsum(take, 0) - take
    col = torch.arange(table.shape[1], device=dev)[None, :]
    fresh = (col >= have[:, None]) & (col < need[:, None])
    idx = (first[:, None] + col - have[:, None]).clamp(0, st["free"].numel() - 1)
    table.copy_(torch.where(fresh, st["free"][idx], table))
    cu = torch.zeros(B + 1, dtype=torch.int32, device=dev)
    cu[1:] = torch.cumsum(new, 0)
    n = st["n_rows"]
    seq = torch.repeat_interleave(torch.arange(B, device=dev), new, output_size=n)
    pos = kv[seq] + torch.arange(n, device=dev) - cu[seq].long()
    slots = table[seq, pos // page].long() * page + pos % page
    out = [table, (st["cursor"].long() + take.sum()).int(), cu, seq.int(), pos.int(), slots, (pos + 1).int()]
    if rpt:
        nt = (new + rpt - 1) // rpt
        ts = torch.repeat_interleave(torch.arange(B, device=dev), nt, output_size=st["n_tiles"])
        at = (torch.arange(st["n_tiles"], device=dev) - (torch.cumsum(nt, 0) - nt)[ts]) * rpt
        out.append(torch.stack([cu[ts].long() + at, torch.minimum(new[ts] - at, torch.full_like(at, rpt)), ts], 1).int())
    return out


def _norm_rotate(x, w, pos, table, inter, math_t):
    """RMS norm of each head, then the rotation of its first columns by the row's angles."""
    x = x.to(math_t)
    y = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * w.to(math_t)
    rd = table.shape[1]
    cs = table[pos].to(math_t)
    cos, sin = cs[:, None, :rd // 2], cs[:, None, rd // 2:]
    r = y[..., :rd]
    a, b = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., :rd // 2], r[..., rd // 2:])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    r = torch.stack([ra, rb], dim=-1).flatten(-2) if inter else torch.cat([ra, rb], dim=-1)
    return torch.cat([r, y[..., rd:]], dim=-1)


def _run_rope(st):
    c = st["case"]
    cached = c["page"] >= 0
    if own:
        from detkernels_b200.kernels.rope import qk_norm_rope
        if cached:
            q, _ = qk_norm_rope(st["q"], st["k"], st["pos"], st["qw"], st["kw"], st["table"], EPS,
                                interleaved=c["inter"], v=st["v"], k_cache=st["kc"], v_cache=st["vc"],
                                slots=st["slots"])
            return [q, st["kc"], st["vc"]]
        return list(qk_norm_rope(st["q"], st["k"], st["pos"], st["qw"], st["kw"], st["table"], EPS,
                                 interleaved=c["inter"]))
    dt = st["q"].dtype
    q, k = (_norm_rotate(x, w, st["pos"], st["table"], c["inter"], torch.float32).to(dt)
            for x, w in ((st["q"], st["qw"]), (st["k"], st["kw"])))
    if not cached:
        return [q, k]
    cap = st["kc"].shape[2]
    n, t = st["slots"] // cap, st["slots"] % cap
    st["kc"][n, :, t] = k
    st["vc"][n, :, t] = st["v"]
    return [q, st["kc"], st["vc"]]


def _seq_kv(cache, bt, s, n):
    """The first n tokens of sequence s: [Hkv, n, D]."""
    if bt is None:
        return cache[s, :, :n]
    page = cache.shape[2]
    b = cache[bt[s, :-(-n // page)].long()]                 # [pages, Hkv, page, D]
    return b.transpose(0, 1).reshape(cache.shape[1], -1, cache.shape[3])[:, :n]


def _prefix_kv(st, name, P):
    if st["pblocks"] is None:
        return st[name]
    b = st[name][st["pblocks"].long()]
    return b.transpose(0, 1).reshape(b.shape[1], -1, b.shape[3])[:, :P]


def _attn_plain(st, math_t):
    c = st["case"]
    H, Hkv, D, P = c["H"], c["Hkv"], c["D"], c["P"]
    G = H // Hkv
    scale = 1.0 / math.sqrt(D)
    q = st["q"].to(math_t)
    R = q.shape[0]
    qg = q.view(R, Hkv, G, D).permute(1, 0, 2, 3).reshape(Hkv, R * G, D)
    sp = torch.matmul(qg, _prefix_kv(st, "kp", P).to(math_t).transpose(1, 2)) * scale       # [Hkv, R G, P]
    vp = _prefix_kv(st, "vp", P).to(math_t)
    if c["rows"]:
        out = torch.empty(Hkv, R * G, D, dtype=math_t, device=q.device)
        at = 0
        for s, n in enumerate(st["seq_lens"]):
            sl = slice(at * G, (at + n) * G)
            at += n
            ks, vs = (_seq_kv(st[x], st["bt"], s, n).to(math_t) for x in ("kc", "vc"))
            ss = torch.matmul(qg[:, sl], ks.transpose(1, 2)) * scale
            row = torch.arange(n * G, device=q.device)[:, None] // G
            ss = torch.where(torch.arange(n, device=q.device)[None, :] <= row, ss, -math.inf)
            m = torch.maximum(sp[:, sl].amax(-1, keepdim=True), ss.amax(-1, keepdim=True))
            pp, ps = torch.exp(sp[:, sl] - m), torch.exp(ss - m)
            out[:, sl] = (torch.matmul(pp, vp) + torch.matmul(ps, vs)) / (pp.sum(-1, keepdim=True) +
                                                                          ps.sum(-1, keepdim=True))
        return out.view(Hkv, R, G, D).permute(1, 0, 2, 3).reshape(R, H, D)
    n = max(1, st["max_len"])
    if st["bt"] is None:
        ks, vs = (st[x][:, :, :n].to(math_t) for x in ("kc", "vc"))
    else:
        page = st["kc"].shape[2]
        ids = st["bt"][:, :-(-n // page)].long()
        ks, vs = (st[x][ids].transpose(1, 2).reshape(R, Hkv, -1, D)[:, :, :n].to(math_t) for x in ("kc", "vc"))
    ss = torch.matmul(q.view(R, Hkv, G, D), ks.transpose(2, 3)) * scale                      # [R, Hkv, G, n]
    valid = torch.arange(n, device=q.device)[None, :] < st["lens"][:, None]
    ss = torch.where(valid[:, None, None, :], ss, -math.inf).permute(1, 0, 2, 3)             # [Hkv, R, G, n]
    sp = sp.view(Hkv, R, G, P)
    m = torch.maximum(sp.amax(-1, keepdim=True), ss.amax(-1, keepdim=True))
    pp, ps = torch.exp(sp - m), torch.exp(ss - m)
    num = torch.matmul(pp.reshape(Hkv, R * G, P), vp).view(Hkv, R, G, D)
    num = num + torch.matmul(ps.permute(1, 0, 2, 3), vs).permute(1, 0, 2, 3)
    out = num / (pp.sum(-1, keepdim=True) + ps.sum(-1, keepdim=True))
    return out.permute(1, 0, 2, 3).reshape(R, H, D)


def _run_attn(st):
    if own:
        from detkernels_b200.kernels.attention import attention_shared_prefix
        return attention_shared_prefix(st["q"], st["kp"], st["vp"], st["kc"], st["vc"], st["lens"],
                                       prefix_len=st["case"]["P"], prefix_blocks=st["pblocks"],
                                       block_table=st["bt"], row_tiles=st["tiles"], max_kv_len=st["max_len"])
    return _attn_plain(st, torch.float32).to(st["q"].dtype)


# --------------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "plan":
        return _exact_plan(st)
    if case["op"] == "rope":
        return _exact_rope(st)
    return _exact_attn(st)


def _exact_plan(st):
    """Sequence by sequence on the host: the definition read aloud."""
    c = st["case"]
    page, rpt = c["page"], c["rpt"]
    table = st["table"].cpu().numpy().copy()
    kv, new, free = (st[x].cpu().numpy().astype(np.int64) for x in ("kv_lens", "new_lens", "free"))
    cursor = int(st["cursor"])
    seq, pos, slots, tiles, cu = [], [], [], [], [0]
    for b in range(len(kv)):
        have, need = -(-kv[b] // page), -(-(kv[b] + new[b]) // page)
        table[b, have:need] = free[cursor:cursor + need - have]
        cursor += int(need - have)
        p = np.arange(kv[b], kv[b] + new[b])
        seq.append(np.full(new[b], b))
        pos.append(p)
        slots.append(table[b, p // page].astype(np.int64) * page + p % page)
        if rpt:
            tiles += [(cu[-1] + i, min(rpt, new[b] - i), b) for i in range(0, int(new[b]), rpt)]
        cu.append(cu[-1] + int(new[b]))
    pos = np.concatenate(pos)
    out = [_i32(table), _i32(np.array([cursor])), _i32(np.array(cu)), _i32(np.concatenate(seq)), _i32(pos),
           torch.from_numpy(np.concatenate(slots)).cuda(), _i32(pos + 1)]
    return out + [_i32(np.array(tiles).reshape(-1, 3))] if rpt else out


def _exact_rope(st):
    c = st["case"]
    rd = c["rd"]
    cs = st["table"].double()[st["pos"].long()]
    half = rd // 2
    z = torch.complex(cs[:, :half], cs[:, half:])[:, None, :]      # the rotation as a unit complex factor
    res = []
    for x, w in ((st["q"], st["qw"]), (st["k"], st["kw"])):
        x = x.double()
        y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()
        r = y[..., :rd]
        if c["inter"]:
            rot = torch.view_as_real(torch.view_as_complex(r.reshape(*r.shape[:-1], half, 2).contiguous()) * z)
            rot = rot.flatten(-2)
        else:
            u = torch.complex(r[..., :half].contiguous(), r[..., half:].contiguous()) * z
            rot = torch.cat([u.real, u.imag], dim=-1)
        res.append(torch.cat([rot, y[..., rd:]], dim=-1))
    if c["page"] < 0:
        return res
    kc, vc = st["kc"].double(), st["vc"].double()
    flat = st["slots"]
    cap = kc.shape[2]
    kc[flat // cap, :, flat % cap] = res[1]
    vc[flat // cap, :, flat % cap] = st["v"].double()
    return [res[0], kc, vc]


def _exact_attn(st):
    """Row by row over [prefix | own tokens] (the rows of one KV head at once where they fit)."""
    c = st["case"]
    H, Hkv, D, P = c["H"], c["Hkv"], c["D"], c["P"]
    G = H // Hkv
    R = st["q"].shape[0]
    if 4.0 * R * H * D * P > 4e11:
        return None
    kp, vp = _prefix_kv(st, "kp", P).double(), _prefix_kv(st, "vp", P).double()
    out = torch.empty(R, H, D, dtype=torch.float64, device=st["q"].device)
    seqs = np.repeat(np.arange(c["B"]), st["seq_lens"]) if c["rows"] else np.arange(c["B"])
    lens = st["lens"].cpu().numpy()
    step = max(1, int(2e8 // (P * H)))
    for r0 in range(0, R, step):        # the prefix part of some rows at a time
        q = st["q"][r0:r0 + step].double()
        n = q.shape[0]
        qh = q.view(n, Hkv, G, D).transpose(0, 1).reshape(Hkv, n * G, D)
        sp = torch.bmm(qh, kp.transpose(1, 2)).mul_(D ** -0.5)
        m = sp.amax(-1)
        p = sp.sub_(m[..., None]).exp_()
        den, num = p.sum(-1), torch.bmm(p, vp)
        for i in range(n):              # joined with the row's own tokens
            L = int(lens[r0 + i])
            a, d, o = (t[:, i * G:(i + 1) * G] for t in (m, den, num))
            if L:
                s = int(seqs[r0 + i])
                ks, vs = (_seq_kv(st[x], st["bt"], s, L).double() for x in ("kc", "vc"))
                ss = torch.bmm(q[i].view(Hkv, G, D), ks.transpose(1, 2)) * D ** -0.5
                t = torch.maximum(a, ss.amax(-1))
                e = torch.exp(ss - t[..., None])
                f = torch.exp(a - t)
                d = d * f + e.sum(-1)
                o = o * f[..., None] + torch.bmm(e, vs)
            out[r0 + i] = (o / d[..., None]).reshape(H, D)
    return out
