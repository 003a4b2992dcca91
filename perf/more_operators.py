"""What is measured of the operators for drafted tokens: attention of a tree of drafts over a KV cache, the log
probabilities of given tokens, the accepted path of a tree, and forking, compacting and freeing the pages of a cache.

``run`` computes each operator with elementary torch operations in 32 bits, or, where ``own`` is
true, through the package's entry points.  ``exact`` gives the same outputs from the definitions in
64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# --------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------
def listed():
    return [
        # --- attention of drafted tokens: t_lo..t_hi nodes a request behind kv_lo..kv_hi cached tokens ---
        # a few requests with short drafts in a contiguous cache (the smallest: latency)
        dict(name="tree_attn_4", op="attn", dt="f16", B=4, t_lo=1, t_hi=6, kv_lo=0, kv_hi=700, H=8, Hkv=8, D=64, page=0),
        # a verification step of a serving batch: trees of up to 32 nodes, grouped heads, paged
        dict(name="tree_attn_64", op="attn", dt="bf16", B=64, t_lo=8, t_hi=32, kv_lo=200, kv_hi=4000, H=32, Hkv=8, D=128,
             page=64),
        # large trees of a few long requests: several hundred query rows a KV head
        dict(name="tree_attn_long", op="attn", dt="f16", B=9, t_lo=40, t_hi=64, kv_lo=8000, kv_hi=20000, H=32, Hkv=4,
             D=128, page=256),
        # --- log probabilities of given tokens over the vocabulary ---
        # one decode step of 8 requests with 20 alternatives each, the benchmark's vocabulary (the smallest: latency)
        dict(name="logprobs_8", op="lp", dt="bf16", R=8, V=32000, k=20),
        # the rows of a verification step in 32 bits, a few alternatives
        dict(name="logprobs_verify", op="lp", dt="f32", R=1531, V=32000, k=5),
        # scoring whole prompts: many rows of an odd vocabulary, whose rows are not aligned; no alternatives
        dict(name="logprobs_score", op="lp", dt="bf16", R=4096, V=50001, k=0),
        # --- the accepted path of each request's tree ---
        # small trees of a few requests (the smallest: latency)
        dict(name="accept_7", op="accept", B=7, t_lo=1, t_hi=24),
        # a large batch of trees of up to 64 nodes
        dict(name="accept_4099", op="accept", B=4099, t_lo=1, t_hi=64),
        # --- forking requests: pages shared or copied ---
        # four samples of each of 7 prompts: whole pages shared, the open page copied (latency)
        dict(name="fork_7x4", op="fork", dt="bf16", B=7, n=4, lo=1, hi=1500, layers=4, Hkv=16, D=64, page=64, shares=True),
        # 24 prompts copied whole, all layers (the traffic of a copy)
        dict(name="fork_copy_24", op="fork", dt="bf16", B=24, n=1, lo=100, hi=3000, layers=4, Hkv=16, D=64, page=64,
             shares=False),
        # --- accepted drafts moved together, the pages behind them given back ---
        # the end of a verification step of 256 requests: a few tokens of each tree are kept
        dict(name="compact_256", op="compact", dt="bf16", B=256, kv_lo=1, kv_hi=600, t_lo=1, t_hi=24, keep=0.2, layers=4,
             Hkv=16, D=64, page=64, shares=True),
        # long caches thinned out to half of their tokens
        dict(name="compact_long", op="compact", dt="f16", B=8, kv_lo=0, kv_hi=64, t_lo=6000, t_hi=16000, keep=0.5, layers=4,
             Hkv=8, D=128, page=128, shares=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.4e12 + w["flops"] / 1.6e15


def draw(rng):
    largest = {}
    for c in listed():
        largest[c["op"]] = max(largest.get(c["op"], 0.0), _cost(c))
    while True:
        op = rng.choice(["attn", "attn", "attn", "lp", "lp", "accept", "fork", "compact"])
        if op == "attn":
            hkv = rng.choice([1, 2, 3, 4, 8, 16])
            kv_hi = _log_int(rng, 1, 20000)
            t_hi = _log_int(rng, 1, 64) if rng.random() < 0.8 else _log_int(rng, 64, 150)
            c = dict(op=op, dt=rng.choice(["bf16", "f16"]), B=_log_int(rng, 1, 128), t_lo=rng.choice([0, 1]) if t_hi < 4 else
                     rng.choice([0, 1, t_hi // 2]), t_hi=t_hi, kv_lo=rng.choice([0, kv_hi // 4, kv_hi]), kv_hi=kv_hi,
                     H=hkv * rng.choice([1, 2, 3, 4, 5, 8, 16]), Hkv=hkv, D=rng.choice([32, 64, 64, 128, 128]),
                     page=rng.choice([0, 0, 64, 128, 256]))
            # the plain form keeps every score and the gathered keys of the batch in 32 bits
            n = c["kv_hi"] + c["t_hi"]
            if c["B"] * c["t_hi"] * c["H"] * n > 8e8 or c["B"] * c["Hkv"] * n * c["D"] > 6e8:
                continue
        elif op == "lp":
            c = dict(op=op, dt=rng.choice(["bf16", "f16", "f32"]), R=_log_int(rng, 1, 5000), V=_log_int(rng, 500, 270000),
                     k=rng.choice([0, 1, 5, 20, 32]))
            if c["R"] * c["V"] > 2.5e8:
                continue
        elif op == "accept":
            c = dict(op=op, B=_log_int(rng, 1, 5000), t_lo=rng.choice([0, 1]), t_hi=_log_int(rng, 1, 150))
        elif op == "fork":
            c = dict(op=op, dt=rng.choice(["bf16", "f16", "f32"]), B=_log_int(rng, 1, 60), n=_log_int(rng, 1, 16),
                     lo=rng.choice([0, 1]), hi=_log_int(rng, 1, 4000), layers=_log_int(rng, 1, 8),
                     Hkv=rng.choice([1, 2, 3, 4, 8, 16]), D=rng.choice([32, 64, 80, 96, 128, 256]),
                     page=rng.choice([16, 64, 128, 256]), shares=rng.random() < 0.6)
        else:
            long = rng.random() < 0.3
            c = dict(op=op, dt=rng.choice(["bf16", "f16", "f32"]), B=_log_int(rng, 1, 30 if long else 500), kv_lo=0,
                     kv_hi=_log_int(rng, 1, 2000), t_lo=rng.choice([0, 1]), t_hi=_log_int(rng, 1, 8000 if long else 64),
                     keep=rng.choice([0.0, 0.1, 0.3, 0.9]), layers=_log_int(rng, 1, 8), Hkv=rng.choice([1, 2, 3, 4, 8, 16]),
                     D=rng.choice([32, 64, 80, 96, 128, 256]), page=rng.choice([16, 64, 128, 256]),
                     shares=rng.random() < 0.5)
        if _cost(c) > largest[op]:
            continue
        if op in ("fork", "compact") and _pool_elements(c) > 1e9:
            continue
        return c


def _spread(n, lo, hi, salt):
    """n whole numbers of [lo, hi], the same ones for every seed (their order is the seed's)."""
    return np.random.default_rng([n, lo, hi, salt]).integers(lo, hi + 1, size=n).astype(np.int64)


def _lens(case, seed):
    """What a case's sequences hold (and, where they have drafts, how many), in the seed's order."""
    r = np.random.default_rng(seed + 1)
    if case["op"] == "fork":
        return r.permutation(_spread(case["B"], case["lo"], case["hi"], 1)), None
    order = r.permutation(case["B"])
    t = _spread(case["B"], case["t_lo"], case["t_hi"], 2)[order]
    if case["op"] == "accept":
        return None, t
    return _spread(case["B"], case["kv_lo"], case["kv_hi"], 3)[order], t


def _kept(case, t):
    """How many of each sequence's t tokens are kept."""
    return np.minimum(t, np.ceil(t * case["keep"]).astype(np.int64))


def _pages(n, page):
    return -(-n // page)


def _pool_elements(case):
    kv, t = _lens(case, 0)
    per = case["Hkv"] * case["D"] * case["page"] * case["layers"] * 2
    if case["op"] == "fork":
        return int(_pages(kv, case["page"]).sum() * (1 + case["n"])) * per
    return int(_pages(kv + t, case["page"]).sum()) * per


def work(case):
    op = case["op"]
    e = 4 if case.get("dt") == "f32" else 2
    if op == "lp":
        R, V, k = case["R"], case["V"], case["k"]
        return {"bytes": R * V * e + R * (8 + 4 + 4 + k * 12), "flops": 6 * R * V}
    kv, t = _lens(case, 0)
    if op == "attn":
        H, Hkv, D = case["H"], case["Hkv"], case["D"]
        live = t > 0
        tokens = int(((kv + t) * live).sum())
        rows = int(t.sum())
        table = 4 * int(_pages((kv + t) * live, case["page"]).sum()) if case["page"] else 0
        return {"bytes": tokens * Hkv * D * 2 * e + 2 * rows * H * D * e + rows * 8 * _words(case) + 12 * case["B"] + table,
                "flops": 4 * H * D * int((t * (kv + t)).sum())}
    if op == "accept":
        rows = int(t.sum())
        # each node's parent, token and pick; the path, its length and the next token a request
        return {"bytes": rows * 20 + case["B"] * (4 + 4 + 8) + 4 * case["B"] * _max_keep(case), "flops": rows}
    row = case["layers"] * 2 * case["Hkv"] * case["D"] * e
    if op == "fork":
        n, page = case["n"], case["page"]
        copied = int((kv % page if case["shares"] else kv).sum()) * n
        entries = int(_pages(kv, page).sum()) * n
        return {"bytes": copied * row * 2 + entries * (16 if case["shares"] else 12) + case["B"] * n * 16,
                "flops": entries}
    kept = _kept(case, t)
    back = int((_pages(kv + t, case["page"]) - _pages(kv + kept, case["page"])).sum())
    # kept tokens that already lie at their place need no copy: the path's first tokens mostly do not move
    moved = int(np.where(kept < t, kept, 0).sum())
    return {"bytes": moved * row * 2 + int(kept.sum()) * 4 + case["B"] * 16 + back * 16, "flops": moved}


# --------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _dev(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a).astype(dtype)).cuda()


def _randn(g, *shape, dtype):
    out = torch.empty(*shape, device="cuda", dtype=dtype)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 28):      # in pieces: a whole cache in 32 bits would not be small
        n = min(1 << 28, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, device="cuda", generator=g, dtype=torch.float32).to(dtype)
    return out


def _words(case):
    return max(1, _pages(case["t_hi"], 64))


def _max_keep(case):
    return min(case["t_hi"], 24) if case["t_hi"] else 1


def _trees(rng, t):
    """Parents of each sequence's nodes (node 0 the root), in the order of a drafter that extends recent nodes."""
    n = int(t.sum())
    at = np.arange(n) - np.repeat(np.cumsum(t) - t, t)
    back = 1 + np.minimum(rng.integers(0, 8, size=n), np.maximum(at - 1, 0))
    return np.where(at == 0, -1, at - back), at


def _masks(parents, at, words):
    """Bit j of a node's words: j is the node or one of its ancestors."""
    n = len(parents)
    mask = np.zeros((n, words), np.uint64)
    mask[np.arange(n), at // 64] = np.uint64(1) << (at % 64).astype(np.uint64)
    up = np.where(parents < 0, np.arange(n), np.arange(n) - at + parents)
    for _ in range(max(1, int(at.max(initial=0))).bit_length()):
        mask |= mask[up]
        up = up[up]
    return mask.view(np.int64)


def _table(lens, page, rng, extra=0, reserved=1, rows=None, width=None):
    """Scattered blocks for sequences of these lengths: (table, blocks in all, the blocks left over)."""
    need = _pages(np.asarray(lens), page)
    n_blocks = reserved + int(need.sum()) + extra
    order = rng.permutation(np.arange(reserved, n_blocks))
    table = np.zeros((rows or len(lens), width or max(1, int(need.max(initial=0)))), np.int64)
    first = np.cumsum(need) - need
    seq = np.repeat(np.arange(len(lens)), need)
    col = np.arange(int(need.sum())) - np.repeat(first, need)
    table[seq, col] = order[:len(seq)]
    return table, n_blocks, order[len(seq):]


def prepare(case, seed):
    op = case["op"]
    rng = np.random.default_rng(seed)
    g = _gen(seed)
    st = {"case": case}
    if op == "lp":
        R, V = case["R"], case["V"]
        dt = DTYPES[case["dt"]]
        x = torch.empty(R, V, device="cuda", dtype=dt)
        for i in range(0, R, 256):      # a broad spread and, in each row, a few likely tokens
            y = torch.randn(min(256, R - i), V, device="cuda", generator=g) * 2.2
            hot = torch.randint(0, V, (y.shape[0], 6), device="cuda", generator=g)
            y.scatter_add_(1, hot, torch.rand(hot.shape, device="cuda", generator=g) * 14)
            x[i:i + 256] = y.to(dt)
            if i == 0:
                likely = hot[:, 0]
        tokens = torch.randint(0, V, (R,), device="cuda", generator=g)
        tokens[:likely.numel()] = torch.where(tokens[:likely.numel()] % 2 == 0, likely, tokens[:likely.numel()])
        st.update(x=x, tokens=tokens)
        return st
    kv, t = _lens(case, seed)
    if op == "accept":
        parents, at = _trees(rng, t)
        n = len(parents)
        tokens = rng.integers(0, 32000, size=n)
        picked = rng.integers(0, 32000, size=n)
        # the model agrees with most nodes' last child (later children overwrite earlier ones)
        kids = np.nonzero((parents >= 0) & (rng.random(n) < 0.8))[0]
        picked[(kids - at[kids] + parents[kids])] = tokens[kids]
        st.update(parents=_dev(parents), tokens=_dev(tokens, np.int64), picked=_dev(picked, np.int64),
                  cu=_dev(np.concatenate([[0], np.cumsum(t)])))
        return st
    dt = DTYPES[case["dt"]]
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    if op == "attn":
        H, W = case["H"], _words(case)
        rows = int(t.sum())
        parents, at = _trees(rng, t)
        st.update(q=_randn(g, rows, H, D, dtype=dt), kv=_dev(kv), cu=_dev(np.concatenate([[0], np.cumsum(t)])),
                  mask=torch.from_numpy(_masks(parents, at, W) if rows else np.zeros((0, W), np.int64)).cuda(),
                  max_len=int((kv + t).max()), max_rows=int(t.max()), seq=_dev(np.repeat(np.arange(len(t)), t), np.int64),
                  at=_dev(at, np.int64), lens=[(int(a), int(b)) for a, b in zip(kv, t)])
        if page:
            table, n, _ = _table(kv + t, page, rng)
            st.update(kc=_randn(g, n, Hkv, page, D, dtype=dt), vc=_randn(g, n, Hkv, page, D, dtype=dt), bt=_dev(table))
        else:
            cap = max(64, _pages(int((kv + t).max()), 64) * 64)
            st.update(kc=_randn(g, case["B"], Hkv, cap, D, dtype=dt), vc=_randn(g, case["B"], Hkv, cap, D, dtype=dt),
                      bt=None)
        return st
    if op == "fork":
        B, n = case["B"], case["n"]
        src = np.repeat(np.arange(B), n)
        dst = B + rng.permutation(B * n)
        new = kv[src] % page > 0 if case["shares"] else _pages(kv[src], page)
        table, n_blocks, free = _table(kv, page, rng, extra=int(new.sum()) + 2, rows=B * (1 + n))
        st.update(table=_dev(table), kv=_dev(np.concatenate([kv, np.zeros(B * n, np.int64)])), src=_dev(src), dst=_dev(dst),
                  free=_dev(np.concatenate([[0], free])), cursor=_dev([1]), longest=int(kv.max()),
                  shares=torch.zeros(n_blocks, dtype=torch.int32, device="cuda") if case["shares"] else None)
    else:
        B = case["B"]
        kept = _kept(case, t)
        K = max(1, int(kept.max()))
        keep = np.full((B, K), -1, np.int64)
        for b in range(B):
            keep[b, :kept[b]] = np.sort(rng.permutation(int(t[b]))[:kept[b]])
        table, n_blocks, _ = _table(kv + t, page, rng)
        handed = int(_pages(kv + t, page).sum())
        shares = torch.zeros(n_blocks, dtype=torch.int32, device="cuda") if case["shares"] else None
        st.update(table=_dev(table), kv=_dev(kv), new=_dev(t), keep=_dev(keep), n_keep=_dev(kept),
                  free=torch.zeros(handed + 4, dtype=torch.int32, device="cuda"), cursor=_dev([handed]), shares=shares)
    st["pools"] = [_randn(g, n_blocks, Hkv, page, D, dtype=dt) for _ in range(2 * case["layers"])]
    return st


# --------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------
def run(state):
    return {"attn": _run_attn, "lp": _run_lp, "accept": _run_accept, "fork": _run_fork,
            "compact": _run_compact}[state["case"]["op"]](state)


def _run_attn(st):
    c = st["case"]
    if own:
        from detkernels_b200.kernels.attention import attention_tree
        return attention_tree(st["q"], st["kc"], st["vc"], st["kv"], st["cu"], st["mask"], block_table=st["bt"],
                              max_kv_len=st["max_len"], max_rows=st["max_rows"])
    B, H, Hkv, D = c["B"], c["H"], c["Hkv"], c["D"]
    G, T, n = H // Hkv, st["max_rows"], max(1, st["max_len"])
    q = st["q"].float()
    if q.shape[0] == 0:
        return st["q"].clone()
    # the rows of a sequence side by side, and its keys and values in one run
    qp = torch.zeros(B, T, H, D, device=q.device)
    qp[st["seq"], st["at"]] = q
    if st["bt"] is None:
        ks, vs = (st[x][:, :, :n].float() for x in ("kc", "vc"))
    else:
        ids = st["bt"][:, :_pages(n, c["page"])].long()
        ks, vs = (st[x][ids].transpose(1, 2).reshape(B, Hkv, -1, D)[:, :, :n].float() for x in ("kc", "vc"))
    qp = qp.view(B, T, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, T * G, D)
    s = torch.matmul(qp, ks.transpose(2, 3)) / math.sqrt(D)                     # [B, Hkv, T G, n]
    j = torch.arange(n, device=q.device)[None, None, :] - st["kv"].long()[:, None, None]    # draft of a token, [B, 1, n]
    mask = torch.zeros(B, T, st["mask"].shape[1], dtype=torch.int64, device=q.device)
    mask[st["seq"], st["at"]] = st["mask"]
    word = mask.gather(2, (j.clamp(min=0) // 64).clamp(max=mask.shape[2] - 1).expand(B, T, n))
    t = (st["cu"][1:] - st["cu"][:-1]).long()[:, None, None]
    sees = (j < 0) | ((j < t) & ((word >> (j.clamp(min=0) % 64)) & 1).bool())   # [B, T, n]
    s = torch.where(sees[:, None, :, None, :], s.view(B, Hkv, T, G, n), -math.inf).view(B, Hkv, T * G, n)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    out = torch.matmul(p, vs) / torch.where(l == 0, 1.0, l)
    out = out.view(B, Hkv, T, G, D).permute(0, 2, 1, 3, 4).reshape(B, T, H, D)
    return out[st["seq"], st["at"]].to(st["q"].dtype)


def _rank_key(x):
    """Whole numbers in the order of the values (x: 32-bit, finite)."""
    b = (x + 0.0).contiguous().view(torch.int32).long()
    return torch.where(b < 0, -(b & 0x7fffffff), b)


def _run_lp(st):
    k = st["case"]["k"]
    if own:
        from detkernels_b200.kernels.logprobs import token_logprobs
        r = token_logprobs(st["x"], st["tokens"], top_k=k)
        return [r.logprobs, r.entropy] + ([r.top_ids, r.top_logprobs] if k else [])
    V = st["x"].shape[1]
    outs = []
    for x, tok in zip(st["x"].split(512), st["tokens"].split(512)):     # some rows at a time: 32-bit copies of them
        x = x.float()
        d = x - x.amax(-1, keepdim=True)
        p = torch.exp(d)
        z = p.sum(-1, keepdim=True)
        logz = torch.log(z)
        row = [(d.gather(1, tok[:, None]) - logz)[:, 0], (logz - (p * d).sum(-1, keepdim=True) / z)[:, 0]]
        if k:   # values first, then the lowest index
            key = _rank_key(x) * 2 ** 20 + (V - 1 - torch.arange(V, device=x.device))
            ids = V - 1 - (key.topk(k, dim=1).values & (2 ** 20 - 1))
            row += [ids, d.gather(1, ids) - logz]
        outs.append(row)
    return [torch.cat(o) for o in zip(*outs)]


def _run_accept(st):
    K = _max_keep(st["case"])
    if own:
        from detkernels_b200.kernels.drafts import tree_accept
        r = tree_accept(st["parents"], st["tokens"], st["picked"], st["cu"], max_keep=K)
        return [r.keep, r.n_keep, r.next_tokens]
    cu = st["cu"].long()
    B, R, dev = cu.numel() - 1, st["parents"].numel(), cu.device
    n = cu[1:] - cu[:-1]
    if R == 0:
        return [torch.full((B, K), -1, dtype=torch.int32, device=dev), torch.zeros(B, dtype=torch.int32, device=dev),
                torch.full((B,), -1, dtype=torch.int64, device=dev)]
    row = torch.arange(R, device=dev)
    seq = torch.repeat_interleave(torch.arange(B, device=dev), n, output_size=R)
    at = row - cu[seq]
    par = st["parents"].long()
    follows = (par >= 0) & (st["tokens"] == st["picked"][(cu[seq] + par).clamp(0, R - 1)])
    # each node's first agreeing child
    child = torch.full((R + 1,), R, dtype=torch.int64, device=dev)
    child.scatter_reduce_(0, torch.where(follows, cu[seq] + par, R), torch.where(follows, row, R), "amin")
    child[R] = R
    cur = torch.where(n > 0, cu[:-1], R)
    path = []
    for _ in range(K):
        path.append(cur)
        cur = child[cur]
    path = torch.stack(path, 1)                                       # [B, K]
    live = path < R
    n_keep = live.sum(1)
    at = torch.cat([at, at.new_tensor([-1])])
    last = path.gather(1, (n_keep - 1).clamp(min=0)[:, None])[:, 0]
    picked = torch.cat([st["picked"], st["picked"].new_full((1,), -1)])
    return [at[path].int(), n_keep.int(), picked[last]]


def _run_fork(st):
    c = st["case"]
    page = c["page"]
    if own:
        from detkernels_b200.kernels.paging import paged_fork
        cursor = paged_fork(st["table"], st["kv"], st["src"], st["dst"], page, free_blocks=st["free"], cursor=st["cursor"],
                            pools=st["pools"], shares=st["shares"])
        return [st["table"], st["kv"], cursor] + ([st["shares"]] if c["shares"] else []) + st["pools"]
    table, kv, src, dst = st["table"], st["kv"], st["src"].long(), st["dst"].long()
    n = kv[src].long()
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    held = col < ((n + page - 1) // page)[:, None]
    new = held & (col >= (n // page)[:, None]) if c["shares"] else held      # entries that need a block of their own
    take = new.sum(1)
    first = st["cursor"].long() + torch.cumsum(take, 0) - take
    order = first[:, None] + torch.cumsum(new, 1) - 1
    old = table[src].long()
    rows = torch.where(new, st["free"][order.clamp(0, st["free"].numel() - 1)].long(), old)
    table[dst] = torch.where(held, rows.int(), table[dst])
    kv[dst] = n.int()
    cursor = (st["cursor"].long() + take.sum()).int()
    if c["shares"]:
        st["shares"].index_add_(0, old[held & ~new], torch.ones_like(old[held & ~new], dtype=torch.int32))
    i, j = torch.nonzero(new, as_tuple=True)
    tok = torch.arange(page, device=table.device)
    for a in range(0, i.numel(), 4096):
        ia, ja = i[a:a + 4096], j[a:a + 4096]
        live = tok[None, :] < (n[ia] - ja * page)[:, None]                   # tokens behind the sequence stay
        s, d = old[ia, ja], rows[ia, ja]
        for pool in st["pools"]:
            pool[d] = torch.where(live[:, None, :, None], pool[s], pool[d])
    return [table, kv, cursor] + ([st["shares"]] if c["shares"] else []) + st["pools"]


def _run_compact(st):
    c = st["case"]
    page = c["page"]
    if own:
        from detkernels_b200.kernels.paging import paged_compact
        r = paged_compact(st["table"], st["kv"], st["new"], st["n_keep"], page, keep=st["keep"], pools=st["pools"],
                          free_blocks=st["free"], cursor=st["cursor"], shares=st["shares"])
        return [r.lens, r.cursor, st["free"]] + ([st["shares"]] if c["shares"] else []) + st["pools"]
    table, kv, new, keep, nk = st["table"].long(), st["kv"].long(), st["new"].long(), st["keep"].long(), st["n_keep"].long()
    lens = kv + nk
    b, j = torch.nonzero(torch.arange(keep.shape[1], device=kv.device)[None, :] < nk[:, None], as_tuple=True)
    src, dst = kv[b] + keep[b, j], kv[b] + j
    sb, db = table[b, src // page], table[b, dst // page]
    for pool in st["pools"]:
        pool[db, :, dst % page] = pool[sb, :, src % page].clone()
    lo, hi = (lens + page - 1) // page, (kv + new + page - 1) // page
    col = torch.arange(table.shape[1], device=kv.device)[None, :]
    blocks = table[(col >= lo[:, None]) & (col < hi[:, None])]
    if c["shares"]:     # every page that is given back here has no other holder
        last = st["shares"][blocks] == 0
        st["shares"][blocks] = torch.where(last, 0, st["shares"][blocks] - 1).int()
        blocks = blocks[last]
    cursor = st["cursor"] - blocks.numel()
    st["free"][cursor.long() + torch.arange(blocks.numel(), device=kv.device)] = blocks.int()
    return [lens.int(), cursor.int(), st["free"]] + ([st["shares"]] if c["shares"] else []) + st["pools"]


# --------------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"attn": _exact_attn, "lp": _exact_lp, "accept": _exact_accept, "fork": _exact_fork,
            "compact": _exact_compact}[case["op"]](st)


def _exact_attn(st):
    """Sequence by sequence over its own tokens."""
    c = st["case"]
    H, Hkv, D, page = c["H"], c["Hkv"], c["D"], c["page"]
    G = H // Hkv
    if work(c)["flops"] > 4e11:
        return None
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    bits = np.unpackbits(st["mask"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")    # bit j of the words
    r0 = 0
    for b, (n, t) in enumerate(st["lens"]):
        if t == 0:
            continue
        if st["bt"] is None:
            k, v = (st[x][b, :, :n + t].double() for x in ("kc", "vc"))
        else:
            ids = st["bt"][b, :_pages(n + t, page)].long()
            k, v = (st[x][ids].transpose(0, 1).reshape(Hkv, -1, D)[:, :n + t].double() for x in ("kc", "vc"))
        sees = np.concatenate([np.ones((t, n), bool), bits[r0:r0 + t, :t].astype(bool)], 1)
        hide = torch.from_numpy(~sees).to(k.device)
        q = st["q"][r0:r0 + t].double()
        for h in range(H):
            s = (q[:, h] @ k[h // G].T) * D ** -0.5
            s = s.masked_fill(hide, -math.inf)
            e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
            z = e.sum(-1, keepdim=True)
            out[r0:r0 + t, h] = (e @ v[h // G]) / z.clamp(min=1e-300)
        r0 += t
    return out


def _exact_lp(st):
    k = st["case"]["k"]
    outs = []
    for x, tok in zip(st["x"].split(256), st["tokens"].split(256)):
        lp = torch.log_softmax(x.double(), dim=-1)
        p = lp.exp()
        row = [lp[torch.arange(len(tok), device=tok.device), tok], -(p * lp).sum(-1)]
        if k:
            # stable, so that equal values stay in the order of their indices
            ids = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :k]
            row += [ids, lp.gather(1, ids)]
        outs.append(row)
    return [torch.cat(o) for o in zip(*outs)]


def _exact_accept(st):
    """Request by request on the host: the definition read aloud."""
    K = _max_keep(st["case"])
    par, tok, pick, cu = (st[x].cpu().numpy() for x in ("parents", "tokens", "picked", "cu"))
    keep, n_keep, nxt = [], [], []
    for a, b in zip(cu[:-1], cu[1:]):
        path = [0] if b > a else []
        while path and len(path) < K:
            cur = path[-1]
            kids = [i for i in range(cur + 1, b - a) if par[a + i] == cur and tok[a + i] == pick[a + cur]]
            if not kids:
                break
            path.append(kids[0])
        keep.append(path + [-1] * (K - len(path)))
        n_keep.append(len(path))
        nxt.append(int(pick[a + path[-1]]) if path else -1)
    return [_dev(np.array(keep)), _dev(np.array(n_keep)), _dev(np.array(nxt), np.int64)]


def _exact_fork(st):
    """Fork by fork on the host; the pools' copies block by block."""
    c = st["case"]
    page = c["page"]
    table, kv, src, dst, free = (st[x].cpu().numpy().astype(np.int64) for x in ("table", "kv", "src", "dst", "free"))
    shares = st["shares"].cpu().numpy().copy() if c["shares"] else None
    at = int(st["cursor"])
    pairs = []
    for s, d in zip(src, dst):
        n = kv[s]
        for j in range(_pages(n, page)):
            if c["shares"] and (j + 1) * page <= n:
                table[d, j] = table[s, j]
                shares[table[s, j]] += 1
            else:
                table[d, j] = free[at]
                at += 1
                pairs.append((table[s, j], table[d, j], min(page, n - j * page)))
        kv[d] = n
    pools = [p.clone() for p in st["pools"]]
    for s, d, n in pairs:
        for p in pools:
            p[d, :, :n] = p[s, :, :n]
    return [_dev(table), _dev(kv), _dev([at])] + ([_dev(shares)] if c["shares"] else []) + pools


def _exact_compact(st):
    """Sequence by sequence."""
    c = st["case"]
    page = c["page"]
    table, kv, new, keep, nk = (st[x].cpu().numpy().astype(np.int64) for x in ("table", "kv", "new", "keep", "n_keep"))
    back = []
    pools = [p.clone() for p in st["pools"]]
    for b in range(len(kv)):
        s = kv[b] + keep[b, :nk[b]]
        d = kv[b] + np.arange(nk[b])
        (sb, so, db, do) = (torch.from_numpy(x).cuda() for x in (table[b, s // page], s % page, table[b, d // page], d % page))
        for p in pools:
            p[db, :, do] = p[sb, :, so].clone()
        back += list(table[b, _pages(kv[b] + nk[b], page):_pages(kv[b] + new[b], page)])
    free = st["free"].clone()
    cursor = int(st["cursor"]) - len(back)
    free[cursor:cursor + len(back)] = _dev(np.array(back))
    return [_dev(kv + nk), _dev([cursor]), free] + ([st["shares"].clone()] if c["shares"] else []) + pools
