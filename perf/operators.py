"""Operators of steps that serve many requests at once, and what they are held to.

Three operators: drawing each request's next token with its own temperature, top-k, top-p and min-p from given random numbers;
copying pages of the paged cache (children of a forked sequence, pages moved together); low-rank adapters of many requests beside
a projection that all of them share.  ``run`` computes them in plain torch operations, or, with ``own``, by the framework.

Sizes are those of the repository's benchmark (widths 2048 and 4096, 8 key/value heads of 64 and 128, pages of 64 tokens,
vocabularies of 32000, 128256 and 151936) and odd ones beside them.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ITEM = {"fp16": 2, "bf16": 2, "fp32": 4}


# ------------------------------------------------------------------ the cases
def _sample(name, rows, vocab, kind, spread):
    return dict(name=name, op="sample", rows=rows, vocab=vocab, kind=kind, spread=spread)


def _fork(name, layers, heads, dim, page, dtype, pool, parents, children, state):
    return dict(name=name, op="pages", kind="fork", layers=layers, heads=heads, dim=dim, page=page, dtype=dtype, pool=pool, parents=parents,
                children=children, state=state)


def _compact(name, layers, heads, dim, page, dtype, pages, live, seqs):
    return dict(name=name, op="pages", kind="compact", layers=layers, heads=heads, dim=dim, page=page, dtype=dtype, pages=pages, live=live, seqs=seqs)


def _adapters(name, tokens, seqs, adapters, rank, K, N, dtype):
    """`tokens` rows of `seqs` requests (as many rows as requests: one token each)"""
    return dict(name=name, op="adapters", tokens=tokens, seqs=seqs, adapters=adapters, rank=rank, K=K, N=N, dtype=dtype)


def listed():
    return [
        # one conversation, one token, the usual settings together: latency
        _sample("sample-one", 1, 32000, "all", 3.0),
        # a small batch whose requests all have settings of their own, the greedy one among them
        _sample("sample-mixed-8", 8, 128256, "mixed", 3.0),
        # creative writing: nucleus and min-p over nearly flat rows, where tens of thousands of tokens are kept
        _sample("sample-flat-48", 48, 151936, "nucleus", 1.5),
        # a full batch with settings of their own
        _sample("sample-mixed-256", 256, 128256, "mixed", 3.0),
        # one conversation continued three ways: a pooled-window layer and a recurrent one of a test-sized model
        _fork("fork-small", 1, 2, 24, 16, "fp32", 7, 1, 3, 4096),
        # a batch of prompts, four samples of each: 12 layers of 8 heads of 128 and two recurrent layers
        _fork("fork-batch", 12, 8, 128, 64, "bf16", 16, 16, 3, 65536),
        # a store of 24 layers after hours of serving, pages moved to its front
        _compact("compact-store", 24, 8, 128, 64, "bf16", 320, 200, 24),
        # one token of one request
        _adapters("adapter-one", 1, 1, 4, 8, 2048, 2560, "bf16"),
        # a batch of single tokens, most of them with an adapter of their own
        _adapters("adapter-batch-64", 64, 64, 48, 16, 4096, 6144, "bf16"),
        # a test-sized model in true fp32, odd sizes
        _adapters("adapter-odd-fp32", 33, 9, 5, 10, 184, 520, "fp32"),
        # prompts of a ragged batch that start together
        _adapters("adapter-prompts", 1999, 7, 4, 32, 4096, 4096, "fp16"),
        # a long prompt's chunk over few adapters of a high rank
        _adapters("adapter-prompts-wide", 8192, 16, 6, 64, 4096, 6144, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("sample", "sample", "pages", "adapters", "adapters"))
    if op == "sample":
        vocab = _log(rng, 1000, 152000)
        rows = min(_log(rng, 1, 256), 32_000_000 // vocab)
        return dict(op=op, rows=rows, vocab=vocab, kind=rng.choice(("all", "mixed", "nucleus", "top", "plain")), spread=round(rng.uniform(0.5, 5.0), 3))
    if op == "pages":
        layers, heads, dim, page = rng.randint(1, 24), rng.choice((1, 2, 4, 8)), rng.choice((24, 25, 40, 64, 72, 96, 128, 256)), rng.choice((7, 16, 32, 50, 64, 128))
        dtype = rng.choice(("fp16", "bf16", "fp32"))
        each = 2 * layers * heads * dim * page * ITEM[dtype]
        if rng.random() < 0.5:
            parents, children = _log(rng, 1, 32), rng.randint(1, 7)
            parents = max(1, min(parents, int(1.2e9 / each) // (children + 1)))
            return dict(op=op, kind="fork", layers=layers, heads=heads, dim=dim, page=page, dtype=dtype, pool=rng.choice((0, 0, 3, 16)), parents=parents, children=children,
                        state=rng.choice((0, 1000, 16384, 40001)))
        pages = max(8, min(_log(rng, 16, 600), int(1.6e9 / each)))
        return dict(op=op, kind="compact", layers=layers, heads=heads, dim=dim, page=page, dtype=dtype, pages=pages, live=rng.randint(pages // 4, pages - 2), seqs=rng.randint(1, 33))
    rank = rng.choice((1, 4, 8, 10, 16, 24, 32, 64, 100, 128))
    K, N = _log(rng, 100, 4096), _log(rng, 100, 6144)
    dtype, adapters = rng.choice(("fp16", "bf16", "bf16", "fp32")), _log(rng, 1, 64)
    seqs = _log(rng, 1, 100)
    tokens = seqs if rng.random() < 0.5 else max(seqs, _log(rng, seqs, 8192))
    if tokens > 256:
        adapters = min(adapters, 8)
    return dict(op=op, tokens=tokens, seqs=seqs, adapters=adapters, rank=rank, K=K, N=N, dtype=dtype)


# ------------------------------------------------------------------ inputs
def _settings(kind, rows, vocab, g, dev):
    """temperature, top-k, top-p, min-p of every row"""
    r = torch.rand(4, rows, generator=g, device=dev)
    t, k, p, m = 0.5 + r[0], torch.zeros(rows, dtype=torch.int32, device=dev), torch.ones(rows, device=dev), torch.zeros(rows, device=dev)
    some_k, some_p, some_m = (1 + r[1] * 99).to(torch.int32), 0.8 + 0.19 * r[2], 0.02 + 0.1 * r[3]
    if kind == "all":
        k, p, m = some_k, some_p, some_m
    elif kind == "nucleus":
        p, m = some_p, torch.where(r[3] < 0.5, some_m * 0.02, m)
    elif kind == "top":
        k = (1 + r[1] * min(vocab, 2000)).to(torch.int32)
    elif kind == "mixed":                         # by row: greedy, top-k, nucleus, min-p, all together, none
        at = torch.arange(rows, device=dev) % 6
        t = torch.where(at == 0, 0.0, t)
        k = torch.where((at == 1) | (at == 4), some_k, k)
        p = torch.where((at == 2) | (at == 4), some_p, p)
        m = torch.where((at == 3) | (at == 4), some_m, m)
    return t.float(), k.contiguous(), p.float().contiguous(), m.float().contiguous()


def _lengths(total, parts, g):
    """`parts` lengths of at least one that add up to `total`"""
    cuts = torch.randperm(total - 1, generator=g)[:parts - 1].sort().values + 1 if parts > 1 else torch.zeros(0, dtype=torch.long)
    edges = torch.cat([torch.zeros(1, dtype=torch.long), cuts, torch.tensor([total])])
    return (edges[1:] - edges[:-1]).tolist()


def _pool_rows(tensors, per, row_dims):
    """what the framework's page operators take: one row a pool of address, bytes a page, groups, rows, bytes a row, tokens a row"""
    said = []
    for t in tensors:
        groups, rows, row = (1, 1, t[0].numel()) if row_dims is None else t.shape[1:]
        said.append([t.data_ptr(), t[0].numel() * t.element_size(), groups, rows, row * t.element_size(), per])
    return torch.tensor(said, dtype=torch.int64).reshape(-1, 6)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    c = torch.Generator().manual_seed(seed)
    if case["op"] == "sample":
        rows, V = case["rows"], case["vocab"]
        x = torch.randn(rows, V, generator=g, device=dev) * case["spread"]
        # a few tokens that the model has good reason for, and some that a grammar rules out
        at = torch.randint(0, V, (rows, 8), generator=g, device=dev)
        x.scatter_add_(1, at, 2.0 * case["spread"] * torch.rand(rows, 8, generator=g, device=dev))
        x[1::3] = x[1::3].masked_fill(torch.rand(V, generator=g, device=dev) < 0.1, float("-inf"))
        t, k, p, m = _settings(case["kind"], rows, V, g, dev)
        return dict(case=case, logits=x, temperature=t, top_k=k, top_p=p, min_p=m, uniforms=torch.rand(rows, generator=g, device=dev))
    if case["op"] == "pages":
        return _prepare_pages(case, g, c, dev)
    T, S, R, K, N, dt = case["tokens"], case["adapters"], case["rank"], case["K"], case["N"], DTYPES[case["dtype"]]
    lens = torch.tensor(_lengths(T, case["seqs"], c))
    # one in eight requests runs the base model alone
    of_seq = torch.where(torch.rand(case["seqs"], generator=c) < 0.125, -1, torch.randint(0, S, (case["seqs"],), generator=c))
    rank = torch.where(torch.rand(S, generator=c) < 0.25, max(1, R // 2), R)
    return dict(case=case, base=torch.randn(T, N, generator=g, device=dev), x=torch.randn(T, K, generator=g, device=dev).to(dt),
                a=(torch.randn(S, R, K, generator=g, device=dev) * K ** -0.5).to(dt), b=(torch.randn(S, N, R, generator=g, device=dev) * 0.3 * R ** -0.5).to(dt),
                adapter=torch.repeat_interleave(of_seq, lens).to(torch.int32).to(dev), scale=(0.5 + torch.rand(S, generator=c)).to(dev), rank=rank.to(torch.int32).to(dev))


def _prepare_pages(case, g, c, dev):
    L, G, D, page, dt = case["layers"], case["heads"], case["dim"], case["page"], DTYPES[case["dtype"]]
    bits = torch.int32 if dt == torch.float32 else torch.int16
    top = 1 << (8 * ITEM[case["dtype"]] - 1)
    if case["kind"] == "fork":
        n, kids = case["parents"] * (1 + case["children"]) + 3, case["parents"] * case["children"]
    else:
        n = case["pages"]
    # keys and values of every layer; bits of any kind, since nothing is computed of them
    kv = torch.randint(-top, top, (2 * L, n, G, page, D), generator=g, dtype=bits, device=dev)
    s = dict(case=case, kv=kv, pools=_pool_rows(list(kv), 1, 3), n_pages=n, pooled=None, states=None, table=None)
    order = torch.randperm(n, generator=c)
    if case["kind"] == "fork":
        src = order[:case["parents"]].repeat_interleave(case["children"])
        # the page that the prompt has begun: its children go on in pages of their own
        tokens = torch.randint(1, page + 1, (case["parents"],), generator=c).repeat_interleave(case["children"])
        s["moves"] = torch.stack([src, order[case["parents"]:case["parents"] + kids], tokens], 1).to(torch.int32).to(dev)
        if case["pool"]:
            s["pooled"] = torch.randint(-1 << 31, 1 << 31, (2 * L, n, G, -(-page // case["pool"]), D), generator=g, dtype=torch.int32, device=dev)
            s["pools"] = torch.cat([s["pools"], _pool_rows(list(s["pooled"]), case["pool"], 3)])
        if case["state"]:
            slots = case["parents"] + kids + 2
            s["states"] = torch.randint(-1 << 31, 1 << 31, (2, slots, case["state"]), generator=g, dtype=torch.int32, device=dev)
            s["state_pools"], at = _pool_rows(list(s["states"]), 0, None), torch.randperm(slots, generator=c)
            s["slots"] = torch.stack([at[:case["parents"]].repeat_interleave(case["children"]), at[case["parents"]:case["parents"] + kids],
                                      torch.ones(kids, dtype=torch.long)], 1).to(torch.int32).to(dev)
        return s
    live = order[:case["live"]]
    src, free = live[live >= case["live"]], torch.ones(n, dtype=torch.bool)
    free[live] = False
    dst = torch.arange(n)[free][:src.numel()]                # the free pages at the front are as many as the live ones behind it
    where = torch.arange(n)
    where[src] = dst
    most = -(-case["live"] // case["seqs"])
    table = torch.zeros(case["seqs"], n, dtype=torch.int32)
    for q in range(case["seqs"]):
        own_pages = live[q * most:(q + 1) * most]
        table[q, :own_pages.numel()] = own_pages.to(torch.int32)
    s.update(moves=torch.stack([src, dst, torch.full_like(src, page)], 1).to(torch.int32).to(dev), table=table.to(dev), where=where.to(torch.int32).to(dev))
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if op == "sample":
        return _run_sample(state)
    if op == "pages":
        return _run_pages(state)
    return _run_adapters(state)


def _run_sample(s):
    if own:
        from umbrella_amd.speculation.sampling import sample_rows
        tokens, probs = sample_rows(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return dict(tokens=tokens, probs=probs)
    x = torch.where(s["logits"].isnan(), float("-inf"), s["logits"])
    v, index = torch.sort(x, dim=1, descending=True, stable=True)
    V = v.shape[1]
    t, u = s["temperature"].double()[:, None], s["uniforms"].double()[:, None]
    greedy, k = ~(t > 0), s["top_k"][:, None]
    # 64 bits: the draw is compared with sums over the whole vocabulary, next to whose borders 32 bits choose another token
    w = torch.where(v == v[:, :1], 1.0, torch.exp((v.double() - v[:, :1].double()) / torch.where(greedy, 1.0, t)))
    rank = torch.arange(V, device=x.device)[None]
    w = torch.where(((k <= 0) | (rank < k)) & (v > float("-inf")), w, 0.0)
    upto = w.cumsum(1)
    front = torch.cat([torch.zeros_like(upto[:, :1]), upto[:, :-1]], 1)
    keep = (w > 0) & ((rank == 0) | (~greedy & (front < s["top_p"].double()[:, None] * upto[:, -1:]) & (w >= s["min_p"].double()[:, None])))
    n, mass = keep.sum(1, keepdim=True), torch.where(keep, w, 0.0).sum(1, keepdim=True)
    at = torch.minimum(((upto <= u * mass) & keep).sum(1, keepdim=True), n - 1).clamp(min=0)
    tokens = torch.where(n > 0, index.gather(1, at), -1)
    probs = torch.where(n > 0, w.gather(1, at) / mass, 0.0)
    return dict(tokens=tokens[:, 0].to(torch.int32), probs=probs[:, 0].float())


def _copy_rows(store, moves, per):
    """the first rows of every group of the pages moves[:, 0] to the pages moves[:, 1]; store [pools, pages, groups, rows, row]"""
    src, dst, tokens = moves[:, 0].long(), moves[:, 1].long(), moves[:, 2]
    took = torch.arange(store.shape[3], device=store.device)[None] * per < tokens[:, None]
    store[:, dst] = torch.where(took[None, :, None, :, None], store[:, src], store[:, dst])


def _run_pages(s):
    if own:
        from umbrella_amd.attn.cache import copy_pages
        copy_pages(s["pools"], s["moves"], s["n_pages"], table=s["table"], where=s.get("where"))
        if s["states"] is not None:
            copy_pages(s["state_pools"], s["slots"], s["states"].shape[1])
    else:
        _copy_rows(s["kv"], s["moves"], 1)
        if s["pooled"] is not None:
            _copy_rows(s["pooled"], s["moves"], s["case"]["pool"])
        if s["states"] is not None:
            s["states"][:, s["slots"][:, 1].long()] = s["states"][:, s["slots"][:, 0].long()]
        if s["table"] is not None:
            s["table"].copy_(s["where"][s["table"].long()])
    return {k: s[k] for k in ("kv", "pooled", "states", "table") if s[k] is not None}


def _run_adapters(s):
    if own:
        from umbrella_amd.models.adapters import add_adapters
        return add_adapters(s["base"], s["x"], s["a"], s["b"], s["adapter"], scale=s["scale"], rank=s["rank"])
    S, R, K = s["a"].shape
    T, N = s["base"].shape
    # every row against every adapter, those that are not its own multiplied by nothing
    mine = torch.arange(S, device=s["x"].device)[None] == s["adapter"][:, None]
    low = (s["x"].float() @ s["a"].float().reshape(S * R, K).t()).reshape(T, S, R)
    low = torch.where(mine[:, :, None] & (torch.arange(R, device=low.device)[None] < s["rank"][:, None])[None], low * s["scale"][None, :, None], 0.0)
    return s["base"] + low.reshape(T, S * R) @ s["b"].float().permute(0, 2, 1).reshape(S * R, N)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * 4 + 28), "flops": 2 * case["rows"] * case["vocab"]}
    if case["op"] == "pages":
        whole = 2 * case["layers"] * case["heads"] * case["dim"] * case["page"] * ITEM[case["dtype"]]
        if case["kind"] == "fork":
            kids = case["parents"] * case["children"]
            pooled = 2 * case["layers"] * case["heads"] * -(-case["page"] // case["pool"]) * case["dim"] * 4 if case["pool"] else 0
            return {"bytes": (case["parents"] + kids) * ((whole + pooled) * (case["page"] + 1) // (2 * case["page"]) + 8 * case["state"]), "flops": 0}
        behind = case["live"] * (case["pages"] - case["live"]) / case["pages"]
        return {"bytes": 2 * behind * whole + 8 * case["seqs"] * case["pages"], "flops": 0}
    T, S, R, K, N, e = case["tokens"], min(case["adapters"], case["seqs"]), case["rank"], case["K"], case["N"], ITEM[case["dtype"]]
    return {"bytes": T * (K * e + 8 * N) + S * R * (K + N) * e, "flops": 2 * T * R * (K + N)}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pages":
        return None                               # nothing is computed
    if case["op"] == "adapters":
        out = s["base"].double()
        for a in range(case["adapters"]):
            rows = (s["adapter"] == a).nonzero()[:, 0]
            r = int(s["rank"][a])
            if rows.numel():
                out[rows] += s["scale"][a].double() * ((s["x"][rows].double() @ s["a"][a, :r].double().t().contiguous()) @ s["b"][a, :, :r].double().t().contiguous())
        return out
    probs = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
    for r in range(case["rows"]):
        x = s["logits"][r].double()
        order = torch.argsort(x, descending=True, stable=True)
        order = order[x[order] > float("-inf")]
        if s["top_k"][r] > 0:
            order = order[:int(s["top_k"][r])]
        t = float(s["temperature"][r])
        if not t > 0:
            probs[r] = 1.0
            continue
        p = torch.softmax(x[order] / t, 0)
        front = p.cumsum(0) - p
        n = max(1, min(int((front < float(s["top_p"][r])).sum()), int((p >= float(s["min_p"][r]) * p[0]).sum())))
        p = p[:n] / p[:n].sum()
        at = min(int((p.cumsum(0) <= float(s["uniforms"][r])).sum()), n - 1)
        probs[r] = p[at]
    return dict(tokens=None, probs=probs)
