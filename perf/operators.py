"""Cases of the attention-side and expert-side operators that stand between the projections of one
decode, verify or prompt step, with their plain forms.

- ``rope_append``: rotary positions on q and k, and k and v appended to a paged cache;
- ``tree_attention``: attention of each request's drafted tokens (a tree, a chain, or one token) over
  that cache, with an optional sigmoid output gate;
- ``route``: the router's logits to each token's top-k experts and their weights.

A case's ``op`` names its operator. Head layouts are ``heads`` / ``kv_heads`` / ``dim``: 16 / 2 / 64 is
the per-GPU share of the qkv_gate projection (with its 16 x 64 gate), 32 / 8 / 128 the 6144-row QKV
projection, 64 / 8 / 128 the 10240-row one; 256 experts is the router's output width.
"""

import math

import torch

own = False

LAYOUTS = ((16, 2, 64), (32, 8, 128), (64, 8, 128))
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SPARE_PAGES = 3


def listed():
    return [
        # One decoded token of one request on the qkv_gate share: the launch is the cost.
        {"op": "rope_append", "name": "rope decode 1 token", "tokens": 1, "heads": 16, "kv_heads": 2, "dim": 64, "rotary": 64,
         "interleaved": False, "page": 16, "start": 5001, "factor": 1.0, "pad": 0, "dtype": "bf16"},
        # A verify step's drafted tokens: interleaved pairs over half of each head, padded rows among them.
        {"op": "rope_append", "name": "rope verify 201 tokens", "tokens": 201, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 64,
         "interleaved": True, "page": 32, "start": 777, "factor": 1.0, "pad": 9, "dtype": "fp16"},
        # A prompt of 4096 tokens (the prefill projection's M) stretched to a longer context.
        {"op": "rope_append", "name": "rope prompt 4096 tokens", "tokens": 4096, "heads": 64, "kv_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "page": 64, "start": 28673, "factor": 4.0, "pad": 0, "dtype": "bf16"},
        # One token of one short conversation, with the output gate: latency.
        {"op": "tree_attention", "name": "attention decode 1x700", "requests": 1, "draft": 1, "ragged": False, "context": 700, "heads": 16,
         "kv_heads": 2, "dim": 64, "page": 16, "gate": True, "tree": False, "dtype": "bf16"},
        # A decode batch with contexts of every length up to 4096.
        {"op": "tree_attention", "name": "attention decode 32x4096", "requests": 32, "draft": 1, "ragged": False, "context": 4096, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "gate": False, "tree": False, "dtype": "bf16"},
        # One token over a very long context: the split over the cache carries it.
        {"op": "tree_attention", "name": "attention decode 1x131072", "requests": 1, "draft": 1, "ragged": False, "context": 131072, "heads": 64,
         "kv_heads": 8, "dim": 128, "page": 64, "gate": False, "tree": False, "dtype": "bf16"},
        # Small trees of drafted tokens on the qkv_gate share.
        {"op": "tree_attention", "name": "attention tree 8x16 gated", "requests": 8, "draft": 16, "ragged": False, "context": 4001, "heads": 16,
         "kv_heads": 2, "dim": 64, "page": 16, "gate": True, "tree": True, "dtype": "bf16"},
        # Chains and trees of unequal, odd sizes in one launch, one request with nothing drafted.
        {"op": "tree_attention", "name": "attention ragged 11x13", "requests": 11, "draft": 13, "ragged": True, "context": 2999, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 32, "gate": False, "tree": True, "dtype": "fp16"},
        # Wide trees over long contexts: the largest verify step, bound by the matrix products.
        {"op": "tree_attention", "name": "attention tree 16x64", "requests": 16, "draft": 64, "ragged": False, "context": 8192, "heads": 64,
         "kv_heads": 8, "dim": 128, "page": 64, "gate": False, "tree": True, "dtype": "bf16"},
        # One token's experts: sigmoid scores, a balance bias, 4 of 8 groups.
        {"op": "route", "name": "route 1 token", "tokens": 1, "experts": 256, "top_k": 8, "scoring": "sigmoid", "bias": True, "groups": 8,
         "top_groups": 4, "renormalize": True, "scale": 2.5, "dtype": "fp32"},
        # A verify step with an odd number of experts, softmax scores.
        {"op": "route", "name": "route 255 tokens softmax", "tokens": 255, "experts": 100, "top_k": 6, "scoring": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "renormalize": False, "scale": 1.0, "dtype": "bf16"},
        # A prompt batch of 8192 tokens (the prefill projection's largest M).
        {"op": "route", "name": "route 8192 tokens", "tokens": 8192, "experts": 256, "top_k": 8, "scoring": "sigmoid", "bias": True, "groups": 8,
         "top_groups": 4, "renormalize": True, "scale": 2.5, "dtype": "fp32"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rope_append", "tree_attention", "tree_attention", "route"))
    if op == "route":
        experts = rng.choice((8, 60, 64, 100, 128, 160, 256, 384, 512))
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if experts % g == 0 and experts // g >= 2])
        top_groups = rng.randint(1, groups)
        sigmoid = rng.random() < 0.5
        return {"op": op, "tokens": _log_int(rng, 1, 8192 * 256 // max(256, experts)), "experts": experts,
                "top_k": rng.randint(1, min(12, experts // groups * top_groups)), "scoring": "sigmoid" if sigmoid else "softmax",
                "bias": sigmoid and rng.random() < 0.7, "groups": groups, "top_groups": top_groups, "renormalize": rng.random() < 0.5,
                "scale": rng.choice((1.0, 2.5)), "dtype": rng.choice(("fp32", "fp32", "bf16", "fp16"))}
    heads, kv_heads, dim = rng.choice(LAYOUTS + ((8, 8, 128), (12, 4, 64), (5, 1, 128)))
    page = rng.choice((8, 16, 32, 64, 128))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if op == "rope_append":
        tokens = _log_int(rng, 1, 4096)
        return {"op": op, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rng.choice((dim, dim // 2, dim // 4 + 4)),
                "interleaved": rng.random() < 0.5, "page": page, "start": _log_int(rng, 1, 120000), "factor": rng.choice((1.0, 4.0)),
                "pad": rng.randint(0, tokens // 8), "dtype": dtype}
    draft = rng.choice((1, 1, _log_int(rng, 2, 64), _log_int(rng, 2, 64)))
    requests = _log_int(rng, 1, 64)
    most = min(131072, (131072 * 8 * 128) // (requests * kv_heads * dim), (16 * 64 * 8192 * 64 * 128) // (requests * draft * heads * dim))
    return {"op": op, "requests": requests, "draft": draft, "ragged": draft > 1 and rng.random() < 0.5, "context": _log_int(rng, 1, most),
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "gate": rng.random() < 0.5, "tree": rng.random() < 0.7, "dtype": dtype}


# ---- inputs -------------------------------------------------------------------------------------


def _contexts(case):
    """Context lengths, spread evenly from `context` down to a quarter of it."""
    n, top = case["requests"], case["context"]
    return [top - (b * (top - top // 4)) // max(1, n - 1) for b in range(n)]


def _drafts(case):
    """Drafted tokens of each request: `draft`, or (ragged) from there down to one, the last of three or more with none."""
    n, top = case["requests"], case["draft"]
    if not case["ragged"]:
        return [top] * n
    got = [top - (b * (top - 1)) // max(1, n - 1) for b in range(n)]
    return got[:-1] + [0] if n >= 3 else got


def _rope_inputs(case, gen):
    m, hq, hk, d, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    dtype, rot = TYPES[case["dtype"]], case["rotary"]
    # q, k and v are slices of one projection output, as the QKV projection leaves them.
    qkv = torch.randn((m, (hq + 2 * hk) * d), generator=gen, device="cuda").to(dtype)
    q = qkv[:, :hq * d].view(m, hq, d)
    k = qkv[:, hq * d:(hq + hk) * d].view(m, hk, d)
    v = qkv[:, (hq + hk) * d:].view(m, hk, d)
    pages = (m + page - 1) // page + 1 + SPARE_PAGES
    order = torch.randperm(pages - 1, generator=gen, device="cuda")  # the last page stays free
    at = torch.arange(m, device="cuda") + case["start"] % page
    slots = order[at // page] * page + at % page
    positions = torch.arange(case["start"], case["start"] + m, device="cuda", dtype=torch.int32)
    if case["pad"]:  # rows that a fixed-size step carries without a token
        slots[torch.randperm(m, generator=gen, device="cuda")[:case["pad"]]] = -1
    most = case["start"] + m
    angle = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] / case["factor"] * (
        10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot))
    rope = torch.cat((angle.cos(), angle.sin()), dim=1).float()
    cache = [torch.randn((pages, hk, page, d), generator=gen, device="cuda").to(dtype) for _ in range(2)]
    return {"q": q, "k": k, "v": v, "positions": positions, "slots": slots, "rope": rope, "k_pages": cache[0], "v_pages": cache[1]}


def _tree_bits(drafts, most, tree, seed):
    """Visibility words [tokens, words] of random trees (or chains): bit j of a token's row is set where
    drafted token j of its request is the token itself or one of its ancestors."""
    import numpy as np

    rng = np.random.RandomState(seed % (1 << 31))
    words = (most + 31) // 32
    rows = []
    for t in drafts:
        seen = np.zeros((t, words * 32), np.uint8)
        for i in range(t):
            parent = (rng.randint(-1, i) if tree else i - 1) if i else -1
            if parent >= 0:
                seen[i] = seen[parent]
            seen[i, i] = 1
        rows.append(seen)
    every = np.concatenate(rows)
    return np.packbits(every, axis=1, bitorder="little").view(np.int32).reshape(len(every), words).copy()


def _attention_inputs(case, gen, seed):
    hq, hk, d, page, dtype = case["heads"], case["kv_heads"], case["dim"], case["page"], TYPES[case["dtype"]]
    order = torch.randperm(case["requests"], generator=gen, device="cuda").tolist()
    contexts, drafts = _contexts(case), _drafts(case)
    contexts, drafts = [contexts[b] for b in order], [drafts[b] for b in order]
    starts = [0]
    for t in drafts:
        starts.append(starts[-1] + t)
    n = starts[-1]
    # A token's row of the projection: q, k, v and the gate side by side.
    row = torch.randn((n, (2 * hq + 2 * hk) * d), generator=gen, device="cuda")
    row[:, :hq * d] *= 2.0
    row = row.to(dtype)
    q = row[:, :hq * d].view(n, hq, d)
    gate = row[:, (hq + 2 * hk) * d:].view(n, hq, d) if case["gate"] else None
    need = [(c + t + page - 1) // page for c, t in zip(contexts, drafts)]
    pages = sum(need) + SPARE_PAGES
    perm = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(need), max(need)), dtype=torch.int32, device="cuda")
    used = 0
    for b, c in enumerate(need):
        table[b, :c] = perm[used:used + c]
        used += c
    cache = [torch.randn((pages, hk, page, d), generator=gen, device="cuda", dtype=dtype) for _ in range(2)]
    mask = torch.from_numpy(_tree_bits(drafts, case["draft"], case["tree"], seed)).cuda() if case["draft"] > 1 else None
    return {"q": q, "gate": gate, "k_pages": cache[0], "v_pages": cache[1], "page_table": table,
            "context": torch.tensor(contexts, dtype=torch.int32, device="cuda"),
            "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"), "mask": mask, "draft": case["draft"]}


def _route_inputs(case, gen):
    logits = (1.5 * torch.randn((case["tokens"], case["experts"]), generator=gen, device="cuda")).to(TYPES[case["dtype"]])
    bias = 0.05 * torch.randn(case["experts"], generator=gen, device="cuda") if case["bias"] else None
    return {"logits": logits, "bias": bias}


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "rope_append":
        return _rope_inputs(case, gen)
    if case["op"] == "tree_attention":
        return _attention_inputs(case, gen, seed)
    return _route_inputs(case, gen)


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# ---- one pass -----------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rope_append": _own_rope, "tree_attention": _own_attention, "route": _own_route}[op](state)
    return {"rope_append": _plain_rope, "tree_attention": _plain_attention, "route": _plain_route}[op](state)


def _own_rope(s):
    from muse_bf16_proj_b200.attention import rope_append

    q = rope_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["k_pages"], s["v_pages"], s["rope"],
                    interleaved=s["case"]["interleaved"])
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_attention(s):
    from muse_bf16_proj_b200.attention import tree_attention

    return tree_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["context"], s["starts"], s["draft"],
                          tree_mask=s["mask"], gate=s["gate"])


def _own_route(s):
    from muse_bf16_proj_b200.routing import route

    c = s["case"]
    weights, experts = route(s["logits"], c["top_k"], scoring=c["scoring"], bias=s["bias"], groups=c["groups"], top_groups=c["top_groups"],
                             renormalize=c["renormalize"], scale=c["scale"])
    return {"weights": weights, "experts": experts}


def _rotate(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    turn, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = turn[..., :rot // 2], turn[..., rot // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _plain_rope(s):
    dtype, half = s["q"].dtype, s["rope"].shape[1] // 2
    angle = s["rope"][s["positions"].long()][:, None, :]
    cos, sin = angle[..., :half], angle[..., half:]
    q = _rotate(s["q"].float(), cos, sin, s["case"]["interleaved"]).to(dtype)
    k = _rotate(s["k"].float(), cos, sin, s["case"]["interleaved"]).to(dtype)
    pages, _, page, _ = s["k_pages"].shape
    # A row without a slot puts the free last page's last entry back as it is.
    here = torch.where(s["slots"] < 0, pages * page - 1, s["slots"])
    at, off, keep = here // page, here % page, (s["slots"] < 0)[:, None, None]
    s["k_pages"][at, :, off] = torch.where(keep, s["k_pages"][at, :, off], k)
    s["v_pages"][at, :, off] = torch.where(keep, s["v_pages"][at, :, off], s["v"])
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attention(s):
    q, page = s["q"], s["k_pages"].shape[2]
    n, hq, d = q.shape
    hk, most = s["k_pages"].shape[1], s["draft"]
    batch, length = s["page_table"].shape[0], s["page_table"].shape[1] * page
    at = torch.arange(length, device=q.device)
    # Keys and values in order, [requests, kv heads, length, dim].
    keys, values = (p[s["page_table"].long()].transpose(1, 2).reshape(batch, hk, length, d).float() for p in (s["k_pages"], s["v_pages"]))
    first, drafts = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()
    step = torch.arange(most, device=q.device)
    token = (first[:, None] + step).clamp(max=n - 1)  # [requests, most]
    rows = q[token].float().view(batch, most, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(batch, hk, -1, d)
    scores = torch.matmul(rows, keys.transpose(2, 3)).view(batch, hk, hq // hk, most, length) / math.sqrt(d)
    inner = at[None, :] - s["context"].long()[:, None]  # [requests, length]: which drafted token, if one
    drafted = (inner >= 0) & (inner < drafts[:, None])
    if s["mask"] is None:
        bits = inner[:, None, :] <= step[None, :, None]
    else:
        index = inner.clamp(0, most - 1)[:, None, :].expand(batch, most, length)
        words = s["mask"][token].long()
        bits = (torch.gather(words, 2, index // 32) >> (index % 32)) & 1 == 1
    seen = (inner < 0)[:, None, :] | (drafted[:, None, :] & bits)
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = torch.matmul(p.view(batch, hk, -1, length), values)
    out = out.view(batch, hk, hq // hk, most, d).permute(0, 3, 1, 2, 4).reshape(batch * most, hq, d)
    # Back to one row for each token: row t of request b is its token starts[b] + t.
    owner = torch.bucketize(torch.arange(n, device=q.device), s["starts"][1:].long(), right=True)
    out = out[owner * most + torch.arange(n, device=q.device) - first[owner]]
    if s["gate"] is not None:
        out = out / (1.0 + torch.exp(-s["gate"].float()))
    return out.to(q.dtype)


def _plain_route(s):
    c = s["case"]
    x = s["logits"].float()
    m, e = x.shape
    if c["scoring"] == "softmax":
        raised = torch.exp(x - x.amax(-1, keepdim=True))
        scores = raised / raised.sum(-1, keepdim=True)
    else:
        scores = 1.0 / (1.0 + torch.exp(-x))
    # Without a bias the order of the scores is the order of the logits.
    choice = x if s["bias"] is None else scores + s["bias"]
    if c["groups"] > 1:
        best = choice.view(m, c["groups"], -1).sort(-1, descending=True)[0]
        worth = best[..., 0] if s["bias"] is None else best[..., 0] + best[..., 1]
        kept = worth.sort(dim=-1, descending=True, stable=True)[1][:, :c["top_groups"]]
        member = torch.zeros_like(worth).scatter_(1, kept, 1.0) > 0
        choice = torch.where(member.repeat_interleave(e // c["groups"], 1), choice, -math.inf)
    experts = choice.sort(dim=-1, descending=True, stable=True)[1][:, :c["top_k"]]
    weights = torch.gather(scores, 1, experts)
    if c["renormalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    return {"weights": weights * c["scale"], "experts": experts.int()}


# ---- what one pass cannot do without ------------------------------------------------------------


def work(case):
    if case["op"] == "rope_append":
        m, hq, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        moved = 2 * 2 * (m * hq * d + (m - case["pad"]) * 2 * hk * d)  # q, k, v in; q and the cache's rows out
        return {"bytes": moved + m * (4 * case["rotary"] + 4 + 8), "flops": 3 * m * (hq + hk) * case["rotary"]}
    if case["op"] == "tree_attention":
        hq, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
        pairs = [(c, t) for c, t in zip(_contexts(case), _drafts(case)) if t]
        n, cached = sum(t for _, t in pairs), sum(c + t for c, t in pairs)
        words = (case["draft"] + 31) // 32 if case["draft"] > 1 else 0
        moved = 2 * 2 * cached * hk * d + 2 * n * hq * d * (3 if case["gate"] else 2) + 4 * n * words
        moved += 4 * (sum((c + t + page - 1) // page for c, t in pairs) + 2 * case["requests"] + 1)
        return {"bytes": moved, "flops": 4 * sum(t * (c + t) for c, t in pairs) * hq * d}
    m, e = case["tokens"], case["experts"]
    size = 4 if case["dtype"] == "fp32" else 2
    return {"bytes": m * (e * size + 8 * case["top_k"]) + (4 * e if case["bias"] else 0), "flops": 6 * m * e}


# ---- the definitions in 64 bits -----------------------------------------------------------------


def exact(case, seed):
    s = _inputs(case, seed)
    return {"rope_append": _exact_rope, "tree_attention": _exact_attention, "route": _exact_route}[case["op"]](case, s)


def _exact_rope(case, s):
    """Each pair of a head's first `rotary` entries as a complex number, turned by its angle."""
    rot = case["rotary"]

    def turned(x):
        x = x.double().clone()
        pair = x[..., :rot].reshape(x.shape[:2] + ((rot // 2, 2) if case["interleaved"] else (2, rot // 2)))
        pair = pair if case["interleaved"] else pair.transpose(2, 3)
        # The table is an input: its 32-bit entries are the operator's angles.
        by = torch.complex(s["rope"][:, :rot // 2].double(), s["rope"][:, rot // 2:].double())[s["positions"].long()]
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * by[:, None, :])
        x[..., :rot] = (z if case["interleaved"] else z.transpose(2, 3)).reshape(x.shape[:2] + (rot,))
        return x

    got = {"q": turned(s["q"]), "k_pages": s["k_pages"].double(), "v_pages": s["v_pages"].double()}
    rows = torch.nonzero(s["slots"] >= 0)[:, 0]
    slots, page = s["slots"][rows], case["page"]
    for name, new in (("k_pages", turned(s["k"])), ("v_pages", s["v"].double())):
        flat = got[name].transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])  # in the order of slots
        flat[slots] = new[rows]
        got[name] = flat.view(-1, page, case["kv_heads"], case["dim"]).transpose(1, 2).contiguous()
    return got


def _exact_attention(case, s):
    """Request by request and head by head: softmax over the tokens that each row sees."""
    hq, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if 4 * sum(t * (c + t) for c, t in zip(_contexts(case), _drafts(case))) * hq * d > 4e11:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    starts, contexts = s["starts"].tolist(), s["context"].tolist()
    for b, context in enumerate(contexts):
        lo, hi = starts[b], starts[b + 1]
        if lo == hi:
            continue
        t = hi - lo
        pages = s["page_table"][b, :(context + t + page - 1) // page].long()
        seen = torch.ones((t, context + t), dtype=torch.bool, device="cuda")
        if s["mask"] is None:
            seen[:, context:] = torch.ones((t, t), dtype=torch.bool, device="cuda").tril()
        else:
            j = torch.arange(t, device="cuda")
            seen[:, context:] = (s["mask"][lo:hi].long()[:, j // 32] >> (j % 32)[None]) % 2 != 0
        for h in range(hk):
            group = slice(h * (hq // hk), (h + 1) * (hq // hk))
            k = s["k_pages"][pages, h].reshape(-1, d)[:context + t].double()
            v = s["v_pages"][pages, h].reshape(-1, d)[:context + t].double()
            rows = s["q"][lo:hi, group].double()
            a = torch.einsum("tgd,ld->tgl", rows, k) * d ** -0.5
            a = a.masked_fill(~seen[:, None], -math.inf).softmax(-1)
            out[lo:hi, group] = torch.einsum("tgl,ld->tgd", a, v)
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double())
    return out


def _exact_route(case, s):
    """The weights alone: which experts are chosen goes by 32-bit scores, ties and near ties included."""
    experts = _plain_route({"case": case, **s})["experts"].long()
    x = s["logits"].double()
    scores = x.softmax(-1) if case["scoring"] == "softmax" else x.sigmoid()
    weights = scores.gather(1, experts)
    if case["renormalize"]:
        weights /= weights.sum(1, keepdim=True)
    return {"weights": weights * case["scale"], "experts": None}
