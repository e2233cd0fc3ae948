"""The serving operators of ``npu_amd.ops`` for a batch of sequences, as they are measured:
rotary positions with the append to a paged key-value cache, attention of one new token over
that cache, attention over packed prompts, and sampling.

``run`` makes one pass through one operator: with ``own`` the framework's call, without it the
same result from elementary torch operations in 32 bits (64 where 32 lose what matters).
``exact`` is the operators' definition in 64 bits.

Sizes: attention heads (16, 2, 256) with 64 rotated dims and the vocabulary of 248,320 are the
decoder's own (npu_amd.qwen_core.Config); the other head layouts, vocabularies and lengths are
generic.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
#: (query heads, key-value heads, head dim, rotated dims)
HEADS = ((16, 2, 256, 64), (32, 8, 128, 128), (8, 8, 64, 64), (24, 4, 128, 64), (12, 4, 64, 32), (7, 1, 256, 128))
VOCABS = (248_320, 131_072, 50_001, 32_000, 1_001)


def listed():
    return [
        # the new tokens of eight sequences: norms, three-axis rotation and the cache rows of one decode step
        {"name": "rope_step", "op": "rope", "tokens": 8, "hq": 16, "hkv": 2, "dim": 256, "rot": 64, "axes": 3,
         "dtype": "float32", "cache": "bfloat16", "norm": True, "far": 40_000, "page": 64},
        # a prompt with an image in it, as the projections leave it (fp32, q and its gate interleaved)
        {"name": "rope_prompt", "op": "rope", "tokens": 2_021, "hq": 16, "hkv": 2, "dim": 256, "rot": 64, "axes": 3,
         "dtype": "float32", "cache": "bfloat16", "norm": True, "far": 200_000, "page": 64},
        # many packed prompts of a 16-bit model, whole heads rotated, one axis, no norms
        {"name": "rope_packed", "op": "rope", "tokens": 16_384, "hq": 32, "hkv": 8, "dim": 128, "rot": 128, "axes": 1,
         "dtype": "bfloat16", "cache": "bfloat16", "norm": False, "far": 1_000_000, "page": 16},
        # one sequence, the decoder's own heads and fp32 activations: latency counts
        {"name": "decode_one", "op": "decode", "batch": 1, "longest": 4_001, "ragged": False, "hq": 16, "hkv": 2,
         "dim": 256, "dtype": "float32", "cache": "bfloat16", "page": 64, "gate": True},
        # a batch of sequences of very different lengths
        {"name": "decode_batch", "op": "decode", "batch": 64, "longest": 8_192, "ragged": True, "hq": 16, "hkv": 2,
         "dim": 256, "dtype": "bfloat16", "cache": "bfloat16", "page": 64, "gate": True},
        # a few very long ones
        {"name": "decode_long", "op": "decode", "batch": 4, "longest": 131_071, "ragged": False, "hq": 32, "hkv": 8,
         "dim": 128, "dtype": "float16", "cache": "float16", "page": 16, "gate": False},
        # a handful of short questions packed together
        {"name": "prompt_short", "op": "prompt", "batch": 5, "tokens": 301, "cached": 0, "hq": 16, "hkv": 2,
         "dim": 256, "dtype": "bfloat16", "paged": False, "page": 64, "gate": True},
        # the packed prompts of a busy server
        {"name": "prompt_packed", "op": "prompt", "batch": 11, "tokens": 8_192, "cached": 0, "hq": 32, "hkv": 8,
         "dim": 128, "dtype": "float16", "paged": False, "page": 16, "gate": False},
        # one long document, written to the cache before
        {"name": "prompt_long", "op": "prompt", "batch": 1, "tokens": 16_000, "cached": 0, "hq": 16, "hkv": 2,
         "dim": 256, "dtype": "bfloat16", "paged": True, "page": 64, "gate": True},
        # the next token of one sequence
        {"name": "sample_one", "op": "sample", "batch": 1, "vocab": 248_320, "dtype": "float32", "filters": "all"},
        # a batch whose users ask for different things
        {"name": "sample_batch", "op": "sample", "batch": 64, "vocab": 248_320, "dtype": "float32", "filters": "mixed"},
        # a large batch with the nucleus alone, no top-k to shorten the search
        {"name": "sample_nucleus", "op": "sample", "batch": 256, "vocab": 248_320, "dtype": "bfloat16",
         "filters": "nucleus"},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["rope", "decode", "prompt", "sample"])
    hq, hkv, dim, rot = rng.choice(HEADS)
    page = rng.choice([16, 32, 64, 128])
    if op == "rope":
        dtype, cache = rng.choice([("float32", "bfloat16"), ("float32", "float16"), ("bfloat16", "bfloat16"),
                                   ("float16", "float16")])
        return {"op": op, "tokens": _log(rng, 1, 8_192), "hq": hq, "hkv": hkv, "dim": dim, "rot": rot,
                "axes": rng.choice([1, 3]), "dtype": dtype, "cache": cache, "norm": rng.random() < 0.5,
                "far": _log(rng, 100, 1_000_000), "page": page}
    if op == "decode":
        dtype, cache = rng.choice([("float32", "bfloat16"), ("float32", "float16"), ("bfloat16", "bfloat16"),
                                   ("float16", "float16")])
        batch = _log(rng, 1, 100)
        return {"op": op, "batch": batch, "longest": _log(rng, 1, min(131_071, 500_000 // (batch * max(1, hkv // 2)))),
                "ragged": rng.random() < 0.6, "hq": hq, "hkv": hkv, "dim": dim, "dtype": dtype, "cache": cache,
                "page": page, "gate": rng.random() < 0.5}
    if op == "prompt":
        return {"op": op, "batch": _log(rng, 1, 24), "tokens": _log(rng, 30, 8_000),
                "cached": rng.choice([0, 0, _log(rng, 1, 2_000)]), "hq": hq, "hkv": hkv, "dim": dim,
                "dtype": rng.choice(["bfloat16", "float16"]), "paged": rng.random() < 0.5, "page": page,
                "gate": rng.random() < 0.5}
    return {"op": op, "batch": _log(rng, 1, 128), "vocab": rng.choice(VOCABS),
            "dtype": rng.choice(["float32", "float32", "bfloat16", "float16"]),
            "filters": rng.choice(["all", "mixed", "nucleus", "none"])}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _lengths(case, g, batch):
    """The sequences' lengths, the new token with them: all the longest, or anything up to it."""
    if not case["ragged"]:
        return torch.full((batch,), case["longest"], dtype=torch.int32, device="cuda")
    r = torch.rand(batch, generator=g, device="cuda")
    n = (r * r * case["longest"]).to(torch.int32) + 1
    n[0] = case["longest"]
    return n.clamp_(max=case["longest"])


def _pages(g, lengths, page):
    """(block table, number of pages): every sequence's pages anywhere in the cache, -1 past its last."""
    need = (lengths.long() + page - 1) // page
    total, width = int(need.sum()), int(need.max())
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    first = torch.cumsum(need, 0) - need
    at = torch.arange(width, device="cuda")
    table = torch.where(at < need[:, None], order[(first[:, None] + at).clamp_(max=total - 1)], -1)
    return table.to(torch.int32).contiguous(), total


def _split(case, g):
    """cu_q of the packed prompts: `tokens` tokens cut at random places, an empty sequence possible."""
    b, t = case["batch"], case["tokens"]
    cuts = torch.randint(0, t + 1, (b - 1,), generator=g, device="cuda").sort().values
    zero = torch.zeros(1, dtype=torch.long, device="cuda")
    return torch.cat([zero, cuts, zero + t]).to(torch.int32)


def _rope_tables(case):
    """(inv_freq [rot / 2] fp64, axis [rot / 2] int32): pair i turns with axis i % 3 while the shorter
    axes last, then with axis 0."""
    half = case["rot"] // 2
    inv = 1e7 ** (-torch.arange(half, dtype=torch.float64) / half)
    i = torch.arange(half)
    axis = torch.where(i < half // 3 * 3, i % 3, 0) if case["axes"] == 3 else torch.zeros(half, dtype=torch.long)
    return inv.cuda(), axis.to(torch.int32).cuda()


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": dict(case)}
    op, dt = case["op"], TYPES[case["dtype"]]
    if op == "sample":
        b, v = case["batch"], case["vocab"]
        x = torch.randn(b, v, generator=g, device="cuda") * 2.5
        likely = torch.randint(0, v, (b, max(8, v // 1000)), generator=g, device="cuda")
        lift = torch.empty(likely.shape, device="cuda").exponential_(0.25, generator=g)
        x.scatter_add_(1, likely, lift)
        x[:, v - v // 100:] = float("-inf")                 # the padding of the vocabulary
        s["logits"] = x.to(dt)
        s["u"] = torch.rand(b, generator=g, device="cuda")
        r = torch.rand(4, b, generator=g, device="cuda")
        f = case["filters"]
        s["temperature"] = 0.5 + r[0]
        s["top_k"] = s["top_p"] = s["min_p"] = None
        if f == "all":
            s["top_k"] = (10 + r[1] * 40).to(torch.int32)
            s["top_p"], s["min_p"] = 0.8 + 0.19 * r[2], 0.05 * r[3]
        elif f == "mixed":                                   # greedy rows, rows without a filter, odd ones
            s["temperature"] = torch.where(r[0] < 0.1, 0.0, 0.3 + r[0])
            s["top_k"] = torch.where(r[1] < 0.4, 0, (r[1] * 300).to(torch.int32)).to(torch.int32)
            s["top_p"] = torch.where(r[2] < 0.3, 1.0, 0.5 + 0.5 * r[2])
            s["min_p"] = torch.where(r[3] < 0.5, 0.0, 0.1 * r[3])
        elif f == "nucleus":
            s["top_p"] = 0.85 + 0.14 * r[2]
        return s
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    if op == "rope":
        t = case["tokens"]
        row = _randn(g, t, (2 * hq + 2 * hkv) * dim, dtype=dt)      # the projection's row: [q | gate] per head, k, v
        s["q"] = row[:, :2 * hq * dim].view(t, hq, 2 * dim)[..., :dim]
        s["k"] = row[:, 2 * hq * dim:(2 * hq + hkv) * dim].view(t, hkv, dim)
        s["v"] = row[:, (2 * hq + hkv) * dim:].view(t, hkv, dim)
        s["positions"] = torch.randint(0, case["far"], (case["axes"], t), generator=g, device="cuda", dtype=torch.int32)
        s["inv_freq"], s["axis"] = _rope_tables(case)
        s["q_norm"] = 1 + _randn(g, dim, scale=0.1) if case["norm"] else None
        s["k_norm"] = 1 + _randn(g, dim, scale=0.1) if case["norm"] else None
        n = -(-t // case["page"]) + 3
        s["slots"] = torch.randperm(n * case["page"], generator=g, device="cuda")[:t].to(torch.int32)
        s["slots"][t // 2:t // 2 + t // 8] = -1                      # padded tokens: nothing is written
        s["k_pages"] = _randn(g, n, case["page"], hkv, dim, dtype=TYPES[case["cache"]])
        s["v_pages"] = _randn(g, n, case["page"], hkv, dim, dtype=TYPES[case["cache"]])
        return s
    s["scale"] = dim ** -0.5
    if op == "decode":
        b, ct = case["batch"], TYPES[case["cache"]]
        s["lengths"] = _lengths(case, g, b)
        s["table"], n = _pages(g, s["lengths"], case["page"])
        s["k"], s["v"] = (_randn(g, n, case["page"], hkv, dim, dtype=ct) for _ in range(2))
        row = _randn(g, b, hq, 2 * dim, dtype=dt)
    else:
        s["cu_q"] = _split(case, g)
        new = s["cu_q"][1:] - s["cu_q"][:-1]
        s["lengths"] = new + case["cached"]
        if case["paged"]:
            s["table"], n = _pages(g, s["lengths"].clamp(min=1), case["page"])
            s["k"], s["v"] = (_randn(g, n, case["page"], hkv, dim, dtype=dt) for _ in range(2))
        else:
            s["cu_k"] = torch.cat([s["cu_q"][:1], torch.cumsum(s["lengths"], 0).to(torch.int32)])
            n = case["tokens"] + case["batch"] * case["cached"]
            s["k"], s["v"] = (_randn(g, n, hkv, dim, dtype=dt) for _ in range(2))
        row = _randn(g, case["tokens"], hq, 2 * dim, dtype=dt)
        s["longest_q"], s["longest_k"] = int(new.max()), int(s["lengths"].max())
    s["q"] = row[..., :dim]
    s["gate"] = row[..., dim:] if case["gate"] else None
    return s


# ------------------------------------------------------------ plain forms
def _norm(x, w, eps):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w


def _rope_plain(s):
    c = s["case"]
    half = c["rot"] // 2
    pos = s["positions"][s["axis"].long()].t().double()             # [T, rot / 2]: far positions in 64 bits
    ang = pos * s["inv_freq"]
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]

    def turn(x, w):
        x = _norm(x.float(), w, 1e-6)
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)

    kp, vp = s["k_pages"], s["v_pages"]
    live = s["slots"] >= 0
    at = s["slots"][live].long()
    kp.view(-1, c["hkv"], c["dim"])[at] = turn(s["k"], s["k_norm"])[live].to(kp.dtype)
    vp.view(-1, c["hkv"], c["dim"])[at] = s["v"][live].to(vp.dtype)
    return {"q": turn(s["q"], s["q_norm"]).to(kp.dtype), "k_pages": kp, "v_pages": vp}


def _decode_plain(s):
    c = s["case"]
    b, hq, hkv, dim, page = c["batch"], c["hq"], c["hkv"], c["dim"], c["page"]
    at = s["table"].clamp(min=0).long()
    k = s["k"][at].view(b, -1, hkv, dim).permute(0, 2, 1, 3).float()   # [B, Hkv, L, D]
    v = s["v"][at].view(b, -1, hkv, dim).permute(0, 2, 1, 3).float()
    q = s["q"].float().view(b, hkv, hq // hkv, dim)
    x = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    live = torch.arange(k.shape[2], device=k.device) < s["lengths"][:, None, None, None]
    x = x.masked_fill(~live, float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.view(b, hq, dim)
    if s["gate"] is not None:
        o = o * (1 / (1 + torch.exp(-s["gate"].float())))
    return o.to(TYPES[c["dtype"]])


def _prompt_plain(s):
    c = s["case"]
    b, hq, hkv, dim = c["batch"], c["hq"], c["hkv"], c["dim"]
    nq, nk = s["longest_q"], s["longest_k"]
    new = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    i, j = torch.arange(nq, device="cuda"), torch.arange(nk, device="cuda")
    if c["paged"]:
        k, v = (x[s["table"].clamp(min=0).long()].view(b, -1, hkv, dim)[:, :nk] for x in (s["k"], s["v"]))
    else:
        at = (s["cu_k"][:-1, None].long() + j).clamp_(max=s["k"].shape[0] - 1)
        k, v = s["k"][at], s["v"][at]
    k, v = (x.permute(0, 2, 1, 3).float() for x in (k, v))             # [B, Hkv, nk, D]
    row = s["cu_q"][:-1, None].long() + i                               # [B, nq]
    q = s["q"].float()[row.clamp(max=c["tokens"] - 1)].permute(0, 2, 1, 3)
    q = q.reshape(b, hkv, hq // hkv * nq, dim)
    x = (torch.matmul(q, k.transpose(-1, -2)) * s["scale"]).view(b, hkv, hq // hkv, nq, nk)
    last = i + (s["lengths"].long() - new)[:, None]                     # the row's last key
    x = x.masked_fill((j > last[..., None])[:, None, None], float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    del x
    total = p.sum(-1, keepdim=True).view(b, hkv, -1, 1)
    o = torch.matmul(p.view(b, hkv, -1, nk), v) / total
    o = o.view(b, hq, nq, dim).permute(0, 2, 1, 3)[i < new[:, None]]    # the packed rows again
    if s["gate"] is not None:
        o = o * (1 / (1 + torch.exp(-s["gate"].float())))
    return o.to(TYPES[c["dtype"]])


def _sample_plain(s):
    x = s["logits"].double()                              # 64 bits: a pick next to a border of the sums
    b, v = x.shape
    t = s["temperature"].double()[:, None]
    y, order = torch.sort(x, dim=1, descending=True, stable=True)      # ties: the lowest index first
    w = torch.exp((y - y[:, :1]) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(v, device=x.device)
    keep = torch.where(t > 0, w > 0, rank == 0)
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        keep &= (k <= 0) | (rank < k)
    w = torch.where(keep, w, 0.0)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        before = torch.cumsum(w, 1) - w
        keep &= (p >= 1) | (rank == 0) | (before < p * w.sum(1, keepdim=True))
    if s["min_p"] is not None:
        keep &= (w >= s["min_p"].double()[:, None]) | (rank == 0)
    w = torch.where(keep, w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)                       # in the vocabulary's order
    total = torch.cumsum(w, 1)
    past = total > s["u"].double()[:, None] * total[:, -1:]
    return (past & (w > 0)).to(torch.int8).argmax(1)


# ------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    if not own:
        return {"rope": _rope_plain, "decode": _decode_plain, "prompt": _prompt_plain, "sample": _sample_plain}[c["op"]](s)
    from npu_amd import ops
    if c["op"] == "rope":
        q = ops.rope_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["k_pages"], s["v_pages"],
                            s["slots"], axis=s["axis"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6)
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if c["op"] == "decode":
        return ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], scale=s["scale"], gate=s["gate"])
    if c["op"] == "prompt":
        if c["paged"]:
            return ops.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], block_table=s["table"],
                                        lengths=s["lengths"], scale=s["scale"], gate=s["gate"])
        return ops.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], cu_k=s["cu_k"], scale=s["scale"], gate=s["gate"])
    return ops.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                      min_p=s["min_p"])


def _mean_keys(case):
    """Keys that a query row sees on average, and the cached rows in all (cut lengths: their expectation)."""
    b, t = case["batch"], case["tokens"]
    return case["cached"] + (t / b if b == 1 else 2 * t / (b + 1)) / 2, t + b * case["cached"]


def work(case):
    size = {"float32": 4, "bfloat16": 2, "float16": 2}
    e = size[case["dtype"]]
    if case["op"] == "sample":
        return {"bytes": case["batch"] * case["vocab"] * e, "flops": 0}
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    if case["op"] == "rope":
        t = case["tokens"]
        ce = size[case["cache"]]
        return {"bytes": t * dim * ((hq + 2 * hkv) * e + hq * ce + 2 * hkv * ce), "flops": 6 * t * dim * (hq + hkv)}
    gate = 1 if case["gate"] else 0
    if case["op"] == "decode":
        keys = case["batch"] * case["longest"] / (3 if case["ragged"] else 1)
        return {"bytes": 2 * keys * hkv * dim * size[case["cache"]] + (2 + gate) * case["batch"] * hq * dim * e,
                "flops": 4 * keys * hq * dim}
    keys, rows = _mean_keys(case)
    return {"bytes": 2 * rows * hkv * dim * e + (2 + gate) * case["tokens"] * hq * dim * e,
            "flops": 4 * case["tokens"] * keys * hq * dim}


# ------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    if case["op"] == "sample":
        return None
    if case["op"] == "prompt" and 4 * case["tokens"] * _mean_keys(case)[0] * case["hq"] * case["dim"] > 1e13:
        return None

    def attend(q, k, v, scale, first):
        """One sequence and kv head: q [n, G, D] over k, v [m, D], row i seeing the keys up to first + i."""
        out = []
        for at in range(0, q.shape[0], 1024):
            part = q[at:at + 1024].double()
            x = torch.einsum("igd,md->igm", part, k) * scale
            last = first + at + torch.arange(part.shape[0], device=q.device)
            x = x.masked_fill(torch.arange(k.shape[0], device=q.device) > last[:, None, None], -math.inf)
            out.append(torch.einsum("igm,md->igd", torch.softmax(x, -1), v))
        return torch.cat(out)

    def attention(s):
        hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
        o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        lengths = s["lengths"].tolist()
        cu = s["cu_q"].tolist() if case["op"] == "prompt" else list(range(case["batch"] + 1))
        ck = s["cu_k"].tolist() if "cu_k" in s else None
        for b, n in enumerate(lengths):
            if cu[b] == cu[b + 1]:
                continue
            if ck is None:
                pages = s["table"][b, :-(-n // case["page"])].long()
                k, v = (x[pages].reshape(-1, hkv, dim)[:n].double() for x in (s["k"], s["v"]))
            else:
                k, v = (x[ck[b]:ck[b + 1]].double() for x in (s["k"], s["v"]))
            q = s["q"][cu[b]:cu[b + 1]].reshape(cu[b + 1] - cu[b], hkv, hq // hkv, dim)
            for h in range(hkv):
                o[cu[b]:cu[b + 1], h * (hq // hkv):(h + 1) * (hq // hkv)] = attend(
                    q[:, h], k[:, h].contiguous(), v[:, h].contiguous(), s["scale"], n - (cu[b + 1] - cu[b]))
        return o if s["gate"] is None else o * torch.sigmoid(s["gate"].double())

    s = prepare(case, seed)
    if case["op"] != "rope":
        return attention(s)
    half = case["rot"] // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       torch.stack([s["positions"][a].double() * f for a, f in zip(s["axis"].tolist(), s["inv_freq"])], -1))

    def rotate(x, w):
        x = x.double().clone()
        if w is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn[:, None]
        x[..., :half], x[..., half:2 * half] = z.real, z.imag
        return x

    pages = {}
    for name, rows in (("k_pages", rotate(s["k"], s["k_norm"])), ("v_pages", s["v"].double())):
        p = s[name].double()
        flat = p.view(-1, case["hkv"], case["dim"])
        for at in (s["slots"] >= 0).nonzero().split(4096):
            flat[s["slots"][at[:, 0]].long()] = rows[at[:, 0]]
        pages[name] = p
    return {"q": rotate(s["q"], s["q_norm"]), **pages}
