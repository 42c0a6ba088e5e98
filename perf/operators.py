"""Cases for the operators around the MoE layer of a decode step.

Three operators that a decode step needs next to its MoE layers:

  append   keys and values of new tokens, rotated by their positions, written
           into a paged cache (and the queries rotated by the same angles);
  attend   attention of a batch over that cache, where all sequences share one
           long prefix and each has its own tokens behind it;
  sample   a token for each row of logits by temperature, top-k, top-p and
           min-p, from given uniform numbers.

`run` computes them in a plain form out of elementary torch operations, or,
where `own` is true, through warp_route's entry points.
"""
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
THETA = 1e6  # base of the rotation frequencies


def _warp_route():
    pkg = os.path.join(os.getcwd(), "warp-route_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import warp_route

    return warp_route


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one token of one sequence: the append of every single-stream decode step (latency)
        dict(name="append_one", op="append", tokens=1, heads_q=32, heads_kv=8, dim=128, rot=128, page=16, pages=512, far=4000,
             interleaved=False, padded=0, dtype="bf16"),
        # a prompt of odd length entering the cache at far positions, the batch padded at its end
        dict(name="append_prompt", op="append", tokens=8191, heads_q=32, heads_kv=8, dim=128, rot=128, page=16, pages=1024, far=900000,
             interleaved=False, padded=61, dtype="bf16"),
        # fp32, as many key heads as query heads, interleaved pairs, half of the head rotated
        dict(name="append_f32", op="append", tokens=1000, heads_q=16, heads_kv=16, dim=128, rot=64, page=32, pages=64, far=30000,
             interleaved=True, padded=0, dtype="f32"),
        # one short conversation, no prefix: latency
        dict(name="attend_one", op="attend", batch=1, q_max=1, heads_q=32, heads_kv=8, dim=128, page=16, prefix=0, own_max=300,
             dtype="bf16", lse=False),
        # one sequence of 64 Ki tokens, most of them a cached document: one row of queries, a long axis
        dict(name="attend_long", op="attend", batch=1, q_max=1, heads_q=32, heads_kv=8, dim=128, page=16, prefix=61003, own_max=4500,
             dtype="bf16", lse=False),
        # a small batch behind a system prompt whose end lies inside a page
        dict(name="attend_batch", op="attend", batch=16, q_max=1, heads_q=32, heads_kv=8, dim=128, page=16, prefix=2055, own_max=700,
             dtype="bf16", lse=False),
        # a large batch behind a long document, six query heads a key head
        dict(name="attend_large", op="attend", batch=256, q_max=1, heads_q=48, heads_kv=8, dim=128, page=64, prefix=16384, own_max=500,
             dtype="bf16", lse=False),
        # several tokens a sequence (checking drafted tokens), ragged, with the log-sum-exp
        dict(name="attend_drafts", op="attend", batch=24, q_max=9, heads_q=32, heads_kv=8, dim=128, page=32, prefix=5000, own_max=1000,
             dtype="bf16", lse=True),
        # fp32, one query head a key head
        dict(name="attend_f32", op="attend", batch=12, q_max=1, heads_q=16, heads_kv=16, dim=128, page=16, prefix=1000, own_max=700,
             dtype="f32", lse=False),
        # one row of a small vocabulary, top-k and top-p: latency
        dict(name="sample_one", op="sample", batch=1, vocab=32000, temperature=0.8, top_k=50, top_p=0.9, min_p=0.0, mixed=False,
             dtype="f32"),
        # bf16 logits (many equal ones), odd vocabulary, the nucleus alone
        dict(name="sample_nucleus", op="sample", batch=64, vocab=100277, temperature=1.0, top_k=0, top_p=0.95, min_p=0.0, mixed=False,
             dtype="bf16"),
        # a large batch of requests, each with settings of its own
        dict(name="sample_mixed", op="sample", batch=256, vocab=131072, temperature=0.9, top_k=200, top_p=0.95, min_p=0.02, mixed=True,
             dtype="f32"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 250)


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8, 16])
    return kv, kv * rng.choice([1, 2, 4, 6, 8])


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sample"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if op == "append":
        kv, q = _heads(rng)
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        page = rng.choice([16, 32, 64])
        tokens = _spread(rng, 1, 8192)
        while True:
            case = dict(op=op, tokens=tokens, heads_q=q, heads_kv=kv, dim=dim, rot=rng.choice([dim, dim, dim // 2]), page=page,
                        pages=-(-tokens // page) + rng.randint(1, 200), far=_spread(rng, tokens, 1000000),
                        interleaved=rng.random() < 0.4, padded=rng.randint(0, tokens // 2), dtype=dtype)
            if _cost(case) <= _cost(_named("append_prompt")):
                return case
            tokens = max(1, tokens // 2)
    if op == "attend":
        kv, q = _heads(rng)
        batch = _spread(rng, 1, 256)
        prefix = rng.choice([0, _spread(rng, 1, 32768), _spread(rng, 64, 32768)])
        q_max = 1 if rng.random() < 0.7 else rng.randint(2, 64)
        own_max = max(q_max, _spread(rng, 1, 4096))
        case = dict(op=op, batch=batch, q_max=q_max, heads_q=q, heads_kv=kv, dim=rng.choice([64, 96, 128, 128, 128, 256]),
                    page=rng.choice([16, 32, 64]), prefix=prefix, own_max=own_max, dtype=dtype, lse=rng.random() < 0.3)
        top = _cost(_named("attend_large")) / (16 if dtype == "f32" else 1)
        while _cost(case) > top:
            case["batch"] = max(1, case["batch"] // 2)
            case["prefix"] = case["prefix"] * 2 // 3
            case["own_max"] = max(q_max, case["own_max"] * 3 // 4)
        return case
    vocab = _spread(rng, 1000, 160000)
    batch = _spread(rng, 1, 256)
    case = dict(op=op, batch=batch, vocab=vocab, temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]),
                top_k=rng.choice([0, 1, 20, 50, _spread(rng, 2, vocab)]), top_p=rng.choice([1.0, 0.1, 0.5, 0.9, 0.99]),
                min_p=rng.choice([0.0, 0.0, 0.01, 0.1]), mixed=rng.random() < 0.5, dtype=dtype)
    while _cost(case) > _cost(_named("sample_mixed")):
        case["batch"] = max(1, case["batch"] // 2)
    return case


def _named(name):
    return next(c for c in listed() if c["name"] == name)


def _lengths(case):
    """Tokens that each sequence asks with, and its own tokens in the cache (those among them): ragged, by the case alone."""
    r = random.Random(case["batch"] * 7919 + case["own_max"])
    asks = [case["q_max"] if b == 0 else r.randint(1, case["q_max"]) for b in range(case["batch"])]
    return asks, [case["own_max"] if b == 0 else r.randint(n, case["own_max"]) for b, n in enumerate(asks)]


def work(case):
    """Each input read once and each output written once; two operations a multiply and add."""
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "append":
        t, hq, hk, d = case["tokens"], case["heads_q"], case["heads_kv"], case["dim"]
        live = t - case["padded"]
        # queries read and written for all tokens, keys and values for those that have a slot
        return {"bytes": 2 * t * hq * d * e + 4 * live * hk * d * e + 16 * t, "flops": 3 * case["rot"] * (t * hq + live * hk)}
    if case["op"] == "attend":
        asks, owned = _lengths(case)
        hq, hk, d = case["heads_q"], case["heads_kv"], case["dim"]
        keys = case["prefix"] + sum(owned)
        # token i of the n that a sequence asks with sees all its own tokens but the n - 1 - i last
        seen = sum(n * (case["prefix"] + c) - n * (n - 1) // 2 for n, c in zip(asks, owned))
        return {"bytes": 2 * keys * hk * d * e + 2 * sum(asks) * hq * d * e + (4 * sum(asks) * hq if case["lse"] else 0),
                "flops": 4 * seen * hq * d}
    # a comparison, an exponential and a sum for each value
    return {"bytes": case["batch"] * (case["vocab"] * e + 4 + 8 + (16 if case["mixed"] else 0)), "flops": 3 * case["batch"] * case["vocab"]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    if case["op"] == "append":
        t, hq, hk, d = case["tokens"], case["heads_q"], case["heads_kv"], case["dim"]
        slots = torch.randperm(case["pages"] * case["page"], generator=g, device="cuda")[:t].clone()
        if case["page"] <= t:  # whole pages in order, as an allocator hands them out
            pages = torch.randperm(case["pages"], generator=g, device="cuda")
            at = torch.arange(t, device="cuda")
            slots = pages[at // case["page"]] * case["page"] + at % case["page"]
        live = t - case["padded"]
        slots[live:] = -1
        first = int(torch.randint(0, case["far"] - t + 1, (1,), generator=g, device="cuda"))
        rot = case["rot"]
        return dict(case=case, qkv=normal(t, (hq + 2 * hk) * d), slots=slots,
                    positions=torch.arange(t, device="cuda") + first,
                    inv_freq=(THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)).float(),
                    k_cache=normal(case["pages"], hk, case["page"], d), v_cache=normal(case["pages"], hk, case["page"], d))
    if case["op"] == "attend":
        asks, owned = _lengths(case)
        hq, hk, d, ps = case["heads_q"], case["heads_kv"], case["dim"], case["page"]
        shared = -(-case["prefix"] // ps)
        counts = [-(-c // ps) for c in owned]
        wide = max(counts)
        total = shared + sum(counts) + 3
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        n_pages = torch.tensor(counts, device="cuda")
        start = shared + torch.cumsum(n_pages, 0) - n_pages
        col = torch.arange(wide, device="cuda")
        tables = order[(start[:, None] + col).clamp(max=total - 1)]
        tables = torch.where(col < n_pages[:, None], tables, torch.zeros_like(tables))  # what lies behind a row's pages is not read
        asks_t = torch.tensor(asks, dtype=torch.int32, device="cuda")
        q_start = torch.zeros(case["batch"] + 1, dtype=torch.int32, device="cuda")
        q_start[1:] = torch.cumsum(asks_t, 0)
        k_cache, v_cache = normal(total, hk, ps, d), normal(total, hk, ps, d)
        k_cache[order[-1].long()] = float("nan")  # a page that nobody owns: memory never written
        v_cache[order[-1].long()] = float("nan")
        return dict(case=case, q=normal(sum(asks), hq, d), k_cache=k_cache, v_cache=v_cache, tables=tables.contiguous(),
                    lens=torch.tensor(owned, dtype=torch.int32, device="cuda"), q_start=None if case["q_max"] == 1 else q_start,
                    q_max=case["q_max"], prefix_pages=order[:shared].contiguous())
    b, v = case["batch"], case["vocab"]
    x = torch.randn(b, v, generator=g, device="cuda") * 2.5
    heads = torch.randint(0, v, (b, 24), generator=g, device="cuda")  # the tokens that the model means
    x.scatter_(1, heads, 9.0 + 2.5 * torch.randn(b, 24, generator=g, device="cuda"))
    state = dict(case=case, logits=x.to(dt), uniforms=torch.rand(b, generator=g, device="cuda").clamp(max=1 - 2.0 ** -24),
                 temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
    if case["mixed"]:  # each row is a request with settings of its own
        row = torch.arange(b, device="cuda")
        state["temperature"] = torch.where(row % 5 == 0, 0.0, case["temperature"] * (0.5 + (row % 7) / 7)).float()
        state["top_k"] = torch.where(row % 2 == 0, case["top_k"], 0).int()
        state["top_p"] = torch.where(row % 3 == 0, 1.0, case["top_p"]).float()
        state["min_p"] = torch.where(row % 4 == 1, case["min_p"], 0.0).float()
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    if own:
        return {"append": _own_append, "attend": _own_attend, "sample": _own_sample}[state["case"]["op"]](state)
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[state["case"]["op"]](state)


def _split(state):
    """The three parts of a fused projection, as views."""
    c, qkv = state["case"], state["qkv"]
    hq, hk, d = c["heads_q"], c["heads_kv"], c["dim"]
    heads = qkv.view(qkv.shape[0], hq + 2 * hk, d)
    return heads[:, :hq], heads[:, hq:hq + hk], heads[:, hq + hk:]


def _own_append(s):
    q, k, v = _split(s)
    q = _warp_route().append_paged_kv(k, v, s["k_cache"], s["v_cache"], s["slots"], positions=s["positions"], inv_freq=s["inv_freq"], q=q,
                                      interleaved=s["case"]["interleaved"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_attend(s):
    out = _warp_route().shared_prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], prefix_pages=s["prefix_pages"],
                                                prefix_len=s["case"]["prefix"], q_start=s["q_start"], return_lse=s["case"]["lse"])
    return {"out": out[0], "lse": out[1]} if s["case"]["lse"] else {"out": out}


def _own_sample(s):
    return {"ids": _warp_route().sample_tokens(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                               min_p=s["min_p"])}


def _rotate(x, cos, sin, interleaved):
    """x [T, heads, dim] in 32 bits; the first 2 * cos.shape[1] values of each head turn in pairs."""
    half = cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _plain_append(s):
    c = s["case"]
    q, k, v = _split(s)
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()  # 64 bits: 32 lose the angles of far positions
    cos, sin = angle.cos().float(), angle.sin().float()
    k = _rotate(k.float(), cos, sin, c["interleaved"]).to(k.dtype)
    # tokens without a slot repeat what the first one with a slot writes
    has = s["slots"] >= 0
    source = torch.where(has, torch.arange(c["tokens"], device=has.device), has.int().argmax())
    slots = s["slots"][source]
    page, row = slots // c["page"], slots % c["page"]
    s["k_cache"][page, :, row] = k[source]
    s["v_cache"][page, :, row] = v[source]
    return {"q": _rotate(q.float(), cos, sin, c["interleaved"]).to(q.dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attend(s):
    c, q = s["case"], s["q"].float()
    hk, d, t = c["heads_kv"], c["dim"], q.shape[0]
    group, low = c["heads_q"] // hk, float("-inf")
    q = (q * d ** -0.5).view(t, hk, group, d)
    # the prefix, once for all tokens: [hk, t * group, prefix]
    at = s["prefix_pages"].long()
    kp = s["k_cache"][at].transpose(0, 1).reshape(hk, -1, d)[:, :c["prefix"]].float()
    vp = s["v_cache"][at].transpose(0, 1).reshape(hk, -1, d)[:, :c["prefix"]].float()
    sp = (q.transpose(0, 1).reshape(hk, t * group, d) @ kp.transpose(1, 2)).view(hk, t, group, -1).transpose(0, 1)
    # own tokens: sequences padded to the same number of questions and keys: [b, hk, q_max * group, keys]
    b, wide = s["tables"].shape
    if s["q_start"] is None:
        seq, nth, asks = torch.arange(t, device=q.device), torch.zeros(t, dtype=torch.long, device=q.device), torch.ones(b, dtype=torch.long, device=q.device)
    else:
        first = s["q_start"].long()
        seq = torch.searchsorted(first, torch.arange(t, device=q.device), right=True) - 1
        nth, asks = torch.arange(t, device=q.device) - first[seq], first[1:] - first[:-1]
    at = s["tables"].long()
    ko = s["k_cache"][at].transpose(1, 2).reshape(b, hk, wide * c["page"], d).float()
    vo = s["v_cache"][at].transpose(1, 2).reshape(b, hk, wide * c["page"], d).float()
    key = torch.arange(wide * c["page"], device=q.device)
    vo = torch.where((key < s["lens"][:, None])[:, None, :, None], vo, 0.0)
    qo = torch.zeros(b, s["q_max"], hk, group, d, device=q.device)
    qo[seq, nth] = q
    so = (qo.transpose(1, 2).reshape(b, hk, -1, d) @ ko.transpose(2, 3)).view(b, hk, s["q_max"], group, -1).transpose(1, 2)[seq, nth]
    seen = key < (s["lens"] - asks)[seq][:, None] + nth[:, None] + 1
    so = torch.where(seen[:, None, None], so, low)
    # one softmax over both
    top = so.amax(-1, keepdim=True)
    if c["prefix"]:
        top = torch.maximum(top, sp.amax(-1, keepdim=True))
    level = torch.where(top == low, 0.0, top)
    po = (so - level).exp()
    total = po.sum(-1, keepdim=True)
    full = torch.zeros(b, s["q_max"], hk, group, po.shape[-1], device=q.device)
    full[seq, nth] = po
    out = (full.transpose(1, 2).reshape(b, hk, -1, po.shape[-1]) @ vo).view(b, hk, s["q_max"], group, d).transpose(1, 2)[seq, nth]
    if c["prefix"]:
        pp = (sp - level).exp()
        total = total + pp.sum(-1, keepdim=True)
        out = out + (pp.transpose(0, 1).reshape(hk, t * group, -1) @ vp).view(hk, t, group, d).transpose(0, 1)
    out = torch.where(total > 0, out / total, 0.0).view(t, -1, d).to(s["q"].dtype)
    return {"out": out, "lse": (top + total.log()).view(t, -1)} if c["lse"] else {"out": out}


def _plain_sample(s):
    # 64 bits: where a sum passes a border decides which token it is
    x = s["logits"].double()
    x = torch.where(x.isnan(), float("-inf"), x)
    b, v = x.shape

    def column(a):
        return (a if isinstance(a, torch.Tensor) else torch.full((b,), a, dtype=torch.float32, device=x.device)).view(b, 1)

    heat, top_k, top_p, min_p = (column(s[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    heat, top_p, min_p = heat.double(), top_p.double(), min_p.double()
    top_k = torch.where(heat == 0, 1, torch.where((top_k < 1) | (top_k > v), v, top_k))
    x, index = x.sort(dim=1, descending=True, stable=True)  # equal ones: the lowest index first
    top = x[:, :1]
    w = torch.where(x == top, 0.0, (x - top) / torch.where(heat == 0, 1.0, heat)).exp()
    w = torch.where(torch.arange(v, device=x.device) < top_k, w, 0.0)
    upto = w.cumsum(1)
    before = torch.cat([torch.zeros_like(top), upto[:, :-1]], 1)
    keep = ((before < top_p * upto[:, -1:]) | (top_p >= 1)) & (w >= min_p)
    keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, index, torch.where(keep, w, 0.0))
    upto = w.cumsum(1)
    ids = (upto <= s["uniforms"].double()[:, None] * upto[:, -1:]).sum(1)
    return {"ids": torch.where(top[:, 0] == float("-inf"), -1, ids)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](case, s)


def _exact_append(case, s):
    hq, hk, d, half = case["heads_q"], case["heads_kv"], case["dim"], case["rot"] // 2
    x = s["qkv"].double().cpu().numpy().reshape(case["tokens"], hq + 2 * hk, d)
    # a pair is a complex number, its turn a product with exp(i * angle)
    turn = np.exp(1j * np.outer(s["positions"].cpu().numpy().astype(np.float64), s["inv_freq"].double().cpu().numpy()))[:, None, :]
    first = np.arange(half) * 2 if case["interleaved"] else np.arange(half)
    second = first + (1 if case["interleaved"] else half)
    z = (x[:, :hq + hk, first] + 1j * x[:, :hq + hk, second]) * turn
    x[:, :hq + hk, first], x[:, :hq + hk, second] = z.real, z.imag
    caches = [s["k_cache"].double().cpu().numpy(), s["v_cache"].double().cpu().numpy()]
    slots = s["slots"].cpu().numpy()
    live = np.nonzero(slots >= 0)[0]
    for cache, lo in zip(caches, (hq, hq + hk)):
        cache[slots[live] // case["page"], :, slots[live] % case["page"]] = x[live, lo:lo + hk]
    return {"q": x[:, :hq], "k_cache": caches[0], "v_cache": caches[1]}


def _exact_attend(case, s):
    if work(case)["flops"] > 5e11:
        return None
    asks, owned = _lengths(case)
    hk, d, ps = case["heads_kv"], case["dim"], case["page"]
    group = case["heads_q"] // hk
    k, v, q = s["k_cache"], s["v_cache"], s["q"].double()

    def rows(cache, pages, n):  # [hk, n, d]
        return cache[pages.long()].double().transpose(0, 1).reshape(hk, -1, d)[:, :n]

    kp, vp = rows(k, s["prefix_pages"], case["prefix"]), rows(v, s["prefix_pages"], case["prefix"])
    outs, sums, at = [], [], 0
    for b in range(case["batch"]):
        n, c = asks[b], owned[b]
        pages = s["tables"][b, :-(-c // ps)]
        kk, vv = torch.cat([kp, rows(k, pages, c)], 1), torch.cat([vp, rows(v, pages, c)], 1)
        qq = q[at:at + n].view(n, hk, group, d).permute(1, 2, 0, 3).reshape(hk, group * n, d)
        sc = (qq @ kk.transpose(1, 2)).view(hk, group, n, -1) / d ** 0.5
        last = case["prefix"] + c - n + torch.arange(n, device=q.device)
        sc = sc.masked_fill(torch.arange(kk.shape[1], device=q.device) > last[:, None], float("-inf"))
        p = sc.softmax(-1).view(hk, group * n, -1)
        outs.append((p @ vv).view(hk, group, n, d).permute(2, 0, 1, 3).reshape(n, hk * group, d))
        sums.append(sc.logsumexp(-1).permute(2, 0, 1).reshape(n, hk * group))
        at += n
    out = {"out": torch.cat(outs).cpu().numpy()}
    return {**out, "lse": torch.cat(sums).cpu().numpy()} if case["lse"] else out


def _exact_sample(case, s):
    x, u = s["logits"].double().cpu().numpy(), s["uniforms"].double().cpu().numpy()
    b, v = x.shape

    def column(a):
        return a.double().cpu().numpy() if isinstance(a, torch.Tensor) else np.full(b, a, np.float32).astype(np.float64)

    # the settings are numbers of 32 bits
    heat, top_k, top_p, min_p = (column(s[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    ids = np.empty(b, np.int64)
    for r in range(b):
        order = np.argsort(-x[r], kind="stable")
        if heat[r] == 0:
            ids[r] = order[0]
            continue
        if top_k[r] >= 1:
            order = order[:int(top_k[r])]
        w = np.exp((x[r, order] - x[r, order[0]]) / heat[r])
        keep = w >= min_p[r]
        if top_p[r] < 1:
            keep &= np.concatenate([[0.0], np.cumsum(w)[:-1]]) < top_p[r] * w.sum()
        keep[0] = True
        kept = np.sort(order[keep])
        c = np.cumsum(np.exp((x[r, kept] - x[r, order[0]]) / heat[r]))
        ids[r] = kept[np.searchsorted(c, u[r] * c[-1], side="right")]
    return {"ids": ids}
