"""Cases, plain forms and exact values of the paged-cache operators.

Four operators of a server that keeps many requests' keys and values in one
pool of pages:

  norm    RMS norm of every query and key head and the rotation by position
  append  the same pass, writing keys and values into the pages
  attend  attention of one new token per sequence over its pages, optionally
          adding each position's attention weight to a running sum
  evict   keeps, per sequence and key head, the most recent positions and of
          the others those with the largest running sum, packed in order

The caches are [pages, kv_heads, page, d]; a sequence's positions p lie in
page table[b, p // page], slot p % page.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
EPS = 1e-6

# A drawn case costs no more than the largest listed one.
MOST_BYTES = 1.0e9


def _attend(name, type, batch, heads, kv_heads, d, page, low, high, weights):
    return {"name": name, "op": "attend", "type": type, "batch": batch, "heads": heads,
            "kv_heads": kv_heads, "d": d, "page": page, "low": low, "high": high,
            "weights": weights}


def _norm(name, type, tokens, heads, kv_heads, d, rot, interleaved, table):
    return {"name": name, "op": "norm", "type": type, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "d": d, "rot": rot, "interleaved": interleaved, "table": table}


def _append(name, type, batch, heads, kv_heads, d, rot, interleaved, page, low, high, new, table):
    return {"name": name, "op": "append", "type": type, "batch": batch, "heads": heads,
            "kv_heads": kv_heads, "d": d, "rot": rot, "interleaved": interleaved, "page": page,
            "low": low, "high": high, "new": new, "table": table}


def _evict(name, type, batch, kv_heads, d, page, low, high, keep, recent):
    return {"name": name, "op": "evict", "type": type, "batch": batch, "kv_heads": kv_heads,
            "d": d, "page": page, "low": low, "high": high, "keep": keep, "recent": recent}


def listed():
    return [
        # one GPT-2-small request in mid answer: 32 prompt tokens and 128 of its own
        _attend("attend fp32 one request", "fp32", 1, 12, 12, 64, 16, 160, 160, False),
        # a batch of GPT-2-small requests anywhere in the 1024-token context, with running sums
        _attend("attend fp32 batch 32", "fp32", 32, 12, 12, 64, 16, 1, 1024, True),
        # an ordinary batch with grouped heads
        _attend("attend bf16 batch 16", "bf16", 16, 32, 8, 128, 16, 300, 4099, False),
        # one request with a very long context: few rows, all of the work along the length
        _attend("attend fp16 one long", "fp16", 1, 64, 8, 128, 64, 130937, 130937, False),
        # a full server, lengths from one token up, with running sums for the eviction
        _attend("attend bf16 batch 64 sums", "bf16", 64, 32, 8, 128, 32, 1, 8191, True),
        # the query and key heads of one decode step, before a dense cache
        _norm("norm fp32 four tokens", "fp32", 4, 12, 12, 64, 32, True, 2048),
        # those of a long prompt
        _norm("norm bf16 prompt", "bf16", 8190, 32, 8, 128, 128, False, 40960),
        # one new token for each of a batch's requests
        _append("append bf16 one each", "bf16", 64, 32, 8, 128, 128, False, 16, 1, 4099, 1, 40960),
        # the prompts of a few requests behind what their caches hold already
        _append("append fp16 prompts", "fp16", 5, 16, 4, 96, 64, True, 64, 1500, 6001, 1400,
                8192),
        # one GPT-2-small request back from its context's end to half of it
        _evict("evict fp32 one request", "fp32", 1, 12, 64, 16, 1024, 1024, 512, 64),
        # a batch that has grown past its budget
        _evict("evict bf16 batch 16", "bf16", 16, 8, 128, 16, 4100, 4352, 4096, 256),
        # long prompts cut down once they are read
        _evict("evict fp16 long", "fp16", 3, 8, 128, 64, 20011, 65521, 8192, 1024),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        type_ = rng.choice(["fp32", "fp16", "bf16"])
        d = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256])
        page = rng.choice([8, 16, 16, 24, 32, 64, 128])
        kv_heads = rng.randint(1, 16)
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
        rot = rng.choice([d, d, d // 2, d // 4])
        interleaved = rng.random() < 0.4
        op = rng.choice(["attend", "attend", "attend", "norm", "append", "evict"])
        if op == "attend":
            batch, high = _log(rng, 1, 160), _log(rng, 16, 150000)
            low = high if rng.random() < 0.3 else rng.randint(0, high)
            case = _attend("", type_, batch, heads, kv_heads, d, page, low, high,
                           rng.random() < 0.4)
            room = batch * heads * high * 4
        elif op == "norm":
            case = _norm("", type_, _log(rng, 1, 20000), heads, kv_heads, d, rot, interleaved,
                         _log(rng, 32, 131072))
            room = 0
        elif op == "append":
            batch, new = _log(rng, 1, 160), rng.choice([1, 1, _log(rng, 2, 4000)])
            high = new + _log(rng, 1, 8000)
            case = _append("", type_, batch, heads, kv_heads, d, rot, interleaved, page,
                           rng.randint(new, high), high, new, high + _log(rng, 1, 50000))
            room = batch * kv_heads * high * d * BYTES[type_]
        else:
            batch, high = _log(rng, 1, 64), _log(rng, 40, 65536)
            keep = rng.randint(max(1, high // 8), high)
            case = _evict("", type_, batch, kv_heads, d, page, rng.randint(keep // 2, high), high,
                          keep, rng.randint(0, keep))
            room = 0
        del case["name"]
        if work(case)["bytes"] <= MOST_BYTES and room <= 4e8 and _held(case) <= 4e9:
            return case


def _lens(case):
    """Lengths spread over [low, high]; the same multiset for every seed."""
    b, low, high = case["batch"], case["low"], case["high"]
    if b == 1:
        return [high]
    return [low + int(round((high - low) * ((0.6180339887498949 * i) % 1.0))) for i in range(b)]


def _news(case):
    """New tokens of each sequence: one each, or ragged up to `new`."""
    if case["new"] == 1:
        return [1] * case["batch"]
    lens = _lens(case)
    return [min(n, 1 + int((case["new"] - 1) * ((0.7548776662466927 * i + 0.9) % 1.0)))
            for i, n in enumerate(lens)]


def _pages(case):
    return [-(-n // case["page"]) for n in _lens(case)]


def _held(case):
    """Bytes of the caches as the plain form spreads them out."""
    if case["op"] == "norm":
        return 0
    wide = max(_pages(case)) * case["page"]
    return 8 * case["batch"] * case["kv_heads"] * wide * case["d"]


def work(case):
    es, op = BYTES[case["type"]], case["op"]
    d, hk = case["d"], case["kv_heads"]
    if op == "attend":
        n, b, h = sum(_lens(case)), case["batch"], case["heads"]
        nbytes = 2 * n * hk * d * es + 2 * b * h * d * es + 4 * sum(_pages(case)) + 4 * b
        if case["weights"]:
            nbytes += 8 * n * hk
        return {"bytes": nbytes, "flops": 4 * n * h * d}
    if op == "evict":
        lens = _lens(case)
        kept = sum(min(n, case["keep"]) for n in lens)
        nbytes = 8 * sum(lens) * hk + 4 * kept * hk + 4 * kept * hk * d * es
        return {"bytes": nbytes, "flops": 2 * sum(lens) * hk}
    tokens = case["tokens"] if op == "norm" else sum(_news(case))
    heads = case["heads"] + hk
    nbytes = 2 * tokens * heads * d * es + tokens * (4 * case["rot"] + 4)
    if op == "append":
        nbytes += 2 * tokens * hk * d * es
    return {"bytes": nbytes, "flops": tokens * heads * (4 * d + 3 * case["rot"])}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _table(case, g):
    """The rotation's cosines and sines, computed in 64 bits once per model."""
    half = case["rot"] // 2
    base = 10000.0 + 10.0 * float(torch.rand((), generator=g, device="cuda"))
    inv = base ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = torch.arange(case["table"], device="cuda", dtype=torch.float64)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def _cache(case, g, pages):
    shape = (pages, case["kv_heads"], case["page"], case["d"])
    t = TYPES[case["type"]]
    k = torch.randn(shape, generator=g, device="cuda", dtype=t)
    v = torch.randn(shape, generator=g, device="cuda", dtype=t)
    return k, v


def _paged(case, g, spare=0):
    """Caches, page table and lengths; `spare`: further pages for each sequence.
    The pages of a pool in use lie in no order."""
    b = case["batch"]
    order = torch.randperm(b, generator=g, device="cuda")
    lens = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")[order]
    wide = max(max(_pages(case)), 1)
    # a few pages that no sequence of this batch holds
    pool = b * (wide + spare) + 3
    ids = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = ids[: b * wide].reshape(b, wide).contiguous()
    more = ids[b * wide: b * (wide + spare)].reshape(b, spare).contiguous()
    k, v = _cache(case, g, pool)
    return {"order": order, "lens": lens, "table": table, "more": more, "k": k, "v": v}


def _rows(case, g, tokens):
    """Query, key and value heads as column blocks of one projection's rows."""
    h, hk, d = case["heads"], case["kv_heads"], case["d"]
    rows = torch.randn(tokens, (h + 2 * hk) * d, generator=g, device="cuda",
                       dtype=TYPES[case["type"]])
    return (rows[:, : h * d].view(tokens, h, d), rows[:, h * d: (h + hk) * d].view(tokens, hk, d),
            rows[:, (h + hk) * d:].view(tokens, hk, d))


def prepare(case, seed):
    g = _generator(seed)
    op, d = case["op"], case["d"]
    s = {"case": case}
    if op == "norm":
        s["q"], s["k"], _ = _rows(case, g, case["tokens"])
        s["positions"] = torch.randint(0, case["table"], (case["tokens"],), generator=g,
                                       device="cuda", dtype=torch.int32)
    elif op == "append":
        s.update(_paged(case, g))
        news = torch.tensor(_news(case), dtype=torch.int32, device="cuda")[s["order"]]
        tokens = sum(_news(case))
        s["q"], s["kn"], s["vn"] = _rows(case, g, tokens)
        s["cu"] = torch.zeros(case["batch"] + 1, dtype=torch.int32, device="cuda")
        s["cu"][1:] = news.cumsum(0)
        # the rotation's position is the slot's, or further where rows were evicted before
        seq = torch.repeat_interleave(torch.arange(case["batch"], device="cuda"), news.long())
        at = torch.arange(tokens, device="cuda") - s["cu"][seq]
        slot = s["lens"][seq] - news[seq] + at
        s["positions"] = (slot + (case["table"] - case["high"]) // 2).to(torch.int32)
    elif op == "attend":
        s.update(_paged(case, g))
        s["q"] = _rows(case, g, case["batch"])[0]
        s["weights"] = None
        if case["weights"]:
            wide = s["table"].shape[1] * case["page"]
            s["weights"] = torch.rand(case["batch"], case["kv_heads"], wide, generator=g,
                                      device="cuda")
    else:
        spare = -(-case["keep"] // case["page"])
        s.update(_paged(case, g, spare))
        wide = s["table"].shape[1] * case["page"]
        shape = (case["batch"], case["kv_heads"], wide)
        # sums of attention weights: a few positions hold most, many have none at all
        w = torch.exp(3 * torch.randn(shape, generator=g, device="cuda"))
        none = torch.rand(shape, generator=g, device="cuda") < 0.1
        s["weights"] = torch.where(none, 0.0, w)
        s["weights_out"] = torch.zeros_like(s["weights"])
    if op in ("norm", "append"):
        s["cos"], s["sin"] = _table(case, g)
        s["q_gamma"] = 1 + 0.1 * torch.randn(d, generator=g, device="cuda")
        s["k_gamma"] = 1 + 0.1 * torch.randn(d, generator=g, device="cuda")
    if own and op != "norm":
        from inferc_b200 import ops
        s["kv"] = ops.PagedKV(s["k"], s["v"], s["table"], s["lens"])  # a view of the cache, no data
    return s


def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    return {"norm": _plain_norm, "append": _plain_append, "attend": _plain_attend,
            "evict": _plain_evict}[op](s)


def _own(s, op):
    from inferc_b200 import ops
    if op == "attend":
        out = ops.PagedDecodeAttention(s["q"], s["kv"], weights=s["weights"])
        return {"out": out, "weights": s["weights"]}
    if op == "evict":
        lens, kept, weights = ops.PagedKVEvict(
            s["kv"], s["weights"], s["case"]["keep"], s["case"]["recent"], dst_table=s["more"],
            weights_out=s["weights_out"])
        return {"k": s["k"], "v": s["v"], "lens": lens, "kept": kept, "weights": weights}
    if op == "norm":
        q, k = ops.QKNormRotary(s["q"], s["k"], s["q_gamma"], s["k_gamma"], EPS, s["cos"],
                                s["sin"], s["positions"], s["case"]["interleaved"])
        return {"q": q, "k": k}
    q = ops.QKNormRotaryAppend(s["kv"], s["q"], s["kn"], s["vn"], s["q_gamma"], s["k_gamma"], EPS,
                               s["cos"], s["sin"], s["positions"], s["case"]["interleaved"],
                               s["cu"])
    return {"q": q, "k": s["k"], "v": s["v"]}


# ------------------------------------------------------------- plain forms


def _plain_heads(x, gamma, s):
    """Norm and rotation of [T, heads, d], in 32 bits, rounded once."""
    case = s["case"]
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * gamma
    at = s["positions"].long()
    c, n = s["cos"][at][:, None], s["sin"][at][:, None]
    rot, rest = y[..., : case["rot"]], y[..., case["rot"]:]
    if case["interleaved"]:
        a, b = rot[..., 0::2], rot[..., 1::2]
        turned = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    else:
        a, b = rot.chunk(2, -1)
        turned = torch.cat([a * c - b * n, b * c + a * n], -1)
    return torch.cat([turned, rest], -1).to(x.dtype)


def _plain_norm(s):
    return {"q": _plain_heads(s["q"], s["q_gamma"], s), "k": _plain_heads(s["k"], s["k_gamma"], s)}


def _plain_append(s):
    page, tokens = s["case"]["page"], s["q"].shape[0]
    token = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(s["cu"].long(), token, right=True) - 1
    slot = s["lens"].long()[seq] - s["cu"].long()[seq + 1] + token
    at = s["table"].long()[seq, slot // page]
    s["k"][at, :, slot % page] = _plain_heads(s["kn"], s["k_gamma"], s)
    s["v"][at, :, slot % page] = s["vn"]
    return {"q": _plain_heads(s["q"], s["q_gamma"], s), "k": s["k"], "v": s["v"]}


def _spread(cache, table):
    """The sequences' rows in order: [B, kv_heads, positions, d], in 32 bits."""
    x = cache[table.long()].transpose(1, 2)
    return x.flatten(2, 3).float()


def _plain_attend(s):
    case, q = s["case"], s["q"]
    b, h, d = q.shape
    hk = case["kv_heads"]
    k, v = _spread(s["k"], s["table"]), _spread(s["v"], s["table"])
    scores = q.float().view(b, hk, h // hk, d) @ k.transpose(2, 3) * d ** -0.5
    held = torch.arange(k.shape[2], device="cuda") < s["lens"][:, None]
    held = held[:, None, None]
    scores = torch.where(held, scores, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
    p = e / torch.where(held.any(-1, keepdim=True), e.sum(-1, keepdim=True), 1.0)
    out = (p @ v).reshape(b, h, d).to(q.dtype)
    if s["weights"] is not None:
        s["weights"] += p.sum(2)
    return {"out": out, "weights": s["weights"]}


def _plain_evict(s):
    keep, recent, page = s["case"]["keep"], s["case"]["recent"], s["case"]["page"]
    w, n = s["weights"], s["lens"].long()[:, None, None]
    wide, hk = w.shape[2], w.shape[1]
    j = torch.arange(wide, device="cuda")
    rank = torch.where(j >= n - recent, torch.inf, w)
    rank = torch.where(j >= n, -torch.inf, rank)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    i = torch.arange(order.shape[2], device="cuda")
    order = torch.sort(torch.where(i < n, order, wide), dim=-1).values
    held = i < n
    order = torch.where(held, order, 0)
    b = torch.arange(w.shape[0], device="cuda")[:, None, None]
    head = torch.arange(hk, device="cuda")[:, None]
    src, dst = s["table"].long()[b, order // page], s["more"].long()[b, (i // page)[None, None]]
    s["k"][dst, head, i % page] = torch.where(held[..., None], s["k"][src, head, order % page],
                                              s["k"][dst, head, i % page])
    s["v"][dst, head, i % page] = torch.where(held[..., None], s["v"][src, head, order % page],
                                              s["v"][dst, head, i % page])
    kept_w = torch.where(held, torch.gather(w, 2, order), 0.0)
    s["weights_out"][:] = torch.where(j < n, 0.0, s["weights_out"])
    s["weights_out"][..., : order.shape[2]] = torch.where(held, kept_w,
                                                          s["weights_out"][..., : order.shape[2]])
    kept = torch.full((w.shape[0], hk, keep), -1, dtype=torch.int32, device="cuda")
    kept[..., : order.shape[2]] = torch.where(held, order, -1).to(torch.int32)
    return {"k": s["k"], "v": s["v"], "lens": s["lens"].clamp(max=keep), "kept": kept,
            "weights": s["weights_out"]}


# ------------------------------------------------------------ exact values


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "append": _exact_append, "attend": _exact_attend,
            "evict": _exact_evict}[case["op"]](case, s)


def _exact_turn(case, x, gamma, s):
    """The rotation as a product of complex numbers."""
    x = x.double()
    x = gamma.double() * x / (EPS + (x * x).sum(-1, keepdim=True) / case["d"]).sqrt()
    half = case["rot"] // 2
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()].unsqueeze(1)
    y = x.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
        z = torch.complex(x[:, :, a], x[:, :, b]) * turn[:, :, i]
        y[:, :, a], y[:, :, b] = z.real, z.imag
    return y


def _exact_norm(case, s):
    return {"q": _exact_turn(case, s["q"], s["q_gamma"], s),
            "k": _exact_turn(case, s["k"], s["k_gamma"], s)}


def _exact_append(case, s):
    k, v = s["k"].double(), s["v"].double()
    kn, page = _exact_turn(case, s["kn"], s["k_gamma"], s), case["page"]
    lens, cu, table = s["lens"].tolist(), s["cu"].tolist(), s["table"].long()
    for b, n in enumerate(lens):
        new = cu[b + 1] - cu[b]
        p = torch.arange(n - new, n, device="cuda")
        at = table[b, p // page]
        k[at, :, p % page] = kn[cu[b]: cu[b + 1]]
        v[at, :, p % page] = s["vn"][cu[b]: cu[b + 1]].double()
    return {"q": _exact_turn(case, s["q"], s["q_gamma"], s), "k": k, "v": v}


def _exact_attend(case, s):
    h, hk, d, page = case["heads"], case["kv_heads"], case["d"], case["page"]
    g = h // hk
    out = torch.zeros(case["batch"], h, d, dtype=torch.float64, device="cuda")
    sums = None if s["weights"] is None else s["weights"].double()
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        pages = s["table"][b, : -(-n // page)].long()
        for i in range(hk):
            k = s["k"][pages, i].reshape(-1, d)[:n].double()
            v = s["v"][pages, i].reshape(-1, d)[:n].double()
            scores = k @ s["q"][b, i * g: (i + 1) * g].double().T / math.sqrt(d)
            p = torch.softmax(scores, 0)
            out[b, i * g: (i + 1) * g] = p.T @ v
            if sums is not None:
                sums[b, i, :n] += p.sum(1)
    return {"out": out, "weights": sums}


def _exact_evict(case, s):
    keep, recent, page = case["keep"], case["recent"], case["page"]
    k, v = s["k"].double(), s["v"].double()
    wout = s["weights_out"].double()
    kept = torch.full((case["batch"], case["kv_heads"], keep), -1, dtype=torch.int32)
    lens = s["lens"].tolist()
    for b, n in enumerate(lens):
        m = min(n, keep)
        for i in range(case["kv_heads"]):
            if n <= keep:
                at = torch.arange(n, device="cuda")
            else:
                old = s["weights"][b, i, : n - recent]
                best = torch.sort(-old, stable=True).indices[: keep - recent]
                last = torch.arange(n - recent, n, device="cuda")
                at = torch.cat([torch.sort(best).values, last])
            kept[b, i, :m] = at.to(torch.int32).cpu()
            to = torch.arange(m, device="cuda")
            src, dst = s["table"][b, at // page].long(), s["more"][b, to // page].long()
            k[dst, i, to % page] = s["k"][src, i, at % page].double()
            v[dst, i, to % page] = s["v"][src, i, at % page].double()
            wout[b, i, :n] = 0
            wout[b, i, :m] = s["weights"][b, i, at].double()
    return {"k": k, "v": v, "lens": torch.tensor([min(n, keep) for n in lens], dtype=torch.int32),
            "kept": kept, "weights": wout}
