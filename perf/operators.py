"""Timed cases of the paged key/value cache operators: attention of new tokens
over a paged cache (full, or a sliding window with first tokens that stay
visible), the same with the accumulated attention weights of the cache slots,
and the eviction of cache slots by those weights.

`run` computes a case in its plain form (elementary torch operations in 32
bits) or, with `own` set, through this package's entry points. `exact` has the
same results in 64 bits.

A case: `kind` "attend" (with `weights`: the accumulated weights too) or
"evict"; `batch` sequences whose lengths lie in [kv * (1 - spread), kv]
cache slots, the new tokens included, and which bring 1..`q` new tokens each
(`q` all of them where `even` is set); `heads` / `kv_heads` query and
key/value heads of `dim` elements; `page` cache slots per page; `window` and
`sinks` as the operators take them (window 0: every earlier slot is visible)."""
import math
import random

import torch

own = False

HEADS = [(32, 8, 128), (64, 8, 128), (16, 4, 64), (16, 16, 64), (28, 4, 128), (12, 2, 64)]


def _attend(name, batch, q, kv, heads, kv_heads, dim, page, dtype, window=0, sinks=0, spread=0.0, even=True,
            weights=False):
    return {"name": name, "kind": "attend", "batch": batch, "q": q, "kv": kv, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "dtype": dtype, "window": window, "sinks": sinks, "spread": spread,
            "even": even, "weights": weights}


def _evict(name, batch, kv, budget, recent, sinks, kv_heads, dim, page, dtype, spread=0.0):
    return {"name": name, "kind": "evict", "batch": batch, "kv": kv, "budget": budget, "recent": recent,
            "sinks": sinks, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "spread": spread}


def listed():
    return [
        # the first tokens of an answer to a short prompt, one user: latency alone counts
        _attend("decode_one", 1, 1, 97, 16, 4, 64, 16, "float16"),
        # one decode step of a busy server, sequences of every length
        _attend("decode_batch", 32, 1, 4096, 32, 8, 128, 16, "float16", spread=0.95),
        # one decode step over two very long documents
        _attend("decode_long", 2, 1, 131072, 64, 8, 128, 64, "bfloat16", spread=0.4),
        # decode with a sliding window and first tokens that stay visible, pages older than the window still held
        _attend("decode_window", 24, 1, 16384, 32, 8, 128, 32, "bfloat16", window=4096, sinks=4, spread=0.9),
        # checking a few drafted tokens per sequence at once
        _attend("verify_draft", 16, 7, 6000, 32, 8, 128, 16, "float16", spread=0.7, even=False),
        # a mixed step: sequences that decode beside chunks of prompts
        _attend("chunk_mixed", 8, 512, 8192, 32, 8, 128, 64, "bfloat16", spread=0.9, even=False),
        # the last chunk of a long prompt
        _attend("prompt_chunk", 1, 4096, 16384, 32, 8, 128, 64, "bfloat16"),
        # a chunk of a long prompt under a sliding window, one key/value head per query head
        _attend("prompt_window", 2, 3000, 11111, 16, 16, 64, 32, "float16", window=1024, sinks=4, spread=0.2),
        # a decode step of a server that keeps the weights for eviction
        _attend("decode_weights", 16, 1, 8192, 32, 8, 128, 16, "float16", spread=0.8, weights=True),
        # a chunk of a prompt whose weights decide what is kept of it
        _attend("chunk_weights", 2, 1024, 4096, 32, 8, 128, 64, "bfloat16", spread=0.3, weights=True),
        # a small cache brought back to its budget while decoding
        _evict("evict_step", 4, 1100, 1024, 128, 4, 4, 64, 16, "float16", spread=0.3),
        # long prompts cut to a quarter before decoding begins
        _evict("evict_prompt", 8, 32768, 8192, 1024, 4, 8, 128, 64, "bfloat16", spread=0.5),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype, page = rng.choice(["float16", "bfloat16"]), rng.choice([16, 32, 64])
    heads, kv_heads, dim = rng.choice(HEADS)
    kind = rng.choice(["decode", "decode", "window", "draft", "chunk", "prompt", "weights", "evict"])
    spread = rng.choice([0.0, 0.5, 0.95])
    if kind == "evict":
        batch = _log(rng, 1, 8)
        kv = _log(rng, 65, 32768)
        budget = max(16, int(kv * rng.uniform(0.1, 0.95)))
        c = _evict("", batch, kv, budget, int(budget * rng.uniform(0, 0.5)), rng.randint(0, 8), kv_heads, dim, page,
                   dtype, spread)
    elif kind in ("chunk", "prompt") or (kind == "weights" and rng.random() < 0.5):
        batch = _log(rng, 1, 8) if kind != "prompt" else 1
        q = _log(rng, 33, 512 if kind == "chunk" else 4096 if kind == "prompt" else 1024)
        kv = q + _log(rng, 1, 8192)
        window = rng.choice([0, 0, _log(rng, 64, 4096)])
        while batch > 1 and batch * q * kv > 20e6:
            batch -= 1
        c = _attend("", batch, q, kv, heads, kv_heads, dim, page, dtype, window, rng.randint(0, 8) if window else 0,
                    spread, rng.random() < 0.5, kind == "weights")
    else:
        batch, q = _log(rng, 1, 64), rng.randint(2, 8) if kind == "draft" else 1
        kv = q + _log(rng, 1, 65536)
        batch = max(1, min(batch, 65536 // kv))
        window = _log(rng, 16, 4096) if kind == "window" else 0
        c = _attend("", batch, q, kv, heads, kv_heads, dim, page, dtype, window, rng.randint(0, 8) if window else 0,
                    spread, rng.random() < 0.5, kind == "weights")
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, cache slots) of each sequence: the first is the longest, the others spread below it."""
    rng = random.Random(case["batch"] * 1000003 + case["kv"])
    got = []
    for b in range(case["batch"]):
        q = case.get("q", 0)
        if b and not case.get("even", True):
            q = rng.randint(1, q)
        low = max(q, int(case["kv"] * (1 - case["spread"])), 1)
        got.append((q, case["kv"] if b == 0 else rng.randint(low, max(low, case["kv"]))))
    return got


def work(case):
    size, dim, hk = 2, case["dim"], case["kv_heads"]
    if case["kind"] == "evict":
        kept = sum(min(n, case["budget"]) for _, n in _lengths(case))
        read = sum(n for _, n in _lengths(case))
        return {"bytes": hk * (kept * (2 * 2 * dim * size + 8) + read * 4), "flops": 0}
    window, sinks, hq = case["window"], case["sinks"], case["heads"]
    slots = pairs = tokens = slots_all = 0
    for q, n in _lengths(case):
        tokens += q
        slots_all += n
        first = n - q  # cache slot of the first new token
        if not window:
            slots += first
            pairs += q * first + q * (q + 1) // 2
        else:
            start = max(0, first - window + 1)
            slots += first - start + min(sinks, start)
            for p in range(first, n):
                pairs += min(p + 1, window) + min(sinks, max(0, p + 1 - window))
    moved = hk * dim * 2 * size * (slots + 2 * tokens)  # old keys and values in, new ones in and out
    moved += 2 * tokens * hq * dim * size + tokens * hq * 4
    if case["weights"]:
        moved += hk * 8 * (slots + tokens)
    return {"bytes": moved, "flops": 4 * dim * hq * pairs}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    hk, dim, page = case["kv_heads"], case["dim"], case["page"]
    lengths = _lengths(case)
    batch, longest = len(lengths), max(n for _, n in lengths)
    columns = -(-longest // page)
    rows = -(-case["budget"] // page) if case["kind"] == "evict" else 0
    pages = batch * (columns + rows) + 3
    order = torch.randperm(pages, generator=g, device="cuda").int()
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    k_pages, v_pages = randn(pages, page, hk, dim), randn(pages, page, hk, dim)
    s = {"case": case, "k_pages": k_pages, "v_pages": v_pages,
         "page_table": order[: batch * columns].reshape(batch, columns).contiguous(),
         "kv_len": torch.tensor([n for _, n in lengths], dtype=torch.int32, device="cuda")}
    # weights as attention leaves them: most near nothing, some slots never looked at, a few heavy ones
    if case["kind"] == "evict" or case["weights"]:
        w = torch.exp(2.5 * torch.randn(batch, hk, columns * page, generator=g, device="cuda") - 3)
        w[torch.rand(w.shape, generator=g, device="cuda") < 0.15] = 0
        s["weights"] = w
    if case["kind"] == "evict":
        s["new_table"] = order[batch * columns: batch * (columns + rows)].reshape(batch, rows).contiguous()
        s["kept"] = torch.empty(batch, hk, case["budget"], dtype=torch.int32, device="cuda")
        s["new_len"] = torch.empty(batch, dtype=torch.int32, device="cuda")
        s["new_weights"] = torch.empty(batch, hk, case["budget"], device="cuda")
    else:
        hq = case["heads"]
        # the first slots draw attention, as the first tokens of a text do
        sink = torch.nn.functional.normalize(torch.randn(hk, dim, generator=g, device="cuda"), dim=-1)
        heavy = s["page_table"][:, 0].long()
        k_pages[heavy, :2] += (3.0 * dim ** 0.5 * sink).to(dtype)
        tokens = sum(q for q, _ in lengths)
        # one projection's result holds the queries and the new keys and values
        qkv = randn(tokens, hq + 2 * hk, dim)
        qkv[:, :hq] += sink.repeat_interleave(hq // hk, 0).to(dtype)
        s["q"], s["k_new"], s["v_new"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        starts = [0]
        for q, _ in lengths:
            starts.append(starts[-1] + q)
        s["q_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["max_q"] = max(q for q, _ in lengths)
        s["output"] = torch.empty(tokens, hq, dim, dtype=dtype, device="cuda")
        s["lse"] = torch.empty(tokens, hq, device="cuda")
        if own:
            from leanstream_b200 import PagedAttention

            s["attention"] = PagedAttention(hq, hk, dim, page_size=page, dtype=dtype, max_sequences=batch,
                                            max_tokens=tokens, max_queries=s["max_q"],
                                            max_weights_length=columns * page if case["weights"] else 0)
    return s


def _updated(s):
    names = ("output", "lse", "weights", "k_pages", "v_pages")
    if s["case"]["kind"] == "evict":
        names = ("kept", "new_len", "new_weights", "k_pages", "v_pages")
    return {n: s[n] for n in names if n in s}


def run(s):
    case = s["case"]
    if not own:
        (_plain_evict if case["kind"] == "evict" else _plain_attend)(s)
    elif case["kind"] == "evict":
        from leanstream_b200 import evict_cache

        evict_cache(k_pages=s["k_pages"], v_pages=s["v_pages"], page_table=s["page_table"], kv_len=s["kv_len"],
                    weights=s["weights"], budget=case["budget"], sinks=case["sinks"], recent=case["recent"],
                    new_table=s["new_table"], new_len=s["new_len"], kept=s["kept"], new_weights=s["new_weights"])
    else:
        s["attention"].run(q=s["q"], k_new=s["k_new"], v_new=s["v_new"], k_pages=s["k_pages"], v_pages=s["v_pages"],
                           page_table=s["page_table"], kv_len=s["kv_len"], q_start=s["q_start"], max_q=s["max_q"],
                           output=s["output"], lse=s["lse"], window=case["window"], sinks=case["sinks"],
                           weights=s.get("weights"))
    return _updated(s)


def _plain_attend(s):
    case = s["case"]
    hk, dim, page, most = case["kv_heads"], case["dim"], case["page"], s["max_q"]
    group = case["heads"] // hk
    table, kv_len, q_start = s["page_table"].long(), s["kv_len"].long(), s["q_start"].long()
    batch, length = table.shape[0], table.shape[1] * page
    new = (q_start[1:] - q_start[:-1])[:, None]  # [batch, 1]
    t = torch.arange(most, device="cuda")[None]
    slot = kv_len[:, None] - new + t  # [batch, most]: the new tokens' cache slots
    real = t < new
    # the new keys and values go to their slots
    b_at, t_at = real.nonzero(as_tuple=True)
    at = slot[b_at, t_at]
    token = q_start[b_at] + t_at
    for pages, fresh in ((s["k_pages"], s["k_new"]), (s["v_pages"], s["v_new"])):
        pages[table[b_at, at // page], at % page] = fresh[token]
    k = s["k_pages"][table].reshape(batch, length, hk, dim).permute(0, 2, 3, 1).float()
    q = s["q"].new_zeros(batch, most, hk * group, dim)
    q[b_at, t_at] = s["q"][token]
    q = q.float().reshape(batch, most, hk, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, hk, group * most, dim)
    x = torch.matmul(q, k) * dim ** -0.5
    del k
    x = x.reshape(batch, hk, group, most, length)
    n = torch.arange(length, device="cuda")
    seen = (n <= slot[..., None]) & real[..., None]
    if case["window"]:
        seen &= (n > slot[..., None] - case["window"]) | (n < case["sinks"])
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp_min(-3e38)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    lse = (torch.log(total) + top)[..., 0]
    x = x / total.clamp_min(1e-38)
    v = s["v_pages"][table].reshape(batch, length, hk, dim).permute(0, 2, 1, 3).float()
    o = torch.matmul(x.reshape(batch, hk, group * most, length), v).reshape(batch, hk, group, most, dim)
    s["output"][token] = o.permute(0, 3, 1, 2, 4).reshape(batch, most, hk * group, dim)[b_at, t_at].to(s["q"].dtype)
    s["lse"][token] = lse.permute(0, 3, 1, 2).reshape(batch, most, hk * group)[b_at, t_at]
    if case["weights"]:
        got = x.sum((2, 3))
        fresh = (n >= (kv_len[:, None] - new))[:, None]
        held = (n < kv_len[:, None])[:, None]
        w = s["weights"]
        w.copy_(torch.where(held, got + torch.where(fresh, torch.zeros_like(w), w), w))


def _plain_evict(s):
    case = s["case"]
    page, budget = case["page"], case["budget"]
    w, kv_len = s["weights"], s["kv_len"].long()
    batch, hk, length = w.shape
    n = torch.arange(length, device="cuda")[None, None]
    count = kv_len[:, None, None]
    rank = torch.where((n < case["sinks"]) | (n >= count - case["recent"]), torch.full_like(w, math.inf), w)
    rank = torch.where(n < count, rank, torch.full_like(w, -math.inf))
    at = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    if at.shape[-1] < budget:
        at = torch.cat([at, at.new_full((batch, hk, budget - at.shape[-1]), length)], -1)
    at = torch.sort(torch.where(at < count, at, torch.full_like(at, length)), dim=-1).values
    real = at < count
    s["kept"].copy_(torch.where(real, at, torch.full_like(at, -1)))
    s["new_len"].copy_(kv_len.clamp_max(budget))
    b, h, j = real.nonzero(as_tuple=True)
    source = at[b, h, j]
    s["new_weights"].zero_()
    s["new_weights"][b, h, j] = w[b, h, source]
    old, new = s["page_table"].long()[b, source // page], s["new_table"].long()[b, j // page]
    for pages in (s["k_pages"], s["v_pages"]):
        pages[new, j % page, h] = pages[old, source % page, h]


def exact(case, seed):
    s = prepare(case, seed)
    page, hk, dim = case["page"], case["kv_heads"], case["dim"]
    table = s["page_table"].long()
    if case["kind"] == "evict":
        weights, new = s["weights"].double(), s["new_table"].long()
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        new_weights = torch.zeros(s["new_weights"].shape, dtype=torch.float64, device="cuda")
        for b, (_, n) in enumerate(_lengths(case)):
            for h in range(hk):
                keep = list(range(n))
                if n > case["budget"]:
                    sinks, recent = list(range(case["sinks"])), list(range(n - case["recent"], n))
                    value = weights[b, h, :n].tolist()
                    middle = sorted(range(case["sinks"], n - case["recent"]), key=lambda i: (-value[i], i))
                    keep = sinks + sorted(middle[: case["budget"] - len(sinks) - len(recent)]) + recent
                keep, to = torch.tensor(keep, device="cuda"), torch.arange(len(keep), device="cuda")
                new_weights[b, h, to] = weights[b, h, keep]
                for pages in (k_pages, v_pages):
                    pages[new[b, to // page], to % page, h] = pages[table[b, keep // page], keep % page, h]
        return {"kept": None, "new_len": None, "new_weights": new_weights, "k_pages": k_pages, "v_pages": v_pages}
    hq, group = case["heads"], case["heads"] // hk
    output = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if case["weights"] else None
    at = 0
    for b, (count, n) in enumerate(_lengths(case)):
        tokens = slice(at, at + count)
        i = torch.arange(n, device="cuda")
        where = table[b, i // page]
        for pages, fresh in ((s["k_pages"], s["k_new"]), (s["v_pages"], s["v_new"])):
            pages[where[n - count:], i[n - count:] % page] = fresh[tokens]
        keys, values = s["k_pages"][where, i % page].double(), s["v_pages"][where, i % page].double()
        position = torch.arange(n - count, n, device="cuda")[:, None]
        hidden = i[None] > position
        if case["window"]:
            hidden |= (i[None] <= position - case["window"]) & (i[None] >= case["sinks"])
        if weights is not None:
            weights[b, :, n - count:n] = 0
        for h in range(hq):
            z = (s["q"][tokens, h].double() @ keys[:, h // group].T) / math.sqrt(dim)
            z[hidden] = -math.inf
            lse[tokens, h] = torch.logsumexp(z, -1)
            z = torch.softmax(z, -1)
            output[tokens, h] = z @ values[:, h // group]
            if weights is not None:
                weights[b, h // group, :n] += z.sum(0)
        at += count
    got = {"output": output, "lse": lse, "weights": weights, "k_pages": s["k_pages"].double(),
           "v_pages": s["v_pages"].double()}
    return got if weights is not None else {k: v for k, v in got.items() if k != "weights"}
