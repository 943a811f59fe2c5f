"""Timed cases of the operators that fill and read a paged key/value cache in
16 or 8 bits: appending the new tokens' keys and values with the position
rotation applied on the way (queries rotated too), and attention over a cache
of 8-bit integers with a power-of-two scale for each block of 16 slots and head.

`run` computes a case in its plain form (elementary torch operations in 32
bits) or, with `own` set, through this package's entry points. `exact` has the
same results in 64 bits.

A case: `kind` "append" or "attend"; `batch` sequences whose lengths lie in
[kv * (1 - spread), kv] cache slots, the new tokens included, and which bring
1..`q` new tokens each (`q` all of them where `even` is set); `heads` /
`kv_heads` query and key/value heads of `dim` elements; `page` cache slots per
page. Append: `rotary` elements of a head are rotated, as two halves or, with
`interleaved`, as neighbours; positions lie `ahead` of the slots (a cache that
was cut back); `int8` is the cache in 8 bits, whose contents are returned as
the values that they stand for. Attend: `window` and `sinks` as the operator
takes them (window 0: every earlier slot is visible)."""
import math
import random

import torch

own = False

BLOCK = 16  # slots that share a scale
HEADS = [(32, 8, 128), (64, 8, 128), (16, 4, 64), (16, 16, 64), (28, 4, 128), (12, 2, 64)]


def _append(name, batch, q, kv, heads, kv_heads, dim, page, dtype, int8, rotary, interleaved=False, ahead=0,
            spread=0.0, even=True):
    return {"name": name, "kind": "append", "batch": batch, "q": q, "kv": kv, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "dtype": dtype, "int8": int8, "rotary": rotary, "interleaved": interleaved,
            "ahead": ahead, "spread": spread, "even": even}


def _attend(name, batch, q, kv, heads, kv_heads, dim, page, dtype, window=0, sinks=0, spread=0.0, even=True):
    return {"name": name, "kind": "attend", "batch": batch, "q": q, "kv": kv, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "dtype": dtype, "window": window, "sinks": sinks, "spread": spread,
            "even": even}


def listed():
    return [
        # the token that one user decodes, 16-bit cache: latency alone counts
        _append("append_one", 1, 1, 97, 16, 4, 64, 16, "float16", False, 64),
        # a prompt's chunk on its way into a 16-bit cache
        _append("append_prompt", 1, 4096, 8192, 32, 8, 128, 64, "bfloat16", False, 128),
        # one decode step of a busy server whose answers have just begun, cache in 8 bits, positions past an eviction
        _append("append_step_8", 64, 1, 60, 64, 8, 128, 16, "bfloat16", True, 128, ahead=5000, spread=0.8),
        # chunks of several prompts into a cache in 8 bits; half of each head is rotated, as neighbours
        _append("append_chunk_8", 4, 900, 1000, 32, 8, 128, 32, "float16", True, 64, True, spread=0.4, even=False),
        # the first tokens of an answer to a short prompt, one user
        _attend("decode_one_8", 1, 1, 130, 16, 4, 64, 16, "float16"),
        # one decode step of a busy server, sequences of every length
        _attend("decode_batch_8", 48, 1, 5000, 32, 8, 128, 16, "float16", spread=0.95),
        # one decode step over two very long documents
        _attend("decode_long_8", 2, 1, 150000, 64, 8, 128, 64, "bfloat16", spread=0.4),
        # decode with a sliding window and first tokens that stay visible
        _attend("decode_window_8", 20, 1, 20000, 64, 8, 128, 32, "bfloat16", window=4096, sinks=4, spread=0.9),
        # checking a few drafted tokens per sequence at once
        _attend("verify_draft_8", 12, 5, 9000, 32, 8, 128, 16, "float16", spread=0.7, even=False),
        # a mixed step: short runs beside chunks of prompts
        _attend("chunk_mixed_8", 6, 700, 9000, 32, 8, 128, 64, "bfloat16", spread=0.9, even=False),
        # the last chunk of a long prompt
        _attend("prompt_chunk_8", 1, 4096, 16384, 32, 8, 128, 64, "bfloat16"),
        # chunks of two prompts, one key/value head per query head
        _attend("prompt_heads_8", 2, 2500, 7777, 16, 16, 64, 32, "float16", spread=0.2),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype, page = rng.choice(["float16", "bfloat16"]), rng.choice([16, 32, 64])
    heads, kv_heads, dim = rng.choice(HEADS)
    spread = rng.choice([0.0, 0.5, 0.95])
    kind = rng.choice(["append", "append", "decode", "decode", "window", "draft", "chunk", "prompt"])
    if kind == "append":
        q = 1 if rng.random() < 0.5 else _log(rng, 2, 4096)
        batch = max(1, min(_log(rng, 1, 64), 4096 // q))
        c = _append("", batch, q, q + _log(rng, 1, 150), heads, kv_heads, dim, page, dtype, rng.random() < 0.6,
                    rng.choice([dim, dim, 32, 48]), rng.random() < 0.4, rng.choice([0, _log(rng, 1, 30000)]), spread,
                    rng.random() < 0.5)
    elif kind in ("chunk", "prompt"):
        batch = _log(rng, 1, 8) if kind == "chunk" else 1
        q = _log(rng, 33, 700 if kind == "chunk" else 4096)
        kv = q + _log(rng, 1, 8192)
        window = rng.choice([0, 0, _log(rng, 64, 4096)])
        while batch > 1 and batch * q * kv > 20e6:
            batch -= 1
        c = _attend("", batch, q, kv, heads, kv_heads, dim, page, dtype, window, rng.randint(0, 8) if window else 0,
                    spread, rng.random() < 0.5)
    else:
        batch, q = _log(rng, 1, 64), rng.randint(2, 8) if kind == "draft" else 1
        kv = q + _log(rng, 1, 65536)
        batch = max(1, min(batch, 65536 // kv))
        window = _log(rng, 16, 4096) if kind == "window" else 0
        c = _attend("", batch, q, kv, heads, kv_heads, dim, page, dtype, window, rng.randint(0, 8) if window else 0,
                    spread, rng.random() < 0.5)
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, cache slots) of each sequence: the first is the longest, the others spread below it."""
    rng = random.Random(case["batch"] * 1000003 + case["kv"])
    got = []
    for b in range(case["batch"]):
        q = case["q"]
        if b and not case["even"]:
            q = rng.randint(1, q)
        low = max(q, int(case["kv"] * (1 - case["spread"])), 1)
        got.append((q, case["kv"] if b == 0 else rng.randint(low, max(low, case["kv"]))))
    return got


def work(case):
    dim, hk, hq = case["dim"], case["kv_heads"], case["heads"]
    lengths = _lengths(case)
    tokens = sum(q for q, _ in lengths)
    if case["kind"] == "append":
        blocks = sum((n - 1) // BLOCK - (n - q) // BLOCK + 1 for q, n in lengths)
        # queries in and out, keys, values and angles in
        moved = tokens * (4 * hq * dim + 4 * hk * dim + 4 * case["rotary"])
        moved += tokens * 2 * hk * dim + 2 * hk * blocks if case["int8"] else tokens * 4 * hk * dim
        return {"bytes": moved, "flops": 3 * tokens * (hq + hk) * case["rotary"]}
    window, sinks = case["window"], case["sinks"]
    slots = pairs = 0
    for q, n in lengths:
        first = n - q  # cache slot of the first new token
        if not window:
            slots += n
            pairs += q * first + q * (q + 1) // 2
        else:
            start = max(0, first - window + 1)
            slots += n - start + min(sinks, start)
            for p in range(first, n):
                pairs += min(p + 1, window) + min(sinks, max(0, p + 1 - window))
    moved = hk * slots * 2 * (dim + 1 / BLOCK) + tokens * hq * (4 * dim + 4)
    return {"bytes": moved, "flops": 4 * dim * hq * pairs}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    hk, hq, dim, page = case["kv_heads"], case["heads"], case["dim"], case["page"]
    lengths = _lengths(case)
    batch, longest, tokens = len(lengths), max(n for _, n in lengths), sum(q for q, _ in lengths)
    columns = -(-longest // page)
    pages = batch * columns + 3
    order = torch.randperm(pages, generator=g, device="cuda").int()
    starts = [0]
    for q, _ in lengths:
        starts.append(starts[-1] + q)
    s = {"case": case, "page_table": order[: batch * columns].reshape(batch, columns).contiguous(),
         "kv_len": torch.tensor([n for _, n in lengths], dtype=torch.int32, device="cuda"),
         "q_start": torch.tensor(starts, dtype=torch.int32, device="cuda"), "max_q": max(q for q, _ in lengths)}
    if case.get("int8", True):
        # codes as blocks have them: the largest of each near 127, scales that differ from block to block
        def codes():
            made = torch.empty(pages, page, hk, dim, dtype=torch.int8, device="cuda")
            for at in range(0, pages, 4096):
                part = made[at:at + 4096]
                part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(32).round_().clamp_(-127, 127))
            return made

        s["k_pages"], s["v_pages"] = codes(), codes()
        s["exponents"] = torch.randint(-6, -3, (pages, hk, page // BLOCK, 2), dtype=torch.int8, device="cuda",
                                       generator=g)
    else:
        s["k_pages"], s["v_pages"] = (torch.randn(pages, page, hk, dim, generator=g, device="cuda", dtype=dtype)
                                      for _ in range(2))
    # one projection's result holds the queries and the new keys and values
    qkv = torch.randn(tokens, hq + 2 * hk, dim, generator=g, device="cuda", dtype=dtype)
    s["q"] = qkv[:, :hq]
    if case["kind"] == "append":
        s["k_new"], s["v_new"] = qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        s["v_new"] *= 0.5
        s["q_out"] = torch.empty(tokens, hq, dim, dtype=dtype, device="cuda")
        slot = torch.cat([torch.arange(n - q, n) for q, n in lengths])
        s["positions"] = (slot + case["ahead"]).int().cuda() if case["ahead"] else None
        half = case["rotary"] // 2
        angle = torch.arange(longest + case["ahead"], device="cuda").double()[:, None] * \
            10000.0 ** (-torch.arange(half, device="cuda").double() / half)
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], -1).float()
    else:
        # the first slots draw attention, as the first tokens of a text do
        sink = torch.nn.functional.normalize(torch.randn(hk, dim, generator=g, device="cuda"), dim=-1)
        heavy = s["page_table"][:, 0].long()
        s["exponents"][heavy, :, 0, 0] = -4
        first = torch.randn(batch, 2, hk, dim, generator=g, device="cuda") + 3.0 * dim ** 0.5 * sink
        s["k_pages"][heavy, :2] = first.mul_(16).round_().clamp_(-127, 127).to(torch.int8)
        s["q"] += sink.repeat_interleave(hq // hk, 0).to(dtype)
        s["output"] = torch.empty(tokens, hq, dim, dtype=dtype, device="cuda")
        s["lse"] = torch.empty(tokens, hq, device="cuda")
        if own:
            from leanstream_b200 import PagedAttention

            s["attention"] = PagedAttention(hq, hk, dim, page_size=page, dtype=dtype, cache_dtype="int8",
                                            max_sequences=batch, max_tokens=tokens, max_queries=s["max_q"])
    return s


def run(s):
    case = s["case"]
    if case["kind"] == "attend":
        if not own:
            _plain_attend(s)
        else:
            s["attention"].run(q=s["q"], k_pages=s["k_pages"], v_pages=s["v_pages"], exponents=s["exponents"],
                               page_table=s["page_table"], kv_len=s["kv_len"], q_start=s["q_start"],
                               max_q=s["max_q"], output=s["output"], lse=s["lse"], window=case["window"],
                               sinks=case["sinks"])
        return {"output": s["output"], "lse": s["lse"]}
    if not own:
        _plain_append(s)
    else:
        from leanstream_b200 import append_cache

        append_cache(q=s["q"], q_out=s["q_out"], k_new=s["k_new"], v_new=s["v_new"], k_pages=s["k_pages"],
                     v_pages=s["v_pages"], exponents=s.get("exponents"), page_table=s["page_table"],
                     q_start=s["q_start"], kv_len=s["kv_len"], cos_sin=s["cos_sin"], positions=s["positions"],
                     interleaved=case["interleaved"])
    if not case["int8"]:
        return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    step = torch.exp2(s["exponents"]).to(s["q"].dtype)  # (the products below are exact)
    return {"q": s["q_out"], "k_pages": _values(s["k_pages"], step[..., 0]),
            "v_pages": _values(s["v_pages"], step[..., 1])}


def _values(codes, step):
    """What codes [pages][page][kv_heads][dim] stand for; step [pages][kv_heads][blocks]."""
    pages, page, hk, dim = codes.shape
    blocks = codes.view(pages, page // BLOCK, BLOCK, hk, dim)
    return (blocks * step.transpose(1, 2)[:, :, None, :, None]).view(codes.shape)


def _tokens(s):
    """For each new token: its sequence, its cache slot, and whether it is real; [batch, max_q] each but the first."""
    kv_len, q_start = s["kv_len"].long(), s["q_start"].long()
    new = (q_start[1:] - q_start[:-1])[:, None]
    t = torch.arange(s["max_q"], device="cuda")[None]
    real = t < new
    b_at, t_at = real.nonzero(as_tuple=True)
    return b_at, t_at, q_start[b_at] + t_at, kv_len[:, None] - new + t, real


def _rotate(x, cos, sin, rotary, interleaved):
    """x [tokens][heads][dim], cos and sin [tokens][rotary / 2], in 32 bits."""
    y, half = x.float(), rotary // 2
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = y[..., 0:rotary:2], y[..., 1:rotary:2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), y[..., rotary:]], -1)
    a, b = y[..., :half], y[..., half:rotary]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., rotary:]], -1)


def _plain_append(s):
    case = s["case"]
    page, rotary, hk, dim = case["page"], case["rotary"], case["kv_heads"], case["dim"]
    table = s["page_table"].long()
    b_at, t_at, token, slot, _ = _tokens(s)
    at = slot[b_at, t_at]
    where = s["positions"][token].long() if s["positions"] is not None else at
    angle = s["cos_sin"][where]
    cos, sin = angle[:, :rotary // 2], angle[:, rotary // 2:]
    q = _rotate(s["q"][token], cos, sin, rotary, case["interleaved"])
    k = _rotate(s["k_new"][token], cos, sin, rotary, case["interleaved"])
    s["q_out"][token] = q.to(s["q"].dtype)
    if not case["int8"]:
        s["k_pages"][table[b_at, at // page], at % page] = k.to(s["q"].dtype)
        s["v_pages"][table[b_at, at // page], at % page] = s["v_new"][token]
        return
    # the blocks with new rows, one after another: (sequence, block), their first slots and pages
    blocks = table.shape[1] * (page // BLOCK)
    key, which = torch.unique(b_at * blocks + at // BLOCK, return_inverse=True)
    b, first = key // blocks, key % blocks * BLOCK
    at_page, in_page = table[b, first // page], first % page
    old_rows = (slot[b, 0] - first).clamp(0, BLOCK)  # rows of the block that were there before
    row = in_page[:, None] + torch.arange(BLOCK, device="cuda")
    lowest, highest = (-24, 9) if s["q"].dtype == torch.float16 else (-126, 120)
    for kv, pages, fresh in ((0, s["k_pages"], k), (1, s["v_pages"], s["v_new"][token].float())):
        most = torch.zeros(len(key), hk, device="cuda")
        most.index_reduce_(0, which, fresh.abs().amax(-1), "amax")
        # the smallest power of two of which 127 reach the largest value
        mantissa, power = torch.frexp(most)
        e = (power - 7 + (mantissa > 127 / 128)).clamp(lowest, highest)
        e = torch.where(most > 0, e, torch.full_like(e, lowest))
        before = s["exponents"][at_page, :, in_page // BLOCK, kv].int()
        e = torch.where(old_rows[:, None] > 0, torch.maximum(e, before), e)
        # older rows of the block, rounded to the new step
        was = pages[at_page[:, None], row]
        now = torch.round(was.float() * torch.exp2((before - e).float())[:, None, :, None]).to(torch.int8)
        old = torch.arange(BLOCK, device="cuda") < old_rows[:, None]
        pages[at_page[:, None], row] = torch.where(old[..., None, None], now, was)
        code = torch.round(fresh * torch.exp2(-e.float())[which][..., None]).clamp(-127, 127)
        pages[table[b_at, at // page], at % page] = code.to(torch.int8)
        s["exponents"][at_page, :, in_page // BLOCK, kv] = e.to(torch.int8)


def _plain_attend(s):
    case = s["case"]
    hk, dim, page, most = case["kv_heads"], case["dim"], case["page"], s["max_q"]
    group = case["heads"] // hk
    table = s["page_table"].long()
    batch, length = table.shape[0], table.shape[1] * page
    b_at, t_at, token, slot, real = _tokens(s)
    step = torch.exp2(s["exponents"])[table]  # [batch, columns, kv_heads, blocks, 2]

    def held(codes, kv):  # [batch, kv_heads, length, dim]
        got = codes[table].view(batch, -1, page // BLOCK, BLOCK, hk, dim)
        got = got * step[..., kv].transpose(2, 3)[:, :, :, None, :, None]
        return got.view(batch, length, hk, dim).transpose(1, 2)

    q = s["q"].new_zeros(batch, most, hk * group, dim)
    q[b_at, t_at] = s["q"][token]
    q = q.float().reshape(batch, most, hk, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, hk, group * most, dim)
    x = torch.matmul(q, held(s["k_pages"], 0).transpose(2, 3)) * dim ** -0.5
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
    o = torch.matmul(x.reshape(batch, hk, group * most, length), held(s["v_pages"], 1))
    o = o.reshape(batch, hk, group, most, dim)
    s["output"][token] = o.permute(0, 3, 1, 2, 4).reshape(batch, most, hk * group, dim)[b_at, t_at].to(s["q"].dtype)
    s["lse"][token] = lse.permute(0, 3, 1, 2).reshape(batch, most, hk * group)[b_at, t_at]


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if case["kind"] == "append" else _exact_attend(s)


def _two_to(e):
    """2 ** e in 64 bits with no rounding, for whole e."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_append(s):
    case = s["case"]
    page, hk, dim, rotary = case["page"], case["kv_heads"], case["dim"], case["rotary"]
    half, table = rotary // 2, s["page_table"].long()
    # pairs of elements that turn together
    i = torch.arange(half, device="cuda")
    low, high = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    q, k, v = s["q"].double(), s["k_new"].double(), s["v_new"].double()
    pools = [s["k_pages"].double(), s["v_pages"].double()]
    if case["int8"]:
        for kv in (0, 1):
            scale = _two_to(s["exponents"][..., kv])
            pools[kv] *= scale.repeat_interleave(BLOCK, 2).transpose(1, 2)[..., None]
    lowest, highest = (-24, 9) if s["q"].dtype == torch.float16 else (-126, 120)
    at = 0
    for b, (count, n) in enumerate(_lengths(case)):
        slots = torch.arange(n - count, n, device="cuda")
        turn = s["cos_sin"][slots + case["ahead"]].double()
        cos, sin = turn[:, None, :half], turn[:, None, half:]
        for x in (q[at:at + count], k[at:at + count]):
            a, c = x[..., low].clone(), x[..., high].clone()
            x[..., low], x[..., high] = a * cos - c * sin, c * cos + a * sin
        for kv, fresh in ((0, k[at:at + count]), (1, v[at:at + count])):
            if not case["int8"]:
                pools[kv][table[b, slots // page], slots % page] = fresh
                continue
            for block in range((n - count) // BLOCK, (n - 1) // BLOCK + 1):
                start, begin, end = block * BLOCK, max(block * BLOCK, n - count), min((block + 1) * BLOCK, n)
                where, row = int(table[b, start // page]), start % page
                rows = fresh[begin - (n - count):end - (n - count)]
                most = rows.abs().amax((0, 2)).clamp_min(1e-300)
                e = torch.round(torch.log2(most / 127))
                e = (e + (most > 127 * _two_to(e))).clamp(lowest, highest)
                before = s["exponents"][where, :, row // BLOCK, kv].double()
                if begin > start:
                    e = torch.maximum(e, before)
                size = _two_to(e)[:, None]
                # what lies behind the last token keeps its codes
                pools[kv][where, row + end - start:row + BLOCK] *= _two_to(e - before)[:, None]
                old = pools[kv][where, row:row + begin - start]
                old.copy_(torch.round(old / size) * size)
                pools[kv][where, row + begin - start:row + end - start] = \
                    torch.round(rows / size).clamp(-127, 127) * size
        at += count
    return {"q": q, "k_pages": pools[0], "v_pages": pools[1]}


def _exact_attend(s):
    case = s["case"]
    page, hk, dim, hq = case["page"], case["kv_heads"], case["dim"], case["heads"]
    table, group = s["page_table"].long(), hq // hk
    output = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, (count, n) in enumerate(_lengths(case)):
        tokens = slice(at, at + count)
        i = torch.arange(n, device="cuda")
        where = table[b, i // page]
        position = torch.arange(n - count, n, device="cuda")[:, None]
        hidden = i[None] > position
        if case["window"]:
            hidden |= (i[None] <= position - case["window"]) & (i[None] >= case["sinks"])
        for h in range(hk):
            scale = _two_to(s["exponents"][where, h, i % page // BLOCK])
            keys = s["k_pages"][where, i % page, h].double() * scale[:, :1]
            values = s["v_pages"][where, i % page, h].double() * scale[:, 1:]
            for head in range(h * group, (h + 1) * group):
                z = (s["q"][tokens, head].double() @ keys.T) / math.sqrt(dim)
                z[hidden] = -math.inf
                lse[tokens, head] = torch.logsumexp(z, -1)
                output[tokens, head] = torch.softmax(z, -1) @ values
        at += count
    return {"output": output, "lse": lse}
