"""What the paged KV cache's operators are measured on.

Three operators share one cache and one batch plan: writing the keys and values
of new tokens into pages (in fp16, or in 8 bits with a scale for each token and
head), reading tokens back, and attention of new tokens over the cached ones. A
batch holds sequences of different lengths, packed one behind the other.
"""

import importlib
import math

import torch

own = False

PACKAGE = "gpu-kernel-for-transformer_b200"
DTYPES = {"fp16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}  # the largest code of each 8-bit type


def _case(name, op, dtype, batch, q, kv, heads, group, hd, page, order="head"):
    """q, kv: smallest and largest number of new tokens and of tokens in all, over the batch;
    heads: key/value heads, each read by `group` query heads; order: what a page holds as a
    block, a "head" (its tokens together) or a "token" (its heads together)."""
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "q_min": q[0], "q_max": q[1],
            "kv_min": kv[0], "kv_max": kv[1], "heads": heads, "group": group, "hd": hd,
            "page": page, "order": order}


def listed():
    return [
        # One step of 64 running sequences: the latency of a write, and of reading it again.
        _case("append_step_int8", "append", "int8", 64, (1, 1), (100, 2100), 16, 1, 64, 16),
        # New prompts, written whole: the longest writes of a server.
        _case("append_prompts_e4m3", "append", "e4m3", 12, (37, 8192), (37, 8192), 16, 1, 64, 64),
        # Sequences taken out of the cache (to move or to keep them) in fp16.
        _case("read_sequences_int8", "read", "int8", 8, (5001, 16384), (5001, 16384), 16, 1, 64,
              32, "token"),
        _case("read_small_e4m3", "read", "e4m3", 3, (1, 900), (1, 900), 2, 1, 32, 16),
        # One user's next token: latency.
        _case("decode_one_fp16", "attention", "fp16", 1, (1, 1), (1777, 1777), 16, 1, 64, 16),
        # A batch of users of different ages, wide heads, the cache in token order.
        _case("decode_batch_fp16", "attention", "fp16", 32, (1, 1), (500, 8192), 4, 1, 256, 32,
              "token"),
        # The longest contexts, in 8 bits.
        _case("decode_long_int8", "attention", "int8", 4, (1, 1), (77777, 100000), 16, 1, 64, 128),
        # Grouped heads, many users: the ordinary load of a large server.
        _case("decode_grouped_e4m3", "attention", "e4m3", 64, (1, 1), (1000, 16000), 8, 4, 128, 64),
        # A few drafted tokens a sequence, checked in one pass.
        _case("verify_drafts_int8", "attention", "int8", 16, (2, 8), (300, 6000), 4, 4, 128, 16),
        # Small heads, running sequences and short new prompts in one batch.
        _case("mixed_small_heads_fp16", "attention", "fp16", 40, (1, 200), (200, 2000), 4, 1, 32,
              16),
        # The next part of two long prompts.
        _case("prompt_part_fp16", "attention", "fp16", 2, (1500, 2048), (15000, 20000), 16, 1, 64,
              64),
        # The same with grouped heads and an 8-bit cache, ragged.
        _case("prompt_parts_grouped_int8", "attention", "int8", 6, (100, 1024), (4000, 12000), 8, 4,
              128, 128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "attention", "attention"])
    dtype = rng.choice(["fp16", "int8", "e4m3"])
    hd = rng.choice([8, 16, 32, 64, 64, 128, 128, 256] if dtype == "fp16" else
                    [16, 32, 64, 64, 128, 128, 256])
    heads = rng.choice([1, 2, 3, 4, 8, 16])
    group = rng.choice([1, 1, 2, 3, 4, 5, 8]) if op == "attention" else 1
    batch = _log(rng, 1, 64)
    if op == "attention":
        q_max = {0: 1, 1: rng.randint(2, 8), 2: _log(rng, 9, 2048)}[rng.randrange(3)]
        q_min = rng.randint(1, q_max)
        kv_max = _log(rng, max(q_max, 16), 100000)
    else:
        kv_max = _log(rng, 1, 16384)
        q_max = 1 if op == "append" and rng.random() < 0.3 else kv_max
        q_min = rng.randint(1, q_max)
    kv_min = rng.randint(max(q_min, kv_max // 20), kv_max)
    case = {"op": op, "dtype": dtype, "batch": batch, "q_min": q_min, "q_max": q_max,
            "kv_min": max(kv_min, q_min), "kv_max": kv_max, "heads": heads, "group": group,
            "hd": hd, "page": rng.choice([16, 32, 64, 128, 256]),
            "order": rng.choice(["head", "token"])}
    # No more than the largest listed ones: in values held, in pairs of tokens, in work.
    most = [work(c) for c in listed()]
    while True:
        w = work(case)
        width = case["batch"] * case["kv_max"] * heads * hd
        pairs = case["batch"] * case["q_max"] * case["kv_max"] * heads * group
        if (width <= 1.4e8 and pairs <= 1.3e9 and w["bytes"] <= max(m["bytes"] for m in most)
                and w["flops"] <= max(m["flops"] for m in most)):
            return case
        if case["batch"] > 1:
            case["batch"] = max(1, int(case["batch"] * 0.7))
        else:
            case["kv_max"] = max(16, int(case["kv_max"] * 0.7))
            case["q_max"] = min(case["q_max"], case["kv_max"])
            case["q_min"] = min(case["q_min"], case["q_max"])
            case["kv_min"] = min(case["kv_min"], case["kv_max"])


def _lengths(case):
    """New tokens and tokens in all of each sequence, spread over the case's ranges."""
    n, kv = [], []
    for b in range(case["batch"]):
        f, g = (0.618034 * b + 0.999) % 1.0, (0.754878 * b + 0.999) % 1.0
        kv.append(case["kv_min"] + int(round(g * (case["kv_max"] - case["kv_min"]))))
        n.append(case["q_min"] + int(round(f * (case["q_max"] - case["q_min"]))))
    if case["op"] == "read" or (case["op"] == "append" and case["q_max"] == case["kv_max"]):
        n = kv  # whole sequences
    return [min(a, b) for a, b in zip(n, kv)], kv


def work(case):
    n, kv = _lengths(case)
    values = case["heads"] * case["hd"]  # of one token's keys
    code = 2 if case["dtype"] == "fp16" else 1
    cached = 2 * (values * code + (0 if code == 2 else 4 * case["heads"]))  # of one token, K and V
    table = 4 * sum(-(-m // case["page"]) for m in kv)
    tokens = sum(n)
    if case["op"] == "append":
        read_again = 4 * values * tokens if code == 1 else 0
        return {"bytes": 4 * values * tokens + cached * tokens + read_again + table, "flops": 0}
    if case["op"] == "read":
        return {"bytes": 4 * values * tokens + cached * tokens + table, "flops": 0}
    rows = values * case["group"]  # of one token's queries
    pairs = sum(m * k - m * (m - 1) // 2 for m, k in zip(n, kv))  # each token sees itself and before
    return {"bytes": 4 * rows * tokens + cached * sum(kv) + table,
            "flops": 4 * case["hd"] * case["heads"] * case["group"] * pairs}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    n, kv = _lengths(case)
    page, heads, hd, quant = case["page"], case["heads"], case["hd"], case["dtype"] != "fp16"
    pages = [-(-m // page) for m in kv]
    pool = sum(pages) + 3
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(kv), max(pages)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, m in enumerate(pages):
        table[b, :m] = order[at:at + m]
        at += m
    # Channels of keys differ in size, as a projection's do; values are closer to each other.
    gain = 0.4 + 1.2 * torch.rand(heads, hd, generator=g, device=dev)
    tokens = sum(n)
    state = {"case": case, "table": table, "tokens": tokens, "longest": max(n),
             "longest_kv": max(kv),
             "kv_len": torch.tensor(kv, dtype=torch.int32, device=dev),
             "query_start": torch.tensor([sum(n[:b]) for b in range(len(n) + 1)],
                                         dtype=torch.int32, device=dev)}
    # Tokens written earlier: codes and scales as a write leaves them.
    for name in ("k", "v"):
        codes, scales = [], []
        for lo in range(0, pool, 512):  # in parts, so that the fp32 values stay small
            x = randn(min(512, pool - lo), heads, page, hd)
            x = (x * gain[:, None] if name == "k" else x).half()
            if quant:
                s = x.float().abs().amax(-1) / TOP[case["dtype"]]
                y = x.float() / s[..., None]
                codes.append((y.round() if case["dtype"] == "int8" else y).to(DTYPES[case["dtype"]]))
                scales.append(s)
            else:
                codes.append(x)
        c = torch.cat([x.view(torch.uint8) if quant else x for x in codes])
        c = c if case["order"] == "head" else c.transpose(1, 2).contiguous()
        c = c.view(DTYPES[case["dtype"]])
        # [pages, tokens of a page, heads, hd], whatever the order in memory
        state[name + "_cache"] = c.transpose(1, 2) if case["order"] == "head" else c
        state[name + "_scale"] = torch.cat(scales) if quant else None
    if case["op"] == "append":  # slices of one projection's output
        new = randn(tokens, 2, heads, hd)
        new[:, 0] *= gain
        new = new.half()
        state["k"], state["v"] = new[:, 0], new[:, 1]
    if case["op"] == "attention":
        state["q"] = (1.5 * randn(tokens, heads * case["group"], hd)).half()
    if own:
        tfx = importlib.import_module(PACKAGE)
        state["cache"] = tfx.PagedKVCache.from_tensors(
            state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"])
        state["batch"] = tfx.PagedBatch(table, state["query_start"], state["kv_len"], tokens,
                                        max_query_len=max(n), max_kv_len=max(kv))
        state["ops"] = tfx.ops
    return state


def run(state):
    op = state["case"]["op"]
    if op == "append":
        return _append(state)
    if op == "read":
        if own:
            return state["ops"].paged_read(state["cache"], state["batch"])
        return _read(state)
    if own:
        return state["ops"].paged_attention(state["q"], state["cache"], state["batch"])
    return _attention(state)


def _append(state):
    """fp16: the cache itself. 8 bits: the new tokens as they read back, and the scales."""
    if own:
        state["ops"].paged_append(state["k"], state["v"], state["cache"], state["batch"])
    else:
        _, at = _slots(state)
        for name in ("k", "v"):
            _write(state[name], state[name + "_cache"], state[name + "_scale"], at)
    if state["k_scale"] is None:
        return state["k_cache"], state["v_cache"]
    k, v = (state["ops"].paged_read(state["cache"], state["batch"]) if own else _read(state))
    return k, v, state["k_scale"], state["v_scale"]


def _slots(state):
    """The sequence of each row, and its token's place in the pool (page * page size + slot)."""
    start, kv = state["query_start"].long(), state["kv_len"].long()
    page = state["case"]["page"]
    rows = torch.arange(state["tokens"], device=start.device)
    seq = torch.searchsorted(start[1:].contiguous(), rows, right=True)
    pos = kv[seq] - (start[seq + 1] - start[seq]) + (rows - start[seq])
    return seq, state["table"][seq, pos // page].long() * page + pos % page


def _write(x, cache, scale, at):
    page = cache.shape[1]
    if scale is None:
        cache[at // page, at % page] = x
        return
    x = x.double()  # 64 bits: quotients that lie next to the border of two codes
    top = TOP["int8" if cache.dtype == torch.int8 else "e4m3"]
    s = (x.abs().amax(-1) / top).float()
    y = torch.where(s[..., None] > 0, x / s[..., None].double(), 0.0)
    if cache.dtype == torch.int8:
        code = y.round().clamp(-127, 127)
    else:  # 3 bits behind the leading one; below 2^-6 the step stays 2^-9
        step = torch.exp2((torch.frexp(y)[1] - 1).clamp(min=-6).double() - 3)
        code = ((y / step).round() * step).clamp(-448, 448).float()
    code = code.to(cache.dtype).view(torch.uint8)
    cache.view(torch.uint8)[at // page, at % page] = code
    scale[at // page, :, at % page] = s


def _values(cache, scale, page, slot):
    """Cached tokens in fp32, [..., heads, hd], for pages and slots of any one shape."""
    if scale is None:
        return cache[page, slot].float()
    code = cache.view(torch.uint8)[page, slot].view(cache.dtype).float()
    return code * scale[page, :, slot][..., None]


def _read(state):
    _, at = _slots(state)
    page = state["case"]["page"]
    return tuple(_values(state[n + "_cache"], state[n + "_scale"], at // page, at % page).half()
                 for n in ("k", "v"))


def _attention(state):
    """Every sequence padded to the longest, in fp32."""
    case = state["case"]
    q, table, page, group = state["q"], state["table"], case["page"], case["group"]
    start, kv = state["query_start"].long(), state["kv_len"].long()
    n = start[1:] - start[:-1]
    # keys and values [B, heads, S, hd]
    j = torch.arange(state["longest_kv"], device=q.device)
    at = table[:, j // page].long().clamp(min=0)
    held = j < kv[:, None]
    k, v = (_values(state[c + "_cache"], state[c + "_scale"], at, (j % page).expand_as(at))
            .masked_fill(~held[..., None, None], 0.0).transpose(1, 2) for c in ("k", "v"))
    # queries [B, heads, longest * group, hd]
    longest = state["longest"]
    i = torch.arange(longest, device=q.device)
    row = (start[:-1, None] + i).clamp(max=q.shape[0] - 1)
    x = q[row].float().view(len(n), longest, case["heads"], group, case["hd"])
    x = x.transpose(1, 2).reshape(len(n), case["heads"], longest * group, case["hd"])
    scores = torch.matmul(x, k.transpose(-1, -2)).mul_(case["hd"] ** -0.5)
    last = (kv - n)[:, None] + i  # the position of each query
    hidden = (j > last[..., None]) | ~held[:, None, :]
    hidden = hidden[:, None, :, None, :].expand(-1, 1, -1, group, -1).flatten(2, 3)
    scores = scores.masked_fill_(hidden, -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores, v) / torch.where(total > 0, total, 1.0)
    out = out.view(len(n), case["heads"], longest, group, case["hd"]).transpose(1, 2)
    out = out.reshape(len(n), longest, -1)
    return out[i < n[:, None]].half()


def exact(case, seed):
    """In 64 bits, a sequence at a time, from the definitions."""
    s = prepare(case, seed)
    n, kv = _lengths(case)
    page = case["page"]
    names = ("k", "v")
    codes = {c: s[c + "_cache"] for c in names}
    scales = {c: s[c + "_scale"] for c in names}
    first = [sum(n[:b]) for b in range(len(n))]

    def places(b, lo):
        p = torch.arange(lo, kv[b], device="cuda")
        return s["table"][b].long()[p // page], p % page

    def held(c, b, lo=0):
        at, slot = places(b, lo)
        if scales[c] is None:
            return codes[c][at, slot].double()
        x = codes[c].view(torch.uint8)[at, slot].view(codes[c].dtype).float().double()
        return x * scales[c][at, :, slot][..., None].double()

    if case["op"] == "append":
        # every positive code's value, and the borders halfway between neighbours
        if case["dtype"] == "int8":
            grid = torch.arange(128, device="cuda").double()
        elif case["dtype"] == "e4m3":
            grid = torch.arange(127, device="cuda", dtype=torch.uint8).view(
                torch.float8_e4m3fn).float().double()
        written = {}
        for c in names:
            new = s[c].double()
            if scales[c] is None:
                codes[c] = codes[c].clone()
                for b in range(len(n)):
                    at, slot = places(b, kv[b] - n[b])
                    codes[c][at, slot] = s[c][first[b]:first[b] + n[b]]
                continue
            scale = (new.abs().max(-1).values / grid[-1]).float()
            rows = []
            for x, m in zip(new.split(4096), scale.split(4096)):  # a part at a time
                y = torch.nan_to_num(x.abs() / m[..., None].double())
                near = torch.searchsorted(grid, y.contiguous()).clamp(1, len(grid) - 1)
                low, high = grid[near - 1], grid[near]
                up = (y - low > high - y) | ((y - low == high - y) & (near % 2 == 0))
                rows.append(torch.where(up, high, low) * x.sign() * m[..., None].double())
            written[c] = torch.cat(rows)
            scales[c] = scales[c].clone()
            for b in range(len(n)):
                at, slot = places(b, kv[b] - n[b])
                scales[c][at, :, slot] = scale[first[b]:first[b] + n[b]]
        if not written:
            return tuple(codes[c].double() for c in names)
        return written["k"], written["v"], scales["k"].double(), scales["v"].double()
    if case["op"] == "read":
        return tuple(torch.cat([held(c, b, kv[b] - n[b]) for b in range(len(n))]) for c in names)
    group, hd = case["group"], case["hd"]
    out = torch.empty(sum(n), case["heads"] * group, hd, dtype=torch.float64, device="cuda")
    for b in range(len(n)):
        keys, values = held("k", b), held("v", b)
        rows = s["q"][first[b]:first[b] + n[b]].double()
        seen = (torch.arange(kv[b], device="cuda")[None, :]
                <= torch.arange(kv[b] - n[b], kv[b], device="cuda")[:, None])
        for h in range(case["heads"] * group):
            w = rows[:, h] @ keys[:, h // group].T / math.sqrt(hd)
            w = torch.softmax(torch.where(seen, w, -math.inf), dim=-1)
            out[first[b]:first[b] + n[b], h] = w @ values[:, h // group]
    return out.flatten(1)
