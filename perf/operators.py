"""The paged key/value cache's operators as workloads: quantising rows into the cache and reading them back, attention
of new rows over it (single tokens and chunks), and the same with a sliding window and always-visible first tokens.

A cache holds, per layer, `pages` pages of `page` tokens; a sequence's block table names its pages in order.  Per
token and KV head it keeps one vector of keys and one of values with an f32 scale each:
  i8   q = the integer nearest to 127 x / amax (ties to even), scale = amax / 127; the value is q * scale
  f16  the vector over 2^e as f16, scale = 2^e, with amax / 2^e in [2^14, 2^15)
Row i of a sequence that has `position` tokens before its new rows stands at position + i and attends to the tokens t
with t <= position + i and, with a window, t > position + i - window or t < sinks.
"""
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    base = {"heads": 16, "kv_heads": 2, "head_dim": 256, "page": 64, "fmt": "i8", "dtype": "f32", "seqs": 1, "rows": 1,
            "ctx": 4096, "window": 0, "sinks": 0}

    def case(name, kind, **k):
        return {"name": name, "kind": kind, **base, **k}

    return [
        # the rows of one verify pass enter the cache and are read back: launch latency
        case("store_verify_4rows", "store", rows=4, ctx=2052),
        # a ragged prefill of several prompts in bf16, pages of 16
        case("store_prefill_bf16", "store", dtype="bf16", seqs=7, rows=4099, ctx=4099, page=16),
        # a long sequence's whole cache goes out for a session image
        case("read_image_f32", "read", ctx=65531, rows=65531),
        # f16 cache with small heads, many short sequences
        case("read_f16_heads64", "read", dtype="f16", fmt="f16", heads=8, head_dim=64, seqs=33, rows=517, ctx=517, page=32),
        # decoding one token of one sequence in the model's own f32 rows
        case("attend_token_4k", "attend", ctx=4096),
        # a batch of 64 sequences of mixed lengths, one token each
        case("attend_tokens_batch64", "attend", dtype="bf16", seqs=64, ctx=8209),
        # one token at the longest context the configurations allow
        case("attend_token_256k_f16", "attend", dtype="f16", fmt="f16", ctx=262144, page=128),
        # speculative verification: up to 4 rows for each of 16 sequences
        case("attend_verify_16x4", "attend", seqs=16, rows=4, ctx=4127, page=32),
        # a prefill chunk of 512 rows in f32 after 2048 tokens
        case("attend_chunk_512_f32", "attend", rows=512, ctx=2560),
        # a long prompt's last chunk: 2048 rows, 32768 tokens
        case("attend_chunk_2048_bf16", "attend", dtype="bf16", rows=2048, ctx=32768, page=128),
        # streaming decode: a window of 4096 and 64 first tokens, long sequences
        case("window_tokens_batch24", "attend", dtype="bf16", seqs=24, ctx=50021, window=4096, sinks=64, page=32),
        # a chunk of a long stream under a window, f16 cache, heads of 128
        case("window_chunk_1111_f16", "attend", dtype="f16", fmt="f16", heads=32, kv_heads=8, head_dim=128, rows=1111, ctx=20011,
             window=1023, sinks=5),
    ]


def _span(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv_heads, head_dim = rng.choice([(16, 2, 256), (16, 2, 256), (8, 2, 64), (32, 8, 128), (12, 4, 128), (14, 2, 64), (4, 4, 128)])
    dtype = rng.choice(["f32", "bf16", "f16"])
    c = {"kind": rng.choice(["store", "read", "attend", "attend", "attend", "attend"]), "heads": heads, "kv_heads": kv_heads,
         "head_dim": head_dim, "page": rng.choice([16, 32, 64, 128]), "fmt": rng.choice(["i8", "i8", "f16"]), "dtype": dtype, "seqs": 1,
         "rows": 1, "ctx": 1, "window": 0, "sinks": 0}
    if c["kind"] in ("store", "read"):
        total = _span(rng, 4, 60000) * 512 // (kv_heads * head_dim)
        c["seqs"] = min(total, _span(rng, 1, 40))
        c["rows"] = max(1, total // c["seqs"])
        c["ctx"] = c["rows"] + (rng.randrange(0, 300) if c["kind"] == "store" else 0)
        return c
    form = rng.choice(["token", "tokens", "verify", "chunk", "chunk"])
    if form == "token":
        c["ctx"] = _span(rng, 64, 200000)
    elif form == "tokens":
        c["seqs"], c["ctx"] = _span(rng, 2, 64), _span(rng, 64, 7000)
    elif form == "verify":
        c["seqs"], c["rows"], c["ctx"] = _span(rng, 1, 20), rng.randrange(2, 9), _span(rng, 64, 5000)
    else:
        c["seqs"], c["rows"] = rng.choice([1, 1, 2, 3]), _span(rng, 9, 1200)
        c["ctx"] = c["rows"] + _span(rng, 1, 16000 // c["seqs"])
    c["ctx"] = max(c["ctx"], c["rows"])
    if rng.random() < 0.35:
        c["window"], c["sinks"] = _span(rng, 16, 4000), rng.choice([0, 1, 4, 63, 128])
    return c


def _lengths(case):
    """[(rows, context with those rows)] of every sequence: the first is the longest, the others are mixed."""
    r = random.Random(case["seqs"] * 1000003 + case["ctx"] * 101 + case["rows"])
    got = [(case["rows"], case["ctx"])]
    for _ in range(case["seqs"] - 1):
        n = r.randint(1, case["rows"])
        got.append((n, n + int((case["ctx"] - case["rows"]) * r.uniform(0.2, 1.0))))
    return got


def _pairs(n, ctx, window, sinks):
    """Visible (row, token) pairs of a sequence, and the tokens that any of its rows sees."""
    if not window:
        return n * ctx - n * (n - 1) // 2, ctx
    total = 0
    for p in range(ctx - n, ctx):
        low = max(0, p - window + 1)
        total += p + 1 - low + min(sinks, low)
    low = max(0, ctx - n - window + 1)
    return total, ctx - low + min(sinks, low)


def work(case):
    item = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    held = case["kv_heads"] * 2 * (case["head_dim"] * (1 if case["fmt"] == "i8" else 2) + 4)
    rows = sum(n for n, _ in _lengths(case))
    vectors = rows * case["kv_heads"] * 2 * case["head_dim"]
    if case["kind"] == "read":
        return {"bytes": rows * held + vectors * item, "flops": vectors}
    if case["kind"] == "store":
        return {"bytes": 2 * rows * held + 2 * vectors * item, "flops": 4 * vectors}
    pairs, tokens = map(sum, zip(*(_pairs(n, ctx, case["window"], case["sinks"]) for n, ctx in _lengths(case))))
    return {"bytes": tokens * held + 2 * rows * case["heads"] * case["head_dim"] * item,
            "flops": 4 * pairs * case["heads"] * case["head_dim"]}


def _inputs(case, seed):
    """What is made from the seed: block tables, keys and values of every cached token, and the new rows."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv, hd, page, dt = case["kv_heads"], case["head_dim"], case["page"], DT[case["dtype"]]
    lens = _lengths(case)
    cols = max(-(-ctx // page) for _, ctx in lens)
    counts = [-(-ctx // page) for _, ctx in lens]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), cols, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    tokens = sum(ctx for _, ctx in lens)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    # normalised keys with a few strong channels; values of mixed size from token to token
    channel = 1.0 + 3.0 * (torch.rand(kv, hd, generator=g, device="cuda") > 0.97)
    k = (normal(tokens, kv, hd) * channel / channel.square().mean(-1, keepdim=True).sqrt()).to(dt)
    v = (normal(tokens, kv, hd) * torch.exp(0.5 * normal(tokens, 1, 1))).to(dt)
    q = (1.5 * normal(starts[-1], case["heads"], hd)).to(dt) if case["kind"] == "attend" else None
    return {"lens": lens, "table": table, "pages": pages, "k": k, "v": v, "q": q, "starts": starts,
            "row_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
            "position": torch.tensor([ctx - n for n, ctx in lens], dtype=torch.int32, device="cuda")}


def _row_of(lens, all_tokens, device="cuda"):
    """(sequence, position) of every new row, or of every cached token."""
    seq = torch.cat([torch.full((ctx if all_tokens else n,), s) for s, (n, ctx) in enumerate(lens)])
    pos = torch.cat([torch.arange(0 if all_tokens else ctx - n, ctx) for n, ctx in lens])
    return seq.to(device), pos.to(device)


def _quantise(x, fmt):
    """(codes, scale) of vectors along the last axis; borders between two codes are decided in 64 bits."""
    amax = x.float().abs().amax(-1, keepdim=True)
    if fmt == "i8":
        codes = torch.where(amax > 0, torch.round(127.0 * x.double() / amax.double()), 0.0).to(torch.int8)
        return codes, amax / 127.0
    scale = torch.where(amax > 0, torch.exp2(torch.floor(torch.log2(amax.double())) - 14), 1.0)
    return (x.double() / scale).float().to(torch.float16), scale.float()


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    lens, page, fmt = st["lens"], case["page"], case["fmt"]
    seq, pos = _row_of(lens, True)
    new, newpos = _row_of(lens, False)
    first = torch.cat([torch.zeros(1, dtype=torch.long), torch.tensor([ctx for _, ctx in lens]).cumsum(0)[:-1]]).cuda()
    at = first[new] + newpos  # the new rows among all tokens
    st["new_k"], st["new_v"] = st["k"][at].contiguous(), st["v"][at].contiguous()
    store = case["kind"] == "store"
    if own:
        from inferq_b200.kv import KvBatch, KvCache

        st["cache"] = KvCache(case["kv_heads"], case["head_dim"], st["pages"], page_tokens=page, format=fmt)
        st["batch"] = KvBatch(st["table"], st["position"], st["row_start"], max_rows=case["rows"])
        if not store:
            every = KvBatch(st["table"], torch.zeros_like(st["position"]),
                            torch.tensor([0] + [ctx for _, ctx in lens], dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32),
                            max_rows=case["ctx"])
            st["cache"].append(st["k"], st["v"], every)
    else:
        shape = (st["pages"], page, case["kv_heads"], case["head_dim"])
        held = torch.int8 if fmt == "i8" else torch.float16
        st["codes"] = [torch.zeros(shape, dtype=held, device="cuda") for _ in range(2)]
        st["scales"] = [torch.zeros(shape[:3] + (1,), device="cuda") for _ in range(2)]
        if not store:
            slot = st["table"][seq, pos // page].long(), pos % page
            for codes, scales, x in zip(st["codes"], st["scales"], (st["k"], st["v"])):
                codes[slot], scales[slot] = _quantise(x, fmt)
        # the plan of a padded pass: which row stands at [sequence, i], and where each row of the ragged form is
        most = max(n for n, _ in lens)
        st["slot"] = st["table"][new, newpos // page].long(), newpos % page
        start = torch.tensor(st["starts"][:-1], device="cuda")
        st["padded"] = torch.minimum(start[:, None] + torch.arange(most, device="cuda"), torch.tensor(st["starts"][-1] - 1, device="cuda"))
        st["ragged"] = new, newpos - st["position"][new]
    st["k"] = st["v"] = None
    return st


def run(st):
    case = st["case"]
    dt = DT[case["dtype"]]
    if own:
        cache, batch = st["cache"], st["batch"]
        if case["kind"] == "attend":
            return cache.attend(st["q"], batch, window=case["window"], sinks=case["sinks"])
        if case["kind"] == "store":
            cache.append(st["new_k"], st["new_v"], batch)
        return cache.read(batch, dtype=dt, rows=st["starts"][-1])
    if case["kind"] != "attend":
        if case["kind"] == "store":
            for codes, scales, x in zip(st["codes"], st["scales"], (st["new_k"], st["new_v"])):
                codes[st["slot"]], scales[st["slot"]] = _quantise(x, case["fmt"])
        return tuple((codes[st["slot"]].float() * scales[st["slot"]]).to(dt) for codes, scales in zip(st["codes"], st["scales"]))
    kv, hd, page = case["kv_heads"], case["head_dim"], case["page"]
    table = st["table"].long()
    seqs, tokens = table.shape[0], table.shape[1] * page
    # [sequence, KV head, token, head_dim] in 32 bits
    k, v = ((codes[table].float() * scales[table]).view(seqs, tokens, kv, hd).transpose(1, 2)
            for codes, scales in zip(st["codes"], st["scales"]))
    q = st["q"][st["padded"]].float().view(seqs, -1, kv, case["heads"] // kv, hd).permute(0, 2, 3, 1, 4)
    at = torch.arange(tokens, device="cuda")
    row = st["position"][:, None] + torch.arange(q.shape[3], device="cuda")
    seen = at <= row[:, :, None]
    if case["window"]:
        seen &= (at > row[:, :, None] - case["window"]) | (at < case["sinks"])
    s = (q / math.sqrt(hd)).flatten(2, 3) @ k.transpose(2, 3)
    s = s.view(seqs, kv, -1, q.shape[3], tokens).masked_fill_(~seen[:, None, None], float("-inf"))
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    o = (s.flatten(2, 3) @ v).view(*total.shape[:-1], hd) / total
    return o.permute(0, 3, 1, 2, 4).reshape(seqs, -1, case["heads"], hd)[st["ragged"]].to(dt)


def exact(case, seed):
    st = _inputs(case, seed)
    lens = st["lens"]
    if case["kind"] == "attend" and sum(n * ctx for n, ctx in lens) * case["heads"] * case["head_dim"] > 3e12:
        return None

    def held(x):
        """The values that the cache stands for."""
        x = x.double()
        top = x.abs().amax(-1, keepdim=True)
        if case["fmt"] == "i8":
            return torch.where(top > 0, torch.round(127 * x / top) * (top / 127), 0.0)
        unit = torch.exp2(torch.frexp(x).exponent.double() - 11)  # 11 significant bits, fewer far below the largest
        unit = torch.maximum(unit, torch.exp2(torch.frexp(top).exponent.double() - 15 - 24))
        return torch.where(x != 0, torch.round(x / unit) * unit, 0.0)

    begin = [0]
    for _, ctx in lens:
        begin.append(begin[-1] + ctx)
    if case["kind"] != "attend":
        return tuple(torch.cat([held(x[b + ctx - n:b + ctx]) for b, (n, ctx) in zip(begin, lens)]) for x in (st["k"], st["v"]))
    group = case["heads"] // case["kv_heads"]
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    for (n, ctx), b, r in zip(lens, begin, st["starts"]):
        k, v = held(st["k"][b:b + ctx]), held(st["v"][b:b + ctx])
        for i in range(0, n, 256):
            p = torch.arange(ctx - n + i, ctx - n + min(n, i + 256), device="cuda")[:, None]
            t = torch.arange(ctx, device="cuda")[None]
            hidden = t > p
            if case["window"]:
                hidden = hidden | ((p - t >= case["window"]) & (t >= case["sinks"]))
            for h in range(case["heads"]):
                s = st["q"][r + i:r + i + len(p), h].double() @ k[:, h // group].T / math.sqrt(case["head_dim"])
                out[r + i:r + i + len(p), h] = torch.softmax(s.masked_fill(hidden, float("-inf")), -1) @ v[:, h // group]
    return out
