"""The operators of an 8-bit K/V cache and its pages, as measured cases.

Format of the cache.  The 128 elements of a (token, kv head) row are 8-bit codes (e4m3 or signed
integers); `block` consecutive tokens of one kv head share one fp32 scale:

    scale = max(fl32(amax / qmax), 2^-126)      qmax = 448 (e4m3), 127 (int8)
    code  = round_to_nearest_even(fl32(x * fl32(1 / scale)))
    value = code * scale

The tokens of a sequence's last, not yet full block stay in 16 bits in an "open" buffer of `block`
rows per (request, kv head) and are quantised together when the block fills.

Operators:
    append    new K / V rows into the cache (prompts, chunks, single tokens)
    dense     decode attention over every cached token, optionally with the filter layer's scores
    sparse    decode attention over selected rows of the cache and a 16-bit tail
    fork      free, fork and extend sequences of a paged pool (a step of several continuations)
    compact   move a pool's used pages to its lowest ones

Codes are bit patterns that both sides must agree on exactly (every rounding above is fixed), so the
append cases return the stored codes as they are, next to the scales.
"""
import random

import torch

own = False

HKV, D = 8, 128  # 32 query heads on 8 kv heads, the shape of this repository's benchmark
QMAX = {"e4m3": 448.0, "int8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TYPE = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------ cases
def _append(name, fmt, dtype, block, batch, new, start, page=0, close=False, hkv=HKV):
    return {"name": name, "op": "append", "fmt": fmt, "dtype": dtype, "block": block, "batch": batch, "new": new,
            "start": start, "page": page, "close": close, "hkv": hkv}


def _dense(name, fmt, dtype, block, batch, lo, hi, page=0, selector="", group=4, hkv=HKV):
    return {"name": name, "op": "dense", "fmt": fmt, "dtype": dtype, "block": block, "batch": batch, "lo": lo, "hi": hi,
            "page": page, "selector": selector, "group": group, "hkv": hkv}


def _sparse(name, fmt, dtype, block, batch, lo, hi, pick, tail, page=0, group=4, hkv=HKV):
    return {"name": name, "op": "sparse", "fmt": fmt, "dtype": dtype, "block": block, "batch": batch, "lo": lo, "hi": hi,
            "pick": pick, "tail": tail, "page": page, "group": group, "hkv": hkv}


def _fork(name, parents, lo, hi, more, layers, block=16, page=16, hkv=HKV):
    return {"name": name, "op": "fork", "parents": parents, "lo": lo, "hi": hi, "more": more, "layers": layers,
            "block": block, "page": page, "hkv": hkv}


def _compact(name, pages, used, layers, block=16, page=16, hkv=HKV):
    return {"name": name, "op": "compact", "pages": pages, "used": used, "layers": layers, "block": block, "page": page,
            "hkv": hkv}


def listed():
    return [
        # a 128K prompt goes into one layer's cache
        _append("append prompt 128K", "e4m3", "bf16", 64, 1, 131072, 0, close=True),
        # one decode step of sixteen requests on 16-token pages: the smallest call of the write path
        _append("append token x16", "int8", "bf16", 16, 16, 1, 700, page=16),
        # decode attention of a full layer at the longest context the benchmark has
        _dense("dense 450K", "int8", "bf16", 64, 1, 450000, 450000),
        # the filter layer of a 128K decode step: attention and the selector's scores in one pass
        _dense("dense 128K scored", "e4m3", "bf16", 64, 1, 131073, 131073, selector="softmax_before_last"),
        # sixteen ragged requests on shuffled 16-token pages
        _dense("dense paged x16", "e4m3", "bf16", 16, 16, 8192, 32768, page=16),
        # chat-sized requests, shorter than one block to a few blocks long: a chain of latencies
        _dense("dense short x4", "int8", "f16", 32, 4, 1, 333),
        # a sparse layer of the 128K decode step: 6.7% of the rows and the tokens generated so far
        _sparse("sparse 128K", "e4m3", "bf16", 64, 1, 131072, 131072, 0.067, 77),
        # the sparse layers of the ragged batch, their rows addressed as token slots of the pool
        _sparse("sparse slots x16", "int8", "f16", 16, 16, 8192, 32768, 0.067, 33, page=16),
        # two prompts fan out into two continuations: the smallest call of the page operations
        _fork("fork x2", 2, 20, 90, 1, 2),
        # sixty-four sequences of sixteen layers fork at once and grow by a chunk
        _fork("fork x64", 64, 500, 1700, 33, 16),
        # a small pool after a few requests ended
        _compact("compact 96 pages", 96, 0.4, 2),
        # a pool of 64K tokens, half of it free, sixteen layers
        _compact("compact 4096 pages", 4096, 0.5, 16),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    fmt, dtype = rng.choice(["e4m3", "int8"]), rng.choice(["bf16", "f16"])
    page = rng.choice([0, 16, 32, 48, 64])
    block = rng.choice([16, 32, 64, 128] if not page else [b for b in (16, 32, 64) if page % b == 0])
    hkv, group = rng.choice([1, 2, 5, 8, 8, 8]), rng.choice([1, 2, 4, 4, 7, 8])
    op = rng.choice(["append", "append", "dense", "dense", "dense", "sparse", "sparse", "fork", "compact"])
    if op == "append":
        batch = rng.choice([1, 1, 2, 5, 16])
        new = log(1, 100000 // batch)
        close = rng.random() < 0.2
        c = _append("", fmt, dtype, block, batch, new, 0 if close else rng.choice([0, log(1, 3000)]), page, close, hkv)
    elif op == "dense":
        batch = rng.choice([1, 1, 2, 3, 8, 16])
        hi = log(1, 400000 // batch)
        selector = rng.choice(["", "", "last", "softmax_before_last", "softmax_sum_last"])
        c = _dense("", fmt, dtype, block, batch, max(1, hi // rng.choice([1, 2, 4])), hi, page, selector, group, hkv)
    elif op == "sparse":
        batch = rng.choice([1, 1, 2, 3, 8, 16])
        hi = log(40, 400000 // batch)
        c = _sparse("", fmt, dtype, block, batch, max(1, hi // rng.choice([1, 2, 4])), hi,
                    round(rng.uniform(0.03, 0.5), 4), rng.choice([0, 1, log(1, 600)]), page, group, hkv)
    elif op == "fork":
        hi = log(8, 1700)
        c = _fork("", log(1, 64), max(1, hi // rng.choice([1, 3, 9])), hi, rng.choice([1, 1, 5, 40]), rng.choice([1, 2, 3, 8]),
                  block if page else 16, page or 16, hkv)
    else:
        c = _compact("", log(20, 4000), round(rng.uniform(0.1, 0.9), 3), rng.choice([1, 2, 3, 8]), block if page else 16,
                     page or 16, hkv)
    del c["name"]
    return c


def _lens(c):
    """The requests' lengths: part of the case, spread over [lo, hi] with the two ends among them."""
    r = random.Random("%d %d %d" % (c["batch"], c["lo"], c["hi"]))
    got = [r.randint(c["lo"], c["hi"]) for _ in range(c["batch"])]
    got[0] = c["hi"]
    if len(got) > 1:
        got[-1] = c["lo"]
    return got


def _picks(c):
    return [max(1, int(n * c["pick"])) for n in _lens(c)]


def _fork_lens(c):
    r = random.Random("%d %d %d" % (c["parents"], c["lo"], c["hi"]))
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["parents"])]


def _fork_parents(c):
    r = random.Random("parents %d" % c["parents"])
    return [r.randrange(c["parents"]) for _ in range(c["parents"])]


def _compact_lens(c):
    """Sequences that hold `used` of the pool's pages between them."""
    r = random.Random("%d %g" % (c["pages"], c["used"]))
    left, got = max(1, int(c["pages"] * c["used"])), []
    while left:
        n = min(left, r.randint(1, max(1, c["pages"] // 16)))
        got.append(n * c["page"] - r.randrange(c["page"]))
        left -= n
    return got


def _page_bytes(c):
    return c["layers"] * c["hkv"] * (2 * c["page"] * D + 2 * 4 * (c["page"] // c["block"]))


def work(c):
    if c["op"] == "append":
        rows = c["batch"] * c["new"] * c["hkv"]
        if c["new"] >= c["block"]:  # 16-bit rows in, codes and scales out
            return {"bytes": rows * 2 * (2 * D + D) + rows // c["block"] * 2 * 4, "flops": rows * 2 * D * 3}
        # rows land in the open block; every block-th token also quantises the block it fills
        return {"bytes": rows * 2 * (2 * D + 2 * D) + rows * 2 * 3 * D, "flops": rows * 2 * D * 3}
    hq = c["hkv"] * c.get("group", 1)
    if c["op"] in ("dense", "sparse"):
        row = c["hkv"] * 2 * (D + 4 / c["block"])
        if c["op"] == "dense":
            lens = _lens(c)
            rows8, rows16, extra = sum(n // c["block"] * c["block"] for n in lens), sum(n % c["block"] for n in lens), 0
            if c["selector"]:
                extra = sum(lens) * 4
        else:
            picks = _picks(c)
            row = c["hkv"] * 2 * (D + 4)
            rows8, rows16, extra = sum(picks), c["tail"] * c["batch"], sum(picks) * 4
        return {"bytes": rows8 * row + rows16 * c["hkv"] * 2 * 2 * D + 2 * c["batch"] * hq * D * 2 + extra,
                "flops": (rows8 + rows16) * hq * D * 4}
    if c["op"] == "fork":
        lens, page = _fork_lens(c), c["page"]
        kids = [lens[p] for p in _fork_parents(c)]
        table = sum(-(-n // page) for n in kids) * 4
        copies = sum(1 for n in kids if n % page)
        return {"bytes": 4 * table + 2 * copies * _page_bytes(c), "flops": 0}
    n = sum(-(-x // c["page"]) for x in _compact_lens(c))
    moves = int(round(n * (1 - n / c["pages"])))
    return {"bytes": 2 * moves * _page_bytes(c) + 2 * 4 * (n + c["pages"]), "flops": 0}


# ------------------------------------------------------------------------------------------ inputs
def _quantise(x, fmt):
    """x (..., block, D) in 16 bits -> codes of the same shape, scales (...)."""
    x = x.float()
    amax = x.abs().amax((-1, -2))
    # the two quotients in 64 bits, rounded once each: next to a border the last bit of fp32 decides the code
    scale = torch.clamp((amax.double() / QMAX[fmt]).float(), min=2.0 ** -126)
    y = x * (1.0 / scale.double()).float()[..., None, None]
    if fmt == "int8":
        return torch.clamp(torch.round(y), -127, 127).to(torch.int8), scale
    return torch.clamp(y, -448.0, 448.0).to(torch.float8_e4m3fn), scale


def _rows(g, shape, dtype, device, gain=1.0):
    """Rows as projections leave them: a few channels far larger than the others."""
    chan = torch.ones(D, device=device)
    chan[torch.randperm(D, generator=g, device=device)[:6]] = 4.0
    x = torch.randn(shape, generator=g, device=device, dtype=dtype)
    return x * (chan * gain).to(dtype)


def _store(g, c, tokens, device):
    """Codes and scales of `tokens` quantised tokens per request (a multiple of the block): contiguous
    (batch, heads, tokens, D) with scales (batch, heads, blocks)."""
    dtype, b, hkv, blk = TYPE[c["dtype"]], c["batch"], c["hkv"], c["block"]
    s = {}
    for name in "kv":
        codes = torch.empty((b, hkv, tokens, D), dtype=CODE[c["fmt"]], device=device)
        scales = torch.empty((b, hkv, tokens // blk), dtype=torch.float32, device=device)
        step = 16384 // blk * blk
        for i in range(b):
            for lo in range(0, tokens, step):
                n = min(step, tokens - lo)
                x = _rows(g, (hkv, n // blk, blk, D), dtype, device, 0.5 if name == "k" else 1.0)
                q, sc = _quantise(x, c["fmt"])
                codes[i, :, lo:lo + n] = q.view(hkv, n, D)
                scales[i, :, lo // blk:(lo + n) // blk] = sc
        s[name], s[name + "_scale"] = codes, scales
    return s


def _paginate(g, c, s, device):
    """The same rows on shuffled pages: pools (pages, page, heads, D), scales (pages, page / block, heads)."""
    b, hkv, tokens, _ = s["k"].shape
    page, per = c["page"], tokens // c["page"]
    table = torch.randperm(b * per, generator=g, device=device).to(torch.int32).view(b, per)
    at = table.view(-1).long()
    for name in "kv":
        pool = torch.empty((b * per, page, hkv, D), dtype=s[name].dtype, device=device)
        pool.view(torch.uint8)[at] = (s[name].view(torch.uint8).view(b, hkv, per, page, D).permute(0, 2, 3, 1, 4)
                                      .reshape(b * per, page, hkv, D))
        sc = torch.empty((b * per, page // c["block"], hkv), dtype=torch.float32, device=device)
        sc[at] = (s[name + "_scale"].view(b, hkv, per, page // c["block"]).permute(0, 2, 3, 1)
                  .reshape(b * per, page // c["block"], hkv))
        s[name], s[name + "_scale"] = pool, sc
    s["table"] = table
    return s


def _i32(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


def prepare(case, seed):
    c = case
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": c}
    if c["op"] in ("fork", "compact"):
        return _prepare_pages(s, c, g, random.Random(seed), dev)
    dtype, b, blk = TYPE[c["dtype"]], c["batch"], c["block"]
    unit = c["page"] or blk
    hq = c["hkv"] * c.get("group", 1)
    if c["op"] == "append":
        r = random.Random("%d %d" % (b, c["start"]))
        starts = [c["start"] + r.randrange(2 * blk) if c["start"] else 0 for _ in range(b)]
        tokens = -(-(max(starts) + c["new"] + 2 * blk) // unit) * unit
        for name in "kv":
            s[name] = torch.zeros((b, c["hkv"], tokens, D), dtype=torch.uint8, device=dev).view(CODE[c["fmt"]])
            s[name + "_scale"] = torch.zeros((b, c["hkv"], tokens // blk), dtype=torch.float32, device=dev)
            s["open_" + name] = _rows(g, (b, c["hkv"], blk, D), dtype, dev)
            s["new_" + name] = _rows(g, (b, c["new"], c["hkv"], D), dtype, dev).transpose(1, 2)
        s["starts"] = _i32(starts, dev)
        if c["page"]:
            _paginate(g, c, s, dev)
        return s
    lens = _lens(c)
    tokens = -(-max(lens) // unit) * unit
    s.update(_store(g, c, tokens, dev))
    s["lens"] = _i32(lens, dev)
    s["q"] = _rows(g, (b, hq, D), dtype, dev, 0.75)
    if c["op"] == "dense":
        for name in "kv":
            s["open_" + name] = _rows(g, (b, c["hkv"], blk, D), dtype, dev, 0.5 if name == "k" else 1.0)
        if c["selector"]:
            s["scores"] = torch.zeros((b, max(lens)), dtype=torch.float32, device=dev)
    else:
        picks = _picks(c)
        idx = torch.full((b, max(picks)), -1, dtype=torch.int32, device=dev)
        for i, (n, k) in enumerate(zip(lens, picks)):
            idx[i, :k] = torch.randperm(n, generator=g, device=dev)[:k].sort()[0].to(torch.int32)
        s["idx"], s["picks"] = idx, _i32(picks, dev)
        if c["tail"]:
            for name in "kv":
                s["tail_" + name] = _rows(g, (b, c["hkv"], c["tail"], D), dtype, dev, 0.5 if name == "k" else 1.0)
    if c["page"]:
        _paginate(g, c, s, dev)
    if c["op"] == "sparse" and c["page"]:  # composed once per selection by the caller: rows of the pool seen flat
        t = s["idx"].clamp(min=0).long()
        flat = s["table"].gather(1, t // c["page"]).long() * c["page"] + t % c["page"]
        s["slots"] = torch.where(s["idx"] < 0, s["idx"], flat.to(torch.int32))
    return s


def _prepare_pages(s, c, g, r, dev):
    page = c["page"]
    lens = _fork_lens(c) if c["op"] == "fork" else _compact_lens(c)
    n = len(lens)
    count = [-(-x // page) for x in lens]
    if c["op"] == "fork":
        # the continuations of the step before: each still holds one page of its own
        pages = sum(count) + n * (2 + -(-c["more"] // page)) + 7
        width = max(count) + 2 + -(-c["more"] // page)
    else:
        pages, width = c["pages"], max(count) + 1
    order = r.sample(range(pages), sum(count) + (n if c["op"] == "fork" else 0))
    rows = 2 * n if c["op"] == "fork" else n
    table, refs, at = [[-1] * width for _ in range(rows)], [0] * pages, 0
    for i in range(n):
        table[i][:count[i]] = order[at:at + count[i]]
        at += count[i]
    all_lens = list(lens)
    if c["op"] == "fork":
        for i in range(n):
            table[n + i][0] = order[at]
            at += 1
            all_lens.append(1 + r.randrange(page))
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    s["page_table"], s["refs"], s["seq_lens"] = _i32(table, dev), _i32(refs, dev), _i32(all_lens, dev)
    for name in "kv":
        s[name] = torch.randint(0, 120, (c["layers"], pages, page, c["hkv"], D), generator=g, device=dev, dtype=torch.uint8)
        s[name + "_scale"] = torch.rand((c["layers"], pages, page // c["block"], c["hkv"]), generator=g, device=dev)
    s["buffers"] = [s[name][i] for i in range(c["layers"]) for name in ("k", "v", "k_scale", "v_scale")]
    if c["op"] == "fork":
        s["from"], s["to"] = _i32(_fork_parents(c), dev), _i32(list(range(n, 2 * n)), dev)
        s["grow"] = torch.full((n,), c["more"], dtype=torch.int32, device=dev)
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _values(s, name, at=None):
    """(batch, heads, tokens, D) fp32 values of the cache; at: (batch, n) token positions instead of all."""
    c = s["case"]
    blk = c["block"]
    if c["page"]:
        if at is None:
            per = s["table"].shape[1] * c["page"]
            at = torch.arange(per, device=s["k"].device).expand(c["batch"], per)
        slot = s["table"].gather(1, at // c["page"]).long() * c["page"] + at % c["page"]
        x = s[name].flatten(0, 1).view(torch.uint8)[slot].view(CODE[c["fmt"]]).float()
        x = x * s[name + "_scale"].flatten(0, 1)[slot // blk][..., None]
        return x.transpose(1, 2)
    if at is None:
        x = s[name].float().unflatten(2, (-1, blk)) * s[name + "_scale"][..., None, None]
        return x.flatten(2, 3)
    i = at[:, None, :].expand(-1, c["hkv"], -1)
    x = s[name].view(torch.uint8).gather(2, i[..., None].expand(-1, -1, -1, D)).view(CODE[c["fmt"]]).float()
    return x * s[name + "_scale"].gather(2, i // blk)[..., None]


def _softmax_attention(q, k, v, valid, hkv):
    """q (b, Hq, D), k / v (b, heads, n, D) fp32, valid (b, n) -> logits (b, Hq, n), output (b, Hq, D)."""
    b, hq, _ = q.shape
    qg = q.float().view(b, hkv, hq // hkv, D).transpose(2, 3).contiguous()
    logits = torch.matmul(k, qg).transpose(2, 3).reshape(b, hq, -1) * D ** -0.5
    masked = logits.masked_fill(~valid[:, None], float("-inf"))
    p = torch.exp(masked - masked.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, hkv, hq // hkv, -1), v.contiguous())
    return logits, out.reshape(b, hq, D).to(q.dtype)


def _plain_append(s):
    c = s["case"]
    blk, b, hkv, new = c["block"], c["batch"], c["hkv"], c["new"]
    dev = s["k"].device
    start = s["starts"].long()
    first, have = start // blk * blk, start % blk
    span = -(-(new + blk - 1) // blk) * blk if c["start"] else -(-new // blk) * blk
    i = torch.arange(span, device=dev)
    from_new = (i[None] >= have[:, None]) & (i[None] < (have + new)[:, None])  # (b, span)
    done = torch.arange(blk, span + 1, blk, device=dev)[None] <= (have + new)[:, None]  # (b, blocks)
    if c["close"]:
        done = torch.arange(0, span, blk, device=dev)[None] < (have + new)[:, None]
    pos = first[:, None] + i[None]
    for name in "kv":
        src = (i[None] - have[:, None]).clamp(0, new - 1)[:, None, :, None].expand(-1, hkv, -1, D)
        x = s["new_" + name].gather(2, src)
        old = s["open_" + name].gather(2, (i % blk)[None, None, :, None].expand(b, hkv, -1, D))
        x = torch.where(from_new[:, None, :, None], x, old)
        held = x.masked_fill((i[None] >= (have + new)[:, None])[:, None, :, None], 0.0)  # a closed last block is short
        codes, scale = _quantise(held.unflatten(2, (-1, blk)), c["fmt"])
        codes, row_ok = codes.flatten(2, 3).view(torch.uint8), done.repeat_interleave(blk, 1) & (i[None] < (have + new)[:, None])
        if c["page"]:
            slot = s["table"].gather(1, pos // c["page"]).long() * c["page"] + pos % c["page"]
            flat = s[name].view(torch.uint8).flatten(0, 1)
            flat[slot] = torch.where(row_ok[..., None, None], codes.transpose(1, 2), flat[slot])
            sc, at = s[name + "_scale"].flatten(0, 1), slot[:, ::blk] // blk
            sc[at] = torch.where(done[..., None], scale.transpose(1, 2), sc[at])
        else:
            at = pos[:, None, :, None].expand(-1, hkv, -1, D)
            flat = s[name].view(torch.uint8)
            flat.scatter_(2, at, torch.where(row_ok[:, None, :, None], codes, flat.gather(2, at)))
            sc, at = s[name + "_scale"], (pos[:, ::blk] // blk)[:, None].expand(-1, hkv, -1)
            sc.scatter_(2, at, torch.where(done[:, None], scale, sc.gather(2, at)))
        if not c["close"]:
            # rows of the block that is still open
            end = have + new
            at = (end // blk * blk)[:, None] + torch.arange(blk, device=dev)[None]  # (b, blk) within the span
            ok = (at >= have[:, None]) & (at < end[:, None])
            rows = x.gather(2, at.clamp(max=span - 1)[:, None, :, None].expand(-1, hkv, -1, D))
            s["open_" + name].copy_(torch.where(ok[:, None, :, None], rows, s["open_" + name]))
    return _appended(s)


def _appended(s):
    return [s["k"], s["v"], s["k_scale"], s["v_scale"], s["open_k"], s["open_v"]]


def _reduce_scores(logits, valid, selector):
    if selector == "last":
        return logits.amax(1)
    logits = logits.masked_fill(~valid[:, None], float("-inf"))
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return p.amax(1) if selector == "softmax_before_last" else p.sum(1)


def _plain_dense(s):
    c = s["case"]
    blk, n = c["block"], c["hi"]
    lens = s["lens"].long()
    pos = torch.arange(n, device=lens.device)[None]
    closed = lens // blk * blk
    kv = []
    for name in "kv":
        x = _values(s, name)[:, :, :n]
        late = s["open_" + name].float().gather(2, (pos % blk)[:, None, :, None].expand(c["batch"], c["hkv"], -1, D))
        kv.append(torch.where((pos >= closed[:, None])[:, None, :, None], late, x))
    valid = pos < lens[:, None]
    logits, out = _softmax_attention(s["q"], kv[0], kv[1], valid, c["hkv"])
    if not c["selector"]:
        return out
    scores = _reduce_scores(logits, valid, c["selector"])
    s["scores"].copy_(torch.where(valid, scores, s["scores"]))
    return [out, s["scores"]]


def _plain_sparse(s):
    c = s["case"]
    at = s["idx"].clamp(min=0).long()
    k, v = _values(s, "k", at), _values(s, "v", at)
    valid = torch.arange(at.shape[1], device=at.device)[None] < s["picks"][:, None]
    if c["tail"]:
        k = torch.cat([k, s["tail_k"].float()], 2)
        v = torch.cat([v, s["tail_v"].float()], 2)
        valid = torch.cat([valid, valid.new_ones((c["batch"], c["tail"]))], 1)
    return _softmax_attention(s["q"], k, v, valid, c["hkv"])[1]


def _plain_free(table, lens, refs, seqs):
    rows = table[seqs]
    held = rows[rows >= 0].long()
    refs.index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    table[seqs] = -1
    lens[seqs] = 0


def _plain_fork(s):
    c = s["case"]
    page, table, refs, lens = c["page"], s["page_table"], s["refs"], s["seq_lens"]
    src, dst = s["from"].long(), s["to"].long()
    _plain_free(table, lens, refs, dst)
    # shared: the parents' full pages; the partly filled last one is copied to a free page
    col = torch.arange(table.shape[1], device=table.device)[None]
    rows, n = table[src], lens[src].long()
    full, part = n // page, n % page > 0
    table[dst] = torch.where(col < full[:, None], rows, -1)
    lens[dst] = lens[src]
    held = rows[col < full[:, None]].long()
    refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    fresh = torch.nonzero(refs == 0)[:, 0][: int(part.sum())]
    old = rows[part, full[part]].long()
    for buf in s["buffers"]:
        buf[fresh] = buf[old]
    table[dst[part], full[part]] = fresh.to(torch.int32)
    refs[fresh] = 1
    # room for `grow` more tokens: the lowest free pages, sequence by sequence
    want = lens[dst].long() + s["grow"].long()
    have, need = -(-lens[dst].long() // page), -(-want // page)
    r, x = torch.nonzero((col >= have[:, None]) & (col < need[:, None]), as_tuple=True)
    fresh = torch.nonzero(refs == 0)[:, 0][: r.numel()]
    table[dst[r], x] = fresh.to(torch.int32)
    refs[fresh] = 1
    lens[dst] = want.to(torch.int32)
    return [table, refs, lens] + [s[n] for n in ("k", "v", "k_scale", "v_scale")]


def _plain_compact(s):
    table, refs = s["page_table"], s["refs"]
    used = refs > 0
    n = int(used.sum())
    src, dst = torch.nonzero(used[n:])[:, 0] + n, torch.nonzero(~used[:n])[:, 0]
    to = torch.arange(refs.numel(), device=refs.device, dtype=torch.int32)
    to[src] = dst.to(torch.int32)
    for buf in s["buffers"]:
        buf[dst] = buf[src]
    refs_out = torch.zeros_like(refs)
    refs_out[to[used].long()] = refs[used]
    table_out = torch.where(table >= 0, to[table.clamp(min=0).long()], table)
    return [table_out, refs_out] + [s[n] for n in ("k", "v", "k_scale", "v_scale")]


_plain = {"append": _plain_append, "dense": _plain_dense, "sparse": _plain_sparse, "fork": _plain_fork,
          "compact": _plain_compact}


# ------------------------------------------------------------------------------------------ the framework's calls
def _cache(s):
    """The handle a program keeps next to its tensors."""
    from omnikv_amd import ops

    if "cache" not in s:
        s["cache"] = ops.KV8(s["k"], s["v"], s["k_scale"], s["v_scale"], s["case"]["block"], open_k=s.get("open_k"),
                             open_v=s.get("open_v"), page_table=s.get("table"))
    return ops, s["cache"]


def _own_append(s):
    ops, cache = _cache(s)
    c = s["case"]
    ops.kv8_append(cache, s["new_k"], s["new_v"], 0 if not c["start"] else s["starts"], close=c["close"])
    return _appended(s)


def _own_dense(s):
    ops, cache = _cache(s)
    c = s["case"]
    if not c["selector"]:
        return ops.kv8_dense_attn(s["q"], cache, seq_len=c["hi"], seq_lens=s["lens"])
    out, scores = ops.kv8_dense_attn(s["q"], cache, seq_len=c["hi"], seq_lens=s["lens"], selector=c["selector"],
                                     score_len=c["hi"], score_lens=s["lens"], scores_out=s["scores"])
    return [out, scores]


def _own_sparse(s):
    ops, cache = _cache(s)
    tail = {"tail_k": s["tail_k"], "tail_v": s["tail_v"]} if s["case"]["tail"] else {}
    if "slots" in s:
        return ops.kv8_sparse_attn(s["q"], cache, slots=s["slots"], sel_lens=s["picks"], **tail)
    return ops.kv8_sparse_attn(s["q"], cache, idx=s["idx"], sel_lens=s["picks"], **tail)


def _buffers(s):
    """The list of the layers' arrays, made once by a program."""
    from omnikv_amd import ops

    if "handle" not in s:
        s["handle"] = ops.PageBuffers(s["buffers"])
    return ops, s["handle"]


def _own_fork(s):
    ops, buffers = _buffers(s)
    page, state = s["case"]["page"], (s["page_table"], s["seq_lens"], s["refs"])
    ops.pages_free(*state, s["to"], page)
    ops.pages_fork(*state, s["from"], s["to"], page, buffers)
    ops.pages_extend(*state, s["to"], s["grow"], page)
    return [s["page_table"], s["refs"], s["seq_lens"]] + [s[n] for n in ("k", "v", "k_scale", "v_scale")]


def _own_compact(s):
    ops, buffers = _buffers(s)
    table, refs, _ = ops.pages_compact(s["page_table"], s["refs"], buffers)
    return [table, refs] + [s[n] for n in ("k", "v", "k_scale", "v_scale")]


_own = {"append": _own_append, "dense": _own_dense, "sparse": _own_sparse, "fork": _own_fork, "compact": _own_compact}


# ------------------------------------------------------------------------------------------ 64 bits
def _exact_rows(s, name):
    """Every cached row of every request in 64 bits, (batch, heads, tokens, D), request by request."""
    c = s["case"]
    got = []
    for b in range(c["batch"]):
        if c["page"]:
            pages = s["table"][b].long()
            codes = s[name][pages].double().flatten(0, 1)  # (tokens, heads, D)
            scale = s[name + "_scale"][pages].double().flatten(0, 1).repeat_interleave(c["block"], 0)
            got.append((codes * scale[..., None]).permute(1, 0, 2))
        else:
            scale = s[name + "_scale"][b].double().repeat_interleave(c["block"], 1)
            got.append(s[name][b].double() * scale[..., None])
    return got


def _exact_attention(s):
    c = s["case"]
    keys, vals = _exact_rows(s, "k"), _exact_rows(s, "v")
    outs, scores = [], s["scores"].double() if c.get("selector") else None
    for b, n in enumerate(_lens(c)):
        k, v = keys[b], vals[b]
        if c["op"] == "dense":
            closed = n // c["block"] * c["block"]
            late = n - closed
            k = torch.cat([k[:, :closed], s["open_k"][b, :, :late].double()], 1)
            v = torch.cat([v[:, :closed], s["open_v"][b, :, :late].double()], 1)
        else:
            at = s["idx"][b, :_picks(c)[b]].long()
            k, v = k[:, at], v[:, at]
            if c["tail"]:
                k, v = torch.cat([k, s["tail_k"][b].double()], 1), torch.cat([v, s["tail_v"][b].double()], 1)
        q = s["q"][b].double().view(c["hkv"], -1, D)
        x = torch.bmm(q, k.transpose(1, 2).contiguous()) / D ** 0.5  # (heads, group, n)
        p = torch.softmax(x, -1)
        outs.append(torch.bmm(p, v.contiguous()).reshape(-1, D))
        if scores is not None:
            y = x if c["selector"] == "last" else p
            y = y.reshape(-1, n)
            scores[b, :n] = y.sum(0) if c["selector"] == "softmax_sum_last" else y.amax(0)
    return torch.stack(outs) if scores is None else [torch.stack(outs), scores]


def _to_e4m3(y):
    """The nearest e4m3 value (ties to even) of a 64-bit number within +-448."""
    a = y.abs().clamp(min=2.0 ** -6)
    step = a / torch.frexp(a)[0] / 16  # a = m 2^e with m in [1/2, 1): three bits behind the leading one
    return torch.round(y / step) * step


def _exact_append(s):
    c = s["case"]
    blk, n = c["block"], c["new"]
    out = {}
    for name in "kv":
        codes, scales, opened = s[name].double(), s[name + "_scale"].double(), s["open_" + name].double()
        for b, start in enumerate(s["starts"].tolist()):
            have, first = start % blk, start // blk
            x = torch.cat([opened[b][:, :have], s["new_" + name][b].double()], 1)  # from the first touched block on
            full = -(-x.shape[1] // blk) if c["close"] else x.shape[1] // blk
            late = x[:, full * blk:]
            short = max(0, full * blk - x.shape[1])
            y = torch.nn.functional.pad(x[:, :full * blk], (0, 0, 0, short)).unflatten(1, (full, blk))
            # the format fixes three fp32 roundings: of the scale, of its reciprocal and of the product
            sc = (y.abs().amax((2, 3)) / QMAX[c["fmt"]]).float().double().clamp(min=2.0 ** -126)
            y = (y * (1 / sc).float().double()[..., None, None]).float().double()
            y = torch.round(y).clamp(-127, 127) if c["fmt"] == "int8" else _to_e4m3(y.clamp(-448, 448))
            y = y.flatten(1, 2)[:, :full * blk - short]
            if c["page"]:
                per = c["page"] // blk
                for j in range(full):
                    p, o = int(s["table"][b, (first + j) // per]), (first + j) % per
                    rows = y[:, j * blk:(j + 1) * blk].transpose(0, 1)
                    codes[p, o * blk:o * blk + rows.shape[0]] = rows
                    scales[p, o] = sc[:, j]
            else:
                codes[b, :, first * blk:first * blk + y.shape[1]] = y
                scales[b, :, first:first + full] = sc
            if not c["close"]:
                at = 0 if full else have
                opened[b][:, at:late.shape[1]] = late[:, at:]
        out[name], out[name + "_scale"], out["open_" + name] = codes, scales, opened
    if c["fmt"] == "int8":  # whole numbers are compared as they are
        out["k"] = out["v"] = None
    return [out[n] for n in ("k", "v", "k_scale", "v_scale", "open_k", "open_v")]


def exact(case, seed):
    if case["op"] in ("fork", "compact"):  # pages and whole numbers: nothing is computed in floating point
        return None
    if case["op"] == "append" and case["page"] and case["new"] > 4096:
        return None
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attention(s)
