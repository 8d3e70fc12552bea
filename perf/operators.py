"""Cases for measuring the paged K/V cache operators (cache_write, cache_read, cache_attn) and their plain forms.

A cache holds rows of 128 values per token and K/V head in pages of `page` tokens: bf16 values, or e4m3 values with one
power-of-two exponent per row (byte = exponent + 127).  A batch names, per sequence b, its pages (`pages[b]`), how many
tokens it holds (`lengths[b]`) and which rows of a packed tensor are its newest tokens (`starts[b] .. starts[b + 1]`):
row i of the n_b rows is the token at position lengths[b] - n_b + i.

With `own` false everything is computed in elementary torch operations in fp32; with `own` true by the package's calls.
"""
import random

import torch

own = False

D = 128
HEADS = 40        # heads of the joint attention
FRAME = 30 * 52   # tokens of one latent frame at the 480p-like size
CLIP = 49384      # the whole 480p-like sequence: 31 frames and 1,024 audio tokens


def listed():
    def c(name, op, batch, new, length, heads, kv_heads, page, quantised, causal=False):
        return {"name": name, "op": op, "batch": batch, "new_min": new[0], "new_max": new[1], "len_min": length[0], "len_max": length[1],
                "heads": heads, "kv_heads": kv_heads, "page": page, "quantised": quantised, "causal": causal}

    return [
        # the newest token of four sequences enters the cache: a call whose latency counts
        c("write tokens e4m3", "write", 4, (1, 1), (77, 4096), 40, 40, 16, True),
        # a ragged batch of prompts is cached unquantised, K/V heads shared by groups of query heads
        c("write prompts bf16", "write", 5, (33, 1157), (33, 2341), 40, 8, 48, False),
        # K and V of a whole clip are quantised into the cache
        c("write clip e4m3", "write", 1, (CLIP, CLIP), (CLIP, CLIP), 40, 40, 128, True),
        # two text prompts are read back
        c("read prompts e4m3", "read", 2, (77, 512), (77, 512), 40, 40, 16, True),
        # half a clip's frames are read back for a dense call
        c("read frames e4m3", "read", 2, (8 * FRAME, 8 * FRAME), (8 * FRAME, CLIP), 40, 40, 64, True),
        # one new token of one sequence
        c("attn token short bf16", "attn", 1, (1, 1), (1023, 1023), 40, 40, 16, False, True),
        # one new token of each of 32 sequences of very different lengths
        c("attn tokens ragged e4m3", "attn", 32, (1, 1), (200, 16384), 40, 8, 32, True, True),
        # one new token each over two long contexts
        c("attn token long bf16", "attn", 2, (1, 1), (65537, 131072), 40, 8, 128, False, True),
        # small ragged chunks with an odd group of query heads and pages that do not divide a tile
        c("attn chunks ragged bf16", "attn", 5, (3, 301), (450, 9001), 21, 3, 48, False, True),
        # a chunk of a long prompt over a quantised context
        c("attn chunk e4m3", "attn", 1, (2048, 2048), (20011, 20011), 40, 8, 64, True, True),
        # three new frames see each other and the whole clip before them
        c("attn frames bf16", "attn", 1, (3 * FRAME, 3 * FRAME), (CLIP, CLIP), 40, 40, 128, False, False),
        # three frames and one frame over the cached states of two prompts of another length
        c("attn text e4m3", "attn", 2, (FRAME, 3 * FRAME), (77, 512), 40, 40, 16, True, False),
    ]


def draw(rng):
    def log(a, b):
        return max(a, min(b, int(round(a * (b / a) ** rng.random()))))

    while True:
        op = rng.choice(("write", "read", "attn", "attn", "attn"))
        batch = log(1, 40)
        kv_heads = rng.choice((1, 2, 3, 5, 8, 10, 20, 40))
        heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 5, 7, 8))
        page = 16 * log(1, 16)
        quantised = rng.random() < 0.5
        causal = op == "attn" and rng.random() < 0.6
        len_max = log(16, 140000)
        len_min = log(1, len_max)
        new_max = 1 if op == "attn" and rng.random() < 0.4 else log(1, CLIP if op != "attn" else 3 * FRAME)
        if op != "attn" or causal:
            new_max = min(new_max, len_max)
        new_min = log(1, new_max)
        case = {"op": op, "batch": batch, "new_min": new_min, "new_max": new_max, "len_min": len_min, "len_max": len_max,
                "heads": heads, "kv_heads": kv_heads, "page": page, "quantised": quantised, "causal": causal}
        n, length = _extents(case)
        if sum(-(-x // page) for x in length) * page * kv_heads > 2 * CLIP * HEADS // (1 if quantised else 2) or heads > 64:
            continue
        if op == "attn" and (batch * max(n) * max(length) * heads > 3 * FRAME * CLIP * HEADS // 2 or batch * max(length) * kv_heads > 4 * CLIP * HEADS):
            continue
        return case


def _extents(case):
    """New tokens and lengths of the batch's sequences: spread evenly over the logarithm, in an order of their own."""
    b = case["batch"]
    r = random.Random(b * 1000003 + case["len_max"] * 101 + case["new_max"])

    def spread(lo, hi):
        v = [hi] if b == 1 else [int(round(lo * (hi / lo) ** (i / (b - 1)))) for i in range(b)]
        r.shuffle(v)
        return v

    n, length = spread(case["new_min"], case["new_max"]), spread(case["len_min"], case["len_max"])
    if case["op"] != "attn" or case["causal"]:
        length = [max(x, y) for x, y in zip(n, length)]
    return n, length


# ---------------------------------------------------------------------------------------------------- e4m3 rows
def _quantise(x):
    """Rows of x [..., 128] fp32 as (e4m3 values, exponent bytes): the smallest power of two that brings the row's largest
    magnitude to at most 448 divides the row."""
    m, e = torch.frexp(x.abs().amax(-1))
    k = torch.where(m <= 0.875, e - 9, e - 8).clamp(-120, 120)
    k = torch.where(m == 0, torch.full_like(k, -120), k)
    return (x * _power(-k)[..., None]).to(torch.float8_e4m3fn), (k + 127).to(torch.uint8)


def _power(k):
    """2^k in fp32, from its bits."""
    return ((k.int() + 127) << 23).view(torch.float32)


def _power64(k):
    return ((k.long() + 1023) << 52).view(torch.float64)


def _put(s, x, page, at, rows):
    if s["exp_" + x] is None:
        s["pool_" + x][page, at] = rows
    else:
        rows, exps = _quantise(rows.float())
        s["pool_" + x].view(torch.uint8)[page, at] = rows.view(torch.uint8)
        s["exp_" + x][page, at] = exps


def _take(s, x, page, at):
    """Cached rows as fp32 values."""
    if s["exp_" + x] is None:
        return s["pool_" + x][page, at].float()
    rows = s["pool_" + x].view(torch.uint8)[page, at].view(torch.float8_e4m3fn)
    return rows.float() * _power(s["exp_" + x][page, at].int() - 127)[..., None]


# ---------------------------------------------------------------------------------------------------- states
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 13)
    n, length = _extents(case)
    page, hk = case["page"], case["kv_heads"]
    per = [-(-x // page) for x in length]
    n_pages = sum(per) + 3
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    pages = torch.zeros(case["batch"], max(per), dtype=torch.int32, device=dev)
    at = 0
    for b, x in enumerate(per):
        pages[b, :x] = order[at : at + x]
        at += x
    starts = [0]
    for x in n:
        starts.append(starts[-1] + x)
    s = {"op": case["op"], "causal": case["causal"], "page": page, "rows": starts[-1], "new_max": max(n), "len_max": max(length),
         "pages": pages, "lengths": torch.tensor(length, dtype=torch.int32, device=dev),
         "starts": torch.tensor(starts, dtype=torch.int32, device=dev)}
    pool = lambda: torch.randn(n_pages, hk, page, D, generator=g, device=dev, dtype=torch.bfloat16)  # noqa: E731
    # head-major inside a page, as the package lays pages out: the logical order is [pages, page, heads, 128]
    for x in ("k", "v"):
        rows, exps = pool(), None
        if case["quantised"]:
            rows, exps = _quantise(rows.float())
            exps = exps.transpose(1, 2)
        s["pool_" + x], s["exp_" + x] = rows.transpose(1, 2), exps
    if case["op"] == "write":
        for x in ("k", "v"):  # rows as a projection leaves them: unit rows with a scale of their own
            s[x] = torch.randn(s["rows"], hk, D, generator=g, device=dev, dtype=torch.bfloat16)
            s[x] *= torch.exp(torch.randn(s["rows"], hk, 1, generator=g, device=dev)).bfloat16()
    if case["op"] == "attn":
        s["q"] = torch.randn(s["rows"], case["heads"], D, generator=g, device=dev, dtype=torch.bfloat16)
    if own:
        import pika_h3_flex_b200 as h3

        s["h3"] = h3
        s["cache"] = h3.KVCache(s["pool_k"], s["pool_v"], s["exp_k"], s["exp_v"])
        s["batch"] = h3.CacheBatch(s["pages"], s["lengths"], s["starts"])
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        h3 = s["h3"]
        if s["op"] == "write":
            h3.cache_write(s["cache"], s["batch"], s["k"], s["v"])
            return _pools(s)
        if s["op"] == "read":
            return h3.cache_read(s["cache"], s["batch"], s["rows"])
        return h3.cache_attn(s["q"], s["cache"], s["batch"], causal=s["causal"], return_lse=True)
    return {"write": _write, "read": _read, "attn": _attn}[s["op"]](s)


def _pools(s):
    return [s["pool_k"], s["pool_v"]] + ([] if s["exp_k"] is None else [s["exp_k"], s["exp_v"]])


def _sequence_of_rows(s):
    """Sequence and position of each packed row."""
    t = torch.arange(s["rows"], device=s["starts"].device)
    b = torch.searchsorted(s["starts"][1:].long(), t, right=True)
    first = (s["lengths"] - (s["starts"][1:] - s["starts"][:-1])).long()
    return t, b, first[b] + t - s["starts"].long()[b]


def _write(s):
    _, b, pos = _sequence_of_rows(s)
    page, at = s["pages"].long()[b, pos // s["page"]], pos % s["page"]
    for x in ("k", "v"):
        _put(s, x, page, at, s[x])
    return _pools(s)


def _read(s):
    _, b, pos = _sequence_of_rows(s)
    page, at = s["pages"].long()[b, pos // s["page"]], pos % s["page"]
    return [_take(s, x, page, at).bfloat16() for x in ("k", "v")]


def _attn(s):
    q, starts, length = s["q"], s["starts"].long(), s["lengths"].long()
    rows, heads = q.shape[:2]
    batch, kv_heads = length.numel(), s["pool_k"].shape[2]
    group, n_max, l_max = heads // kv_heads, s["new_max"], s["len_max"]
    n = starts[1:] - starts[:-1]
    j = torch.arange(l_max, device=q.device)
    page, at = s["pages"].long()[:, j // s["page"]], (j % s["page"]).expand(batch, l_max)
    k, v = (_take(s, x, page, at).transpose(1, 2) for x in ("k", "v"))
    i = torch.arange(n_max, device=q.device)
    x = q[(starts[:-1, None] + i).clamp(max=rows - 1)].float().view(batch, n_max, kv_heads, group, D)
    x = x.permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, n_max * group, D)
    p = (x * D ** -0.5) @ k.transpose(2, 3)
    seen = j < length[:, None, None]
    if s["causal"]:
        seen = seen & (j <= (length - n)[:, None, None] + i[:, None])
    p.view(batch, kv_heads, n_max, group, l_max).masked_fill_(~seen[:, None, :, None, :], float("-inf"))
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    total = p.sub_(top).exp_().sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (total.log() + top).view(batch, kv_heads, n_max, group)
    t, b, _ = _sequence_of_rows(s)
    r = t - starts[b]
    out = o.view(batch, kv_heads, n_max, group, D)[b, :, r].reshape(rows, heads, D).bfloat16()
    return [out, lse[b, :, r].reshape(rows, heads).transpose(0, 1).contiguous()]


# ---------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    n, length = _extents(case)
    page, quantised = case["page"], case["quantised"]

    def stored(x, b, lo, hi):
        """Rows lo..hi of sequence b in 64 bits, [hi - lo, kv_heads, 128]."""
        p = torch.arange(lo, hi, device=s["starts"].device)
        ids = s["pages"][b].long()[torch.div(p, page, rounding_mode="floor")]
        if not quantised:
            return s["pool_" + x][ids, p % page].double()
        rows = s["pool_" + x].view(torch.uint8)[ids, p % page].view(torch.float8_e4m3fn)
        return rows.double() * _power64(s["exp_" + x][ids, p % page].int() - 127)[..., None]

    if case["op"] == "read":
        return [torch.cat([stored(x, b, length[b] - n[b], length[b]) for b in range(case["batch"])]) for x in ("k", "v")]
    if case["op"] == "write":
        found = []
        for x in ("k", "v"):
            pool = s["pool_" + x].double()
            at = 0
            for b in range(case["batch"]):
                rows = s[x][at : at + n[b]].double()
                at += n[b]
                if quantised:
                    # the least exponent k with largest <= 448 * 2^k; then 4 significant bits, 2^-9 the least step
                    largest = rows.abs().amax(-1, keepdim=True)
                    k = torch.ceil(torch.log2(largest / 448.0)).clamp(-120, 120)
                    k = torch.where(largest <= 448.0 * _power64(k - 1), k - 1, torch.where(largest > 448.0 * _power64(k), k + 1, k)).clamp(-120, 120)
                    y = rows / _power64(k)
                    _, e = torch.frexp(y.abs().clamp(min=2.0 ** -6))
                    step = _power64(e - 4)
                    rows = torch.round(y / step) * step
                p = torch.arange(length[b] - n[b], length[b], device=rows.device)
                pool[s["pages"][b].long()[torch.div(p, page, rounding_mode="floor")], p % page] = rows
            found.append(pool)
        return found + ([None, None] if quantised else [])
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["rows"], case["heads"], D, dtype=torch.float64, device=s["q"].device)
    lse = torch.full((case["heads"], s["rows"]), float("-inf"), dtype=torch.float64, device=s["q"].device)
    at = 0
    for b in range(case["batch"]):
        k, v = stored("k", b, 0, length[b]), stored("v", b, 0, length[b])
        position = length[b] - n[b] + torch.arange(n[b], device=k.device)
        hidden = torch.arange(length[b], device=k.device)[None, :] > position[:, None]
        for h in range(case["heads"]):
            logits = s["q"][at : at + n[b], h].double() @ k[:, h // group].T / D ** 0.5
            if case["causal"]:
                logits = logits.masked_fill(hidden, float("-inf"))
            z = torch.logsumexp(logits, 1)
            out[at : at + n[b], h] = torch.exp(logits - z[:, None]) @ v[:, h // group]
            lse[h, at : at + n[b]] = z
        at += n[b]
    return [out, lse]


# ---------------------------------------------------------------------------------------------------- what it takes
def work(case):
    n, length = _extents(case)
    row = D + 1 if case["quantised"] else 2 * D  # bytes of one cached row
    if case["op"] != "attn":  # K and V: bf16 rows on one side, cached rows on the other
        return {"bytes": 2 * sum(n) * case["kv_heads"] * (2 * D + row), "flops": 0}
    seen = [x * y - (x * (x - 1) // 2 if case["causal"] else 0) for x, y in zip(n, length)]
    return {"bytes": sum(n) * case["heads"] * (4 * D + 4) + 2 * sum(length) * case["kv_heads"] * row,
            "flops": 4 * D * case["heads"] * sum(seen)}
