"""Operators of generating text for many sequences at once, as cases that can be timed.

Four kinds of work, next to one another in a decoding program:

* ``write``   the rotary step of new rows and their keys and values into a cache of 4-bit numbers, and those rows read back;
* ``attn``    attention of one row (a decoded token) or several rows (drafted tokens, a piece of a prompt) of each sequence
              over such a cache;
* ``pages``   pages of the cache copied, in all layers: when a sequence is forked, or a cache compacted;
* ``sample``  the next token of each sequence from its logits: temperature, top-k, top-p, min-p and a given random number.

The cache lies in pages of 64 positions, ``pool`` uint8 [pages][kv_heads][64 * (hd + hd / 8)] per layer, and ``table`` names the
pages of a sequence in order.  The record of a page and head holds the codes of the keys [64][hd / 2], those of the values, then
(scale, low) of the keys as fp16 [64][hd / 64][2], then of the values.  64 numbers next to one another in a row are a group:

    low = min, scale = half((max - min) / 15), code = min(15, rint((x - low) * (1 / scale))), value = low + scale * code

with every step in 32-bit arithmetic.  Byte j of a group's 32 bytes holds the numbers 2j (low half) and 2j + 1, and the groups of
position p are stored in the order g ^ f(p), see `_order`.  A rotated number is the exact a * cos - b * sin rounded to 32 and then to
16 bits.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64


def listed():
    return [
        # one new token of each of sixteen sequences of a 7B decoder: launch latency
        {"name": "write_token_16", "kind": "write", "batch": 16, "m": 1, "heads": 32, "kv_heads": 32, "hd": 128, "first": 40, "last": 2000},
        # the rows of a prompt, 70B heads, starting and ending inside a page
        {"name": "write_prompt", "kind": "write", "batch": 1, "m": 1537, "heads": 64, "kv_heads": 8, "hd": 128, "first": 211, "last": 211},
        # a small decoder's token early in a text: the smallest call
        {"name": "attn_token_small", "kind": "attn", "batch": 1, "m": 1, "heads": 4, "kv_heads": 2, "hd": 64, "first": 99, "last": 99, "ragged": False},
        # one token of sixteen sequences of different lengths, 7B heads
        {"name": "attn_token_16", "kind": "attn", "batch": 16, "m": 1, "heads": 32, "kv_heads": 32, "hd": 128, "first": 300, "last": 4000, "ragged": False},
        # one token of three sequences with long texts, 70B heads: the cache's bytes
        {"name": "attn_token_long", "kind": "attn", "batch": 3, "m": 1, "heads": 64, "kv_heads": 8, "hd": 128, "first": 70001, "last": 100003, "ragged": False},
        # up to five drafted tokens of six sequences, 70B heads, fewer rows in some of them
        {"name": "attn_draft", "kind": "attn", "batch": 6, "m": 5, "heads": 64, "kv_heads": 8, "hd": 128, "first": 1000, "last": 6000, "ragged": True},
        # the last piece of a 2048-token prompt, 7B heads: the matrix products
        {"name": "attn_prompt", "kind": "attn", "batch": 1, "m": 512, "heads": 32, "kv_heads": 32, "hd": 128, "first": 1536, "last": 1536, "ragged": False},
        # a sequence of a small decoder forked once: one page copied in two layers
        {"name": "pages_fork_small", "kind": "pages", "layers": 2, "pages": 16, "kv_heads": 2, "hd": 64, "pairs": 1},
        # the last, partly filled pages of fifteen forks of one prompt, 32 layers, 7B heads
        {"name": "pages_fork_15", "kind": "pages", "layers": 32, "pages": 36, "kv_heads": 32, "hd": 128, "pairs": 15},
        # one sequence's next token, the usual filters
        {"name": "sample_token", "kind": "sample", "rows": 1, "vocab": 32000, "bits": 16, "filters": "k_p"},
        # 64 sequences that ask for different things, 32-bit logits
        {"name": "sample_mixed_64", "kind": "sample", "rows": 64, "vocab": 32000, "bits": 32, "filters": "mixed"},
        # a large vocabulary of odd size, top-p alone
        {"name": "sample_large_48", "kind": "sample", "rows": 48, "vocab": 131071, "bits": 16, "filters": "p"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


def draw(rng):
    kind = rng.choice(("write", "attn", "attn", "attn", "pages", "sample", "sample"))
    most = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        heads, kv_heads = rng.choice(((32, 32), (64, 8), (4, 2), (8, 8), (10, 2), (28, 4), (16, 1), (7, 7)))
        hd = rng.choice((64, 128, 128, 128, 256))
        if kind == "write":
            m = rng.choice((1, _log(rng, 2, 2000)))
            first = _log(rng, 1, 4000) - 1
            case = {"kind": kind, "batch": _log(rng, 1, 64) if m == 1 else _log(rng, 1, 4), "m": m, "heads": heads, "kv_heads": kv_heads, "hd": hd,
                    "first": first, "last": first + rng.randrange(500)}
        elif kind == "attn":
            m = rng.choice((1, 1, _log(rng, 2, 9), _log(rng, 10, 600)))
            first = _log(rng, 1, 30000 if m == 1 else 6000) - 1
            case = {"kind": kind, "batch": _log(rng, 1, 48) if m < 10 else _log(rng, 1, 3), "m": m, "heads": heads, "kv_heads": kv_heads, "hd": hd,
                    "first": first, "last": first + _log(rng, 1, 4000) - 1, "ragged": m > 1 and rng.random() < 0.5}
        elif kind == "pages":
            case = {"kind": kind, "layers": rng.choice((2, 32, 40, 80)), "pages": _log(rng, 8, 64), "kv_heads": kv_heads, "hd": hd, "pairs": 0}
            case["pairs"] = _log(rng, 1, case["pages"] // 2)
            if case["layers"] * case["pages"] * kv_heads * PAGE * (hd + hd // 8) > 380e6:
                continue
        else:
            case = {"kind": kind, "rows": _log(rng, 1, 128), "vocab": _log(rng, 500, 200000), "bits": rng.choice((16, 16, 32)),
                    "filters": rng.choice(("none", "k", "p", "k_p", "min", "mixed"))}
        if _cost(case) <= most and (kind != "attn" or _scores(case) <= 2e8):
            return case


def _scores(case):
    """32-bit scores of the plain form."""
    return case["batch"] * case["heads"] * case["m"] * (case["last"] + case["m"])


def _firsts(case):
    """The position of each sequence's first new row: spread evenly over first .. last."""
    b, lo, hi = case["batch"], case["first"], case["last"]
    return [hi if b == 1 else lo + (hi - lo) * i // (b - 1) for i in range(b)]


def _rows_of(case):
    return [1 + (i * 3) % case["m"] if case.get("ragged") else case["m"] for i in range(case["batch"])]


def _random(shape, gen, device, spread=None):
    x = torch.randn(shape, device=device, generator=gen)
    return x if spread is None else x * spread


def _spread(hd, gen, device):
    """A few dimensions of keys and values are several times larger than the others, as in real caches."""
    s = torch.ones(hd, device=device)
    s[torch.randperm(hd, generator=gen, device=device)[: max(1, hd // 32)]] = 4.0
    return s


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(int(seed))
    s = {"case": dict(case)}
    kind = case["kind"]
    if kind == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a broad body with a tail of likelier tokens
        x = 2.0 * torch.randn(rows, vocab, device=device, generator=gen) + 2.5 * torch.rand(rows, vocab, device=device, generator=gen).pow(40)
        peaks = torch.randint(0, vocab, (rows, 12), device=device, generator=gen)
        x.scatter_add_(1, peaks, 6.0 * torch.rand(rows, 12, device=device, generator=gen))
        s["logits"] = x.half() if case["bits"] == 16 else x
        s["u"] = torch.rand(rows, device=device, generator=gen)
        pick = torch.rand(5, rows, device=device, generator=gen)
        f = case["filters"]
        mixed = f == "mixed"
        s["temperature"] = 0.5 + pick[0]
        s["top_k"] = (1 + 99 * pick[1]).int() if f in ("k", "k_p", "mixed") else torch.zeros(rows, dtype=torch.int32, device=device)
        s["top_p"] = 0.8 + 0.19 * pick[2] if f in ("p", "k_p", "mixed") else torch.ones(rows, device=device)
        s["min_p"] = 0.02 + 0.1 * pick[3] if f in ("min", "mixed") else torch.zeros(rows, device=device)
        if mixed:  # every sequence has some of the filters only, and some are greedy
            s["temperature"][pick[4] < 0.1] = 0.0
            s["top_k"][(pick[4] > 0.3) & (pick[4] < 0.6)] = 0
            s["top_p"][pick[4] > 0.5] = 1.0
            s["min_p"][pick[4] < 0.7] = 0.0
        s["token"] = torch.zeros(rows, dtype=torch.int64, device=device)
        return s
    kvh, hd = case["kv_heads"], case["hd"]
    record = PAGE * (hd + hd // 8)
    if kind == "pages":
        s["pool"] = torch.randint(0, 256, (case["layers"], case["pages"], kvh, record), dtype=torch.uint8, device=device, generator=gen)
        order = torch.randperm(case["pages"], generator=torch.Generator().manual_seed(int(seed))).tolist()
        s["src"], s["dst"] = order[: case["pairs"]], order[case["pairs"]: 2 * case["pairs"]]
        return s
    batch, m, heads = case["batch"], case["m"], case["heads"]
    firsts = _firsts(case)
    width = (max(firsts) + m - 1) // PAGE + 1
    pages = batch * width + 3
    s["pos"] = torch.tensor(firsts, dtype=torch.int64, device=device)
    s["table"] = torch.randperm(pages, device=device, generator=gen)[: batch * width].view(batch, width).int()
    # what no row was written to holds what was there before
    s["pool"] = torch.randint(0, 256, (pages, kvh, record), dtype=torch.uint8, device=device, generator=gen)
    s["q"] = _random((batch, m, heads * hd), gen, device).half()
    if kind == "write":
        s["k"] = _random((batch, m, kvh, hd), gen, device, _spread(hd, gen, device)).half().view(batch, m, kvh * hd)
        s["v"] = _random((batch, m, kvh, hd), gen, device, _spread(hd, gen, device)).half().view(batch, m, kvh * hd)
        inv = 10000.0 ** (-torch.arange(0, hd, 2, device=device, dtype=torch.float64) / hd)
        angle = torch.arange(width * PAGE, device=device, dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_out"] = torch.zeros_like(s["q"])
        s["k_out"] = torch.zeros(batch, m, kvh, hd, device=device)
        s["v_out"] = torch.zeros_like(s["k_out"])
        return s
    s["rows"] = torch.tensor(_rows_of(case), dtype=torch.int32, device=device) if case["ragged"] else None
    s["out"] = torch.zeros_like(s["q"])
    s["scale"] = 1.0 / math.sqrt(hd)
    k_spread, v_spread = _spread(hd, gen, device), _spread(hd, gen, device)
    for b in range(batch):  # the sequence's rows, page by page; what lies behind its last row stays as it was
        n = firsts[b] + _rows_of(case)[b]
        own_pages = s["table"][b, : (n - 1) // PAGE + 1].long()
        old = s["pool"][own_pages]
        new = _record(_random((own_pages.numel(), kvh, PAGE, hd), gen, device, k_spread).half(),
                      _random((own_pages.numel(), kvh, PAGE, hd), gen, device, v_spread).half())
        written = (torch.arange(own_pages.numel() * PAGE, device=device) < n).view(-1, 1, PAGE)
        s["pool"][own_pages] = torch.where(_by_byte(written.expand(-1, kvh, -1), hd), new, old)
    return s


# ---- the format --------------------------------------------------------------------------------------


def _order(groups, device):
    """[64][groups]: which group lies at place g of position p (and, the order being its own inverse, where group g lies)."""
    p = torch.arange(PAGE, device=device)
    f = (p & 3) ^ ((p >> 1) & 2)
    f = f if groups == 4 else f >> 1 if groups == 2 else torch.zeros_like(f)
    return torch.arange(groups, device=device)[None, :] ^ f[:, None]


def _quantise(x):
    """x fp16 [..., hd] -> codes uint8 [..., groups, 64], scale and low fp16 [..., groups]."""
    g = x.float().unflatten(-1, (-1, 64))
    low, high = g.amin(-1), g.amax(-1)
    scale = ((high - low) / 15.0).half()
    inv = torch.where(scale > 0, 1.0 / scale.float(), torch.zeros_like(low))
    codes = ((g - low[..., None]) * inv[..., None]).round().clamp(max=15.0)
    return codes.to(torch.uint8), scale, low.half()


def _value(codes, scale, low):
    return (codes.float() * scale.float()[..., None] + low.float()[..., None]).flatten(-2)


def _record(k, v):
    """k, v fp16 [..., 64, hd] of a page and head -> its record, uint8 [..., 64 * (hd + hd / 8)]."""
    codes, params = [], []
    for x in (k, v):
        c, scale, low = _quantise(x)
        place = _order(c.shape[-2], x.device)[..., None].expand(c.shape)
        c = c.gather(-2, place)
        codes.append((c[..., 0::2] | (c[..., 1::2] << 4)).flatten(-3))
        params.append(torch.stack((scale, low), -1).flatten(-3).contiguous().view(torch.uint8))
    return torch.cat(codes + params, -1)


def _by_byte(written, hd):
    """[..., 64] truth values of the positions -> [..., record] of the bytes."""
    codes, params = written.repeat_interleave(hd // 2, -1), written.repeat_interleave(hd // 16, -1)
    return torch.cat((codes, codes, params, params), -1)


def _values(records, hd):
    """Records [..., 64 * (hd + hd / 8)] -> keys and values in 32 bits, [..., 64, hd]."""
    groups, n = hd // 64, PAGE * hd // 2
    got = []
    for i in range(2):
        c = records[..., i * n:(i + 1) * n].unflatten(-1, (PAGE, groups, 32))
        c = torch.stack((c & 15, c >> 4), -1).flatten(-2)
        c = c.gather(-2, _order(groups, c.device)[..., None].expand(c.shape))
        p = records[..., 2 * n + i * n // 8: 2 * n + (i + 1) * n // 8].contiguous().view(torch.float16).unflatten(-1, (PAGE, groups, 2))
        got.append(_value(c, p[..., 0], p[..., 1]))
    return got


# ---- one pass ----------------------------------------------------------------------------------------


def run(s):
    kind = s["case"]["kind"]
    if own:
        return _own(s, kind)
    return {"write": _plain_write, "attn": _plain_attention, "pages": _plain_pages, "sample": _plain_sample}[kind](s)


def _own(s, kind):
    from shiftaddllm_b200 import decode_ops

    c = s["case"]
    if kind == "write":
        decode_ops.rope_kv4_write(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["pos"], s["table"], s["pool"], s["q_out"], c["heads"], c["kv_heads"], c["hd"])
        decode_ops.read_kv4(s["pool"], s["table"], s["pos"], s["k_out"], s["v_out"], c["kv_heads"], c["hd"])
        return s["q_out"], s["k_out"], s["v_out"]
    if kind == "attn":
        if "workspace" not in s:
            s["workspace"] = decode_ops.attention_kv4_workspace(c["batch"], c["m"], c["heads"], c["kv_heads"], c["hd"], s["q"].device)
        decode_ops.attention_kv4(s["q"], s["pool"], s["table"], s["pos"], s["out"], c["heads"], c["kv_heads"], c["hd"], s["scale"], s["workspace"], s["rows"])
        return s["out"]
    if kind == "pages":
        decode_ops.copy_kv4_pages(s["pool"], s["src"], s["dst"])
        return s["pool"]
    decode_ops.sample_token(s["logits"], s["u"], s["token"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    return s["token"]


def _rotated(x, cos, sin, heads):
    """x fp16 [batch, m, heads * hd] at angles [batch, m, hd / 2]: first half and second half of a head are the pair's numbers."""
    a, b = x.double().unflatten(-1, (heads, 2, -1)).unbind(-2)
    cos, sin = cos.double()[:, :, None, :], sin.double()[:, :, None, :]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).float().half()


def _plain_write(s):
    c = s["case"]
    at = s["pos"][:, None] + torch.arange(c["m"], device=s["pos"].device)
    cos, sin = s["cos"][at], s["sin"][at]
    q = _rotated(s["q"], cos, sin, c["heads"])
    k = _rotated(s["k"], cos, sin, c["kv_heads"])
    return q.flatten(-2), _value(*_quantise(k)), _value(*_quantise(s["v"].unflatten(-1, (c["kv_heads"], c["hd"]))))


def _plain_attention(s):
    c = s["case"]
    batch, m, kvh, hd = c["batch"], c["m"], c["kv_heads"], c["hd"]
    rows = s["rows"] if s["rows"] is not None else torch.full((batch,), m, dtype=torch.int32, device=s["pos"].device)
    k, v = _values(s["pool"][s["table"].long()], hd)                                  # [batch, pages, kv_heads, 64, hd]
    k, v = k.transpose(1, 2).flatten(2, 3), v.transpose(1, 2).flatten(2, 3)           # [batch, kv_heads, T, hd]
    t = torch.arange(k.shape[2], device=k.device)
    written = (t < (s["pos"] + rows)[:, None])[:, None, :, None]
    k, v = torch.where(written, k, torch.zeros((), device=k.device)), torch.where(written, v, torch.zeros((), device=v.device))
    q = s["q"].float().view(batch, m, kvh, -1, hd).permute(0, 2, 3, 1, 4).flatten(2, 3)   # [batch, kv_heads, rep * m, hd]
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(s["scale"])
    last = (s["pos"][:, None] + torch.arange(m, device=k.device)).repeat(1, c["heads"] // kvh)
    score.masked_fill_((t > last[:, :, None])[:, None], float("-inf"))
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.unflatten(2, (-1, m)).permute(0, 3, 1, 2, 4).reshape(batch, m, -1).half()
    valid = (torch.arange(m, device=k.device) < rows[:, None])[..., None]
    return torch.where(valid, o, s["out"])


def _plain_pages(s):
    pool = s["pool"]
    device = pool.device
    pool[:, torch.tensor(s["dst"], device=device)] = pool[:, torch.tensor(s["src"], device=device)]
    return pool


def _plain_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    temperature = s["temperature"].double()[:, None]
    greedy = temperature <= 0
    x, index = x.sort(dim=-1, descending=True, stable=True)               # equal logits: the lower index first
    w = ((x - x[:, :1]) / torch.where(greedy, torch.ones_like(temperature), temperature)).exp()
    rank = torch.arange(vocab, device=x.device)[None, :]
    k = s["top_k"][:, None]
    w = torch.where((k > 0) & (rank >= k), torch.zeros_like(w), w)
    before = w.cumsum(-1) - w
    p = s["top_p"].double()[:, None]
    w = torch.where((p < 1) & (before >= p * w.sum(-1, keepdim=True)) & (rank > 0), torch.zeros_like(w), w)
    w = torch.where(w < s["min_p"].double()[:, None], torch.zeros_like(w), w)
    w = torch.where(greedy, (rank == 0).double(), w)
    w = torch.zeros_like(w).scatter_(1, index, w)                          # back in the vocabulary's order
    total = w.cumsum(-1)
    last = (w > 0).double().mul_(rank).amax(-1).long()                     # the last token that is left
    return torch.minimum((total <= s["u"].double()[:, None] * total[:, -1:]).sum(-1), last)


# ---- what a pass cannot do without -----------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * case["bits"] // 8 + case["rows"] * 28, "flops": 4 * n}
    kvh, hd = case["kv_heads"], case["hd"]
    row = hd + hd // 8          # bytes of a position and head: the codes and parameters of its key and its value
    if kind == "pages":
        return {"bytes": 2 * case["layers"] * case["pairs"] * kvh * PAGE * row, "flops": 0}
    batch, m, heads = case["batch"], case["m"], case["heads"]
    if kind == "write":
        n = batch * m
        moved = n * (2 * heads + 2 * kvh) * hd * 2 + n * hd * 4 + 2 * n * kvh * row + n * 2 * kvh * hd * 4
        return {"bytes": moved, "flops": n * (heads + kvh) * hd * 3 + n * 2 * kvh * hd * 4}
    firsts, rows = _firsts(case), _rows_of(case)
    positions = sum(f + r for f, r in zip(firsts, rows))
    pairs = sum(r * f + r * (r + 1) // 2 for f, r in zip(firsts, rows))
    return {"bytes": positions * kvh * row + 2 * sum(rows) * heads * hd * 2, "flops": 4 * pairs * heads * hd}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "pages":
        return None
    if kind == "sample":
        return _exact_sample(s)
    return _exact_write(s) if kind == "write" else _exact_attention(s)


def _exact_sample(s):
    tokens = []
    per_row = [s[n].cpu().numpy().astype(np.float64) for n in ("u", "temperature", "top_p", "min_p")]
    for x, u, t, p, least, k in zip(s["logits"].cpu().numpy().astype(np.float64), *per_row, s["top_k"].tolist()):
        if t <= 0:
            tokens.append(int(np.argmax(x)))
            continue
        best = np.argsort(-x, kind="stable")[: k if k > 0 else x.size]
        w = np.exp((x[best] - x.max()) / t)
        kept = len(best)
        if p < 1:
            kept = max(1, int(np.count_nonzero(np.cumsum(w) - w < p * w.sum())))
        chosen = sorted((int(i), float(v)) for i, v in zip(best[:kept], w[:kept]) if v >= least)
        goal, have = u * math.fsum(v for _, v in chosen), 0.0
        token = chosen[-1][0]
        for i, v in chosen:
            have += v
            if have > goal:
                token = i
                break
        tokens.append(token)
    return torch.tensor(tokens, dtype=torch.int64)


def _exact_write(s):
    c = s["case"]
    kvh, hd = c["kv_heads"], c["hd"]
    half = hd // 2

    def turned(x, heads):
        x = x.cpu().numpy().astype(np.float64).reshape(c["batch"], c["m"], heads, hd)
        at = s["pos"].cpu().numpy()[:, None] + np.arange(c["m"])
        cos, sin = (s[n].cpu().numpy().astype(np.float64)[at][:, :, None, :] for n in ("cos", "sin"))
        y = np.empty_like(x)
        y[..., :half] = x[..., :half] * cos - x[..., half:] * sin
        y[..., half:] = x[..., half:] * cos + x[..., :half] * sin
        return y.astype(np.float32).astype(np.float16)

    def kept(x):   # the format's own roundings are part of its definition
        g = x.astype(np.float32).reshape(*x.shape[:-1], hd // 64, 64)
        low, high = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
        scale = ((high - low) / np.float32(15)).astype(np.float16).astype(np.float32)
        with np.errstate(divide="ignore"):
            inv = np.where(scale > 0, np.float32(1) / scale, np.float32(0))
        code = np.minimum(np.rint((g - low) * inv), 15)
        return torch.from_numpy((low.astype(np.float64) + scale.astype(np.float64) * code).reshape(x.shape))

    v = s["v"].cpu().numpy().reshape(c["batch"], c["m"], kvh, hd)
    q = turned(s["q"], c["heads"]).astype(np.float64).reshape(c["batch"], c["m"], -1)
    return torch.from_numpy(q), kept(turned(s["k"], kvh)), kept(v)


def _exact_attention(s):
    c = s["case"]
    heads, kvh, hd, m = c["heads"], c["kv_heads"], c["hd"], c["m"]
    groups = hd // 64
    out = torch.zeros(c["batch"], m, heads, hd, dtype=torch.float64, device=s["q"].device)
    place = torch.tensor([[g ^ ({4: f, 2: f >> 1, 1: 0}[groups]) for g in range(groups)] for f in ((p & 3) ^ ((p >> 1) & 2) for p in range(PAGE))])

    def numbers(record, of_values):    # [n, 64 * (hd + hd / 8)] -> [n * 64, hd] in 64 bits
        n = record.shape[0]
        size = 32 * hd
        codes = record[:, of_values * size:(of_values + 1) * size].reshape(n, PAGE, groups, 32)
        start = 2 * size + of_values * (size // 8)
        params = record[:, start:start + size // 8].contiguous().view(torch.float16).double().reshape(n, PAGE, groups, 2)
        got = torch.empty(n, PAGE, groups, 64, dtype=torch.float64, device=record.device)
        where = torch.arange(PAGE)
        for g in range(groups):
            block = codes[:, where.to(record.device), place[:, g].to(record.device)].double()      # [n, 64, 32]
            got[:, :, g, 0::2] = block.remainder(16)
            got[:, :, g, 1::2] = block.div(16).floor()
        return (got * params[..., :1] + params[..., 1:]).reshape(n * PAGE, hd)

    for b, (first, count) in enumerate(zip(_firsts(c), _rows_of(c))):
        total = first + count
        used = s["table"][b, : (total - 1) // PAGE + 1].long()
        q = s["q"][b, :count].double().view(count, heads, hd)
        limit = torch.arange(first, total, device=q.device)
        for h in range(kvh):
            records = s["pool"][used, h]
            k, v = numbers(records, 0)[:total], numbers(records, 1)[:total]
            for j in range(h * (heads // kvh), (h + 1) * (heads // kvh)):
                w = (q[:, j] @ k.T) * s["scale"]
                w = w.masked_fill(torch.arange(total, device=q.device)[None, :] > limit[:, None], -math.inf)
                out[b, :count, j] = torch.softmax(w, -1) @ v
    return out.view(c["batch"], m, -1)
