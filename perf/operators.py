"""Performance cases of the batched serving operators: a paged key-value cache, the attentions that read it, and sampling.

The operators serve several sequences at once beside the batch-1 token loop:

  append   rotates the queries and keys of new tokens to their positions (split-half RoPE) and writes keys and values
           into the pages of their sequences (fp16, or Q8_0: int8 with one fp16 scale per 64 values)
  gather   reads cached tokens back as fp16 rows, for a prompt that continues a cached prefix
  paged    attention of one new token of each sequence over its pages
  packed   causal attention of prompts of different lengths packed behind each other, queries grouped over key heads,
           each prompt's queries the last rows of its keys
  sample   a token of each row of logits: temperature, top-k, top-p, min-p, and a given uniform number

``listed()`` holds the fixed cases, ``draw(rng)`` makes further ones over the same ranges.  ``prepare`` makes what a
program has in hand before the call, ``run`` makes one call: in plain torch, or, with ``own``, through the library's
binding.  ``exact`` computes the same outputs in 64 bits, apart from the plain form.
"""
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

VOCAB = 129280
THETA = 10000.0


def listed():
    return [
        # the new tokens of 16 sequences in one decode step: latency of a small call
        {"name": "append-f16-decode-16", "kind": "append", "qtype": "f16", "heads": 10, "kv_heads": 10, "dim": 128, "page": 64,
         "seqs": 16, "low": 1, "high": 1, "mix": 1, "far": 4000},
        # three prompts into Q8 pages, read back as rows
        {"name": "append-q8-prompts-3", "kind": "append", "qtype": "q8", "heads": 10, "kv_heads": 10, "dim": 128, "page": 16,
         "seqs": 3, "low": 932, "high": 2048, "mix": 2, "far": 0},
        # the cached prefix that a second question about one page starts from
        {"name": "gather-f16-932", "kind": "gather", "qtype": "f16", "heads": 10, "kv_heads": 10, "dim": 128, "page": 64,
         "seqs": 1, "low": 932, "high": 932, "mix": 3},
        # prefixes of several long documents out of Q8 pages
        {"name": "gather-q8-long-6", "kind": "gather", "qtype": "q8", "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "seqs": 6, "low": 1500, "high": 8000, "mix": 4},
        # a decode step of one sequence at the headline prompt: latency
        {"name": "paged-f16-1x932", "kind": "paged", "qtype": "f16", "heads": 10, "kv_heads": 10, "dim": 128, "page": 64,
         "seqs": 1, "low": 932, "high": 932, "mix": 5},
        # a decode step of a batch near the headline's mean context, Q8 pages
        {"name": "paged-q8-16x1044", "kind": "paged", "qtype": "q8", "heads": 10, "kv_heads": 10, "dim": 128, "page": 16,
         "seqs": 16, "low": 880, "high": 1208, "mix": 6},
        # a full batch of very different lengths, grouped heads
        {"name": "paged-f16-64-ragged", "kind": "paged", "qtype": "f16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "seqs": 64, "low": 300, "high": 16384, "mix": 7},
        # the prompts of a few crops in one pass
        {"name": "packed-crops-6", "kind": "packed", "heads": 10, "kv_heads": 10, "dim": 128, "seqs": 6, "low": 60, "high": 932,
         "mix": 8, "prefix": 0},
        # long prompts, grouped heads, each continuing a cached prefix
        {"name": "packed-long-4", "kind": "packed", "heads": 32, "kv_heads": 8, "dim": 128, "seqs": 4, "low": 1000, "high": 4001,
         "mix": 9, "prefix": 900},
        # one row of fp16 logits with every filter on: latency
        {"name": "sample-f16-1-all", "kind": "sample", "type": "f16", "rows": 1, "vocab": VOCAB, "filters": "all"},
        # a batch of fp32 logits, the nucleus alone
        {"name": "sample-f32-16-top_p", "kind": "sample", "type": "f32", "rows": 16, "vocab": VOCAB, "filters": "top_p"},
        # a full batch, each request with settings of its own
        {"name": "sample-f16-192-mixed", "kind": "sample", "type": "f16", "rows": 192, "vocab": VOCAB, "filters": "mixed"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["append", "gather", "paged", "paged", "packed", "packed", "sample", "sample"])
    if kind == "sample":
        vocab = _log(rng, 1000, 200000)
        return {"kind": kind, "type": rng.choice(["f16", "f32"]), "rows": _log(rng, 1, max(1, min(192, 192 * VOCAB // vocab))),
                "vocab": vocab, "filters": rng.choice(["all", "top_k", "top_p", "min_p", "none", "mixed"])}
    heads, kv_heads = rng.choice([(10, 10), (32, 8), (16, 2), (12, 12), (20, 5), (26, 1), (9, 3)])
    c = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": rng.choice([128, 128, 64]), "mix": rng.randrange(1 << 20)}
    if kind == "packed":
        high = _log(rng, 2, 4001)
        most = max(1, min(48, 4 * 32 * 4001 ** 2 // (heads * high * high), 16384 // high))
        return {**c, "seqs": _log(rng, 1, most), "low": rng.randint(1, high), "high": high,
                "prefix": rng.choice([0, 0, rng.randint(1, high)]) if high < 2000 else 0}
    c |= {"qtype": rng.choice(["f16", "q8"]), "page": 1 << rng.randint(3, 8)}
    if kind == "paged":
        high = _log(rng, 1, 100000)
        seqs = _log(rng, 1, max(1, min(128, 8 * 64 * 16384 // (kv_heads * high), 32 * 64 * 16384 // (heads * high))))
    else:
        high = _log(rng, 1, 8000)
        seqs = _log(rng, 1, max(1, min(64, 8 * 24000 // (kv_heads * high))))
    c |= {"seqs": seqs, "low": rng.randint(max(1, high // 50), high), "high": high}
    if kind == "append":
        c["far"] = rng.choice([0, 0, 5000, 1000000])
    return c


def _lengths(case):
    """The lengths of a case's sequences: spread over their logarithm, the longest one among them."""
    rng = random.Random(case["mix"])
    n = [_log(rng, case["low"], case["high"]) for _ in range(case["seqs"])]
    n[rng.randrange(len(n))] = case["high"]
    return n


def _starts(n):
    return [0] + list(np.cumsum(n))


# ---- inputs -------------------------------------------------------------------


class _Rand:
    """Seeded values on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda")

    def half(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float16)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda")


def _ints(v):
    return torch.tensor(np.asarray(v, np.int32), device="cuda")


def _cache(case, r, seed, tokens, filled):
    """Pages that hold `tokens[i]` tokens of sequence i, in the order that a running server hands them out, two of them free."""
    kvh, dim, page, n = case["kv_heads"], case["dim"], case["page"], case["seqs"]
    count = [-(-t // page) for t in tokens]
    pages = sum(count) + 2
    order = np.random.default_rng(int(seed)).permutation(pages)
    table = np.full((n, max(count)), -1, np.int32)
    at = 0
    for i, c in enumerate(count):
        table[i, :c] = order[at:at + c]
        at += c
    s = {"table": _ints(table)}
    shape = (pages, kvh, page, dim)
    for x in "kv":
        if case["qtype"] == "f16":
            s[x + "_pages"], s[x + "_scales"] = (r.half(*shape) if filled else torch.zeros(shape, dtype=torch.float16, device="cuda")), None
        elif filled:
            s[x + "_pages"] = torch.randint(-127, 128, shape, generator=r.g, device="cuda", dtype=torch.int8)
            s[x + "_scales"] = ((0.5 + r.uniform(*shape[:3], dim // 64)) / 60).half()
        else:
            s[x + "_pages"] = torch.zeros(shape, dtype=torch.int8, device="cuda")
            s[x + "_scales"] = torch.zeros(*shape[:3], dim // 64, dtype=torch.float16, device="cuda")
    return s


def _zeros(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


def prepare(case, seed):
    kind, r = case["kind"], _Rand(seed)
    if kind == "sample":
        s = _logits(case, r)
    else:
        n, h, kvh, dim = _lengths(case), case["heads"], case["kv_heads"], case["dim"]
        if kind == "packed":
            # a prompt that continues a prefix: the queries are the rows behind it
            keys = [x + case["prefix"] for x in n]
            qs, ks = _starts(n), _starts(keys)
            s = {"q": r.half(qs[-1], h, dim), "k": r.half(ks[-1], kvh, dim), "v": r.half(ks[-1], kvh, dim), "q_starts": _ints(qs),
                 "k_starts": _ints(ks), "out": _zeros(qs[-1], h, dim)}
        elif kind == "paged":
            s = _cache(case, r, seed, n, True)
            s |= {"q": r.half(len(n), h, dim), "lengths": _ints(n), "out": _zeros(len(n), h, dim)}
        else:
            # new tokens stand behind what their sequence holds already; pages before them are absent where that is far off
            far = case.get("far", 0)
            at = [random.Random(case["mix"] + i).randint(far // 2, far) for i in range(len(n))] if far else [0] * len(n)
            skip = [a // case["page"] for a in at]
            s = _cache(case, r, seed, [x + a - b * case["page"] for x, a, b in zip(n, at, skip)], kind == "gather")
            table = s["table"].cpu().numpy()
            wide = np.full((len(n), max(b + table.shape[1] for b in skip)), -1, np.int32)
            for i, b in enumerate(skip):
                wide[i, b:b + table.shape[1]] = table[i]
            s["table"] = _ints(wide)
            s["seq"] = _ints(np.repeat(np.arange(len(n)), n))
            s["pos"] = _ints(np.concatenate([np.arange(a, a + x) for a, x in zip(at, n)]))
            t = sum(n)
            s |= {"k_rows": _zeros(t, kvh, dim), "v_rows": _zeros(t, kvh, dim)}
            if kind == "append":
                qkv = r.half(t, h + 2 * kvh, dim)  # one projection's output: rows of queries, keys and values
                s |= {"q": qkv[:, :h], "k": qkv[:, h:h + kvh], "v": qkv[:, h + kvh:], "q_out": _zeros(t, h, dim), "k_out": _zeros(t, kvh, dim)}
    s["case"] = case
    torch.cuda.synchronize()  # the library's stream does not order itself behind torch's
    return s


def _logits(case, r):
    """Logits of a language model: a broad bulk and a few tokens well above it; settings as requests have them."""
    rows, vocab, f = case["rows"], case["vocab"], case["filters"]
    x = r.normal(rows, vocab) * 2.0
    hot = torch.randint(0, vocab, (rows, 40), generator=r.g, device="cuda")
    x.scatter_add_(1, hot, 6.0 + 5.0 * r.uniform(rows, 40))
    u = r.uniform(rows, 4)
    kind = torch.arange(rows, device="cuda") % 6 if f == "mixed" else None

    def on(name, i):
        if kind is not None:
            return (kind == i) | (kind == 4)
        return torch.full((rows,), f in (name, "all"), device="cuda")

    temperature = 0.4 + 1.1 * u[:, 0]
    if kind is not None:
        temperature = torch.where(kind == 5, torch.zeros_like(temperature), temperature)
    return {"logits": x.half() if case["type"] == "f16" else x, "temperature": temperature,
            "top_k": torch.where(on("top_k", 1), 1 + 200 * u[:, 1], torch.zeros_like(u[:, 1])).int(),
            "top_p": torch.where(on("top_p", 2), 0.5 + 0.49 * u[:, 2], torch.ones_like(u[:, 2])),
            "min_p": torch.where(on("min_p", 3), 0.01 + 0.1 * u[:, 3], torch.zeros_like(u[:, 3])),
            "uniform": r.uniform(rows), "token": _zeros(rows, dtype=torch.int32), "prob": _zeros(rows, dtype=torch.float32)}


# ---- one pass -------------------------------------------------------------------


def run(s):
    return (_run_own if own else _run_plain)(s, s["case"])


_LIBRARY = []


def _library():
    """The library's binding, imported on the first call."""
    if not _LIBRARY:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "unlimitedocr.c_amd"))
        import uocr

        _LIBRARY.append(uocr)
    return _LIBRARY[0]


def _run_own(s, case):
    """The library's calls: operands by address, on the operator stream."""
    uocr, kind = _library(), case["kind"]
    if kind == "sample":
        f32 = case["type"] == "f32"
        uocr.op_sample(uocr.QT_F32 if f32 else uocr.QT_F16, case["rows"], case["vocab"], s["logits"].data_ptr(), case["vocab"],
                       s["temperature"].data_ptr(), s["top_k"].data_ptr(), s["top_p"].data_ptr(), s["min_p"].data_ptr(), s["uniform"].data_ptr(),
                       _kept(uocr, "sample", case["rows"], case["vocab"]), s["token"].data_ptr(), s["prob"].data_ptr())
        return {"token": s["token"], "prob": s["prob"]}
    h, kvh, dim = case["heads"], case["kv_heads"], case["dim"]
    if kind == "packed":
        uocr.op_packed_attention(case["seqs"], s["q_starts"].data_ptr(), s["q"].shape[0], s["k_starts"].data_ptr(), s["k"].shape[0], h, kvh, dim, 0.0,
                                 s["q"].data_ptr(), h * dim, s["k"].data_ptr(), kvh * dim, s["v"].data_ptr(), kvh * dim, s["out"].data_ptr(), h * dim)
        return s["out"]
    pages = s.get("pages")
    if pages is None:  # the descriptor that a program fills when it makes its cache
        pages = s["pages"] = uocr.CKvPages(
            qtype=uocr.QT_F16 if case["qtype"] == "f16" else uocr.QT_Q8, kv_heads=kvh, head_dim=dim, page_tokens=case["page"],
            n_pages=s["k_pages"].shape[0], n_seqs=case["seqs"], table_stride=s["table"].shape[1], page_stride=0,
            k=s["k_pages"].data_ptr(), v=s["v_pages"].data_ptr(), k_scales=_at(s["k_scales"]), v_scales=_at(s["v_scales"]),
            page_table=s["table"].data_ptr())
    if kind == "paged":
        uocr.op_paged_attention(pages, s["lengths"].data_ptr(), h, 0.0, s["q"].data_ptr(), h * dim, _kept(uocr, "paged", case["seqs"], h, kvh, dim),
                                s["out"].data_ptr(), h * dim)
        return s["out"]
    t, seq, pos = s["pos"].shape[0], s["seq"].data_ptr(), s["pos"].data_ptr()
    if kind == "append":
        uocr.op_kv_append(pages, t, seq, pos, h, THETA, s["q"].data_ptr(), s["q"].stride(0), s["q_out"].data_ptr(), h * dim,
                          s["k"].data_ptr(), s["k"].stride(0), s["k_out"].data_ptr(), kvh * dim, s["v"].data_ptr(), s["v"].stride(0))
        if case["qtype"] == "f16":
            return {"q": s["q_out"], "k": s["k_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    uocr.op_kv_gather(pages, t, seq, pos, s["k_rows"].data_ptr(), kvh * dim, s["v_rows"].data_ptr(), kvh * dim)
    if kind == "append":
        return {"q": s["q_out"], "k": s["k_out"], "k_rows": s["k_rows"], "v_rows": s["v_rows"]}
    return {"k_rows": s["k_rows"], "v_rows": s["v_rows"]}


def _at(t):
    return None if t is None else t.data_ptr()


_WORKSPACES = {}


def _kept(uocr, kind, *sizes):
    """The workspace of a kind of call, which a program makes once at its largest size."""
    need = (uocr.sample_workspace_bytes if kind == "sample" else uocr.paged_attention_workspace_bytes)(*sizes)
    if kind not in _WORKSPACES or _WORKSPACES[kind].nbytes < need:
        _WORKSPACES[kind] = uocr.DeviceBuffer(need)
    return _WORKSPACES[kind]


def _run_plain(s, case):
    return {"sample": _plain_sample, "packed": _plain_packed, "paged": _plain_paged, "append": _plain_append, "gather": _plain_gather}[case["kind"]](s, case)


def _softmax(scores, seen):
    """Softmax over the keys that are seen, in 32 bits; a row that sees none has no weight."""
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_packed(s, case):
    """Every prompt in a row of its own, padded to the longest."""
    h, kvh, dim = case["heads"], case["kv_heads"], case["dim"]
    qs, ks = s["q_starts"].long(), s["k_starts"].long()
    nq, nk = qs[1:] - qs[:-1], ks[1:] - ks[:-1]
    i, j = torch.arange(case["high"], device="cuda"), torch.arange(case["high"] + case["prefix"], device="cuda")
    q = s["q"].float()[(qs[:-1, None] + i).clamp_max(s["q"].shape[0] - 1)]
    rows = (ks[:-1, None] + j).clamp_max(s["k"].shape[0] - 1)
    k, v = s["k"].float()[rows], s["v"].float()[rows]
    n = q.shape[0]
    q = q.view(n, len(i), kvh, h // kvh, dim).permute(0, 2, 3, 1, 4).reshape(n, kvh, -1, dim)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(n, kvh, h // kvh, len(i), len(j)).mul_(dim ** -0.5)
    seen = (j < nk[:, None])[:, None, :] & (j <= i[:, None] + (nk - nq)[:, None, None])
    p = _softmax(scores, seen[:, None, None])
    out = torch.matmul(p.view(n, kvh, -1, len(j)), v.permute(0, 2, 1, 3).contiguous())
    out = out.view(n, kvh, h // kvh, len(i), dim).permute(0, 3, 1, 2, 4).reshape(n, len(i), h, dim)
    return out[i < nq[:, None]].half()


def _values(s, x, index):
    """Cached rows at `index` (pages first, then head and token in the page), in 32 bits."""
    rows = s[x + "_pages"][index].float()
    if s[x + "_scales"] is None:
        return rows
    return (rows.unflatten(-1, (-1, 64)) * s[x + "_scales"][index].float().unsqueeze(-1)).flatten(-2)


def _plain_paged(s, case):
    h, kvh, dim = case["heads"], case["kv_heads"], case["dim"]
    table = s["table"].long().clamp_min(0)
    n = table.shape[0]
    k, v = (_values(s, x, table).transpose(1, 2).reshape(n, kvh, -1, dim) for x in "kv")
    q = s["q"].float().view(n, kvh, h // kvh, dim)
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(dim ** -0.5)
    seen = torch.arange(k.shape[2], device="cuda") < s["lengths"][:, None]
    return torch.matmul(_softmax(scores, seen[:, None, None]), v).reshape(n, h, dim).half()


def _slots(s, case):
    """(page, token in the page) of each token, as indices over the heads of a page."""
    pos, page = s["pos"].long(), case["page"]
    return s["table"][s["seq"].long(), pos // page].long()[:, None], torch.arange(case["kv_heads"], device="cuda")[None], (pos % page)[:, None]


def _rotated(x, pos):
    """Split-half rotation in 32 bits; the angles of far positions in 64."""
    half = x.shape[-1] // 2
    angle = pos.double()[:, None] * THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    c, n = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :half].float(), x[..., half:].float()
    return torch.cat([a * c - b * n, a * n + b * c], -1)


def _quantised(x):
    """Q8_0 of groups of 64 values: the payload and its fp16 scales."""
    g = x.unflatten(-1, (-1, 64))
    top = g.abs().amax(-1, keepdim=True)
    scale = torch.where(top == 0, torch.ones_like(top), top / 127)
    return (g / scale).round_().clamp_(-127, 127).to(torch.int8).flatten(-2), scale[..., 0].half()


def _plain_append(s, case):
    at = _slots(s, case)
    q, k = _rotated(s["q"], s["pos"]), _rotated(s["k"], s["pos"])
    if case["qtype"] == "f16":
        s["k_pages"][at], s["v_pages"][at] = k.half(), s["v"]
        return {"q": q.half(), "k": k.half(), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    s["k_pages"][at], s["k_scales"][at] = _quantised(k)
    s["v_pages"][at], s["v_scales"][at] = _quantised(s["v"].float())
    return {"q": q.half(), "k": k.half(), **_plain_gather(s, case)}


def _plain_gather(s, case):
    at = _slots(s, case)
    return {x + "_rows": _values(s, x, at).half() for x in "kv"}


def _plain_sample(s, case):
    """In 64 bits: a weight next to a border decides which token it is."""
    x = s["logits"].double()
    x = torch.where(x.isnan(), -math.inf, x)
    x, order = x.sort(dim=1, descending=True, stable=True)  # equal logits: the lowest id first
    rank = torch.arange(x.shape[1], device="cuda")
    t = s["temperature"].double()[:, None]
    w = torch.exp(torch.where(x == x[:, :1], 0.0, x - x[:, :1]) / torch.where(t > 0, t, 1.0))
    k = s["top_k"].long()[:, None]
    w = w * torch.where(t > 0, (k <= 0) | (rank < k), rank < 1)
    before = torch.cat([torch.zeros_like(t), w.cumsum(1)], 1)
    p = s["top_p"].double()[:, None]
    w = w * ((p >= 1) | (rank == 0) | (before[:, :-1] < p * before[:, -1:])) * (w >= s["min_p"].double()[:, None])
    w = torch.zeros_like(w).scatter_(1, order, w)  # by id again
    sums = w.cumsum(1)
    token = (sums <= s["uniform"].double()[:, None] * sums[:, -1:]).sum(1, keepdim=True)
    return {"token": token[:, 0].int(), "prob": (w.gather(1, token) / sums[:, -1:])[:, 0].float()}


# ---- what a pass cannot do without ----------------------------------------------


def _row_bytes(case, qtype):
    return case["dim"] * 2 if qtype == "f16" else case["dim"] + case["dim"] // 32


def work(case):
    kind = case["kind"]
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["type"] == "f16" else 4) + case["rows"] * 28, "flops": n}
    n, h, kvh, dim = _lengths(case), case["heads"], case["kv_heads"], case["dim"]
    t = sum(n)
    if kind == "packed":
        keys, pairs = t + len(n) * case["prefix"], sum(x * (x + 1) // 2 + x * case["prefix"] for x in n)
        return {"bytes": 2 * dim * (2 * t * h + 2 * keys * kvh), "flops": 4 * dim * h * pairs}
    if kind == "paged":
        return {"bytes": 2 * t * kvh * _row_bytes(case, case["qtype"]) + 4 * len(n) * h * dim, "flops": 4 * dim * h * t}
    pages, rows = 2 * kvh * _row_bytes(case, case["qtype"]), 2 * dim
    if kind == "gather":
        return {"bytes": t * (pages + 2 * kvh * rows), "flops": t * 2 * kvh * dim}
    read_back = pages + 2 * kvh * rows if case["qtype"] == "q8" else 0
    return {"bytes": t * (rows * (2 * h + 3 * kvh) + pages + read_back), "flops": t * dim * 3 * (h + kvh)}


# ---- 64-bit results --------------------------------------------------------------


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "sample":
        return _exact_sample(s, case)
    h, kvh, dim, n = case["heads"], case["kv_heads"], case["dim"], _lengths(case)
    g = h // kvh

    def attend(q, k, v, lead):
        """q [rows][heads][dim] over k, v [keys][kv heads][dim]: row i sees keys up to i + lead."""
        out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
        hide = torch.arange(k.shape[0], device="cuda")[None] > torch.arange(q.shape[0], device="cuda")[:, None] + lead
        for x in range(h):
            a = q[:, x].double() @ k[:, x // g].double().T / math.sqrt(dim)
            out[:, x] = torch.softmax(a.masked_fill(hide, -math.inf), -1) @ v[:, x // g].double()
        return out

    if kind == "packed":
        qs, ks = _starts(n), _starts([x + case["prefix"] for x in n])
        return torch.cat([attend(s["q"][qs[i]:qs[i + 1]], s["k"][ks[i]:ks[i + 1]], s["v"][ks[i]:ks[i + 1]], case["prefix"]) for i in range(len(n))])

    def cached(x, i, tokens):
        """Tokens [0, tokens) of sequence i as 64-bit rows [tokens][kv heads][dim]."""
        t = torch.arange(tokens, device="cuda")
        page = s["table"][i].long()[t // case["page"]]
        rows = s[x + "_pages"][page, :, t % case["page"]].double()
        if s[x + "_scales"] is not None:
            rows = rows * s[x + "_scales"][page, :, t % case["page"]].double().repeat_interleave(64, -1)
        return rows

    if kind == "paged":
        return torch.cat([attend(s["q"][i:i + 1], cached("k", i, n[i]), cached("v", i, n[i]), n[i] - 1) for i in range(len(n))])
    if kind == "gather":
        return {x + "_rows": torch.cat([cached(x, i, n[i]) for i in range(len(n))]) for x in "kv"}

    def turned(x):
        """Each pair as a complex number times exp(i angle)."""
        f = torch.exp(-math.log(THETA) * 2 / dim * torch.arange(dim // 2, device="cuda", dtype=torch.float64))
        z = torch.complex(x[..., :dim // 2].double(), x[..., dim // 2:].double()) * torch.exp(1j * s["pos"].double()[:, None, None] * f)
        return torch.cat([z.real, z.imag], -1)

    q, k, v = turned(s["q"]), turned(s["k"]), s["v"].double()
    if case["qtype"] == "q8":
        def stored(x):
            x = x.reshape(-1, 64)
            top = x.abs().max(1, keepdim=True).values / 127
            return (torch.round(x / top.clamp_min(1e-300)) * top.half().double()).view(v.shape)

        return {"q": q, "k": k, "k_rows": stored(k), "v_rows": stored(v)}
    pages = {x: s[x + "_pages"].double() for x in "kv"}
    seq, pos = s["seq"].cpu().numpy(), s["pos"].cpu().numpy()
    page = torch.from_numpy(s["table"].cpu().numpy()[seq, pos // case["page"]]).long().cuda()
    slot = torch.from_numpy(pos % case["page"]).long().cuda()
    for x, rows in (("k", k), ("v", v)):
        pages[x].transpose(1, 2)[page, slot] = rows
    return {"q": q, "k": k, "k_pages": pages["k"], "v_pages": pages["v"]}


def _exact_sample(s, case):
    """Row by row: the kept set from sorted arrays, then the first id whose running sum passes the uniform number."""
    a = {x: s[x].double().cpu().numpy() for x in ("logits", "temperature", "top_k", "top_p", "min_p", "uniform")}
    token, prob = [], []
    for x, t, k, p, m, u in zip(a["logits"], a["temperature"], a["top_k"], a["top_p"], a["min_p"], a["uniform"]):
        if not t > 0:
            token.append(int(x.argmax()))
            prob.append(1.0)
            continue
        order = np.argsort(-x, kind="stable")
        if k > 0:
            order = order[:int(k)]
        w = np.exp((x[order] - x[order[0]]) / t)
        if p < 1:
            order = order[:max(1, int(np.searchsorted(np.cumsum(w), p * w.sum())) + 1)]
        w = w[:len(order)]
        ids = np.sort(order[w >= m])
        w = np.exp((x[ids] - x.max()) / t)
        at = min(int(np.searchsorted(np.cumsum(w), u * w.sum(), side="right")), len(ids) - 1)
        token.append(int(ids[at]))
        prob.append(w[at] / w.sum())
    return {"token": torch.tensor(token, dtype=torch.int32), "prob": torch.tensor(prob, dtype=torch.float64)}
