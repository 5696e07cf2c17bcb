"""64-bit numpy results of the operators that serve several sequences, and the
error bounds that the kernels' roundings give.

A value rounded to fp16 is off by at most 2^-11 of itself (2^-25 below the
normal range), one rounded to fp32 by 2^-24."""
from __future__ import annotations

import numpy as np

H16, H32, SUB16 = 2.0 ** -11, 2.0 ** -24, 2.0 ** -25


def rotated(x, pos, theta):
    """Split-half rotation of [tokens][heads][dim] and its error bound: the
    angle in turns is exact to 2^-25 (fp64 product of an int32 position) and
    rounded to fp32 (half turns: 2^-24), sine and cosine are within 2 ulp, and
    the fp32 product and sum round twice: (pi (2^-24 + 2^-24) + 4 2^-24 + 2 2^-24)
    (|x1| + |x2|) < 2^-20 (|x1| + |x2|), then one rounding to fp16."""
    x = x.astype(np.float64)
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    if theta == 0.0:
        return x, np.zeros_like(x)
    ang = (pos.astype(np.float64)[:, None] * theta ** (-np.arange(half) / half))[:, None]
    c, s = np.cos(ang), np.sin(ang)
    y = np.concatenate([a * c - b * s, a * s + b * c], -1)
    slack = 2.0 ** -20 * np.concatenate([np.abs(a) + np.abs(b)] * 2, -1)
    return y, slack


def stored(payload, scales):
    """The values of a cache's rows [..., dim]."""
    if scales is None:
        return payload.astype(np.float64)
    return payload.astype(np.float64) * np.repeat(scales.astype(np.float64), 64, -1)


def attend(q, k, v, seen, scale, top=1.0):
    """One head: q [rows][dim], k, v [keys][dim] (fp64), seen [rows][keys].
    Returns the result and its bound.  Scores: fp32 sums of dim exact products,
    dim 2^-24 sum |q k| each, and the exponent's argument rounds twice; so a
    weight is off by delta, at most twice that in the quotient.  Weights round
    to fp16 (2^-11, or 2^-25 beside a largest one of 1 to 256); their sum and the sum of
    products round once per key in fp32.  Q8_0: it is a weight times its scale,
    over up to twice the largest scale, that rounds; top is how much larger that
    makes the least step beside a value (2 times largest over least scale)."""
    rows, dim = q.shape
    out, tol = np.zeros((rows, v.shape[1])), np.zeros((rows, v.shape[1]))
    for i in range(rows):
        j = np.nonzero(seen[i])[0]
        if not len(j):
            tol[i] = 0.0
            continue
        s = scale * (k[j] @ q[i])
        w = np.exp(s - s.max())
        w /= w.sum()
        out[i] = w @ v[j]
        mass = w @ np.abs(v[j])
        delta = H32 * (scale * dim * (np.abs(k[j]) @ np.abs(q[i])).max() + 8 * np.abs(s).max() + 8)
        n = len(j)
        tol[i] = mass * (H16 + 4 * delta + 4 * n * H32) + n * top * SUB16 * np.abs(v[j]).max(0) + H16 * np.abs(out[i]) + SUB16
    return out, tol


def packed(q, k, v, qs, ks, scale):
    """[rows][heads][dim] of packed prompts; rows outside every prompt are NaN."""
    rows, heads, dim = q.shape
    kvh = k.shape[1]
    out, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    for s in range(len(qs) - 1):
        nq, nk = qs[s + 1] - qs[s], ks[s + 1] - ks[s]
        if nq <= 0:
            continue
        seen = np.arange(nk)[None, :] <= np.arange(nq)[:, None] + (nk - nq)
        for h in range(heads):
            g = h // (heads // kvh)
            o, t = attend(q[qs[s]:qs[s + 1], h].astype(np.float64), k[ks[s]:ks[s + 1], g].astype(np.float64),
                          v[ks[s]:ks[s + 1], g].astype(np.float64), seen, scale)
            out[qs[s]:qs[s + 1], h], tol[qs[s]:qs[s + 1], h] = o, t
    return out, tol


class Pages:
    """A paged cache on the host; `fill` stands in slots that hold no token."""

    def __init__(self, rng, qtype, kv_heads, dim, page, lengths, absent=(), gap=0, extra=3, stride_extra=1, fill=np.nan):
        self.qtype, self.kv_heads, self.dim, self.page = qtype, kv_heads, dim, page
        count = [-(-n // page) for n in lengths]
        self.n_pages = sum(count) + extra
        self.n_seqs, self.table_stride = len(lengths), max(count + [1]) + stride_extra
        self.page_stride = kv_heads * page * dim + gap
        order = rng.permutation(self.n_pages)
        self.table = np.full((self.n_seqs, self.table_stride), self.n_pages + 7, np.int32)
        at = 0
        for i, c in enumerate(count):
            self.table[i, :c] = order[at:at + c]
            at += c
        for i, p in absent:
            self.table[i, p] = -1
        n = self.n_pages * self.page_stride
        self.scales = [None, None]
        if qtype == 1:
            self.data = [np.full(n, fill, np.float16) for _ in range(2)]
        else:
            self.data = [rng.integers(-127, 128, n, dtype=np.int8) for _ in range(2)]
            self.scales = [np.full(n // 64, fill, np.float16) for _ in range(2)]

    def slot(self, seq, pos, head):
        """Index of a row's first value, or None."""
        p, at = divmod(int(pos), self.page)
        if seq < 0 or seq >= self.n_seqs or pos < 0 or p >= self.table_stride:
            return None
        page = int(self.table[seq, p])
        if not 0 <= page < self.n_pages:
            return None
        return page * self.page_stride + (head * self.page + at) * self.dim

    def put(self, side, seq, pos, head, row, scales=None):
        i = self.slot(seq, pos, head)
        if i is not None:
            self.data[side][i:i + self.dim] = row
            if scales is not None:
                self.scales[side][i // 64:(i + self.dim) // 64] = scales

    def row(self, side, seq, pos, head):
        i = self.slot(seq, pos, head)
        if i is None:
            return None
        s = None if self.scales[side] is None else self.scales[side][i // 64:(i + self.dim) // 64]
        return stored(self.data[side][i:i + self.dim], s)

    def fill(self, rng, lengths):
        for s, n in enumerate(lengths):
            for pos in range(n):
                for h in range(self.kv_heads):
                    for side in range(2):
                        if self.qtype == 1:
                            self.put(side, s, pos, h, rng.standard_normal(self.dim).astype(np.float16))
                        else:
                            self.put(side, s, pos, h, rng.integers(-127, 128, self.dim, dtype=np.int8),
                                     rng.uniform(0.005, 0.02, self.dim // 64).astype(np.float16))

    def upload(self, uocr):
        self.dev = [uocr.DeviceBuffer.of(d) for d in self.data]
        self.dev_s = [None if s is None else uocr.DeviceBuffer.of(s) for s in self.scales]
        self.dev_t = uocr.DeviceBuffer.of(self.table)
        return uocr.CKvPages(qtype=self.qtype, kv_heads=self.kv_heads, head_dim=self.dim, page_tokens=self.page, n_pages=self.n_pages,
                             n_seqs=self.n_seqs, table_stride=self.table_stride, page_stride=self.page_stride, k=self.dev[0].ptr,
                             v=self.dev[1].ptr, k_scales=self.dev_s[0].ptr if self.dev_s[0] else None,
                             v_scales=self.dev_s[1].ptr if self.dev_s[1] else None, page_table=self.dev_t.ptr)

    def download(self):
        """What the device holds now, as a cache of its own."""
        import copy
        other = copy.copy(self)
        other.data = [b.download(d.dtype) for b, d in zip(self.dev, self.data)]
        other.scales = [None if b is None else b.download(np.float16) for b in self.dev_s]
        return other


def paged(pages, lengths, q, scale, top=None):
    """[seqs][heads][dim] of one new token each, and the bound."""
    n, heads, dim = q.shape
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(n):
        cap = pages.table_stride * pages.page
        rows = [p for p in range(min(max(int(lengths[s]), 0), cap)) if pages.slot(s, p, 0) is not None]
        for g in range(pages.kv_heads):
            k = np.array([pages.row(0, s, p, g) for p in rows]).reshape(len(rows), dim)
            v = np.array([pages.row(1, s, p, g) for p in rows]).reshape(len(rows), dim)
            per = heads // pages.kv_heads
            o, t = attend(q[s, g * per:(g + 1) * per].astype(np.float64), k, v, np.ones((per, len(rows)), bool), scale, top or (8.0 if pages.qtype == 3 else 1.0))
            out[s, g * per:(g + 1) * per], tol[s, g * per:(g + 1) * per] = o, t
    return out, tol


def sample(x, t, k, p, m, u):
    """(token, probability, distance of the deciding sums from their limits)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    t, p, m, u = float(t), float(p), float(m), float(u)
    if not np.any(x > -np.inf):
        return 0, 0.0, 1.0
    if not t > 0:
        return int(x.argmax()), 1.0, 1.0
    order = np.argsort(-x, kind="stable")
    d = np.where(x[order] == x[order[0]], 0.0, x[order] - x[order[0]])
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        w = np.where(d == -np.inf, 0.0, np.exp(d / t))
    keep = np.arange(len(x)) < (k if k > 0 else len(x))
    w, order = w[keep], order[keep]
    margin = 1.0
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        keep = before < p * w.sum()
        keep[0] = True
        if p > 0 and len(w) > 1:  # the first is always kept
            margin = min(margin, np.abs(before[1:] - p * w.sum()).min() / w.sum())
        w, order = w[keep], order[keep]
    if m > 0:
        keep = w >= min(m, 1.0)
        near = np.abs(w - min(m, 1.0))
        margin = min(margin, near[near > 0].min() if np.any(near > 0) else 1.0)
        w, order = w[keep], order[keep]
    by = np.argsort(order)
    w, order = w[by], order[by]
    sums = np.cumsum(w)
    u = min(u, float(np.float32(0.99999994))) if u > 0 else 0.0
    at = int(np.argmax(sums > u * sums[-1]))
    if u > 0:
        margin = min(margin, np.abs(sums - u * sums[-1]).min() / sums[-1])
    return int(order[at]), w[at] / sums[-1], margin
