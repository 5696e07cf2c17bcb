"""The operators that serve several sequences against 64-bit results
(serve_reference.py, where the bounds are derived)."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import convert_q8, rand_f16
from serve_reference import H16, H32, SUB16, Pages, attend, packed, paged, rotated, sample, stored

pytestmark = pytest.mark.gpu


def dev(uocr, a):
    return None if a is None else uocr.DeviceBuffer.of(np.ascontiguousarray(a))


def near(got, ref, tol, what):
    got = got.astype(np.float64)
    if ref.size == 0:
        return
    with np.errstate(invalid="ignore"):
        ok = np.where(np.isnan(ref), np.isnan(got), np.where(np.isinf(ref), got == ref, np.abs(got - ref) <= tol))
    at = np.unravel_index(int(np.argmin(ok)), ok.shape)
    assert ok.all(), f"{what}: {(~ok).sum()} of {ok.size} off, first {at}: {got[at]} for {ref[at]} (bound {np.broadcast_to(tol, ok.shape)[at]})"


# ---- append and gather -------------------------------------------------------------

def append_case(uocr, rng, qtype, heads, kvh, dim, page, seqs, pos, n_seqs, theta=1e4, q_gap=0, in_place=False, k_out=True, gap=0, shift=0, absent=()):
    """Appends tokens (seqs[i], pos[i]); checks rows, pages and what has to stay."""
    t = len(pos)
    lengths = [max([p + 1 for s, p in zip(seqs, pos) if s == i] + [1]) for i in range(n_seqs)]
    c = Pages(rng, qtype, kvh, dim, page, lengths, absent=absent, gap=gap)
    desc = c.upload(uocr)
    stride = (heads + 2 * kvh) * dim + q_gap
    rows = rand_f16(rng, t * stride + shift)
    d = dev(uocr, rows)
    view = rows[shift:].reshape(t, stride)
    q, k, v = (view[:, a:b].reshape(t, -1, dim) for a, b in ((0, heads * dim), (heads * dim, (heads + kvh) * dim), ((heads + kvh) * dim, (heads + 2 * kvh) * dim)))
    at = d.ptr + 2 * shift
    q_out, k_rows = dev(uocr, np.full((t, heads, dim), 7, np.float16)), dev(uocr, np.full((t, kvh, dim), 7, np.float16))
    plain = seqs == list(range(t))
    uocr.op_kv_append(desc, t, None if plain else dev(uocr, np.array(seqs, np.int32)), dev(uocr, np.array(pos, np.int32)), heads if heads else 0, theta,
                      at if heads else None, stride, (at if in_place else q_out) if heads else None, stride if in_place else heads * dim, at + 2 * heads * dim,
                      stride, (at + 2 * heads * dim if in_place else k_rows) if k_out else None, stride if in_place else kvh * dim,
                      at + 2 * (heads + kvh) * dim, stride)
    uocr.sync()
    skip = np.array([s < 0 or s >= n_seqs or p < 0 or p // page >= c.table_stride for s, p in zip(seqs, pos)])
    yq, sq = rotated(q, np.array(pos), theta)
    yk, sk = rotated(k, np.array(pos), theta)
    if in_place:
        got = d.download(np.float16)[shift:].reshape(t, stride)
        gq, gk = got[:, :heads * dim].reshape(t, heads, dim), got[:, heads * dim:(heads + kvh) * dim].reshape(t, kvh, dim)
        assert np.array_equal(got[:, (heads + kvh) * dim:], view[:, (heads + kvh) * dim:]), "values and gaps"
        old_q, old_k = q, k
    else:
        gq, gk = q_out.download(np.float16).reshape(t, heads, dim), k_rows.download(np.float16).reshape(t, kvh, dim)
        old_q, old_k = np.full_like(gq, 7), np.full_like(gk, 7)
    near(gq[~skip], yq[~skip], H16 * np.abs(yq[~skip]) + SUB16 + sq[~skip], "q")
    assert np.array_equal(gq[skip], old_q[skip])
    if k_out:
        near(gk[~skip], yk[~skip], H16 * np.abs(yk[~skip]) + SUB16 + sk[~skip], "k")
        assert np.array_equal(gk[skip], old_k[skip])
    elif not in_place:
        assert np.all(gk == 7)
    after = c.download()
    touched = [np.zeros(x.shape, bool) for x in c.data]
    for i in np.nonzero(~skip)[0]:
        for h in range(kvh):
            a = c.slot(seqs[i], pos[i], h)
            if a is None:
                continue
            for side, y, slack in ((0, yk[i, h], sk[i, h]), (1, v[i, h].astype(np.float64), 0.0)):
                touched[side][a:a + dim] = True
                got = after.data[side][a:a + dim]
                if qtype == 1:
                    near(got, y, (H16 * np.abs(y) + SUB16 + slack) if side == 0 else 0.0, "page")
                    continue
                sc = after.scales[side][a // 64:(a + dim) // 64]
                if side == 1 or theta == 0.0:  # nothing is computed before the quantiser: its bytes
                    w, s = convert_q8(y.astype(np.float32).reshape(1, -1))
                    assert np.array_equal(got, w[0]) and np.array_equal(sc, s[0])
                    continue
                # half a step, the rotation's error, the scale's rounding of up to 127 steps
                step = np.repeat(np.abs(y).reshape(-1, 64).max(1) / 127, 64)
                near(stored(got, sc), y, 0.5 * step * (1 + 2.0 ** -20) + slack + 127 * (H16 * step + SUB16), "page")
    for side in range(2):
        same = after.data[side].view(np.uint16 if qtype == 1 else np.int8) == c.data[side].view(np.uint16 if qtype == 1 else np.int8)
        assert same[~touched[side]].all(), "slots of no new token"
    return c, after, desc


@pytest.mark.parametrize("qtype", [1, 3])
@pytest.mark.parametrize("heads,kvh,dim,page", [(10, 10, 128, 64), (4, 1, 64, 16), (6, 2, 64, 1), (32, 8, 128, 32), (9, 3, 128, 8), (0, 3, 64, 4)])
def test_append_rows_and_pages(gpu, qtype, heads, kvh, dim, page):
    rng = np.random.default_rng(heads + dim + qtype)
    seqs = [0] * 37 + [1] + [2] * 5
    pos = list(range(37)) + [90] + list(range(60, 65))
    append_case(gpu, rng, qtype, heads, kvh, dim, page, seqs, pos, 3)


@pytest.mark.parametrize("qtype", [1, 3])
def test_append_in_place_padding_and_absent_pages(gpu, qtype):
    """Padding rows, sequences and positions out of range and absent pages; rows at odd places; pages with gaps."""
    rng = np.random.default_rng(11)
    seqs = [0, -1, 1, 5, 1, 0, 2, 0]
    pos = [0, 3, 17, 2, -1, 5000, 20, 33]
    for in_place in (False, True):
        append_case(gpu, rng, qtype, 5, 5, 64, 16, seqs, pos, 3, in_place=in_place, q_gap=7, gap=128, shift=1, absent=[(2, 1), (0, 2)])
    append_case(gpu, rng, qtype, 2, 2, 128, 16, [0, 1, 2, 3], [5, 0, 9, 31], 4, k_out=False)


@pytest.mark.parametrize("theta", [0.0, 1.0, 10000.0, 5.0e5])
def test_append_far_positions(gpu, theta):
    rng = np.random.default_rng(5)
    far = [0, 1, 2047, 65535, 1000003, 16777217, 100000007, 2000000011]
    t = len(far)
    c = Pages(rng, 1, 2, 128, 65536, [4], stride_extra=0)
    c.table = np.full((1, 32000), -1, np.int32)
    c.table_stride = 32000
    desc = c.upload(gpu)
    q, k = rand_f16(rng, (t, 3, 128)), rand_f16(rng, (t, 2, 128))
    dq, dk, oq, ok = dev(gpu, q), dev(gpu, k), gpu.DeviceBuffer(q.nbytes), gpu.DeviceBuffer(k.nbytes)
    gpu.op_kv_append(desc, t, dev(gpu, np.zeros(t, np.int32)), dev(gpu, np.array(far, np.int32)), 3, theta, dq, 384, oq, 384, dk, 256, ok, 256, dk, 256)
    gpu.sync()
    for got, x in ((oq, q), (ok, k)):
        y, slack = rotated(x, np.array(far), theta)
        near(got.download(np.float16).reshape(x.shape), y, H16 * np.abs(y) + SUB16 + slack, "rotation")


def test_append_q8_special_groups(gpu):
    """Zero groups keep scale 1; a group with inf or NaN gets a NaN scale, its neighbours stay."""
    rng = np.random.default_rng(2)
    c = Pages(rng, 3, 1, 128, 8, [4])
    desc = c.upload(gpu)
    x = rand_f16(rng, (4, 1, 128))
    x[0, 0, :64] = 0
    x[1, 0, 3] = np.inf
    x[2, 0, 100] = np.nan
    x[3] = 65504
    d = dev(gpu, x)
    gpu.op_kv_append(desc, 4, dev(gpu, np.zeros(4, np.int32)), dev(gpu, np.arange(4, dtype=np.int32)), 0, 0.0, None, 0, None, 0, d, 128, None, 0, d, 128)
    gpu.sync()
    after = c.download()
    for side in range(2):
        s = np.array([after.scales[side][after.slot(0, i, 0) // 64:][:2] for i in range(4)])
        assert s[0, 0] == 1 and np.isnan(s[1, 0]) and np.isnan(s[2, 1]) and np.isfinite(s[[0, 1, 2], [1, 1, 0]]).all()
        assert np.array_equal(after.data[side][after.slot(0, 0, 0):][:64], np.zeros(64, np.int8))
        assert np.all(after.data[side][after.slot(0, 3, 0):][:128] == 127)


@pytest.mark.parametrize("qtype", [1, 3])
@pytest.mark.parametrize("kvh,dim,page", [(10, 128, 64), (3, 64, 16), (1, 64, 1), (8, 128, 8)])
def test_gather(gpu, qtype, kvh, dim, page):
    rng = np.random.default_rng(kvh + dim)
    lengths = [70, 1, 0, 33]
    c = Pages(rng, qtype, kvh, dim, page, lengths, gap=dim, absent=[(3, 0)])
    c.fill(rng, lengths)
    desc = c.upload(gpu)
    where = [(s, p) for s, n in enumerate(lengths) for p in range(n)] + [(-1, 0), (9, 1), (0, -4), (1, 10 ** 6), (0, 5), (0, 5)]
    rng.shuffle(where)
    seqs, pos = (np.array(x, np.int32) for x in zip(*where))
    ref = np.zeros((2, len(where), kvh, dim))
    for i, (s, p) in enumerate(where):
        for h in range(kvh):
            for side in range(2):
                row = c.row(side, s, p, h)
                ref[side, i, h] = 0 if row is None else row
    ref = ref.astype(np.float16)
    ds, dp = dev(gpu, seqs), dev(gpu, pos)
    for sides, stride, shift in (((0, 1), kvh * dim, 0), ((0,), kvh * dim + 3, 1), ((1,), kvh * dim + 8, 0)):
        out = [dev(gpu, np.full(len(where) * stride + shift, 7, np.float16)) if i in sides else None for i in range(2)]
        at = [None if o is None else o.ptr + 2 * shift for o in out]
        gpu.op_kv_gather(desc, len(where), ds, dp, at[0], stride, at[1], stride)
        gpu.sync()
        for i in sides:
            got = out[i].download(np.float16)
            assert np.all(got[:shift] == 7)
            got = got[shift:].reshape(-1, stride)
            assert np.array_equal(got[:, :kvh * dim].reshape(-1, kvh, dim), ref[i])
            assert np.all(got[:, kvh * dim:] == 7)
    # token i of sequence i
    out = gpu.DeviceBuffer(2 * 4 * kvh * dim)
    gpu.op_kv_gather(desc, 4, None, dev(gpu, np.array([69, 0, 0, 20], np.int32)), out, kvh * dim, None, 0)
    gpu.sync()
    rows = [c.row(0, s, p, h) for s, p in enumerate([69, 0, 0, 20]) for h in range(kvh)]
    want = np.array([np.zeros(dim) if r is None else r for r in rows]).astype(np.float16)
    assert np.array_equal(out.download(np.float16).reshape(-1, dim), want)


# ---- attention of one token ----------------------------------------------------------

def paged_case(uocr, rng, qtype, heads, kvh, dim, page, lengths, scale=0.0, gap=0, absent=(), q_gap=0, shift=0, said=None, q=None, change=None, ws=None, top=None):
    c = Pages(rng, qtype, kvh, dim, page, lengths, gap=gap, absent=absent)
    c.fill(rng, lengths)
    if change:
        change(c)
    desc = c.upload(uocr)
    n = len(lengths)
    stride = heads * dim + q_gap
    said = lengths if said is None else said
    q = rand_f16(rng, (n, heads, dim)) if q is None else q
    rows = np.full((n, stride), 7, np.float16)
    rows[:, :heads * dim] = q.reshape(n, -1)
    dq = dev(uocr, np.concatenate([np.zeros(shift, np.float16), rows.reshape(-1)]))
    out = dev(uocr, np.full(n * stride + shift, 9, np.float16))
    ws = ws or uocr.DeviceBuffer(uocr.paged_attention_workspace_bytes(n, heads, kvh, dim))
    dl = dev(uocr, np.array(said, np.int32))
    uocr.op_paged_attention(desc, dl, heads, scale, dq.ptr + 2 * shift, stride, ws, out.ptr + 2 * shift, stride)
    uocr.sync()
    got = out.download(np.float16)
    assert np.all(got[:shift] == 9)
    got = got[shift:].reshape(n, stride)
    assert np.all(got[:, heads * dim:] == 9)
    got = got[:, :heads * dim].reshape(n, heads, dim)
    ref, tol = paged(c, said, q, scale or dim ** -0.5, top)
    near(got, ref, tol, "paged")
    return got


@pytest.mark.parametrize("qtype", [1, 3])
@pytest.mark.parametrize("heads,kvh,dim", [(10, 10, 128), (8, 2, 128), (4, 4, 64), (24, 1, 64), (5, 1, 128), (34, 2, 64)])
@pytest.mark.parametrize("page", [1, 16, 64])
def test_paged_attention(gpu, qtype, heads, kvh, dim, page):
    rng = np.random.default_rng(heads * page + dim)
    paged_case(gpu, rng, qtype, heads, kvh, dim, page, [1, 131, 0, 17, 300], gap=dim, q_gap=3, shift=1)


@pytest.mark.parametrize("qtype", [1, 3])
@pytest.mark.parametrize("lengths", [[127], [128], [129], [2500], [1000, 3, 257, 511, 1, 64, 0, 640, 33, 31, 32], [5] * 300], ids=lambda v: f"{len(v)}x{max(v)}")
def test_paged_attention_lengths(gpu, qtype, lengths):
    rng = np.random.default_rng(len(lengths))
    paged_case(gpu, rng, qtype, 2, 1, 128, 32, lengths)


def test_paged_attention_more_tiles_than_blocks(gpu):
    """Sets that span blocks, blocks that span sets, both at once."""
    rng = np.random.default_rng(77)
    paged_case(gpu, rng, 1, 8, 8, 64, 64, [4000, 1, 9000, 130, 0, 2600, 700], scale=0.3)


def test_paged_attention_absent_pages_and_bad_lengths(gpu):
    rng = np.random.default_rng(8)
    lengths = [100, 64, 40, 48, 16]
    for qtype in (1, 3):
        paged_case(gpu, rng, qtype, 4, 2, 64, 16, lengths, absent=[(0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (1, 3), (2, 2)],
                   said=[100, 64, 33, -5, 2 ** 31 - 1])


def test_paged_attention_values_that_are_not_finite(gpu):
    """Where no token is, nothing matters (Pages fills it with NaN); a token's own NaN or inf goes through."""
    rng = np.random.default_rng(9)

    def change(c):
        a = c.slot(1, 20, 0)
        c.data[1][a + 3] = np.inf
        c.data[1][a + 4] = -np.inf
        c.data[1][a + 5] = np.nan
        c.data[1][c.slot(1, 22, 0) + 4] = np.inf
        c.data[0][c.slot(2, 7, 0) + 1] = np.nan
        for p in range(40):  # a key side that is all NaN
            c.data[0][c.slot(3, p, 0)] = np.nan

    with np.errstate(invalid="ignore"):
        paged_case(gpu, rng, 1, 2, 1, 64, 16, [40, 41, 42, 40], change=change)


def test_paged_attention_far_scores(gpu):
    """Scores of thousands: one key takes all, or all are equal."""
    rng = np.random.default_rng(10)
    q = np.full((2, 2, 128), 30, np.float16)

    def change(c):
        for p in range(300):
            for h in range(1):
                c.data[0][c.slot(0, p, h):][:128] = -20 if p != 211 else 20
                c.data[0][c.slot(1, p, h):][:128] = 25

    paged_case(gpu, rng, 1, 2, 1, 128, 32, [300, 300], scale=1.0, q=q, change=change)


def test_paged_attention_one_workspace_for_all_sizes(gpu):
    """Calls of different heads, dims and batches take turns on one workspace."""
    rng = np.random.default_rng(14)
    size = max(gpu.paged_attention_workspace_bytes(9, *h) for h in ((10, 10, 128), (32, 8, 64), (32, 1, 128)))
    ws = gpu.DeviceBuffer(size)
    for heads, kvh, dim, lengths in ((10, 10, 128, [932]), (32, 1, 128, [900, 2000]), (32, 8, 64, [300, 700, 1, 4000]), (4, 4, 128, [600] * 9)) * 2:
        paged_case(gpu, rng, 1, heads, kvh, dim, 16, lengths, ws=ws)


def test_paged_attention_q8_scales_far_apart(gpu):
    """Scales that grow along the cache, by powers of two and more."""
    rng = np.random.default_rng(15)

    def change(c):
        for p in range(400):
            for h in range(2):
                a = c.slot(0, p, h)
                c.scales[1][a // 64:a // 64 + 2] = np.array([0.001 * 1.03 ** p, 2.0 ** (p // 40 - 12)], np.float16)

    paged_case(gpu, rng, 3, 4, 2, 128, 16, [400], change=change, top=2.0 ** 18)


def test_paged_attention_in_place_and_repeated(gpu):
    """out may be q; the same bits every time from one workspace, whose counters are left at zero."""
    rng = np.random.default_rng(12)
    lengths = [700, 90, 1500]
    c = Pages(rng, 1, 2, 128, 16, lengths)
    c.fill(rng, lengths)
    desc = c.upload(gpu)
    q = rand_f16(rng, (3, 4, 128))
    n = gpu.paged_attention_workspace_bytes(3, 4, 2, 128)
    ws = gpu.DeviceBuffer(n)
    dl, out = dev(gpu, np.array(lengths, np.int32)), gpu.DeviceBuffer(q.nbytes)
    dq = dev(gpu, q)
    gpu.op_paged_attention(desc, dl, 4, 0.0, dq, 512, ws, out, 512)
    gpu.op_paged_attention(desc, dl, 4, 0.0, dq, 512, ws, dq, 512)
    gpu.sync()
    first = out.download(np.uint16)
    assert np.array_equal(first, dq.download(np.uint16))
    ref, tol = paged(c, lengths, q, 128 ** -0.5)
    near(first.view(np.float16).reshape(q.shape), ref, tol, "paged")


def test_paged_attention_largest_pages(gpu):
    """Pages of 65,536 tokens, the second one hardly begun."""
    rng = np.random.default_rng(16)
    for qtype, lengths in ((1, [65541, 3]), (3, [65537])):
        paged_case(gpu, rng, qtype, 2, 1, 64, 65536, lengths)


@pytest.mark.parametrize("qtype", [1, 3])
def test_offsets_past_32_bits(gpu, qtype):
    """Pages 2^31 values apart, rows of keys 2^22 - 64: appended, read back, read by both attentions."""
    rng = np.random.default_rng(17)
    heads, kvh, dim, page, n, far = 2, 1, 64, 512, 1100, 2 ** 31
    size = 2 if qtype == 1 else 1
    pages = gpu.DeviceBuffer((2 * far + 2 * page * dim) * size)  # v's pages stand behind k's
    scales = gpu.DeviceBuffer((2 * far + 2 * page * dim) // 64 * 2) if qtype == 3 else None
    table = dev(gpu, np.array([[2, 0, 1]], np.int32))
    desc = gpu.CKvPages(qtype=qtype, kv_heads=kvh, head_dim=dim, page_tokens=page, n_pages=3, n_seqs=1, table_stride=3, page_stride=far, k=pages.ptr,
                        v=pages.ptr + page * dim * size, k_scales=scales.ptr if scales else None, v_scales=scales.ptr + page * dim // 64 * 2 if scales else None,
                        page_table=table.ptr)
    rows = rand_f16(rng, (3, n, 1, dim))
    q, k, v = (dev(gpu, x) for x in rows)
    seqs, pos = dev(gpu, np.zeros(n, np.int32)), dev(gpu, np.arange(n, dtype=np.int32))
    gpu.op_kv_append(desc, n, seqs, pos, 0, 0.0, None, 0, None, 0, k, dim, None, 0, v, dim)
    near_k, near_v = gpu.DeviceBuffer(2 * n * dim), gpu.DeviceBuffer(2 * n * dim)
    gpu.op_kv_gather(desc, n, seqs, pos, near_k, dim, near_v, dim)
    gpu.sync()
    kk, vv = (b.download(np.float16).reshape(n, 1, dim) for b in (near_k, near_v))
    held = [x.astype(np.float64).reshape(n, dim) for x in rows[1:]]
    if qtype == 3:
        for i, (q8, sc) in enumerate(convert_q8(x.astype(np.float32).reshape(n, dim)) for x in rows[1:]):
            held[i] = q8.astype(np.float64) * sc.astype(np.float64)
    for got, want in zip((kk, vv), held):
        assert np.array_equal(got.reshape(n, dim), want.astype(np.float16))
    qq = rows[0, :2].reshape(1, 2, dim)
    out, ws = gpu.DeviceBuffer(2 * 2 * dim), gpu.DeviceBuffer(gpu.paged_attention_workspace_bytes(1, heads, kvh, dim))
    gpu.op_paged_attention(desc, dev(gpu, np.array([n], np.int32)), heads, 0.0, dev(gpu, qq), heads * dim, ws, out, heads * dim)
    stride = 2 ** 22 - 64
    if qtype == 1:  # 9 GB of rows: keys and values beside each other
        wide = gpu.DeviceBuffer((n * stride) * 2)
        gpu.op_kv_gather(desc, n, seqs, pos, wide, stride, wide.ptr + 2 * dim, stride)
        packed_out = gpu.DeviceBuffer(2 * n * dim)
        gpu.op_packed_attention(1, dev(gpu, np.array([0, n], np.int32)), n, None, n, 1, 1, dim, 0.0, q, dim, wide, stride, wide.ptr + 2 * dim, stride,
                                packed_out, dim)
        gpu.sync()
        ref, tol = packed(rows[0], kk, vv, [0, n], [0, n], dim ** -0.5)
        near(packed_out.download(np.float16).reshape(n, 1, dim), ref, tol, "packed")
    gpu.sync()
    ref, tol = attend(qq[0].astype(np.float64), held[0], held[1], np.ones((2, n), bool), dim ** -0.5, 8.0 if qtype == 3 else 1.0)
    near(out.download(np.float16).reshape(2, dim), ref, tol, "paged")


# ---- packed prompts --------------------------------------------------------------------

def packed_case(uocr, rng, heads, kvh, dim, nq, nk=None, scale=0.0, lead_rows=0, tail_rows=0, gaps=(0, 0, 0, 0), shift=0, change=None):
    qs = lead_rows + np.concatenate([[0], np.cumsum(nq)])
    ks = qs if nk is None else np.concatenate([[0], np.cumsum(nk)])
    tq = int(qs[-1]) + tail_rows
    tk = tq if nk is None else int(ks[-1]) + 2
    q, k, v = rand_f16(rng, (tq, heads, dim)), rand_f16(rng, (tk, kvh, dim)), rand_f16(rng, (tk, kvh, dim))
    if change:
        change(q, k, v)
    bufs, ptrs, strides = [], [], []
    for x, gap in ((q, gaps[0]), (k, gaps[1]), (v, gaps[2]), (np.full_like(q, 9), gaps[3])):
        stride = x.shape[1] * dim + gap
        rows = np.full((x.shape[0], stride), 9, np.float16)
        rows[:, :x.shape[1] * dim] = x.reshape(x.shape[0], -1)
        bufs.append(dev(uocr, np.concatenate([np.zeros(shift, np.float16), rows.reshape(-1)])))
        ptrs.append(bufs[-1].ptr + 2 * shift)
        strides.append(stride)
    dqs, dks = dev(uocr, qs.astype(np.int32)), None if nk is None else dev(uocr, ks.astype(np.int32))
    uocr.op_packed_attention(len(nq), dqs, tq, dks, tk, heads, kvh, dim, scale, ptrs[0], strides[0], ptrs[1], strides[1], ptrs[2], strides[2],
                             ptrs[3], strides[3])
    uocr.sync()
    got = bufs[3].download(np.float16)[shift:].reshape(tq, strides[3])
    assert np.all(got[:, heads * dim:] == 9)
    got = got[:, :heads * dim].reshape(tq, heads, dim)
    with np.errstate(invalid="ignore"):
        ref, tol = packed(q, k, v, qs, ks, scale or dim ** -0.5)
    outside = np.ones(tq, bool)
    outside[qs[0]:qs[-1]] = False
    assert np.all(got[outside] == 9), "rows outside every prompt"
    near(got[~outside], ref[~outside], tol[~outside], "packed")
    return got


@pytest.mark.parametrize("heads,kvh,dim", [(10, 10, 128), (4, 2, 128), (8, 1, 64), (3, 3, 64), (9, 3, 128)])
def test_packed_attention(gpu, heads, kvh, dim):
    rng = np.random.default_rng(heads + dim)
    packed_case(gpu, rng, heads, kvh, dim, [1, 129, 0, 33, 64, 200, 2])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nq,nk", [([5, 1, 40], [70, 300, 40]), ([1], [513]), ([64, 3, 7], [0, 3, 5]), ([130], [129]), ([2, 0, 31], [1, 9, 95])], ids=str)
def test_packed_attention_prefixes(gpu, dim, nq, nk):
    """Queries behind a cached prefix; more queries than keys (the first rows see nothing)."""
    rng = np.random.default_rng(dim + len(nq))
    packed_case(gpu, rng, 4, 2, dim, nq, nk)


@pytest.mark.parametrize("dim", [64, 128])
def test_packed_attention_strides(gpu, dim):
    """Rows off 16-byte boundaries, gaps between them, rows before the first and behind the last prompt."""
    rng = np.random.default_rng(dim)
    packed_case(gpu, rng, 4, 2, dim, [70, 90], lead_rows=5, tail_rows=9, gaps=(3, 1, 5, 7), shift=1, scale=0.2)
    packed_case(gpu, rng, 4, 2, dim, [70, 90], lead_rows=0, tail_rows=3, gaps=(8, 16, 24, 8))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [31, 32, 63, 64, 65, 127, 128, 257, 700])
def test_packed_attention_lengths(gpu, dim, n):
    rng = np.random.default_rng(n)
    packed_case(gpu, rng, 1, 1, dim, [n, 1])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,nq,nk", [(24, [300, 1000], None), (12, [700, 1, 650], [700, 900, 651]), (40, [90] * 12, None), (16, [260, 129, 511, 400], None)],
                         ids=["24x2", "12x3", "40x12", "16x4"])
def test_packed_attention_tile_choices(gpu, dim, heads, nq, nk):
    """Few long and many short prompts: every way of sharing out tiles; strided rows too."""
    rng = np.random.default_rng(heads)
    packed_case(gpu, rng, heads, 4, dim, nq, nk)
    packed_case(gpu, rng, heads, 4, dim, nq, nk, gaps=(1, 3, 3, 1), shift=1)


def test_packed_attention_many_short(gpu):
    rng = np.random.default_rng(3)
    packed_case(gpu, rng, 2, 1, 64, list(rng.integers(0, 6, 700)))


@pytest.mark.parametrize("heads,n", [(2, 150), (2, 400), (20, 700), (40, 400), (90, 400)])
@pytest.mark.parametrize("dim", [64, 128])
def test_packed_attention_values_that_are_not_finite(gpu, dim, heads, n):
    """Keys and values that a row does not see never reach it; those it sees go through."""
    rng = np.random.default_rng(4)

    def change(q, k, v):
        v[40, 0, 5], v[70, 0, 6], v[70, 0, 7], v[90, 0, 6] = np.inf, np.inf, -np.inf, -np.inf
        v[100, 0, 9], k[120, 0, 3] = np.nan, np.nan
        v[n - 1, 0, :], k[n, 0, :], v[n, 0, :] = np.nan, np.nan, np.inf

    packed_case(gpu, rng, heads, 1, dim, [n, 50], change=change)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,n", [(2, 400), (90, 400)])
def test_packed_attention_not_finite_values_of_little_weight(gpu, dim, heads, n):
    """A value that is not finite reaches every row that sees it, also where its weight rounds to zero in fp16."""
    rng = np.random.default_rng(19)

    def change(q, k, v):
        q[:, :, 0], k[:, :, 0] = 2, 2
        k[[10, 70, 130], 0, 0] = -6  # e^-24 of the others and less
        v[10, 0, 5], v[70, 0, 6], v[130, 0, 7], v[70, 0, 8], v[130, 0, 8] = np.inf, -np.inf, np.nan, np.inf, -np.inf

    packed_case(gpu, rng, heads, 1, dim, [n, 50], scale=1.5, change=change)


def test_packed_attention_in_place(gpu):
    """out may be q, a value that is not finite among the rows that others do not see too."""
    rng = np.random.default_rng(18)
    nq, heads, kvh, dim = [300, 70], 6, 2, 128
    starts = np.concatenate([[0], np.cumsum(nq)])
    q, k, v = (rand_f16(rng, (370, h, dim)) for h in (heads, kvh, kvh))
    v[299, 1, 7] = np.inf
    d = [dev(gpu, x) for x in (q, k, v)]
    gpu.op_packed_attention(2, dev(gpu, starts.astype(np.int32)), 370, None, 370, heads, kvh, dim, 0.0, d[0], heads * dim, d[1], kvh * dim, d[2], kvh * dim,
                            d[0], heads * dim)
    gpu.sync()
    ref, tol = packed(q, k, v, starts, starts, dim ** -0.5)
    near(d[0].download(np.float16).reshape(q.shape), ref, tol, "packed")


def test_packed_attention_bad_starts(gpu):
    """Starts out of range or decreasing read and write only what is there."""
    rng = np.random.default_rng(6)
    q, k = rand_f16(rng, (64, 2, 64)), rand_f16(rng, (64, 1, 64))
    dq, dk = dev(gpu, q), dev(gpu, k)
    for starts in ([0, 40, 20, 64], [-7, 10, 500, 900], [64, 0, 64, 0], [5, 5, 5, 5], [2 ** 31 - 1, -2 ** 31, 3, 60]):
        buf = dev(gpu, np.full(64 * 128 + 4096, 9, np.float16))
        gpu.op_packed_attention(3, dev(gpu, np.array(starts, np.int32)), 64, None, 64, 2, 1, 64, 0.0, dq, 128, dk, 64, dk, 64, buf.ptr + 4096, 128)
        gpu.sync()
        got = buf.download(np.float16)
        assert np.all(got[:2048] == 9) and np.all(got[2048 + 64 * 128:] == 9)


# ---- sampling -----------------------------------------------------------------------------

def sample_case(uocr, x, f32, t=None, k=None, p=None, m=None, u=None, shift=0, gap=0):
    rows, vocab = x.shape
    x = x.astype(np.float32 if f32 else np.float16)
    stride = vocab + gap
    padded = np.full((rows, stride), 500, x.dtype)
    padded[:, :vocab] = x
    logits = dev(uocr, np.concatenate([np.full(shift, 500, x.dtype), padded.reshape(-1)]))
    u = np.full(rows, 0.5) if u is None else np.asarray(u)

    def param(v, dt):
        return None if v is None else np.broadcast_to(np.asarray(v, dt), (rows,)).copy()

    t, k, p, m, u = param(t, np.float32), param(k, np.int32), param(p, np.float32), param(m, np.float32), param(u, np.float32)
    d = [dev(uocr, v) for v in (t, k, p, m, u)]
    token, prob = dev(uocr, np.full(rows + 1, -9, np.int32)), dev(uocr, np.full(rows + 1, -9, np.float32))
    ws = uocr.DeviceBuffer.of(np.full(max(16, uocr.sample_workspace_bytes(rows, vocab)), 0xff, np.uint8))
    uocr.op_sample(uocr.QT_F32 if f32 else uocr.QT_F16, rows, vocab, logits.ptr + shift * x.itemsize, stride, *d, ws, token, prob)
    uocr.sync()
    got, pr = token.download(np.int32), prob.download(np.float32)
    assert got[-1] == -9 and pr[-1] == -9
    for i in range(rows):
        with np.errstate(all="ignore"):
            rt, rp, margin = sample(x[i], 1.0 if t is None else t[i], 0 if k is None else k[i], 1.0 if p is None else p[i], 0.0 if m is None else m[i], u[i])
        # the sums are integers of at least 2^-38 of the largest weight per token: decisions further than that from their limits are the same
        assert margin > 1e-10 or margin == 0.0, f"row {i}: inputs at a border ({margin})"
        assert got[i] == rt, f"row {i}: token {got[i]} (logit {x[i][got[i]]}) for {rt} (logit {x[i][rt]}), margin {margin}"
        # one rounding to fp32, and 2^-38 of the largest weight that a weight may be off
        assert abs(pr[i] - rp) <= H32 * rp + 2.0 ** -37, f"row {i}: probability {pr[i]} for {rp}"
    uocr.op_sample(uocr.QT_F32 if f32 else uocr.QT_F16, rows, vocab, logits.ptr + shift * x.itemsize, stride, *d, ws, token, None)
    uocr.sync()
    assert np.array_equal(token.download(np.int32), got)
    return got[:rows]


SETTINGS = [dict(), dict(k=40), dict(p=0.9), dict(m=0.05), dict(t=0.7, k=50, p=0.95, m=0.02), dict(t=1.7), dict(t=0.0), dict(k=1), dict(p=0.3, k=7)]


@pytest.mark.parametrize("f32", [False, True], ids=["f16", "f32"])
@pytest.mark.parametrize("vocab", [1, 2, 63, 513, 4097, 129280])
@pytest.mark.parametrize("s", SETTINGS, ids=lambda s: "-".join(f"{a}{b}" for a, b in s.items()) or "plain")
def test_sample(gpu, f32, vocab, s):
    rng = np.random.default_rng(vocab + len(s))
    rows = 3 if vocab > 5000 else 9
    sample_case(gpu, rng.standard_normal((rows, vocab)) * 3, f32, u=rng.uniform(0, 1, rows), shift=1, gap=3, **s)


@pytest.mark.parametrize("f32", [False, True], ids=["f16", "f32"])
def test_sample_equal_logits(gpu, f32):
    """Few different values: ties at every limit go to the lowest id; crowded bins."""
    rng = np.random.default_rng(21)
    x = rng.integers(0, 3, (8, 9001)).astype(np.float32)
    u = rng.uniform(0, 1, 8)
    for s in (dict(k=100), dict(p=0.37), dict(k=4000, p=0.77), dict(k=8999), dict(t=5.0, p=0.5), dict(t=1e6, p=0.613), dict(m=0.2), dict(m=1.0)):
        sample_case(gpu, x, f32, u=u, **s)
    sample_case(gpu, np.zeros((2, 30000)), f32, k=[7777, 0], p=[1.0, 0.311], u=[0.9, 0.2])


@pytest.mark.parametrize("f32", [False, True], ids=["f16", "f32"])
def test_sample_special_values(gpu, f32):
    rng = np.random.default_rng(22)
    x = (rng.standard_normal((10, 1000)) * 2).astype(np.float32)
    x[0, ::2] = -np.inf
    x[1] = -np.inf
    x[2] = np.nan
    x[3, 5:900] = np.nan
    x[4, [7, 300, 999]] = np.inf
    x[5, :] = -np.inf
    x[5, 777] = -3
    x[6, 10:20] = 0.0
    x[6, 15:17] = -0.0
    x[7] = -60000 if not f32 else -3e38
    x[8, 0] = 60000
    x[9, 0::3] = -0.0
    u = rng.uniform(0, 1, 10)
    for s in (dict(), dict(k=10), dict(p=0.8), dict(m=0.1), dict(k=600, p=0.99, m=0.001), dict(t=0.0), dict(t=float("inf")), dict(t=float("inf"), k=30, p=0.5)):
        sample_case(gpu, x, f32, u=u, **s)


def test_sample_settings_at_their_ends(gpu):
    rng = np.random.default_rng(23)
    x = rng.standard_normal((1, 700)) * 2
    for s in (dict(t=-1.0), dict(t=float("nan")), dict(t=1e-30), dict(t=1e-45), dict(t=1e30), dict(k=-3), dict(k=700), dict(k=2 ** 31 - 1), dict(p=0.0), dict(p=-1.0),
              dict(p=1e-20), dict(p=5.0), dict(p=float("nan")), dict(m=-1.0), dict(m=float("nan")), dict(m=1.0), dict(m=9.0), dict(u=[0.0]), dict(u=[1.0]), dict(u=[-2.0]),
              dict(u=[3.0]), dict(u=[float("nan")]), dict(u=[0.0], p=0.5), dict(u=[0.99999994], k=5)):
        sample_case(gpu, x, True, **s)


def test_sample_mixed_rows(gpu):
    """A batch whose rows have settings of their own."""
    rng = np.random.default_rng(24)
    rows = 70
    sample_case(gpu, rng.standard_normal((rows, 2500)) * 2, False, t=rng.choice([0.0, 0.5, 1.0, 1.5], rows), k=rng.choice([0, 1, 20, 900], rows),
                p=rng.choice([1.0, 0.9, 0.2], rows), m=rng.choice([0.0, 0.05], rows), u=rng.uniform(0, 1, rows))


@pytest.mark.parametrize("f32", [False, True], ids=["f16", "f32"])
def test_sample_long_crowded_rows(gpu, f32):
    """Few different values in rows that several blocks share."""
    rng = np.random.default_rng(25)
    x = rng.integers(0, 3, (8, 40001)).astype(np.float32)
    u = rng.uniform(0, 1, 8)
    for s in (dict(k=100), dict(p=0.37), dict(k=4000, p=0.77), dict(k=40000), dict(t=5.0, p=0.5), dict(t=1e6, p=0.613), dict(m=0.2), dict(m=1.0)):
        sample_case(gpu, x, f32, u=u, **s)
    x[:, ::7] = -np.inf
    x[1, :] = 2.0
    x[2, 1:] = np.nan
    x[3, ::2] = np.inf
    x[4] = -np.inf
    x[4, 39999] = 1.0
    x[5] = -np.inf
    for s in (dict(), dict(k=1024), dict(k=1025, p=0.9), dict(p=0.999), dict(t=0.0), dict(t=float("inf"), k=30000, p=0.51)):
        sample_case(gpu, x, f32, u=u, **s)


@pytest.mark.parametrize("f32", [False, True], ids=["f16", "f32"])
@pytest.mark.parametrize("vocab", [3000, 40003])
def test_sample_flat_rows(gpu, f32, vocab):
    """Logits within little of each other, some rows with most tokens masked or with a few far below, NaN between."""
    rng = np.random.default_rng(26)
    x = (rng.standard_normal((9, vocab)) * rng.choice([0.01, 0.1, 0.5], (9, 1))).astype(np.float32)
    x[3, rng.random(vocab) < 0.97] = -np.inf
    x[4, rng.random(vocab) < 0.5] = np.nan
    x[5, ::3] -= 40
    x[6, 512:] -= 3  # the first step is not like the others
    x[7, :-512] -= 0.5
    u = rng.uniform(0, 1, 9)
    for s in (dict(p=0.9), dict(p=0.999999), dict(k=2000, p=0.5), dict(k=700), dict(k=vocab - 1), dict(p=0.5, t=3.0), dict(p=0.7, m=0.9), dict(p=0.9, t=0.05)):
        sample_case(gpu, x, f32, u=u, **s)


@pytest.mark.parametrize("rows,vocab", [(1, 16384), (1, 16385), (64, 32768), (64, 32769), (63, 20000), (128, 32768), (128, 32769), (2, 300007), (1, 1500000)])
def test_sample_one_block_or_several(gpu, rows, vocab):
    """Sizes on both sides of where rows are shared, rows of more than 512 steps, each row with settings of its own."""
    rng = np.random.default_rng(rows + vocab)
    sample_case(gpu, rng.standard_normal((rows, vocab)) * 3, True, t=rng.choice([0.6, 1.0, 1.3], rows), k=rng.choice([0, 30, 700], rows),
                p=rng.choice([1.0, 0.9, 0.5], rows), m=rng.choice([0.0, 0.01], rows), u=rng.uniform(0, 1, rows), gap=5)


# ---- together -------------------------------------------------------------------------------

def test_prompts_then_decode(gpu):
    """As a server runs them: prompts packed (the second one behind a cached prefix), their rows rotated and cached, then decode steps
    of append, paged attention, logits and sampling, captured once and replayed: each step equals the eager calls on a cache of its
    own, and the caches agree at the end."""
    rng = np.random.default_rng(31)
    heads, kvh, dim, page, vocab = 4, 2, 64, 16, 1000
    hidden, rows = heads * dim, (heads + 2 * kvh) * dim
    prompts, prefix, steps = [37, 20, 5], [0, 33, 0], 6
    total = [a + b for a, b in zip(prompts, prefix)]
    wqkv = rand_f16(rng, (rows, hidden), 0.05)
    head, embed = rand_f16(rng, (vocab, hidden), 0.2), rand_f16(rng, (vocab, hidden))
    dw, dh, de = dev(gpu, wqkv), dev(gpu, head), dev(gpu, embed)
    x0 = rand_f16(rng, (sum(total), hidden))
    u = rng.uniform(0, 1, (steps, 3)).astype(np.float32)

    def start():
        """The prompts through packed attention; returns the cache and the last rows' attention."""
        c = Pages(rng, 1, kvh, dim, page, [n + steps for n in total])
        desc = c.upload(gpu)
        where = np.concatenate([[0]] * 37 + [[1]] * 53 + [[2]] * 5).astype(np.int32)
        pos = np.concatenate([np.arange(n) for n in total]).astype(np.int32)
        dx, qkv = dev(gpu, x0), gpu.DeviceBuffer(2 * len(pos) * rows)
        gpu.op_gemm(gpu.QT_F16, dw, None, len(pos), rows, hidden, dx, None, qkv)
        # the prefix of sequence 1 is cached by an earlier call
        first = np.where((where == 1) & (pos < 33), where, -1).astype(np.int32)
        later = np.where((where == 1) & (pos < 33), -1, where).astype(np.int32)
        q, k = gpu.DeviceBuffer(2 * len(pos) * hidden), gpu.DeviceBuffer(2 * len(pos) * kvh * dim)
        for seqs in (first, later):
            gpu.op_kv_append(desc, len(pos), dev(gpu, seqs), dev(gpu, pos), heads, 1e4, qkv, rows, q, hidden, qkv.ptr + 2 * hidden, rows, k, kvh * dim,
                             qkv.ptr + 2 * (hidden + kvh * dim), rows)
        gpu.sync()
        # keys and values of every token out of the cache, queries of the new ones
        kk, vv = gpu.DeviceBuffer(k.nbytes), gpu.DeviceBuffer(k.nbytes)
        gpu.op_kv_gather(desc, len(pos), dev(gpu, where), dev(gpu, pos), kk, kvh * dim, vv, kvh * dim)
        gpu.sync()
        assert np.array_equal(kk.download(np.uint16), k.download(np.uint16))
        new = later >= 0
        qn = q.download(np.float16).reshape(-1, hidden)[new]
        qs, ks = np.concatenate([[0], np.cumsum(prompts)]), np.concatenate([[0], np.cumsum(total)])
        out = gpu.DeviceBuffer(qn.nbytes)
        gpu.op_packed_attention(3, dev(gpu, qs.astype(np.int32)), int(qs[-1]), dev(gpu, ks.astype(np.int32)), int(ks[-1]), heads, kvh, dim, 0.0,
                                dev(gpu, qn), hidden, kk, kvh * dim, vv, kvh * dim, out, hidden)
        gpu.sync()
        got = out.download(np.float16).reshape(-1, heads, dim)
        ref, tol = packed(qn.reshape(-1, heads, dim), kk.download(np.float16).reshape(-1, kvh, dim), vv.download(np.float16).reshape(-1, kvh, dim), qs, ks, dim ** -0.5)
        near(got, ref, tol, "prompts")
        # the last row of each prompt is also what one token's attention over the cache gives
        last = qn.reshape(-1, heads, dim)[qs[1:] - 1]
        ws = gpu.DeviceBuffer(gpu.paged_attention_workspace_bytes(3, heads, kvh, dim))
        one = gpu.DeviceBuffer(last.nbytes)
        gpu.op_paged_attention(desc, dev(gpu, np.array(total, np.int32)), heads, 0.0, dev(gpu, last), hidden, ws, one, hidden)
        gpu.sync()
        near(one.download(np.float16).reshape(3, heads, dim), ref[qs[1:] - 1], tol[qs[1:] - 1], "last rows")
        return c, desc, got[qs[1:] - 1].reshape(3, hidden)

    def loop(desc, first, graph):
        state = {n: dev(gpu, v) for n, v in dict(x=first, pos=np.zeros(3, np.int32), len=np.zeros(3, np.int32), u=u[0], t=np.full(3, 0.8, np.float32),
                                                 k=np.array([0, 30, 5], np.int32), p=np.array([0.9, 1, 0.8], np.float32)).items()}
        b = {n: gpu.DeviceBuffer(2 * s) for n, s in dict(qkv=3 * rows, q=3 * hidden, ctx=3 * hidden, logits=3 * vocab).items()}
        tok = gpu.DeviceBuffer(12)
        ws = gpu.DeviceBuffer(gpu.paged_attention_workspace_bytes(3, heads, kvh, dim))
        sws = gpu.DeviceBuffer(gpu.sample_workspace_bytes(3, vocab))

        def step():
            gpu.op_gemm(gpu.QT_F16, dw, None, 3, rows, hidden, state["x"], None, b["qkv"])
            gpu.op_kv_append(desc, 3, None, state["pos"], heads, 1e4, b["qkv"], rows, b["q"], hidden, b["qkv"].ptr + 2 * hidden, rows, None, 0,
                             b["qkv"].ptr + 2 * (hidden + kvh * dim), rows)
            gpu.op_paged_attention(desc, state["len"], heads, 0.0, b["q"], hidden, ws, b["ctx"], hidden)
            gpu.op_gemm(gpu.QT_F16, dh, None, 3, vocab, hidden, b["ctx"], None, b["logits"])
            gpu.op_sample(gpu.QT_F16, 3, vocab, b["logits"], vocab, state["t"], state["k"], state["p"], None, state["u"], sws, tok, None)

        cap = None
        tokens, ctxs = [], []
        for i in range(steps):
            state["pos"].upload(np.array(total, np.int32) + i)
            state["len"].upload(np.array(total, np.int32) + i + 1)
            state["u"].upload(u[i])
            if graph and cap is None:
                with gpu.Capture() as cap:
                    step()
            if graph:
                cap.replay(1)
            else:
                step()
            gpu.sync()
            t = tok.download(np.int32)
            logits = b["logits"].download(np.float16).reshape(3, vocab)
            for s in range(3):
                want, _, margin = sample(logits[s], np.float32(0.8), [0, 30, 5][s], np.float32([0.9, 1, 0.8][s]), 0.0, u[i][s])
                assert margin < 1e-10 or t[s] == want
            tokens.append(t)
            ctxs.append(b["ctx"].download(np.uint16))
            state["x"].upload(embed[t])
        if cap is not None:
            cap.release()
        return np.array(tokens), np.array(ctxs)

    rng_state = rng.bit_generator.state
    c1, d1, f1 = start()
    rng.bit_generator.state = rng_state
    c2, d2, f2 = start()
    assert np.array_equal(f1, f2)
    eager, graph = loop(d1, f1, False), loop(d2, f2, True)
    assert np.array_equal(eager[0], graph[0]) and np.array_equal(eager[1], graph[1])
    for side in range(2):
        assert np.array_equal(c1.download().data[side].view(np.uint16), c2.download().data[side].view(np.uint16))


def test_replays_of_every_operator(gpu):
    """One graph with all operators (paged attention with both ways of joining, sampling in one block and in several) on shared
    workspaces, replayed with other contents of its arrays, eager calls and synchronizations in between: the eager results' bits."""
    rng = np.random.default_rng(33)
    dim, page, n = 64, 16, 3
    lengths = [700, 33, 1200]
    sizes = [(32, 2), (8, 4)]  # joined by a launch of its own, and by the last block
    caches = [Pages(rng, t, kvh, dim, page, [x + 8 for x in lengths]) for t, (_, kvh) in zip((1, 3), sizes)]
    for c in caches:
        c.fill(rng, lengths)
    ws = gpu.DeviceBuffer(max(gpu.paged_attention_workspace_bytes(n, h, kvh, dim) for h, kvh in sizes))
    vocabs = [900, 40000]
    sws = gpu.DeviceBuffer(max(gpu.sample_workspace_bytes(n, x) for x in vocabs))
    x = {name: gpu.DeviceBuffer(size) for name, size in dict(q=2 * n * 32 * dim, k=2 * n * 4 * dim, v=2 * n * 4 * dim, pos=4 * n, len=4 * n, starts=4 * (n + 1),
                                                             logits=4 * n * vocabs[1], u=4 * n, top_p=4 * n, top_k=4 * n).items()}

    def fresh(i):
        r = np.random.default_rng(100 + i)
        for name in ("q", "k", "v"):
            x[name].upload(rand_f16(r, x[name].nbytes // 2))
        pos = np.array(lengths, np.int32) + i
        x["pos"].upload(pos)
        x["len"].upload(pos + 1)
        x["starts"].upload(np.array([0, i % 3, 2, 3], np.int32))
        x["logits"].upload((r.standard_normal(n * vocabs[1]) * 3).astype(np.float32))
        x["u"].upload(r.uniform(0, 1, n).astype(np.float32))
        x["top_p"].upload(np.array([0.9, 1.0, 0.5], np.float32))
        x["top_k"].upload(np.array([0, 40, 600], np.int32))

    def outputs():
        return [gpu.DeviceBuffer(size) for size in [2 * n * 32 * dim] * 4 + [2 * n * 4 * dim] * 4 + [4 * n] * 4]

    def run(descs, o):
        for i, ((h, kvh), desc) in enumerate(zip(sizes, descs)):
            gpu.op_kv_append(desc, n, None, x["pos"], h, 1e4, x["q"], h * dim, o[i], h * dim, x["k"], kvh * dim, None, 0, x["v"], kvh * dim)
            gpu.op_paged_attention(desc, x["len"], h, 0.0, o[i], h * dim, ws, o[2 + i], h * dim)
            gpu.op_kv_gather(desc, n, None, x["pos"], o[4 + 2 * i], kvh * dim, o[5 + 2 * i], kvh * dim)
            gpu.op_packed_attention(n, x["starts"], n, None, n, h, kvh, dim, 0.0, o[i], h * dim, o[4 + 2 * i], kvh * dim, o[5 + 2 * i], kvh * dim, o[i], h * dim)
            gpu.op_sample(gpu.QT_F32, n, vocabs[i], x["logits"], vocabs[i], None, x["top_k"], x["top_p"], None, x["u"], sws, o[8 + 2 * i], o[9 + 2 * i])

    eager, held = outputs(), outputs()
    d1 = [c.upload(gpu) for c in caches]
    keep = [(c.dev, c.dev_s, c.dev_t) for c in caches]
    d2 = [c.upload(gpu) for c in caches]
    fresh(0)
    run(d1, eager)
    gpu.sync()
    with gpu.Capture() as cap:
        run(d2, held)
    for i in range(6):
        fresh(i)
        run(d1, eager)
        if i % 2:
            gpu.sync()
        cap.replay(1)
        gpu.sync()
        for j, (a, b) in enumerate(zip(eager, held)):
            assert np.array_equal(a.download(np.uint16), b.download(np.uint16)), f"replay {i}, output {j}"
    cap.release()
    assert len(keep) == 2
