"""Paged cache of the decode step on the GPU against plain 64-bit integers: every output has equal bits."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

I64_MIN = -(1 << 63)


# ---------------------------------------------------------------------------------- plain restatement
def rdiv(x, s):
    q = np.floor_divide(x + (1 << s) // 2, 1 << s)
    return q, x - q * (1 << s)


class Pool:
    """Pages of a cache on the host, logical [page][head][slot][channel], in either memory order; `gap` elements
    between the rows show what is written where nothing should be."""

    def __init__(self, rng, pages, heads, slots, dim, bits, layout="head", gap=0, std=1000.0):
        self.dtype = np.dtype(np.int16 if bits == 16 else np.int32)
        row = dim + gap
        shape = (pages, heads, slots, row) if layout == "head" else (pages, slots, heads, row)
        self.raw = np.clip(np.rint(rng.normal(0, std, shape)), -(1 << (bits - 1)), (1 << (bits - 1)) - 1).astype(self.dtype)
        view = self.raw if layout == "head" else self.raw.transpose(0, 2, 1, 3)
        self.view = view[..., :dim]
        self.strides = tuple(x // self.raw.itemsize for x in view.strides[:3])


def table_for(rng, n_pages, tokens, page, width=None):
    counts = [-(-n // page) for n in tokens]
    width = max([1] + counts) if width is None else width
    order = rng.permutation(n_pages)[:sum(counts)]
    t = np.full((len(tokens), width), -1, np.int32)
    at = 0
    for b, n in enumerate(counts):
        t[b, :n] = order[at:at + n]
        at += n
    return t


def upload(ctx, a):
    return ctx.upload(np.ascontiguousarray(a)) if a is not None else None


def fetch(ctx, buf, like):
    return ctx.download(buf, like.nbytes, dtype=like.dtype).reshape(like.shape)


def make_cache(ctx, k, v, page, heads, dim, bits, k_shift=0, v_shift=0, bounds=None):
    from grape_b200.decode import KVCache
    dk, dv, db = upload(ctx, k.raw), upload(ctx, v.raw), upload(ctx, bounds)
    return KVCache(ctx, k.raw.shape[0], page, heads, dim, bits=bits, k_shift=k_shift, v_shift=v_shift, d_k=dk, d_v=dv, d_bounds=db,
                   strides=k.strides)


# ---------------------------------------------------------------------------------- append
def plain_append(k, v, bounds, table, start, offsets, q, keys, values, cos, sin, rot, shift, inter, k_shift, v_shift, page):
    """Token by token; every value as a Python integer where 64 bits could wrap."""
    lim = 1 << (8 * k.dtype.itemsize - 1)
    idx = np.arange(rot // 2)
    first, second = (2 * idx, 2 * idx + 1) if inter else (idx, idx + rot // 2)
    out = {n: (np.zeros(x.shape, np.int32), np.zeros(x.shape, np.int32)) for n, x in (("q", q), ("k", keys), ("v", values))}
    saturated = False

    def turned(x, p):
        y = x.astype(object) * (1 << shift)
        if rot:
            a, b = x[:, first].astype(object), x[:, second].astype(object)
            c, s = cos[p].astype(object), sin[p].astype(object)
            y[:, first], y[:, second] = a * c - b * s, b * c + a * s
        return y

    for b in range(len(start)):
        for t in range(offsets[b], offsets[b + 1]):
            p = int(start[b]) + t - int(offsets[b])
            pg, slot = table[b, p // page], p % page
            kq, kr = rdiv(turned(keys[t], p), shift + k_shift)
            vq, vr = rdiv(values[t].astype(object), v_shift)
            qq, qr = rdiv(turned(q[t], p), shift)
            saturated |= any((x < -lim).any() or (x >= lim).any() for x in (kq, vq))
            saturated |= (qq < -(1 << 31)).any() or (qq >= 1 << 31).any()
            kq, vq = np.clip(kq, -lim, lim - 1).astype(k.dtype), np.clip(vq, -lim, lim - 1).astype(k.dtype)
            out["q"][0][t], out["q"][1][t] = np.clip(qq, -(1 << 31), (1 << 31) - 1), qr
            out["k"][1][t], out["v"][1][t] = kr, vr
            k.view[pg, :, slot], v.view[pg, :, slot] = kq, vq
            if bounds is not None:
                bounds[pg, :, 0] = kq if slot == 0 else np.minimum(bounds[pg, :, 0], kq)
                bounds[pg, :, 1] = kq if slot == 0 else np.maximum(bounds[pg, :, 1], kq)
    return out, saturated


APPEND = [
    # new tokens, starts, heads, kv_heads, dim, rot, bits, page, interleaved, layout, shift, k_shift, v_shift, gap
    ([1], [0], 1, 1, 8, 8, 32, 1, True, "head", 16, 0, 0, 0),
    ([1], [2047], 1, 1, 4096, 4096, 32, 64, True, "head", 16, 0, 0, 0),
    ([1, 1, 0, 1], [5, 0, 3, 16], 4, 2, 64, 64, 16, 16, False, "token", 16, 6, 6, 0),
    ([70, 0, 3, 129], [0, 9, 63, 60], 3, 3, 24, 16, 32, 64, True, "head", 14, 2, 1, 8),
    ([70, 0, 3, 129], [0, 9, 63, 60], 5, 1, 40, 16, 32, 64, False, "token", 14, 2, 1, 8),
    ([33, 17], [1, 0], 8, 2, 128, 0, 16, 7, True, "head", 0, 8, 4, 0),
    ([33, 17], [1, 0], 8, 2, 128, 0, 16, 7, False, "token", 9, 0, 4, 8),
    ([300], [11], 2, 2, 72, 72, 16, 100, True, "token", 16, 5, 5, 0),
    ([65, 66, 2, 2], [63, 63, 63, 64], 7, 7, 80, 80, 32, 64, False, "head", 30, 0, 30, 0),
    ([5] * 70, list(range(70)), 2, 1, 16, 8, 32, 3, True, "head", 16, 0, 0, 0),
]


@pytest.mark.parametrize("case", APPEND, ids=str)
@pytest.mark.parametrize("extreme", [False, True])
def test_append(gctx, case, extreme):
    from grape_b200 import decode
    new, start, H, KV, D, rot, bits, page, inter, layout, shift, k_shift, v_shift, gap = case
    rng = np.random.default_rng(7)
    T, offsets = sum(new), np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    tokens = [s + n for s, n in zip(start, new)]
    table = table_for(rng, sum(-(-n // page) for n in tokens) + 2, tokens, page)
    P = sum(-(-n // page) for n in tokens) + 2
    k, v = (Pool(rng, P, KV, page, D, bits, layout, gap) for _ in range(2))
    bounds = np.stack([k.view.min(axis=2), k.view.max(axis=2)], axis=2).copy()
    x = rng.integers(-(1 << 31), 1 << 31, (T, (H + 2 * KV) * D + 4)) if extreme else np.rint(rng.normal(0, 65536, (T, (H + 2 * KV) * D + 4)))
    x = x.astype(np.int32)
    if extreme:
        x[0, :8] = [-(1 << 31), -(1 << 31), (1 << 31) - 1, (1 << 31) - 1, -(1 << 31), (1 << 31) - 1, 0, 1]
    pos = max(tokens)
    ang = np.arange(pos)[:, None] * 10000.0 ** (-np.arange(rot // 2) / max(rot // 2, 1))
    cos, sin = (np.rint(f(ang) * (1 << shift)).astype(np.int32) for f in (np.cos, np.sin))
    rows = x[:, :(H + 2 * KV) * D].reshape(T, H + 2 * KV, D)
    cache = make_cache(gctx, k, v, page, KV, D, bits, k_shift, v_shift, bounds)
    dx, dt, ds, do, dc, dsn = (upload(gctx, a) for a in (x, table, np.array(start, np.int32), offsets, cos, sin))
    outs = {n: gctx.upload(np.full((T, h, D), 77, np.int32)) for n, h in (("q", H), ("q_rem", H), ("k_rem", KV), ("v_rem", KV))}
    rotation = decode.Rotation(dc if rot else None, dsn if rot else None, pos, rot, shift, inter)
    stride = x.shape[1]
    gctx.status()
    decode.kv_append(cache, dt, table.shape[1], len(new), ds, do, T, dx.at(4 * H * D), dx.at(4 * (H + KV) * D), rotation=rotation, d_q=dx,
                     heads=H, d_q_out=outs["q"], d_q_rem=outs["q_rem"], d_k_rem=outs["k_rem"], d_v_rem=outs["v_rem"], q_stride=stride,
                     k_stride=stride, v_stride=stride)
    status = gctx.status()
    want, saturated = plain_append(k, v, bounds, table, start, offsets, rows[:, :H], rows[:, H:H + KV], rows[:, H + KV:], cos, sin, rot,
                                   shift, inter, k_shift, v_shift, page)
    assert status == (decode.STATUS_RANGE if saturated else 0)
    assert saturated or not extreme or bits == 32
    assert np.array_equal(fetch(gctx, outs["q"], want["q"][0]), want["q"][0])
    for n in ("q", "k", "v"):
        assert np.array_equal(fetch(gctx, outs[n + "_rem"], want[n][1]), want[n][1]), n
    # the raw pools: gaps, other slots and other pages are as they were
    assert np.array_equal(fetch(gctx, cache.k, k.raw), k.raw)
    assert np.array_equal(fetch(gctx, cache.v, v.raw), v.raw)
    assert np.array_equal(fetch(gctx, cache.bounds, bounds), bounds)


def test_append_without_queries_rotation_bounds_or_remainders(gctx):
    from grape_b200 import decode
    rng = np.random.default_rng(3)
    k, v = (Pool(rng, 5, 2, 16, 32, 32) for _ in range(2))
    x = rng.integers(-9, 9, (20, 2, 2, 32)).astype(np.int32)
    table, start, offsets = np.array([[4, 1]], np.int32), [6], np.array([0, 20], np.int32)
    cache = make_cache(gctx, k, v, 16, 2, 32, 32)
    dk, dv, dt, ds, do = (upload(gctx, a) for a in (x[:, 0], x[:, 1], table, np.array(start, np.int32), offsets))
    decode.kv_append(cache, dt, 2, 1, ds, do, 20, dk, dv)
    plain_append(k, v, None, table, start, offsets, x[:, 0], x[:, 0], x[:, 1], None, None, 0, 0, True, 0, 0, 16)
    assert np.array_equal(fetch(gctx, cache.k, k.raw), k.raw) and np.array_equal(fetch(gctx, cache.v, v.raw), v.raw)
    assert gctx.status() == 0


@pytest.mark.parametrize("fault", ["page -1", "page too large", "table too short", "position", "start", "offsets", "order"])
def test_append_skips_what_lies_outside(gctx, fault):
    """Bad device data sets the status bit; everything else is appended, nothing is written elsewhere."""
    from grape_b200 import decode
    rng = np.random.default_rng(4)
    P, KV, D, page = 6, 1, 16, 8
    k, v = (Pool(rng, P, KV, page, D, 32) for _ in range(2))
    bounds = np.stack([k.view.min(axis=2), k.view.max(axis=2)], axis=2).copy()
    x = rng.integers(-1000, 1000, (24, 2, KV, D)).astype(np.int32)
    table, start, offsets = np.array([[0, 1], [2, 3]], np.int32), np.array([4, 0], np.int32), np.array([0, 10, 24], np.int32)
    cos, sin = (rng.integers(-65536, 65536, (16, 8)).astype(np.int32) for _ in range(2))
    cache = make_cache(gctx, k, v, page, KV, D, 32, bounds=bounds)
    good_table, skipped, positions = table.copy(), [], 16
    if fault == "page -1":
        table[0, 1], skipped = -1, range(4, 10)
    elif fault == "page too large":
        table[0, 1], skipped = P, range(4, 10)
    elif fault == "table too short":
        start[0], skipped = 10, range(6, 10)      # positions 16..19 have no page
    elif fault == "position":
        positions, skipped = 11, [7, 8, 9, 21, 22, 23]
    elif fault == "start":
        start[0], skipped = -3, range(0, 10)
    elif fault == "offsets":
        offsets[2], skipped = 25, range(10, 24)
    else:
        offsets[1], skipped = -1, range(0, 24)
    dx, dt, ds, do, dc, dn = (upload(gctx, a) for a in (x, table, start, offsets, cos, sin))
    gctx.status()
    rem = gctx.upload(np.full((24, KV, D), 5, np.int32))
    decode.kv_append(cache, dt, 2, 2, ds, do, 24, dx, dx.at(4 * KV * D), k_stride=2 * KV * D, v_stride=2 * KV * D, d_k_rem=rem,
                     rotation=decode.Rotation(dc, dn, positions, 16))
    assert gctx.status() == decode.STATUS_PLACE
    got = fetch(gctx, rem, x[:, 0])
    if fault == "order":
        assert np.array_equal(fetch(gctx, cache.k, k.raw)[[4, 5]], k.raw[[4, 5]])
        return
    want = np.full((24, KV, D), 5, np.int32)
    for b in range(2):
        for t in range(offsets[b], min(offsets[b + 1], 24)):
            if t in skipped:
                continue
            one, _ = plain_append(k, v, bounds, good_table, [start[b] + t - offsets[b] if i == b else 0 for i in range(2)],
                                  [0, 1, 1] if b == 0 else [0, 0, 1], x[t:t + 1, 0], x[t:t + 1, 0], x[t:t + 1, 1], cos, sin, 16, 16, True,
                                  0, 0, page)
            want[t] = one["k"][1][0]
    assert np.array_equal(got, want)
    assert np.array_equal(fetch(gctx, cache.k, k.raw), k.raw) and np.array_equal(fetch(gctx, cache.v, v.raw), v.raw)
    assert np.array_equal(fetch(gctx, cache.bounds, bounds), bounds)


# ---------------------------------------------------------------------------------- select
def plain_select(bounds, table, lens, q, KV, page, n, recent):
    B, H, D = q.shape
    P = bounds.shape[0]
    sel, bound = np.full((B, KV, n), -1, np.int32), np.full((B, KV, table.shape[1]), 99, np.int64)
    for b in range(B):
        pages = -(-int(lens[b]) // page)
        for g in range(KV):
            for i in range(pages):
                pg = table[b, i]
                if not 0 <= pg < P:
                    bound[b, g, i] = I64_MIN
                    continue
                lo, hi = (bounds[pg, g, j].astype(object) for j in range(2))
                bound[b, g, i] = max(int(sum(max(a, c) for a, c in zip(x * lo, x * hi)))
                                     for x in q[b, g * (H // KV):(g + 1) * (H // KV)].astype(object))
            old = max(0, pages - recent)
            best = sorted(range(old), key=lambda i: (-int(bound[b, g, i]), i))[:max(0, min(n, pages) - (pages - old))]
            chosen = sorted(best + list(range(old, pages)))
            sel[b, g, :len(chosen)] = chosen
    return sel, bound


SELECT = [
    # lengths, heads, kv_heads, dim, bits, page, n_select, recent
    ([1], 1, 1, 8, 32, 1, 1, 0),
    ([0, 5, 64, 65], 4, 2, 64, 32, 16, 2, 1),
    ([1021], 8, 8, 64, 32, 16, 8, 1),
    ([3000, 1, 1700], 6, 2, 72, 16, 24, 40, 4),
    ([640, 0], 14, 2, 128, 16, 8, 80, 3),
    ([640, 600], 5, 1, 4096, 32, 100, 3, 0),
    ([2100, 2047], 9, 1, 24, 32, 1, 300, 300),
    ([1500], 2, 2, 200, 16, 2, 600, 1),
    # one head a group and several, for rows of every width: a few 16-byte pieces, warps, blocks
    ([300, 17], 3, 3, 40, 16, 3, 20, 2),
    ([800, 90], 2, 2, 1024, 16, 16, 9, 1),
    ([130], 2, 2, 520, 32, 4, 7, 0),
    ([333, 12], 6, 2, 1032, 16, 8, 12, 1),
    ([700, 1], 2, 1, 32, 32, 2, 50, 5),
    ([5000] * 40, 4, 4, 48, 32, 4, 30, 1),
    ([6000] * 30, 9, 3, 128, 16, 3, 30, 1),
]


@pytest.mark.parametrize("case", SELECT, ids=str)
@pytest.mark.parametrize("kind", ["normal", "ties", "extreme"])
def test_select(gctx, case, kind):
    from grape_b200 import decode
    lens, H, KV, D, bits, page, n, recent = case
    rng = np.random.default_rng(11)
    P = sum(-(-x // page) for x in lens) + 1
    table = table_for(rng, P, lens, page)
    top = 1 << (bits - 1)
    if kind == "ties":       # few different pages: most bounds are equal
        bounds = np.sort(rng.integers(-3, 4, (3, KV, 2, D)), axis=2)[rng.integers(0, 3, P)]
        q = rng.integers(-2, 3, (len(lens), H, D))
    elif kind == "extreme":  # the largest magnitudes that keep the sum below 2^63, in two channels
        bounds, q = np.zeros((P, KV, 2, D), np.int64), np.zeros((len(lens), H, D), np.int64)
        bounds[..., 1:3] = np.sort(rng.choice([-top, top - 1, 0, 1, -1], (P, KV, 2, 2)), axis=2)
        q[..., 1:3] = rng.choice([-(1 << 31) + 1, (1 << 31) - 1, 0, 1], (len(lens), H, 2))
    else:
        bounds = np.sort(np.rint(rng.normal(0, 3000, (P, KV, 2, D))), axis=2)
        q = np.rint(rng.normal(0, 65536, (len(lens), H, D)))
    bounds, q = bounds.astype(np.int16 if bits == 16 else np.int32), q.astype(np.int32)
    want, want_bound = plain_select(bounds, table, lens, q, KV, page, n, recent)
    cache = decode.KVCache(gctx, P, page, KV, D, bits=bits, d_bounds=upload(gctx, bounds), d_k=0, d_v=0)
    dt, dl, dq = upload(gctx, table), upload(gctx, np.array(lens, np.int32)), upload(gctx, q)
    gctx.status()
    for with_bound in (True, False):
        ds, db = gctx.upload(np.full(want.shape, 55, np.int32)), gctx.upload(np.full(want_bound.shape, 99, np.int64))
        decode.kv_select(cache, dt, table.shape[1], len(lens), dl, dq, H, n, ds, recent=recent, d_bound=db if with_bound else None)
        assert np.array_equal(fetch(gctx, ds, want), want)
        assert not with_bound or np.array_equal(fetch(gctx, db, want_bound), want_bound)
    assert gctx.status() == 0


def test_select_with_bad_pages_and_lengths(gctx):
    from grape_b200 import decode
    rng = np.random.default_rng(12)
    bounds = np.sort(rng.integers(-99, 99, (9, 1, 2, 16)), axis=2).astype(np.int32)
    table = np.array([[0, -1, 2, 9, 4], [5, 6, 7, 8, 0], [1, 2, 3, 4, 5]], np.int32)
    q = rng.integers(-99, 99, (3, 2, 16)).astype(np.int32)
    cache = decode.KVCache(gctx, 9, 4, 1, 16, d_bounds=upload(gctx, bounds), d_k=0, d_v=0)
    dt, dq = upload(gctx, table), upload(gctx, q)
    lens = np.array([20, -1, 21], np.int32)              # bad pages; negative; longer than the table
    want, want_bound = plain_select(bounds, table, [20, 0, 20], q, 1, 4, 4, 1)
    gctx.status()
    ds, db = gctx.upload(np.zeros(want.shape, np.int32)), gctx.upload(np.full(want_bound.shape, 99, np.int64))
    decode.kv_select(cache, dt, 5, 3, upload(gctx, lens), dq, 2, 4, ds, recent=1, d_bound=db)
    assert np.array_equal(fetch(gctx, ds, want), want) and np.array_equal(fetch(gctx, db, want_bound), want_bound)
    assert gctx.status() == decode.STATUS_PLACE


# ---------------------------------------------------------------------------------- attend
WITNESS = ("score", "score_rem", "exp_in", "exp_out", "softmax")


def plain_attend(k, v, table, lens, q, exp, low, page, score_shift, soft_shift, max_keys, selected=None, fill=33):
    B, H, D = q.shape
    P, KV = k.view.shape[:2]
    out = {n: np.full((B, H, max_keys), fill, np.int32) for n in WITNESS}
    out |= {"out": np.zeros((B, H, D), np.int32), "out_rem": np.zeros((B, H, D), np.int32), "sum": np.zeros((B, H), np.int64)}
    status = 0
    for b in range(B):
        n = int(lens[b])
        for g in range(KV):
            if selected is None:
                cols = [(i, i) for i in range(min(n, max_keys))]
                status |= 16 if n > max_keys else 0
            else:
                cols = [(r * page + s, p * page + s) for r, p in enumerate(selected[b, g]) for s in range(page) if 0 <= p]
                if any(p >= table.shape[1] for r, p in enumerate(selected[b, g]) if r * page < max_keys) and n:
                    status |= 16
                cols = [(i, t) for i, t in cols if t < n and t // page < table.shape[1] and i < max_keys]
            bad = [t for _, t in cols if not 0 <= table[b, t // page] < P]
            status |= 16 if bad else 0
            cols = [(i, t) for i, t in cols if t not in set(bad)]
            if not cols:
                status |= 32 if bad or (selected is not None and n) else 0
                continue
            at = np.array([i for i, _ in cols])
            tok = np.array([t for _, t in cols])
            kk, vv = (x.view[table[b, tok // page], g, tok % page] for x in (k, v))
            # Python integers wherever the products could pass 2^62
            wide = max(abs(int(kk.min())), abs(int(kk.max()))) * int(np.abs(q[b].astype(np.int64)).max()) * D >= 1 << 62
            kk, vv = kk.astype(object if wide else np.int64), vv.astype(object if wide else np.int64)
            for h in range(g * (H // KV), (g + 1) * (H // KV)):
                s, r = rdiv(kk.dot(q[b, h].astype(kk.dtype)), score_shift)
                if max(s) >= 1 << 31 or min(s) < -(1 << 31):
                    status |= 8
                s = np.clip(s, -(1 << 31), (1 << 31) - 1)
                x = s - max(s)
                status |= 32 if min(x) < low else 0
                x = np.maximum(x, low).astype(np.int64)
                e = exp[x - low].astype(np.int64)
                z = int(e.sum())
                status |= 32 if z == 0 else 0
                o = np.floor_divide(e * (1 << soft_shift) + z // 2, z) if z else e * 0
                y, yr = rdiv(o.astype(vv.dtype).dot(vv), soft_shift)
                for name, a in (("score", s), ("score_rem", r), ("exp_in", x), ("exp_out", e), ("softmax", o)):
                    out[name][b, h, at] = a
                if max(y) >= 1 << 31 or min(y) < -(1 << 31):
                    status |= 8
                out["out"][b, h], out["out_rem"][b, h], out["sum"][b, h] = np.clip(y, -(1 << 31), (1 << 31) - 1), yr, z
    return out, status


def run_attend(ctx, cache, table, lens, q, exp, low, score_shift, soft_shift, max_keys, selected=None, witness=True, q_stride=None):
    from grape_b200 import decode
    B, H, D = q.shape
    like = {n: np.full((B, H, max_keys), 33, np.int32) for n in WITNESS}
    like |= {"out": np.full((B, H, D), 33, np.int32), "out_rem": np.full((B, H, D), 33, np.int32), "sum": np.full((B, H), 33, np.int64)}
    bufs = {n: ctx.upload(a) for n, a in like.items()}
    rows = np.zeros((B, q_stride or H * D), np.int32)
    rows[:, :H * D] = q.reshape(B, H * D)
    dt, dl, dq, de, ds = (upload(ctx, a) for a in (table, np.array(lens, np.int32), rows, exp, selected))
    w = {"d_" + n: bufs[n] for n in WITNESS + ("sum", "out_rem")} if witness else {}
    decode.kv_attend(cache, dt, table.shape[1], B, dl, dq, H, decode.ExpTable(de, low, exp.size), bufs["out"], score_shift=score_shift,
                     soft_shift=soft_shift, max_keys=max_keys, d_selected=ds, n_select=0 if selected is None else selected.shape[2],
                     q_stride=q_stride, **w)
    status = ctx.status()
    return {n: fetch(ctx, bufs[n], like[n]) for n in (bufs if witness else ["out"])}, status


def exp_table(n, top=1023, width=8.0):
    return np.rint(top * np.exp(-np.arange(n)[::-1] * width / n)).astype(np.int32)


ATTEND = [
    # lengths, heads, kv_heads, dim, bits, page, layout, gap, max_keys beyond the longest, soft_shift
    ([1], 1, 1, 8, 32, 1, "head", 0, 0, 16),
    ([17], 4, 4, 64, 32, 16, "head", 0, 0, 16),
    ([0, 1, 15, 16, 17, 33], 2, 2, 40, 32, 16, "token", 8, 5, 16),
    ([300, 0, 257, 256, 255], 8, 2, 128, 16, 64, "token", 0, 3, 16),
    ([130, 9], 1, 1, 4096, 32, 64, "head", 0, 0, 16),
    ([130, 9], 2, 1, 2048, 16, 24, "head", 8, 1, 20),
    ([1000, 77], 5, 1, 72, 32, 100, "head", 0, 0, 16),
    ([1000, 77], 7, 1, 80, 16, 7, "token", 0, 0, 1),
    ([333], 32, 2, 96, 32, 128, "head", 0, 2, 16),
    ([513, 700], 9, 3, 24, 16, 32, "head", 0, 0, 11),
    ([2600], 3, 1, 8, 16, 8, "head", 0, 0, 20),
    ([2049, 31], 24, 8, 120, 32, 48, "token", 0, 0, 16),
    ([640], 33, 1, 16, 32, 256, "head", 0, 0, 16),
    ([129], 12, 4, 256, 16, 16, "head", 0, 0, 16),
]


# rows too long for one block: every width of key rows, one to nine heads a key head, many short sequences beside long ones
ATTEND_LONG = [
    ([3001, 40, 2048], 8, 2, 128, 16, 32, "token", 0, 3, 16),
    ([5000], 2, 1, 64, 32, 24, "head", 0, 0, 16),
    ([4097, 1], 4, 4, 128, 32, 100, "head", 0, 0, 20),
    ([2500, 2499, 0, 7], 6, 2, 128, 32, 64, "head", 8, 1, 16),
    ([3000], 9, 1, 128, 16, 64, "head", 0, 0, 16),
    ([700, 600], 8, 1, 512, 16, 16, "token", 0, 0, 16),
    ([700, 601], 3, 1, 512, 32, 7, "head", 0, 0, 16),
    ([33, 500], 2, 1, 1024, 32, 16, "head", 0, 2, 16),
    ([40000, 3], 1, 1, 8, 32, 256, "head", 0, 0, 20),
    ([900] + [5, 0, 1, 17] * 20, 2, 2, 256, 32, 16, "head", 0, 0, 16),
    ([3, 0, 1, 2] * 66, 1, 1, 520, 32, 8, "head", 0, 1, 16),
]


def attend_setup(gctx, case, kind, seed=21):
    lens, H, KV, D, bits, page, layout, gap, more, soft_shift = case
    rng = np.random.default_rng(seed)
    P = sum(-(-n // page) for n in lens) + 2
    table = table_for(rng, P, lens, page)
    k, v = (Pool(rng, P, KV, page, D, bits, layout, gap, std=65536 if bits == 32 else 1024) for _ in range(2))
    q = np.rint(rng.normal(0, 65536, (len(lens), H, D))).astype(np.int32)
    shift = 16 + int(round(np.log2(D) / 2)) - (6 if bits == 16 else 0)
    if kind == "extreme":    # full range: keys and queries in two channels (their sum stays below 2^63), all values
        top = 1 << (bits - 1)
        k.raw[...] = 0
        k.raw[..., 3:5] = rng.choice([-top, top - 1, -1, 0, 1, 128, -128, 255], k.raw[..., 3:5].shape)
        v.raw[...] = rng.choice([-top, top - 1, -1, 0, 1], v.raw.shape)
        q[...] = 0
        q[..., 3:5] = rng.choice([-(1 << 31) + 1, (1 << 31) - 1, 127, -129, 0x7f7f7f80, -0x7f7f7f80], q[..., 3:5].shape)
        shift = 31 if bits == 32 else 20
    cache = make_cache(gctx, k, v, page, KV, D, bits)
    return rng, table, k, v, q, shift, cache


@pytest.mark.parametrize("case", ATTEND + ATTEND_LONG, ids=lambda x: str(x)[:60])
@pytest.mark.parametrize("kind", ["normal", "extreme"])
def test_attend(gctx, case, kind):
    lens, H, KV, D, bits, page, layout, gap, more, soft_shift = case
    rng, table, k, v, q, shift, cache = attend_setup(gctx, case, kind)
    n = 1 << 20
    exp, max_keys = exp_table(n, width=16.0), max(lens) + more
    want, status = plain_attend(k, v, table, lens, q, exp, 1 - n, page, shift, soft_shift, max_keys)
    gctx.status()
    got, seen = run_attend(gctx, cache, table, lens, q, exp, 1 - n, shift, soft_shift, max_keys, q_stride=H * D + 4)
    for name in want:
        assert np.array_equal(got[name], want[name]), name
    assert seen == status
    alone, _ = run_attend(gctx, cache, table, lens, q, exp, 1 - n, shift, soft_shift, max_keys, witness=False)
    assert np.array_equal(alone["out"], want["out"])


@pytest.mark.parametrize("case", ATTEND + ATTEND_LONG, ids=lambda x: str(x)[:60])
def test_attend_selected_pages(gctx, case):
    """Lists with holes: nothing selected, the partial page in the middle, a page twice, numbers outside the table."""
    lens, H, KV, D, bits, page, layout, gap, more, soft_shift = case
    rng, table, k, v, q, shift, cache = attend_setup(gctx, case, "normal")
    width = table.shape[1]
    n_select = min(9 if case in ATTEND else 60, width + 2)
    sel = rng.integers(-1, width + 1, (len(lens), KV, n_select)).astype(np.int32)
    sel[0, 0, 0] = (lens[0] - 1) // page
    n = 1 << 20
    exp, max_keys = exp_table(n, width=16.0), max(1, n_select * page - 3 + more)
    want, status = plain_attend(k, v, table, lens, q, exp, 1 - n, page, shift, soft_shift, max_keys, selected=sel)
    gctx.status()
    got, seen = run_attend(gctx, cache, table, lens, q, exp, 1 - n, shift, soft_shift, max_keys, selected=sel)
    for name in want:
        assert np.array_equal(got[name], want[name]), name
    assert seen == status


def test_attend_bad_pages_lengths_and_tables(gctx):
    from grape_b200 import decode
    case = ([70, 64, 90, 50], 4, 2, 32, 32, 16, "head", 0, 0, 16)
    rng, table, k, v, q, shift, cache = attend_setup(gctx, case, "normal")
    n = 1 << 20
    exp = exp_table(n, width=16.0)
    table[0, 1], table[1, :], table[2, 5] = -1, 10 ** 6, -7
    want, status = plain_attend(k, v, table, [70, 64, 90, 50], q, exp, 1 - n, 16, shift, 16, 64)   # 70 and 90 do not fit max_keys
    gctx.status()
    got, seen = run_attend(gctx, cache, table, [70, 64, 90, 50], q, exp, 1 - n, shift, 16, 64)
    for name in want:
        assert np.array_equal(got[name], want[name]), name
    assert seen == status == decode.STATUS_PLACE | decode.STATUS_EXP
    # lengths outside the table: cut, negative: empty
    want, _ = plain_attend(k, v, table, [0, 0, 96, 50], q, exp, 1 - n, 16, shift, 16, 96)
    got, seen = run_attend(gctx, cache, table, [-5, 0, 1 << 30, 50], q, exp, 1 - n, shift, 16, 96)
    assert seen & decode.STATUS_PLACE and all(np.array_equal(got[name], want[name]) for name in want)
    # an exp table that is too short, and one of zeros
    table = np.arange(24, dtype=np.int32).reshape(4, 6) % k.raw.shape[0]
    for exp, low in ((exp_table(500), -499), (np.zeros(1 << 20, np.int32), 1 - (1 << 20))):
        want, status = plain_attend(k, v, table, [70, 64, 90, 50], q, exp, low, 16, shift, 16, 96)
        got, seen = run_attend(gctx, cache, table, [70, 64, 90, 50], q, exp, low, shift, 16, 96)
        assert seen == status == decode.STATUS_EXP and all(np.array_equal(got[name], want[name]) for name in want)


def test_any_bound_of_columns_without_a_witness(gctx):
    """The largest max_keys: the call keeps no more than the table's columns."""
    from grape_b200 import decode
    case = ([1500, 900], 8, 2, 64, 32, 16, "head", 0, 0, 16)
    rng, table, k, v, q, shift, cache = attend_setup(gctx, case, "normal")
    n = 1 << 20
    exp = exp_table(n, width=16.0)
    want, status = plain_attend(k, v, table, [1500, 900], q, exp, 1 - n, 16, shift, 16, 1500)
    gctx.status()
    dt, dl, dq, de = (upload(gctx, a) for a in (table, np.array([1500, 900], np.int32), q, exp))
    out, total = gctx.upload(np.zeros(q.shape, np.int32)), gctx.upload(np.zeros(q.shape[:2], np.int64))
    decode.kv_attend(cache, dt, table.shape[1], 2, dl, dq, 8, decode.ExpTable(de, 1 - n, n), out, score_shift=shift,
                     max_keys=(1 << 31) - 1, d_sum=total)
    assert np.array_equal(fetch(gctx, out, want["out"]), want["out"])
    assert np.array_equal(fetch(gctx, total, want["sum"]), want["sum"])
    assert gctx.status() == status


def test_offsets_beyond_32_bits(gctx):
    """A cache of three far pages: 2 x 13 GB, elements beyond 2^32."""
    from grape_b200 import decode
    rng = np.random.default_rng(31)
    stride, page, D = (1 << 31) + 4096, 16, 64
    dk, dv = (gctx.alloc((2 * stride + page * D) * 2) for _ in range(2))
    cache = decode.KVCache(gctx, 3, page, 1, D, bits=16, k_shift=6, v_shift=6, d_k=dk, d_v=dv, strides=(stride, D * page, D))
    x = np.rint(rng.normal(0, 65536, (40, 3, D))).astype(np.int32)
    table, start, offsets = np.array([[2, 0, 1]], np.int32), np.zeros(1, np.int32), np.array([0, 40], np.int32)
    dx, dt, ds, do = (upload(gctx, a) for a in (x, table, start, offsets))
    decode.kv_append(cache, dt, 3, 1, ds, do, 40, dx.at(4 * D), dx.at(8 * D), k_stride=3 * D, v_stride=3 * D)
    k, v = (Pool(rng, 3, 1, page, D, 16) for _ in range(2))
    plain_append(k, v, None, table, start, offsets, x[:, :1], x[:, 1:2], x[:, 2:3], None, None, 0, 0, True, 6, 6, page)
    exp = exp_table(1 << 20, width=16.0)
    want, _ = plain_attend(k, v, table, [40], x[39:, :1], exp, 1 - (1 << 20), page, 13, 16, 40)
    got, status = run_attend(gctx, cache, table, [40], x[39:, :1], exp, 1 - (1 << 20), 13, 16, 40)
    assert status == 0 and all(np.array_equal(got[name], want[name]) for name in want)
    dk.free()
    dv.free()


# ---------------------------------------------------------------------------------- together
class Step:
    """A batch whose tokens are appended and attended step by step."""

    def __init__(self, ctx, seed, B=3, H=8, KV=2, D=64, page=16, bits=32, width=12):
        from grape_b200 import decode
        self.ctx, self.B, self.H, self.KV, self.D, self.page, self.width = ctx, B, H, KV, D, page, width
        rng = self.rng = np.random.default_rng(seed)
        P = B * width
        self.table = rng.permutation(P).astype(np.int32).reshape(B, width)
        self.k, self.v = (Pool(rng, P, KV, page, D, bits) for _ in range(2))
        self.bounds = np.zeros((P, KV, 2, D), self.k.dtype)
        self.sh = 6 if bits == 16 else 0
        self.cache = make_cache(ctx, self.k, self.v, page, KV, D, bits, self.sh, self.sh, self.bounds)
        ang = np.arange(width * page)[:, None] * 10000.0 ** (-np.arange(D // 2) / (D // 2))
        self.cos, self.sin = (np.rint(f(ang) * 65536).astype(np.int32) for f in (np.cos, np.sin))
        self.exp = exp_table(1 << 20, width=16.0)
        self.d = {n: upload(ctx, a) for n, a in (("table", self.table), ("cos", self.cos), ("sin", self.sin), ("exp", self.exp))}
        self.rotation = decode.Rotation(self.d["cos"], self.d["sin"], width * page, D)
        self.n_select, self.keys = 4, 4 * page
        shapes = {"start": (B,), "len": (B,), "offsets": (B + 1,), "q_out": (B * 40, H, D), "selected": (B, KV, 4), "out": (B, H, D),
                  "softmax": (B, H, self.keys), "x": (B * 40, (H + 2 * KV) * D)}
        self.like = {n: np.zeros(s, np.int32) for n, s in shapes.items()}
        self.d |= {n: ctx.upload(a) for n, a in self.like.items()}

    def put(self, name, a):
        a = np.ascontiguousarray(a, np.int32)
        self.ctx._check(self.ctx.lib.grape_h2d(self.ctx.handle, self.d[name].ptr, a.ctypes.data, a.nbytes))
        self.ctx.sync()

    def issue(self, tokens):
        """append, select, attend, on the buffers as they are (tokens rows of x in all, the last B of q_out are used)"""
        from grape_b200 import decode
        d, B, H, KV, D = self.d, self.B, self.H, self.KV, self.D
        row = (H + 2 * KV) * D
        decode.kv_append(self.cache, d["table"], self.width, B, d["start"], d["offsets"], tokens, d["x"].at(4 * H * D),
                         d["x"].at(4 * (H + KV) * D), rotation=self.rotation, d_q=d["x"], heads=H, d_q_out=d["q_out"], q_stride=row,
                         k_stride=row, v_stride=row)
        q = d["q_out"].at(4 * (tokens - B) * H * D)
        decode.kv_select(self.cache, d["table"], self.width, B, d["len"], q, H, self.n_select, d["selected"])
        decode.kv_attend(self.cache, d["table"], self.width, B, d["len"], q, H, decode.ExpTable(d["exp"], 1 - (1 << 20), 1 << 20), d["out"],
                         score_shift=19 - self.sh, max_keys=self.keys, d_selected=d["selected"], n_select=self.n_select,
                         d_softmax=d["softmax"])

    def want(self, x, start, new):
        H, KV, D = self.H, self.KV, self.D
        offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        rows = x.reshape(-1, H + 2 * KV, D)
        got, _ = plain_append(self.k, self.v, self.bounds, self.table, start, offsets, rows[:, :H], rows[:, H:H + KV], rows[:, H + KV:],
                              self.cos, self.sin, D, 16, True, self.sh, self.sh, self.page)
        lens = [s + n for s, n in zip(start, new)]
        q = got["q"][0][-self.B:]
        sel, _ = plain_select(self.bounds, self.table, lens, q, KV, self.page, self.n_select, 1)
        out, _ = plain_attend(self.k, self.v, self.table, lens, q, self.exp, 1 - (1 << 20), self.page, 19 - self.sh, 16, self.keys,
                              selected=sel, fill=0)
        return sel, out

    def rows(self, n):
        return np.rint(self.rng.normal(0, 65536, (n, (self.H + 2 * self.KV) * self.D))).astype(np.int32)


def one_step(s, start, new):
    x = s.rows(sum(new))
    s.put("x", x)
    s.put("start", start)
    s.put("offsets", np.concatenate([[0], np.cumsum(new)]))
    s.put("len", [a + n for a, n in zip(start, new)])
    s.put("softmax", s.like["softmax"])
    return x


@pytest.mark.parametrize("bits", [32, 16])
def test_prompt_then_tokens(gctx, bits):
    """Prompts of 40 tokens, then single tokens across page borders, on one cache."""
    s = Step(gctx, 5, bits=bits)
    start, new = [0, 0, 0], [40, 40, 40]
    gctx.status()
    for _ in range(12):
        x = one_step(s, start, new)
        s.issue(sum(new))
        if new[0] == 40:      # queries of the last B rows are those of the last sequence: only the cache matters here
            rows = x.reshape(-1, s.H + 2 * s.KV, s.D)
            plain_append(s.k, s.v, s.bounds, s.table, start, np.array([0, 40, 80, 120]), rows[:, :s.H], rows[:, s.H:s.H + s.KV],
                         rows[:, s.H + s.KV:], s.cos, s.sin, s.D, 16, True, s.sh, s.sh, s.page)
        else:
            sel, out = s.want(x, start, new)
            assert np.array_equal(fetch(gctx, s.d["selected"], sel), sel)
            assert np.array_equal(fetch(gctx, s.d["out"], out["out"]), out["out"])
            soft = fetch(gctx, s.d["softmax"], out["softmax"])
            assert np.array_equal(soft, out["softmax"])
        assert gctx.status() == 0
        start, new = [a + n for a, n in zip(start, new)], [1, 1, 1]


def test_captured_steps_replay_on_new_data():
    """One step captured from the context's stream and replayed with other inputs; two graphs share the workspace."""
    import grape_b200
    import torch
    ctx = grape_b200.Context(0)
    s, t = Step(ctx, 6), Step(ctx, 7, B=5, H=4, KV=4, D=32, bits=16)
    stream = torch.cuda.ExternalStream(ctx.stream)
    start = {s: [0] * s.B, t: [0] * t.B}
    for st in (s, t):
        for n in (30, 1):
            x = one_step(st, start[st], [n] * st.B)
            st.issue(n * st.B)
            rows = x.reshape(-1, st.H + 2 * st.KV, st.D)
            plain_append(st.k, st.v, st.bounds, st.table, start[st], np.arange(st.B + 1) * n, rows[:, :st.H], rows[:, st.H:st.H + st.KV],
                         rows[:, st.H + st.KV:], st.cos, st.sin, st.D, 16, True, st.sh, st.sh, st.page)
            start[st] = [a + n for a in start[st]]
    ctx.sync()
    graphs = {}
    for st in (s, t):
        one_step(st, start[st], [1] * st.B)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            st.issue(st.B)
        graphs[st] = g
    for _ in range(3):
        for st in (s, t):
            x = one_step(st, start[st], [1] * st.B)
            with torch.cuda.stream(stream):
                graphs[st].replay()
            ctx.sync()
            sel, out = st.want(x, start[st], [1] * st.B)
            assert np.array_equal(fetch(ctx, st.d["selected"], sel), sel)
            assert np.array_equal(fetch(ctx, st.d["out"], out["out"]), out["out"])
            start[st] = [a + 1 for a in start[st]]
    assert ctx.status() == 0
    del graphs
    ctx.close()


def test_captured_long_rows_replay_on_new_queries():
    """The three passes of long rows, and the choice of pages, captured together; two replays without waiting between."""
    import grape_b200
    import torch
    from grape_b200 import decode
    ctx = grape_b200.Context(0)
    case = ([2500, 2499, 0, 7], 6, 2, 128, 32, 64, "head", 8, 1, 16)
    rng, table, k, v, q, shift, cache = attend_setup(ctx, case, "normal")
    lens, H, KV, D, page, n, keys = case[0], 6, 2, 128, 64, 1 << 20, 2500
    exp = exp_table(n, width=16.0)
    bounds = np.stack([k.view.min(axis=2), k.view.max(axis=2)], axis=2).copy()
    cache = decode.KVCache(ctx, k.raw.shape[0], page, KV, D, d_k=cache.k, d_v=cache.v, d_bounds=upload(ctx, bounds), strides=k.strides)
    d = {name: upload(ctx, a) for name, a in (("table", table), ("len", np.array(lens, np.int32)), ("q", q), ("exp", exp),
                                              ("out", q), ("sel", np.zeros((4, KV, 5), np.int32)), ("sum", np.zeros((4, H), np.int64)))}

    def issue():
        decode.kv_select(cache, d["table"], table.shape[1], 4, d["len"], d["q"], H, 5, d["sel"])
        decode.kv_attend(cache, d["table"], table.shape[1], 4, d["len"], d["q"], H, decode.ExpTable(d["exp"], 1 - n, n), d["out"],
                         score_shift=shift, max_keys=keys, d_sum=d["sum"])

    issue()
    ctx.sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(ctx.stream)):
        issue()
    for seed in range(3):
        q = np.rint(np.random.default_rng(seed).normal(0, 65536, q.shape)).astype(np.int32)
        ctx._check(ctx.lib.grape_h2d(ctx.handle, d["q"].ptr, q.ctypes.data, q.nbytes))
        ctx.sync()
        with torch.cuda.stream(torch.cuda.ExternalStream(ctx.stream)):
            g.replay()
            g.replay()
        ctx.sync()
        sel, _ = plain_select(bounds, table, lens, q, KV, page, 5, 1)
        want, _ = plain_attend(k, v, table, lens, q, exp, 1 - n, page, shift, 16, keys)
        assert np.array_equal(fetch(ctx, d["sel"], sel), sel)
        assert np.array_equal(fetch(ctx, d["out"], want["out"]), want["out"]) and np.array_equal(fetch(ctx, d["sum"], want["sum"]), want["sum"])
    assert ctx.status() == 0
    del g
    ctx.close()


def test_a_capture_that_would_have_to_allocate_is_refused():
    import grape_b200
    import torch
    from grape_b200 import decode
    ctx = grape_b200.Context(0)
    cache = decode.KVCache(ctx, 4, 16, 1, 64)
    table = ctx.upload(np.zeros((1, 1 << 20), np.int32))
    zeros = ctx.upload(np.zeros(1 << 20, np.int32))
    stream = torch.cuda.ExternalStream(ctx.stream)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(grape_b200.GrapeError, match="outside the capture"):
        with torch.cuda.graph(g, stream=stream):
            decode.kv_select(cache, table, 1 << 20, 1, zeros, zeros, 1, 4, zeros)
    decode.kv_select(cache, table, 1 << 20, 1, zeros, zeros, 1, 4, zeros)     # the context still works
    assert ctx.status() == 0
    ctx.close()


def test_two_contexts_at_once():
    """Steps of two contexts interleaved without waiting for either; each has its own stream and workspace."""
    import grape_b200
    a, b = grape_b200.Context(0), grape_b200.Context(0)
    s, t = Step(a, 8), Step(b, 9, D=128, H=4, KV=1)
    xs = [one_step(st, [0] * st.B, [1] * st.B) for st in (s, t)]
    for _ in range(20):      # appending the same token again changes nothing
        s.issue(s.B)
        t.issue(t.B)
    for st, x in zip((s, t), xs):
        sel, out = st.want(x, [0] * st.B, [1] * st.B)
        assert np.array_equal(fetch(st.ctx, st.d["out"], out["out"]), out["out"])
        assert st.ctx.status() == 0
    a.close()
    b.close()


def test_the_workspace_takes_what_there_is():
    """Where twice the last workspace finds no room, the call gets what it needs."""
    import torch
    from grape_b200 import decode, host
    ctx = host.Context(0)
    width = (40 << 20, 50 << 20)                                  # 8 bytes a page of the table: 320 and 400 MB
    cache = decode.KVCache(ctx, 1, 1, 1, 8)
    dt, dl = ctx.alloc(width[1] * 4), ctx.upload(np.zeros(1, np.int32))
    dq, ds = ctx.upload(np.ones(8, np.int32)), ctx.upload(np.zeros(2, np.int32))
    torch.cuda.empty_cache()
    hold = torch.empty(torch.cuda.mem_get_info()[0] - (900 << 20), dtype=torch.uint8, device="cuda")
    for w in width:
        decode.kv_select(cache, dt, w, 1, dl, dq, 1, 2, ds)
        assert ctx.download(ds, 8, np.int32).tolist() == [-1, -1]
    with pytest.raises(host.GrapeError, match="workspace"):
        decode.kv_select(cache, dt, 1 << 30, 1, dl, dq, 1, 2, ds)
    assert ctx.status() == 0
    del hold
    torch.cuda.empty_cache()
    cache.close()
    ctx.close()


def test_empty_calls(gctx):
    from grape_b200 import decode
    cache = decode.KVCache(gctx, 1, 16, 1, 64)
    decode.kv_append(cache, None, 0, 0, None, None, 0, None, None)
    decode.kv_select(cache, None, 0, 0, None, None, 1, 1, None)
    decode.kv_attend(cache, None, 0, 0, None, None, 1, decode.ExpTable(upload(gctx, np.ones(1, np.int32)), 0, 1), None, score_shift=1, max_keys=1)
    zero = upload(gctx, np.zeros(4, np.int32))
    decode.kv_append(cache, zero, 1, 1, zero, zero, 0, None, None)      # a sequence that receives nothing
    assert gctx.status() == 0


def test_refusals_reach_the_user(gctx):
    import grape_b200
    from grape_b200 import decode
    cache = decode.KVCache(gctx, 1, 16, 1, 64)
    with pytest.raises(grape_b200.GrapeError, match="n_select"):
        decode.kv_select(cache, 1 << 20, 1, 1, 1 << 20, 1 << 20, 1, 0, 1 << 20)
    assert isinstance(C.string_at(gctx.lib.grape_ctx_error(gctx.handle)), bytes)
