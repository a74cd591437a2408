"""Calls of the decode step at the edges of what its documentation allows, against plain 64-bit integers."""
import warnings

import numpy as np
import pytest

from test_gpu_kv_decode import (WITNESS, Pool, exp_table, fetch, make_cache, plain_append, plain_attend, plain_select,
                                run_attend, table_for, upload)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------- append
def taken_sequences(offsets, tokens):
    """Sequences whose rows lie in the call's and, where offsets fall, behind those of the sequences before."""
    got, end = [], 0
    for b, (lo, hi) in enumerate(zip(offsets[:-1], offsets[1:])):
        if 0 <= lo <= hi <= tokens:
            if lo >= end:
                got.append(b)
            end = max(end, hi)
    return got


def scattered_offsets(n, tokens, seed):
    """Offsets of n sequences, a few of which fall, lie below 0 or behind the rows."""
    rng = np.random.default_rng(seed)
    o = np.sort(rng.integers(0, tokens + 1, n + 1))
    at = rng.choice(n + 1, 5, replace=False)
    o[at] = rng.integers(-50, tokens + 50, 5)
    return [int(x) for x in o]


OFFSETS = [
    # offsets, sequences that are appended
    ([-1, 10, 24], [1]),
    ([0, 24, 2, 24], [0]),
    ([0, 20, 2, 24], [0]),
    ([0, 10, 5, 24], [0]),
    ([8, 3, 3, 24], [1, 2]),
    ([0, 30, 10, 24], [2]),
    ([40, 50, 24], []),
    ([0, 8, 8, 16, 4, 24], [0, 1, 2]),
    ([0, 24, -(1 << 31), 24], [0]),
    ([0, (1 << 31) - 1, 8, 24], [2]),
    ([0, 6, 6, 24, 24], [0, 1, 2, 3]),
    ([5, 9, 20], [0, 1]),
    (scattered_offsets(40, 300, 1), None),
    (scattered_offsets(700, 900, 2), None),
    (scattered_offsets(700, 900, 3), None),
]


@pytest.mark.parametrize("offsets, want_taken", OFFSETS, ids=lambda x: str(x)[:30])
def test_append_with_bad_offsets(gctx, offsets, want_taken):
    """A sequence whose rows lie outside or run backwards is skipped and reported, wherever it stands; of sequences that
    share rows the first has them; all others are appended."""
    from grape_b200 import decode
    rng = np.random.default_rng(8)
    tokens = 24 if want_taken is not None else 300 if len(offsets) == 41 else 900
    taken = taken_sequences(offsets, tokens)
    assert want_taken is None or taken == want_taken
    B, KV, D, page = len(offsets) - 1, 2, 8, 8
    start = [(4 + 5 * b) % 11 for b in range(B)]
    ends = [s + max(0, min(hi, tokens) - max(lo, 0)) for s, lo, hi in zip(start, offsets[:-1], offsets[1:])]
    P = sum(-(-n // page) for n in ends) + 2
    table = table_for(rng, P, ends, page)
    k, v = (Pool(rng, P, KV, page, D, 32) for _ in range(2))
    bounds = np.stack([k.view.min(axis=2), k.view.max(axis=2)], axis=2).copy()
    x = rng.integers(-1000, 1000, (tokens, 2, KV, D)).astype(np.int32)
    cache = make_cache(gctx, k, v, page, KV, D, 32, bounds=bounds)
    dx, dt, ds, do = (upload(gctx, a) for a in (x, table, np.array(start, np.int32), np.array(offsets, np.int32)))
    rem = gctx.upload(np.full((tokens, KV, D), 5, np.int32))
    gctx.status()
    decode.kv_append(cache, dt, table.shape[1], B, ds, do, tokens, dx, dx.at(4 * KV * D), k_stride=2 * KV * D, v_stride=2 * KV * D,
                     d_k_rem=rem)
    whole = all(0 <= lo <= hi <= tokens for lo, hi in zip(offsets[:-1], offsets[1:]))
    assert gctx.status() == (0 if whole else decode.STATUS_PLACE)
    want = np.full((tokens, KV, D), 5, np.int32)
    for b in taken:
        plain_append(k, v, bounds, table[b:b + 1], [start[b]], offsets[b:b + 2], x[:, 0], x[:, 0], x[:, 1], None, None, 0, 0, True, 0, 0, page)
        want[offsets[b]:offsets[b + 1]] = 0
    assert np.array_equal(fetch(gctx, rem, want), want)
    assert np.array_equal(fetch(gctx, cache.k, k.raw), k.raw) and np.array_equal(fetch(gctx, cache.v, v.raw), v.raw)
    assert np.array_equal(fetch(gctx, cache.bounds, bounds), bounds)


@pytest.mark.parametrize("batch, bits, interleaved", [(4097, 32, True), (9001, 16, False)])
def test_append_to_very_many_sequences(gctx, batch, bits, interleaved):
    """None, one or two tokens a sequence, more sequences than a launch takes; one of the last runs outside its table."""
    from grape_b200 import decode
    rng = np.random.default_rng(batch)
    KV, D, page = 1, 16, 8
    new = rng.integers(0, 3, batch)
    new[-1], start = 1, rng.integers(0, 6, batch).astype(np.int32)
    start[-1] = 11                                             # its second page is not there
    offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    T, table = int(offsets[-1]), rng.permutation(batch).astype(np.int32).reshape(batch, 1)
    k, v = (Pool(rng, batch, KV, page, D, bits) for _ in range(2))
    x = rng.integers(-1000, 1000, (T, 2, KV, D)).astype(np.int32)
    cos, sin = (rng.integers(-65536, 65536, (12, D // 2)).astype(np.int32) for _ in range(2))
    cache = make_cache(gctx, k, v, page, KV, D, bits)
    dx, dt, ds, do, dc, dn = (upload(gctx, a) for a in (x, table, start, offsets, cos, sin))
    gctx.status()
    decode.kv_append(cache, dt, 1, batch, ds, do, T, dx, dx.at(4 * KV * D), k_stride=2 * KV * D, v_stride=2 * KV * D,
                     rotation=decode.Rotation(dc, dn, 12, D, interleaved=interleaved))
    assert gctx.status() == decode.STATUS_PLACE
    seq = np.repeat(np.arange(batch), new)[:-1]
    pos = start[seq] + np.arange(T - 1) - offsets[seq]
    idx = np.arange(D // 2)
    first, second = (2 * idx, 2 * idx + 1) if interleaved else (idx, idx + D // 2)
    key, c, s = x[:-1, 0, 0].astype(np.int64), cos[pos].astype(np.int64), sin[pos].astype(np.int64)
    turned = np.empty_like(key)
    turned[:, first], turned[:, second] = key[:, first] * c - key[:, second] * s, key[:, second] * c + key[:, first] * s
    k.view[table[seq, 0], 0, pos] = (turned + (1 << 15)) >> 16
    v.view[table[seq, 0], 0, pos] = x[:-1, 1, 0]
    assert np.array_equal(fetch(gctx, cache.k, k.raw), k.raw) and np.array_equal(fetch(gctx, cache.v, v.raw), v.raw)


# ---------------------------------------------------------------------------------- select
@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("heads, kv_heads, dim", [(4, 1, 3048), (3, 1, 3056), (8, 2, 3064), (2, 1, 4088), (4, 1, 4096)])
def test_select_with_wide_heads(gctx, heads, kv_heads, dim, bits):
    """Heads whose queries fill a block's default shared memory up to the last hundred bytes, and wider ones."""
    from grape_b200 import decode
    rng = np.random.default_rng(dim + bits)
    lens, page, n = [90, 33], 4, 5
    P = sum(-(-x // page) for x in lens) + 1
    table = table_for(rng, P, lens, page)
    bounds = np.sort(np.rint(rng.normal(0, 3000, (P, kv_heads, 2, dim))), axis=2).astype(np.int16 if bits == 16 else np.int32)
    q = np.rint(rng.normal(0, 65536, (2, heads, dim))).astype(np.int32)
    want, want_bound = plain_select(bounds, table, lens, q, kv_heads, page, n, 1)
    cache = decode.KVCache(gctx, P, page, kv_heads, dim, bits=bits, d_bounds=upload(gctx, bounds), d_k=0, d_v=0)
    dt, dl, dq = upload(gctx, table), upload(gctx, np.array(lens, np.int32)), upload(gctx, q)
    ds, db = gctx.upload(np.full(want.shape, 55, np.int32)), gctx.upload(np.full(want_bound.shape, 99, np.int64))
    gctx.status()
    decode.kv_select(cache, dt, table.shape[1], 2, dl, dq, heads, n, ds, d_bound=db)
    assert np.array_equal(fetch(gctx, ds, want), want) and np.array_equal(fetch(gctx, db, want_bound), want_bound)
    assert gctx.status() == 0


# ---------------------------------------------------------------------------------- attend
class SparseTable:
    """An exp table of which only a few entries are not zero."""

    def __init__(self, entries):
        self.entries = entries

    def __getitem__(self, at):
        return np.array([self.entries.get(int(i), 0) for i in at], np.int32)


@pytest.mark.parametrize("length, more", [(40, 0), (6000, 0), (6000, 1)])
def test_attend_with_the_longest_exp_table(gctx, length, more):
    """Arguments from -2^31 to 0: 2^31 + 1 entries, the last of them 2^31 entries behind the first."""
    from grape_b200 import decode
    rng = np.random.default_rng(length)
    D, page, low, size = 64, 16, -(1 << 31), (1 << 31) + 1
    table = table_for(rng, -(-length // page), [length], page)
    k, v = (Pool(rng, -(-length // page), 1, page, D, 32) for _ in range(2))
    k.raw[...] = 0
    k.raw[..., 0] = rng.choice([-1, -7, -1000000, low], k.raw.shape[:-1])
    k.raw[table[0, 0], 0, 3, 0] = 0                                  # the row's largest score
    q = np.zeros((1, 1, D), np.int32)
    q[0, 0, 0] = 1
    entries = {size - 1: 1000, size - 2: 900, size - 8: 500, size - 1000001: 77, 0: 3}
    want, status = plain_attend(k, v, table, [length], q, SparseTable(entries), low, page, 0, 16, length + more)
    assert status == 0 and want["exp_in"].min() == low
    exp = gctx.alloc(4 * size)
    gctx._check(gctx.lib.grape_dev_zero(gctx.handle, exp.ptr, 4 * size))
    for at, value in entries.items():
        one = np.array([value], np.int32)
        gctx._check(gctx.lib.grape_h2d(gctx.handle, exp.at(4 * at), one.ctypes.data, 4))
        gctx.sync()
    cache = make_cache(gctx, k, v, page, 1, D, 32)
    dt, dl, dq = upload(gctx, table), upload(gctx, np.array([length], np.int32)), upload(gctx, q)
    bufs = {n: gctx.upload(np.full(a.shape, 33, a.dtype)) for n, a in want.items()}
    gctx.status()
    decode.kv_attend(cache, dt, table.shape[1], 1, dl, dq, 1, decode.ExpTable(exp, low, size), bufs["out"], score_shift=0,
                     max_keys=length + more, **{"d_" + n: bufs[n] for n in WITNESS + ("sum", "out_rem")})
    for name, a in want.items():
        assert np.array_equal(fetch(gctx, bufs[name], a), a), name
    assert gctx.status() == 0
    exp.free()


@pytest.mark.parametrize("length", [70, 4000])
@pytest.mark.parametrize("missing", [-5, 0, 1, 16])
def test_columns_of_selected_pages_are_not_cut_without_a_word(gctx, length, missing):
    """A call whose max_keys is below the columns of the selected pages says so; its outputs are those of the columns before."""
    rng = np.random.default_rng(length)
    H, KV, D, page, n = 2, 1, 64, 16, 1 << 20
    pages = -(-length // page)
    n_select = min(pages, 150)
    table = table_for(rng, pages, [length], page)
    k, v = (Pool(rng, pages, KV, page, D, 32, std=65536) for _ in range(2))
    q = np.rint(rng.normal(0, 65536, (1, H, D))).astype(np.int32)
    selected = np.sort(rng.choice(pages - 1, n_select - 1, replace=False)).astype(np.int32)
    selected = np.append(selected, pages - 1).astype(np.int32).reshape(1, 1, n_select)
    exp, max_keys = exp_table(n, width=16.0), n_select * page - missing
    cache = make_cache(gctx, k, v, page, KV, D, 32)
    want, status = plain_attend(k, v, table, [length], q, exp, 1 - n, page, 19, 16, max_keys, selected=selected)
    gctx.status()
    with warnings.catch_warnings(record=True) as said:
        warnings.simplefilter("always")
        got, seen = run_attend(gctx, cache, table, [length], q, exp, 1 - n, 19, 16, max_keys, selected=selected)
    assert [str(w.message) for w in said] == ([f"max_keys {max_keys} cuts the {n_select * page} columns of the selected pages"] if missing > 0 else [])
    assert seen == status == 0 and all(np.array_equal(got[name], a) for name, a in want.items())
