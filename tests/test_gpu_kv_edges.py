"""Calls of the decode step at the edges of what its documentation allows, against plain 64-bit integers."""
import numpy as np
import pytest

from test_gpu_kv_decode import WITNESS, Pool, fetch, make_cache, plain_attend, plain_select, table_for, upload

pytestmark = pytest.mark.gpu


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
