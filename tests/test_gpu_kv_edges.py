"""Calls of the decode step at the edges of what its documentation allows, against plain 64-bit integers."""
import numpy as np
import pytest

from test_gpu_kv_decode import fetch, plain_select, table_for, upload

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
