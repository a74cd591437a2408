"""What outlives what: memory of lookups, caches and their contexts."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def free_bytes():
    import torch
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


def some_lookups(ctx):
    from grape_b200.host import Lookup
    return [Lookup(ctx, -(1 << 19), 1 << 20), Lookup(ctx, 1 - (1 << 20), 1 << 20, np.arange(1 << 20, dtype=np.int32))]


@pytest.mark.parametrize("context_first", [True, False])
def test_a_lookup_gives_its_memory_back(context_first):
    """About 230 MB of two lookups, whichever goes first, the context or they."""
    import grape_b200
    warm = grape_b200.Context(0)
    for lookup in some_lookups(warm):
        lookup.close()
    before = free_bytes()
    for _ in range(3):
        ctx = grape_b200.Context(0)
        lookups = some_lookups(ctx)
        assert before - free_bytes() > 200 << 20
        if context_first:
            ctx.close()
        for lookup in lookups:
            lookup.close()
            lookup.close()      # a second time does nothing
        ctx.close()
    assert before - free_bytes() < 64 << 20
    warm.close()


def test_a_lookup_is_proven_while_others_come_and_go(gctx):
    """Lookups of one context are destroyed in any order beside one that is in use."""
    import grape_b200
    from grape_b200.host import Lookup
    rng = np.random.default_rng(3)
    first, kept, last = (Lookup(gctx, 0, 256) for _ in range(3))
    first.close()
    n = 1024
    s = gctx.upload(rng.integers(0, 256, n).astype(np.int32))
    fr, A = gctx.alloc(n * 32), gctx.alloc(n * 32)
    gctx.fr_from_i32(s, n, fr)
    keep = gctx.clone(fr, n * 32)
    last.close()
    v = [int(x) for x in rng.integers(1, 1 << 60, 10)]
    claim, _ = kept.prove(fr, n, A, v)
    assert claim == gctx.fr_eval(keep, n, v)
    kept.close()
    with pytest.raises(grape_b200.GrapeError):
        kept.prove(fr, n, A, v)
    assert gctx.status() == 0
