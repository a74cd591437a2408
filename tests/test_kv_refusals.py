"""Refusals of the decode-step calls.  Arguments are checked before the context, so no GPU is needed."""
import ctypes as C

import pytest


def lib():
    import grape_b200
    return grape_b200._lib.load()


def cache(**change):
    from grape_b200 import decode
    f = dict(d_k=1 << 20, d_v=1 << 21, d_bounds=1 << 22, page_stride=2 * 16 * 64, head_stride=16 * 64, slot_stride=64, n_pages=9,
             page_size=16, kv_heads=2, head_dim=64, bits=32, k_shift=0, v_shift=0)
    f.update(change)
    return decode._Cache(**f)


CACHE_FAULTS = [
    (dict(bits=8), "bits"), (dict(head_dim=0), "head_dim"), (dict(head_dim=60), "head_dim"), (dict(head_dim=4104), "head_dim"),
    (dict(page_size=0), "page_size"), (dict(page_size=4097), "page_size"), (dict(kv_heads=0), "kv_heads"), (dict(n_pages=0), "n_pages"),
    (dict(n_pages=1 << 31), "n_pages"), (dict(slot_stride=68), "multiples of 8"), (dict(slot_stride=56), "smaller"),
    (dict(head_stride=32), "smaller"), (dict(page_stride=8), "smaller"), (dict(page_stride=1 << 61), "too large"),
    (dict(k_shift=31), "shifts"), (dict(v_shift=31), "shifts"),
]


def append(c, **change):
    from grape_b200 import decode
    f = dict(table=1 << 23, width=4, batch=3, start=1 << 24, offsets=1 << 25, tokens=10,
             rotation=decode._Rotation(1 << 26, 1 << 27, 100, 64, 16, 1), q=1 << 28, q_stride=4 * 64, heads=4, k=1 << 29, k_stride=128,
             v=1 << 30, v_stride=128, q_out=1 << 31, q_rem=None, k_rem=None, v_rem=None)
    f.update(change)
    r = f["rotation"]
    L = lib()
    rc = L.grape_kv_append(None, C.byref(c) if c is not None else None, f["table"], f["width"], f["batch"], f["start"], f["offsets"],
                           f["tokens"], C.byref(r) if r is not None else None, f["q"], f["q_stride"], f["heads"], f["k"], f["k_stride"],
                           f["v"], f["v_stride"], f["q_out"], f["q_rem"], f["k_rem"], f["v_rem"])
    return rc, L.grape_kv_error().decode()


def select(c, **change):
    f = dict(table=1 << 23, width=4, batch=3, len=1 << 24, q=1 << 28, q_stride=4 * 64, heads=4, n_select=3, recent=1, selected=1 << 29,
             bound=None)
    f.update(change)
    L = lib()
    rc = L.grape_kv_select(None, C.byref(c) if c is not None else None, *[f[n] for n in (
        "table", "width", "batch", "len", "q", "q_stride", "heads", "n_select", "recent", "selected", "bound")])
    return rc, L.grape_kv_error().decode()


def attend(c, witness=None, **change):
    f = dict(table=1 << 23, width=4, batch=3, len=1 << 24, selected=None, n_select=0, q=1 << 28, q_stride=4 * 64, heads=4, score_shift=19,
             exp=1 << 29, exp_low=-15, exp_len=16, soft_shift=16, max_keys=64, out=1 << 30)
    f.update(change)
    L = lib()
    rc = L.grape_kv_attend(None, C.byref(c) if c is not None else None, *[f[n] for n in (
        "table", "width", "batch", "len", "selected", "n_select", "q", "q_stride", "heads", "score_shift", "exp", "exp_low", "exp_len",
        "soft_shift", "max_keys", "out")], C.byref(witness) if witness is not None else None)
    return rc, L.grape_kv_error().decode()


def test_only_the_context_is_missing():
    for rc, text in (append(cache()), select(cache()), attend(cache())):
        assert rc == 1 and text == "null context"


@pytest.mark.parametrize("call", [append, select, attend])
@pytest.mark.parametrize("change, word", CACHE_FAULTS)
def test_cache_faults(call, change, word):
    rc, text = call(cache(**change))
    assert rc == 1 and word in text


@pytest.mark.parametrize("call", [append, select, attend])
def test_common_faults(call):
    assert call(None) == (1, "cache is null")
    assert "page table" in call(cache(), table=None)[1]
    assert "page table" in call(cache(), width=0)[1]
    assert call(cache(page_size=4096), width=1 << 20)[0] == 5     # table_width * page_size
    assert "multiple of 4" in call(cache(), q_stride=252)[1]      # shorter than a row
    assert "multiple of 4" in call(cache(), q_stride=258)[1]
    assert "16 bytes" in call(cache(), q=(1 << 28) + 4)[1]


def test_append_faults():
    from grape_b200.decode import _Rotation
    assert "without pages" in append(cache(d_k=None))[1]
    assert "without pages" in append(cache(d_v=None))[1]
    assert append(cache(d_bounds=None))[1] == "null context"      # bounds are optional here
    assert "16 bytes" in append(cache(d_v=(1 << 21) + 8))[1]
    for r, word in ((_Rotation(None, 1 << 27, 100, 64, 16, 1), "tables"), (_Rotation(1 << 26, 1 << 27, 100, 60, 16, 1), "dim"),
                    (_Rotation(1 << 26, 1 << 27, 100, 72, 16, 1), "dim"), (_Rotation(1 << 26, 1 << 27, 100, 64, 31, 1), "shift"),
                    (_Rotation(1 << 26, 1 << 27, 100, 64, 16, 2), "pairing")):
        rc, text = append(cache(), rotation=r)
        assert rc == 1 and word in text
    assert "shift" in append(cache(k_shift=15))[1]                # 16 + 15 > 30
    assert append(cache(), rotation=None)[1] == "null context"
    assert "start" in append(cache(), start=None)[1]
    assert "start" in append(cache(), offsets=None)[1]
    assert "keys" in append(cache(), k=None)[1]
    assert "values" in append(cache(), v_stride=64)[1]
    assert "without an output" in append(cache(), q_out=None)[1]
    assert "not given" in append(cache(), q=None)[1]
    assert append(cache(), q=None, q_out=None)[1] == "null context"
    assert "heads" in append(cache(), heads=0)[1]
    assert "16 bytes" in append(cache(), k_rem=(1 << 31) + 4)[1]
    assert append(cache(), tokens=1 << 31)[0] == 5


def test_select_faults():
    assert "bounds" in select(cache(d_bounds=None))[1]
    assert select(cache(d_k=None, d_v=None))[1] == "null context"  # keys are not read
    assert "multiple of kv_heads" in select(cache(), heads=3)[1]
    assert "n_select" in select(cache(), n_select=0)[1]
    assert "n_select" in select(cache(), n_select=(1 << 20) + 1)[1]
    assert "recent" in select(cache(), recent=4)[1]
    assert "lengths" in select(cache(), len=None)[1]
    assert "selected" in select(cache(), selected=None)[1]
    assert "8 bytes" in select(cache(), bound=(1 << 29) + 4)[1]


def test_attend_faults():
    from grape_b200.decode import _Witness
    assert "multiple of kv_heads" in attend(cache(), heads=5)[1]
    assert "score_shift" in attend(cache(), score_shift=32)[1]
    assert "soft_shift" in attend(cache(), soft_shift=0)[1]
    assert "soft_shift" in attend(cache(), soft_shift=21)[1]
    assert "max_keys" in attend(cache(), max_keys=0)[1]
    assert "max_keys" in attend(cache(), max_keys=1 << 31)[1]
    for change in (dict(exp=None), dict(exp_low=1), dict(exp_low=-16), dict(exp_len=0)):
        assert "exp table" in attend(cache(), **change)[1]
    assert "n_select" in attend(cache(), n_select=3)[1]
    assert "n_select" in attend(cache(), selected=1 << 29)[1]
    assert "lengths" in attend(cache(), len=None)[1]
    assert "output" in attend(cache(), out=None)[1]
    assert "16 bytes" in attend(cache(), witness=_Witness(d_score=(1 << 29) + 4))[1]
    assert "16 bytes" in attend(cache(), witness=_Witness(d_sum=(1 << 29) + 4))[1]
    assert attend(cache(), witness=_Witness())[1] == "null context"


def test_empty_batches_need_no_pointers():
    """A batch of no sequences is no error (the context alone is missing)."""
    nothing = dict(table=None, width=0, batch=0, q=None)
    assert append(cache(), start=None, offsets=None, k=None, v=None, q_out=None, **nothing)[1] == "null context"
    assert select(cache(), len=None, selected=None, **nothing)[1] == "null context"
    assert attend(cache(), len=None, out=None, **nothing)[1] == "null context"


def test_python_cache_checks():
    from grape_b200.decode import KVCache
    with pytest.raises(ValueError):
        KVCache(None, 1, 16, 1, 64, bits=8)
    with pytest.raises(ValueError):
        KVCache(None, 1, 16, 1, 64, strides=(1024, 1024, 64))


class NoGpu:
    """A context's memory without a GPU."""
    handle = None

    def __init__(self):
        self.lib, self.next = lib(), 1 << 20

    def alloc(self, nbytes):
        from grape_b200.host import DeviceBuffer
        buf = DeviceBuffer.__new__(DeviceBuffer)
        self.next += -(-nbytes // 256) * 256
        buf.ctx, buf.nbytes, buf.ptr = self, nbytes, self.next
        return buf

    def _check(self, rc):
        pass


def test_a_closed_cache_is_refused():
    """The memory of a cache that allocated it is gone with close(): the calls see a cache without pages."""
    from grape_b200.decode import KVCache
    own = KVCache(NoGpu(), 9, 16, 2, 64)
    assert append(own._struct)[1] == select(own._struct)[1] == attend(own._struct)[1] == "null context"
    own.close()
    own.close()
    assert append(own._struct)[1] == attend(own._struct)[1] == "cache without pages"
    assert select(own._struct)[1] == "cache without bounds"
    given = KVCache(NoGpu(), 9, 16, 2, 64, d_k=1 << 20, d_v=1 << 21, d_bounds=1 << 22)
    given.close()     # the caller's memory is still the caller's
    assert append(given._struct)[1] == select(given._struct)[1] == "null context"


@pytest.mark.parametrize("change, gens, word", [
    (dict(keys=1), 16384, "pad the columns"), (dict(rows=2, dim=4), 16384, "pad the columns"), (dict(scale=64), 16384, "scale"),
    (dict(softmax_len=64), 16384, "softmax_len"), (dict(exp_len=64), 16384, "exp_len"), (dict(), 1024, "scale of 65536"),
    (dict(softmax_len=1 << 18), 4096, "8192 generators"), (dict(exp_len=1 << 20), 4096, "16384 generators")])
def test_steps_that_cannot_be_proven(change, gens, word):
    """Shapes that an opening or a lookup would refuse in the middle of a proof are refused before it."""
    from types import SimpleNamespace

    import numpy as np
    from grape_b200.decode import StepProver, StepShape
    shape = StepShape(**{**dict(rows=1, keys=16, dim=64, exp_len=512, exp_low=-511), **change})
    with pytest.raises(ValueError, match=word):
        StepProver(None, shape, SimpleNamespace(n_gens=gens), None, np.zeros(shape.exp_len, np.int32))


def test_append_takes_no_more_work_than_a_call_can_end():
    """Sequences times pages of tokens: a million of each passes, sixteen million do not."""
    assert append(cache(), batch=1 << 20, tokens=1 << 20)[1] == "null context"
    rc, text = append(cache(), batch=1 << 24, tokens=1 << 24)
    assert rc == 5 and "too many sequences" in text
