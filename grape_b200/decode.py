"""Attention of generated tokens over a paged key-value cache, in the integers that the provers take.

``layer_full.synthesize_layer`` makes the tensors of a whole prompt; here are those of one new token per
sequence, on the GPU: ``kv_append`` turns keys and queries by their position and writes keys and values to
the cache, ``kv_select`` chooses the pages whose keys can matter, ``kv_attend`` computes scores, softmax and
output with every quotient and remainder.  ``StepProver`` proves the attention of such a step.

Device tensors are :class:`DeviceBuffer` objects or raw device addresses, on the context's stream; every
call is asynchronous, and what it finds outside the cache, the rotation or the exp table is reported by
``Context.status`` (bits ``STATUS_*``).
"""
from __future__ import annotations

import ctypes as C

from .host import Context, _p

#: a quotient did not fit its type and was stored as the nearest value
STATUS_RANGE = 8
#: a length, position or page outside the cache, its table or the rotation was skipped
STATUS_PLACE = 16
#: a score further behind its row's maximum than the exp table reaches, or a row whose sum is zero
STATUS_EXP = 32


class _Cache(C.Structure):
    _fields_ = [("d_k", C.c_void_p), ("d_v", C.c_void_p), ("d_bounds", C.c_void_p), ("page_stride", C.c_uint64),
                ("head_stride", C.c_uint64), ("slot_stride", C.c_uint64), ("n_pages", C.c_uint32),
                ("page_size", C.c_uint32), ("kv_heads", C.c_uint32), ("head_dim", C.c_uint32), ("bits", C.c_uint32),
                ("k_shift", C.c_uint32), ("v_shift", C.c_uint32)]


class _Rotation(C.Structure):
    _fields_ = [("d_cos", C.c_void_p), ("d_sin", C.c_void_p), ("positions", C.c_uint32), ("dim", C.c_uint32),
                ("shift", C.c_uint32), ("interleaved", C.c_uint32)]


class _Witness(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("d_score", "d_score_rem", "d_exp_in", "d_exp_out", "d_softmax", "d_sum", "d_out_rem")]


class KVCache:
    """Pages of keys and values of one layer.  Element (page, head, slot, channel) lies at ``strides`` =
    (page, head, slot) elements; the default is dense [n_pages][kv_heads][page_size][head_dim].  The memory is
    allocated (zeroed) unless ``d_k`` and ``d_v`` give it; ``d_bounds`` is [n_pages][kv_heads][2][head_dim] in the
    cache's type, ``bounds=False`` leaves it out where pages are never selected."""

    def __init__(self, ctx: Context, n_pages: int, page_size: int, kv_heads: int, head_dim: int, bits: int = 32,
                 k_shift: int = 0, v_shift: int = 0, d_k=None, d_v=None, d_bounds=None, strides=None, bounds: bool = True):
        if bits not in (16, 32):
            raise ValueError("bits must be 16 or 32")
        self.ctx = ctx
        self.n_pages, self.page_size, self.kv_heads, self.head_dim, self.bits = n_pages, page_size, kv_heads, head_dim, bits
        self.k_shift, self.v_shift = k_shift, v_shift
        self._owned = []
        nbytes = n_pages * kv_heads * page_size * head_dim * bits // 8
        if d_k is None and d_v is None:
            if strides is not None:
                raise ValueError("strides describe memory that is given")
            d_k, d_v = self._zeros(nbytes), self._zeros(nbytes)
            if bounds and d_bounds is None:
                d_bounds = self._zeros(2 * n_pages * kv_heads * head_dim * bits // 8)
        self.k, self.v, self.bounds = d_k, d_v, d_bounds
        page, head, slot = strides if strides is not None else (kv_heads * page_size * head_dim, page_size * head_dim, head_dim)
        self._struct = _Cache(_p(d_k) or None, _p(d_v) or None, _p(d_bounds) or None, page, head, slot, n_pages, page_size,
                              kv_heads, head_dim, bits, k_shift, v_shift)
        self._ref = C.byref(self._struct)

    def _zeros(self, nbytes: int):
        buf = self.ctx.alloc(nbytes)
        self.ctx._check(self.ctx.lib.grape_dev_zero(self.ctx.handle, buf.ptr, nbytes))
        self._owned.append(buf)
        return buf

    def close(self):
        for b in self._owned:
            b.free()
        self._owned = []


class Rotation:
    """Cosines and sines, int32 [positions][dim / 2] at scale 2^shift, of the first ``dim`` channels; pairs are
    neighbours (``interleaved``, LLaMA's complex pairs) or ``dim / 2`` apart."""

    def __init__(self, d_cos, d_sin, positions: int, dim: int, shift: int = 16, interleaved: bool = True):
        self.d_cos, self.d_sin = d_cos, d_sin    # kept alive
        self._struct = _Rotation(_p(d_cos) or None, _p(d_sin) or None, positions, dim, shift, int(bool(interleaved)))
        self._ref = C.byref(self._struct)


class ExpTable:
    """``length`` int32 values of the exp mapping from argument ``low`` on, as ``host.Lookup`` proves it."""

    def __init__(self, d_values, low: int, length: int):
        self.d_values, self.low, self.length = d_values, low, length


def kv_append(cache: KVCache, d_table, table_width: int, batch: int, d_start, d_offsets, tokens: int, d_k, d_v, rotation=None,
              d_q=None, heads: int = 0, d_q_out=None, d_q_rem=None, d_k_rem=None, d_v_rem=None, q_stride: int | None = None,
              k_stride: int | None = None, v_stride: int | None = None):
    """``grape_kv_append``: sequence b, which holds d_start[b] tokens, receives rows d_offsets[b] .. d_offsets[b+1]-1
    of keys and values; queries are turned alike into ``d_q_out``.  Row strides default to dense."""
    ctx, row = cache.ctx, cache.kv_heads * cache.head_dim
    ctx._check(ctx.lib.grape_kv_append(
        ctx.handle, cache._ref, _p(d_table), table_width, batch, _p(d_start), _p(d_offsets), tokens,
        rotation._ref if rotation is not None else None, _p(d_q), heads * cache.head_dim if q_stride is None else q_stride, heads,
        _p(d_k), row if k_stride is None else k_stride, _p(d_v), row if v_stride is None else v_stride, _p(d_q_out), _p(d_q_rem),
        _p(d_k_rem), _p(d_v_rem)))


def kv_select(cache: KVCache, d_table, table_width: int, batch: int, d_len, d_q, heads: int, n_select: int, d_selected,
              recent: int = 1, d_bound=None, q_stride: int | None = None):
    """``grape_kv_select``: the ``recent`` newest pages and those of the largest bounds, ``n_select`` per sequence
    and key head, ascending, -1 behind the last."""
    ctx = cache.ctx
    ctx._check(ctx.lib.grape_kv_select(ctx.handle, cache._ref, _p(d_table), table_width, batch, _p(d_len), _p(d_q),
                                       heads * cache.head_dim if q_stride is None else q_stride, heads, n_select, recent,
                                       _p(d_selected), _p(d_bound)))


def kv_attend(cache: KVCache, d_table, table_width: int, batch: int, d_len, d_q, heads: int, exp: ExpTable, d_out,
              score_shift: int, max_keys: int, soft_shift: int = 16, d_selected=None, n_select: int = 0, d_out_rem=None,
              d_score=None, d_score_rem=None, d_exp_in=None, d_exp_out=None, d_softmax=None, d_sum=None,
              q_stride: int | None = None):
    """``grape_kv_attend``: attention of one token per sequence over its cached positions, or over those of the
    selected pages, with the tensors of its proof (rows of ``max_keys`` columns)."""
    ctx = cache.ctx
    w = _Witness(_p(d_score), _p(d_score_rem), _p(d_exp_in), _p(d_exp_out), _p(d_softmax), _p(d_sum), _p(d_out_rem))
    ctx._check(ctx.lib.grape_kv_attend(ctx.handle, cache._ref, _p(d_table), table_width, batch, _p(d_len), _p(d_selected),
                                       n_select, _p(d_q), heads * cache.head_dim if q_stride is None else q_stride, heads,
                                       score_shift, _p(exp.d_values), exp.low, exp.length, soft_shift, max_keys, _p(d_out),
                                       C.byref(w)))
