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
import warnings
from dataclasses import dataclass

import numpy as np

from ._lib import CUT
from .host import FR_MODULUS as R
from .host import Context, Lookup, _p, decode_field, prove_matmul, reassemble_vectors
from .layer import FFNTrace, ProofError, log2ceil
from .layer_full import LayerProver, LayerShape

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
        if self._owned:      # no call may meet the addresses again
            self._struct.d_k = self._struct.d_v = self._struct.d_bounds = None
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
        ctx.handle, cache._ref, d_table, table_width, batch, d_start, d_offsets, tokens,
        rotation._ref if rotation is not None else None, d_q, heads * cache.head_dim if q_stride is None else q_stride, heads,
        d_k, row if k_stride is None else k_stride, d_v, row if v_stride is None else v_stride, d_q_out, d_q_rem,
        d_k_rem, d_v_rem))


def kv_select(cache: KVCache, d_table, table_width: int, batch: int, d_len, d_q, heads: int, n_select: int, d_selected,
              recent: int = 1, d_bound=None, q_stride: int | None = None):
    """``grape_kv_select``: the ``recent`` newest pages and those of the largest bounds, ``n_select`` per sequence
    and key head, ascending, -1 behind the last."""
    ctx = cache.ctx
    ctx._check(ctx.lib.grape_kv_select(ctx.handle, cache._ref, d_table, table_width, batch, d_len, d_q,
                                       heads * cache.head_dim if q_stride is None else q_stride, heads, n_select, recent,
                                       d_selected, d_bound))


def kv_attend(cache: KVCache, d_table, table_width: int, batch: int, d_len, d_q, heads: int, exp: ExpTable, d_out,
              score_shift: int, max_keys: int, soft_shift: int = 16, d_selected=None, n_select: int = 0, d_out_rem=None,
              d_score=None, d_score_rem=None, d_exp_in=None, d_exp_out=None, d_softmax=None, d_sum=None,
              q_stride: int | None = None):
    """``grape_kv_attend``: attention of one token per sequence over its cached positions, or over those of the
    selected pages, with the tensors of its proof (rows of ``max_keys`` columns).  Warns where ``max_keys`` cuts the
    columns of the selected pages, of which the newest come last."""
    ctx = cache.ctx
    w = _Witness(_p(d_score), _p(d_score_rem), _p(d_exp_in), _p(d_exp_out), _p(d_softmax), _p(d_sum), _p(d_out_rem))
    rc = ctx.lib.grape_kv_attend(ctx.handle, cache._ref, d_table, table_width, batch, d_len, d_selected,
                                 n_select, d_q, heads * cache.head_dim if q_stride is None else q_stride, heads,
                                 score_shift, exp.d_values, exp.low, exp.length, soft_shift, max_keys, d_out, C.byref(w))
    if rc == CUT:
        warnings.warn(ctx.lib.grape_kv_error().decode(), RuntimeWarning, stacklevel=2)
    else:
        ctx._check(rc)


# ----------------------------------------------------------------------------- proof of a step
@dataclass
class StepShape:
    """One key head of a step: the heads that share it, the (padded) columns, the head's channels and the scales.  rows, keys
    and dim are powers of two, rows * keys and rows * dim at least 16; the three lookups' lengths at least 128."""
    rows: int
    keys: int
    dim: int
    scale: int = 1 << 16             # softmax and output rescale, 2^soft_shift
    score_scale: int = 1 << 22       # 2^score_shift
    exp_low: int = -(1 << 20) + 1
    exp_len: int = 1 << 20
    softmax_len: int = 1 << 16       # range of the softmax rounding residual: at least twice the largest row sum


def pad_step(shape: StepShape, q, k, v, witness: dict) -> dict:
    """The tensors of :meth:`StepProver.prove_attention` from those of ``kv_attend``, all of n <= ``shape.keys`` columns: q
    [rows][dim], k and v [n][dim] (the cached rows of the columns), witness["score"], ["score_rem"], ["exp_in"],
    ["exp_out"], ["softmax"] [rows][n] and ["out"], ["out_rem"] [rows][dim].  A column behind the last has key, value,
    score and softmax zero and the exp table's first entry, which has to be zero for that."""
    n = witness["score"].shape[1]
    wide = lambda a, fill=0: np.pad(a, ((0, 0), (0, shape.keys - n)), constant_values=fill).astype(np.int32)
    rows = lambda a: np.pad(a, ((0, shape.keys - n), (0, 0))).astype(np.int32)
    return {"xq_q": np.asarray(q, np.int32), "xk_q": rows(k), "xv_q": np.ascontiguousarray(rows(v).T), "scores_q": wide(witness["score"]),
            "scores_rem": wide(witness["score_rem"]), "exp_in": wide(witness["exp_in"], shape.exp_low),
            "exp_out": wide(witness["exp_out"]), "softmax": wide(witness["softmax"]), "qkv_q": witness["out"].astype(np.int32),
            "qkv_rem": witness["out_rem"].astype(np.int32)}


class StepProver(LayerProver):
    """Proof of the attention of one new token over one key head, the same walk as a layer's (test/llm.cu:356-452) with
    the heads that share the key head for rows and the cached columns for keys: output remainder, softmax x V, the
    softmax relation, the exp mapping, the score remainder, Q K^T.  What is left are claims on the query, the keys
    and the values, for the proofs of the tokens that made them.

    What the walk does not bind, in a layer's proof either: ``exp_in`` to the scores and their row's maximum (any
    arguments pass whose values, softmax and output go with them), the score remainder to its range (a quotient one
    larger passes with a remainder ``score_scale`` smaller), and the claim of the softmax relation's range check to the
    softmax and the exp values it was computed from (of which the latter are opened at its point).  A verifier who needs
    those links has to make them from the tensors."""

    def __init__(self, ctx: Context, shape: StepShape, table, G_jacobian, exp_table):
        for name in ("rows", "keys", "dim"):
            if getattr(shape, name) < 1 or getattr(shape, name) & (getattr(shape, name) - 1):
                raise ValueError(f"{name} must be a power of two")
        exp_table = np.asarray(exp_table, np.int32)
        if exp_table.shape != (shape.exp_len,) or exp_table[0] != 0:
            raise ValueError("the exp table must have exp_len entries, the first of them zero")
        # an opening takes rows of 16 elements at least, and a lookup commits its multiplicities in rows of 16 sqrt(entries)
        if min(shape.rows * shape.keys, shape.rows * shape.dim) < 16:
            raise ValueError("rows * keys and rows * dim must be at least 16: pad the columns")
        for name in ("scale", "softmax_len", "exp_len"):
            entries = log2ceil(getattr(shape, name))
            if entries < 7:
                raise ValueError(f"{name} must be at least 128")
            if table.n_gens < 16 << entries // 2:
                raise ValueError(f"{name} of {getattr(shape, name)} needs a table of {16 << entries // 2} generators, not {table.n_gens}")
        self.step = shape
        self.ctx, self.table, self.G = ctx, table, G_jacobian
        self.shape = LayerShape(layer_num=1, tokens=shape.keys, dim=shape.dim, ffn=shape.dim, scale1=shape.scale, npoints=shape.dim)
        self.c = decode_field(ctx.random_fr(1))[0]
        self.rs = Lookup(ctx, -(shape.scale // 2), shape.scale)
        self.softmax_range = Lookup(ctx, 0, shape.softmax_len)
        self.exp = Lookup(ctx, shape.exp_low, shape.exp_len, exp_table)

    def _n(self, size: int) -> int:
        """Row length (over 16) of a tensor's commitments and openings."""
        return max(1, min(size, self.table.n_gens) // 16)

    def _padded(self, ints, n: int, fill: int = 0):
        """int32 tensor -> Fr tensor of at least n elements (a lookup takes no fewer queries than its table has entries)."""
        flat = np.ascontiguousarray(ints, dtype=np.int32).reshape(-1)
        if flat.size < n:
            flat = np.concatenate([flat, np.full(n - flat.size, fill, np.int32)])
        return self._fr(flat)

    def _remainder(self, ints, point, trace, name):
        """Range check of a remainder at a point of its own, tied to the tensor by an opening; returns the opening at
        ``point`` (of the tensor without its padding)."""
        keep, size = self._padded(ints, self.rs.n)
        work, A = self._clone(keep, size * 32), self._alloc(size * 32)
        v = self._draw(log2ceil(size))
        trace.lookups += 1
        with self._phase(trace, "lookup"):
            claim, _ = self.rs.prove(work, size, A, v, table=self.table, msm_size=min(self._n(size), self._n(self.rs.n)))
        if self._open(keep, size, v, self._n(size), trace)["result"] != claim:
            raise ProofError(f"{name}: opening of the remainder disagrees with the lookup claim")
        value = self._open(keep, size, list(point) + [0] * (log2ceil(size) - len(point)), self._n(size), trace)["result"]
        self._release(keep, work, A)
        return value

    def prove_attention(self, t: dict) -> FFNTrace:
        ctx, s = self.ctx, self.step
        lR, lS, lD = log2ceil(s.rows), log2ceil(s.keys), log2ceil(s.dim)
        ssize, osize = s.rows * s.keys, s.rows * s.dim
        trace = FFNTrace()
        # ---- output: quotient opened, remainder looked up
        out, _ = self._fr(t["qkv_q"])
        e2 = self._draw(log2ceil(osize))
        out_value = self._open(out, osize, e2, self._n(osize), trace)["result"]
        self._release(out)
        value = (out_value * s.scale + self._remainder(t["qkv_rem"], e2, trace, "qkv")) % R
        trace.values["out"], trace.values["out_point"] = out_value, list(e2)
        # ---- softmax x V, V transposed [dim][keys]
        soft, _ = self._fr(t["softmax"])
        soft_keep = self._clone(soft, ssize * 32)
        xv, _ = self._fr(t["xv_q"])
        e3 = self._draw(lS)
        trace.matmuls += 1
        with self._phase(trace, "matmul"):
            soft_cl, v_cl, _, _ = prove_matmul(ctx, soft, xv, 1, s.rows, s.dim, s.keys, e2, e3, value)
        e2, e3 = reassemble_vectors(e2, e3, lR, lS, lD)
        trace.values["v"], trace.values["v_point"] = v_cl, list(e3)
        if self._open(soft_keep, ssize, e2, self._n(ssize), trace)["result"] != soft_cl:
            raise ProofError("softmax x V: opening of the softmax disagrees")
        self._release(soft, xv)
        # ---- softmax relation: 2 scale e - (2 o - 1) rowsum(e) in [0, softmax_len)
        e_out, _ = self._fr(t["exp_out"])
        rsize = max(ssize, self.softmax_range.n)
        resid, tmp, A = self._alloc(rsize * 32), self._alloc(ssize * 32), self._alloc(rsize * 32)
        ctx._check(ctx.lib.grape_dev_zero(ctx.handle, resid.ptr, rsize * 32))
        consts = ctx.fr_upload([2 * s.scale, 2, -1])
        ctx.fr_binary("scale", e_out, consts, resid, ssize)
        ctx.fr_binary("scale", soft_keep, consts.at(32), soft_keep, ssize)
        ctx.fr_binary("add_scalar", soft_keep, consts.at(64), soft_keep, ssize)
        ctx.fr_rowsum(e_out, tmp, s.rows, s.keys)
        ctx.fr_binary("mul", soft_keep, tmp, soft_keep, ssize)
        ctx.fr_binary("sub", resid, soft_keep, resid, ssize)
        e1 = self._draw(log2ceil(rsize))
        trace.lookups += 1
        with self._phase(trace, "lookup"):
            self.softmax_range.prove(resid, rsize, A, e1, table=self.table, msm_size=min(self._n(rsize), self._n(self.softmax_range.n)))
        self._open(e_out, ssize, e1[:log2ceil(ssize)], self._n(ssize), trace)    # the padding's variables come last
        self._release(resid, tmp, A, soft_keep, e_out)
        consts.free()
        # ---- exp mapping, padded with the table's first pair
        e_in, esize = self._padded(t["exp_in"], self.exp.n, s.exp_low)
        e_out, _ = self._padded(t["exp_out"], self.exp.n)
        e1 = self._draw(log2ceil(esize))
        work, A = self._alloc(esize * 32), self._alloc(esize * 32)
        trace.lookups += 1
        with self._phase(trace, "lookup"):
            lookup_value, _ = self.exp.prove_pairs(e_in, e_out, esize, work, A, e1, table=self.table,
                                                   msm_size=min(self._n(esize), self._n(self.exp.n)))
        in_value = self._open(e_in, esize, e1, self._n(esize), trace)["result"]
        out_value = self._open(e_out, esize, e1, self._n(esize), trace)["result"]
        if lookup_value != (in_value + out_value * self.exp.r) % R:
            raise ProofError("exp: lookup claim disagrees with the two openings")
        self._release(e_in, e_out, work, A)
        # ---- scores (quotient evaluated, remainder opened, as a layer's) and Q K^T
        sc, _ = self._fr(t["scores_q"])
        sc_rem, _ = self._fr(t["scores_rem"])
        e1 = self._draw(log2ceil(ssize))
        score_value = ctx.fr_eval(sc, ssize, e1)
        score_value = (score_value * s.score_scale + self._open(sc_rem, ssize, e1, self._n(ssize), trace)["result"]) % R
        self._release(sc, sc_rem)
        xq, _ = self._fr(t["xq_q"])
        xk, _ = self._fr(t["xk_q"])
        e2 = self._draw(lD)
        trace.matmuls += 1
        with self._phase(trace, "matmul"):
            q_cl, k_cl, _, _ = prove_matmul(ctx, xq, xk, 1, s.rows, s.keys, s.dim, e1, e2, score_value)
        e1, e2 = reassemble_vectors(e1, e2, lR, lD, lS)
        self._release(xq, xk)
        trace.values.update({"q": q_cl, "q_point": e1, "k": k_cl, "k_point": e2})
        return trace
