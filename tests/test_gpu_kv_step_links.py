"""Which tensors the proof of a generated token's attention ties together, and which it does not."""
import numpy as np
import pytest

from test_gpu_kv_proof import evaluate, prover, step  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def finish(p):
    p.release_pool()
    p.table.close()


def test_the_exp_values_are_opened_at_the_point_of_the_softmax_relation(gctx, step):  # noqa: F811
    shape, t, exp = step
    p = prover(gctx, shape, exp, 7)
    points, opened = [], []
    prove, open_ = p.softmax_range.prove, p._open

    def record_prove(resid, size, A, v, **more):
        points.append(list(v))
        return prove(resid, size, A, v, **more)

    def record_open(buf, size, e, N, trace):
        got = open_(buf, size, e, N, trace)
        opened.append((size, list(e), got["result"]))
        return got

    p.softmax_range.prove, p._open = record_prove, record_open
    p.prove_attention(t)
    point = points[0][:int(np.log2(t["exp_out"].size))]
    assert (t["exp_out"].size, point, evaluate(gctx, t["exp_out"], point)) in opened
    finish(p)


def proven(gctx, shape, exp, t, seed):
    p = prover(gctx, shape, exp, seed)
    trace = p.prove_attention(t)
    for name, tensor in (("q", t["xq_q"]), ("k", t["xk_q"]), ("v", t["xv_q"]), ("out", t["qkv_q"])):
        assert trace.values[name] == evaluate(gctx, tensor, trace.values[name + "_point"]), name
    finish(p)


def test_a_score_and_its_remainder_may_be_shifted_together(gctx, step):  # noqa: F811
    """The score remainder is opened, its range is not checked: the documentation says so."""
    shape, t, exp = step
    t = {n: a.copy() for n, a in t.items()}
    t["scores_q"][1, 7] += 1
    t["scores_rem"][1, 7] -= shape.score_scale
    assert abs(int(t["scores_rem"][1, 7])) > shape.score_scale // 2
    proven(gctx, shape, exp, t, 8)


def test_exp_arguments_are_not_tied_to_the_scores(gctx, step):  # noqa: F811
    """The arguments of other columns, with the values, softmax and output that go with them: the documentation says so."""
    shape, t, exp = step
    t = {n: a.copy() for n, a in t.items()}
    for n in ("exp_in", "exp_out", "softmax"):
        t[n] = np.ascontiguousarray(t[n][:, ::-1])
    acc = t["softmax"].astype(np.int64) @ t["xv_q"].astype(np.int64).T
    quotient = (acc + shape.scale // 2) // shape.scale
    assert not np.array_equal(quotient, t["qkv_q"])
    t["qkv_q"], t["qkv_rem"] = quotient.astype(np.int32), (acc - quotient * shape.scale).astype(np.int32)
    proven(gctx, shape, exp, t, 9)


@pytest.mark.parametrize("rows, cached, keys, dim, exp_len, softmax_len", [
    (1, 1, 16, 16, 128, 128), (16, 1, 1, 1, 512, 128), (2, 1, 8, 8, 512, 128), (1, 200, 256, 64, 512, 4096), (8, 300, 512, 64, 512, 8192),
    (1, 16, 16, 4096, 128, 1024), (4096, 1, 1, 1, 128, 128)])
def test_the_smallest_steps_and_lopsided_ones(gctx, rows, cached, keys, dim, exp_len, softmax_len):
    """A first token, one head, one channel, many heads: every claim that is left holds."""
    from grape_b200 import decode
    rng = np.random.default_rng(rows + keys + dim)
    q, k, v = (np.rint(rng.normal(0, 64, s)).astype(np.int64) for s in ((rows, dim), (cached, dim), (cached, dim)))
    exp = np.rint(7 * np.exp(-np.arange(exp_len)[::-1] * 9 / exp_len)).astype(np.int32)
    exp[0] = 0
    acc = q @ k.T
    score = (acc + 256) >> 9
    exp_in = np.maximum(score - score.max(axis=1, keepdims=True), 1 - exp_len)
    exp_out = exp[exp_in - (1 - exp_len)].astype(np.int64)
    total = exp_out.sum(axis=1, keepdims=True)
    assert 2 * total.max() <= softmax_len
    softmax = ((exp_out << 8) + total // 2) // total
    product = softmax @ v
    out = (product + 128) >> 8
    shape = decode.StepShape(rows=rows, keys=keys, dim=dim, scale=1 << 8, score_scale=1 << 9, exp_low=1 - exp_len, exp_len=exp_len,
                             softmax_len=softmax_len)
    t = decode.pad_step(shape, q, k, v, {"score": score, "score_rem": acc - (score << 9), "exp_in": exp_in, "exp_out": exp_out,
                                         "softmax": softmax, "out": out, "out_rem": product - (out << 8)})
    proven(gctx, shape, exp, t, 11)
