"""A generated token's attention from the cache to its proof: append, attend, prove; every claim that is left equals the
tensors' multilinear evaluation, and a witness that was tampered with breaks a check."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

SHIFT, EXP_LEN, HEADS, DIM, PAGE, TOKENS = 8, 512, 4, 32, 16, 50


@pytest.fixture(scope="module")
def step(gctx):
    """4 heads on one key head over 50 cached tokens, the last of them the new one; columns padded to 64."""
    from grape_b200 import decode
    rng = np.random.default_rng(41)
    ctx = gctx
    cache = decode.KVCache(ctx, 5, PAGE, 1, DIM)
    table = np.array([[3, 0, 4, 1]], np.int32)
    x = np.rint(rng.normal(0, 64, (TOKENS, HEADS + 2, DIM))).astype(np.int32)
    ang = np.arange(TOKENS)[:, None] * 10000.0 ** (-np.arange(DIM // 2) / (DIM // 2))
    cos, sin = (np.rint(f(ang) * (1 << SHIFT)).astype(np.int32) for f in (np.cos, np.sin))
    exp = np.rint(7 * np.exp(-np.arange(EXP_LEN)[::-1] / 60.0)).astype(np.int32)
    d = {n: ctx.upload(a) for n, a in (("x", x), ("table", table), ("cos", cos), ("sin", sin), ("exp", exp), ("start", np.zeros(1, np.int32)),
                                       ("off", np.array([0, TOKENS], np.int32)), ("len", np.array([TOKENS], np.int32)))}
    row = (HEADS + 2) * DIM
    like = {"q": np.zeros((TOKENS, HEADS, DIM), np.int32), "out": np.zeros((1, HEADS, DIM), np.int32),
            "out_rem": np.zeros((1, HEADS, DIM), np.int32)}
    like |= {n: np.zeros((1, HEADS, TOKENS), np.int32) for n in ("score", "score_rem", "exp_in", "exp_out", "softmax")}
    buf = {n: ctx.upload(a) for n, a in like.items()}
    ctx.status()
    decode.kv_append(cache, d["table"], 4, 1, d["start"], d["off"], TOKENS, d["x"].at(4 * HEADS * DIM), d["x"].at(4 * (HEADS + 1) * DIM),
                     rotation=decode.Rotation(d["cos"], d["sin"], TOKENS, DIM, shift=SHIFT), d_q=d["x"], heads=HEADS, d_q_out=buf["q"],
                     q_stride=row, k_stride=row, v_stride=row)
    q_last = buf["q"].at(4 * (TOKENS - 1) * HEADS * DIM)
    decode.kv_attend(cache, d["table"], 4, 1, d["len"], q_last, HEADS, decode.ExpTable(d["exp"], 1 - EXP_LEN, EXP_LEN), buf["out"],
                     score_shift=9, soft_shift=SHIFT, max_keys=TOKENS, d_out_rem=buf["out_rem"], d_score=buf["score"],
                     d_score_rem=buf["score_rem"], d_exp_in=buf["exp_in"], d_exp_out=buf["exp_out"], d_softmax=buf["softmax"])
    assert ctx.status() == 0
    got = {n: ctx.download(buf[n], a.nbytes, dtype=np.int32).reshape(a.shape) for n, a in like.items()}
    pages = 5 * PAGE * DIM
    k, v = (ctx.download(b, pages * 4, dtype=np.int32).reshape(5, PAGE, DIM)[table[0]].reshape(-1, DIM)[:TOKENS] for b in (cache.k, cache.v))
    shape = decode.StepShape(rows=HEADS, keys=64, dim=DIM, scale=1 << SHIFT, score_scale=1 << 9, exp_low=1 - EXP_LEN, exp_len=EXP_LEN,
                             softmax_len=1024)
    tensors = decode.pad_step(shape, got["q"][-1], k, v, {n: a[0] for n, a in got.items() if n != "q"})
    return shape, tensors, exp


def prover(gctx, shape, exp, seed):
    import grape_b200 as g
    from grape_b200 import decode, workloads as wl
    gens = wl.make_generators(gctx, 1024, seed=90)
    table = g.GeneratorTable(gctx, gens, 8, 1)
    gctx.seed(seed)
    return decode.StepProver(gctx, shape, table, gens[0], exp)


def evaluate(ctx, ints, point):
    flat = np.ascontiguousarray(ints, np.int32).reshape(-1)
    d = ctx.upload(flat)
    fr = ctx.alloc(flat.size * 32)
    ctx.fr_from_i32(d, flat.size, fr)
    return ctx.fr_eval(fr, flat.size, point)


def test_relations_of_the_witness(step):
    """The padded tensors satisfy the relations that the proof is about."""
    shape, t, exp = step
    q, k, v = (t[n].astype(np.int64) for n in ("xq_q", "xk_q", "xv_q"))
    assert np.array_equal(q @ k.T, t["scores_q"].astype(np.int64) * shape.score_scale + t["scores_rem"])
    assert np.array_equal(exp[t["exp_in"] - shape.exp_low], t["exp_out"])
    total = t["exp_out"].sum(axis=1, keepdims=True).astype(np.int64)
    resid = 2 * shape.scale * t["exp_out"].astype(np.int64) - (2 * t["softmax"].astype(np.int64) - 1) * total
    assert resid.min() >= 0 and resid.max() < shape.softmax_len
    assert np.array_equal(t["softmax"].astype(np.int64) @ v.T, t["qkv_q"].astype(np.int64) * shape.scale + t["qkv_rem"])


def test_step_is_proven_and_its_claims_hold(gctx, step):
    shape, t, exp = step
    p = prover(gctx, shape, exp, 5)
    trace = p.prove_attention(t)
    assert trace.matmuls == 2 and trace.lookups == 3
    for name, tensor in (("q", t["xq_q"]), ("k", t["xk_q"]), ("v", t["xv_q"]), ("out", t["qkv_q"])):
        assert trace.values[name] == evaluate(gctx, tensor, trace.values[name + "_point"]), name
    p.release_pool()
    p.table.close()


@pytest.mark.parametrize("name", ["softmax", "scores_q", "exp_out", "qkv_rem", "xq_q"])
def test_a_tampered_step_is_rejected(gctx, step, name):
    import grape_b200 as g
    from grape_b200.layer import ProofError
    shape, t, exp = step
    t = dict(t)
    t[name] = t[name].copy()
    t[name].reshape(-1)[5] += 1 if t[name].reshape(-1)[5] < 100 else -1
    p = prover(gctx, shape, exp, 6)
    with pytest.raises((g.GrapeError, ProofError)):
        p.prove_attention(t)
    gctx.status()
    p.release_pool()
    p.table.close()


def test_shapes_that_are_refused(gctx, step):
    from grape_b200 import decode
    shape, _, exp = step
    for change in (dict(rows=3), dict(keys=50), dict(dim=24)):
        with pytest.raises(ValueError, match="power of two"):
            decode.StepProver(gctx, decode.StepShape(**{**shape.__dict__, **change}), None, None, exp)
    with pytest.raises(ValueError, match="first of them zero"):
        decode.StepProver(gctx, shape, None, None, exp + 1)
