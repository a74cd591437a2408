"""Measured cases of the decode step's operators over a paged key-value cache, in the prover's integers:
appending keys and values with their position rotation, selecting pages by the bounds of their keys, and the
attention of one new token with every tensor its proof needs.

All values are integers at scale 2^16 (activations, rotations, softmax), products are brought back by a
rounded division by a power of two, and the remainders of those divisions are outputs too: the provers
range-check them.  So every output is a whole number and has to be equal.
"""
import math

import numpy as np
import torch

own = False

SCALE_BITS = 16           # activations, rotation tables and softmax are integers at scale 2^16
EXP_LEN = 1 << 20         # entries of the exp table, the layer prover's length
EXP_LOW = 1 - EXP_LEN     # its lowest argument; the highest is 0, a row's maximum
INT_MIN = -(1 << 63)


def listed():
    return [
        # one new token of the single-head layer that the layer prover proves (dim 4096): latency
        dict(name="append one token, one head of 4096", op="append", batch=1, new_low=1, new_high=1, start=2047, heads=1,
             kv_heads=1, dim=4096, rot=4096, bits=32, page=64, interleaved=True, layout="head", remainders=True),
        # a batch of sequences that each add a token to a 16-bit cache
        dict(name="append 64 tokens, 32 heads on 8, 16 bits", op="append", batch=64, new_low=1, new_high=1, start=4000,
             heads=32, kv_heads=8, dim=128, rot=128, bits=16, page=64, interleaved=False, layout="token", remainders=True),
        # the prompt of the layer prover: 2048 tokens of dim 4096, all remainders for the proof
        dict(name="append a prompt of 2048, one head of 4096", op="append", batch=1, new_low=2048, new_high=2048, start=0,
             heads=1, kv_heads=1, dim=4096, rot=4096, bits=32, page=64, interleaved=True, layout="head", remainders=True),
        # ragged prompts behind cached prefixes, nothing to prove yet
        dict(name="append ragged prompts, 32 heads on 8", op="append", batch=7, new_low=37, new_high=3001, start=811, heads=32,
             kv_heads=8, dim=128, rot=128, bits=32, page=48, interleaved=True, layout="head", remainders=False),
        # one sequence, short cache: latency
        dict(name="select 8 of 64 pages", op="select", batch=1, len_low=1021, len_high=1021, heads=8, kv_heads=8, dim=64,
             bits=32, page=16, select=8, recent=1, bounds=True),
        # long caches of a batch
        dict(name="select 64 of 2048 pages, 16 long caches", op="select", batch=16, len_low=100003, len_high=131072, heads=32,
             kv_heads=8, dim=128, bits=32, page=64, select=64, recent=2, bounds=True),
        # the smallest attention: a few cached tokens
        dict(name="attend 17 keys, 4 heads of 64", op="attend", batch=1, len_low=17, len_high=17, heads=4, kv_heads=4, dim=64,
             bits=32, page=16, layout="head", select=0),
        # one token of the layer prover's model over its 2048-token context
        dict(name="attend 2048 keys, one head of 4096", op="attend", batch=1, len_low=2048, len_high=2048, heads=1, kv_heads=1,
             dim=4096, bits=32, page=64, layout="head", select=0),
        # a ragged batch with shared key heads
        dict(name="attend 32 ragged caches, 32 heads on 8", op="attend", batch=32, len_low=301, len_high=4099, heads=32,
             kv_heads=8, dim=128, bits=32, page=64, layout="head", select=0),
        # few sequences, long caches of 16 bits: the split over the length
        dict(name="attend 2 caches of 100000, 16 bits", op="attend", batch=2, len_low=90001, len_high=100000, heads=16,
             kv_heads=4, dim=128, bits=16, page=32, layout="token", select=0),
        # the pages that select chose
        dict(name="attend 64 selected pages of 16 caches", op="attend", batch=16, len_low=30011, len_high=32768, heads=32,
             kv_heads=8, dim=128, bits=32, page=64, layout="head", select=64),
        # the largest: every head has its own keys
        dict(name="attend 8 caches of 8000, 32 heads of 128", op="attend", batch=8, len_low=7601, len_high=8000, heads=32,
             kv_heads=32, dim=128, bits=32, page=64, layout="head", select=0),
    ]


def draw(rng):
    """One more case of the ranges above."""
    def log_int(low, high):
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    op = rng.choice(["append", "select", "attend", "attend"])
    heads, kv_heads, dim = rng.choice([(1, 1, 4096), (1, 1, 2048), (4, 4, 64), (8, 8, 80), (8, 2, 96), (8, 1, 128), (16, 2, 128),
                                       (32, 8, 128), (32, 32, 128), (12, 12, 64), (14, 2, 64), (16, 16, 72), (8, 4, 256), (24, 8, 120)])
    bits = rng.choice([16, 32])
    page = rng.choice([8, 16, 24, 32, 48, 64, 100, 128, 256])
    layout = rng.choice(["head", "token"])
    if op == "append":
        batch = log_int(1, 64)
        rows = max(1, 8_000_000 // ((heads + 2 * kv_heads) * dim * batch))
        high = log_int(1, min(4096, rows))
        rot = rng.choice([dim, dim, dim // 2 // 8 * 8, 0])
        return dict(op=op, batch=batch, new_low=rng.randint(1, high), new_high=high, start=log_int(1, 8000) - 1, heads=heads,
                    kv_heads=kv_heads, dim=dim, rot=rot, bits=bits, page=page, interleaved=rng.choice([True, False]),
                    layout=layout, remainders=rng.choice([True, False]))
    batch = log_int(1, 32)
    if op == "select":
        most = min(4096, 60_000_000 // (batch * kv_heads * dim * 2))
        pages = log_int(2, max(2, most))
        high = rng.randint((pages - 1) * page + 1, pages * page)
        select = log_int(1, max(1, min(pages, 256)))
        return dict(op=op, batch=batch, len_low=rng.randint(1, high), len_high=high, heads=heads, kv_heads=kv_heads, dim=dim,
                    bits=bits, page=page, select=select, recent=rng.randint(0, min(4, select)), bounds=rng.choice([True, False]))
    high = log_int(1, min(100000, max(16, min(200_000_000 // (batch * kv_heads * dim), 12_000_000 // (batch * heads)))))
    pages = -(-high // page)
    select = log_int(1, pages) if pages > 4 and rng.random() < 0.35 else 0
    return dict(op=op, batch=batch, len_low=rng.randint(1, high), len_high=high, heads=heads, kv_heads=kv_heads, dim=dim,
                bits=bits, page=page, layout=layout, select=select)


# ---------------------------------------------------------------------------------------------- inputs
def ragged(n, low, high):
    """n lengths between low and high, the first of them high."""
    return [high - (high - low) * (i * 618 % 1000) // 1000 for i in range(n)]


def lengths(case):
    return ragged(case["batch"], case["len_low"], case["len_high"])


def shift_of(case):
    """What a 16-bit cache divides its keys and values by (in bits): they stay within a few thousand."""
    return 6 if case["bits"] == 16 else 0


def score_bits(case):
    """Division of the scores: the scale of one operand and the root of the head size, less the cache's own shift."""
    return SCALE_BITS + int(round(math.log2(case["dim"]) / 2)) - shift_of(case)


def normal(gen, shape, std, device):
    return torch.round(torch.randn(shape, generator=gen, device=device) * std).to(torch.int32)


def paged(gen, case, n_pages, device, std):
    """A pool of pages, [n_pages][kv_heads][page][dim] by index; `layout` says which of heads and slots is outer in memory."""
    P, H, S, D = n_pages, case["kv_heads"], case["page"], case["dim"]
    dtype = torch.int16 if case["bits"] == 16 else torch.int32
    shape = (P, H, S, D) if case.get("layout", "head") == "head" else (P, S, H, D)
    t = normal(gen, shape, std, device).to(dtype)
    return t if case.get("layout", "head") == "head" else t.permute(0, 2, 1, 3)


def page_table(gen, case, tokens, device):
    """Every sequence's pages, scattered over the pool: [batch][width] (-1 behind a sequence's last page), and the pool's size."""
    counts = [-(-n // case["page"]) for n in tokens]
    width, total = max(counts), sum(counts)
    order = torch.randperm(total + 3, generator=gen, device=device)[:total].to(torch.int32)
    c = torch.tensor(counts, device=device)
    at = torch.arange(width, device=device)[None, :]
    table = torch.where(at < c[:, None], order[(torch.cumsum(c, 0) - c)[:, None].add(at).clamp(max=total - 1)], -1)
    return table.to(torch.int32).contiguous(), total + 3


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(int(seed))
    unit = float(1 << SCALE_BITS)
    small = unit / (1 << shift_of(case))
    B, H, KV, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    st = {"case": case}
    if case["op"] == "append":
        new = ragged(B, case["new_low"], case["new_high"])
        start = [max(0, case["start"] - 29 * b) for b in range(B)]
        st["tokens"] = T = sum(new)
        st["table"], st["n_pages"] = page_table(gen, case, [a + n for a, n in zip(start, new)], device)
        st["start"] = torch.tensor(start, dtype=torch.int32, device=device)
        st["offsets"] = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device=device)
        # one fused projection: queries, keys and values of a token lie behind one another
        st["qkv"] = normal(gen, (T, (H + 2 * KV) * D), unit, device)
        st["k"], st["v"] = (paged(gen, case, st["n_pages"], device, small) for _ in range(2))
        st["bounds"] = torch.stack([st["k"].amin(dim=2), st["k"].amax(dim=2)], dim=2).contiguous()
        st["positions"] = max(a + n for a, n in zip(start, new))
        half = case["rot"] // 2
        angle = torch.arange(st["positions"], device=device, dtype=torch.float64)[:, None] * \
            torch.pow(10000.0, -torch.arange(half, device=device, dtype=torch.float64) / max(half, 1))[None, :]
        st["cos"], st["sin"] = (torch.round(f(angle) * unit).to(torch.int32).contiguous() for f in (torch.cos, torch.sin))
        st["q_out"] = torch.zeros((T, H, D), dtype=torch.int32, device=device)
        if case["remainders"]:
            st["q_rem"] = torch.zeros_like(st["q_out"])
            st["k_rem"], st["v_rem"] = (torch.zeros((T, KV, D), dtype=torch.int32, device=device) for _ in range(2))
    else:
        n = lengths(case)
        st["len"] = torch.tensor(n, dtype=torch.int32, device=device)
        st["table"], st["n_pages"] = page_table(gen, case, n, device)
        st["q"] = normal(gen, (B, H, D), unit, device)
        if case["op"] == "select":
            # the keys themselves are not read: a page's bounds are those of `page` draws around a page's own mean
            shape = (st["n_pages"], KV, 1, D)
            dtype = torch.int16 if case["bits"] == 16 else torch.int32
            mean = torch.randn(shape, generator=gen, device=device) * small * 0.5
            spread = (0.5 + torch.rand((st["n_pages"], KV, 2, D), generator=gen, device=device)) * small * math.sqrt(math.log(case["page"] + 1))
            st["bounds"] = torch.round(mean + torch.tensor([-1.0, 1.0], device=device)[:, None] * spread).to(dtype).contiguous()
            st["selected"] = torch.zeros((B, KV, case["select"]), dtype=torch.int32, device=device)
            if case["bounds"]:
                st["bound"] = torch.zeros((B, KV, st["table"].shape[1]), dtype=torch.int64, device=device)
        else:
            st["k"], st["v"] = (paged(gen, case, st["n_pages"], device, small) for _ in range(2))
            # the layer prover's kind of table: exp over 16 units of the score's scale, the maximum at 0
            arg = torch.arange(EXP_LOW, 1, device=device, dtype=torch.float64)
            st["exp"] = torch.round(1023.0 * torch.exp(arg / unit)).to(torch.int32)
            keys = max(n)
            if case["select"]:
                pages = (st["len"].to(torch.int64) + case["page"] - 1) // case["page"]
                st["selected"] = pick(gen, pages, KV, case["select"], st["table"].shape[1], device)
                keys = case["select"] * case["page"]
            st["keys"] = keys
            for name in ("score", "score_rem", "exp_in", "exp_out", "softmax"):
                st[name] = torch.zeros((B, H, keys), dtype=torch.int32, device=device)
            st["sum"] = torch.zeros((B, H), dtype=torch.int64, device=device)
            st["out"], st["out_rem"] = (torch.zeros((B, H, D), dtype=torch.int32, device=device) for _ in range(2))
    if own:
        handles(st)
    torch.cuda.synchronize()
    return st


def pick(gen, pages, kv_heads, n, width, device):
    """Random distinct pages of every sequence, its newest among them, in ascending order, -1 behind the last."""
    B = pages.shape[0]
    key = torch.rand((B, kv_heads, width), generator=gen, device=device)
    at = torch.arange(width, device=device)
    key = torch.where(at[None, None] == pages[:, None, None] - 1, 2.0, key)
    key = torch.where(at[None, None] < pages[:, None, None], key, -1.0)
    got = torch.sort(key, dim=2, descending=True, stable=True)[1][:, :, :n]
    got = torch.where(torch.arange(got.shape[2], device=device)[None, None] < pages[:, None, None], got, width)
    got = torch.sort(got, dim=2)[0]
    got = torch.where(got == width, -1, got)
    return torch.nn.functional.pad(got, (0, n - got.shape[2]), value=-1).to(torch.int32).contiguous()


_contexts = {}


def handles(st):
    """The context, cache and tables that a program keeps."""
    from grape_b200 import Context
    from grape_b200.decode import ExpTable, KVCache, Rotation
    case = st["case"]
    if "ctx" not in _contexts:
        _contexts["ctx"] = Context(0)
    ctx = _contexts["ctx"]
    k, v = (st[n].data_ptr() if n in st else 0 for n in ("k", "v"))
    strides = st["k"].stride()[:3] if "k" in st else None
    st["cache"] = KVCache(ctx, st["n_pages"], case["page"], case["kv_heads"], case["dim"], bits=case["bits"],
                          k_shift=shift_of(case), v_shift=shift_of(case), d_k=k, d_v=v,
                          d_bounds=st["bounds"].data_ptr() if "bounds" in st else 0, strides=strides)
    if case["op"] == "append":
        st["rotation"] = Rotation(st["cos"].data_ptr(), st["sin"].data_ptr(), positions=st["positions"], dim=case["rot"],
                                  shift=SCALE_BITS, interleaved=case["interleaved"])
    elif case["op"] == "attend":
        st["table_exp"] = ExpTable(st["exp"].data_ptr(), EXP_LOW, EXP_LEN)


# ---------------------------------------------------------------------------------------------- a pass
def run(st):
    if own:
        return run_own(st)
    return {"append": plain_append, "select": plain_select, "attend": plain_attend}[st["case"]["op"]](st)


def at(st, name):
    return st[name].data_ptr() if name in st else None


def run_own(st):
    from grape_b200.decode import kv_append, kv_attend, kv_select
    case = st["case"]
    B, H, KV, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    table, width = st["table"].data_ptr(), st["table"].shape[1]
    if case["op"] == "append":
        q, row = st["qkv"].data_ptr(), (H + 2 * KV) * D
        kv_append(st["cache"], table, width, B, at(st, "start"), at(st, "offsets"), st["tokens"], q + 4 * H * D,
                  q + 4 * (H + KV) * D, rotation=st["rotation"], d_q=q, heads=H, d_q_out=at(st, "q_out"), d_q_rem=at(st, "q_rem"),
                  d_k_rem=at(st, "k_rem"), d_v_rem=at(st, "v_rem"), q_stride=row, k_stride=row, v_stride=row)
        return {n: st[n] for n in ("k", "v", "bounds", "q_out", "q_rem", "k_rem", "v_rem") if n in st}
    if case["op"] == "select":
        kv_select(st["cache"], table, width, B, at(st, "len"), at(st, "q"), H, case["select"], at(st, "selected"),
                  recent=case["recent"], d_bound=at(st, "bound"))
        return {n: st[n] for n in ("selected", "bound") if n in st}
    kv_attend(st["cache"], table, width, B, at(st, "len"), at(st, "q"), H, st["table_exp"], at(st, "out"),
              score_shift=score_bits(case), soft_shift=SCALE_BITS, max_keys=st["keys"], d_selected=at(st, "selected"),
              n_select=case["select"], d_out_rem=at(st, "out_rem"), d_score=at(st, "score"), d_score_rem=at(st, "score_rem"),
              d_exp_in=at(st, "exp_in"), d_exp_out=at(st, "exp_out"), d_softmax=at(st, "softmax"), d_sum=at(st, "sum"))
    return {n: st[n] for n in ("out", "out_rem", "score", "score_rem", "exp_in", "exp_out", "softmax", "sum")}


def divide(x, bits):
    """Rounded quotient by 2^bits and its remainder."""
    q = (x + ((1 << bits) >> 1)) >> bits
    return q, x - (q << bits)


def rotate(x, cos, sin, rot, interleaved):
    """[tokens][heads][dim] at the product of the two scales; cos, sin: [tokens][rot/2]."""
    x = x.to(torch.int64)
    c, s = cos.to(torch.int64)[:, None], sin.to(torch.int64)[:, None]
    rest = x[..., rot:] << SCALE_BITS
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).reshape(x.shape[:-1] + (rot,))
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def plain_append(st):
    case, T = st["case"], st["tokens"]
    H, KV, D, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    t = torch.arange(T, device=st["qkv"].device)
    seq = torch.searchsorted(st["offsets"].to(torch.int64), t, right=True) - 1
    pos = st["start"].to(torch.int64)[seq] + t - st["offsets"].to(torch.int64)[seq]
    page, slot = st["table"].to(torch.int64)[seq, pos // ps], pos % ps
    q, k, v = st["qkv"].split([H * D, KV * D, KV * D], dim=1)
    cos, sin = st["cos"][pos], st["sin"][pos]
    top = (1 << (case["bits"] - 1)) - 1
    q_out, q_rem = divide(rotate(q.reshape(T, H, D), cos, sin, case["rot"], case["interleaved"]), SCALE_BITS)
    key, k_rem = divide(rotate(k.reshape(T, KV, D), cos, sin, case["rot"], case["interleaved"]), SCALE_BITS + shift_of(case))
    val, v_rem = divide(v.reshape(T, KV, D).to(torch.int64), shift_of(case))
    key = key.clamp(-top - 1, top).to(st["k"].dtype)
    st["k"][page, :, slot] = key
    st["v"][page, :, slot] = val.clamp(-top - 1, top).to(st["v"].dtype)
    # bounds: over the keys written since a page's slot 0 was written
    fresh = torch.zeros(st["n_pages"], dtype=torch.int64, device=t.device).scatter_add_(0, page, (slot == 0).to(torch.int64)) > 0
    fresh = fresh[:, None, None]
    where = page[:, None, None].expand(T, KV, D)
    new = [torch.full((st["n_pages"], KV, D), f, dtype=torch.int32, device=t.device).scatter_reduce_(0, where, key.to(torch.int32), how)
           for f, how in ((top, "amin"), (-top - 1, "amax"))]
    low, high = st["bounds"][:, :, 0].to(torch.int32), st["bounds"][:, :, 1].to(torch.int32)
    st["bounds"][:, :, 0] = torch.where(fresh, new[0], torch.minimum(low, new[0])).to(st["k"].dtype)
    st["bounds"][:, :, 1] = torch.where(fresh, new[1], torch.maximum(high, new[1])).to(st["k"].dtype)
    out = {"k": st["k"], "v": st["v"], "bounds": st["bounds"], "q_out": q_out.to(torch.int32)}
    if case["remainders"]:
        out |= {"q_rem": q_rem.to(torch.int32), "k_rem": k_rem.to(torch.int32), "v_rem": v_rem.to(torch.int32)}
    return out


def plain_select(st):
    case = st["case"]
    B, H, KV, D, n = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["select"]
    width = st["table"].shape[1]
    pages = (st["len"].to(torch.int64) + case["page"] - 1) // case["page"]
    i = torch.arange(width, device=pages.device)
    valid = (i[None] < pages[:, None])[:, None]
    b = st["bounds"][st["table"].to(torch.int64).clamp(min=0)].to(torch.int64)        # [B][W][KV][2][D]
    q = st["q"].to(torch.int64).reshape(B, 1, KV, H // KV, D)
    bound = torch.maximum(q * b[:, :, :, None, 0], q * b[:, :, :, None, 1]).sum(-1).amax(-1).transpose(1, 2)
    key = torch.where((i[None] >= pages[:, None] - case["recent"])[:, None], (1 << 63) - 1, bound)
    key = torch.where(valid, key, INT_MIN)
    got = torch.sort(key, dim=2, descending=True, stable=True)[1][:, :, :n]
    got = torch.where(torch.arange(got.shape[2], device=got.device)[None, None] < pages[:, None, None], got, width)
    got = torch.sort(got, dim=2)[0]
    got = torch.nn.functional.pad(torch.where(got == width, -1, got), (0, n - got.shape[2]), value=-1)
    out = {"selected": got.to(torch.int32)}
    if case["bounds"]:
        out["bound"] = torch.where(valid, bound, 0)
    return out


def plain_attend(st):
    case = st["case"]
    B, H, KV, D, ps, keys = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"], st["keys"]
    j = torch.arange(keys, device=st["q"].device)
    n = st["len"].to(torch.int64)
    table = st["table"].to(torch.int64)
    if case["select"]:
        logical = st["selected"].to(torch.int64)[:, :, j // ps]                       # [B][KV][keys]
        token = logical * ps + j % ps
        valid = (logical >= 0) & (token < n[:, None, None])
    else:
        logical = (j // ps)[None, None].expand(B, KV, keys)
        valid = (j[None, None] < n[:, None, None]).expand(B, KV, keys)
    page = torch.gather(table, 1, logical.clamp(min=0).reshape(B, KV * keys)).reshape(B, KV, keys).clamp(min=0)
    head = torch.arange(KV, device=j.device)[None, :, None]
    k, v = (st[name][page, head, (j % ps)[None, None]].to(torch.float64) for name in ("k", "v"))
    # products of these integers and all their partial sums stay far below 2^53: exact in 64-bit floating point
    q = st["q"].reshape(B, KV, H // KV, D).to(torch.float64)
    acc = torch.matmul(q, k.transpose(2, 3)).to(torch.int64)
    valid = valid[:, :, None]
    score, score_rem = (torch.where(valid, x, 0) for x in divide(acc, score_bits(case)))
    top = torch.where(valid, score, INT_MIN).amax(-1, keepdim=True)
    exp_in = torch.where(valid, (score - top).clamp(min=EXP_LOW), 0)
    exp_out = torch.where(valid, st["exp"].to(torch.int64)[exp_in - EXP_LOW], 0)
    total = exp_out.sum(-1, keepdim=True)
    softmax = torch.where(valid, ((exp_out << SCALE_BITS) + total // 2) // total.clamp(min=1), 0)
    out, out_rem = divide(torch.matmul(softmax.to(torch.float64), v).to(torch.int64), SCALE_BITS)
    got = {"out": out, "out_rem": out_rem, "score": score, "score_rem": score_rem, "exp_in": exp_in, "exp_out": exp_out,
           "softmax": softmax}
    got = {name: x.reshape(B, H, -1).to(torch.int32) for name, x in got.items()}
    got["sum"] = total.reshape(B, H)
    return got


# ---------------------------------------------------------------------------------------------- work
def work(case):
    H, KV, D, e = case["heads"], case["kv_heads"], case["dim"], case["bits"] // 8
    if case["op"] == "append":
        new = ragged(case["batch"], case["new_low"], case["new_high"])
        T = sum(new)
        read = 4 * T * (H + 2 * KV) * D + 4 * T * case["rot"]
        written = 4 * T * H * D + 2 * e * T * KV * D + (4 * T * (H + 2 * KV) * D if case["remainders"] else 0)
        touched = sum((max(0, case["start"] - 29 * b) + m - 1) // case["page"] - max(0, case["start"] - 29 * b) // case["page"] + 1
                      for b, m in enumerate(new))
        return {"bytes": read + written + 2 * touched * 2 * KV * D * e, "flops": 3 * T * (H + KV) * case["rot"]}
    n = lengths(case)
    if case["op"] == "select":
        pages = sum(-(-x // case["page"]) for x in n)
        out = 4 * case["batch"] * KV * case["select"] + (8 * pages * KV if case["bounds"] else 0)
        return {"bytes": pages * KV * 2 * D * e + 4 * case["batch"] * H * D + 4 * pages + out, "flops": 2 * pages * H * D}
    if case["select"]:
        n = [min(x, case["select"] * case["page"]) for x in n]
    scores = sum(n) * H
    data = 2 * sum(n) * KV * D * e + 3 * 4 * case["batch"] * H * D + 8 * case["batch"] * H
    return {"bytes": data + 20 * scores + 4 * min(scores, EXP_LEN), "flops": 4 * scores * D}


# ---------------------------------------------------------------------------------------------- exact
def floor_div(x, bits):
    q = np.floor_divide(x + (1 << bits) // 2, 1 << bits)
    return q, x - q * (1 << bits)


def exact(case, seed):
    """The same outputs from the definitions, sequence by sequence in numpy's 64-bit integers."""
    if work(case)["flops"] > 1_500_000_000 or work(case)["bytes"] > 500_000_000:
        return None
    st = {n: (x.cpu().numpy() if isinstance(x, torch.Tensor) else x) for n, x in prepare(case, seed).items()}
    return {"append": exact_append, "select": exact_select, "attend": exact_attend}[case["op"]](case, st)


def exact_append(case, st):
    H, KV, D, ps, rot = case["heads"], case["kv_heads"], case["dim"], case["page"], case["rot"]
    sh, unit = shift_of(case), 1 << SCALE_BITS
    lim = (1 << (case["bits"] - 1)) - 1
    idx = np.arange(rot // 2)
    first, second = (2 * idx, 2 * idx + 1) if case["interleaved"] else (idx, idx + rot // 2)
    rows = st["qkv"].astype(np.int64).reshape(st["tokens"], H + 2 * KV, D)
    acc = rows[:, :H + KV] * unit
    pos, seq = np.zeros(st["tokens"], np.int64), np.zeros(st["tokens"], np.int64)
    for b in range(case["batch"]):
        lo, hi = st["offsets"][b], st["offsets"][b + 1]
        pos[lo:hi], seq[lo:hi] = st["start"][b] + np.arange(hi - lo), b
    z = (rows[:, :H + KV, first].astype(np.int64), rows[:, :H + KV, second].astype(np.int64))
    c, s = st["cos"][pos].astype(np.int64)[:, None], st["sin"][pos].astype(np.int64)[:, None]
    acc[:, :, first] = z[0] * c - z[1] * s
    acc[:, :, second] = z[0] * s + z[1] * c
    q_out, q_rem = floor_div(acc[:, :H], SCALE_BITS)
    key, k_rem = floor_div(acc[:, H:], SCALE_BITS + sh)
    val, v_rem = floor_div(rows[:, H + KV:], sh)
    key, val = np.clip(key, -lim - 1, lim), np.clip(val, -lim - 1, lim)
    k, v, bounds = st["k"].copy(), st["v"].copy(), st["bounds"].copy()
    for t in range(st["tokens"]):
        page, slot = st["table"][seq[t], pos[t] // ps], pos[t] % ps
        k[page, :, slot], v[page, :, slot] = key[t], val[t]
        if slot == 0:
            bounds[page, :, 0] = bounds[page, :, 1] = key[t]
        else:
            bounds[page, :, 0] = np.minimum(bounds[page, :, 0], key[t])
            bounds[page, :, 1] = np.maximum(bounds[page, :, 1], key[t])
    out = {"k": k, "v": v, "bounds": bounds, "q_out": q_out.astype(np.int32)}
    if case["remainders"]:
        out |= {"q_rem": q_rem.astype(np.int32), "k_rem": k_rem.astype(np.int32), "v_rem": v_rem.astype(np.int32)}
    return out


def exact_select(case, st):
    B, H, KV, n = case["batch"], case["heads"], case["kv_heads"], case["select"]
    selected = np.full((B, KV, n), -1, np.int32)
    bound = np.zeros((B, KV, st["table"].shape[1]), np.int64)
    for b, length in enumerate(lengths(case)):
        pages = -(-length // case["page"])
        for g in range(KV):
            rows = st["bounds"][st["table"][b, :pages], g].astype(np.int64)
            q = st["q"][b, g * (H // KV):(g + 1) * (H // KV)].astype(np.int64)
            up, down = np.maximum(q, 0), np.minimum(q, 0)
            bound[b, g, :pages] = (rows[:, 1] @ up.T + rows[:, 0] @ down.T).max(axis=1)
            old = max(0, pages - case["recent"])
            best = sorted(range(old), key=lambda i: (-int(bound[b, g, i]), i))[:max(0, n - (pages - old))]
            chosen = sorted(best + list(range(old, pages)))[-n:]
            selected[b, g, :len(chosen)] = chosen
    return {"selected": selected} | ({"bound": bound} if case["bounds"] else {})


def exact_attend(case, st):
    B, H, KV, D, ps, keys = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"], st["keys"]
    got = {n: np.zeros((B, H, keys), np.int32) for n in ("score", "score_rem", "exp_in", "exp_out", "softmax")}
    out, out_rem, total = np.zeros((B, H, D), np.int32), np.zeros((B, H, D), np.int32), np.zeros((B, H), np.int64)
    for b, length in enumerate(lengths(case)):
        for g in range(KV):
            chosen = [p for p in st["selected"][b, g] if p >= 0] if case["select"] else range(-(-length // ps))
            tokens = np.concatenate([np.arange(p * ps, min((p + 1) * ps, length)) for p in chosen])
            page, slot, m = st["table"][b, tokens // ps], tokens % ps, len(tokens)
            k, v = st["k"][page, g, slot].astype(np.int64), st["v"][page, g, slot].astype(np.int64)
            for h in range(g * (H // KV), (g + 1) * (H // KV)):
                s, r = floor_div(k @ st["q"][b, h].astype(np.int64), score_bits(case))
                x = np.maximum(s - s.max(), EXP_LOW)
                e = st["exp"][x - EXP_LOW].astype(np.int64)
                z = int(e.sum())
                o = np.floor_divide(e * (1 << SCALE_BITS) + z // 2, z)
                for name, a in (("score", s), ("score_rem", r), ("exp_in", x), ("exp_out", e), ("softmax", o)):
                    got[name][b, h, :m] = a
                out[b, h], out_rem[b, h] = floor_div(o @ v, SCALE_BITS)
                total[b, h] = z
    return {"out": out, "out_rem": out_rem} | got | {"sum": total}
