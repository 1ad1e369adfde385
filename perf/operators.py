"""The serving operators in cases that can be timed and compared.

Five operators: ``rms_norm`` (with the residual's addition, to int8 rows),
``rope``, ``cache_append`` (to a paged int8 cache), ``cache_attention`` (over
that cache) and ``dequantize``.  ``run`` computes a case with elementary torch
operations in 32 bits, or, where ``own`` is true, with the calls a user makes
of ``xtile``; ``exact`` computes it from the definition in 64 bits.

Lengths of ragged cases are spread over their range by a fixed sequence, so a
case's work is known; the seed only deals them out to the sequences.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f32": 4}
_EPS = 1e-5


def listed():
    return [
        # eight sequences each decode one token: the norm before the projections, to int8 rows for an int8 matmul
        dict(name="norm decode", op="norm", rows=8, cols=4096, dtype="bf16", residual=True, out="i8"),
        # the same norm over a prompt of 8192 tokens
        dict(name="norm prompt", op="norm", rows=8192, cols=4096, dtype="bf16", residual=True, out="i8"),
        # queries of 16 decoding sequences, a view into the packed projection rows
        dict(name="rope decode", op="rope", tokens=16, heads=32, dim=128, rot=128, interleaved=False, dtype="bf16",
             packed=48, inverse=False),
        # queries of a long prompt as an f32 matmul leaves them, half of each head rotated, pairs side by side
        dict(name="rope prompt", op="rope", tokens=8192, heads=32, dim=128, rot=64, interleaved=True, dtype="f32",
             packed=32, inverse=False),
        # 64 sequences append one token each, most of them into a block that has tokens already
        dict(name="append decode", op="append", seqs=64, new=1, context=128, kv_heads=8, dim=128, page=64, block=16,
             rot=128, interleaved=False, dtype="bf16"),
        # ragged prompts enter the cache
        dict(name="append prompts", op="append", seqs=7, new=4000, context=4000, kv_heads=8, dim=128, page=64,
             block=16, rot=128, interleaved=False, dtype="bf16"),
        # one sequence decodes: the latency of a single user
        dict(name="attend one", op="attend", seqs=1, new=1, context=777, q_heads=32, kv_heads=8, dim=128, page=64,
             block=16, window=0, softcap=0.0, dtype="bf16"),
        # a full decode batch of ragged contexts
        dict(name="attend batch", op="attend", seqs=64, new=1, context=8192, q_heads=32, kv_heads=8, dim=128, page=64,
             block=16, window=0, softcap=0.0, dtype="bf16"),
        # several drafted tokens a sequence, f32 heads of 64 with a window and capped scores, pages of 48
        dict(name="attend drafted", op="attend", seqs=9, new=5, context=3001, q_heads=16, kv_heads=16, dim=64,
             page=48, block=8, window=1000, softcap=30.0, dtype="f32"),
        # prompt chunks of 2048 tokens behind what is in the cache already
        dict(name="attend prompt", op="attend", seqs=2, new=2048, context=4096, q_heads=32, kv_heads=8, dim=128,
             page=64, block=16, window=0, softcap=0.0, dtype="bf16"),
        # a few int8 rows read back
        dict(name="read rows", op="read", runs=100, run=1000, dtype="f32"),
        # a cache's blocks read back, to move sequences elsewhere
        dict(name="read blocks", op="read", runs=32768, run=2048, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rope", "append", "attend", "attend", "read"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    page, block = rng.choice([(64, 16), (64, 64), (16, 16), (48, 8), (128, 32), (32, 1), (40, 20)])
    if op == "norm":
        cols = rng.choice([1024, 2048, 4096, 5120, 8192, _log_int(rng, 64, 8192)])
        rows = _log_int(rng, 1, min(16384, 33554432 // cols))
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, residual=rng.random() < 0.7,
                    out=rng.choice(["i8", "i8", "same"]))
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        heads = rng.choice([1, 4, 8, 12, 32])
        tokens = _log_int(rng, 1, min(16384, 33554432 // (heads * dim)))
        return dict(op=op, tokens=tokens, heads=heads, dim=dim, rot=rng.choice([dim, dim, dim // 2]),
                    interleaved=rng.random() < 0.5, dtype=dtype, packed=heads + rng.choice([0, 2, 7]),
                    inverse=rng.random() < 0.25)
    if op == "append":
        dim, kv_heads = rng.choice([64, 80, 128, 256]), rng.choice([1, 2, 5, 8])
        seqs = _log_int(rng, 1, 128)
        new = 1 if rng.random() < 0.4 else _log_int(rng, 2, max(2, 12000000 // (seqs * kv_heads * dim)))
        context = new + rng.choice([0, rng.randrange(1, 300)])
        return dict(op=op, seqs=seqs, new=new, context=context, kv_heads=kv_heads, dim=dim, page=page, block=block,
                    rot=rng.choice([0, dim, dim // 2]), interleaved=rng.random() < 0.5, dtype=dtype)
    if op == "attend":
        dim, kv_heads = rng.choice([64, 80, 96, 128, 128, 256]), rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 4, 5, 7, 8, 16])
        seqs = _log_int(rng, 1, 96)
        context = _log_int(rng, 8, min(200000, 300000000 // (seqs * kv_heads * dim)))
        most = 100000000000 // (4 * seqs * kv_heads * group * dim * context)
        most = max(1, min(most, context, 500000000 // (seqs * kv_heads * group * context), 4096))
        new = 1 if rng.random() < 0.5 else _log_int(rng, 1, most)
        return dict(op=op, seqs=seqs, new=new, context=context, q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    page=page, block=block, window=rng.choice([0, 0, 0, _log_int(rng, 1, context)]),
                    softcap=rng.choice([0.0, 0.0, 30.0]), dtype=dtype)
    run = rng.choice([16 * 128, 8 * 64, _log_int(rng, 16, 8192)])
    return dict(op=op, runs=_log_int(rng, 1, 67108864 // run), run=run, dtype=dtype)


def _spread(n, lo, hi):
    """``n`` whole numbers over [lo, hi]; the first is hi."""
    at = [(0.6180339887498949 * i + 1.0) % 1.0 for i in range(n)]
    return [hi - int(a * (hi - lo)) for a in at]


def _lengths(case):
    """(new tokens, tokens in all) of each sequence of a ragged case, in no order."""
    total = _spread(case["seqs"], max(case["context"] // 4, 1), case["context"])
    new = [min(n, t) for n, t in zip(_spread(case["seqs"], max(case["new"] // 2, 1), case["new"]), total)]
    return new, total


def _tables(case, rand):
    """starts, lengths and the page table of a ragged case on the GPU, and how many pages there are."""
    new, total = _lengths(case)
    order = rand.permutation(case["seqs"])
    new, total = np.array(new)[order], np.array(total)[order]
    page = case["page"]
    need = (total + page - 1) // page
    count = int(need.sum())
    free = rand.permutation(count)
    pages = np.zeros((case["seqs"], int(need.max())), np.int32)
    at = 0
    for b, n in enumerate(need):
        pages[b, :n] = free[at:at + n]
        at += n
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return put(starts), put(total.astype(np.int32)), put(pages), count, int(starts[-1])


def _cache(case, count, gen):
    """The four tensors of a filled cache: int8 keys and values of normal tokens, and their blocks' scales."""
    h, d, page, nb = case["kv_heads"], case["dim"], case["page"], case["page"] // case["block"]
    parts = []
    for _ in range(2):
        q = torch.empty(count, h, page, d, dtype=torch.int8, device="cuda")
        for c in range(0, count, 4096):
            x = torch.empty(q[c:c + 4096].shape, dtype=torch.bfloat16, device="cuda").normal_(0, 40, generator=gen)
            q[c:c + 4096] = x.round_().clamp_(-127, 127)
        parts.append(q)
    scales = [torch.empty(count, h, nb, device="cuda").uniform_(0.015, 0.035, generator=gen) for _ in range(2)]
    return parts[0], parts[1], scales[0], scales[1]


def _cos_sin(positions, rot):
    """cos and sin of every position and frequency, made in 64 bits: [positions, rot / 2, 2]."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * f
    return torch.stack([a.cos(), a.sin()], dim=-1).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = np.random.RandomState(seed % (1 << 31))
    op, s = case["op"], {"case": case}
    dtype = _TYPES[case["dtype"]]

    def normal(*shape, std=1.0, type=dtype):
        return torch.empty(*shape, device="cuda").normal_(0, std, generator=gen).to(type)

    def empty(*shape, type=dtype):
        return torch.empty(*shape, dtype=type, device="cuda")

    if op == "norm":
        r, c = case["rows"], case["cols"]
        s["x"] = normal(r, c)
        s["residual"] = normal(r, c, std=4.0) if case["residual"] else None
        s["weight"] = (1 + 0.1 * normal(c, type=torch.float32)).to(dtype)
        s["sum"] = empty(r, c) if case["residual"] else None
        s["y"] = empty(r, c, type=torch.int8 if case["out"] == "i8" else dtype)
        s["scales"] = empty(r, type=torch.float32)
        s["values"] = empty(r, c, type=torch.bfloat16)
    elif op == "rope":
        t, h, d = case["tokens"], case["heads"], case["dim"]
        s["x"] = normal(t, case["packed"] * d)[:, :h * d].view(t, h, d)  # the queries of packed projection rows
        s["positions"] = torch.from_numpy(rand.randint(0, 16384, t).astype(np.int32)).cuda()
        s["cos_sin"] = _cos_sin(16384, case["rot"])
        s["y"] = empty(t, h, d)
    elif op == "append":
        s["starts"], s["lengths"], s["pages"], count, tokens = _tables(case, rand)
        h, d = case["kv_heads"], case["dim"]
        kv = normal(tokens, 2, h, d) * (1 + 3 * torch.rand(d, device="cuda", generator=gen) ** 8).to(dtype)
        s["k"], s["v"] = kv[:, 0], kv[:, 1]  # keys and values of packed projection rows
        s["cache"] = _cache(case, count, gen)
        s["cos_sin"] = _cos_sin(case["context"], case["rot"]) if case["rot"] else None
        s["values"] = [empty(c.shape, type=torch.bfloat16) for c in s["cache"][:2]]
    elif op == "attend":
        s["starts"], s["lengths"], s["pages"], count, tokens = _tables(case, rand)
        s["q"] = normal(tokens, case["q_heads"], case["dim"], std=1.5)
        s["cache"] = _cache(case, count, gen)
        s["new"] = case["new"]  # a program that batches sequences knows the most new tokens that one has
        s["y"] = empty(s["q"].shape)
    else:
        s["q"] = empty(case["runs"], case["run"]).normal_(0, 40, generator=gen).round_().clamp_(-127, 127).to(torch.int8)
        s["scales"] = empty(case["runs"], type=torch.float32).uniform_(0.01, 0.04, generator=gen)
        s["values"] = empty(case["runs"], case["run"])
    if own:
        import xtile as xt

        if "cache" in s:
            s["cache"] = xt.KVCache(*s["cache"])
        if s.get("cos_sin") is not None:
            s["cos_sin"] = xt.RopeTable(s["cos_sin"], interleaved=case["interleaved"])
    return s


# ----------------------------------------------------------------- plain forms

def _quantize(x, dims):
    """int8 values and scales of f32 ``x``, one scale over ``dims``."""
    scale = x.abs().amax(dims, keepdim=True) / 127.0
    q = torch.where(scale > 0, (x / scale).round(), torch.zeros_like(x)).clamp(-127, 127)
    return q, scale


def _rotate(x, cos_sin, interleaved, inverse=False):
    """Rotates the pairs of f32 ``x`` [tokens, heads, dim] by each token's row of cos_sin [tokens, rot / 2, 2]."""
    half = cos_sin.shape[1]
    c, s = cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
    s = -s if inverse else s
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * c - b * s, a * s + b * c
    return y


def _plain_norm(s, case):
    h = s["x"].float()
    if case["residual"]:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS) * s["weight"].float()
    out = {"sum": h.to(s["x"].dtype)} if case["residual"] else {}
    if case["out"] != "i8":
        return {**out, "y": y.to(s["x"].dtype)}
    q, scale = _quantize(y, -1)
    return {**out, "values": (q * scale).to(torch.bfloat16), "scales": scale[:, 0]}


def _plain_append(s, case):
    kq, vq, ks, vs = s["cache"]
    starts, lengths, pages = s["starts"].long(), s["lengths"].long(), s["pages"].long()
    page, block, nb = case["page"], case["block"], case["page"] // case["block"]
    tokens = s["k"].shape[0]
    token = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(starts, token, right=True) - 1
    position = lengths[seq] - starts[seq + 1] + token
    into = pages[seq, position // page]
    blk = into * nb + position % page // block  # the block of each token among all blocks
    begin = lengths - (starts[1:] - starts[:-1])
    held = begin[seq] - position // block * block  # rows of its block that earlier calls filled
    old = held > 0
    k, v = s["k"].float(), s["v"].float()
    if case["rot"]:
        k = _rotate(k, s["cos_sin"][position], case["interleaved"])
    h = case["kv_heads"]
    values = []
    for x, q, scale in ((k, kq, ks), (v, vq, vs)):
        flat = scale.transpose(1, 2).reshape(-1, h)  # [pages * nb, heads]
        top = x.abs().amax(-1) / 127.0
        new = torch.zeros_like(flat).index_reduce_(0, blk, top, "amax")
        touched = torch.zeros(flat.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, blk, True)
        kept = torch.zeros(flat.shape[0], dtype=torch.long, device="cuda")
        kept[blk[old]] = held[old]
        new = torch.where(kept[:, None] > 0, torch.maximum(new, flat), new)
        ratio = torch.where(new > flat, flat / new, 1.0).view(-1, nb, h).transpose(1, 2)
        earlier = torch.arange(block, device="cuda") < kept.view(-1, 1, nb, 1)  # rows behind them stay as they are
        moved = q.view(-1, h, nb, block, q.shape[-1]).float()
        moved = (moved * torch.where(earlier, ratio[..., None], 1.0)[..., None]).round()
        mine = new[blk]
        fresh = torch.where(mine[..., None] > 0, (x / mine[..., None]).round(), torch.zeros_like(x)).clamp(-127, 127)
        moved = moved.view(q.shape)
        moved[into, :, position % page] = fresh
        q.copy_(moved)
        scale.copy_(torch.where(touched[:, None], new, flat).view(-1, nb, h).transpose(1, 2))
        values.append((moved.view(-1, h, nb, block, q.shape[-1]) * scale[..., None, None]).view(q.shape)
                      .to(torch.bfloat16))
    return {"k": values[0], "v": values[1], "k_scale": ks, "v_scale": vs}


def _plain_attend(s, case):
    kq, vq, ks, vs = s["cache"]
    starts, lengths, pages = s["starts"].long(), s["lengths"].long(), s["pages"].long()
    h, d, page, block = case["kv_heads"], case["dim"], case["page"], case["block"]
    seqs, g = case["seqs"], case["q_heads"] // h
    new = starts[1:] - starts[:-1]
    i = torch.arange(s["new"], device="cuda")
    there = i < new[:, None]  # [seqs, n]: sequences with fewer new tokens leave some out
    row = torch.where(there, starts[:-1, None] + i, 0)
    position = (lengths - new)[:, None] + i
    q = s["q"].float()[row].view(seqs, -1, h, g, d).permute(0, 2, 3, 1, 4)  # [seqs, h, g, n, d]

    def gather(x, scale):  # [seqs, h, tokens, d] in f32
        x = x.view(x.shape[0], h, page // block, block, d)[pages].float() * scale[pages][..., None, None]
        return x.transpose(1, 2).reshape(seqs, h, -1, d)

    k, v = gather(kq, ks), gather(vq, vs)
    score = torch.matmul(q.reshape(seqs, h, -1, d), k.transpose(2, 3)).mul_(1.0 / math.sqrt(d))
    if case["softcap"]:
        score = score.div_(case["softcap"]).tanh_().mul_(case["softcap"])
    j = torch.arange(k.shape[2], device="cuda")
    seen = (j <= position[..., None]) & there[..., None]
    if case["window"]:
        seen &= j > position[..., None] - case["window"]
    score = score.view(seqs, h, g, -1, k.shape[2]).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top > -math.inf, top, 0)).exp_()
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.view(seqs, h, -1, k.shape[2]), v).view(seqs, h, g, -1, d)
    y = torch.where(total > 0, y / total, 0).permute(0, 3, 1, 2, 4).reshape(seqs, -1, h * g, d)
    return {"y": y[there].to(s["q"].dtype)}


def _plain(s, case):
    op = case["op"]
    if op == "norm":
        return _plain_norm(s, case)
    if op == "rope":
        y = _rotate(s["x"].float(), s["cos_sin"][s["positions"].long()], case["interleaved"], case["inverse"])
        return {"y": y.to(s["x"].dtype)}
    if op == "append":
        return _plain_append(s, case)
    if op == "attend":
        return _plain_attend(s, case)
    return {"values": (s["q"].float() * s["scales"][:, None]).to(s["values"].dtype)}


def run(state):
    s, case = state, state["case"]
    if not own:
        return _plain(s, case)
    import xtile as xt

    op = case["op"]
    if op == "norm":
        out = {"sum": s["sum"]} if case["residual"] else {}
        if case["out"] != "i8":
            xt.rms_norm(s["x"], s["weight"], s["y"], residual=s["residual"], residual_out=s["sum"], eps=_EPS)
            return {**out, "y": s["y"]}
        xt.rms_norm(s["x"], s["weight"], s["y"], scales=s["scales"], residual=s["residual"], residual_out=s["sum"],
                    eps=_EPS)
        return {**out, "values": xt.dequantize(s["y"], s["scales"], s["values"]), "scales": s["scales"]}
    if op == "rope":
        return {"y": xt.rope(s["x"], s["positions"], s["cos_sin"], s["y"], inverse=case["inverse"])}
    if op == "append":
        cache = s["cache"]
        xt.cache_append(cache, s["k"], s["v"], s["starts"], s["lengths"], s["pages"], rope=s["cos_sin"])
        return {"k": xt.dequantize(cache.k, cache.k_scale, s["values"][0]), "k_scale": cache.k_scale,
                "v": xt.dequantize(cache.v, cache.v_scale, s["values"][1]), "v_scale": cache.v_scale}
    if op == "attend":
        return {"y": xt.cache_attention(s["cache"], s["q"], s["starts"], s["lengths"], s["pages"], s["y"],
                                        max_new=s["new"], window=case["window"], softcap=case["softcap"])}
    return {"values": xt.dequantize(s["q"], s["scales"], s["values"])}


# ------------------------------------------------------------------------ work

def work(case):
    op, size = case["op"], _BYTES[case["dtype"]]
    if op == "norm":
        n = case["rows"] * case["cols"]
        moved = n * size * (3 if case["residual"] else 1) + case["cols"] * size
        # int8 rows are written, and read back as bf16 values
        moved += n * (1 + 1 + 2) + 4 * case["rows"] if case["out"] == "i8" else n * size
        return {"bytes": moved, "flops": 8 * n}
    if op == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        rows = min(case["tokens"], 16384) * case["rot"] * 4
        return {"bytes": 2 * n * size + rows + 4 * case["tokens"],
                "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    if op == "read":
        n = case["runs"] * case["run"]
        return {"bytes": n * (1 + size) + 4 * case["runs"], "flops": n}
    new, total = _lengths(case)
    h, d, block, page = case["kv_heads"], case["dim"], case["block"], case["page"]
    if op == "append":
        # keys and values are read and written as int8 with their scales, and the cache's pages read back as bf16
        held = sum(-(-t // page) * page for t in total)
        blocks = sum(-(-n // block) for n in new)
        moved = 2 * sum(new) * h * d * (size + 1) + 2 * 4 * blocks * h + 4 * sum(new) * case["rot"]
        return {"bytes": moved + 2 * held * h * (d * 3 + 4 / block), "flops": 2 * sum(new) * h * (4 * d)}
    window = case["window"] or max(total)
    seen = [sum(min(t - n + i + 1, window) for i in range(n)) for n, t in zip(new, total)]
    touched = sum(min(t, window + n - 1) for n, t in zip(new, total))
    moved = touched * h * (2 * d + 8 / block) + 2 * sum(new) * case["q_heads"] * d * size
    return {"bytes": moved, "flops": 4.0 * d * case["q_heads"] * sum(seen)}


# ------------------------------------------------- the definitions, in 64 bits

def _to_int8(x, scale):
    return torch.clamp(torch.round(x / scale), -127, 127) if scale > 0 else torch.zeros_like(x)


def _turned(x, angles, interleaved, inverse):
    """x [tokens, heads, dim] as complex numbers, each token's times exp(i angle) of its own angles."""
    c, s = angles[..., 0].double(), angles[..., 1].double()
    turn = torch.complex(c, -s if inverse else s)[:, None]
    n = turn.shape[-1]
    x = x.double()
    if interleaved:
        z = torch.view_as_complex(x[..., :2 * n].unflatten(-1, (n, 2)).contiguous()) * turn
        head = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., :n], x[..., n:2 * n]) * turn
        head = torch.cat([z.real, z.imag], -1)
    return torch.cat([head, x[..., 2 * n:]], -1)


def _exact_norm(s, case):
    out = {}
    h = s["x"].double()
    if case["residual"]:
        out["sum"] = h = h + s["residual"].double()
    norm = torch.linalg.vector_norm(h, dim=1, keepdim=True)
    y = h * s["weight"].double() / torch.sqrt(norm ** 2 / case["cols"] + _EPS)
    if case["out"] != "i8":
        return {**out, "y": y}
    scale = torch.linalg.vector_norm(y, ord=math.inf, dim=1, keepdim=True) / 127
    return {**out, "values": torch.round(y / scale) * scale, "scales": scale[:, 0]}


def _exact_append(s, case):
    starts, lengths, pages = s["starts"].tolist(), s["lengths"].tolist(), s["pages"].tolist()
    page, block = case["page"], case["block"]
    if sum((n // block + 2) for n in np.diff(starts)) * case["kv_heads"] > 20000:
        return None
    out = {}
    for name, x, q, scale in (("k", s["k"], s["cache"][0], s["cache"][2]), ("v", s["v"], s["cache"][1], s["cache"][3])):
        q, scale = q.double(), scale.double()
        for b in range(case["seqs"]):
            first, last = lengths[b] - (starts[b + 1] - starts[b]), lengths[b]
            at = first
            while at < last:
                lo = at // block * block
                hi = min(lo + block, last)
                p, inside, slot = pages[b][lo // page], lo % page, lo % page // block
                rows = x[starts[b] + at - first:starts[b] + hi - first].double()
                if name == "k" and case["rot"]:
                    rows = _turned(rows, s["cos_sin"][at:hi], case["interleaved"], False)
                for h in range(case["kv_heads"]):
                    was = scale[p, h, slot].item() if at > lo else 0.0
                    now = max(was, rows[:, h].abs().max().item() / 127)
                    if at > lo and now > was:
                        q[p, h, inside:inside + at - lo] = torch.round(q[p, h, inside:inside + at - lo] * (was / now))
                    q[p, h, inside + at - lo:inside + hi - lo] = _to_int8(rows[:, h], now)
                    scale[p, h, slot] = now
                at = hi
        out[name] = (q.view(*scale.shape, block, -1) * scale[..., None, None]).view(q.shape)
        out[name + "_scale"] = scale
    return out


def _exact_attend(s, case):
    starts, lengths, pages = s["starts"].tolist(), s["lengths"].tolist(), s["pages"].long()
    kq, vq, ks, vs = s["cache"]
    d, page, block, g = case["dim"], case["page"], case["block"], case["q_heads"] // case["kv_heads"]
    y = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["seqs"]):
        n, t = starts[b + 1] - starts[b], lengths[b]
        held = pages[b, :-(-t // page)]
        position = torch.arange(t - n, t, device="cuda")[:, None]
        token = torch.arange(t, device="cuda")
        hidden = token > position
        if case["window"]:
            hidden |= token <= position - case["window"]
        for h in range(case["kv_heads"]):
            k = kq[held, h].reshape(-1, d)[:t].double() * ks[held, h].repeat_interleave(block, 1).reshape(-1, 1)[:t]
            v = vq[held, h].reshape(-1, d)[:t].double() * vs[held, h].repeat_interleave(block, 1).reshape(-1, 1)[:t]
            for r in range(h * g, h * g + g):
                score = s["q"][starts[b]:starts[b + 1], r].double() @ k.T / math.sqrt(d)
                if case["softcap"]:
                    score = case["softcap"] * torch.tanh(score / case["softcap"])
                y[starts[b]:starts[b + 1], r] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v
    return {"y": y}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        return _exact_norm(s, case)
    if op == "rope":
        return {"y": _turned(s["x"], s["cos_sin"][s["positions"].long()], case["interleaved"], case["inverse"])}
    if op == "append":
        return _exact_append(s, case)
    if op == "attend":
        return _exact_attend(s, case)
    return {"values": s["q"].double() * s["scales"].double()[:, None]}
