"""The serving operators on a GPU against plain 64-bit forms.

Tolerances follow from the arithmetic.  u = 2^-24 is the f32 unit roundoff; a
bf16 result adds 2^-8 of itself; an int8 value may be half a step of its scale
off.  Each test states what else it allows.
"""
import math

import pytest
import torch

import xtile as xt

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16_STEP = 2.0 ** -8 * 1.01
TYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    assert xt.device_error() == 0


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(gen, *shape, std=1.0, dtype=torch.float32):
    return torch.empty(*shape, device="cuda").normal_(0, std, generator=gen).to(dtype)


def within(got, want, allowed):
    got, want = got.double(), want.double()
    assert torch.equal(got.isnan(), want.isnan())
    off = (got - want).abs() - allowed
    assert not (off > 0).any(), f"{int((off > 0).sum())} of {off.numel()} values, the worst {off.nan_to_num().max():.3g} too far"


def rounding(y, dtype):
    return BF16_STEP * y.abs() if dtype == torch.bfloat16 else 0.0


# ------------------------------------------------------------------- rms norm

def norm_64(x, weight, residual, eps):
    h = x.double() if residual is None else x.double() + residual.double()
    return h, h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * weight.double()


# widths: one element, under and over a warp's vector, odd, the limits of each kernel's registers, and past them
WIDTHS = [1, 2, 8, 31, 250, 256, 264, 1000, 1024, 1032, 2047, 4096, 4097, 8200, 32768, 32776]


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out", ["same", "i8"])
def test_rms_norm_widths(cols, dtype, out):
    g = generator(cols)
    rows, eps = 5, 1e-5
    x, w, r = normal(g, rows, cols, dtype=dtype), normal(g, cols, dtype=dtype), normal(g, rows, cols, std=3, dtype=dtype)
    h, want = norm_64(x, w, r, eps)
    total = torch.full_like(x, float("nan"))
    # f32: the sum of squares over at most 64 sequential and 20 tree terms, halved by the root, rsqrt's 2 ulp, 4 products
    rel = 64 * U
    if out == "same":
        y = xt.rms_norm(x, w, residual=r, residual_out=total, eps=eps)
        assert y.dtype == dtype
        within(y, want, rel * want.abs() + rounding(want, dtype))
    else:
        q, s = xt.rms_norm(x, w, residual=r, residual_out=total, eps=eps, dtype=torch.int8)
        top = want.abs().amax(-1)
        within(s, top / 127, rel * top)
        within(q.double() * s.double()[:, None], want, (0.5 + 1e-3) * s.double()[:, None])
    within(total, h, U * h.abs() + rounding(h, dtype))


@pytest.mark.parametrize("rows", [1, 7, 8, 9, 3000])
@pytest.mark.parametrize("weight_dtype", TYPES)
def test_rms_norm_rows_types_and_strides(rows, weight_dtype):
    g = generator(rows)
    wide = normal(g, rows, 700, dtype=torch.float32)
    x = wide[:, 3:515]  # rows 700 apart that start off the vector boundary
    w = normal(g, 512, dtype=weight_dtype)
    _, want = norm_64(x, w, None, 1e-6)
    base = torch.full((rows, 520), 7.0, device="cuda", dtype=torch.bfloat16)
    y = base[:, :512]
    assert xt.rms_norm(x, w, y) is y
    within(y, want, 64 * U * want.abs() + rounding(want, torch.bfloat16))
    assert (base[:, 512:] == 7.0).all()


@pytest.mark.parametrize("cols", [512, 4099, 40000])
def test_rms_norm_in_place(cols):
    g = generator(3)
    x, r, w = normal(g, 6, cols), normal(g, 6, cols), normal(g, cols)
    h, want = norm_64(x, w, r, 1e-6)
    y = xt.rms_norm(x, w, x, residual=r, residual_out=r)
    assert y is x
    within(y, want, 64 * U * want.abs())
    within(r, h, U * h.abs())


def test_rms_norm_zeros_and_nan():
    x = torch.ones(5, 64, device="cuda")
    x[1] = 0
    x[2, 3] = float("nan")
    x[3, 5] = float("inf")
    x[4] = 1e-30  # normed values of 1e-27 are under eps' reach but above the int8 threshold
    w = torch.ones(64, device="cuda")
    q, s = xt.rms_norm(x, w, dtype=torch.int8)
    assert (q[0] == 127).all() and (q[1] == 0).all() and s[1] == 0
    assert s[2].isnan() and s[3].isnan()  # whoever reads those rows back sees it
    assert (q[4] == 127).all()
    y = xt.rms_norm(x, w)
    assert y[2].isnan().all() and y[3, 5].isnan() and (y[1] == 0).all()


# ----------------------------------------------------------------------- rope

def rope_64(x, cos_sin, interleaved, inverse=False):
    c, s = cos_sin[..., 0].double()[:, None], cos_sin[..., 1].double()[:, None]
    s = -s if inverse else s
    half = c.shape[-1]
    y, x = x.double().clone(), x.double()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    size = torch.zeros_like(y)
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return y, size


@pytest.mark.parametrize("dim, rot", [(64, 64), (80, 40), (80, 80), (96, 48), (128, 64), (128, 128), (256, 256), (6, 2),
                                      (34, 34), (50, 20), (576, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                   (torch.float32, torch.bfloat16)])
def test_rope_layouts(dim, rot, interleaved, types):
    g = generator(dim + rot)
    tokens, heads = 13, 5
    x = normal(g, tokens, heads, dim, dtype=types[0])
    table = xt.RopeTable.build(100, rot, interleaved=interleaved)
    pos = torch.randint(0, 100, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    want, size = rope_64(x, table.cos_sin[pos.long()], interleaved)
    out = torch.empty(x.shape, dtype=types[1], device="cuda")
    assert xt.rope(x, pos, table, out) is out
    within(out, want, 3 * U * size + rounding(want, types[1]))


@pytest.mark.parametrize("tokens, heads", [(1, 1), (1, 32), (3000, 32), (5000, 3)])
@pytest.mark.parametrize("dtype", TYPES)
def test_rope_packed_rows_in_place(tokens, heads, dtype):
    g = generator(tokens)
    packed = normal(g, tokens, (heads + 3) * 64, dtype=dtype)
    before = packed.clone()
    x = packed[:, 64:64 * (heads + 1)].view(tokens, heads, 64)
    table = xt.RopeTable.build(8192, 64)
    pos = torch.arange(tokens, device="cuda", dtype=torch.int32)
    want, size = rope_64(x, table.cos_sin[:tokens], False)
    xt.rope(x, pos, table, x)
    within(x, want, 3 * U * size + rounding(want, dtype))
    assert torch.equal(packed[:, :64], before[:, :64]) and torch.equal(packed[:, 64 * (heads + 1):], before[:, 64 * (heads + 1):])


def test_rope_heads_first_and_odd_offsets():
    g = generator(8)
    x = normal(g, 4, 9, 64, dtype=torch.bfloat16).transpose(0, 1)  # [9, 4, 64], heads outermost in memory
    odd = normal(g, 9 * 4 * 64 + 1, dtype=torch.bfloat16)[1:].view(9, 4, 64)
    table = xt.RopeTable.build(32, 64)
    pos = torch.arange(9, device="cuda", dtype=torch.int32)
    for t in (x, odd):
        want, size = rope_64(t, table.cos_sin[:9], False)
        within(xt.rope(t, pos, table), want, 3 * U * size + rounding(want, torch.bfloat16))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_gradient_is_the_inverse(interleaved):
    g = generator(5)
    x, grad = normal(g, 6, 3, 32), normal(g, 6, 3, 32)
    table = xt.RopeTable.build(50, 16, interleaved=interleaved)
    pos = torch.tensor([0, 49, 3, 3, 17, 8], device="cuda", dtype=torch.int32)
    dx = xt.rope(grad, pos, table, inverse=True)
    leaf = x.double().requires_grad_()
    want, _ = rope_64(grad, table.cos_sin[pos.long()], interleaved, inverse=True)
    within(dx, want, 3 * U * grad.abs().amax() * 2)
    # against differences of the forward call: it is linear, so a step of 1 gives the slope itself
    for i in range(0, x.numel(), 37):
        step = torch.zeros_like(x).view(-1)
        step[i] = 1.0
        forward = xt.rope(step.view(x.shape), pos, table)
        slope = (forward.double() * grad.double()).sum()
        assert abs(slope - dx.double().view(-1)[i]) <= 6 * U * (grad.abs().amax().double() * 2)
    back = xt.rope(xt.rope(x, pos, table), pos, table, inverse=True)
    within(back, leaf.detach(), 16 * U * x.abs().amax())


def test_rope_table_scalings():
    plain = xt.RopeTable.build(64, 32).cos_sin.double()
    slow = xt.RopeTable.build(256, 32, factor=4.0).cos_sin.double()
    within(slow[::4], plain, 2 * U)
    parts = xt.RopeTable.build(64, 32, factor=8.0, trained=4096, low=1.0, high=32.0, amplitude=1.2).cos_sin.double() / 1.2
    freq = 10000.0 ** (-torch.arange(0, 32, 2, dtype=torch.float64) / 32)
    turns = 4096 * freq / (2 * math.pi)
    for i, (f, n) in enumerate(zip(freq.tolist(), turns.tolist())):
        keep = min(max((n - 1) / 31, 0.0), 1.0)
        angle = 5 * f * (keep + (1 - keep) / 8)
        assert abs(parts[5, i, 0].item() - math.cos(angle)) <= 4 * U
        assert abs(parts[5, i, 1].item() - math.sin(angle)) <= 4 * U


def test_rope_position_outside_the_table():
    table = xt.RopeTable.build(8, 32)
    x = torch.ones(3, 2, 64, device="cuda")
    pos = torch.tensor([7, 8, -1], device="cuda", dtype=torch.int32)
    y = xt.rope(x, pos, table)
    assert xt.device_error() == 0x301
    assert y[0].isfinite().all() and y[1:, :, :32].isnan().all() and (y[1:, :, 32:] == 1).all()


# --------------------------------------------------------------- paged batches

class Batch:
    """Sequences of ``total`` tokens, the last ``new`` of them new, over shuffled pages."""

    def __init__(self, new, total, page, seed, spare=2, extra_width=1):
        self.new, self.total = new, total
        g = torch.Generator().manual_seed(seed)
        need = [-(-t // page) for t in total]
        self.pages_held = sum(need) + spare
        order = torch.randperm(self.pages_held, generator=g).tolist()
        width = max(need + [0]) + extra_width
        table = torch.full((len(total), width), -7, dtype=torch.int32)  # never followed behind a sequence's end
        self.table = []
        for b, n in enumerate(need):
            self.table.append([order.pop() for _ in range(n)])
            table[b, :n] = torch.tensor(self.table[-1], dtype=torch.int32)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.first, self.tokens = starts, starts[-1]
        self.args = (torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(total, dtype=torch.int32).cuda(),
                     table.cuda())


def filled_cache(gen, pages, heads, dim, page, block, lo=0.01, hi=0.03):
    cache = xt.KVCache.empty(pages, heads, dim, page=page, block=block)
    for t in (cache.k, cache.v):
        t.copy_(torch.randint(-127, 128, t.shape, generator=gen, device="cuda"))
    for t in (cache.k_scale, cache.v_scale):
        t.copy_(torch.exp(torch.empty_like(t).uniform_(math.log(lo), math.log(hi), generator=gen)))
    return cache


# --------------------------------------------------------------------- append

def check_append(cache, before, batch, k, v, table):
    """Every value of the cache against the definition."""
    page, block, dim = cache.page, cache.block, cache.dim
    for name, x, rot in (("k", k, table), ("v", v, None)):
        q, s = getattr(cache, name), getattr(cache, name + "_scale")
        q0, s0 = before[name], before[name + "_scale"]
        touched = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
        blocks = torch.zeros(s.shape, dtype=torch.bool, device="cuda")
        for b, (n, t) in enumerate(zip(batch.new, batch.total)):
            at = t - n
            while at < t:
                lo = at // block * block
                hi = min(lo + block, t)
                into, row, slot = batch.table[b][lo // page], lo % page, lo % page // block
                rows = x[batch.first[b] + at - (t - n):batch.first[b] + hi - (t - n)]
                slack = 0.0
                want = rows.double()
                if rot is not None:
                    want, size = rope_64(rows, rot.cos_sin[at:hi], rot.interleaved)
                    slack = 4 * U * size.transpose(0, 1)
                want = want.transpose(0, 1)  # [heads, rows, dim]
                top = want.abs().amax((1, 2))
                top_slack = 8 * U * (want.abs() + slack).amax((1, 2)) if rot is not None else 4 * U * top
                scale = top / 127
                if at > lo:
                    scale = torch.maximum(scale, s0[into, :, slot].double())
                got = s[into, :, slot].double()
                within(got, scale, top_slack / 127 + 4 * U * scale)
                step = got[:, None, None]
                new = q[into, :, row + at - lo:row + hi - lo].double()
                within(new * step, want, (0.5 + 1e-4) * step + slack)
                if at > lo:  # the earlier tokens' values moved by at most half a step, and not at all if the scale stayed
                    old0, old = q0[into, :, row:row + at - lo], q[into, :, row:row + at - lo]
                    within(old.double() * step, old0.double() * s0[into, :, slot].double()[:, None, None], (0.5 + 1e-4) * step)
                    same = got == s0[into, :, slot].double()
                    assert torch.equal(old[same], old0[same])
                touched[into, :, row:row + hi - lo] = True
                blocks[into, :, slot] = True
                at = hi
        assert torch.equal(q[~touched], q0[~touched])  # and nothing else moved
        assert torch.equal(s[~blocks], s0[~blocks])


def snapshot(cache):
    return {n: getattr(cache, n).clone() for n in ("k", "v", "k_scale", "v_scale")}


APPENDS = [
    # new, total
    ([1], [1]),
    ([1, 1, 1, 1, 1], [1, 16, 17, 64, 65]),
    ([3, 0, 40, 1], [3, 9, 77, 200]),
    ([200, 131], [200, 131]),
    ([0, 0], [5, 0]),
    ([5] * 40, [5 + 7 * i for i in range(40)]),
    ([1] * 300, [1 + i for i in range(300)]),
]


@pytest.mark.parametrize("new, total", APPENDS)
@pytest.mark.parametrize("dim, rot, interleaved, dtype", [(128, 128, False, torch.bfloat16), (80, 40, True, torch.float32),
                                                          (64, 0, False, torch.float32), (256, 64, False, torch.bfloat16),
                                                          (16, 6, True, torch.bfloat16)])
@pytest.mark.parametrize("page, block", [(64, 16), (48, 8), (16, 1), (40, 40)])
def test_cache_append(new, total, dim, rot, interleaved, dtype, page, block):
    g = generator(len(new) + dim)
    batch = Batch(new, total, page, seed=dim)
    heads = 3
    cache = filled_cache(g, batch.pages_held, heads, dim, page, block)
    before = snapshot(cache)
    kv = normal(g, max(batch.tokens, 1), 2, heads, dim, dtype=dtype)[:batch.tokens]
    kv[:, :, 1] *= 3  # one head's scales rise, the others' mostly too
    kv[:, :, 2] *= 0.1  # and one head's stay
    table = xt.RopeTable.build(max(total) + 1, rot, interleaved=interleaved) if rot else None
    xt.cache_append(cache, kv[:, 0], kv[:, 1], *batch.args, rope=table)
    check_append(cache, before, batch, kv[:, 0], kv[:, 1], table)


@pytest.mark.parametrize("dim, rot, interleaved, dtype", [(128, 128, False, torch.float32), (80, 40, True, torch.float32),
                                                          (80, 40, False, torch.bfloat16), (128, 64, True, torch.bfloat16)])
@pytest.mark.parametrize("new, total", [([5 + i % 30 for i in range(100)], [40 + 3 * i for i in range(100)]), ([900], [1000])])
def test_cache_append_many_blocks(new, total, dim, rot, interleaved, dtype):
    """Enough blocks that each belongs to one warp, at the sizes where a few of them would have a CTA each."""
    g = generator(dim)
    batch = Batch(new, total, 64, seed=dim)
    cache = filled_cache(g, batch.pages_held, 8, dim, 64, 16)
    before = snapshot(cache)
    kv = normal(g, batch.tokens, 2, 8, dim, dtype=dtype)
    kv[:, :, 1] *= 3
    kv[:, :, 2] *= 0.1
    table = xt.RopeTable.build(max(total) + 1, rot, interleaved=interleaved)
    xt.cache_append(cache, kv[:, 0], kv[:, 1], *batch.args, rope=table)
    check_append(cache, before, batch, kv[:, 0], kv[:, 1], table)


def test_cache_append_token_by_token_and_at_once():
    """A prompt appended at once and token by token: the same scales, values within the steps of the roundings."""
    g = generator(2)
    page, block, t = 32, 16, 37
    batch = Batch([t], [t], page, seed=1)
    kv = normal(g, t, 2, 2, 64)
    once, steps = (xt.KVCache.empty(batch.pages_held, 2, 64, page=page, block=block) for _ in range(2))
    xt.cache_append(once, kv[:, 0], kv[:, 1], *batch.args)
    for i in range(t):
        starts = torch.tensor([0, 1], dtype=torch.int32).cuda()
        lengths = torch.tensor([i + 1], dtype=torch.int32).cuda()
        xt.cache_append(steps, kv[i:i + 1, 0], kv[i:i + 1, 1], starts, lengths, batch.args[2])
    assert torch.equal(once.k_scale, steps.k_scale) and torch.equal(once.v_scale, steps.v_scale)
    a, b = (xt.dequantize(c.k, c.k_scale, dtype=torch.float32).double() for c in (once, steps))
    # each of at most block - 1 new scales adds half a step at the time, and steps only grow: 8 steps bound block = 16
    bound = 8 * once.k_scale.double().repeat_interleave(block, 2)[..., None]
    within(b, a, bound)


def test_cache_append_zeros_and_nan():
    batch = Batch([2, 2], [2, 20], 16, seed=1)
    cache = filled_cache(generator(1), batch.pages_held, 1, 16, 16, 16)
    k = torch.zeros(4, 1, 16, device="cuda")
    v = torch.ones(4, 1, 16, device="cuda")
    v[3, 0, 4] = float("nan")
    before = snapshot(cache)
    xt.cache_append(cache, k, v, *batch.args)
    into0, into1 = batch.table[0][0], batch.table[1][1]
    assert cache.k_scale[into0, 0, 0] == 0 and (cache.k[into0, 0, :2] == 0).all()
    assert cache.k_scale[into1, 0, 0] == before["k_scale"][into1, 0, 0]  # zeros leave a block's scale
    assert cache.v_scale[into1, 0, 0].isnan()


def test_cache_append_reports_bad_tables():
    batch = Batch([1, 1, 1], [3, 5, 7], 16, seed=1)
    starts, lengths, table = batch.args
    k = torch.ones(3, 1, 16, device="cuda")
    for fault in ("page", "length", "starts", "position"):
        cache = filled_cache(generator(1), batch.pages_held, 1, 16, 16, 16)
        before = snapshot(cache)
        s, n, t, rope = starts.clone(), lengths.clone(), table.clone(), None
        if fault == "page":
            t[1, 0] = batch.pages_held
        elif fault == "length":
            n[1] = 1000
        elif fault == "starts":
            s[3] = 5  # behind the rows that are there
        else:
            rope = xt.RopeTable.build(4, 16)
        xt.cache_append(cache, k, k, s, n, t, rope=rope)
        assert xt.device_error() == (0x301 if fault == "position" else 0x302)
        b = 2 if fault == "starts" else 1
        into = batch.table[b][0]
        if fault == "position":
            assert cache.k_scale[into].isnan().all()
        else:
            assert torch.equal(cache.k[into], before["k"][into])
        assert not torch.equal(cache.k[batch.table[0][0]], before["k"][batch.table[0][0]])


# ------------------------------------------------------------------ attention

def attend_64(cache, batch, q, scale, window, softcap):
    """By the definition, sequence by sequence: the result, the sum of |weight * value|, the largest sum of
    |q_d k_d| * scale and the largest |value|."""
    dim, g = cache.dim, q.shape[1] // cache.heads
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    size, steep, most = torch.zeros_like(out), 0.0, 0.0
    for b, (n, t) in enumerate(zip(batch.new, batch.total)):
        if n == 0 or t == 0:
            continue
        held = torch.tensor(batch.table[b], device="cuda")
        k, v = (((x[held].double().view(len(held), cache.heads, -1, cache.block, dim) * s[held].double()[..., None, None])
                 .view(len(held), cache.heads, cache.page, dim).transpose(0, 1).reshape(cache.heads, -1, dim)[:, :t])
                for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        pos = torch.arange(t - n, t, device="cuda")[:, None]
        j = torch.arange(t, device="cuda")
        seen = j <= pos
        if window:
            seen &= j > pos - window
        rows = q[batch.first[b]:batch.first[b + 1]].double().transpose(0, 1).view(cache.heads, g, n, dim)
        z = rows @ k[:, None].transpose(2, 3) * scale
        steep = max(steep, (rows.abs() @ k[:, None].abs().transpose(2, 3) * scale * seen).max().item())
        most = max(most, v.abs().max().item())
        if softcap:
            z = softcap * torch.tanh(z / softcap)
        z = z.masked_fill(~seen, -math.inf)
        top = z.amax(-1, keepdim=True)
        p = torch.exp(z - torch.where(top > -math.inf, top, 0.0))
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        y, a = p @ v[:, None], p @ v[:, None].abs()
        out[batch.first[b]:batch.first[b + 1]] = y.view(-1, n, dim).transpose(0, 1)
        size[batch.first[b]:batch.first[b + 1]] = a.view(-1, n, dim).transpose(0, 1)
    return out, size, steep, most


def allowed(want, size, steep, most, tokens, dtype):
    # scores: up to dim / 16 = 16 rounded-down steps and 8 roundings of sums up to ``steep``, in the exponent of both the
    # weight and the sum; the sum of the weights: a lane's run of tokens / 4; f32 weights go in with 2^-21
    f32 = 2.0 ** -20 + 2 * 24 * 2 * U * (1 + steep) + U * (tokens / 4 + 40)
    # a weight is an f16 value 2^10 over the row's largest: half a subnormal step is 2^-35 of that one
    lost = 2.0 ** -35 * tokens * most
    if dtype == torch.float32:
        return f32 * size + lost
    # bf16: weights rounded to f16 (2^-11), the result to bf16
    return (f32 + 2.0 ** -11) * size + BF16_STEP * want.abs() + lost


def check_attention(cache, batch, q, window=0, softcap=0.0, scale=None, out=None, **kw):
    y = xt.cache_attention(cache, q, *batch.args, out, window=window, softcap=softcap, scale=scale, **kw)
    want, size, steep, most = attend_64(cache, batch, q, cache.dim ** -0.5 if scale is None else scale, window, softcap)
    within(y, want, allowed(want, size, steep, most, max(batch.total + [0]), q.dtype))
    return y


LENGTHS = [
    ([1], [1]),
    ([1] * 9, [1, 2, 15, 16, 17, 63, 64, 65, 300]),
    ([4, 0, 1, 33], [4, 50, 700, 129]),
    ([0, 0, 7], [0, 3, 7]),
    ([130], [130]),
    ([5, 3], [2, 3]),  # more new tokens than tokens: the first queries see nothing
    ([1, 2], [0, 40]),  # no token at all
]


@pytest.mark.parametrize("new, total", LENGTHS)
@pytest.mark.parametrize("dim, heads, group", [(128, 2, 4), (64, 3, 1), (256, 1, 8), (80, 2, 5), (16, 1, 16), (96, 2, 7),
                                               (128, 1, 32), (192, 2, 2)])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_shapes(new, total, dim, heads, group, dtype):
    g = generator(dim + group)
    page, block = {128: (64, 16), 64: (48, 8), 256: (16, 16), 80: (40, 20), 16: (32, 1)}.get(dim, (64, 64))
    batch = Batch(new, total, page, seed=dim)
    cache = filled_cache(g, batch.pages_held, heads, dim, page, block)
    check_attention(cache, batch, normal(g, batch.tokens, heads * group, dim, std=1.5, dtype=dtype))


@pytest.mark.parametrize("window", [1, 5, 16, 100, 10000])
@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_window_and_cap(window, softcap, dtype):
    g = generator(window)
    batch = Batch([1, 40, 3, 200], [333, 40, 500, 777], 64, seed=3)
    cache = filled_cache(g, batch.pages_held, 2, 128, 64, 16)
    check_attention(cache, batch, normal(g, batch.tokens, 8, 128, dtype=dtype), window=window, softcap=softcap)


@pytest.mark.parametrize("page, block", [(1, 1), (3, 3), (7, 1), (16, 4), (24, 8), (256, 256)])
def test_attention_pages(page, block):
    g = generator(page)
    batch = Batch([1, 20], [100, 75], page, seed=page)
    cache = filled_cache(g, batch.pages_held, 2, 64, page, block)
    check_attention(cache, batch, normal(g, batch.tokens, 4, 64, dtype=torch.bfloat16))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_wide_scales(dtype):
    """Scales from 1e-8 to 1e3 in one sequence, sharp scores, and queries of very different sizes."""
    g = generator(4)
    batch = Batch([1, 3], [900, 400], 64, seed=3)
    cache = filled_cache(g, batch.pages_held, 2, 128, 64, 16)
    spread = torch.empty_like(cache.v_scale).uniform_(math.log(1e-8), math.log(1e3), generator=g)
    cache.v_scale.copy_(spread.exp())
    q = normal(g, batch.tokens, 8, 128, dtype=dtype)
    q[:, ::2] *= 1e-20
    q[:, 1::4] *= 30
    check_attention(cache, batch, q)
    cache.v_scale.mul_(1e-30)
    check_attention(cache, batch, q, scale=1.0)
    cache.v_scale.zero_()
    y = xt.cache_attention(cache, q, *batch.args)
    assert (y == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 3e38])
def test_attention_ignores_what_it_does_not_see(bad):
    """Garbage in a block behind a sequence's end, before its window, and in pages of no sequence."""
    g = generator(6)
    batch = Batch([1, 2], [70, 33], 16, seed=3)
    cache = filled_cache(g, batch.pages_held, 2, 64, 16, 1)
    q = normal(g, batch.tokens, 4, 64, dtype=torch.bfloat16)
    good = check_attention(cache, batch, q, window=20)
    used = torch.zeros_like(cache.k_scale, dtype=torch.bool)
    for b, (n, t) in enumerate(zip(batch.new, batch.total)):
        for j in range(max(0, t - n - 20 + 1), t):
            used[batch.table[b][j // 16], :, j % 16] = True
    for s in (cache.k_scale, cache.v_scale):
        s[~used] = bad
    for c in (cache.k, cache.v):
        c[~used] = -128
    assert torch.equal(xt.cache_attention(cache, q, *batch.args, window=20), good)
    # what is seen comes through
    cache.v_scale[batch.table[0][69 // 16], 0, 69 % 16] = float("nan")
    y = xt.cache_attention(cache, q, *batch.args, window=20)
    assert y[0, :2].isnan().all() and torch.equal(y[0, 2:], good[0, 2:]) and torch.equal(y[1:], good[1:])


def test_attention_nan_query_stays_in_its_row():
    g = generator(7)
    batch = Batch([4], [50], 16, seed=3)
    cache = filled_cache(g, batch.pages_held, 1, 64, 16, 16)
    q = normal(g, 4, 2, 64, dtype=torch.bfloat16)
    good = xt.cache_attention(cache, q, *batch.args)
    q[2, 1, 5] = float("nan")
    y = xt.cache_attention(cache, q, *batch.args)
    assert y[2, 1].isnan().all()
    keep = torch.ones(4, 2, dtype=torch.bool)
    keep[2, 1] = False
    assert torch.equal(y[keep], good[keep])


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_strided_views(dtype):
    g = generator(9)
    batch = Batch([3, 6], [100, 6], 64, seed=3)
    cache = filled_cache(g, batch.pages_held, 2, 64, 64, 16)
    packed = normal(g, batch.tokens, 12 * 64, dtype=dtype)
    q = packed[:, :8 * 64].view(batch.tokens, 8, 64)
    base = torch.full((8, batch.tokens, 64), 5.0, dtype=dtype, device="cuda")
    check_attention(cache, batch, q, out=base.transpose(0, 1))
    wide = torch.cat([batch.args[2], batch.args[2]], 1)[:, :batch.args[2].shape[1]]  # rows of the table further apart
    y = xt.cache_attention(cache, q, batch.args[0], batch.args[1], wide)
    assert torch.equal(y, base.transpose(0, 1))


def test_attention_long_sequence_is_split():
    g = generator(10)
    for new, total in (([1], [50000]), ([1, 1], [7, 30000]), ([6], [20000])):
        batch = Batch(new, total, 64, seed=3)
        cache = filled_cache(g, batch.pages_held, 2, 128, 64, 16)
        for dtype in TYPES:
            q = normal(g, batch.tokens, 8, 128, std=2.0, dtype=dtype)
            y = check_attention(cache, batch, q)
            assert torch.equal(y, xt.cache_attention(cache, q, *batch.args))  # no order of arrival in it


def test_attention_many_sequences():
    g = generator(11)
    total = [1 + (37 * i) % 90 for i in range(1500)]
    batch = Batch([1] * 1500, total, 16, seed=3)
    cache = filled_cache(g, batch.pages_held, 1, 64, 16, 16)
    check_attention(cache, batch, normal(g, 1500, 2, 64, dtype=torch.bfloat16))


def widened(batch, cache, form):
    """The batch with a page table so wide that, as far as the host can tell, its sequences may be very long: their
    tokens are shared out over the whole GPU then, and come as single rows ("rows") or as boxes of rows ("boxes")."""
    starts, lengths, table = batch.args
    tokens = (40 if form == "boxes" else 1) * 16400 * 16 // (cache.heads * max(len(batch.total), 1)) + 1
    if form == "rows":  # but not so long that boxes pay
        assert tokens * len(batch.total) * cache.heads * cache.dim < 64 << 20 or cache.page % 16
    extra = torch.full((table.shape[0], -(-tokens // cache.page)), -9, dtype=torch.int32, device="cuda")
    batch.args = (starts, lengths, torch.cat([table, extra], 1))
    return batch


@pytest.mark.parametrize("form", ["rows", "boxes"])
@pytest.mark.parametrize("new, total", LENGTHS)
@pytest.mark.parametrize("dim, heads, group", [(128, 2, 4), (64, 3, 1), (256, 1, 8), (80, 2, 5), (16, 1, 16), (96, 2, 7),
                                               (128, 1, 32), (192, 2, 2)])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_shapes_shared_out(form, new, total, dim, heads, group, dtype):
    g = generator(dim + group)
    page, block = {128: (64, 16), 64: (48, 8), 256: (16, 16), 80: (40, 20), 16: (32, 1)}.get(dim, (64, 64))
    if form == "rows" and dim > 128:
        page, block = 24, 8
    batch = Batch(new, total, page, seed=dim)
    cache = filled_cache(g, batch.pages_held, heads, dim, page, block)
    widened(batch, cache, form)
    q = normal(g, batch.tokens, heads * group, dim, std=1.5, dtype=dtype)
    y = check_attention(cache, batch, q)
    assert torch.equal(y, xt.cache_attention(cache, q, *batch.args))  # no order of arrival in it


@pytest.mark.parametrize("form", ["rows", "boxes"])
@pytest.mark.parametrize("window, softcap", [(0, 4.0), (1, 0.0), (100, 0.0), (5000, 20.0)])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_long_shared_out(form, window, softcap, dtype):
    g = generator(window)
    batch = Batch([1, 2, 30, 1], [9000, 777, 500, 20000], 64, seed=3)
    cache = filled_cache(g, batch.pages_held, 2, 128, 64, 16)
    widened(batch, cache, form)
    check_attention(cache, batch, normal(g, batch.tokens, 8, 128, std=2.0, dtype=dtype), window=window, softcap=softcap)


@pytest.mark.parametrize("form", ["rows", "boxes"])
def test_attention_edges_shared_out(form):
    """Garbage that nothing sees, NaN that is seen, and wrong tables."""
    g = generator(6)
    batch = Batch([1, 2, 3], [70, 33, 2000], 16, seed=3)
    cache = filled_cache(g, batch.pages_held, 2, 64, 16, 1)
    widened(batch, cache, form)
    q = normal(g, batch.tokens, 4, 64, dtype=torch.bfloat16)
    good = check_attention(cache, batch, q, window=20)
    used = torch.zeros_like(cache.k_scale, dtype=torch.bool)
    for b, (n, t) in enumerate(zip(batch.new, batch.total)):
        for j in range(max(0, t - n - 20 + 1), t):
            used[batch.table[b][j // 16], :, j % 16] = True
    for bad in (float("nan"), float("inf"), 3e38):
        for s in (cache.k_scale, cache.v_scale):
            s[~used] = bad
        for c in (cache.k, cache.v):
            c[~used] = -128
        assert torch.equal(xt.cache_attention(cache, q, *batch.args, window=20), good)
    cache.v_scale[batch.table[0][69 // 16], 0, 69 % 16] = float("nan")
    y = xt.cache_attention(cache, q, *batch.args, window=20)
    assert y[0, :2].isnan().all() and torch.equal(y[0, 2:], good[0, 2:]) and torch.equal(y[1:], good[1:])

    cache = filled_cache(g, batch.pages_held, 2, 64, 16, 1)
    starts, lengths, table = batch.args
    good = xt.cache_attention(cache, q, starts, lengths, table)
    for fault in ("page", "length", "starts"):
        s, n, t = starts.clone(), lengths.clone(), table.clone()
        if fault == "page":
            t[1, 1] = batch.pages_held
        elif fault == "length":
            n[1] = -3
        else:
            s[3] = 9
        y = xt.cache_attention(cache, q, s, n, t)
        assert xt.device_error() == 0x303
        wrong = slice(3, 6) if fault == "starts" else slice(1, 3)
        assert y[wrong].isnan().all(), fault
        assert torch.equal(y[0], good[0])


@pytest.mark.parametrize("seqs, heads, new", [(1, 1, 1), (3, 2, 1), (40, 4, 1), (300, 2, 1), (5, 8, 3), (1, 16, 40)])
@pytest.mark.parametrize("dim, group", [(128, 8), (64, 2), (256, 3)])
def test_attention_clusters(seqs, heads, new, dim, group):
    """Few and many small segments: clusters of every size, rows over several tiles."""
    g = generator(seqs + new)
    total = [max(new, 1 + (97 * i) % 200) for i in range(seqs)]
    batch = Batch([new] * seqs, total, 16, seed=3)
    cache = filled_cache(g, batch.pages_held, heads, dim, 16, 4)
    for dtype in TYPES:
        q = normal(g, batch.tokens, heads * group, dim, dtype=dtype)
        check_attention(cache, batch, q, max_new=new)


@pytest.mark.parametrize("new, total", [([300], [300]), ([257, 64, 500], [1000, 64, 777]), ([128, 1, 129], [2048, 900, 129])])
@pytest.mark.parametrize("dim, group", [(128, 4), (64, 8), (128, 1), (96, 5), (256, 2), (80, 7)])
@pytest.mark.parametrize("window, softcap", [(0, 0.0), (100, 0.0), (0, 20.0)])
def test_attention_prompts(new, total, dim, group, window, softcap):
    g = generator(dim)
    page = 48 if dim == 96 else 64
    batch = Batch(new, total, page, seed=3)
    cache = filled_cache(g, batch.pages_held, 2, dim, page, 16)
    q = normal(g, batch.tokens, 2 * group, dim, std=1.5, dtype=torch.bfloat16)
    y = check_attention(cache, batch, q, window=window, softcap=softcap, max_new=max(new))
    assert y.isfinite().all()


@pytest.mark.parametrize("new, total", [([700, 64, 900], [700, 300, 2500]), ([1700], [1700]), ([33] * 50, [33 + 40 * i for i in range(50)])])
@pytest.mark.parametrize("dim, heads, group, page", [(128, 2, 4, 64), (128, 8, 1, 40), (64, 2, 8, 16), (96, 1, 10, 48), (80, 2, 7, 1),
                                                     (16, 1, 32, 128)])
@pytest.mark.parametrize("window, softcap", [(0, 0.0), (130, 0.0), (0, 20.0), (7, 3.0)])
def test_attention_long_prompts(new, total, dim, heads, group, page, window, softcap):
    """Enough query rows for the kernel that long prompts run in, at every layout it has."""
    g = generator(dim)
    batch = Batch(new, total, page, seed=3)
    cache = filled_cache(g, batch.pages_held, heads, dim, page, 8 if page % 8 == 0 else 1)
    packed = normal(g, batch.tokens, (heads * group + 1) * dim, std=1.5, dtype=torch.bfloat16)
    q = packed[:, :heads * group * dim].view(batch.tokens, heads * group, dim)
    check_attention(cache, batch, q, window=window, softcap=softcap, max_new=max(new))


@pytest.mark.parametrize("new, total", [([64], [2000]), ([128], [1600]), ([512], [1600]), ([70, 3, 90], [4000, 70, 2500])])
@pytest.mark.parametrize("dim, heads, group, page", [(128, 8, 4, 64), (64, 8, 8, 48), (96, 10, 5, 40)])
@pytest.mark.parametrize("window, softcap", [(0, 0.0), (1300, 0.0), (0, 20.0)])
def test_attention_prompt_clusters(new, total, dim, heads, group, page, window, softcap):
    """Few segments of many rows: clusters of two, four and eight that share the tokens of a segment."""
    g = generator(dim + len(new))
    batch = Batch(new, total, page, seed=3)
    cache = filled_cache(g, batch.pages_held, heads, dim, page, 8)
    q = normal(g, batch.tokens, heads * group, dim, std=1.5, dtype=torch.bfloat16)
    y = check_attention(cache, batch, q, window=window, softcap=softcap, max_new=max(new))
    assert torch.equal(y, xt.cache_attention(cache, q, *batch.args, window=window, softcap=softcap, max_new=max(new)))


def test_attention_prompt_cluster_edges():
    """Rows that see nothing, CTAs of a cluster that have no token, NaN in one CTA's share, wrong tables."""
    g = generator(18)
    batch = Batch([128], [1600], 64, seed=3)
    cache = filled_cache(g, batch.pages_held, 8, 128, 64, 1)
    q = normal(g, batch.tokens, 32, 128, std=1.5, dtype=torch.bfloat16)
    starts, lengths, table = batch.args
    good = check_attention(cache, batch, q)
    short = torch.tensor([100], dtype=torch.int32, device="cuda")  # 28 queries before the first token, one tile at most
    y = xt.cache_attention(cache, q, starts, short, table)
    batch.total, batch.args = [100], (starts, short, table)
    assert (y[:28] == 0).all() and torch.equal(y, check_attention(cache, batch, q))
    none = torch.tensor([0], dtype=torch.int32, device="cuda")
    assert (xt.cache_attention(cache, q, starts, none, table) == 0).all()
    where = batch.table[0][700 // 64], 2, 700 % 64
    cache.v_scale[where] = float("nan")
    y = xt.cache_attention(cache, q, starts, lengths, table)
    assert y[:, 8:12].isnan().all() and torch.equal(y[:, :8], good[:, :8]) and torch.equal(y[:, 12:], good[:, 12:])
    cache.v_scale[where] = 0.02
    wrong = table.clone()
    wrong[0, 20] = -1
    assert xt.cache_attention(cache, q, starts, lengths, wrong).isnan().all() and xt.device_error() == 0x303
    over = torch.tensor([1 << 20], dtype=torch.int32, device="cuda")
    assert xt.cache_attention(cache, q, starts, over, table).isnan().all() and xt.device_error() == 0x303


def test_attention_long_prompt_edges():
    """Rows that see nothing, garbage that no row sees, NaN that one sequence's rows see, zero scales, wrong tables."""
    g = generator(16)
    batch = Batch([900, 900, 300], [400, 900, 1500], 64, seed=3)  # the first 500 queries of sequence 0 see nothing
    cache = filled_cache(g, batch.pages_held, 2, 64, 64, 1)
    q = normal(g, batch.tokens, 16, 64, std=1.5, dtype=torch.bfloat16)
    good = check_attention(cache, batch, q)
    assert (good[:500] == 0).all() and torch.equal(good, xt.cache_attention(cache, q, *batch.args))
    used = torch.zeros_like(cache.k_scale, dtype=torch.bool)
    for b, t in enumerate(batch.total):
        for j in range(t):
            used[batch.table[b][j // 64], :, j % 64] = True
    for bad in (float("nan"), float("inf"), 3e38):
        for s in (cache.k_scale, cache.v_scale):
            s[~used] = bad
        assert torch.equal(xt.cache_attention(cache, q, *batch.args), good)
    windowed = check_attention(cache, batch, q, window=50)
    cache.v_scale[batch.table[2][0], 0, 10] = 1e30  # before the window of sequence 2's rows
    cache.k_scale[batch.table[2][0], 0, 11] = float("nan")
    assert torch.equal(xt.cache_attention(cache, q, *batch.args, window=50), windowed)
    y = xt.cache_attention(cache, q, *batch.args)
    assert y[1800:, :8].isnan().all() and torch.equal(y[:1800], good[:1800]) and torch.equal(y[:, 8:], good[:, 8:])
    cache.k_scale[~used] = 0.02
    cache.k_scale[batch.table[2][0], 0, 11] = 0.02
    cache.v_scale.zero_()
    assert (xt.cache_attention(cache, q, *batch.args) == 0).all()
    cache = filled_cache(g, batch.pages_held, 2, 64, 64, 1)
    good = xt.cache_attention(cache, q, *batch.args)
    starts, lengths, table = batch.args
    for fault in ("page", "length", "starts"):
        s, n, t = starts.clone(), lengths.clone(), table.clone()
        if fault == "page":
            t[1, 3] = batch.pages_held
        elif fault == "length":
            n[1] = 1 << 20
        else:
            s[3] = batch.tokens + 5
        y = xt.cache_attention(cache, q, s, n, t)
        assert xt.device_error() == 0x303
        rows = slice(1800, 2100) if fault == "starts" else slice(900 + 3 * 64, 1800) if fault == "page" else slice(900, 1800)
        assert y[rows].isnan().all(), fault
        assert torch.equal(y[:900], good[:900])


def test_attention_long_prompt_scales_and_signs():
    """Value scales of 1e-6 to 1e3 beside each other, a negative and a zero score scale, queries of very different sizes."""
    g = generator(17)
    batch = Batch([800, 600], [1000, 600], 64, seed=3)
    cache = filled_cache(g, batch.pages_held, 2, 128, 64, 16)
    q = normal(g, batch.tokens, 8, 128, dtype=torch.bfloat16)
    q[:, ::2] *= 1e-20
    q[:, 1::4] *= 8
    check_attention(cache, batch, q, scale=-0.1)
    check_attention(cache, batch, q, scale=0.0)
    spread = torch.empty_like(cache.v_scale).uniform_(math.log(1e-6), math.log(1e3), generator=g)
    cache.v_scale.copy_(spread.exp())
    check_attention(cache, batch, q)


def test_attention_hint_does_not_change_what_is_computed():
    g = generator(12)
    batch = Batch([200, 3], [400, 90], 64, seed=3)
    cache = filled_cache(g, batch.pages_held, 2, 128, 64, 16)
    q = normal(g, batch.tokens, 8, 128, dtype=torch.bfloat16)
    for hint in (None, 1, 3, 200, 100000):
        check_attention(cache, batch, q, max_new=hint)


def test_attention_reports_bad_tables():
    g = generator(13)
    batch = Batch([1, 1, 2], [100, 80, 60], 16, seed=3)
    cache = filled_cache(g, batch.pages_held, 1, 64, 16, 16)
    q = normal(g, 4, 2, 64, dtype=torch.bfloat16)
    starts, lengths, table = batch.args
    good = xt.cache_attention(cache, q, starts, lengths, table)
    for fault in ("page", "negative page", "length", "starts"):
        s, n, t = starts.clone(), lengths.clone(), table.clone()
        if fault == "length":
            n[1] = 5000
        elif fault == "starts":
            s[3] = 9
        else:
            t[1, 2] = batch.pages_held if fault == "page" else -1
        y = xt.cache_attention(cache, q, s, n, t)
        assert xt.device_error() == 0x303
        wrong = slice(2, 4) if fault == "starts" else slice(1, 2)
        assert y[wrong].isnan().all(), fault
        assert torch.equal(y[0], good[0])


def test_attention_offsets_past_32_bits():
    """Pages behind 2^31 elements of a cache."""
    heads, dim, page = 8, 128, 64
    pages = (1 << 31) // (heads * dim * page) + 50
    g = generator(14)
    k, v = (torch.empty(pages, heads, page, dim, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(pages, heads, 4, device="cuda") for _ in range(2))
    cache = xt.KVCache(k, v, ks, vs)
    total = [1000]
    small = Batch([1], total, page, seed=3, spare=0)
    last = [pages - 1 - p for p in small.table[0]]
    small.table = [last]
    small.args[2][0, :len(last)] = torch.tensor(last, dtype=torch.int32)
    kv = normal(g, total[0], 2, heads, dim, dtype=torch.bfloat16)
    starts = torch.tensor([0, total[0]], dtype=torch.int32).cuda()
    xt.cache_append(cache, kv[:, 0], kv[:, 1], starts, *small.args[1:])
    held = torch.tensor(last, device="cuda")
    near = xt.KVCache(k[held].contiguous(), v[held].contiguous(), ks[held].contiguous(), vs[held].contiguous())
    flat = Batch([1], total, page, seed=3, spare=0)
    flat.table = [list(range(len(last)))]
    flat.args[2][0, :len(last)] = torch.arange(len(last), dtype=torch.int32)
    q = normal(g, 1, 16, dim, dtype=torch.bfloat16)
    y = check_attention(near, flat, q)
    assert torch.equal(y, xt.cache_attention(cache, q, *small.args))
    want = kv[:, 0].float()
    got = xt.dequantize(near.k, near.k_scale, dtype=torch.float32).transpose(1, 2).reshape(-1, heads, dim)[:total[0]]
    assert (got - want).abs().max() <= 0.51 * ks.max()


# ----------------------------------------------------------------- dequantize

@pytest.mark.parametrize("runs, run", [(1, 1), (7, 1), (3, 5), (100, 16), (33, 17), (1, 1000003), (999, 1000), (64, 2048),
                                       (5000, 3)])
@pytest.mark.parametrize("dtype", TYPES)
def test_dequantize(runs, run, dtype):
    g = generator(run)
    q = torch.randint(-128, 128, (runs, run), generator=g, device="cuda", dtype=torch.int8)
    s = normal(g, runs)
    got = xt.dequantize(q, s, dtype=dtype)
    assert torch.equal(got, (q.float() * s[:, None]).to(dtype))


@pytest.mark.parametrize("run", [4096, 4097])
def test_dequantize_behind_31_bits(run):
    runs = (1 << 31) // run + 3
    q = torch.empty(runs, run, dtype=torch.int8, device="cuda")
    q.view(-1)[:] = 3
    q[-5:] = torch.arange(-60, 60, dtype=torch.int8, device="cuda").repeat(run // 120 + 1)[:run]
    s = torch.arange(runs, device="cuda").float()
    got = xt.dequantize(q, s)
    assert torch.equal(got[-9:], (q[-9:].float() * s[-9:, None]).bfloat16())
    assert torch.equal(got[:, run // 2], (3 * s).bfloat16().where(torch.arange(runs, device="cuda") < runs - 5, got[:, run // 2]))


def test_dequantize_cache_blocks():
    g = generator(1)
    cache = filled_cache(g, 5, 3, 80, 40, 20)
    got = xt.dequantize(cache.v, cache.v_scale, dtype=torch.float32)
    want = cache.v.float().view(5, 3, 2, 20, 80) * cache.v_scale[..., None, None]
    assert torch.equal(got, want.view(5, 3, 40, 80))
    assert xt.dequantize(cache.v[:0], cache.v_scale[:0]).shape == (0, 3, 40, 80)


# ---------------------------------------------------------- streams and graphs

def test_other_streams_and_graphs():
    g = generator(15)
    batch = Batch([1, 1, 1], [40, 100, 9], 16, seed=3)
    heads, dim = 2, 64
    table = xt.RopeTable.build(128, dim)
    weight = normal(g, heads * dim, dtype=torch.bfloat16)
    x, residual = (normal(g, 3, heads * dim, dtype=torch.bfloat16) for _ in range(2))
    kv = normal(g, 3, 2, heads, dim, dtype=torch.bfloat16)
    pos = torch.tensor([39, 99, 8], dtype=torch.int32).cuda()
    start = filled_cache(g, batch.pages_held, heads, dim, 16, 16)

    def step(cache, out, stream=None):
        q8, s = xt.rms_norm(x, weight, residual=residual, dtype=torch.int8, stream=stream)
        q = xt.dequantize(q8, s, stream=stream).view(3, heads, dim)
        xt.rope(q, pos, table, q, stream=stream)
        xt.cache_append(cache, kv[:, 0], kv[:, 1], *batch.args, rope=table, stream=stream)
        return xt.cache_attention(cache, q, *batch.args, out, stream=stream)

    def copy():
        return xt.KVCache(start.k.clone(), start.v.clone(), start.k_scale.clone(), start.v_scale.clone())

    want = step(copy(), None).clone()
    side = torch.cuda.Stream()
    cache = copy()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = step(cache, None)
    side.synchronize()
    assert torch.equal(y, want)
    cache, out = copy(), torch.empty_like(want)
    side.wait_stream(torch.cuda.current_stream())
    held = step(cache, out, stream=side)  # the call's own stream, while another is current
    side.synchronize()
    assert torch.equal(held, want)

    cache, out = copy(), torch.zeros_like(want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cache, out)
    assert (out == 0).all()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# ------------------------------------------------------------------- refusals

def test_refusals():
    x = torch.zeros(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    refused = pytest.raises
    with refused(ValueError, match="shape"):
        xt.rms_norm(x, w[:32])
    with refused(TypeError, match="residual"):
        xt.rms_norm(x, w, residual=x.bfloat16())
    with refused(ValueError, match="expected"):
        xt.rms_norm(x, w.cpu())
    with refused(ValueError, match="contiguous"):
        xt.rms_norm(x.t(), torch.ones(4, device="cuda"))
    with refused(ValueError, match="broadcast"):
        xt.rms_norm(x, w, torch.empty(1, 64, device="cuda").expand(4, 64))
    with refused(ValueError, match="scales"):
        xt.rms_norm(x, w, scales=torch.empty(4, device="cuda"))
    with refused(TypeError, match="out"):
        xt.rms_norm(x, w, x.half())
    table = xt.RopeTable.build(8, 32)
    heads = torch.zeros(4, 2, 64, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    with refused(TypeError, match="positions"):
        xt.rope(heads, pos.long(), table)
    with refused(ValueError, match="turn"):
        xt.rope(heads[..., :16], pos, table)
    with refused(TypeError, match="RopeTable"):
        xt.rope(heads, pos, table.cos_sin)
    with refused(TypeError, match="out"):
        xt.rope(heads.bfloat16(), pos, table, heads)
    cache = xt.KVCache.empty(4, 2, 64)
    starts = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([4], dtype=torch.int32, device="cuda")
    pages = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    with refused(ValueError, match="shape"):
        xt.cache_append(cache, heads[..., :32], heads[..., :32], starts, lengths, pages)
    with refused(TypeError, match="v must"):
        xt.cache_append(cache, heads, heads.bfloat16(), starts, lengths, pages)
    with refused(ValueError, match="starts"):
        xt.cache_append(cache, heads, heads, starts[:1], lengths, pages)
    with refused(TypeError, match="lengths"):
        xt.cache_append(cache, heads, heads, starts, lengths.long(), pages)
    with refused(ValueError, match="turn"):
        xt.cache_append(cache, heads, heads, starts, lengths, pages, rope=xt.RopeTable.build(8, 128))
    with refused(ValueError, match="fit"):
        xt.cache_attention(cache, heads[:, :1], starts, lengths, pages)
    with refused(ValueError, match="multiples of four"):
        xt.cache_attention(cache, torch.zeros(4, 2, 66, device="cuda")[..., 1:65], starts, lengths, pages)
    with refused(ValueError, match="softcap"):
        xt.cache_attention(cache, heads, starts, lengths, pages, softcap=-2.0)
    with refused(ValueError, match="dim must be"):
        xt.KVCache.empty(2, 2, 72)
    with refused(ValueError, match="equal runs"):
        xt.dequantize(cache.k, torch.ones(7, device="cuda"))
    with refused(TypeError, match="float32 or bfloat16"):
        xt.dequantize(cache.k, cache.k_scale, dtype=torch.float16)
