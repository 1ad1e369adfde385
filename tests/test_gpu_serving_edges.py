"""The serving operators where a call meets the rest of a program: streams and
their memory, wrong tables, waits that run out, and values at the edges of
their types.  Tolerances are those of ``test_gpu_serving``."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import xtile as xt
from tests.test_gpu_serving import Batch, allowed, attend_64, filled_cache, generator, normal, widened, within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    assert xt.device_error() == 0


# -------------------------------------------------------------------- streams

def owner(t):
    """The stream whose pool of torch's allocator a tensor's memory is from."""
    at = t.data_ptr()
    return next(s["stream"] for s in torch.cuda.memory_snapshot() if s["address"] <= at < s["address"] + s["total_size"])


def allocating_calls():
    """Every call that allocates its results, as functions of the stream."""
    g = generator(21)
    x, w = normal(g, 64, 512, dtype=torch.bfloat16), normal(g, 512)
    heads = x.view(64, 4, 128)
    table = xt.RopeTable.build(64, 128)
    pos = torch.arange(64, device="cuda", dtype=torch.int32)
    batch = Batch([30, 34], [90, 70], 64, seed=3)
    cache = filled_cache(g, batch.pages_held, 2, 128, 64, 16)
    return {
        "norm": lambda s: [xt.rms_norm(x, w, stream=s)],
        "int8 norm": lambda s: list(xt.rms_norm(x, w, dtype=torch.int8, stream=s)),
        "rope": lambda s: [xt.rope(heads, pos, table, stream=s)],
        "attention": lambda s: [xt.cache_attention(cache, heads, *batch.args, stream=s)],
        "dequantize": lambda s: [xt.dequantize(cache.k, cache.k_scale, stream=s)],
    }


@pytest.mark.parametrize("handle", [False, True])
def test_results_are_of_the_calls_stream(handle):
    """With ``stream`` given its pool has what the call allocates, else the current stream's has it."""
    side = torch.cuda.Stream()
    for name, call in allocating_calls().items():
        want = call(None)
        assert all(owner(t) == 0 for t in want), name
        side.wait_stream(torch.cuda.current_stream())
        got = call(side.cuda_stream if handle else side)
        side.synchronize()
        for a, b in zip(got, want):
            assert owner(a) == side.cuda_stream, name
            assert torch.equal(a, b), name


def test_a_result_takes_no_memory_that_its_stream_does_not_own():
    """A tensor dropped while its stream has yet to read it is not written by a call on another stream."""
    side = torch.cuda.Stream()
    for name, call in allocating_calls().items():
        like = call(None)[0]
        torch.cuda.synchronize()
        held = torch.full_like(like, 3)
        seen = torch.empty_like(like)
        side.wait_stream(torch.cuda.current_stream())
        torch.cuda._sleep(20_000_000)  # about 10 ms
        seen.copy_(held)
        del held  # the current stream's pool may give it out again, to that stream
        call(side)
        torch.cuda.synchronize()
        assert (seen == 3).all(), name


# --------------------------------------------------------------- wrong tables

def starts_of(new, first=0):
    s = [first]
    for n in new:
        s.append(s[-1] + n)
    return s


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# new tokens of three sequences: one slot a token, and one a block
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 3, 70]])
@pytest.mark.parametrize("page, block", [(16, 16), (48, 8)])
def test_append_reports_every_wrong_start(new, page, block):
    a, b, c = new
    batch = Batch(new, [n + 20 for n in new], page, seed=1)
    lengths, table = batch.args[1:]
    k = normal(generator(1), a + b + c, 2, 64)
    start = filled_cache(generator(2), batch.pages_held, 2, 64, page, block)

    def append(starts, lengths=lengths):
        cache = xt.KVCache(start.k.clone(), start.v.clone(), start.k_scale.clone(), start.v_scale.clone())
        xt.cache_append(cache, k, k, ints(starts), lengths, table)
        return cache

    def pages_of(cache, b):
        held = torch.tensor(batch.table[b], device="cuda")
        return [t[held] for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]

    def same(x, y, b):
        return all(torch.equal(s, t) for s, t in zip(pages_of(x, b), pages_of(y, b)))

    good = append(starts_of(new))
    assert xt.device_error() == 0 and not any(same(good, start, b) for b in range(3))
    # starts that fall: a sequence that is wrong by itself is not stored, any other one may be missed
    for wrong in ([0, a + b, a, a + b + c], [0, a, -1, a + b + c], [a, 0, a + b, a + b + c], [0, a, a + b, a - 1]):
        cache = append(wrong)
        assert xt.device_error() == 0x302, wrong
        assert all(same(cache, start, b) for b in range(3) if not 0 <= wrong[b] <= wrong[b + 1]), wrong
    # a negative start: the others' tokens are stored
    for wrong in ([-1, a, a + b, a + b + c], [-1000, a, a + b, a + b + c]):
        cache = append(wrong)
        assert xt.device_error() == 0x302, wrong
        assert same(cache, start, 0) and same(cache, good, 1) and same(cache, good, 2), wrong
    # sequences without a token, or behind all rows
    for wrong, n in (([-5, -5, -2, 0], lengths), ([1000, 1000, 1001, 1002], lengths), ([0, 0, 0, 0], ints([5, -1, 5])),
                     ([0, 0, 0, 0], ints([5, 1 << 20, 5]))):
        cache = append(wrong, n)
        assert xt.device_error() == 0x302, wrong
        assert all(same(cache, start, b) for b in range(3)), wrong


# the forms of the attention: clusters, runs of units over the GPU, whole prompts, prompts in clusters
FORMS = {
    "clusters": (([20, 3, 30], [70, 33, 60]), 64, 8, None),
    "rows": (([20, 3, 30], [70, 33, 60]), 64, 8, "rows"),
    "boxes": (([20, 3, 30], [70, 33, 60]), 64, 8, "boxes"),
    "prompts": (([2000, 500, 900], [2000, 700, 1500]), 64, 8, None),
    "prompt clusters": (([70, 3, 90], [4000, 70, 2500]), 128, 4, None),
}


def form_case(form):
    (new, total), dim, group, wide = FORMS[form]
    heads = 8 if form == "prompt clusters" else 2
    dtype = torch.bfloat16 if "prompt" in form else torch.float32
    batch = Batch(new, total, 64, seed=3)
    cache = filled_cache(generator(5), batch.pages_held, heads, dim, 64, 16)
    if wide:
        widened(batch, cache, wide)
    return new, batch, cache, normal(generator(6), batch.tokens, heads * group, dim, std=1.5, dtype=dtype)


@pytest.mark.parametrize("form", FORMS)
def test_attention_reports_every_wrong_start(form):
    new, batch, cache, q = form_case(form)
    (a, b, c), most = new, max(new)
    lengths, table = batch.args[1:]
    attend = lambda starts, n=lengths: xt.cache_attention(cache, q, ints(starts), n, table, max_new=most)  # noqa: E731
    want, *rest = attend_64(cache, batch, q, cache.dim ** -0.5, 0, 0.0)
    off = allowed(want, *rest, max(batch.total), q.dtype)
    within(attend(starts_of(new)), want, off)
    for wrong in ([0, a + b, a, a + b + c], [0, a, -1, a + b + c], [a, 0, a + b, a + b + c], [0, a, a + b, a - 1]):
        y = attend(wrong)
        assert xt.device_error() == 0x303, wrong
        assert y.isnan().all(), wrong  # starts that fall: no row is sure
    for wrong in ([-1, a, a + b, a + b + c], [-1000, a, a + b, a + b + c]):
        y = attend(wrong)
        assert xt.device_error() == 0x303, wrong
        assert y[:a].isnan().all(), wrong
        within(y[a:], want[a:], off[a:])
    for wrong, n in (([-5, -5, -2, 0], lengths), ([100000, 100000, 100001, 100002], lengths), ([0, 0, 0, 0], ints([5, -1, 5])),
                     ([0, 0, 0, 0], ints([5, 1 << 30, 5]))):
        attend(wrong, n)
        assert xt.device_error() == 0x303, wrong


# --------------------------------------------------------- waits that run out

def rows_good_or_nan(y, good):
    """Every head of a token is what it should be, or NaN throughout.  How many are NaN."""
    lost = y.isnan().all(-1)
    assert torch.equal(y[~lost], good[~lost])
    return int(lost.sum())


WAITS = {
    # new, total, q heads, kv heads, dim, type, form
    "clusters": ([1] * 30, [100 + 60 * i for i in range(30)], 16, 4, 128, torch.bfloat16, None),
    "one warp a segment": ([1] * 600, [96] * 600, 4, 4, 128, torch.bfloat16, None),
    "rows": ([1] * 60, [2000 + 40 * i for i in range(60)], 16, 4, 128, torch.bfloat16, "rows"),
    "boxes": ([1, 3] * 16, [4000 + 100 * i for i in range(32)], 32, 8, 128, torch.bfloat16, "boxes"),
    "many segments a warp": ([1] * 1200, [20 + i % 50 for i in range(1200)], 8, 8, 128, torch.bfloat16, "boxes"),
}


@pytest.mark.parametrize("case", WAITS)
def test_attention_waits_run_out(case):
    """A wait limit of 1 ns: warps that find a tile not yet there give up, their rows are NaN, and the next call is
    whole again.  No copy is lost or held back: every one lands before its warp ends."""
    new, total, q_heads, heads, dim, dtype, form = WAITS[case]
    batch = Batch(new, total, 64, seed=3)
    cache = filled_cache(generator(5), batch.pages_held, heads, dim, 64, 16)
    if form:
        widened(batch, cache, form)
    q = normal(generator(6), batch.tokens, q_heads, dim, std=1.5, dtype=dtype)
    good = xt.cache_attention(cache, q, *batch.args, max_new=max(new))
    assert good.isfinite().all() and xt.device_error() == 0
    flush = torch.empty(1 << 28, dtype=torch.int8, device="cuda")
    for _ in range(100):
        flush.zero_()  # the tiles come from far, the queries do not
        y = torch.zeros_like(q) + q * 0
        with xt.wait_limit(1):
            xt.cache_attention(cache, q, *batch.args, y, max_new=max(new))
        lost = rows_good_or_nan(y, good)
        code = xt.device_error()
        assert code == (0x307 if lost else 0)
        if lost:
            break
    assert lost, "no wait ran out"
    assert torch.equal(xt.cache_attention(cache, q, *batch.args, max_new=max(new)), good)


@pytest.mark.parametrize("limit_ns", [1, 1000, 3000])
@pytest.mark.parametrize("new, total, dim, heads, group, window, softcap", [
    ([700, 64, 900], [700, 300, 2500], 128, 2, 4, 0, 0.0),
    ([700, 64, 900], [700, 300, 2500], 64, 2, 8, 130, 0.0),
    ([1700], [1700], 96, 1, 10, 0, 20.0),
    ([128], [1600], 128, 8, 4, 0, 0.0),  # clusters, as the two below
    ([70, 3, 90], [4000, 70, 2500], 128, 8, 4, 1300, 0.0),
    ([512], [1600], 64, 8, 8, 0, 20.0),
])
def test_attention_prompt_waits_run_out(new, total, dim, heads, group, window, softcap, limit_ns):
    """The tcgen05 kernel's waits run out: every row is whole or NaN, the products that were issued land, the tensor
    memory is freed, and the next call is whole again."""
    batch = Batch(new, total, 64, seed=3)
    cache = filled_cache(generator(5), batch.pages_held, heads, dim, 64, 16)
    q = normal(generator(6), batch.tokens, heads * group, dim, std=1.5, dtype=torch.bfloat16)
    attend = lambda out=None: xt.cache_attention(cache, q, *batch.args, out, window=window, softcap=softcap,  # noqa: E731
                                                 max_new=max(new))
    good = attend()
    assert good.isfinite().all() and xt.device_error() == 0
    for _ in range(3):
        y = torch.zeros_like(q)
        with xt.wait_limit(limit_ns):
            attend(y)
        lost = rows_good_or_nan(y, good)
        code = xt.device_error()
        assert code in ((0x304, 0x305) if lost else (0,))
        assert lost or limit_ns > 1
        assert torch.equal(attend(), good) and xt.device_error() == 0


def test_attention_prompt_waits_have_their_codes():
    """At once the softmax warps give up; with 2000 cycles, which the scores take less than and a stage's way through
    softmax and products more, the converting ones do."""
    batch = Batch([700, 64, 900], [700, 300, 2500], 64, seed=3)
    cache = filled_cache(generator(5), batch.pages_held, 2, 128, 64, 16)
    q = normal(generator(6), batch.tokens, 8, 128, std=1.5, dtype=torch.bfloat16)
    for limit_ns, code in ((1, 0x304), (1000, 0x305)):
        with xt.wait_limit(limit_ns):
            xt.cache_attention(cache, q, *batch.args, max_new=900)
        assert xt.device_error() == code


# --------------------------------------------------------------- sizes at edges

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("new", [[1, 1], [40, 30], [700, 900]])
def test_attention_of_an_empty_page_table(new, dtype):
    """No page at all and so no token: every row is 0."""
    cache = filled_cache(generator(1), 3, 2, 64, 16, 16)
    q = normal(generator(2), sum(new), 16, 64, dtype=dtype)
    pages = torch.empty(2, 0, dtype=torch.int32, device="cuda")
    y = torch.full_like(q, 7)
    xt.cache_attention(cache, q, ints(starts_of(new)), ints([0, 0]), pages, y, max_new=max(new))
    assert (y == 0).all()
    xt.cache_attention(cache, q, ints(starts_of(new)), ints([0, 5]), pages, y, max_new=max(new))
    assert xt.device_error() == 0x303
    assert (y[:new[0]] == 0).all() and y[new[0]:].isnan().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_of_the_widest_window(dtype):
    """The largest window there is hides nothing, also behind queries that see no token."""
    batch = Batch([900, 300], [400, 1500], 64, seed=3)
    cache = filled_cache(generator(1), batch.pages_held, 2, 64, 64, 16)
    q = normal(generator(2), batch.tokens, 16, 64, dtype=dtype)
    want = xt.cache_attention(cache, q, *batch.args, max_new=900)
    for window in (1 << 30, (1 << 31) - 1):
        assert torch.equal(xt.cache_attention(cache, q, *batch.args, max_new=900, window=window), want)


@pytest.mark.parametrize("block", [1, 16])
@pytest.mark.parametrize("sign", [1, -1])
def test_infinities_do_not_come_back_as_values(block, sign):
    """int8 data that cannot hold an infinity says so: its scale is NaN, like that of a NaN."""
    batch = Batch([3], [20], 16, seed=1)
    cache = filled_cache(generator(1), batch.pages_held, 2, 64, 16, block)
    before = cache.k_scale.clone()
    k = normal(generator(2), 3, 2, 64)
    v = k.clone()
    k[1, 0, 5] = sign * float("inf")
    xt.cache_append(cache, k, v, *batch.args)
    into, row = batch.table[0][1], 18 % 16
    assert cache.k_scale[into, 0, row // block].isnan()
    assert cache.k_scale[into, 1].isfinite().all() and cache.v_scale.isfinite().all()
    assert torch.equal(cache.k_scale[batch.table[0][0]], before[batch.table[0][0]])
    y = xt.cache_attention(cache, k.nan_to_num(posinf=1, neginf=1), *batch.args)
    assert y[1:, 0].isnan().all() and y[:, 1].isfinite().all()
    x, w = torch.ones(2, 64, device="cuda"), torch.ones(64, device="cuda")
    w[3] = sign * float("inf")
    assert xt.rms_norm(x, w, dtype=torch.int8)[1].isnan().all()


# ------------------------------------------------------------ torch's own rules

def test_written_tensors_have_a_new_version():
    """Autograd finds a tensor that was saved and then written by its version, as after torch's own in-place calls."""
    g = generator(3)
    x, w = normal(g, 4, 128, dtype=torch.bfloat16), normal(g, 128)
    r, total, y = x.clone(), torch.empty_like(x), torch.empty_like(x)
    q8, s = torch.empty(4, 128, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
    heads, pos, table = x.view(4, 2, 64), ints([0, 1, 2, 3]), xt.RopeTable.build(8, 64)
    batch = Batch([4], [4], 16, seed=1)
    cache = filled_cache(g, batch.pages_held, 2, 64, 16, 16)
    turned, seen, back = torch.empty_like(heads), torch.empty_like(heads), torch.empty_like(cache.k, dtype=torch.float32)
    calls = [
        (lambda: xt.rms_norm(x, w, y, residual=r, residual_out=total), [y, total], [x, w, r]),
        (lambda: xt.rms_norm(x, w, q8, scales=s), [q8, s], [x, w]),
        (lambda: xt.rope(heads, pos, table, turned), [turned], [heads, pos, table.cos_sin]),
        (lambda: xt.cache_append(cache, heads, heads, *batch.args, rope=table),
         [cache.k, cache.v, cache.k_scale, cache.v_scale], [heads, *batch.args]),
        (lambda: xt.cache_attention(cache, heads, *batch.args, seen), [seen], [heads, cache.k, cache.v_scale]),
        (lambda: xt.dequantize(cache.k, cache.k_scale, back), [back], [cache.k, cache.k_scale]),
    ]
    for i, (call, written, read) in enumerate(calls):
        before = [t._version for t in written], [t._version for t in read]
        call()
        assert all(t._version > v for t, v in zip(written, before[0])), i
        assert all(t._version == v for t, v in zip(read, before[1])), i
    with torch.inference_mode():
        held = torch.empty_like(heads)
    xt.rope(heads, pos, table, held)  # has no version
    assert torch.equal(held, turned)
    leaf = x.float().requires_grad_()
    square = (leaf * 1).square_()
    saved = square * square
    xt.rms_norm(square.detach(), w, square.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.sum().backward()


def test_a_flag_without_a_truth_value_is_refused():
    x, pos, table = torch.ones(4, 2, 64, device="cuda"), ints([0, 1, 2, 3]), xt.RopeTable.build(8, 64)
    with pytest.raises(RuntimeError, match="ambiguous"):
        xt.rope(x, pos, table, inverse=torch.ones(2))
    table.interleaved = torch.ones(2)
    with pytest.raises(RuntimeError, match="ambiguous"):
        xt.rope(x, pos, table)


FIRST_IN_A_GRAPH = """
import torch, xtile as xt
x = torch.randn(600, 512, device="cuda").bfloat16(); w = torch.ones(512, device="cuda")
heads = x.view(600, 8, 64); kv = heads[:, :2]
ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
args = ints([0, 600]), ints([600]), torch.arange(4096, dtype=torch.int32, device="cuda").view(1, -1) % 10
one = ints([0, 1]), args[1], args[2]
pos = torch.arange(600, dtype=torch.int32, device="cuda")
table, cache = xt.RopeTable.build(600, 64), xt.KVCache.empty(10, 2, 64)
def calls():
    xt.cache_append(cache, kv, kv, *args, rope=table)
    q8, s = xt.rms_norm(x, w, dtype=torch.int8)
    q = xt.rope(xt.dequantize(q8, s).view(600, 8, 64), pos, table)
    return (xt.cache_attention(cache, q, *args, max_new=600), xt.cache_attention(cache, q[-1:], *one, max_new=1),
            xt.cache_attention(cache, q[-1:], one[0], one[1], args[2][:, :10], max_new=1))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, calls())) and xt.device_error() == 0
print("whole")
"""


def test_the_first_calls_may_be_captured():
    """A process whose first calls are captured in a graph: nothing that they set up breaks the capture."""
    run = subprocess.run([sys.executable, "-c", FIRST_IN_A_GRAPH], capture_output=True, text=True, timeout=300,
                         cwd=Path(__file__).resolve().parents[1])
    assert run.returncode == 0 and "whole" in run.stdout, run.stderr[-2000:]


# ------------------------------------------------------------- what bits are held

@pytest.mark.parametrize("new, total", [([1], [300]), ([400], [700])])
def test_small_elements_of_a_bf16_query(new, total):
    """A row's elements of 2^-20 to 2^-40 of its largest, before keys that are 0 where that one is: what they score is
    off by half a step of the f16 that they enter as, 2^-35 of the row's largest each."""
    batch = Batch(new, total, 64, seed=3)
    cache = filled_cache(generator(1), batch.pages_held, 2, 128, 64, 16)
    cache.k[..., 0] = 0
    q = normal(generator(2), batch.tokens, 16, 128, dtype=torch.float32)
    q *= 2.0 ** -torch.randint(20, 41, q.shape, generator=generator(3), device="cuda").float()
    q[..., 0] = 1.0
    q = q.bfloat16()
    scale = 2.0 ** 20
    y = xt.cache_attention(cache, q, *batch.args, scale=scale, max_new=max(new))
    want, *rest = attend_64(cache, batch, q, scale, 0, 0.0)
    keys = cache.k.float().view(-1, 2, 4, 16, 128) * cache.k_scale[..., None, None]
    off = scale * 2.0 ** -35 * keys.abs().sum(-1).max().item()  # of a score, in the exponent of a weight and of the sum
    assert 2 ** -10 < off < 2 ** -4  # far over the rounding of the scores' sums
    within(y, want, allowed(want, *rest, max(total), q.dtype) + 2.2 * off * rest[0])


@pytest.mark.parametrize("new, total", [([1], [300]), ([400], [700])])
def test_the_largest_bf16_queries(new, total):
    """Queries up to the end of their range, whose scores a small scale brings back."""
    batch = Batch(new, total, 64, seed=3)
    cache = filled_cache(generator(1), batch.pages_held, 2, 128, 64, 16)
    q = normal(generator(2), batch.tokens, 16, 128, dtype=torch.float32)
    q = (q * 2.0 ** torch.arange(110, 126, device="cuda").float()[:, None]).bfloat16()  # sizes head by head
    assert q.isfinite().all() and q.abs().max() > 1e38
    for scale in (2.0 ** -126, 2.0 ** -110):
        y = xt.cache_attention(cache, q, *batch.args, scale=scale, max_new=max(new))
        want, *rest = attend_64(cache, batch, q, scale, 0, 0.0)
        within(y, want, allowed(want, *rest, max(total), q.dtype))


@pytest.mark.parametrize("new, total", [([1] * 4, [307, 250, 120, 77]), ([1, 1], [3000, 2000]), ([5, 40], [900, 700])])
@pytest.mark.parametrize("dim, heads, group", [(256, 4, 1), (256, 2, 8), (128, 4, 4), (80, 2, 16)])
def test_f32_attention_holds_its_bits(new, total, dim, heads, group):
    """The 2-norm of the error, of scores of about 1.  Root mean squares of what a weight is off by: exp2 2^-22.7, the
    query's and the weight's two f16 terms 2^-23 each, four partial scores of eight sums, each rounded toward zero by
    2^-24 of half a score, 2^-21.9; together 3.5e-7, and a mean of values is off by as much.  Twice that is allowed."""
    batch = Batch(new, total, 64, seed=3)
    cache = filled_cache(generator(1), batch.pages_held, heads, dim, 64, 16, 0.015, 0.035)
    q = normal(generator(2), batch.tokens, heads * group, dim)
    want = attend_64(cache, batch, q, dim ** -0.5, 0, 0.0)[0]
    y = xt.cache_attention(cache, q, *batch.args, max_new=max(new))
    assert (y.double() - want).norm() <= 7e-7 * want.norm()


# ------------------------------------------------------------------ int8 chains

@xt.kernel
def int8_product(rows, w, by_column, out, tm, tn, tk):
    i, j = xt.bid(0), xt.bid(1)
    p = xt.matmul(xt.load(rows, index=(i, 0), shape=(tm, tk)), xt.load(w, index=(0, j), shape=(tk, tn), shared=1))
    xt.store(out, index=(i, j), tile=p * xt.load(by_column, index=(0, j), shape=(1, tn)))


@xt.kernel
def rows_scaled(p, by_row, out, tm, tn):
    i, j = xt.bid(0), xt.bid(1)
    xt.store(out, index=(i, j), tile=xt.load(p, index=(i, j), shape=(tm, tn)) * xt.load(by_row, index=(i, 0), shape=(tm, 1)))


def test_int8_rows_through_an_int8_product():
    """``rms_norm``'s int8 rows times int8 weights: the matmul program scales the columns, a program behind it the rows."""
    m, k, n = 256, 512, 384
    g = generator(9)
    x, w = normal(g, m, k, dtype=torch.bfloat16), normal(g, k)
    q8, s = xt.rms_norm(x, w, dtype=torch.int8)
    w8 = torch.randint(-127, 128, (k, n), generator=g, device="cuda", dtype=torch.int8)
    columns = torch.rand(1, n, generator=g, device="cuda")
    product, y = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
    A = xt.Array
    xt.launch(xt.convert(int8_product, args=(A((m, k), xt.int8), A((k, n), xt.int8), A((1, n), xt.float32), A((m, n), xt.float32),
                                             128, 128, k), grid=(m // 128, n // 128, 1)), q8, w8, columns, product)
    xt.launch(xt.convert(rows_scaled, args=(A((m, n), xt.float32), A((m, 1), xt.float32), A((m, n), xt.float32), 8, n),
                         grid=(m // 8, 1, 1)), product, s.view(m, 1), y)
    want = (q8.double() @ w8.double()) * columns.double() * s.double()[:, None]
    within(y, want, 3 * 2.0 ** -24 * want.abs())  # whole numbers under 2^24, times two scales
