"""The serving operators where a call meets the rest of a program: streams and
their memory, wrong tables, waits that run out, and values at the edges of
their types.  Tolerances are those of ``test_gpu_serving``."""
import pytest
import torch

import xtile as xt
from tests.test_gpu_serving import Batch, filled_cache, generator, normal

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
