"""The serving example against its layers written out in 64 bits.

The tolerance: the cache holds keys and values as int8, off by up to half a
step of max|x| / 127, 2^-8 of their block's largest; a score sums dim products
of such errors, which have no common sign, so weights are off by a few percent
of themselves at most and a mean of values by 2^-8 of the largest value and as
much again; bf16 rows and products add 2^-8 of an operand's size.  Every layer
adds such errors of its own: 3 percent of the output's largest magnitude for two.
"""
import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


def load():
    spec = importlib.util.spec_from_file_location("serve_attention", ROOT / "examples" / "serve_attention.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain(server, x):
    """A whole sequence x [tokens, width] through the layers, causal, in 64 bits and without a cache."""
    h, y = torch.zeros_like(x, dtype=torch.float64), x.double()
    cs = server.table.cos_sin.double()[:x.shape[0], None]
    for layer in server.layers:
        h = h + y
        n = h * (h.square().mean(1, keepdim=True) + 1e-6).rsqrt() * layer.norm.double()
        qkv = (n @ layer.qkv.w.double()).view(x.shape[0], -1, layer.dim)
        q, k, v = qkv.split([layer.q_heads, layer.kv_heads, layer.kv_heads], dim=1)

        def turned(z):
            a, b = z.chunk(2, dim=2)
            return torch.cat([a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]], dim=2)

        group = layer.q_heads // layer.kv_heads
        q, k, v = turned(q), turned(k).repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        z = torch.einsum("ihd,jhd->hij", q, k) * layer.dim ** -0.5
        z = z.masked_fill(torch.ones_like(z[0], dtype=torch.bool).triu(1), float("-inf"))
        y = torch.einsum("hij,jhd->ihd", z.softmax(2), v).reshape(x.shape[0], -1) @ layer.out.w.double()
    return h + y


def test_serving_example():
    example = load()
    prompts, steps = [70, 1, 200], 5
    server = example.Server(prompts, steps, width=512, q_heads=4, kv_heads=2, dim=64, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(4)
    xs = [torch.randn(n + steps, 512, generator=gen, device="cuda") for n in prompts]
    got = [[part] for part in server.prefill(torch.cat([x[:n] for x, n in zip(xs, prompts)])).split(prompts)]
    for i in range(steps):
        y = server.decode(torch.stack([x[n + i] for x, n in zip(xs, prompts)]))
        for b, row in enumerate(y.clone()):
            got[b].append(row[None])
    import xtile as xt

    assert xt.device_error() == 0
    assert server.lengths.tolist() == [n + steps for n in prompts]
    for b, x in enumerate(xs):
        want, y = plain(server, x), torch.cat(got[b]).double()
        assert (y - want).abs().max() <= 0.03 * want.abs().max(), b
        keys, values = server.cached(0, b, len(x))
        assert keys.shape == (len(x), 2, 64) and keys.isfinite().all() and values.abs().max() > 0
