"""The serving operators' argument checks that need no GPU: the C entry points
through ctypes, and the Python calls on wrong types and CPU tensors."""
import ctypes
from pathlib import Path

import pytest
import torch

import xtile as xt

LIB = ctypes.CDLL(str(Path(__file__).resolve().parents[1] / "xtile_b200" / "libxt_b200.so"))
LIB.xt_last_error.restype = ctypes.c_char_p
P, I, L, F, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t
F32, BF16, I8 = 0, 1, 2
ARGUMENT = 5  # XT_EARGUMENT


def struct(name, fields):
    return type(name, (ctypes.Structure,), {"_fields_": fields})


Norm = struct("Norm", [("x", P), ("residual", P), ("weight", P), ("y", P), ("sum", P), ("scales", P), ("rows", L),
                       ("cols", L), ("x_stride", L), ("residual_stride", L), ("y_stride", L), ("sum_stride", L),
                       ("elem", I), ("weight_elem", I), ("y_elem", I), ("eps", F)])
Rope = struct("Rope", [("x", P), ("y", P), ("positions", P), ("table", P), ("tokens", L), ("heads", L), ("dim", L),
                       ("rot", L), ("table_rows", L), ("x_token", L), ("x_head", L), ("y_token", L), ("y_head", L),
                       ("elem", I), ("y_elem", I), ("interleaved", I), ("inverse", I)])
Cache = struct("Cache", [("k", P), ("v", P), ("k_scale", P), ("v_scale", P), ("pages", L), ("heads", I), ("page", I),
                         ("dim", I), ("block", I)])
Batch = struct("Batch", [("starts", P), ("lengths", P), ("table", P), ("seqs", I), ("tokens", I), ("table_width", I),
                         ("table_stride", L)])
Append = struct("Append", [("cache", Cache), ("batch", Batch), ("k", P), ("v", P), ("k_token", L), ("k_head", L),
                           ("v_token", L), ("v_head", L), ("rope", P), ("rot", L), ("rope_rows", L), ("elem", I),
                           ("interleaved", I)])
Attend = struct("Attend", [("cache", Cache), ("batch", Batch), ("q", P), ("out", P), ("q_token", L), ("q_head", L),
                           ("out_token", L), ("out_head", L), ("q_heads", I), ("max_new", I), ("window", I),
                           ("scale", F), ("softcap", F), ("elem", I), ("workspace", P), ("workspace_bytes", Z)])
AT = 1 << 20  # an aligned address that no check reads


def norm(**kw):
    return Norm(**{**dict(x=AT, weight=AT, y=AT, scales=AT, rows=4, cols=64, x_stride=64, y_stride=64, elem=BF16,
                          weight_elem=BF16, y_elem=I8, eps=1e-6), **kw})


def rope(**kw):
    return Rope(**{**dict(x=AT, y=AT, positions=AT, table=AT, tokens=4, heads=2, dim=64, rot=64, table_rows=10,
                          x_token=128, x_head=64, y_token=128, y_head=64, elem=BF16, y_elem=BF16), **kw})


def parts(kw):
    cache = dict(k=AT, v=AT, k_scale=AT, v_scale=AT, pages=4, heads=2, page=64, dim=64, block=16)
    batch = dict(starts=AT, lengths=AT, table=AT, seqs=2, tokens=4, table_width=2, table_stride=2)
    for k in list(kw):
        for d in (cache, batch):
            if k in d:
                d[k] = kw.pop(k)
    return dict(cache=Cache(**cache), batch=Batch(**batch))


@pytest.mark.parametrize("args, word", [
    (norm(cols=0), "cols"), (norm(rows=-1), "rows"), (norm(elem=I8), "x and weight"), (norm(weight_elem=3), "weight"),
    (norm(y_elem=3), "y must be"), (norm(scales=None), "scales"), (norm(x=None), "null"), (norm(y=None), "null"),
    (norm(x=AT + 1), "aligned"), (norm(rows=1 << 31), "too many"),
])
def test_rms_norm_refuses(args, word):
    assert LIB.xt_rms_norm(ctypes.byref(args), None) == ARGUMENT
    assert word in LIB.xt_last_error().decode()


@pytest.mark.parametrize("args, word", [
    (rope(dim=63), "dim"), (rope(rot=65), "rot"), (rope(rot=66), "rot"), (rope(rot=-2), "rot"), (rope(x=None), "null"),
    (rope(positions=None), "null"), (rope(elem=BF16, y_elem=F32), "types"), (rope(elem=I8), "types"),
    (rope(table=AT + 4), "aligned"), (rope(tokens=-1), "dim must be"), (rope(tokens=1 << 32), "too many"),
])
def test_rope_refuses(args, word):
    assert LIB.xt_rope(ctypes.byref(args), None) == ARGUMENT
    assert word in LIB.xt_last_error().decode()


CACHE_FAULTS = [
    (dict(dim=72), "dim"), (dict(dim=272), "dim"), (dict(dim=0), "dim"), (dict(block=15), "whole blocks"),
    (dict(pages=0), "positive"), (dict(heads=0), "positive"), (dict(page=0, block=1), "positive"),
    (dict(k_scale=None), "null"), (dict(k=AT + 8), "16-byte"), (dict(starts=None), "null"), (dict(table=None), "null"),
    (dict(seqs=-1), "negative"), (dict(table_width=1 << 30), "too wide"),
]


@pytest.mark.parametrize("kw, word", CACHE_FAULTS + [
    (dict(elem=I8), "f32 or bf16"), (dict(rope=AT, rot=7), "rot"), (dict(rope=AT, rot=66), "rot"),
    (dict(rope=AT, rot=0), "rot"), (dict(rope=AT, rot=64), "no positions"), (dict(k_in=None), "null"),
])
def test_cache_append_refuses(kw, word):
    kw = dict(kw)
    given = kw.pop("k_in", AT)
    base = parts(kw)
    args = Append(**base, **{**dict(elem=BF16), **kw})
    args.k, args.v = given, AT
    assert LIB.xt_cache_append(ctypes.byref(args), None) == ARGUMENT
    assert word in LIB.xt_last_error().decode()


@pytest.mark.parametrize("kw, word", CACHE_FAULTS + [
    (dict(elem=I8), "f32 or bf16"), (dict(q_heads=3), "multiple"), (dict(q_heads=0), "multiple"),
    (dict(window=-1), "negative"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"),
    (dict(q=None), "null"), (dict(q=AT + 4), "aligned"), (dict(q_head=6), "multiples of four"),
])
def test_cache_attention_refuses(kw, word):
    kw = dict(kw)
    base = parts(kw)
    args = Attend(**base, **{**dict(q=AT, out=AT, q_token=128, q_head=64, out_token=128, out_head=64, q_heads=2,
                                    scale=0.125, elem=BF16), **kw})
    assert LIB.xt_cache_attention(ctypes.byref(args), None) == ARGUMENT
    assert word in LIB.xt_last_error().decode()


def test_cache_attention_needs_its_workspace():
    args = Attend(**parts(dict(table_width=1 << 16, table_stride=1 << 16)), q=AT, out=AT, q_heads=2, scale=0.125, elem=BF16)
    need = ctypes.c_size_t()
    assert LIB.xt_cache_attention_workspace(ctypes.byref(args), ctypes.byref(need)) == 0
    args.workspace, args.workspace_bytes = AT, max(need.value, 1) - 1
    assert need.value > 0 and LIB.xt_cache_attention(ctypes.byref(args), None) == ARGUMENT
    assert "workspace" in LIB.xt_last_error().decode()


def test_dequantize_refuses():
    call = lambda q, s, o, n, run, elem: LIB.xt_dequantize(P(q), P(s), P(o), L(n), L(run), I(elem), None)  # noqa: E731
    assert call(AT, AT, AT, -1, 1, F32) == ARGUMENT
    assert call(AT, AT, AT, 16, 0, F32) == ARGUMENT
    assert call(AT, AT, AT, 16, 16, I8) == ARGUMENT
    assert call(None, AT, AT, 16, 16, F32) == ARGUMENT
    assert call(AT + 4, AT, AT, 16, 16, F32) == ARGUMENT
    assert call(None, None, None, 0, 16, F32) == 0  # nothing to do


def test_nothing_to_do_needs_no_arrays():
    assert LIB.xt_rms_norm(ctypes.byref(Norm(rows=0, cols=64, elem=F32, y_elem=F32)), None) == 0
    assert LIB.xt_rope(ctypes.byref(Rope(tokens=0, heads=1, dim=64, rot=64)), None) == 0
    args = Append(**parts(dict(tokens=0)), elem=BF16)
    assert LIB.xt_cache_append(ctypes.byref(args), None) == 0
    args = Attend(**parts(dict(seqs=0)), q_heads=2, elem=BF16)
    assert LIB.xt_cache_attention(ctypes.byref(args), None) == 0


def test_python_calls_refuse_cpu_tensors_and_wrong_types():
    x, w = torch.zeros(4, 64), torch.ones(64)
    with pytest.raises(ValueError, match="CUDA"):
        xt.rms_norm(x, w)
    with pytest.raises(TypeError, match="torch tensor"):
        xt.rms_norm([1.0], w)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        xt.rms_norm(x.half(), w)
    with pytest.raises(ValueError, match="CUDA"):
        xt.rope(torch.zeros(4, 2, 64), None, None)
    with pytest.raises(ValueError, match="CUDA"):
        xt.RopeTable(torch.zeros(4, 32, 2))
    with pytest.raises(ValueError, match="rot"):
        xt.RopeTable.build(10, 7)
    with pytest.raises(ValueError, match="factor"):
        xt.RopeTable.build(10, 8, factor=0.5)
    with pytest.raises(ValueError, match="CUDA"):
        xt.KVCache.empty(2, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="whole blocks"):
        xt.KVCache.empty(2, 2, 64, page=64, block=24, device="cpu")
    with pytest.raises(TypeError, match="int8"):
        xt.dequantize(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        xt.dequantize(x.to(torch.int8), w)


def test_the_example_names_the_device_error(monkeypatch):
    import importlib.util

    spec = importlib.util.spec_from_file_location("serve_attention", Path(__file__).resolve().parents[1] / "examples" / "serve_attention.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    codes = [0x303, 0]  # read and cleared
    monkeypatch.setattr(example.xt, "device_error", lambda: codes.pop(0))
    with pytest.raises(RuntimeError, match="0x303"):
        example.raise_for_device_error()
    example.raise_for_device_error()


def test_cache_attention_refuses_an_infinite_cap():
    base = parts({})
    args = Attend(**base, q=AT, out=AT, q_token=128, q_head=64, out_token=128, out_head=64, q_heads=2, scale=0.125,
                  elem=BF16, softcap=float("inf"))  # its tanh is 0 and the product of both NaN
    assert LIB.xt_cache_attention(ctypes.byref(args), None) == ARGUMENT
    assert "softcap" in LIB.xt_last_error().decode()
