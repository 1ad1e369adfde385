"""The operators between the matmuls of a decoder layer when a model answers.

``rms_norm`` (with the residual's addition, to f32, bf16 or int8 rows),
``rope``, an int8 paged cache (``KVCache``) with ``cache_append`` and
``cache_attention``, and ``dequantize``.  They take torch CUDA tensors the way
``launch`` does: results are written in place into the tensors given for them
(allocated where ``out`` is left out), the call is asynchronous on ``stream``
(default: torch's current stream of the tensors' device), and a wrong argument
raises ``TypeError`` (types) or ``ValueError`` (shapes, devices, layouts)
before anything runs.  Positions, lengths and page tables live on the device:
an entry outside the arrays is not followed, and ``device_error()`` reports it
(0x301 rope, 0x302 append, 0x303 attention).

A ragged batch is described by three int32 tensors: ``starts`` [seqs + 1],
``lengths`` [seqs] and ``pages`` [seqs, width].  Sequence ``b`` has
``lengths[b]`` tokens; the last ``starts[b + 1] - starts[b]`` of them are new
and are rows ``starts[b]`` .. of the packed arrays [tokens, heads, dim].  Its
token ``j`` lies in row ``j % page`` of cache page ``pages[b, j // page]``.
"""
from __future__ import annotations

import math

from ._native import native as _native

_F32, _BF16, _I8 = 0, 1, 2
_ELEM: dict = {}
_torch = None


def _load_torch():
    """torch, imported at the first call: the package itself does not need it."""
    global _torch
    if _torch is None:
        import torch

        _ELEM.update({torch.float32: _F32, torch.bfloat16: _BF16, torch.int8: _I8})
        _torch = torch
    return _torch


def _floats(name, t, rank):
    """Element code of a CUDA tensor of f32 or bf16 values whose last axis is contiguous."""
    torch = _torch or _load_torch()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
    elem = _ELEM.get(t.dtype)
    if elem is None or elem == _I8:
        raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dim() != rank:
        raise ValueError(f"{name} must have {rank} axes, got shape {tuple(t.shape)}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}'s last axis must be contiguous")
    return elem


def _like(name, t, shape, dtype, device):
    """Checks a tensor that goes with others: its type, shape, device and contiguous last axis."""
    if not isinstance(t, _torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}'s last axis must be contiguous")


def _written(name, t):
    """A result's elements must lie apart: no broadcast axis."""
    for n, s in zip(t.shape, t.stride()):
        if s == 0 and n > 1:
            raise ValueError(f"{name} is written and must not be broadcast")


def _call(fn, device, stream, *args):
    """Runs a native launcher on ``stream`` with the tensors' device current."""
    torch = _torch
    if stream is None:
        stream = torch.cuda.current_stream(device)
    handle = stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)
    if torch.cuda.current_device() == device.index:
        fn(*args, handle)
    else:
        with torch.cuda.device(device):
            fn(*args, handle)


def rms_norm(x, weight, out=None, *, residual=None, residual_out=None, scales=None, eps: float = 1e-6, dtype=None,
             stream=None):
    """``h * rsqrt(mean(h^2) + eps) * weight`` of each row of ``h = x + residual``.

    ``x`` [rows, cols] is f32 or bf16, ``residual`` and ``residual_out`` (which
    receives h, and may be ``residual`` or ``x``) are like it; ``weight`` [cols]
    is f32 or bf16.  ``out`` is f32, bf16 or int8 (``dtype`` chooses where it is
    left out; default x's).  Int8 rows carry one f32 scale each in ``scales``
    [rows]: ``int8 = rint(value / scale)``, ``scale = max|value| / 127``.
    Returns ``out``, for int8 rows ``(out, scales)``.
    """
    elem = _floats("x", x, 2)
    torch = _torch
    device, shape = x.device, x.shape
    rows, cols = shape
    if not isinstance(weight, torch.Tensor) or _ELEM.get(weight.dtype, _I8) == _I8:
        raise TypeError("weight must be a float32 or bfloat16 tensor")
    _like("weight", weight, (cols,), weight.dtype, device)
    if out is None:
        out = torch.empty(shape, dtype=dtype or x.dtype, device=device)
        if out.dtype not in _ELEM:
            raise TypeError(f"out must be float32, bfloat16 or int8, got {out.dtype}")
    else:
        if not isinstance(out, torch.Tensor) or out.dtype not in _ELEM or (dtype is not None and out.dtype != dtype):
            raise TypeError(f"out must be a {dtype or 'float32, bfloat16 or int8'} tensor")
        _like("out", out, shape, out.dtype, device)
        _written("out", out)
    y_elem = _ELEM[out.dtype]
    if y_elem == _I8:
        if scales is None:
            scales = torch.empty(rows, dtype=torch.float32, device=device)
        else:
            _like("scales", scales, (rows,), torch.float32, device)
    elif scales is not None:
        raise ValueError("scales go with int8 rows only")
    if residual is not None:
        _like("residual", residual, shape, x.dtype, device)
    if residual_out is not None:
        _like("residual_out", residual_out, shape, x.dtype, device)
        _written("residual_out", residual_out)
    _call(_native.rms_norm, device, stream, x.data_ptr(), residual.data_ptr() if residual is not None else 0,
          weight.data_ptr(), out.data_ptr(), residual_out.data_ptr() if residual_out is not None else 0,
          scales.data_ptr() if scales is not None else 0, rows, cols, x.stride(0),
          residual.stride(0) if residual is not None else 0, out.stride(0),
          residual_out.stride(0) if residual_out is not None else 0, elem, _ELEM[weight.dtype], y_elem, eps)
    return (out, scales) if y_elem == _I8 else out


class RopeTable:
    """Cosines and sines of every position and frequency, and how a head's pairs lie.

    ``cos_sin`` is an f32 CUDA tensor [positions, rot / 2, 2]; the first ``rot``
    elements of a head turn.  Pair ``i`` is elements ``(2i, 2i + 1)`` if
    ``interleaved``, else ``(i, i + rot / 2)``.
    """

    def __init__(self, cos_sin, interleaved: bool = False) -> None:
        _floats("cos_sin", cos_sin, 3)
        if cos_sin.dtype != _torch.float32:
            raise TypeError(f"cos_sin must be float32, got {cos_sin.dtype}")
        if cos_sin.shape[1] < 1 or cos_sin.shape[2] != 2 or not cos_sin.is_contiguous():
            raise ValueError(f"cos_sin must be contiguous [positions, rot / 2, 2], got shape {tuple(cos_sin.shape)}")
        self.cos_sin = cos_sin
        self.positions, self.rot = cos_sin.shape[0], 2 * cos_sin.shape[1]
        self.interleaved = bool(interleaved)

    @classmethod
    def build(cls, positions: int, rot: int, *, base: float = 10000.0, interleaved: bool = False, factor: float = 1.0,
              trained: int = 0, low: float = 1.0, high: float = 32.0, amplitude: float = 1.0,
              device="cuda") -> "RopeTable":
        """The table of frequencies ``base ** (-2i / rot)``, computed in 64 bits.

        ``factor`` > 1 stretches it for contexts longer than the trained one:
        every frequency is divided by ``factor``, or, where ``trained`` gives the
        trained length, only those that turn fewer than ``low`` times over it; the
        ones that turn more than ``high`` times stay, those between are blended
        linearly in their turns.  ``amplitude`` multiplies all cosines and sines.
        """
        torch = _load_torch()
        if rot < 2 or rot % 2 or positions < 0:
            raise ValueError("rot must be even and positive, and positions not negative")
        if factor < 1 or (trained and not 0 <= low < high):
            raise ValueError("factor must be at least 1 and low below high")
        freq = float(base) ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
        if trained:
            turns = trained * freq / (2 * math.pi)
            keep = ((turns - low) / (high - low)).clamp(0, 1)
            freq = freq * (keep + (1 - keep) / factor)
        else:
            freq = freq / factor
        angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
        cos_sin = torch.stack([angle.cos(), angle.sin()], dim=-1) * amplitude
        return cls(cos_sin.float().to(device).contiguous(), interleaved)


def rope(x, positions, table: RopeTable, out=None, *, inverse: bool = False, stream=None):
    """Turns each head of ``x`` [tokens, heads, dim] to its token's position.

    ``positions`` [tokens] is int32.  ``out`` is like ``x``, or bf16 for f32
    input; it may be ``x`` itself.  ``inverse`` turns back: the gradient of the
    forward call with respect to x is ``rope(grad, ..., inverse=True)``.
    """
    elem = _floats("x", x, 3)
    torch = _torch
    tokens, heads, dim = x.shape
    device = x.device
    if not isinstance(table, RopeTable):
        raise TypeError(f"table must be a RopeTable, got {type(table).__name__}")
    if table.cos_sin.device != device:
        raise ValueError(f"table is on {table.cos_sin.device}, expected {device}")
    if dim % 2 or table.rot > dim:
        raise ValueError(f"heads of {dim} elements cannot turn {table.rot} of them")
    _like("positions", positions, (tokens,), torch.int32, device)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=device)
    else:
        dtype = torch.bfloat16 if elem == _F32 and getattr(out, "dtype", None) == torch.bfloat16 else x.dtype
        _like("out", out, x.shape, dtype, device)
        _written("out", out)
    _call(_native.rope, device, stream, x.data_ptr(), out.data_ptr(), positions.data_ptr(), table.cos_sin.data_ptr(),
          tokens, heads, dim, table.rot, table.positions, x.stride(0), x.stride(1), out.stride(0), out.stride(1), elem,
          _ELEM[out.dtype], table.interleaved, inverse)
    return out


class KVCache:
    """A paged cache of int8 keys and values with one f32 scale for each block of tokens and head.

    ``k`` and ``v`` are int8 [pages, heads, page, dim], ``k_scale`` and
    ``v_scale`` f32 [pages, heads, page / block]; a stored value stands for
    ``int8 * scale``.  ``KVCache.empty`` allocates one.
    """

    def __init__(self, k, v, k_scale, v_scale) -> None:
        torch = _load_torch()
        if not isinstance(k, torch.Tensor) or k.dtype != torch.int8:
            raise TypeError("k must be an int8 tensor")
        if not k.is_cuda:
            raise ValueError("k must be a CUDA tensor")
        if k.dim() != 4:
            raise ValueError(f"k must be [pages, heads, page, dim], got shape {tuple(k.shape)}")
        _like("v", v, k.shape, torch.int8, k.device)
        pages, heads, page, dim = k.shape
        blocks = k_scale.shape[-1] if isinstance(k_scale, torch.Tensor) and k_scale.dim() == 3 else 0
        if blocks < 1 or page % blocks:
            raise ValueError("k_scale must be [pages, heads, page / block]")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            _like(name, t, (pages, heads, blocks), torch.float32, k.device)
        if not all(t.is_contiguous() for t in (k, v, k_scale, v_scale)):
            raise ValueError("the cache's tensors must be contiguous")
        if dim % 16 or not 16 <= dim <= 256:
            raise ValueError(f"dim must be a multiple of 16 up to 256, got {dim}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.heads, self.page, self.dim, self.block = pages, heads, page, dim, page // blocks
        self.device = k.device
        self._view = _native.CacheView(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, heads,
                                       page, dim, self.block)

    @classmethod
    def empty(cls, pages: int, heads: int, dim: int, *, page: int = 64, block: int = 16, device="cuda") -> "KVCache":
        torch = _load_torch()
        if block < 1 or page % block:
            raise ValueError("a page must hold whole blocks")
        shape = (pages, heads, page, dim)
        k, v = (torch.zeros(shape, dtype=torch.int8, device=device) for _ in range(2))
        ks, vs = (torch.zeros(shape[:2] + (page // block,), dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, ks, vs)


def _batch(cache, starts, lengths, pages):
    """The three tensors of a ragged batch, checked: (pointers, seqs, width, stride)."""
    torch = _torch
    if not isinstance(cache, KVCache):
        raise TypeError(f"cache must be a KVCache, got {type(cache).__name__}")
    if not isinstance(lengths, torch.Tensor) or lengths.dim() != 1:
        raise ValueError("lengths must be an int32 tensor [seqs]")
    seqs = lengths.shape[0]
    device = cache.device
    _like("lengths", lengths, (seqs,), torch.int32, device)
    _like("starts", starts, (seqs + 1,), torch.int32, device)
    if not isinstance(pages, torch.Tensor) or pages.dim() != 2:
        raise ValueError("pages must be an int32 tensor [seqs, width]")
    _like("pages", pages, (seqs, pages.shape[1]), torch.int32, device)
    return starts.data_ptr(), lengths.data_ptr(), pages.data_ptr(), seqs, pages.shape[1], pages.stride(0)


def cache_append(cache: KVCache, k, v, starts, lengths, pages, *, rope: RopeTable | None = None, stream=None) -> None:
    """Stores the new tokens' keys (turned to their positions if ``rope`` is given) and values.

    ``k`` and ``v`` [tokens, heads, dim] are f32 or bf16; ``lengths`` already
    counts the new tokens.  A block's scale becomes the larger of its old one (if
    it holds earlier tokens) and ``max|x| / 127`` of its new tokens; where it
    rises, the rows of the earlier tokens are rounded anew to it.
    """
    elem = _floats("k", k, 3)
    starts_p, lengths_p, pages_p, seqs, width, stride = _batch(cache, starts, lengths, pages)
    tokens = k.shape[0]
    _like("k", k, (tokens, cache.heads, cache.dim), k.dtype, cache.device)
    _like("v", v, k.shape, k.dtype, cache.device)
    table, rot, positions, interleaved = 0, 0, 0, False
    if rope is not None:
        if not isinstance(rope, RopeTable):
            raise TypeError(f"rope must be a RopeTable, got {type(rope).__name__}")
        if rope.cos_sin.device != cache.device:
            raise ValueError(f"rope is on {rope.cos_sin.device}, expected {cache.device}")
        if rope.rot > cache.dim:
            raise ValueError(f"heads of {cache.dim} elements cannot turn {rope.rot} of them")
        table, rot, positions, interleaved = rope.cos_sin.data_ptr(), rope.rot, rope.positions, rope.interleaved
    _call(_native.cache_append, cache.device, stream, cache._view, starts_p, lengths_p, pages_p, seqs, tokens, width,
          stride, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1), table, rot, positions,
          elem, interleaved)


def cache_attention(cache: KVCache, q, starts, lengths, pages, out=None, *, max_new: int | None = None,
                    scale: float | None = None, window: int = 0, softcap: float = 0.0, stream=None):
    """Attention of the new tokens' queries over their sequences' cached tokens.

    ``q`` [tokens, q_heads, dim] is f32 or bf16, ``out`` like it; consecutive
    ``q_heads / heads`` query heads share a cache head.  A query sees its
    sequence's tokens up to its own (the last ``window`` of them if window > 0); one
    that sees none gives 0.  ``scale`` defaults to ``dim ** -0.5``; ``softcap`` > 0
    caps the scaled scores by ``softcap * tanh(score / softcap)``.  ``max_new``, the
    most new tokens of one sequence, helps to choose the kernel; results do not
    depend on it.
    """
    elem = _floats("q", q, 3)
    torch = _torch
    starts_p, lengths_p, pages_p, seqs, width, stride = _batch(cache, starts, lengths, pages)
    tokens, q_heads, dim = q.shape
    device = cache.device
    if q.device != device:
        raise ValueError(f"q is on {q.device}, expected {device}")
    if dim != cache.dim or q_heads < 1 or q_heads % cache.heads:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {cache.heads} heads of {cache.dim}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
    else:
        _like("out", out, q.shape, q.dtype, device)
        _written("out", out)
    if stream is None:
        stream = torch.cuda.current_stream(device)
    need = _native.cache_attention_workspace(cache._view, seqs, tokens, width, q_heads, max_new or 0, elem)
    workspace = 0
    if need:
        # scratch of this call alone, from the allocator's pool of the stream that it runs on
        if hasattr(stream, "cuda_stream") and stream != torch.cuda.current_stream(device):
            with torch.cuda.stream(stream):
                scratch = torch.empty(need, dtype=torch.uint8, device=device)
        else:
            scratch = torch.empty(need, dtype=torch.uint8, device=device)
        workspace = scratch.data_ptr()
    _call(_native.cache_attention, device, stream, cache._view, starts_p, lengths_p, pages_p, seqs, tokens, width,
          stride, q.data_ptr(), out.data_ptr(), q.stride(0), q.stride(1), out.stride(0), out.stride(1), q_heads,
          max_new or 0, window, dim ** -0.5 if scale is None else scale, softcap, elem, workspace, need)
    return out


def dequantize(q, scales, out=None, *, dtype=None, stream=None):
    """The values that int8 data stands for: ``q * scales``, one scale for each equal run of elements.

    ``rms_norm``'s rows and their scales, or a cache's ``k`` and ``k_scale`` (whose
    blocks are contiguous): the run is ``q.numel() / scales.numel()`` elements.
    ``out`` is f32 or bf16 (``dtype`` chooses where it is left out; default bf16).
    """
    torch = _load_torch()
    if not isinstance(q, torch.Tensor) or q.dtype != torch.int8:
        raise TypeError("q must be an int8 tensor")
    if not q.is_cuda:
        raise ValueError("q must be a CUDA tensor")
    if not isinstance(scales, torch.Tensor) or scales.dtype != torch.float32:
        raise TypeError("scales must be a float32 tensor")
    device = q.device
    if scales.device != device:
        raise ValueError(f"scales is on {scales.device}, expected {device}")
    n, runs = q.numel(), scales.numel()
    if (n and not runs) or (runs and n % runs):
        raise ValueError(f"{n} elements do not divide into {runs} equal runs")
    if out is None:
        out = torch.empty(q.shape, dtype=dtype or torch.bfloat16, device=device)
    else:
        _like("out", out, q.shape, dtype or getattr(out, "dtype", None), device)
    elem = _ELEM.get(out.dtype, _I8)
    if elem == _I8:
        raise TypeError(f"out must be float32 or bfloat16, got {out.dtype}")
    if not (q.is_contiguous() and scales.is_contiguous() and out.is_contiguous()):
        raise ValueError("q, scales and out must be contiguous")
    if n:
        _call(_native.dequantize, device, stream, q.data_ptr(), scales.data_ptr(), out.data_ptr(), n, n // runs, elem)
    return out
