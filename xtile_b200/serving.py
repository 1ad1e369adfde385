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
(0x301 rope, 0x302 append, 0x303 attention; where ``starts`` fall, append may
miss other sequences too, and every row of an attention is NaN; 0x304, 0x305 and
0x307 are bounded waits of the attention kernels that ran out, whose rows are
NaN).

With ``stream`` given, that stream owns what the call allocates, as under
``torch.cuda.stream(stream)``: another stream waits for it before it reads the
result, and calls ``record_stream`` on a result that is dropped while its own
reads are under way.  The same holds for the call's inputs on ``stream``.

The calls are outside autograd: results carry no gradient, whatever the inputs
require, and a tensor that is written gets a new version, so that a backward
pass that saved it finds out.

A ragged batch is described by three int32 tensors: ``starts`` [seqs + 1],
``lengths`` [seqs] and ``pages`` [seqs, width].  Sequence ``b`` has
``lengths[b]`` tokens; the last ``starts[b + 1] - starts[b]`` of them are new
and are rows ``starts[b]`` .. of the packed arrays [tokens, heads, dim].  Its
token ``j`` lies in row ``j % page`` of cache page ``pages[b, j // page]``.
"""
from __future__ import annotations

import importlib
import math

_native = None


def _load():
    """The extension over torch tensors, loaded with torch at the first use: the package itself needs neither."""
    global _native
    if _native is None:
        import torch  # noqa: F401  (its libraries come first)

        try:
            _native = importlib.import_module("xtile_b200._serving")
        except ImportError as exc:  # pragma: no cover - exercised only on an unbuilt tree
            raise ImportError("the xtile_b200 serving extension is not built; run `python xtile_b200/build.py` "
                              f"(or __graft_entry__.build()) first: {exc}") from exc
    return _native


def rms_norm(x, weight, out=None, *, residual=None, residual_out=None, scales=None, eps: float = 1e-6, dtype=None,
             stream=None):
    """``h * rsqrt(mean(h^2) + eps) * weight`` of each row of ``h = x + residual``.

    ``x`` [rows, cols] is f32 or bf16, ``residual`` and ``residual_out`` (which
    receives h, and may be ``residual`` or ``x``) are like it; ``weight`` [cols]
    is f32 or bf16.  ``out`` is f32, bf16 or int8 (``dtype`` chooses where it is
    left out; default x's).  Int8 rows carry one f32 scale each in ``scales``
    [rows]: ``int8 = rint(value / scale)``, ``scale = max|value| / 127`` (NaN for a
    row with a NaN or an infinity).  A matmul program takes such rows as they are,
    and a program behind it multiplies the product's rows by ``scales``: its own
    epilogue scales columns only.
    Returns ``out``, for int8 rows ``(out, scales)``.
    """
    return (_native or _load()).rms_norm(x, weight, out, residual, residual_out, scales, eps, dtype, stream)


class RopeTable:
    """Cosines and sines of every position and frequency, and how a head's pairs lie.

    ``cos_sin`` is an f32 CUDA tensor [positions, rot / 2, 2]; the first ``rot``
    elements of a head turn.  Pair ``i`` is elements ``(2i, 2i + 1)`` if
    ``interleaved``, else ``(i, i + rot / 2)``.
    """

    def __init__(self, cos_sin, interleaved: bool = False) -> None:
        (_native or _load()).check_table(cos_sin)
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
        import torch

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
    cos_sin, interleaved = (table.cos_sin, table.interleaved) if isinstance(table, RopeTable) else (None, False)
    return (_native or _load()).rope(x, positions, cos_sin, interleaved, out, inverse, stream)


class KVCache:
    """A paged cache of int8 keys and values with one f32 scale for each block of tokens and head.

    ``k`` and ``v`` are int8 [pages, heads, page, dim], ``k_scale`` and
    ``v_scale`` f32 [pages, heads, page / block]; a stored value stands for
    ``int8 * scale``.  ``KVCache.empty`` allocates one.
    """

    def __init__(self, k, v, k_scale, v_scale) -> None:
        (_native or _load()).check_cache(k, v, k_scale, v_scale)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.heads, self.page, self.dim = k.shape
        self.block = self.page // k_scale.shape[2]
        self.device = k.device

    @classmethod
    def empty(cls, pages: int, heads: int, dim: int, *, page: int = 64, block: int = 16, device="cuda") -> "KVCache":
        import torch

        if block < 1 or page % block:
            raise ValueError("a page must hold whole blocks")
        shape = (pages, heads, page, dim)
        k, v = (torch.zeros(shape, dtype=torch.int8, device=device) for _ in range(2))
        ks, vs = (torch.zeros(shape[:2] + (page // block,), dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, ks, vs)


def _no_cache(cache):
    raise TypeError(f"cache must be a KVCache, got {type(cache).__name__}")


def cache_append(cache: KVCache, k, v, starts, lengths, pages, *, rope: RopeTable | None = None, stream=None) -> None:
    """Stores the new tokens' keys (turned to their positions if ``rope`` is given) and values.

    ``k`` and ``v`` [tokens, heads, dim] are f32 or bf16; ``lengths`` already
    counts the new tokens.  A block's scale becomes the larger of its old one (if
    it holds earlier tokens) and ``max|x| / 127`` of its new tokens; where it
    rises, the rows of the earlier tokens are rounded anew to it.  A NaN or an
    infinity makes its block's scale NaN.
    """
    if not isinstance(cache, KVCache):
        _no_cache(cache)
    cos_sin, interleaved = None, False
    if rope is not None:
        if not isinstance(rope, RopeTable):
            raise TypeError(f"rope must be a RopeTable, got {type(rope).__name__}")
        cos_sin, interleaved = rope.cos_sin, rope.interleaved
    (_native or _load()).cache_append(cache.k, cache.v, cache.k_scale, cache.v_scale, k, v, starts, lengths, pages,
                                      cos_sin, interleaved, stream)


def cache_attention(cache: KVCache, q, starts, lengths, pages, out=None, *, max_new: int | None = None,
                    scale: float | None = None, window: int = 0, softcap: float = 0.0, stream=None):
    """Attention of the new tokens' queries over their sequences' cached tokens.

    ``q`` [tokens, q_heads, dim] is f32 or bf16, ``out`` like it; consecutive
    ``q_heads / heads`` query heads share a cache head.  A query sees its
    sequence's tokens up to its own (the last ``window`` of them if window > 0); one
    that sees none gives 0, and a row of no sequence stays as it is.  Heads start
    on four elements' bytes; prompts of bf16 queries whose heads start on 16 bytes
    can run on the tensor cores' own kernel.  ``scale`` defaults to ``dim ** -0.5``; ``softcap`` > 0
    caps the scaled scores by ``softcap * tanh(score / softcap)``.  ``max_new``, the
    most new tokens of one sequence, helps to choose the kernel; it changes
    nothing that is computed, only the order of sums and so their last bits.
    """
    if not isinstance(cache, KVCache):
        _no_cache(cache)
    return (_native or _load()).cache_attention(cache.k, cache.v, cache.k_scale, cache.v_scale, q, starts, lengths,
                                                pages, out, max_new, scale, window, softcap, stream)


def dequantize(q, scales, out=None, *, dtype=None, stream=None):
    """The values that int8 data stands for: ``q * scales``, one scale for each equal run of elements.

    ``rms_norm``'s rows and their scales, or a cache's ``k`` and ``k_scale`` (whose
    blocks are contiguous): the run is ``q.numel() / scales.numel()`` elements.
    All are contiguous, and ``q`` and ``out`` start on 16 bytes.
    ``out`` is f32 or bf16 (``dtype`` chooses where it is left out; default bf16).
    """
    return (_native or _load()).dequantize(q, scales, out, dtype, stream)
