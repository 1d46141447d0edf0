"""The attention half of a decoder layer next to the split FFN: rotary positions and an
8-bit paged cache (append, attend, read, fork, compact) over the C ABI.

A cache holds K and V as int8 codes in pages of ``page_tokens`` tokens, with one f32 scale
for each page and head (value = code * scale; scales are finite and not negative, NaN marks a block that
took a non-finite value). A step works on a batch of sequences given by
three int32 device tensors:

* ``tables``  [seqs, width]  page ids of each sequence in order;
* ``lengths`` [seqs]         tokens it holds, the step's new ones included (0: an idle slot);
* ``starts``  [seqs + 1]     rows of its new tokens in q, k and v (None: one row each).

The j-th of a sequence's n new tokens stands at position ``lengths - n + j``. A step is then:
``fork`` (reserve room; also shares, copies and frees pages between steps), and per layer
``append`` (rotates q and k, quantises k and v into the pages) and ``attend``.

Arguments are torch tensors on the cache's device. Shape and type errors raise
``ValueError``; data on the device that a kernel could not use is recorded and raised by
``check``. Calls run on the current stream (or ``stream``) without synchronising and can be
captured in a CUDA graph; calls on one cache must not overlap on the GPU. With a ``stream`` that is not
the current one the caller orders it behind what wrote the arguments (they may be dropped as soon as the
call returns); new outputs belong to that stream. Only ``rotary`` takes part in
autograd: the cache's calls serve, and their results require no gradient.
"""
from __future__ import annotations

import ctypes
import math

from . import _native as N
from .engine import _stream


_module = None


def _bind():
    """The compiled binding of the cache's calls (built with the library)."""
    global _module
    if _module is None:
        import importlib.util

        import torch  # noqa: F401  (its libraries are loaded first)
        N.lib()
        if not N.BIND_PATH.exists():
            raise N.NativeLibraryMissing(f"{N.BIND_PATH} is not built; run `python -m ffn_residual_mesh_b200.build`")
        spec = importlib.util.spec_from_file_location("ffnrm_kv_bind", N.BIND_PATH)
        _module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_module)
    return _module


class RotaryTable:
    """Cosines and sines of every position, f32 [max_positions, rotary_dim] (cosines, then
    sines). Pair i of a head turns by ``position * base ** (-2 i / rotary_dim)``.

    ``scaling`` for contexts longer than the weights were trained on:

    * ``"linear"`` — positions divided by ``factor``;
    * ``"ntk"`` — the base raised to ``base * factor ** (R / (R - 2))``, which leaves the
      fastest pair as it is and slows the slowest one by ``factor``;
    * ``"yarn"`` — per pair: pairs that turn more than ``beta_fast`` times within
      ``original_positions`` stay, those below ``beta_slow`` turns are divided by
      ``factor``, a ramp between; cosines and sines are multiplied by
      ``0.1 ln(factor) + 1`` (YaRN, Peng et al. 2023).
    """

    def __init__(self, rotary_dim: int, max_positions: int, base: float = 10000.0, interleaved: bool = False,
                 scaling: str | None = None, factor: float = 1.0, original_positions: int | None = None,
                 beta_fast: float = 32.0, beta_slow: float = 1.0, device=0):
        import torch
        if rotary_dim <= 0 or rotary_dim % 2 or max_positions <= 0:
            raise ValueError("rotary_dim must be even and positive, max_positions positive")
        if scaling not in (None, "linear", "ntk", "yarn"):
            raise ValueError(f"unknown scaling {scaling!r}")
        if scaling is not None and factor < 1.0:
            raise ValueError("factor must be at least 1")
        if base <= 1.0:
            raise ValueError("base must be above 1")
        pair = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
        gain = 1.0
        if scaling == "ntk" and rotary_dim > 2:
            base = base * factor ** (rotary_dim / (rotary_dim - 2))
        freq = base ** (-pair / rotary_dim)
        if scaling == "linear":
            freq = freq / factor
        elif scaling == "yarn":
            if not original_positions or original_positions <= 0 or beta_fast <= beta_slow:
                raise ValueError("yarn needs original_positions and beta_fast > beta_slow")
            # the (fractional) pair that makes `turns` turns within the original context
            at = [rotary_dim * math.log(original_positions / (turns * 2 * math.pi)) / (2 * math.log(base))
                  for turns in (beta_fast, beta_slow)]
            low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary_dim - 1)
            ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
            freq = freq * (1 - ramp) + freq / factor * ramp
            gain = 0.1 * math.log(factor) + 1.0
        angle = torch.arange(max_positions, dtype=torch.float64)[:, None] * freq
        self._set((torch.cat([angle.cos(), angle.sin()], 1) * gain).float().to(
            torch.device("cuda", device) if isinstance(device, int) else device), interleaved)

    @classmethod
    def from_tensor(cls, cos_sin, interleaved: bool = False) -> "RotaryTable":
        """A table of the caller's own angles: f32 [max_positions, rotary_dim]."""
        self = cls.__new__(cls)
        self._set(cos_sin, interleaved)
        return self

    def _set(self, cos_sin, interleaved):
        import torch
        if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous() or cos_sin.shape[1] % 2 \
                or 0 in cos_sin.shape:
            raise ValueError("cos_sin must be a contiguous float32 tensor [max_positions, rotary_dim]")
        self.cos_sin, self.interleaved = cos_sin, bool(interleaved)
        self.max_positions, self.rotary_dim = cos_sin.shape
        self.flags = N.ROTARY_INTERLEAVED if interleaved else 0


_recorded = None


def _rotary_function():
    """The rotation for autograd: linear in x, its gradient is the other direction at the same positions."""
    global _recorded
    if _recorded is None:
        import torch

        class Rotary(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, positions, table, inverse, stream):
                ctx.save_for_backward(positions, table.cos_sin)
                ctx.interleaved, ctx.inverse = table.interleaved, inverse
                return rotary(x.detach(), positions, table, inverse=inverse, stream=stream)

            @staticmethod
            def backward(ctx, grad):
                positions, cos_sin = ctx.saved_tensors
                if grad.stride(2) != 1:  # as a sum's gradient
                    grad = grad.contiguous()
                table = RotaryTable.from_tensor(cos_sin, ctx.interleaved)
                return rotary(grad, positions, table, inverse=not ctx.inverse), None, None, None, None

        _recorded = Rotary
    return _recorded


def rotary(x, positions, table: RotaryTable, out=None, inverse: bool = False, stream=None):
    """x [T, heads, dim] with its first ``rotary_dim`` channels rotated at ``positions`` (int32
    [T]); ``inverse`` applies the transposed rotation, the gradient of the forward one, which autograd
    uses where x requires it (the table gets none). ``out`` is x or lies apart from it, and is not for
    tensors that require a gradient. A position outside the table gives NaN in the rotated channels."""
    y = (_module or _bind()).rotary(x, positions, table.cos_sin, out, table.flags | (N.ROTARY_INVERSE if inverse else 0), stream)
    return _rotary_function().apply(x, positions, table, inverse, stream) if y is None else y


class PagedKvCache:
    """K and V of ``n_layers`` layers in ``n_pages`` pages of ``page_tokens`` tokens each.

    ``buffers``: (k_codes, v_codes, k_scale, v_scale) to use in place of new ones: int8
    [layers, pages, kv_heads, page_tokens, head_dim] and f32 [layers, pages, kv_heads].
    """

    def __init__(self, n_layers: int, n_pages: int, kv_heads: int, head_dim: int, page_tokens: int = 64,
                 max_seqs: int = 256, device: int = 0, buffers=None):
        import torch
        self.handle = None
        self.lib = N.lib()
        self._calls = _bind()
        self.n_layers, self.n_pages, self.kv_heads, self.head_dim = n_layers, n_pages, kv_heads, head_dim
        self.page_tokens, self.max_seqs = page_tokens, max_seqs
        self.device = torch.device("cuda", device)
        if min(n_layers, n_pages, kv_heads, max_seqs) <= 0 or head_dim not in (64, 128, 256) \
                or page_tokens not in (16, 32, 64, 128):
            raise ValueError(f"n_layers={n_layers}, n_pages={n_pages}, kv_heads={kv_heads}, max_seqs={max_seqs} must be "
                             f"positive, head_dim={head_dim} 64, 128 or 256, page_tokens={page_tokens} 16, 32, 64 or 128")
        codes, scale = (n_layers, n_pages, kv_heads, page_tokens, head_dim), (n_layers, n_pages, kv_heads)
        if buffers is None:
            buffers = [torch.zeros(codes, dtype=torch.int8, device=self.device) for _ in range(2)] + \
                      [torch.zeros(scale, dtype=torch.float32, device=self.device) for _ in range(2)]
            torch.cuda.current_stream(self.device).synchronize()
        for b, shape, dtype in zip(buffers, (codes, codes, scale, scale), (torch.int8, torch.int8, torch.float32, torch.float32)):
            if tuple(b.shape) != shape or b.dtype != dtype or not b.is_contiguous():
                raise ValueError(f"a cache buffer must be a contiguous {dtype} tensor of shape {shape}, "
                                 f"got {b.dtype} {tuple(b.shape)}")
            if b.device != self.device:
                raise ValueError(f"a cache buffer must be on {self.device}, got {b.device}")
        self.k_codes, self.v_codes, self.k_scale, self.v_scale = buffers
        cfg = N.KvConfig(n_layers, n_pages, kv_heads, head_dim, page_tokens, max_seqs)
        handle = ctypes.c_void_p()
        N.check(self.lib.ffnrm_kv_create(ctypes.byref(handle), device, ctypes.byref(cfg),
                                         *(b.data_ptr() for b in buffers)))
        self.handle = handle
        self._geo = (handle.value, kv_heads, head_dim, device)

    # -- lifetime ---------------------------------------------------------
    def close(self) -> None:
        if getattr(self, "handle", None):
            self._geo = None
            N.check(self.lib.ffnrm_kv_destroy(self.handle))
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def check(self, stream=None) -> None:
        """Synchronise and raise what the kernels recorded: MemoryError (too few free pages),
        TimeoutError (a bounded wait ran out), RuntimeError (data that could not be used)."""
        import torch
        N.check(self.lib.ffnrm_kv_check(self.handle, _stream(torch.cuda.current_stream(self.device) if stream is None else stream)))

    # -- a step's work --------------------------------------------------------
    def append(self, layer: int, k, v, tables, lengths, starts=None, rope: RotaryTable | None = None, q=None, q_out=None,
               stream=None):
        """Quantise the step's new k and v [T, kv_heads, head_dim] into their pages. With
        ``rope`` the keys are rotated at their positions first, and with ``q`` [T, heads,
        head_dim] the queries too; returns the rotated queries (``q_out``, which is q or lies
        apart from q, k and v)."""
        return self._calls.append(self._geo, layer, k, v, tables, lengths, starts, rope.cos_sin if rope else None,
                                  rope.flags if rope else 0, q, q_out, stream)

    def attend(self, layer: int, q, tables, lengths, starts=None, out=None, lse=None, scale: float | None = None,
               causal: bool = True, window: int = 0, stream=None):
        """Attention of the step's queries q [T, heads, head_dim] (float16 or bfloat16) over the
        cache, the step's own tokens included. q's and ``out``'s rows start on 16 bytes (views of packed
        rows do where head_dim divides their offsets); ``out`` is q or lies apart from it. ``scale`` defaults to ``head_dim ** -0.5``;
        ``window`` > 0 lets a query see its last ``window`` positions only. ``lse`` (float32
        [T, heads]) receives the natural log of the sum of exponentials."""
        return self._calls.attend(self._geo, layer, q, tables, lengths, starts, out, lse,
                                  self.head_dim ** -0.5 if scale is None else scale, causal, window, stream)

    def read(self, layer: int, tables, lengths, starts, rows: int, dtype=None, stream=None):
        """The last tokens of each sequence back from the cache: k and v [rows, kv_heads,
        head_dim] (code * scale), float32 unless ``dtype``. ``starts`` says how many of each; rows outside
        them are zeros."""
        import torch
        types = {None: N.F32, torch.float32: N.F32, torch.float16: N.F16, torch.bfloat16: N.BF16}
        if dtype not in types:
            raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        return self._calls.read(self._geo, layer, tables, lengths, starts, rows, types[dtype], stream)

    # -- pages between steps --------------------------------------------------
    def fork(self, tables, lengths, parents, extra, out_tables=None, out_lengths=None, info=None, stream=None):
        """The next step's batch: child i continues sequence ``parents[i]`` (-1: an empty one)
        with room for ``extra[i]`` new tokens. A sequence named by several children is
        shared (its open last page is copied), one named by none is freed. Returns (tables,
        lengths, info); info int32 [4] holds the pages held, free, copied and short. ``out_lengths``
        may be ``lengths`` (a fork that is short of pages leaves zeros there), ``out_tables`` lies apart
        from ``tables``."""
        return self._calls.fork(self._geo, tables, lengths, parents, extra, out_tables, out_lengths, info, stream)

    def compact(self, tables, lengths, out_tables=None, info=None, stream=None):
        """Move the held pages to the lowest ids. Returns (tables, info); ``out_tables`` may be
        ``tables``. No held page is overwritten, so the old tables stay readable until the
        next fork hands out the freed pages."""
        return self._calls.compact(self._geo, tables, lengths, out_tables, info, stream)

    def copy_pages(self, src, dst, stream=None) -> None:
        """Copy page src[i] to dst[i] in every layer (int32 [n]; a destination is named once and is
        no source)."""
        self._calls.copy_pages(self._geo, src, dst, stream)
