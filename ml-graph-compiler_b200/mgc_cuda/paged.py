"""Serving operators over a paged cache of keys and values: ``kv_append`` and ``paged_attention``.

A compiled graph computes a whole sequence at a fixed length. Serving a decoder token by token
needs the keys and values of earlier tokens kept on the device: two tensors of pages,
``k_cache`` and ``v_cache`` [pages, page_size, kv_heads, head_dim] (float32, float16 or bfloat16;
any strides, the last 1; both of the same), and per sequence the list of its pages. A call takes a
batch of sequences with any number of new tokens each, packed along one axis:

* ``block_table`` int32 [batch, n]: the pages of each sequence in order,
* ``kv_lens`` int32 [batch]: cached positions of each sequence, its new tokens included,
* ``q_starts`` int32 [batch + 1]: sequence b's new tokens are rows q_starts[b]:q_starts[b + 1].

These three stay on the device: nothing is copied to the host and no call synchronises. All tensors
are torch CUDA tensors on one device; the kernels run on torch's current stream of that device, so
a call can be captured into a CUDA graph. There is no backward pass: where gradients are recorded, an
operand that requires one raises ``GraphError``. The C entry points are
``mgc_cuda_kv_append`` and ``mgc_cuda_paged_attention`` (include/mgc_cuda.h); an operand they cannot
take raises ``GraphError`` or ``CodegenError`` and nothing runs.

What a kernel cannot accept (a page number outside the cache, a position past the block table or
past the rotation table, a row of q_starts that the operands do not have) is skipped and recorded in ``status``, an int32 tensor of one element that
the caller may pass and hand to ``check_status`` when it next synchronises.
"""

from __future__ import annotations

import importlib.util
import threading
from ctypes import c_void_p, cast
from types import ModuleType

import torch

from mgc_cuda import build as _build
from mgc_cuda._errors import CodegenError, GraphError
from mgc_cuda.native import library

_EXT: ModuleType | None = None
_EXT_LOCK = threading.Lock()


def _binding() -> ModuleType:
    """The torch binding (csrc/paged_torch.cpp) with the C entry points handed to it, loaded once (built
    first if its sources, torch or Python changed)."""
    global _EXT
    with _EXT_LOCK:
        if _EXT is None:
            lib = library()
            path = _build.build_binding()
            spec = importlib.util.spec_from_file_location("_mgc_paged", path)
            if spec is None or spec.loader is None:
                raise CodegenError(f"cannot load {path}")
            ext = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(ext)
            entry = [cast(getattr(lib, f"mgc_cuda_{name}"), c_void_p).value
                     for name in ("kv_append", "paged_attention", "paged_attention_workspace", "last_error")]
            ext.bind(*entry, GraphError, CodegenError)
            _EXT = ext
        return _EXT


def kv_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    kv_lens: torch.Tensor,
    q_starts: torch.Tensor,
    *,
    q: torch.Tensor | None = None,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    interleaved: bool = False,
    q_out: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Write the new tokens' ``k`` and ``v`` [tokens, kv_heads, head_dim] into their cache positions.

    With ``cos`` and ``sin`` (float32 [positions, rot / 2], rot <= head_dim) the first rot channels
    of every key are rotated by the token's position on the way, pair i being channels (i, i + rot/2),
    or (2i, 2i + 1) when ``interleaved``. With ``q`` [tokens, heads, head_dim] the queries are rotated
    too: the result (``q_out`` if given, which may be ``q`` itself) is returned in the cache's type;
    rows that no sequence has are copied as they are.
    ``q``, ``k`` and ``v`` are of the cache's type or float32, strided views of a fused projection
    included; the arithmetic is fp32, rounded once."""
    return (_EXT or _binding()).kv_append(k, v, k_cache, v_cache, block_table, kv_lens, q_starts, q, cos, sin, interleaved,
                                          q_out, status)


def paged_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    kv_lens: torch.Tensor,
    q_starts: torch.Tensor,
    *,
    max_q: int | None = None,
    max_kv: int | None = None,
    scale: float | None = None,
    causal: bool = True,
    window: int = 0,
    out: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of the new tokens ``q`` [tokens, heads, head_dim] over their sequences' cached
    positions, head h reading key head h // (heads // kv_heads); returns ``out`` of q's shape.

    A token at position p sees positions j < kv_len, j <= p if ``causal``, and j > p - window if
    ``window`` is positive; a token that sees nothing, or that no sequence has, gets zeros. ``scale`` defaults to
    head_dim ** -0.5. ``max_q`` and ``max_kv``, the longest sequence's new tokens and positions,
    size the launch; without them it is sized by the packed tokens and the block table."""
    return (_EXT or _binding()).paged_attention(q, k_cache, v_cache, block_table, kv_lens, q_starts, max_q, max_kv, scale,
                                                causal, window, out, status)


def check_status(status: torch.Tensor) -> None:
    """Raise if a call with this status tensor met a page or a position it could not use (waits for
    the device)."""
    value = int(status.item())
    if value == 1:
        raise GraphError("a page number, a cache position or a rotation position was out of range")
    if value:
        raise CodegenError(f"device status {value}")
