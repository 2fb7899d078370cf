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
a call can be captured into a CUDA graph. The C entry points are ``mgc_cuda_kv_append`` and
``mgc_cuda_paged_attention`` (include/mgc_cuda.h).

What a kernel cannot accept (a page number outside the cache, a position past the block table or
past the rotation table) is skipped and recorded in ``status``, an int32 tensor of one element that
the caller may pass and hand to ``check_status`` when it next synchronises.
"""

from __future__ import annotations

import struct

import torch

from mgc_cuda._errors import CodegenError, GraphError
from mgc_cuda.native import check, library

_DTYPES = {torch.float32: 0, torch.float16: 7, torch.bfloat16: 8}  # MGC_F32, MGC_F16, MGC_BF16
_I32, _NEEDS_WORKSPACE = torch.int32, 5  # MGC_CUDA_NEEDS_WORKSPACE
_PAGED = "6q4q5q2qq"
_APPEND = struct.Struct("=" + _PAGED + "q" + "3q3q4q3q2q4q")
_ATTEND = struct.Struct("=" + _PAGED + "4q3q2qd2q2q")


# the current stream of a device as an integer, without building a stream object (3 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _fail(what: str, why: str) -> None:
    raise GraphError(f"{what}: {why}")


def _paged(what, k_cache, v_cache, block_table, kv_lens, q_starts, tokens, status):
    """The fields of mgc_cuda_paged, checked as far as the C side cannot (types, devices, shapes)."""
    dtype, device = k_cache.dtype, k_cache.device
    if dtype not in _DTYPES or v_cache.dtype is not dtype:
        _fail(what, f"pages of {dtype} and {v_cache.dtype}: both float32, float16 or bfloat16")
    shape, strides = k_cache.shape, k_cache.stride()
    if len(shape) != 4 or v_cache.shape != shape or v_cache.stride() != strides:
        _fail(what, f"caches {tuple(shape)} and {tuple(v_cache.shape)}: two [pages, page_size, kv_heads, head_dim] of "
                    "the same strides")
    if not k_cache.is_cuda:
        _fail(what, f"the cache is on {device}")
    pages, page_size, kv_heads, head_dim = shape
    ps, ts, hs, cs = strides
    if cs != 1 and head_dim > 1:
        _fail(what, "the cache's channels are not contiguous")
    if block_table.dtype is not _I32 or kv_lens.dtype is not _I32 or q_starts.dtype is not _I32:
        _fail(what, "block_table, kv_lens and q_starts are int32")
    table, table_strides, lens, starts = block_table.shape, block_table.stride(), kv_lens.shape, q_starts.shape
    batch = lens[0] if len(lens) == 1 else -1
    if (len(table) != 2 or batch < 0 or len(starts) != 1 or table[0] != batch or starts[0] != batch + 1
            or (table_strides[1] != 1 and table[1] > 1) or not kv_lens.is_contiguous() or not q_starts.is_contiguous()):
        _fail(what, f"block_table {tuple(table)}, kv_lens {tuple(lens)}, q_starts {tuple(starts)}: [batch, n], [batch], "
                    "[batch + 1], contiguous rows")
    if v_cache.device != device or block_table.device != device or kv_lens.device != device or q_starts.device != device:
        _fail(what, "the tensors are on several devices")
    at = 0
    if status is not None:
        if status.dtype is not _I32 or status.numel() != 1 or status.device != device:
            _fail(what, "status is one int32 on the cache's device")
        at = status.data_ptr()
    return (k_cache.data_ptr(), v_cache.data_ptr(), pages, ps, ts, hs, _DTYPES[dtype], kv_heads, head_dim, page_size,
            block_table.data_ptr(), table_strides[0], table[1], kv_lens.data_ptr(), q_starts.data_ptr(), batch, tokens, at)


def _rows(what, name, x, tokens, heads, dim, device):
    """(pointer, token stride, head stride) of a packed [tokens, heads, head_dim] operand."""
    shape, strides = x.shape, x.stride()
    if len(shape) != 3 or shape[0] != tokens or (heads and shape[1] != heads) or shape[2] != dim:
        _fail(what, f"{name} {tuple(shape)}: [{tokens}, {heads or 'heads'}, {dim}]")
    if x.device != device:
        _fail(what, f"{name} is on {x.device}, the cache on {device}")
    if strides[2] != 1 and dim > 1:
        _fail(what, f"{name}'s channels are not contiguous")
    return x.data_ptr(), strides[0], strides[1]


def _call(fn, what, args, device):
    """The C call on the device's current stream."""
    index = device.index
    if index == torch.cuda.current_device():
        status = fn(args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = fn(args, _raw_stream(index))
    return status


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
    too: the result (``q_out`` if given, which may be ``q`` itself) is returned in the cache's type.
    ``q``, ``k`` and ``v`` are of the cache's type or float32, strided views of a fused projection
    included; the arithmetic is fp32, rounded once."""
    what = "kv_append"
    tokens, device = k.shape[0], k_cache.device
    paged = _paged(what, k_cache, v_cache, block_table, kv_lens, q_starts, tokens, status)
    kv_heads, dim = k_cache.shape[2], k_cache.shape[3]
    src = k.dtype
    if src not in _DTYPES or v.dtype != src or (q is not None and q.dtype != src):
        _fail(what, "q, k and v are of one type")
    fields = (*paged, _DTYPES[src], *_rows(what, "k", k, tokens, kv_heads, dim, device),
              *_rows(what, "v", v, tokens, kv_heads, dim, device))
    if q is None:
        fields += (0, 0, 0, 0, 0, 0, 0)
    else:
        if q_out is None:
            q_out = q.new_empty(q.shape, dtype=k_cache.dtype)
        elif q_out.dtype != k_cache.dtype or q_out.shape != q.shape:
            _fail(what, f"q_out {tuple(q_out.shape)} of {q_out.dtype}")
        fields += (*_rows(what, "q", q, tokens, 0, dim, device), q.shape[1],
                   *_rows(what, "q_out", q_out, tokens, 0, dim, device))
    if (cos is None) != (sin is None):
        _fail(what, "cos and sin come together")
    if cos is None or sin is None:
        fields += (0, 0, 0, 0, 0, 0)
    else:
        if (cos.dim() != 2 or sin.shape != cos.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32
                or cos.stride() != sin.stride() or (cos.stride(1) != 1 and cos.shape[1] > 1)
                or cos.device != device or sin.device != device):
            _fail(what, f"cos {tuple(cos.shape)} and sin {tuple(sin.shape)}: float32 [positions, rot / 2] on the cache's "
                        "device, of the same strides")
        fields += (cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.shape[0], 2 * cos.shape[1], int(interleaved))
    status_code = _call(library().mgc_cuda_kv_append, what, _APPEND.pack(*fields), device)
    if status_code:
        check(status_code, what)
    return q_out if q is not None else None


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
    ``window`` is positive; a token that sees nothing gets zeros. ``scale`` defaults to
    head_dim ** -0.5. ``max_q`` and ``max_kv``, the longest sequence's new tokens and positions,
    size the launch; without them it is sized by the packed tokens and the block table."""
    what = "paged_attention"
    tokens, device, dtype = q.shape[0], k_cache.device, k_cache.dtype
    paged = _paged(what, k_cache, v_cache, block_table, kv_lens, q_starts, tokens, status)
    dim = k_cache.shape[3]
    if q.dtype != dtype:
        _fail(what, f"q of {q.dtype} over a cache of {dtype}")
    if out is None:
        out = q.new_empty(q.shape)
    elif out.dtype != dtype or out.shape != q.shape:
        _fail(what, f"out {tuple(out.shape)} of {out.dtype}")
    q_ptr, q_ts, q_hs = _rows(what, "q", q, tokens, 0, dim, device)
    fields = (*paged, q_ptr, q_ts, q_hs, q.shape[1], *_rows(what, "out", out, tokens, 0, dim, device),
              tokens if max_q is None else max_q,
              block_table.shape[1] * k_cache.shape[1] if max_kv is None else max_kv,
              dim ** -0.5 if scale is None else scale, int(causal), window)
    lib = library()
    status_code = _call(lib.mgc_cuda_paged_attention, what, _ATTEND.pack(*fields, 0, 0), device)
    if status_code == _NEEDS_WORKSPACE:
        # few rows over many keys: partial results of the keys' parts, from torch's stream-ordered
        # allocator (the block returns to this stream's pool after the call)
        need = lib.mgc_cuda_paged_attention_workspace(_ATTEND.pack(*fields, 0, 0))
        space = q.new_empty(need, dtype=torch.uint8)
        status_code = _call(lib.mgc_cuda_paged_attention, what, _ATTEND.pack(*fields, space.data_ptr(), need), device)
    if status_code:
        check(status_code, what)
    return out


def check_status(status: torch.Tensor) -> None:
    """Raise if a call with this status tensor met a page or a position it could not use (waits for
    the device)."""
    value = int(status.item())
    if value == 1:
        raise GraphError("a page number, a cache position or a rotation position was out of range")
    if value:
        raise CodegenError(f"device status {value}")
