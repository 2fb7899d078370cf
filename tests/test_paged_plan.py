"""What the host decides about a paged attention call, seen through the workspace it asks for."""

from __future__ import annotations

import struct

from mgc_cuda.native import library
from test_paged import ATTEND, A


def workspace(**change: int) -> int:
    values = dict(A, **change)
    data = b"".join(struct.pack("=d" if n == "scale" else "=q", values[n]) for n in ATTEND)
    return library().mgc_cuda_paged_attention_workspace(data)


def test_rows_past_32_bits_take_the_row_kernel() -> None:
    """The tiled kernels count a sequence's rows (new tokens times the heads of a key head) in 32 bits;
    the one-warp-a-row kernel, which needs no workspace, counts tokens."""
    heads = dict(q_heads=128, kv_heads=2, q_ts=128 * 64, o_ts=128 * 64)
    assert workspace(tokens=1 << 20, max_q=1 << 20, **heads) > 0
    assert workspace(tokens=1 << 26, max_q=1 << 26, **heads) == 0
    assert workspace(tokens=(1 << 25) - 8, max_q=1, batch=1 << 20, max_kv=1 << 14, table_pages=1 << 10, **heads) > 0
    assert workspace(tokens=1 << 25, max_q=1, batch=1 << 20, max_kv=1 << 14, table_pages=1 << 10, **heads) == 0
