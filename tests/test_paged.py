"""The C entry points of the paged-cache operators refuse what they cannot take, on the host and before
any CUDA call."""

from __future__ import annotations

import ctypes
import struct

import pytest

from mgc_cuda.native import library

PAGED = ("k v pages page_stride token_stride head_stride dtype kv_heads head_dim page_size block_table table_stride "
         "table_pages kv_lens q_starts batch tokens status").split()
ATTEND = [*PAGED, *"q q_ts q_hs q_heads out o_ts o_hs max_q max_kv scale causal window workspace workspace_bytes".split()]
APPEND = [*PAGED, *("src_dtype k_src k_ts k_hs v_src v_ts v_hs q q_ts q_hs q_heads q_out qo_ts qo_hs cos sin table_row "
                    "positions rot interleaved").split()]
P = 1 << 20  # a 16-byte aligned address that nothing reads
BASE = dict(k=P, v=P, pages=4, page_stride=2048, token_stride=128, head_stride=64, dtype=8, kv_heads=2, head_dim=64,
            page_size=16, block_table=P, table_stride=2, table_pages=2, kv_lens=P, q_starts=P, batch=1, tokens=1, status=0)
A = dict(BASE, q=P, q_ts=256, q_hs=64, q_heads=4, out=P, o_ts=256, o_hs=64, max_q=1, max_kv=32, scale=0.125, causal=1,
         window=0, workspace=0, workspace_bytes=0)
B = dict(BASE, src_dtype=8, k_src=P, k_ts=128, k_hs=64, v_src=P, v_ts=128, v_hs=64, q=0, q_ts=0, q_hs=0, q_heads=0, q_out=0,
         qo_ts=0, qo_hs=0, cos=0, sin=0, table_row=0, positions=0, rot=0, interleaved=0)


def call(entry: str, names: list[str], values: dict) -> tuple[int, str]:
    lib = library()
    data = b"".join(struct.pack("=d" if n == "scale" else "=q", values[n]) for n in names)
    status = getattr(lib, entry)(data, None)
    return status, lib.mgc_cuda_last_error().decode()


@pytest.mark.parametrize("change,status,text", [
    (dict(k=0), 2, "NULL"), (dict(q_starts=0), 2, "NULL"), (dict(q=0), 2, "NULL"), (dict(out=0), 2, "NULL"),
    (dict(dtype=1), 3, "type"), (dict(head_dim=0), 2, "negative or zero"), (dict(page_size=0), 2, "negative or zero"),
    (dict(tokens=-1), 2, "negative"), (dict(page_stride=-1), 2, "stride"), (dict(q_heads=3), 2, "heads"),
    (dict(q_heads=0), 2, "heads"), (dict(head_dim=257), 3, "channels"), (dict(scale=0.0), 2, "scale"),
    (dict(scale=float("nan")), 2, "scale"), (dict(window=-1), 2, "window"), (dict(window=3, causal=0), 2, "window"),
    (dict(max_q=-1), 2, "bound"), (dict(table_pages=1 << 30), 3, "32 bits"), (dict(tokens=1 << 31), 3, "32 bits"),
])
def test_attention_refuses(change: dict, status: int, text: str) -> None:
    got, why = call("mgc_cuda_paged_attention", ATTEND, dict(A, **change))
    assert got == status and text in why


@pytest.mark.parametrize("change,status,text", [
    (dict(v=0), 2, "NULL"), (dict(k_src=0), 2, "missing"), (dict(q=P, q_heads=4), 2, "missing"), (dict(rot=3), 2, "rotation"),
    (dict(rot=128), 2, "rotation"), (dict(rot=32), 2, "missing"), (dict(src_dtype=7), 3, "type"), (dict(dtype=2), 3, "type"),
    (dict(q=P, q_out=P, q_heads=4, q_ts=256, q_hs=64, qo_ts=512, qo_hs=64), 2, "in place"), (dict(head_dim=512), 3, "channels"),
    (dict(kv_heads=70000), 3, "32 bits"),
])
def test_append_refuses(change: dict, status: int, text: str) -> None:
    got, why = call("mgc_cuda_kv_append", APPEND, dict(B, **change))
    assert got == status and text in why


def test_null_and_empty_calls() -> None:
    lib = library()
    assert lib.mgc_cuda_kv_append(None, None) == 2 and lib.mgc_cuda_paged_attention(None, None) == 2
    assert lib.mgc_cuda_paged_attention_workspace(None) == -1
    for change in (dict(tokens=0), dict(batch=0)):
        assert call("mgc_cuda_paged_attention", ATTEND, dict(A, **change))[0] == 0
        assert call("mgc_cuda_kv_append", APPEND, dict(B, **change))[0] == 0


def test_struct_sizes_match_the_header() -> None:
    assert len(ATTEND) * 8 == 256 and len(APPEND) * 8 == 304 and len(PAGED) * 8 == 144
    assert ctypes.sizeof(ctypes.c_void_p) == 8
