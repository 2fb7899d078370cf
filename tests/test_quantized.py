"""Quantised pages: what the Python layer and the C entry points refuse, on the host and before any CUDA call."""

from __future__ import annotations

import struct

import pytest

torch = pytest.importorskip("torch")

from mgc_cuda import paged  # noqa: E402
from mgc_cuda._errors import GraphError  # noqa: E402
from mgc_cuda.native import library  # noqa: E402
from quantized_cases import quantise, values  # noqa: E402
from test_paged import APPEND, ATTEND, PAGED  # noqa: E402

QUANT = "bits group k_scales v_scales s_page s_token s_head".split()
HEADS = [*APPEND, *QUANT, "q_norm", "k_norm", "eps"]
READ = [*PAGED, *QUANT, *"k_out ko_ts ko_hs v_out vo_ts vo_hs".split()]
ATTEND_Q = [*ATTEND, *QUANT]
P = 1 << 20
BASE = dict(k=P, v=P, pages=4, page_stride=1024, token_stride=32, head_stride=512, dtype=8, kv_heads=2, head_dim=64,
            page_size=16, block_table=P, table_stride=2, table_pages=2, kv_lens=P, q_starts=P, batch=1, tokens=1, status=0,
            bits=4, group=64, k_scales=P, v_scales=P, s_page=32, s_token=1, s_head=16)
A = dict(BASE, q=P, q_ts=256, q_hs=64, q_heads=4, out=P, o_ts=256, o_hs=64, max_q=1, max_kv=32, scale=0.125, causal=1,
         window=0, workspace=0, workspace_bytes=0)
B = dict(BASE, src_dtype=8, k_src=P, k_ts=128, k_hs=64, v_src=P, v_ts=128, v_hs=64, q=0, q_ts=0, q_hs=0, q_heads=0, q_out=0,
         qo_ts=0, qo_hs=0, cos=0, sin=0, table_row=0, positions=0, rot=0, interleaved=0, q_norm=0, k_norm=0, eps=1e-6)
R = dict(BASE, k_out=P, ko_ts=128, ko_hs=64, v_out=P, vo_ts=128, vo_hs=64)


def call(entry: str, names: list[str], given: dict) -> tuple[int, str]:
    lib = library()
    data = b"".join(struct.pack("=d" if n in ("scale", "eps") else "=q", given[n]) for n in names)
    fn = getattr(lib, entry)
    status = fn(data) if entry.endswith("workspace") else fn(data, None)
    return status, lib.mgc_cuda_last_error().decode()


FORMAT = [
    (dict(bits=3), 3, "bits"), (dict(k_scales=0), 2, "NULL"), (dict(v_scales=0), 2, "NULL"), (dict(head_dim=72), 3, "multiple of 16"),
    (dict(head_dim=272, group=272), 3, "channels"), (dict(group=32), 3, "groups"), (dict(group=0), 3, "groups"), (dict(group=48), 3, "groups"),
    (dict(s_page=-1), 2, "stride"), (dict(token_stride=24), 3, "16 bytes"), (dict(k=P + 8), 3, "16 bytes"), (dict(v=P + 1), 3, "16 bytes"),
    (dict(k_scales=P + 2), 3, "4 bytes"), (dict(k=0), 2, "NULL"), (dict(dtype=1), 3, "type"), (dict(page_size=0), 2, "negative or zero"),
    (dict(tokens=1 << 31), 3, "32 bits"),
]


@pytest.mark.parametrize("change,status,text", [*FORMAT, (dict(q=0), 2, "NULL"), (dict(q_heads=3), 2, "heads"), (dict(scale=0.0), 2, "scale"),
                                                (dict(window=2, causal=0), 2, "window"), (dict(max_kv=-1), 2, "bound")])
def test_attention_refuses(change: dict, status: int, text: str) -> None:
    got, why = call("mgc_cuda_paged_attention_quantized", ATTEND_Q, dict(A, **change))
    assert got == status and text in why
    assert call("mgc_cuda_paged_attention_quantized_workspace", ATTEND_Q, dict(A, **change))[0] == -1


@pytest.mark.parametrize("change,status,text", [*FORMAT[1:], (dict(bits=2), 3, "bits"), (dict(k_src=0), 2, "missing"), (dict(rot=128), 2, "rotation"), (dict(rot=32), 2, "missing"),
                                                (dict(src_dtype=0), 3, "queries"), (dict(eps=-1.0), 2, "eps"), (dict(eps=float("nan")), 2, "eps"),
                                                (dict(bits=0, src_dtype=7), 3, "pages"), (dict(bits=0, head_dim=257), 3, "channels")])
def test_append_refuses(change: dict, status: int, text: str) -> None:
    got, why = call("mgc_cuda_kv_append_heads", HEADS, dict(B, **change))
    assert got == status and text in why


@pytest.mark.parametrize("change,status,text", [*FORMAT, (dict(bits=0), 3, "bits"), (dict(k_out=0), 2, "NULL"), (dict(v_out=0), 2, "NULL")])
def test_read_refuses(change: dict, status: int, text: str) -> None:
    got, why = call("mgc_cuda_kv_read", READ, dict(R, **change))
    assert got == status and text in why


def test_null_and_empty_calls() -> None:
    lib = library()
    assert lib.mgc_cuda_kv_append_heads(None, None) == 2 and lib.mgc_cuda_kv_read(None, None) == 2
    assert lib.mgc_cuda_paged_attention_quantized(None, None) == 2
    assert lib.mgc_cuda_paged_attention_quantized_workspace(None) == -1
    for change in (dict(tokens=0), dict(batch=0)):
        assert call("mgc_cuda_paged_attention_quantized", ATTEND_Q, dict(A, **change))[0] == 0
        assert call("mgc_cuda_paged_attention_quantized_workspace", ATTEND_Q, dict(A, **change))[0] == 0
        assert call("mgc_cuda_kv_append_heads", HEADS, dict(B, **change))[0] == 0
        assert call("mgc_cuda_kv_read", READ, dict(R, **change))[0] == 0


@pytest.mark.parametrize("kw,text", [(dict(bits=2), "bits"), (dict(head_dim=24), "multiple of 16"), (dict(head_dim=512), "channels"),
                                     (dict(group=32), "groups"), (dict(head_dim=96, group=64), "groups")])
def test_quantized_pages_refuses(kw: dict, text: str) -> None:
    with pytest.raises(GraphError, match=text):
        paged.quantized_pages(2, 16, 2, **{"head_dim": 128, "device": "cpu", **kw})


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim,groups", [(16, 1), (48, 1), (64, 1), (80, 1), (128, 2), (192, 3), (256, 4)])
def test_quantized_pages_layout(bits: int, dim: int, groups: int) -> None:
    x = paged.quantized_pages(3, 8, 5, dim, bits=bits, device="cpu")
    assert x.codes.shape == (3, 8, 5, dim * bits // 8) and x.scales.shape == (3, 8, 5, groups, 2) and x.bits == bits
    assert all(s % 16 == 0 for s in x.codes.stride()[:3]) and x.codes.stride(3) == 1


@pytest.mark.parametrize("bits", [4, 8])
def test_a_value_is_off_by_half_a_step(bits: int) -> None:
    """|x - value| <= scale / 2 inside the range; at its ends the pair's rounding cuts off at most 2^-11 of the
    offset's size and L 2^-11 of the step."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(200, 128, generator=g) * torch.exp(torch.randn(200, 1, generator=g))
    codes, scales = quantise(x, bits, 64)
    off = (values(codes, scales, bits) - x.double()).abs().unflatten(-1, (2, 64))
    step, offset = scales[..., :1].double(), scales[..., 1:].double()
    assert bool((off <= step * (0.5 + 2**-11 * ((1 << bits) - 1)) + offset.abs() * 2**-11 + 1e-7).all())


def test_operands_are_refused_on_the_cpu() -> None:
    x = paged.quantized_pages(2, 16, 2, 64, device="cpu")
    i = torch.zeros(1, dtype=torch.int32)
    at = (i.view(1, 1), i, torch.zeros(2, dtype=torch.int32))
    q = torch.zeros(1, 4, 64)
    with pytest.raises(GraphError, match="on cpu"):
        paged.paged_attention(q, x, x, *at)
    with pytest.raises(GraphError, match="on cpu"):
        paged.kv_read(x, x, *at, rows=1)
    with pytest.raises(GraphError, match="quantised and the other"):
        paged.paged_attention(q, x, x.codes, *at)
    with pytest.raises(GraphError, match="bits"):
        paged.paged_attention(q, (x.codes, x.scales, 5), x, *at)
    with pytest.raises(GraphError, match="codes, scales, bits"):
        paged.paged_attention(q, (x.codes, x.scales), x, *at)
    with pytest.raises(GraphError, match="whole number"):
        paged.paged_attention(q, (x.codes, x.scales, None), x, *at)
    with pytest.raises(GraphError, match="not a torch type"):
        paged.kv_read(x, x, *at, rows=1, dtype=4)
    with pytest.raises(GraphError, match="negative"):
        paged.kv_read(x, x, *at, rows=-1)


def test_struct_sizes_match_the_header() -> None:
    assert len(HEADS) * 8 == 304 + 56 + 24 and len(READ) * 8 == 144 + 56 + 48 and len(ATTEND_Q) * 8 == 256 + 56
