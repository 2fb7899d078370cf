"""kv_append with head norms, kv_append and kv_read over quantised pages, and the attention over them, against
their definitions: every type, head layout, page size and mask at the sizes where a kernel can go wrong."""

from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from mgc_cuda import paged  # noqa: E402
from mgc_cuda._errors import GraphError  # noqa: E402
from paged_cases import DTYPES, ROUND, PagedBatch, angles  # noqa: E402
from quantized_cases import QuantizedBatch, attention, compare, normed, quantise, rotated, values, widened, workspace  # noqa: E402

pytestmark = pytest.mark.gpu

ALL = ["f32", "f16", "bf16"]


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---- append --------------------------------------------------------------------------------------
def spots(x, qs, ks):
    """(row, sequence, position) of every packed token."""
    return [(sum(qs[:b]) + i, b, k - q + i) for b, (q, k) in enumerate(zip(qs, ks)) for i in range(q)]


def append(x, qs, ks, *, src, norm, rot, interleaved, seed, odd=False, positions=4096, eps=1e-6, in_place=False):
    """Runs kv_append over batch x and returns what the definition's steps give: (q, k, v, got q)."""
    kv_heads = (x.k.codes if x.__class__ is QuantizedBatch else x.k).shape[2]
    heads, dim, dt = x.q.shape[1], x.q.shape[2], DTYPES[src]
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = sum(qs)
    pad = 3 if odd else 0
    qkv = torch.randn(tokens, heads + 2 * kv_heads, dim + pad, generator=g, device="cuda").to(dt)[..., pad and 1 :][..., :dim]
    q, k, v = qkv[:, :heads], qkv[:, heads : heads + kv_heads], qkv[:, heads + kv_heads :]
    wq, wk = (1 + 0.3 * torch.randn(dim, generator=g, device="cuda") if norm else None for _ in range(2))
    cos, sin = angles(positions, rot) if rot else (None, None)
    pos = torch.tensor([p for _, _, p in spots(x, qs, ks)], device="cuda")
    want_q = rotated(normed(q.float(), wq, eps), cos, sin, pos, interleaved)
    want_k = rotated(normed(k.float(), wk, eps), cos, sin, pos, interleaved)
    want_v = v.float().clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = paged.kv_append(k, v, *x.operands, q=q, cos=cos, sin=sin, interleaved=interleaved, q_norm=wq, k_norm=wk, eps=eps,
                          q_out=q if in_place else None, status=status)
    paged.check_status(status)
    return want_q, want_k, want_v, got


@pytest.mark.parametrize("src", ALL)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim,group,rot,interleaved", [
    (64, 64, 0, False), (64, 64, 64, False), (64, 64, 64, True), (128, 64, 128, False), (128, 128, 64, True), (128, 64, 32, False),
    (80, 80, 32, False), (80, 80, 20, False), (96, 96, 96, False), (16, 16, 16, False), (48, 48, 6, True), (256, 64, 128, False),
    (256, 256, 256, True), (192, 64, 192, False), (112, 112, 2, False), (32, 32, 0, False),
])
def test_append_writes_the_definition_s_codes(src, bits, dim, group, rot, interleaved) -> None:
    for norm, odd, layout in ((True, False, "heads"), (False, False, "tokens"), (True, True, "joint")):
        qs, ks = [1, 37, 0, 5], [9, 37, 4, 70]
        x = QuantizedBatch(qs, ks, heads=6, kv_heads=2, dim=dim, page=16, dtype=src, bits=bits, group=group, layout=layout)
        before = [[t.clone() for t in (c.codes, c.scales)] for c in (x.k, x.v)]
        q, k, v, got = append(x, qs, ks, src=src, norm=norm, rot=rot, interleaved=interleaved, seed=dim + rot, odd=odd, in_place=layout == "tokens")
        assert got.dtype == DTYPES[src]
        assert bool(((got.double() - q.double()).abs() <= ROUND[src] * q.double().abs() + 2.0**-25).all())
        for c, want, old in ((x.k, k, before[0]), (x.v, v, before[1])):
            codes, scales = quantise(want, bits, group)
            for row, b, pos in spots(x, qs, ks):
                at = int(x.table[b, pos // 16]), pos % 16
                old[0][at], old[1][at] = codes[row], scales[row]
            # the new tokens' rows and nothing else
            assert torch.equal(c.codes, old[0])
            assert torch.equal(c.scales.view(torch.int16), old[1].view(torch.int16)) or torch.equal(c.scales.nan_to_num(7.0), old[1].nan_to_num(7.0))


@pytest.mark.parametrize("dtype,src", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("dim,rot,interleaved", [(64, 64, False), (128, 128, False), (128, 64, True), (80, 32, True), (7, 4, False), (1, 0, False),
                                                 (256, 256, False), (100, 50, False), (24, 24, True)])
def test_norms_of_heads_into_plain_pages(dtype, src, dim, rot, interleaved) -> None:
    for odd, layout in ((False, "tokens"), (True, "heads"), (False, "odd")):
        qs, ks = [1, 40, 0, 5], [9, 40, 4, 70]
        x = PagedBatch(qs, ks, heads=6, kv_heads=2, dim=dim, page=16, dtype=dtype, layout=layout)
        old = [x.k.clone(), x.v.clone()]
        q, k, v, got = append(x, qs, ks, src=src, norm=True, rot=rot, interleaved=interleaved, seed=dim, odd=odd, in_place=dtype == src and not odd)
        r = ROUND[dtype]
        assert bool(((got.double() - q.double()).abs() <= r * q.double().abs() + 2.0**-25).all())
        for c, want, before in ((x.k, k, old[0]), (x.v, v, old[1])):
            for row, b, pos in spots(x, qs, ks):
                at = int(x.table[b, pos // 16]), pos % 16
                assert bool(((c[at].double() - want[row].double()).abs() <= r * want[row].double().abs() + 2.0**-25).all())
                before[at] = c[at]
            assert torch.equal(c.nan_to_num(7.0), before.nan_to_num(7.0))


def test_norm_against_64_bits_at_the_ends_of_the_range() -> None:
    """Heads of zeros, of tiny and of huge values: x / sqrt(mean x^2 + eps) w, off by three roundings."""
    for eps in (1e-6, 0.0):
        x = PagedBatch([6], [6], heads=2, kv_heads=1, dim=64, page=16, dtype="f32")
        g = torch.Generator(device="cuda").manual_seed(1)
        q = torch.randn(6, 2, 64, generator=g, device="cuda") * torch.tensor([1e-18, 1e-12, 1.0, 1e4, 1e17, 3e18], device="cuda")[:, None, None]
        if eps:
            q[0] = 0.0
        w = 1 + torch.randn(64, generator=g, device="cuda")
        got = paged.kv_append(q[:, :1], q[:, :1], *x.operands, q=q, q_norm=w, k_norm=w, eps=eps)
        want = q.double() / (q.double().square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
        assert bool(((got.double() - want).abs() <= 3.5 * 2.0**-24 * want.abs()).all())
        assert torch.equal(x.k[x.slots[0]], got[:, :1])


@pytest.mark.parametrize("bits", [4, 8])
def test_groups_that_have_no_range_or_no_bounds(bits) -> None:
    """Constant groups, values past half's range, NaN and infinities: codes as the definition says, and only
    the group that a value is in."""
    x = QuantizedBatch([5], [5], heads=1, kv_heads=1, dim=128, page=16, dtype="f32", bits=bits, group=64)
    k = torch.randn(5, 1, 128, device="cuda")
    k[0, 0, :64] = 0.75
    k[1, 0, 3], k[1, 0, 4] = 1e6, -2e5
    k[2, 0, 70] = math.nan
    k[3, 0, 5] = math.inf
    k[4, 0, :64] = 0.0
    v = torch.where(torch.isfinite(k), -k, -k)
    paged.kv_append(k, v, *x.operands)
    for c, src in ((x.k, k), (x.v, v)):
        codes, scales = quantise(src, bits, 64)
        assert torch.equal(c.codes[x.slots[0]], codes)
        assert torch.equal(c.scales[x.slots[0]].nan_to_num(-3.0), scales.nan_to_num(-3.0))
    back, _ = paged.kv_read(*x.operands, rows=5, dtype=torch.float32)
    assert torch.isnan(back).sum() == 128 and bool((back[0, 0, :64] == 0.75).all()) and bool((back[4, 0, :64] == 0).all())


def test_append_leaves_what_it_cannot_place() -> None:
    """Missing pages, positions past the rotation table, more new tokens than positions, rows that no sequence
    has: nothing is written there, the rest is, and the status tells."""
    for norm in (True, False):
        x = QuantizedBatch([4, 3, 6], [20, 40, 4], heads=2, kv_heads=1, dim=64, page=16, dtype="bf16", bits=4)
        x.block_table[0, 1] = 99
        before = [c.codes.clone() for c in (x.k, x.v)]
        q = torch.randn(16, 2, 64, device="cuda").bfloat16()
        k, v = (torch.randn(16, 1, 64, device="cuda").bfloat16() for _ in range(2))
        cos, sin = angles(39, 64)
        w = torch.full((64,), 2.0, device="cuda") if norm else None
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = paged.kv_append(k, v, *x.operands, q=q, cos=cos, sin=sin, q_norm=w, k_norm=w, status=status)
        assert int(status) == 1
        # sequence 0's tokens 16..19 are on the missing page (their queries are turned all the same), position 39
        # of sequence 1 has no angle, sequence 2 has two tokens before position 0, rows 13..15 belong to none
        copied = [6, 7, 8, 13, 14, 15]
        assert all(torch.equal(got[i], q[i]) for i in copied)
        assert not any(torch.equal(got[i], q[i]) for i in range(13) if i not in copied and i != 9)  # (9: position 0, turned by nothing)
        written = {(int(x.table[1, 2]), 5), (int(x.table[1, 2]), 6), *((int(x.table[2, 0]), i) for i in range(4))}
        for c, old in zip((x.k, x.v), before):
            changed = (c.codes != old).flatten(2).any(-1)
            assert {tuple(i) for i in changed.nonzero().tolist()} == written


# ---- read ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,group,layout", [(64, 64, "heads"), (128, 64, "tokens"), (128, 128, "joint"), (80, 80, "heads"), (16, 16, "tokens"),
                                              (256, 64, "heads"), (192, 192, "joint")])
def test_read(bits, dtype, dim, group, layout) -> None:
    qs, ks = [70, 0, 3, 1], [70, 5, 33, 1]
    x = QuantizedBatch(qs, ks, heads=2, kv_heads=2, dim=dim, page=16, dtype="f16", bits=bits, group=group, layout=layout, spread=2.0)
    rows = 80  # six that no sequence has
    odd = torch.empty(rows, 2, dim + 1, dtype=dtype, device="cuda")[..., 1:]
    for out in (None, odd):
        k, v = paged.kv_read(*x.operands, rows=rows, dtype=dtype, k_out=out)
        assert k.shape == v.shape == (rows, 2, dim) and (out is None or k.data_ptr() == out.data_ptr())
        for c, got in ((x.k, k), (x.v, v)):
            for row, b, pos in spots(x, qs, ks):
                at = int(x.table[b, pos // 16]), pos % 16
                # fp32 as the definition rounds it: the product is exact
                assert torch.equal(got[row], values(c.codes[at], c.scales[at], bits, torch.float32).to(dtype))
            assert bool((got[74:] == 0).all())


def test_read_is_the_inverse_of_append() -> None:
    """Appending what was read back gives the same codes where the extremes are on the grid, as they are."""
    qs = ks = [50, 7]
    x = QuantizedBatch(qs, ks, heads=2, kv_heads=2, dim=64, page=24, dtype="f32", bits=8)
    k, v = paged.kv_read(*x.operands, rows=57, dtype=torch.float32)
    y = QuantizedBatch(qs, ks, heads=2, kv_heads=2, dim=64, page=24, dtype="f32", bits=8, seed=5)
    paged.kv_append(k, v, *y.operands)
    again, _ = paged.kv_read(*y.operands, rows=57, dtype=torch.float32)
    step = y.k.scales[..., 0].float().nan_to_num(0.0).max()
    assert float((again - k).abs().max()) <= float(step) * (0.5 + 255 * 2**-11) + 2**-10


def test_read_without_pages_or_positions() -> None:
    x = QuantizedBatch([5, 4], [5, 2], heads=1, kv_heads=1, dim=64, page=4, dtype="f16", bits=4)
    x.block_table[0, 1] = -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = paged.kv_read(*x.operands, rows=9, status=status)
    assert int(status) == 1
    zero = [4, 5, 6]  # position 4 of sequence 0; sequence 1 has two tokens before position 0
    for got in (k, v):
        assert [i for i in range(9) if bool((got[i] == 0).all())] == zero
    status.zero_()
    k, _ = paged.kv_read(x.k, x.v, x.block_table, x.kv_lens, x.q_starts, rows=7, status=status)  # rows that the call does not have
    assert int(status) == 1 and k.shape[0] == 7
    k, v = paged.kv_read(x.k, x.v, x.block_table[:0], x.kv_lens[:0], x.q_starts[:1], rows=3)
    assert bool((k == 0).all()) and bool((v == 0).all())
    assert paged.kv_read(*x.operands[:4], i32(0, 0, 0), rows=0)[0].shape == (0, 1, 64)


# ---- attention -----------------------------------------------------------------------------------
def attend(x: QuantizedBatch, **kw):
    out = torch.full(x.q.shape, math.nan, dtype=x.q.dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kw.setdefault("max_q", max(x.qs))
    kw.setdefault("max_kv", max(x.ks))
    assert paged.paged_attention(x.q, *x.operands, out=out, status=status, **kw) is out
    paged.check_status(status)
    return out


def expands(x: QuantizedBatch) -> bool:
    """Whether a call without max_kv goes over plain pages."""
    capacity = x.block_table.shape[1] * x.page
    return workspace(x, max(x.qs), capacity) >= 4 * len(x.qs) * capacity * x.q.shape[2]


def many_rows(x: QuantizedBatch) -> bool:
    """Whether there is a way over plain pages: 16 bits, rows enough (288: 18 units of codes against 48 of pages; sequences
    of at most 64 stay on the codes), rows of q in 16 bytes; bf16 with the tcgen05 kernel alone; a head's pages in 1 GiB."""
    return (x.name != "f32" and max(x.qs) * x.share >= 288 and x.q.data_ptr() % 16 == 0 and x.q.stride(0) % 8 == 0 and
            not (x.name == "bf16" and (x.q.shape[2] > 128 or x.page % 8)) and x.k.codes.shape[2] > 1)


def agree(x: QuantizedBatch, causal: bool = True, window: int = 0, **kw) -> None:
    want, bound = attention(x, x.q.shape[2] ** -0.5, causal, window)
    compare(attend(x, causal=causal, window=window, **kw), want, bound)
    if many_rows(x) and not kw and not window:
        y = widened(x)
        assert expands(y)
        compare(attend(y, causal=causal, max_q=max(x.qs), max_kv=None), want, bound)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 1000, 4097])
def test_one_token(dtype, bits, n) -> None:
    agree(QuantizedBatch([1], [n], heads=4, kv_heads=4, dim=64, page=16, dtype=dtype, bits=bits, seed=n))
    agree(QuantizedBatch([1], [n], heads=8, kv_heads=2, dim=128, page=16, dtype=dtype, bits=bits, seed=n, spread=2.0))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (8, 4), (12, 4), (8, 1), (32, 8), (16, 1), (20, 1), (40, 2), (66, 2)])
def test_head_groups(dtype, bits, heads, kv_heads) -> None:
    for qs, ks in (([1, 1, 1], [300, 5, 77]), ([7, 40, 1], [300, 40, 77])):
        agree(QuantizedBatch(qs, ks, heads=heads, kv_heads=kv_heads, dim=64, page=16, dtype=dtype, bits=bits, seed=heads))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim,group", [(16, 16), (32, 32), (48, 48), (64, 64), (80, 80), (96, 96), (112, 112), (128, 64), (128, 128), (144, 144),
                                       (192, 64), (192, 192), (256, 64), (256, 128), (256, 256)])
def test_head_widths_and_groups(dtype, bits, dim, group) -> None:
    for qs, ks in (([1, 1], [150, 33]), ([5, 3], [150, 33]), ([150, 3], [150, 33])):
        agree(QuantizedBatch(qs, ks, heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype, bits=bits, group=group, seed=dim, spread=1.7))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 48, 64, 100, 128, 256, 512])
def test_page_sizes(dtype, bits, page) -> None:
    for qs, ks in (([1, 1], [601, 130]), ([150, 70], [601, 130])):
        agree(QuantizedBatch(qs, ks, heads=4, kv_heads=2, dim=64, page=page, dtype=dtype, bits=bits, seed=page))
        agree(QuantizedBatch(qs, ks, heads=4, kv_heads=2, dim=128, page=page, dtype=dtype, bits=bits, seed=page))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("layout", ["heads", "tokens", "joint"])
def test_cache_layouts_and_query_strides(dtype, bits, layout) -> None:
    for packed in (True, False):
        for qs in ([1, 1], [200, 30]):  # 600 rows: both ways
            for dim in (64, 80):
                agree(QuantizedBatch(qs, [300, 31], heads=6, kv_heads=2, dim=dim, page=16, dtype=dtype, bits=bits, layout=layout, packed=packed))
    x = QuantizedBatch([1, 1], [300, 31], heads=6, kv_heads=2, dim=64, page=16, dtype=dtype, bits=bits, layout=layout)
    x.q = torch.nn.functional.pad(x.q, (1, 2))[..., 1:65]  # rows at odd elements
    agree(x)
    x = QuantizedBatch([90, 1], [300, 31], heads=6, kv_heads=2, dim=64, page=16, dtype=dtype, bits=bits, layout=layout)
    x.q = torch.nn.functional.pad(x.q, (1, 2))[..., 1:65]
    agree(x)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("qs,ks", [
    ([0, 0, 5], [0, 9, 5]),            # sequences without new tokens, without positions
    ([3, 1, 2], [1, 0, 2]),            # more new tokens than positions: rows that see nothing
    ([300, 130], [120, 0]),            # the same over whole tiles
    ([1] * 70, list(range(1, 71))),    # more sequences than a warp has lanes
    ([257, 1, 128, 64, 0, 33], [257, 900, 128, 1000, 40, 64]),
    ([513], [2000]),
])
@pytest.mark.parametrize("causal", [True, False])
def test_ragged_batches(dtype, bits, qs, ks, causal) -> None:
    for kv_heads, dim in ((4, 64), (1, 128)):
        agree(QuantizedBatch(qs, ks, heads=4, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype, bits=bits), causal=causal)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_many_rows_over_plain_pages(dtype, bits) -> None:
    """What a batch may hold, in calls that expand values first: windows, missing pages, NaN, lengths past the table, rows
    that no sequence has, sequences longer than max_kv says, single tokens beside chunks, key heads in passes."""

    def batch(qs, ks, **kw):
        return QuantizedBatch(qs, ks, **{**dict(heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, bits=bits), **kw})

    kw = dict(max_kv=None)
    # windows that leave pages out, whose entries and rows hold anything
    x = batch([300, 200, 1], [900, 333, 100])
    # (the rule counts on the window's keys: a wide one)
    want, bound = attention(x, 64**-0.5, True, 250)
    for b, (nq, nk) in enumerate(zip(x.qs, x.ks)):
        first = max(0, nk - nq - 250 + 1)
        page, row = (t[:first] for t in x.slots[b])
        for c in (x.k, x.v):
            c.scales[page, row] = math.nan
        x.block_table[b, : first // 16] = -1
    compare(attend(widened(x), window=250, **kw), want, bound)
    compare(attend(x, window=250), want, bound)
    # missing pages
    x = batch([300, 3, 290], [333, 90, 400])
    present = [torch.ones(n, dtype=torch.bool, device="cuda") for n in x.ks]
    for b, page, number in ((0, 3, -1), (0, 20, 10**6), (1, 0, -7), (2, 24, 10**9)):
        x.block_table[b, page] = number
        present[b][16 * page : 16 * page + 16] = False
    y = widened(x)
    assert expands(y)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = paged.paged_attention(y.q, *y.operands, max_q=300, status=status)
    assert int(status) == 1
    compare(got, *attention(x, 64**-0.5, present=present))
    # NaN at the last but one position, and a group of one head
    for what in ("k", "v"):
        x = batch([300, 290], [300, 360], dim=128)
        page, row = x.slots[0]
        getattr(x, what).scales[page[298], row[298], :] = math.nan
        page, row = x.slots[1]
        getattr(x, what).scales[page[358], row[358], 1, 1] = math.nan
        agree(x)
    # lengths past the block table
    x = batch([300, 2], [304, 40])
    x.block_table = x.block_table[:, :19].contiguous()
    x.kv_lens = i32(400, 40)
    compare(paged.paged_attention(x.q, *x.operands, max_q=300, max_kv=400), *attention(x, 64**-0.5, lens=[400, 40]))
    # rows that no sequence has
    x = batch([300, 140], [330, 140])
    want, bound = attention(x, 64**-0.5)
    y = widened(x)
    y.q = torch.cat((torch.full_like(x.q[:2], 9.0), x.q, torch.full_like(x.q[:3], math.nan)))
    y.q_starts = x.q_starts + 2
    out = torch.full_like(y.q, math.nan)
    paged.paged_attention(y.q, *y.operands, max_q=300, out=out)
    assert bool((out[:2] == 0).all()) and bool((out[-3:] == 0).all())
    compare(out[2:-3], want, bound)
    # a sequence longer than max_kv says, one that fits, single tokens
    x = batch([700, 500, 1, 3], [6000, 1500, 900, 20], kv_heads=4, heads=8, dim=128)
    compare(attend(x, max_kv=4000), *attention(x, 128**-0.5))
    # key heads in two passes: 2^21 positions of 64 channels take 512 MiB a head
    x = batch([300], [400], kv_heads=3, heads=3)
    x.block_table = torch.nn.functional.pad(x.block_table, (0, (1 << 17) - x.block_table.shape[1]), value=-1)
    assert expands(x) and workspace(x, 300, 1 << 21) < 3 * (1 << 29)
    compare(attend(x, **kw), *attention(x, 64**-0.5))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("window", [1, 2, 16, 100, 128, 1000, 5000])
def test_windows(dtype, window) -> None:
    for qs, ks in (([1, 1, 1], [700, 90, 1]), ([300, 90, 5], [700, 90, 129])):
        for dim, bits in ((64, 8), (128, 4)):
            agree(QuantizedBatch(qs, ks, heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype, bits=bits, seed=window), window=window)


@pytest.mark.parametrize("dtype", ALL)
def test_pages_before_the_window_are_not_read(dtype) -> None:
    for qs, ks, window in (([1, 1], [900, 333], 100), ([60, 200], [900, 333], 70)):
        x = QuantizedBatch(qs, ks, heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, bits=4)
        want, bound = attention(x, 64**-0.5, True, window)
        for b, (nq, nk) in enumerate(zip(qs, ks)):
            first = max(0, nk - nq - window + 1)
            page, row = (t[:first] for t in x.slots[b])
            for c in (x.k, x.v):
                c.scales[page, row] = math.nan
            x.block_table[b, : first // 16] = -1
        compare(attend(x, window=window), want, bound)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("qs", [[1, 1, 1], [9, 3, 70], [200, 90, 70]])
def test_missing_pages_weigh_nothing(dtype, bits, qs) -> None:
    ks = [333, 90, 70]
    x = QuantizedBatch(qs, ks, heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, bits=bits)
    present = [torch.ones(n, dtype=torch.bool, device="cuda") for n in ks]
    for b, page, number in ((0, 3, -1), (0, 20, 10**6), (1, 0, -7)):
        x.block_table[b, page] = number
        present[b][16 * page : 16 * page + 16] = False
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = paged.paged_attention(x.q, *x.operands, max_q=max(qs), max_kv=max(ks), status=status)
    assert int(status) == 1
    compare(got, *attention(x, 64**-0.5, present=present))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("qs", [[1, 1], [6, 30], [150, 60]])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(dtype, bits, qs) -> None:
    ks = [150, 60]
    for what in ("k", "v"):
        x = QuantizedBatch(qs, ks, heads=4, kv_heads=2, dim=128, page=16, dtype=dtype, bits=bits)
        page, row = x.slots[0]
        # the last but one position: a row alone sees it in a chunk; and one group of a head in sequence 1
        getattr(x, what).scales[page[148], row[148], :] = math.nan
        page, row = x.slots[1]
        getattr(x, what).scales[page[59], row[59], 1, 1] = math.nan
        agree(x)


@pytest.mark.parametrize("dtype", ALL)
def test_lengths_past_the_block_table(dtype) -> None:
    """A length that the table cannot hold: what is there is read, tokens keep their positions."""
    for qs in ([1, 2], [80, 2]):
        x = QuantizedBatch(qs, [112, 40], heads=2, kv_heads=1, dim=64, page=16, dtype=dtype, bits=4)
        x.block_table = x.block_table[:, :7].contiguous()
        x.kv_lens = i32(130, 40)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = paged.paged_attention(x.q, *x.operands, max_q=max(qs), max_kv=130, status=status)
        assert int(status) == 1
        compare(got, *attention(x, 64**-0.5, lens=[130, 40]))


@pytest.mark.parametrize("dtype", ALL)
def test_bounds_that_are_too_small_or_absent(dtype) -> None:
    """max_q and max_kv size the launch; longer sequences are computed all the same."""
    for qs, ks in (([1, 1], [900, 40]), ([90, 20], [900, 40])):
        x = QuantizedBatch(qs, ks, heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, bits=4)
        for max_q, max_kv in ((1, 1), (None, None), (max(qs), 1), (1, 900), (max(qs), 100), (10**6, 10**6), (0, 0)):
            compare(attend(x, max_q=max_q, max_kv=max_kv), *attention(x, 64**-0.5))


@pytest.mark.parametrize("dtype", ALL)
def test_rows_that_no_sequence_has_are_zero(dtype) -> None:
    for qs in ([1, 1], [100, 40]):
        x = QuantizedBatch(qs, [130, 40], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, bits=4)
        n = sum(qs)
        want, bound = attention(x, 64**-0.5)
        x.q = torch.cat((torch.full_like(x.q[:2], 9.0), x.q, torch.full_like(x.q[:3], math.nan)))
        x.q_starts += 2
        out = torch.full_like(x.q, math.nan)
        paged.paged_attention(x.q, *x.operands, max_q=max(qs), max_kv=130, out=out)
        assert bool((out[:2] == 0).all()) and bool((out[n + 2 :] == 0).all())
        compare(out[2 : n + 2], want, bound)


def test_rows_of_q_starts_that_q_does_not_have() -> None:
    x = QuantizedBatch([30, 40], [130, 40], heads=4, kv_heads=2, dim=64, page=16, dtype="bf16", bits=4)
    want, bound = attention(x, 64**-0.5)
    guard = torch.full((100, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    guard[:50] = x.q[:50]
    out = torch.full_like(guard, 5.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.paged_attention(guard[:50], *x.operands, max_q=40, max_kv=130, out=out[:50], status=status)
    assert int(status) == 1 and bool((out[50:] == 5.0).all())
    compare(out[:50], want[:50], bound[:50])


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("qs,ks", [([1, 1], [9000, 40]), ([200, 3], [900, 40])])
def test_outputs_at_odd_elements(dtype, qs, ks) -> None:
    """Rows of out that allow single elements only, keys that would be cut into pieces."""
    x = QuantizedBatch(qs, ks, heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, bits=4)
    room = torch.full((sum(qs), 4, 67), 5.0, dtype=x.q.dtype, device="cuda")
    out = room[..., 1:65]
    assert paged.paged_attention(x.q, *x.operands, max_q=max(qs), max_kv=max(ks), out=out) is out
    compare(out, *attention(x, 64**-0.5))
    assert bool((room[..., 0] == 5.0).all()) and bool((room[..., 65:] == 5.0).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_queries_of_every_size(dtype, bits) -> None:
    """Rows of queries from 1e-30 to 1e30, the softmax flat or on one key: half's range does not show."""
    for qs, ks in (([6], [50]), ([120], [300])):
        x = QuantizedBatch(qs, ks, heads=2, kv_heads=1, dim=64, page=16, dtype=dtype, bits=bits)
        size = torch.tensor([1e-30, 1e-6, 1.0, 1e5, 1e20, 1e30], device="cuda").repeat(qs[0] // 6)[:, None, None]
        x.q = (x.q.float() * size).to(x.q.dtype)
        got = attend(x)
        want, _ = attention(x, 64**-0.5)
        # one key's weight is 1 to rounding for the large rows, all weights are equal to 1e-5 for the small ones; those
        # in between have the ordinary bound
        plain, bound = attention(x, 64**-0.5)
        rows = size[:, 0, 0].reshape(-1)
        middle = (rows > 1e-7) & (rows < 1e3)
        compare(got[middle], plain[middle], bound[middle])
        flat, peak = rows < 1e-7, rows > 1e3
        v = values(x.v.codes[x.slots[0]], x.v.scales[x.slots[0]], bits)
        most = float(v.abs().max())
        r = ROUND[dtype]
        assert float((got[flat].double() - want[flat]).abs().max()) <= most * (4 * r + 1e-5)
        assert float((got[peak].double() - want[peak]).abs().max()) <= most * (4 * r + 1e-5)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("bits", [4, 8])
def test_long_contexts(dtype, bits) -> None:
    agree(QuantizedBatch([1], [30011], heads=8, kv_heads=2, dim=128, page=64, dtype=dtype, bits=bits, spread=1.5))
    agree(QuantizedBatch([5, 1], [20000, 12345], heads=4, kv_heads=1, dim=96, page=24, dtype=dtype, bits=bits))
    agree(QuantizedBatch([1] * 40, [100 + 97 * b for b in range(40)], heads=8, kv_heads=2, dim=128, page=16, dtype=dtype, bits=bits))


@pytest.mark.parametrize("dtype", ALL)
def test_sizes_of_values_that_differ_by_thousands(dtype) -> None:
    """Tokens whose scales differ by far, the small ones holding the weight (as first tokens of trained models do)."""
    for n, qs in ((700, [1]), (700, [100])):
        x = QuantizedBatch(qs, [n], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, bits=4, seed=3)
        page, row = x.slots[0]
        g = torch.Generator(device="cuda").manual_seed(4)
        size = 10.0 ** (-4 * torch.rand(n, 1, 1, generator=g, device="cuda"))
        size[0], size[n // 2], size[n - 1] = 1e-4, 2e3, 1e-3
        x.v.codes[page, row], x.v.scales[page, row] = quantise(torch.randn(n, 2, 64, generator=g, device="cuda") * size, 4, 64)
        agree(x)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_scale_that_vanishes(dtype) -> None:
    """Scores that are 0 in fp32: weights are equal, and hidden keys stay hidden."""
    for qs, ks in (([3, 1], [40, 200]), ([300, 2], [333, 90])):
        x = QuantizedBatch(qs, ks, heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, bits=4)
        x.q = x.q * 1e-25
        want, bound = attention(x, 1e-25)
        compare(attend(x, scale=1e-25), want, bound)
        if many_rows(x):
            compare(attend(widened(x), scale=1e-25, max_kv=None), want, bound)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("bits", [4, 8])
def test_a_long_tail_far_below_one_key(dtype, bits) -> None:
    """One key 17 above 16383 others, whose weights are 2^-24.5 of its own, with a value of 0: the output is theirs."""
    for qs in ([1], [2]):
        x = QuantizedBatch(qs, [16384], heads=2, kv_heads=1, dim=64, page=64, dtype=dtype, bits=bits, gain=0.05)
        x.q[:] = x.q[:1, :1]
        q = x.q[0, 0].float()
        page, row = (t[100] for t in x.slots[0])
        x.v.scales[page, row] = 0.0
        x.k.codes[page, row, 0], x.k.scales[page, row, 0] = quantise(q * (17.0 * 8.0 / float(q.square().sum())), bits, 64)
        agree(x)


def test_offsets_that_pass_32_bits() -> None:
    """Pages 2 GiB apart: codes 4 GiB and scales 4 GiB from the first page."""
    dim, page, far = 64, 16, 1 << 31

    def pages():
        codes = torch.empty(2 * far + (1 << 20), dtype=torch.uint8, device="cuda").as_strided((3, page, 2, dim // 2), (far, 64, 32, 1))
        scales = torch.empty(far + (1 << 20), dtype=torch.float16, device="cuda").as_strided((3, page, 2, 1, 2), (far // 2, 4, 2, 2, 1))
        return paged.QuantizedPages(codes, scales, 4)

    x = QuantizedBatch([20, 1], [20, 11], heads=4, kv_heads=2, dim=dim, page=page, dtype="f16", bits=4)
    x.k, x.v = pages(), pages()
    x.block_table = torch.tensor([[2, 0], [1, -1]], dtype=torch.int32, device="cuda")
    x.slots = [(torch.tensor([2] * 16 + [0] * 4, device="cuda"), torch.tensor([*range(16), *range(4)], device="cuda")),
               (torch.full((11,), 1, device="cuda"), torch.arange(11, device="cuda"))]
    k, v = (torch.randn(31, 2, dim, device="cuda").half() for _ in range(2))
    at = (x.block_table, x.kv_lens, i32(0, 20, 31))
    paged.kv_append(k, v, x.k, x.v, *at)
    got = paged.kv_read(x.k, x.v, *at, rows=31)
    for src, back, c in ((k, got[0], x.k), (v, got[1], x.v)):
        codes, scales = quantise(src.float(), 4, dim)
        assert torch.equal(back, values(codes, scales, 4, torch.float32).half())
        assert torch.equal(c.codes[x.slots[0]], codes[:20]) and torch.equal(c.scales[x.slots[1]], scales[20:])
    compare(attend(x), *attention(x, dim**-0.5))


def test_scale_and_masked_rows_of_every_kind() -> None:
    x = QuantizedBatch([4, 3], [2, 300], heads=4, kv_heads=2, dim=64, page=16, dtype="f16", bits=8)
    compare(attend(x, scale=0.01), *attention(x, 0.01))
    got = attend(x)
    assert bool((got[:2] == 0).all())  # two tokens before position 0


@pytest.mark.parametrize("bits", [4, 8])
def test_the_same_call_twice_gives_the_same_bits(bits) -> None:
    for qs, ks in (([1] * 20, [50 * b + 1 for b in range(20)]), ([1], [20000]), ([300, 2], [2000, 900])):
        x = QuantizedBatch(qs, ks, heads=8, kv_heads=2, dim=128, page=16, dtype="bf16", bits=bits)
        a = attend(x)
        assert all(torch.equal(a, attend(x)) for _ in range(3))


# ---- the calls of a program ----------------------------------------------------------------------
def test_a_decoder_s_steps_together() -> None:
    """A prompt and then single tokens, each appended (normalised, rotated, quantised) and attended to, against
    64-bit attention over what kv_read says the cache holds."""
    heads, kv_heads, dim, page, batch = 8, 2, 128, 16, 3
    g = torch.Generator(device="cuda").manual_seed(0)
    k_cache, v_cache = (paged.quantized_pages(40, page, kv_heads, dim, bits=4) for _ in range(2))
    table = torch.randperm(40, generator=g, device="cuda")[:36].view(batch, 12).int()
    cos, sin = angles(256, dim)
    wq, wk = (1 + 0.2 * torch.randn(dim, generator=g, device="cuda") for _ in range(2))
    lens = [0] * batch
    for new in ([70, 5, 33], [1, 1, 1], [1, 0, 1], [3, 2, 4], [1, 1, 1]):
        lens = [a + b for a, b in zip(lens, new)]
        tokens = sum(new)
        at = (table, i32(*lens), i32(*np.concatenate([[0], np.cumsum(new)]).tolist()))
        qkv = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=g, device="cuda").bfloat16()
        q = paged.kv_append(qkv[:, heads : heads + kv_heads], qkv[:, heads + kv_heads :], k_cache, v_cache, *at, q=qkv[:, :heads],
                            cos=cos, sin=sin, q_norm=wq, k_norm=wk)
        got = paged.paged_attention(q, k_cache, v_cache, *at, max_q=max(new), max_kv=max(lens))
        x = QuantizedBatch.__new__(QuantizedBatch)
        x.qs, x.ks, x.share, x.name, x.bits, x.q, x.k, x.v = new, lens, heads // kv_heads, "bf16", 4, q, k_cache, v_cache
        x.slots = [(table[b, torch.arange(n, device="cuda") // page].long(), torch.arange(n, device="cuda") % page) for b, n in enumerate(lens)]
        compare(got, *attention(x, dim**-0.5))
        whole = i32(*np.concatenate([[0], np.cumsum(lens)]).tolist())
        k, v = paged.kv_read(k_cache, v_cache, table, at[1], whole, rows=sum(lens), dtype=torch.float32)
        for b in range(batch):
            part = slice(sum(lens[:b]), sum(lens[: b + 1]))
            assert torch.equal(k[part], values(k_cache.codes[x.slots[b]], k_cache.scales[x.slots[b]], 4, torch.float32))
            assert torch.equal(v[part], values(v_cache.codes[x.slots[b]], v_cache.scales[x.slots[b]], 4, torch.float32))


@pytest.mark.parametrize("qs,ks", [([1, 1, 1], [700, 5, 90]), ([100, 1, 3], [700, 5, 90])])
def test_graphs_and_other_streams(qs, ks) -> None:
    """Captured and replayed with changed contents, two graphs side by side, and on a stream of its own."""
    batches = [QuantizedBatch(qs, ks, heads=8, kv_heads=2, dim=128, page=16, dtype="bf16", bits=4, seed=s) for s in (1, 2)]
    graphs, outs = [], []
    for x in batches:
        kw = dict(max_q=max(qs), max_kv=max(ks))
        paged.paged_attention(x.q, *x.operands, **kw)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged.paged_attention(x.q, *x.operands, **kw))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for x in batches:
        x.q.mul_(0.5)
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for x, out in zip(batches, outs):
        compare(out, *attention(x, 128**-0.5))
    with torch.cuda.stream(streams[0]):
        got = [attend(x) for x in batches]
    for a, b in zip(got, outs):
        assert torch.equal(a, b)


def test_graphs_of_calls_that_expand() -> None:
    x = [widened(QuantizedBatch([300, 1], [700, 90], heads=4, kv_heads=2, dim=64, page=16, dtype="bf16", bits=4, seed=s)) for s in (1, 2)]
    assert all(expands(y) for y in x)
    graphs, outs = [], []
    for y in x:
        attend(y, max_kv=None)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged.paged_attention(y.q, *y.operands, max_q=300))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in x]
    for y in x:
        y.q.mul_(0.5)
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for y, out in zip(x, outs):
        compare(out, *attention(y, 64**-0.5))


def test_refusals() -> None:
    x = QuantizedBatch([1], [40], heads=4, kv_heads=2, dim=64, page=16, dtype="bf16", bits=4)
    table, lens, starts = x.operands[2:]
    with pytest.raises(GraphError, match="uint8 codes"):
        paged.paged_attention(x.q, (x.k.codes.float(), x.k.scales, 4), x.v, table, lens, starts)
    with pytest.raises(GraphError, match="uint8 codes"):
        paged.paged_attention(x.q, (x.k.codes, x.k.scales.float(), 4), x.v, table, lens, starts)
    with pytest.raises(GraphError, match="same bits"):
        paged.paged_attention(x.q, (x.k.codes, x.k.scales, 8), x.v, table, lens, starts)
    with pytest.raises(GraphError, match="scales"):
        paged.paged_attention(x.q, (x.k.codes, x.k.scales[:1], 4), x.v, table, lens, starts)
    with pytest.raises(GraphError, match="64"):
        paged.paged_attention(x.q[..., :32], x.k, x.v, table, lens, starts)
    with pytest.raises(GraphError, match="not quantised"):
        paged.kv_read(torch.zeros(2, 16, 2, 64, device="cuda").half(), torch.zeros(2, 16, 2, 64, device="cuda").half(), table, lens, starts, rows=1)
    with pytest.raises(GraphError, match="dtype"):
        paged.kv_read(*x.operands, rows=1, dtype=torch.float64)
    with pytest.raises(GraphError, match="not of dtype"):
        paged.kv_read(*x.operands, rows=1, k_out=torch.empty(1, 2, 64, device="cuda"))
    with pytest.raises(GraphError, match="gradient"):
        paged.paged_attention(x.q.float().requires_grad_(), *x.operands)
    kv = torch.zeros(1, 2, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(GraphError, match="norm weights"):
        paged.kv_append(kv, kv, *x.operands, k_norm=torch.ones(32, device="cuda"))
    with pytest.raises(GraphError, match="norm weights"):
        paged.kv_append(kv, kv, *x.operands, k_norm=torch.ones(64, device="cuda").half())
    with pytest.raises(GraphError, match="without q"):
        paged.kv_append(kv, kv, *x.operands, q_norm=torch.ones(64, device="cuda"))
    with pytest.raises(GraphError, match="eps is a number"):
        paged.kv_append(kv, kv, *x.operands, eps="x")
    with pytest.raises(GraphError, match="q's type"):
        paged.kv_append(kv, kv, *x.operands, q=x.q, q_out=x.q.float())
    with pytest.raises(GraphError, match="one type"):
        paged.kv_append(kv.float(), kv.float(), *x.operands, q=x.q)


def test_what_a_call_writes_counts_as_changed() -> None:
    x = QuantizedBatch([1], [40], heads=4, kv_heads=2, dim=64, page=16, dtype="bf16", bits=4)
    kv = torch.zeros(1, 2, 64, device="cuda", dtype=torch.bfloat16)
    seen = [t._version for c in (x.k, x.v) for t in (c.codes, c.scales)]
    paged.kv_append(kv, kv, *x.operands)
    assert all(t._version > s for t, s in zip((t for c in (x.k, x.v) for t in (c.codes, c.scales)), seen))
    out = torch.empty_like(kv)
    s = out._version
    paged.kv_read(*x.operands, rows=1, dtype=torch.bfloat16, k_out=out)
    assert out._version > s
