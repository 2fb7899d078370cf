"""paged_attention and kv_append at the borders of their definition, against 64 bits."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from mgc_cuda import paged  # noqa: E402
from mgc_cuda._errors import GraphError  # noqa: E402
from paged_cases import PagedBatch  # noqa: E402
from paged_exact import compare, reference  # noqa: E402

pytestmark = pytest.mark.gpu

ALL = ["f32", "f16", "bf16"]


def attend(x: PagedBatch, status=None, **kw):
    kw.setdefault("max_q", max(x.qs))
    kw.setdefault("max_kv", max(x.ks))
    out = torch.full(x.q.shape, math.nan, dtype=x.q.dtype, device="cuda")
    return paged.paged_attention(x.q, *x.operands, out=out, status=status, **kw)


# ---- keys that cannot be read --------------------------------------------------------------------
BATCHES = [
    ([1, 1, 1], [300, 20, 40]),              # single tokens, a cluster to each
    ([3, 2, 1], [300, 20, 40]),              # a few tokens
    ([200, 3, 17], [300, 20, 40]),           # chunks
    ([1] * 40, [4000, 20, 40, *range(900, 937)]),  # even shares of a batch
    ([300, 150, 40], [1500, 400, 40]),
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("layout", ["tokens", "odd"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (64, 128), (128, 8), (96, 24)])
@pytest.mark.parametrize("qs,ks", BATCHES)
def test_keys_of_bad_pages_are_left_out(dtype: str, layout: str, dim: int, page: int, qs, ks) -> None:
    """A page number outside the cache: its keys weigh nothing, in every kernel; other sequences and the
    rest of its own are untouched. A sequence of bad pages only gets zeros."""
    x = PagedBatch(qs, ks, heads=4, kv_heads=2, dim=dim, page=page, dtype=dtype, layout=layout)
    present = [torch.ones(n, dtype=torch.bool, device="cuda") for n in ks]
    bad = [-1, x.k.shape[0], 1 << 30]
    pages = -(-ks[0] // page)
    for i, slot in enumerate(sorted({0, pages // 2, pages - 1})):
        x.block_table[0, slot] = bad[i]
        present[0][slot * page : (slot + 1) * page] = False
    x.block_table[2] = -1
    present[2][:] = False
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = attend(x, status)
    with pytest.raises(GraphError, match="out of range"):
        paged.check_status(status)
    compare(got, *reference(x, dim**-0.5, present=present))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("layout", ["tokens", "odd"])
@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("length", [37, 0x7FFFFFFF])
@pytest.mark.parametrize("qs,ks", BATCHES)
def test_lengths_past_the_block_table_keep_their_positions(dtype: str, layout: str, window: int, length: int, qs, ks) -> None:
    """Positions that the block table does not reach cannot be read; the new tokens stay where they are."""
    page = 16
    full = -(-max(ks) // page) * page
    ks = [full, *ks[1:]]
    x = PagedBatch(qs, ks, heads=4, kv_heads=2, dim=64, page=page, dtype=dtype, layout=layout)
    x.block_table = x.block_table[:, : full // page].contiguous()
    lens = [full + 37 if length == 37 else length, *ks[1:]]
    x.kv_lens[0] = lens[0]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = attend(x, status, window=window)
    with pytest.raises(GraphError, match="out of range"):
        paged.check_status(status)
    compare(got, *reference(x, 64**-0.5, window=window, lens=lens))


# ---- rows that the operands do not have ----------------------------------------------------------
def inside(x: PagedBatch):
    """x.q, its out and its cache-sized operands as views of larger buffers whose other rows must stay as
    they are: what a kernel reads or writes past the views shows there."""
    room = torch.full((x.q.shape[0] + 600, *x.q.shape[1:]), math.nan, dtype=x.q.dtype, device="cuda")
    room[300:-300] = x.q
    out = torch.full_like(room, 7.0)
    x.q = room[300:-300]
    return out


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("layout", ["tokens", "odd"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shift", [-2, 3, 200])
@pytest.mark.parametrize("qs,ks", BATCHES)
def test_rows_past_the_operands_are_left_out(dtype: str, layout: str, dim: int, shift: int, qs, ks) -> None:
    """q_starts that begin before the first row or end after the last: the rows that exist keep their
    positions, nothing else is read or written, and the status says so."""
    x = PagedBatch(qs, ks, heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype, layout=layout)
    out = inside(x)
    tokens = x.q.shape[0]
    starts = [0]
    for n in qs:
        starts.append(starts[-1] + n)
    if shift < 0:
        starts[0] = shift
    else:
        starts[-1] += shift
    x.q_starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
    # the sequence that is too long has its other tokens before the first row or after the last
    lens = list(x.ks)
    if shift > 0:
        lens[-1] -= shift
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = out[300:-300]
    paged.paged_attention(x.q, *x.operands, out=got, max_q=max(qs) + abs(shift), max_kv=max(ks), status=status)
    with pytest.raises(GraphError, match="out of range"):
        paged.check_status(status)
    compare(got, *reference(x, dim**-0.5, lens=lens))
    assert bool((out[:300] == 7.0).all()) and bool((out[300 + tokens :] == 7.0).all())


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("layout", ["tokens", "odd"])
@pytest.mark.parametrize("starts", [[0, 0x7FFFFFFF], [-0x7FFFFFFF, 0x7FFFFFFF], [5, 3], [100, 400], [-9, -2], [0, -5]])
@pytest.mark.parametrize("tokens", [1, 3, 150])
def test_any_starts_stay_inside_the_operands(dtype: str, layout: str, starts, tokens: int) -> None:
    x = PagedBatch([tokens, 1], [200, 9], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, layout=layout)
    out = inside(x)
    x.q_starts = torch.tensor([*starts, starts[-1]], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.paged_attention(x.q, *x.operands, out=out[300:-300], max_q=tokens, max_kv=200, status=status)
    with pytest.raises(GraphError, match="out of range"):
        paged.check_status(status)
    assert bool((out[:300] == 7.0).all()) and bool((out[-300:] == 7.0).all())


def test_append_with_rows_past_the_operands() -> None:
    x = PagedBatch([3, 4], [40, 9], heads=4, kv_heads=2, dim=64, page=16, dtype="bf16")
    k = torch.randn(7, 2, 64, device="cuda").to(torch.bfloat16)
    x.q_starts = torch.tensor([0, 3, 9], dtype=torch.int32, device="cuda")
    before = x.k.clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.kv_append(k, k, *x.operands, status=status)
    with pytest.raises(GraphError, match="out of range"):
        paged.check_status(status)
    for b, rows, at in ((0, slice(0, 3), slice(37, 40)), (1, slice(3, 7), slice(3, 7))):
        page, row = x.slots[b]
        before[page[at], row[at]] = k[rows]
    assert torch.equal(before.nan_to_num(7.0), x.k.nan_to_num(7.0))


# ---- rows of q that no sequence has --------------------------------------------------------------
def padded(qs, ks, before: int, after: int, **kw) -> PagedBatch:
    """A batch with rows of q in front of the first sequence's and behind the last one's."""
    x = PagedBatch([before, *qs, after], [before, *ks, after], **kw)
    x.qs, x.ks, x.slots = x.qs[1:-1], x.ks[1:-1], x.slots[1:-1]
    x.block_table, x.kv_lens, x.q_starts = x.block_table[1:-1], x.kv_lens[1:-1], x.q_starts[1:-1]
    x.before = before
    x.rows = lambda b: slice(before + sum(x.qs[:b]), before + sum(x.qs[: b + 1]))
    return x


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("layout", ["tokens", "odd"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("before,after", [(0, 5), (3, 0), (2, 300)])
@pytest.mark.parametrize("qs,ks", BATCHES)
def test_rows_of_no_sequence_get_zeros(dtype: str, layout: str, dim: int, before: int, after: int, qs, ks) -> None:
    """A batch padded to a fixed number of rows, as a captured graph runs it."""
    x = padded(qs, ks, before, after, heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype, layout=layout)
    compare(attend(x), *reference(x, dim**-0.5))


@pytest.mark.parametrize("dtype", ALL)
def test_queries_of_no_sequence_are_copied(dtype: str) -> None:
    """kv_append returns them as they are, and caches nothing for them."""
    x = padded([3, 40], [20, 40], 2, 70, heads=4, kv_heads=2, dim=64, page=16, dtype=dtype)
    a = torch.arange(64, device="cuda")[:, None] * torch.linspace(0.1, 1.0, 32, device="cuda")
    k = x.q[:, :2]
    before = [x.k.clone(), x.v.clone()]
    out = torch.full(x.q.shape, math.nan, dtype=x.q.dtype, device="cuda")
    paged.kv_append(k, k, *x.operands, q=x.q, q_out=out, cos=a.cos(), sin=a.sin())
    assert torch.equal(out[:2], x.q[:2]) and torch.equal(out[-70:], x.q[-70:])
    for b in range(2):
        page, row = x.slots[b]
        at = torch.arange(x.ks[b] - x.qs[b], x.ks[b], device="cuda")
        for was, now in zip(before, (x.k, x.v)):
            was[page[at], row[at]] = now[page[at], row[at]]
    for was, now in zip(before, (x.k, x.v)):
        assert torch.equal(was.nan_to_num(7.0), now.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", ALL)
def test_rows_without_any_sequence(dtype: str) -> None:
    x = padded([], [], 3, 4, heads=4, kv_heads=2, dim=64, page=16, dtype=dtype)
    out = torch.full(x.q.shape, math.nan, dtype=x.q.dtype, device="cuda")
    assert not paged.paged_attention(x.q, *x.operands, out=out).any()
    assert torch.equal(paged.kv_append(x.q[:, :2], x.q[:, :2], *x.operands, q=x.q), x.q)


# ---- weights far below the largest ---------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("below", [10.0, 17.0, 17.4])
@pytest.mark.parametrize("qs,n", [([1], 131072), ([1], 16384), ([24], 16384), ([150], 16384)])
def test_one_key_above_a_long_flat_tail(dtype: str, dim: int, below: float, qs, n: int) -> None:
    """The first key's score is `below` above all others', whose weights together still count: below half
    precision's range, 131071 of them hold 3.6e-3 of the mass at 17.4."""
    x = PagedBatch(qs, [n], heads=2, kv_heads=1, dim=dim, page=16, dtype=dtype)
    x.q.zero_()
    x.q[..., 0] = 8.0
    page, row = x.slots[0]
    x.k[page, row, :, 0] = 0.0
    x.k[page[0], row[0], :, 0] = below
    x.v[page, row] = x.v[page, row].abs()
    x.v[page[0], row[0]] = 0.0
    compare(attend(x, scale=0.125), *reference(x, 0.125))


# ---- values that are not finite ------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("layout", ["tokens", "odd"])
@pytest.mark.parametrize("qs,ks", [([1], [300]), ([1, 1], [9000, 40]), ([2], [90]), ([4, 1], [300, 33]), ([9], [100]), ([30], [200])])
def test_infinite_and_nan_values_that_are_seen(dtype: str, layout: str, qs, ks) -> None:
    """A value's infinity or NaN reaches its channel and no other."""
    x = PagedBatch(qs, ks, heads=2, kv_heads=2, dim=64, page=16, dtype=dtype, layout=layout)
    page, row = x.slots[0]
    x.v[page[5], row[5], 0, 3] = math.inf
    x.v[page[6], row[6], 0, 4] = -math.inf
    x.v[page[7], row[7], 1, 5] = math.nan
    x.v[page[8], row[8], 1, 6] = math.inf
    x.v[page[9], row[9], 1, 6] = -math.inf
    if dtype == "f32":
        x.v[page[10], row[10], 0, 7] = 3.4028e38
    compare(attend(x), *reference(x, 64**-0.5))


HIDDEN = [([3], [40], 0), ([2, 1], [300, 40], 0), ([4], [40], 8), ([24], [300], 0), ([24], [300], 50), ([60], [700], 300),
          ([150], [400], 0), ([300], [400], 0), ([300, 40], [1500, 90], 100), ([600], [600], 70)]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("layout", ["tokens", "odd"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("qs,ks,window", HIDDEN)
def test_values_that_a_row_does_not_see_do_not_reach_it(dtype: str, layout: str, dim: int, qs, ks, window: int) -> None:
    """Infinities and NaN at positions that some new tokens see and others, earlier or later ones, do not."""
    x = PagedBatch(qs, ks, heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype, layout=layout)
    page, row = x.slots[0]
    n, first = ks[0], ks[0] - qs[0]
    for i, at in enumerate(sorted({n - 1, n - 2, first + qs[0] // 2, first + 1, max(0, first - window), max(0, first - window + 1)})):
        x.v[page[at], row[at], :, 2 * i] = (math.inf, math.nan, -math.inf)[i % 3]
        x.k[page[at], row[at], 1, 0] = (math.nan, math.inf)[i % 2] if at == n - 1 else x.k[page[at], row[at], 1, 0]
    want, bound = reference(x, dim**-0.5, window=window)
    got = attend(x, window=window)
    # the last token sees a key that is not finite: what its second head group gets is undefined
    want[x.rows(0).stop - 1, 2:], got[x.rows(0).stop - 1, 2:], bound[x.rows(0).stop - 1, 2:] = 0.0, 0.0, 1.0
    compare(got, want, bound)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("qs", [[300], [30]])
def test_rows_computed_again_over_a_long_context(dtype: str, dim: int, qs) -> None:
    """No wait of the other warps runs out meanwhile."""
    x = PagedBatch(qs, [30000], heads=8, kv_heads=2, dim=dim, page=16, dtype=dtype)
    page, row = x.slots[0]
    x.v[page[-1], row[-1], :, 5] = math.nan
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = attend(x, status)
    paged.check_status(status)
    compare(got, *reference(x, dim**-0.5))
