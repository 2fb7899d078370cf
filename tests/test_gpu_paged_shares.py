"""Paged attention whose keys are shared out over all SMs: units cut between blocks, their pieces added
by a second kernel. Every value is marked with its place among the keys, so that a lost, doubled or
misplaced piece of a few keys shows; fp32 at a bound that an unsplit product would miss by far."""

from __future__ import annotations

import math
import threading

import pytest

torch = pytest.importorskip("torch")

from mgc_cuda import paged  # noqa: E402
from paged_cases import PagedBatch  # noqa: E402
from paged_exact import compare, reference, workspace  # noqa: E402

pytestmark = pytest.mark.gpu

ALL = ["f32", "f16", "bf16"]


def marked(x: PagedBatch) -> PagedBatch:
    """Channel c's values are 0 outside the c-th part of the sequence, so an output channel is the weight of
    that part and its error is relative to that."""
    dim = x.v.shape[3]
    for (page, row), n in zip(x.slots, x.ks):
        part = torch.arange(n, device="cuda") * dim // max(n, 1)
        x.v[page, row] = ((1.0 + 0.25 * x.v[page, row].float().abs()) * torch.eye(dim, device="cuda")[part][:, None]).to(x.v.dtype)
    return x


def check(x: PagedBatch, **kw) -> None:
    out = torch.full(x.q.shape, math.nan, dtype=x.q.dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = reference(x, x.q.shape[2] ** -0.5, **kw)
    for _ in range(2):  # the second call's workspace holds the first's pieces
        paged.paged_attention(x.q, *x.operands, max_q=max(x.qs), max_kv=max(x.ks), out=out, status=status, **kw)
        compare(out, *want)
    paged.check_status(status)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("group", [1, 2, 4, 8, 20])
@pytest.mark.parametrize("kv_heads,n,dim", [(1, 131071, 64), (1, 70001, 128), (1, 40000, 256), (3, 50000, 96), (7, 30011, 128)])
def test_one_long_sequence(dtype: str, group: int, kv_heads: int, n: int, dim: int) -> None:
    """With one key head a row is cut into more pieces than four warps' lanes (128)."""
    x = marked(PagedBatch([1], [n], heads=group * kv_heads, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype))
    assert workspace(x) > 0
    check(x)


BATCH = [17, 4096, 1, 0, 300, 2900, 4095, 64, 65, 1500] * 6 + [4000, 9, 128, 2047]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (15, 5), (7, 7), (12, 12), (66, 6)])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_ragged_batches(dtype: str, heads: int, kv_heads: int, dim: int) -> None:
    """Key heads that divide the number of blocks, and ones that do not."""
    x = marked(PagedBatch([1] * 64, BATCH, heads=heads, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype))
    assert workspace(x) > 0
    check(x)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("window", [1, 100, 1900, 3000])
@pytest.mark.parametrize("tokens", [1, 3])
def test_windows_over_cut_units(dtype: str, window: int, tokens: int) -> None:
    x = marked(PagedBatch([tokens] * 64, [max(n, tokens) for n in BATCH], heads=16, kv_heads=8, dim=64, page=16, dtype=dtype))
    assert workspace(x, window=window) > 0 or window < 1000
    check(x, window=window)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("page", [24, 100, 64])
@pytest.mark.parametrize("qs,ks,heads,kv_heads,dim", [
    ([200, 1, 70] * 6, [3000, 5000, 70] * 6, 8, 2, 128), ([40, 1, 33] * 20, [3000, 700, 33] * 20, 6, 6, 64),
    ([5] * 64, [2000, 1300, 40, 5] * 16, 16, 4, 80), ([5] * 128, [2000, 1300, 40, 5] * 32, 8, 4, 64),
    ([150, 3, 64] * 30, [1700, 900, 64] * 30, 2, 1, 256),
])
def test_chunks(dtype: str, page: int, qs, ks, heads: int, kv_heads: int, dim: int) -> None:
    """Row tiles of 16, 32 and 64 on the warp-level products, and the tcgen05 kernel where page and type allow."""
    x = marked(PagedBatch(qs, ks, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype))
    assert workspace(x) > 0
    check(x)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 7, 8, 9, 16, 17, 32, 33, 64, 65])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("n", [1, 17, 300, 2001])
def test_fp32_at_its_own_precision(rows: int, dim: int, n: int) -> None:
    """Every form of the fp32 kernels (1 to 8 rows on the FMA units, 16, 32, 64 in split products), as heads of
    a token and as tokens of a head."""
    check(PagedBatch([1, 1], [n, max(1, n // 3)], heads=rows, kv_heads=1, dim=dim, page=16, dtype="f32", seed=n + rows))
    if rows <= n:
        check(PagedBatch([rows, 1], [n, 5], heads=2, kv_heads=2, dim=dim, page=16, dtype="f32", seed=n + rows))


@pytest.mark.parametrize("dtype", ALL)
def test_bits_repeat_and_are_right(dtype: str) -> None:
    for qs, ks in (([1] * 64, BATCH), ([300, 5], [3000, 900])):
        x = marked(PagedBatch(qs, ks, heads=8, kv_heads=2, dim=128, page=16, dtype=dtype))
        first = paged.paged_attention(x.q, *x.operands, max_q=max(qs), max_kv=max(ks))
        compare(first, *reference(x, 128**-0.5))
        for _ in range(5):
            assert torch.equal(paged.paged_attention(x.q, *x.operands, max_q=max(qs), max_kv=max(ks)), first)


def test_two_threads_with_a_stream_each() -> None:
    """Calls share nothing: each thread's workspace comes from its own stream."""
    batches = [marked(PagedBatch([1] * 64, BATCH, heads=16, kv_heads=4, dim=64, page=16, dtype="bf16", seed=s)) for s in (1, 2)]
    want = [paged.paged_attention(x.q, *x.operands, max_q=1, max_kv=4096) for x in batches]
    torch.cuda.synchronize()
    wrong: list[int] = []

    def serve(i: int) -> None:
        x = batches[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                k = x.q[:, :4].contiguous()
                before = x.k.clone()
                paged.kv_append(k, k, before, x.v.clone(), *x.operands[2:])
                got = paged.paged_attention(x.q, *x.operands, max_q=1, max_kv=4096)
                if not torch.equal(got, want[i]):
                    wrong.append(i)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=serve, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
