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
