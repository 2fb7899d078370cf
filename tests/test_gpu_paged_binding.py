"""What the torch binding of the paged-cache operators takes and refuses beyond types and shapes."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from mgc_cuda import paged  # noqa: E402
from mgc_cuda._errors import GraphError  # noqa: E402
from paged_cases import PagedBatch, angles  # noqa: E402

pytestmark = pytest.mark.gpu


def batch() -> PagedBatch:
    return PagedBatch([2], [9], heads=4, kv_heads=2, dim=64, page=16, dtype="f32")


class Neither:
    def __bool__(self) -> bool:
        raise TypeError("neither true nor false")


@pytest.mark.parametrize("value", [Neither(), torch.tensor([True, False])])
def test_flags_without_a_truth_value_are_refused(value) -> None:
    x = batch()
    with pytest.raises(GraphError, match="causal"):
        paged.paged_attention(x.q, *x.operands, causal=value)
    cos, sin = angles(16, 64)
    for tables in ({}, {"cos": cos, "sin": sin}):
        with pytest.raises(GraphError, match="interleaved"):
            paged.kv_append(x.q[:, :2], x.q[:, :2], *x.operands, interleaved=value, **tables)
