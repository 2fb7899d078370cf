"""The fp32 bound of paged_exact.reference tells a right computation from one with a lost split."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from paged_cases import PagedBatch  # noqa: E402
from paged_exact import reference  # noqa: E402


def tf32(x: torch.Tensor) -> torch.Tensor:
    """Rounded to 11 significant bits."""
    i = x.view(torch.int32)
    return ((i + 0x1000) & ~0x1FFF).view(torch.float32)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [17, 600, 4097])
def test_the_bound_notices_an_unsplit_product(dim: int, n: int) -> None:
    x = PagedBatch([1, 5], [n, 40], heads=4, kv_heads=2, dim=dim, page=16, dtype="f32", device="cpu")
    want, bound = reference(x, dim**-0.5)

    def worst(round_scores, round_values) -> float:
        top = 0.0
        for b, (nq, nk) in enumerate(zip(x.qs, x.ks)):
            k, v, q = x.k[x.slots[b]], x.v[x.slots[b]], x.q[x.rows(b)].contiguous()
            hidden = torch.arange(nk)[None] > torch.arange(nk - nq, nk)[:, None]
            for h in range(4):
                s = round_scores(q[:, h].contiguous()) @ round_scores(k[:, h // 2].contiguous()).T * dim**-0.5
                w = torch.softmax(s.masked_fill(hidden, -torch.inf), -1)
                o = round_values(w) @ round_values(v[:, h // 2].contiguous())
                top = max(top, float(((o.double() - want[x.rows(b), h]).abs() / bound[x.rows(b), h]).max()))
        return top

    assert worst(lambda t: t, lambda t: t) <= 1.0
    assert worst(tf32, lambda t: t) > 3.0
    assert worst(lambda t: t, tf32) > 3.0
