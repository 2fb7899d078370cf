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


# ---- gradients -----------------------------------------------------------------------------------
@pytest.mark.parametrize("which", ["q", "k_cache", "v_cache", "out"])
def test_attention_refuses_to_lose_a_gradient(which: str) -> None:
    """There is no backward pass: a result without history would train nothing and say nothing."""
    x = batch()
    out = torch.empty_like(x.q)
    t = {"q": x.q, "k_cache": x.k, "v_cache": x.v, "out": out}

    def call():
        return paged.paged_attention(t["q"], t["k_cache"], t["v_cache"], *x.operands[2:], out=t["out"])

    want = call().clone()
    t[which] = t[which].detach().requires_grad_()
    with pytest.raises(GraphError, match="gradient"):
        call()
    with torch.no_grad():
        got = call()
    assert torch.equal(got, want) and (which == "out" or not got.requires_grad)


@pytest.mark.parametrize("which", ["k", "v", "q", "k_cache", "v_cache", "cos", "q_out"])
def test_append_refuses_to_lose_a_gradient(which: str) -> None:
    x = batch()
    cos, sin = angles(16, 64)
    t = {"k": x.q[:, :2], "v": x.q[:, 2:], "q": x.q, "k_cache": x.k, "v_cache": x.v, "cos": cos, "q_out": torch.empty_like(x.q)}

    def call():
        return paged.kv_append(t["k"], t["v"], t["k_cache"], t["v_cache"], *x.operands[2:], q=t["q"], cos=t["cos"], sin=sin,
                               q_out=t["q_out"])

    t[which] = t[which].detach().requires_grad_()
    with pytest.raises(GraphError, match="gradient"):
        call()
    with torch.no_grad():
        call()


def test_what_a_call_writes_counts_as_changed() -> None:
    """Autograd sees that a tensor it saved was written since."""
    x = batch()
    out, q_out = torch.empty_like(x.q), torch.empty_like(x.q)
    tensors = [x.k, x.v, out, q_out]
    before = [t._version for t in tensors]
    paged.kv_append(x.q[:, :2], x.q[:, 2:], *x.operands, q=x.q, q_out=q_out)
    paged.paged_attention(x.q, *x.operands, out=out)
    assert all(t._version > v for t, v in zip(tensors, before))
    weight = torch.ones(1, device="cuda", requires_grad=True)
    loss = (weight * x.k.nan_to_num(0.0)).sum() + (weight * x.v).sum()
    paged.kv_append(x.q[:, :2], x.q[:, 2:], *x.operands)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_inference_tensors_are_written() -> None:
    with torch.inference_mode():
        x = batch()
        paged.kv_append(x.q[:, :2], x.q[:, 2:], *x.operands)
        paged.paged_attention(x.q, *x.operands, out=torch.empty_like(x.q))
