"""The token-by-token GPT-2 example: chunks and single tokens over the paged cache against one plain
computation over the whole sequence."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from mgc_cuda import generate  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,precision,tol", [
    # exact-fp32 products and cache: rounding of a few fp32 operations a layer, 1e-4 of unit-size logits
    (torch.float32, generate.FP32, 1e-4),
    # TF32 products (the framework's 2e-2 logit budget), caches of 11 and 8 significant bits within it
    (torch.float32, generate.TF32, 2e-2), (torch.float16, generate.TF32, 2e-2), (torch.bfloat16, generate.TF32, 2e-2),
])
def test_generation_matches_the_whole_sequence(dtype, precision: int, tol: float) -> None:
    model = generate.Gpt2(layers=3, d=128, heads=2, vocab=512, max_pos=256, cache_dtype=dtype, precision=precision)
    prompts = [list(range(1, 91)), [7], list(range(40, 57))]
    out, _, logits = generate.generate(model, prompts, 20, chunk=32)
    for b, seq in enumerate(out):
        assert seq[: len(prompts[b])] == prompts[b] and len(seq) == len(prompts[b]) + 20
        want = model.plain(torch.tensor(seq[:-1], device="cuda"))[0]
        assert float((logits[b].double() - want).abs().max()) <= tol


def test_pages_are_reused_and_run_out() -> None:
    pages = generate.Pages(4, 16, 2, torch.device("cuda"))
    table, lens, starts = pages.extend([33, 5])
    assert lens.tolist() == [33, 5] and starts.tolist() == [0, 33, 38] and table.shape == (2, 3)
    with pytest.raises(RuntimeError, match="no free page"):
        pages.extend([0, 12])
    pages.release(0)
    assert len(pages.free) == 3 and pages.lens[0] == 0


def test_the_command_checks_itself() -> None:
    assert generate.main(["--batch", "2", "--prompt", "40", "--tokens", "5", "--layers", "2", "--check"]) == 0


@pytest.mark.parametrize("d,heads,vocab", [(66, 2, 101), (65, 5, 64), (60, 3, 99)])
@pytest.mark.parametrize("precision,tol", [(generate.FP32, 1e-4), (generate.TF32, 2e-2)])
def test_widths_that_are_no_multiple_of_four(d: int, heads: int, vocab: int, precision: int, tol: float) -> None:
    model = generate.Gpt2(layers=2, d=d, heads=heads, vocab=vocab, max_pos=64, precision=precision)
    out, _, logits = generate.generate(model, [list(range(1, 31)), [7]], 4, chunk=16)
    for b, seq in enumerate(out):
        want = model.plain(torch.tensor(seq[:-1], device="cuda"))[0]
        assert float((logits[b].double() - want).abs().max()) <= tol
