"""The host side of the token-by-token GPT-2 example: pages handed out to sequences, refused prompts."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from mgc_cuda import generate  # noqa: E402


def test_a_failed_extend_changes_nothing() -> None:
    """No free page: the caller releases a sequence and tries again."""
    pages = generate.Pages(4, 16, 3, torch.device("cpu"))
    pages.extend([33, 5, 0])
    before = (list(pages.lens), [list(p) for p in pages.owned], list(pages.free))
    with pytest.raises(RuntimeError, match="no free page"):
        pages.extend([0, 12, 3])
    assert (pages.lens, pages.owned, pages.free) == before
    pages.release(0)
    table, lens, starts = pages.extend([0, 12, 3])
    assert lens.tolist() == [0, 17, 3] and starts.tolist() == [0, 0, 12, 15]
    used = [table[b, : -(-n // 16)].tolist() for b, n in enumerate(lens.tolist())]
    assert len(sum(used, [])) == len(set(sum(used, []))) == 3


def test_empty_prompts_are_refused() -> None:
    """A sequence without a token has no logits to go on from."""

    class Untouched:
        def __getattribute__(self, name: str):
            raise AssertionError(f"{name} was used")

    for prompts in ([[1, 2], []], [[]], []):
        with pytest.raises(ValueError, match="prompt"):
            generate.generate(Untouched(), prompts, 4)
