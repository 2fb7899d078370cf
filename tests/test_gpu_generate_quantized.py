"""The token-by-token GPT-2 over a cache of 4 or 8 bits, against float64 over what its own cache holds."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from mgc_cuda import generate  # noqa: E402
from mgc_cuda.paged import kv_read  # noqa: E402

pytestmark = pytest.mark.gpu


def layer_over(model: generate.Gpt2, ids: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """Logits after the last token of a one-layer model, its queries attending to keys and values [n, heads, dim] that
    are given, in float64."""
    def norm(x: torch.Tensor, ln: tuple[torch.Tensor, torch.Tensor]) -> torch.Tensor:
        return torch.nn.functional.layer_norm(x, (model.d,), ln[0].double(), ln[1].double(), 1e-5)

    n, heads, dim = int(ids.shape[0]), model.heads, model.d // model.heads
    b = model.blocks[0]
    w = {key: (m.double(), c.double()) for key, (m, c) in b.items()}
    x = model.wte[ids[-1:]].double() + model.wpe[n - 1 : n].double()
    q = (norm(x, b["ln1"]) @ w["qkv"][0].T + w["qkv"][1]).view(3, heads, dim)[0]
    p = torch.softmax(torch.einsum("hd,nhd->hn", q, k.double()) * dim**-0.5, -1)
    x = x + torch.einsum("hn,nhd->hd", p, v.double()).reshape(1, model.d) @ w["proj"][0].T + w["proj"][1]
    h = torch.nn.functional.gelu(norm(x, b["ln2"]) @ w["up"][0].T + w["up"][1], approximate="tanh")
    x = x + h @ w["down"][0].T + w["down"][1]
    return norm(x, model.ln) @ model.wte.double().T


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("precision,tol", [(generate.FP32, 1e-4), (generate.TF32, 2e-2)])  # as with unquantised caches
def test_logits_follow_from_the_cache(bits: int, precision: int, tol: float) -> None:
    model = generate.Gpt2(layers=1, d=128, heads=2, vocab=512, max_pos=256, cache_bits=bits, precision=precision)
    pages, cache = generate.Pages(24, 16, 3, model.device), model.cache(24, 16)
    seqs: list[list[int]] = [[], [], []]
    g = torch.Generator().manual_seed(0)
    for new in ([70, 1, 17], [1, 1, 1], [20, 0, 3], [1, 1, 1]):
        ids = [torch.randint(512, (n,), generator=g).tolist() for n in new]
        for seq, part in zip(seqs, ids):
            seq += part
        got = model.step(torch.tensor(sum(ids, []), device="cuda"), new, pages, cache)
        lens = torch.tensor(pages.lens, dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, *torch.tensor(pages.lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
        width = max(len(p) for p in pages.owned)
        table = torch.tensor([p + [0] * (width - len(p)) for p in pages.owned], dtype=torch.int32, device="cuda")
        k, v = kv_read(*cache[0], table, lens, starts, rows=sum(pages.lens), dtype=torch.float32)
        rows = iter(got)
        for b, n in enumerate(new):
            if n:
                part = slice(int(starts[b]), int(starts[b + 1]))
                want = layer_over(model, torch.tensor(seqs[b], device="cuda"), k[part], v[part])
                assert float((next(rows).double() - want[0]).abs().max()) <= tol


@pytest.mark.parametrize("bits", [4, 8])
def test_generation_runs(bits: int) -> None:
    model = generate.Gpt2(layers=3, d=128, heads=2, vocab=512, max_pos=256, cache_bits=bits)
    prompts = [list(range(1, 91)), [7], list(range(40, 57))]
    out, _, logits = generate.generate(model, prompts, 20, chunk=32)
    assert [len(s) for s in out] == [len(p) + 20 for p in prompts] and bool(torch.isfinite(logits).all())
    assert generate.main(["--batch", "2", "--prompt", "40", "--tokens", "3", "--layers", "2", "--cache", f"int{bits}"]) == 0


def test_refusals() -> None:
    with pytest.raises(ValueError, match="cache_bits"):
        generate.Gpt2(layers=1, d=64, heads=1, vocab=16, cache_bits=4, cache_dtype=torch.float16)
    with pytest.raises(SystemExit):
        generate.main(["--cache", "int4", "--check"])
