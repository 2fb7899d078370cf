"""Token-by-token GPT-2 on the kernel ABI: prompts in chunks and then one token at a time over a paged
cache, where a compiled graph computes a whole sequence of fixed length.

``Gpt2`` holds a decoder of the GPT-2 layout (pre-LayerNorm, tanh GELU, learned positions, head tied to
the token embedding; ``zoo.gpt2``'s) with random weights, and runs one step for a batch
of sequences with any number of new tokens each: layer norms, products and epilogues by
``mgc_cuda_layer_norm`` and ``mgc_cuda_gemm``, the cache and its attention by ``mgc_cuda.paged``.
``Pages`` hands out the pages of a cache to sequences.

    python ml-graph-compiler_b200/mgc_cuda/generate.py --batch 4 --prompt 100 --tokens 32

generates greedily from random prompts with random weights and prints the time per step; ``--check``
compares the last step's logits with a plain computation over the whole sequences.
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch  # noqa: E402

from mgc_cuda.native import check, library  # noqa: E402
from mgc_cuda.paged import check_status, kv_append, paged_attention  # noqa: E402

ACT_NONE, ACT_GELU_TANH = 0, 4  # MGC_ACT_*
FP32, TF32 = 0, 1  # MGC_PREC_*


class Pages:
    """The pages of a cache, handed out to sequences as they grow (host side)."""

    def __init__(self, pages: int, page_size: int, batch: int, device: torch.device) -> None:
        self.page_size, self.free = page_size, list(range(pages))
        self.owned: list[list[int]] = [[] for _ in range(batch)]
        self.lens = [0] * batch
        self.device = device

    def extend(self, new: list[int]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Room for ``new[b]`` more tokens of every sequence: (block_table, kv_lens, q_starts). When there
        are too few free pages it raises and nothing changes, so a caller can release a sequence and
        try again."""
        need = [-(-(n + old) // self.page_size) - len(own) for n, old, own in zip(new, self.lens, self.owned)]
        if sum(need) > len(self.free):
            raise RuntimeError("the cache has no free page")
        starts = [0]
        for b, n in enumerate(new):
            self.lens[b] += n
            self.owned[b] += [self.free.pop() for _ in range(need[b])]
            starts.append(starts[-1] + n)
        width = max(1, max(len(p) for p in self.owned))
        table = [p + [0] * (width - len(p)) for p in self.owned]
        i32 = {"dtype": torch.int32, "device": self.device}
        return torch.tensor(table, **i32), torch.tensor(self.lens, **i32), torch.tensor(starts, **i32)

    def release(self, b: int) -> None:
        """Sequence b is done: its pages are free again."""
        self.free += self.owned[b]
        self.owned[b], self.lens[b] = [], 0


class Gpt2:
    """A GPT-2 decoder in fp32 over a paged cache of fp32, float16 or bfloat16."""

    def __init__(self, layers: int = 12, d: int = 768, heads: int = 12, vocab: int = 50257, max_pos: int = 1024, *,
                 cache_dtype: torch.dtype = torch.float32, precision: int = TF32, seed: int = 3, device: str = "cuda") -> None:
        self.layers, self.d, self.heads, self.vocab, self.max_pos = layers, d, heads, vocab, max_pos
        self.cache_dtype, self.precision, self.device = cache_dtype, precision, torch.device(device)
        self.lib = library()
        g = torch.Generator(device=device).manual_seed(seed)

        def normal(*shape: int, std: float = 0.02) -> torch.Tensor:
            return torch.randn(*shape, generator=g, device=device) * std

        # products read their weights as [out, in] rows, what the tensor cores take
        self.wte, self.wpe = normal(vocab, d), normal(max_pos, d, std=0.01)
        self.blocks = [
            {"ln1": (1 + normal(d), normal(d)), "qkv": (normal(3 * d, d), normal(3 * d)), "proj": (normal(d, d), normal(d)),
             "ln2": (1 + normal(d), normal(d)), "up": (normal(4 * d, d), normal(4 * d)), "down": (normal(d, 4 * d), normal(d))}
            for _ in range(layers)
        ]
        self.ln = (1 + normal(d), normal(d))

    def cache(self, pages: int, page_size: int) -> list[tuple[torch.Tensor, torch.Tensor]]:
        """(k, v) pages of every layer."""
        shape = (pages, page_size, self.heads, self.d // self.heads)
        return [tuple(torch.empty(shape, dtype=self.cache_dtype, device=self.device) for _ in range(2))  # type: ignore[misc]
                for _ in range(self.layers)]

    def _stream(self) -> int:
        return torch.cuda.current_stream(self.device).cuda_stream

    def _norm(self, x: torch.Tensor, ln: tuple[torch.Tensor, torch.Tensor]) -> torch.Tensor:
        x = x.contiguous()  # a product's rows may be padded
        y = torch.empty_like(x)
        check(self.lib.mgc_cuda_layer_norm(x.shape[0], x.shape[1], x.data_ptr(), ln[0].data_ptr(), ln[1].data_ptr(), 1e-5,
                                           y.data_ptr(), self._stream()), "mgc_cuda_layer_norm", self.lib)
        return y

    def _product(self, x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None, act: int = ACT_NONE,
                 res: torch.Tensor | None = None) -> torch.Tensor:
        m, k = x.shape
        n = w.shape[0]
        # rows of a multiple of 16 bytes, what TF32 takes: odd widths (the vocabulary's) get padded ones
        ldc = -(-n // 4) * 4
        y = torch.empty(m, ldc, device=x.device)
        precision = self.precision if n % 4 == 0 and k % 4 == 0 else FP32
        check(self.lib.mgc_cuda_gemm(m, n, k, 1, x.data_ptr(), max(x.stride(0), k), 1, 0, w.data_ptr(), 1, k, 0,
                                     y.data_ptr(), ldc, 0, 1.0,
                                     bias.data_ptr() if bias is not None else None, 1 if bias is not None else 0,
                                     res.data_ptr() if res is not None else None, res.stride(0) if res is not None else n, 0,
                                     1.0, act, 0.0, 0.0, precision, self._stream()), "mgc_cuda_gemm", self.lib)
        return y[:, :n]

    def step(self, ids: torch.Tensor, new: list[int], pages: Pages, cache: list[tuple[torch.Tensor, torch.Tensor]],
             status: torch.Tensor | None = None) -> torch.Tensor:
        """``ids`` [sum(new)]: the next ``new[b]`` tokens of every sequence. Caches them and returns the
        logits [batch, vocab] after each sequence's last token (of sequences with new tokens)."""
        before = list(pages.lens)
        if max(n + b for n, b in zip(new, before)) > self.max_pos:
            raise ValueError(f"a sequence passes {self.max_pos} positions")
        at = pages.extend(new)
        positions = torch.cat([torch.arange(b, b + n) for b, n in zip(before, new)]).to(self.device)
        tokens, d, heads = int(ids.shape[0]), self.d, self.heads
        x = self.wte[ids] + self.wpe[positions]
        max_q, max_kv = max(new), max(pages.lens)
        for block, (k_cache, v_cache) in zip(self.blocks, cache):
            qkv = self._product(self._norm(x, block["ln1"]), *block["qkv"]).view(tokens, 3 * heads, d // heads)
            q, k, v = qkv[:, :heads], qkv[:, heads : 2 * heads], qkv[:, 2 * heads :]
            # learned positions: nothing to rotate; q comes back in the cache's type
            same = self.cache_dtype == torch.float32
            turned = kv_append(k, v, k_cache, v_cache, *at, q=None if same else q, status=status)
            o = paged_attention(q if same else turned, k_cache, v_cache, *at, max_q=max_q, max_kv=max_kv, status=status)
            x = self._product(o.reshape(tokens, d).float(), *block["proj"], res=x)
            h = self._product(self._norm(x, block["ln2"]), *block["up"], act=ACT_GELU_TANH)
            x = self._product(h, *block["down"], res=x)
        last = torch.tensor([s for s, n in zip(at[2].tolist()[1:], new) if n], device=self.device) - 1
        return self._product(self._norm(x[last].contiguous(), self.ln), self.wte, None)

    def plain(self, ids: torch.Tensor) -> torch.Tensor:
        """Logits after the last token of one whole sequence, in plain float64 operations."""
        def norm(x: torch.Tensor, ln: tuple[torch.Tensor, torch.Tensor]) -> torch.Tensor:
            return torch.nn.functional.layer_norm(x, (self.d,), ln[0].double(), ln[1].double(), 1e-5)

        n, heads, dim = int(ids.shape[0]), self.heads, self.d // self.heads
        x = self.wte[ids].double() + self.wpe[:n].double()
        hidden = torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1)
        for b in self.blocks:
            w = {k: (m.double(), c.double()) for k, (m, c) in b.items()}
            qkv = (norm(x, b["ln1"]) @ w["qkv"][0].T + w["qkv"][1]).view(n, 3, heads, dim).permute(1, 2, 0, 3)
            s = (qkv[0] @ qkv[1].transpose(1, 2)) * dim**-0.5
            o = torch.softmax(s.masked_fill(hidden, float("-inf")), -1) @ qkv[2]
            x = x + o.transpose(0, 1).reshape(n, self.d) @ w["proj"][0].T + w["proj"][1]
            h = torch.nn.functional.gelu(norm(x, b["ln2"]) @ w["up"][0].T + w["up"][1], approximate="tanh")
            x = x + h @ w["down"][0].T + w["down"][1]
        return norm(x[-1:], self.ln) @ self.wte.double().T


def generate(model: Gpt2, prompts: list[list[int]], tokens: int, *, page_size: int = 16, chunk: int = 256) -> tuple[list[list[int]], list[float], torch.Tensor]:
    """Greedy continuation of every prompt by ``tokens`` tokens: (sequences, seconds of each step, the
    last logits). Prompts, of at least one token each, are cached in chunks of at most ``chunk`` tokens a
    sequence."""
    if not prompts or not all(prompts):
        raise ValueError("every prompt needs a token")
    batch, dev = len(prompts), model.device
    need = sum(-(-(len(p) + tokens) // page_size) for p in prompts)
    pages, cache = Pages(need, page_size, batch, dev), model.cache(need, page_size)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = [list(p) for p in prompts]
    logits = torch.empty(batch, model.vocab, device=dev)
    done = 0
    while done < max(len(p) for p in prompts):
        parts = [p[done : done + chunk] for p in prompts]
        ids = torch.tensor([i for part in parts for i in part], device=dev)
        got = model.step(ids, [len(part) for part in parts], pages, cache, status)
        logits[[b for b, part in enumerate(parts) if part]] = got
        done += chunk
    seconds = []
    for step in range(tokens):
        ids = logits.argmax(-1)
        for seq, i in zip(out, ids.tolist()):
            seq.append(i)
        if step + 1 == tokens:
            break
        start = time.perf_counter()
        logits = model.step(ids, [1] * batch, pages, cache, status)
        torch.cuda.synchronize(dev)
        seconds.append(time.perf_counter() - start)
    check_status(status)
    return out, seconds, logits


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=100, help="longest prompt; the others are shorter")
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--layers", type=int, default=12)
    ap.add_argument("--page-size", type=int, default=16)
    ap.add_argument("--cache", choices=["float32", "float16", "bfloat16"], default="float32")
    ap.add_argument("--check", action="store_true", help="compare the last logits with a plain computation")
    args = ap.parse_args(argv)
    model = Gpt2(layers=args.layers, cache_dtype=getattr(torch, args.cache))
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(model.vocab, (max(1, args.prompt - 7 * b),), generator=g).tolist() for b in range(args.batch)]
    out, seconds, logits = generate(model, prompts, args.tokens, page_size=args.page_size)
    if seconds:
        print(f"{args.batch} sequences, {args.tokens} tokens each: {1e3 * sorted(seconds)[len(seconds) // 2]:.3f} ms per step (median)")
    if args.check:
        for b, seq in enumerate(out):
            want = model.plain(torch.tensor(seq[:-1], device=model.device))
            err = float((logits[b].double() - want[0]).abs().max())
            print(f"sequence {b}: {len(seq)} tokens, max abs logit error {err:.3g}")
            if not err <= 2e-2:
                return 1
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
