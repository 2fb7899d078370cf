"""Batches for the paged-cache tests and the operators' definition in 64 bits (plain loops)."""

from __future__ import annotations

import math

import numpy as np
import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# unit roundoff of one rounding to the type (24, 11 and 8 significant bits)
ROUND = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


def caches(layout: str, pages: int, page: int, heads: int, dim: int, dtype: torch.dtype, device: str):
    """(k, v) [pages, page, heads, dim] in one of the layouts a server may keep."""
    if layout == "tokens":
        k, v = (torch.empty(pages, page, heads, dim, dtype=dtype, device=device) for _ in range(2))
    elif layout == "heads":  # [pages, heads, page, dim]
        k, v = (torch.empty(pages, heads, page, dim, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))
    elif layout == "joint":  # keys and values of a page side by side
        kv = torch.empty(pages, 2, page, heads, dim, dtype=dtype, device=device)
        k, v = kv[:, 0], kv[:, 1]
    elif layout == "odd":  # rows that start at odd elements: no wide access is aligned
        k, v = (torch.empty(pages, page, heads, dim + 3, dtype=dtype, device=device)[..., 1 : dim + 1] for _ in range(2))
    else:
        raise ValueError(layout)
    return k, v


class PagedBatch:
    """Sequences with `qs` new tokens and `ks` cached positions, their pages drawn in a random order.
    Whatever no sequence owns (spare pages, rows past the last position) holds NaN."""

    def __init__(self, qs, ks, *, heads, kv_heads, dim, page, dtype, layout="tokens", seed=0, gain=1.75, device="cuda",
                 packed=True):
        g = torch.Generator(device=device).manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.qs, self.ks, self.page, self.group = list(qs), list(ks), page, heads // kv_heads
        self.dtype, self.name, dt = dtype, dtype, DTYPES[dtype]
        need = [-(-k // page) for k in ks]
        pages = sum(need) + 2
        order = rng.permutation(pages)
        table = np.full((len(ks), max([*need, 1]) + 1), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at : at + n]
            at += n
        self.table = table
        self.k, self.v = caches(layout, pages, page, kv_heads, dim, dt, device)
        self.k.fill_(math.nan)
        self.v.fill_(math.nan)
        self.slots = []
        for b, n in enumerate(ks):
            j = np.arange(n)
            slot = torch.from_numpy(table[b, j // page].astype(np.int64)).to(device), torch.from_numpy(j % page).to(device)
            self.slots.append(slot)
            self.k[slot] = torch.randn(n, kv_heads, dim, generator=g, device=device).to(dt)
            self.v[slot] = torch.randn(n, kv_heads, dim, generator=g, device=device).to(dt)
        tokens = sum(qs)
        qkv = torch.randn(max(tokens, 1), heads + 2 * kv_heads, dim, generator=g, device=device)[:tokens] * gain
        self.q = qkv.to(dt)[:, :heads] if packed else qkv[:, :heads].to(dt).contiguous()
        i32 = torch.int32
        self.block_table = torch.from_numpy(table).to(device)
        self.kv_lens = torch.tensor(ks, dtype=i32, device=device)
        self.q_starts = torch.tensor(np.concatenate([[0], np.cumsum(qs)]), dtype=i32, device=device)

    @property
    def operands(self):
        return self.k, self.v, self.block_table, self.kv_lens, self.q_starts

    def rows(self, b):
        start = sum(self.qs[:b])
        return slice(start, start + self.qs[b])


def attention_exact(x: PagedBatch, scale: float, causal: bool = True, window: int = 0):
    """(output, bound on the error): float64 by the definition, one sequence and head at a time.

    The bound follows a computation that takes scores in fp32 products (or exact splits of them),
    the weights e^(s - m) rounded once to the pages' type, and one rounding at the end:
    a score is off by at most ds = (dim + 8) 2^-21 sum_c |q_c k_c| scale (2^-21 rather than 2^-24
    because the tensor cores truncate and keep 22 bits of split fp32 operands), which scales its
    weight by e^ds; sums over n keys add sqrt(n) 2^-21; so
      |o' - o| <= (2 ds + r + sqrt(n) 2^-21) sum_j w_j |v_j| + r |o|, r the type's roundoff."""
    out = torch.zeros(x.q.shape, dtype=torch.float64, device=x.q.device)
    bound = torch.zeros_like(out)
    r, u = ROUND[x.name], 2.0**-21
    for b, (nq, nk) in enumerate(zip(x.qs, x.ks)):
        if not nq or not nk:
            continue
        k, v = x.k[x.slots[b]].double(), x.v[x.slots[b]].double()
        q = x.q[x.rows(b)].double()
        pos = torch.arange(nk - nq, nk, device=q.device)[:, None]
        j = torch.arange(nk, device=q.device)[None]
        seen = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
        if causal:
            seen &= j <= pos
        if window:
            seen &= j > pos - window
        some = seen.any(1)
        for h in range(q.shape[1]):
            kh, vh = k[:, h // x.group], v[:, h // x.group]
            s = (q[:, h] @ kh.T * scale).masked_fill(~seen, -math.inf)
            w = torch.where(some[:, None], torch.softmax(s, -1), torch.zeros_like(s)).nan_to_num(0.0)
            out[x.rows(b), h] = w @ vh
            size = (q[:, h].abs() @ kh.abs().T * scale).masked_fill(~seen, 0.0).amax(1, keepdim=True)
            ds = (q.shape[2] + 8) * u * size
            bound[x.rows(b), h] = (2 * ds + r + math.sqrt(nk) * u) * (w @ vh.abs()) + r * (w @ vh).abs() + 1e-30
    return out, bound


def rotate_exact(x: torch.Tensor, pos, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """[n, heads, dim] rotated by rows `pos` of the tables, in float64."""
    y = x.double().clone()
    half = cos.shape[1]
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cos[pos, i].double()[:, None], sin[pos, i].double()[:, None]
        y[..., a] = x[..., a].double() * c - x[..., b].double() * s
        y[..., b] = x[..., b].double() * c + x[..., a].double() * s
    return y


def angles(positions: int, rot: int, device: str = "cuda"):
    half = rot // 2
    inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=device) / max(half, 1))
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return a.cos().float(), a.sin().float()
