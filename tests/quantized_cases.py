"""Batches over a quantised paged cache for the tests, the append's steps in plain torch and the attention's
definition in 64 bits with the error that a kernel is allowed."""

from __future__ import annotations

import copy
import math
import struct

import numpy as np
import torch

from paged_cases import DTYPES, ROUND

from mgc_cuda.native import library
from mgc_cuda.paged import QuantizedPages, quantized_pages


def quantise(x: torch.Tensor, bits: int, group: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes [..., D * bits / 8], scales [..., groups, 2]) of fp32 x [..., D], the steps of the definition."""
    top = (1 << bits) - 1
    g = x.unflatten(-1, (-1, group))
    held = g.clamp(-65504.0, 65504.0)
    offset = held.amin(-1, keepdim=True).half()
    scale = ((held.amax(-1, keepdim=True) - offset.float()) * (1.0 / top)).half()
    step = scale.float()
    code = torch.where(step > 0, (g - offset.float()) / step, torch.zeros_like(g)).round().clamp(0, top)
    bad = ~torch.isfinite(g).all(-1, keepdim=True)
    nan = torch.full_like(scale, math.nan)
    code = torch.where(bad, torch.zeros_like(code), code).to(torch.uint8).flatten(-2)
    if bits == 4:
        code = code[..., 0::2] | code[..., 1::2] << 4
    return code, torch.cat((torch.where(bad, nan, scale), torch.where(bad, nan, offset)), -1)


def whole_codes(codes: torch.Tensor, bits: int) -> torch.Tensor:
    return codes if bits == 8 else torch.stack((codes & 15, codes >> 4), -1).flatten(-2)


def values(codes: torch.Tensor, scales: torch.Tensor, bits: int, dtype=torch.float64) -> torch.Tensor:
    x = whole_codes(codes, bits).to(dtype).unflatten(-1, (scales.shape[-2], -1))
    return (x * scales[..., :1].to(dtype) + scales[..., 1:].to(dtype)).flatten(-2)


def pages_like(layout: str, pages: int, page: int, heads: int, dim: int, bits: int, group: int, device: str):
    """(k, v) quantised pages in one of the layouts a server may keep."""
    row = dim * bits // 8
    if layout == "heads":
        return [quantized_pages(pages, page, heads, dim, bits=bits, group=group, device=device) for _ in range(2)]
    if layout == "tokens":
        pad = -(-row // 16) * 16
        return [QuantizedPages(torch.zeros(pages, page, heads, pad, dtype=torch.uint8, device=device)[..., :row],
                               torch.zeros(pages, page, heads, dim // group, 2, dtype=torch.float16, device=device), bits)
                for _ in range(2)]
    if layout == "joint":  # keys and values of a page side by side, rows with room to spare, scales three pairs apart
        pad = -(-row // 16) * 16 + 16
        codes = torch.zeros(pages, 2, page, heads, pad, dtype=torch.uint8, device=device)
        scales = torch.zeros(pages, 2, page, heads, dim // group + 3, 2, dtype=torch.float16, device=device)
        return [QuantizedPages(codes[:, i, ..., :row], scales[:, i, ..., 1 : 1 + dim // group, :], bits) for i in range(2)]
    raise ValueError(layout)


class QuantizedBatch:
    """Sequences with `qs` new tokens and `ks` cached positions over pages of `bits`, drawn in a random
    order. What no sequence owns (spare pages, rows past the last position) has pairs of NaN."""

    def __init__(self, qs, ks, *, heads, kv_heads, dim, page, dtype, bits, group=None, layout="heads", seed=0, gain=1.75,
                 device="cuda", packed=True, spread=1.0):
        g = torch.Generator(device=device).manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.qs, self.ks, self.page, self.share = list(qs), list(ks), page, heads // kv_heads
        self.dtype, self.name, self.bits, dt = dtype, dtype, bits, DTYPES[dtype]
        self.group = group or (64 if dim % 64 == 0 else dim)
        need = [-(-k // page) for k in ks]
        pages = sum(need) + 2
        order = rng.permutation(pages)
        table = np.full((len(ks), max([*need, 1]) + 1), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at : at + n]
            at += n
        self.table = table
        self.k, self.v = pages_like(layout, pages, page, kv_heads, dim, bits, self.group, device)
        for c in (self.k, self.v):
            c.codes.fill_(0xAB)
            c.scales.fill_(math.nan)
        self.slots = []
        mean = torch.randn(kv_heads, dim, generator=g, device=device) * 0.5
        for b, n in enumerate(ks):
            j = np.arange(n)
            slot = torch.from_numpy(table[b, j // page].astype(np.int64)).to(device), torch.from_numpy(j % page).to(device)
            self.slots.append(slot)
            # tokens of different sizes, so that groups have different scales
            size = torch.exp(torch.randn(2, n, 1, 1, generator=g, device=device) * (spread - 1.0))
            for c, m, s in ((self.k, mean, size[0].clamp(max=1.0)), (self.v, 0.0, size[1])):
                c.codes[slot], c.scales[slot] = quantise((torch.randn(n, kv_heads, dim, generator=g, device=device) + m) * s, bits, self.group)
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


def attention(x: QuantizedBatch, scale: float, causal: bool = True, window: int = 0, present=None, lens=None):
    """(output, allowed error). `present[b]`: which of the sequence's positions can be read (all); `lens[b]`:
    its length when that is more than the positions that its pages hold.

    With a = scale_j |code - c| + |offset_j + c scale_j|, c the middle of the codes, the size of what a
    channel's value may be computed from, r the type's roundoff (half a step), and N the root of the sum of
    squared products q_c k_c of a score:
    * scores: codes times 16-bit queries are exact and sums lose at most 2^-22 a step of 16 channels, so
      (dim / 16 + 8) 2^-22 sum |q_c| a_c. fp32 queries are split in two halves, 2^-24 of the row's largest
      left. A kernel may instead take the values rounded to the type: r a value, independent and of deviation
      0.58 r at most, six deviations 3.5 r N (fp32: the split TF32 products' 6 * 0.85 * 2^-21 N + 12 2^-23 N).
    * weights: rounded to 16 bits (r), the exponent's rounding 2^-24 of its size and the score's, 2^-22 of exp2,
      and steps of 2^-36 of the largest weight for those that half cannot hold; fp32: split in two.
    * values: rounded to the type, six deviations 3.5 r of the weighted root of squares, or
      6 * 0.85 * 2^-21 in fp32; sums 2^-22 a step of 16 keys within a tile, 2^-23 a tile of 128 keys.
    * the output: r."""
    dev, dim, dtype = x.q.device, x.q.shape[2], torch.float64
    out = torch.zeros(x.q.shape, dtype=dtype, device=dev)
    bound = torch.full_like(out, 1e-30)
    f32, r, mid = x.name == "f32", ROUND[x.name], 1 << (x.bits - 1)
    rs = 6 * 0.85 * 2.0**-21 + 12 * 2.0**-23 if f32 else 3.5 * r
    for b, (nq, nk) in enumerate(zip(x.qs, x.ks)):
        if not nq or not nk:
            continue
        q = x.q[x.rows(b)].double()
        k, v = (values(c.codes[x.slots[b]], c.scales[x.slots[b]], x.bits) for c in (x.k, x.v))
        size = []
        for c in (x.k, x.v):
            sc = c.scales[x.slots[b]].double().nan_to_num(0.0, 0.0, 0.0)
            code = whole_codes(c.codes[x.slots[b]], x.bits).double().unflatten(-1, (sc.shape[-2], -1))
            size.append((sc[..., :1].abs() * (code - mid).abs() + (sc[..., 1:] + mid * sc[..., :1]).abs()).flatten(-2))
        n = nk if lens is None else lens[b]
        pos = torch.arange(n - nq, n, device=dev)[:, None]
        j = torch.arange(nk, device=dev)[None]
        seen = torch.ones(nq, nk, dtype=torch.bool, device=dev)
        if present is not None:
            seen &= present[b][None]
        if causal:
            seen &= j <= pos
        if window:
            seen &= j > pos - window
        some = seen.any(1, keepdim=True)
        for h in range(q.shape[1]):
            kh, vh, qh = k[:, h // x.share], v[:, h // x.share], q[:, h]
            kf, vf = kh.nan_to_num(0.0), vh.nan_to_num(0.0)
            s = qh @ kf.T
            s = torch.where(torch.isnan(kh).any(1)[None], math.nan, s)
            s = torch.where(seen, s * scale, -math.inf)
            w = torch.where(some, torch.softmax(s, -1), 0.0)
            w = torch.where(some & ~seen, torch.where(w.isnan().any(1, keepdim=True), math.nan, w), w)
            o = torch.where(seen, w, 0.0) @ vf
            lost = torch.isnan(vh)  # a channel's NaN reaches the rows that see its key
            if lost.any():
                o = torch.where((seen.double() @ lost.double()) > 0, math.nan, o)
            o = torch.where(torch.isnan(w).any(1, keepdim=True), math.nan, o)
            w = w.nan_to_num(0.0)
            ks_, vs_ = size[0][:, h // x.share], size[1][:, h // x.share]
            big = (qh.square() @ kf.square().T).sqrt() * scale
            sf = torch.where(seen, s, 0.0).nan_to_num(0.0)
            top = torch.where(seen, s, -1e30).nan_to_num(0.0).amax(1, keepdim=True)
            lin = 2.0**-24 * ((top - sf).clamp(min=0.0) + 2 * sf.abs()) + 2.0**-22 + (0.0 if f32 else r)
            lin = lin + ((dim / 16 + 8) * 2.0**-22 * (qh.abs() @ ks_.T) + 2.0**-24 * qh.abs().amax(1, keepdim=True) * ks_.sum(1)[None]) * scale
            wl, wr = w * lin, (w * big * rs).square()
            of = o.nan_to_num(0.0).abs()
            out[x.rows(b), h] = o
            bound[x.rows(b), h] += (
                wl @ vs_ + wl.sum(1, keepdim=True) * of + 2 * (wr @ vs_.square() + wr.sum(1, keepdim=True) * of.square()).sqrt()
                + rs * (w.square() @ vs_.square()).sqrt() + nk * 2.0**-36 * w.amax(1, keepdim=True) * vs_.amax(0)[None]
                + (16 * 2.0**-22 + (3 * math.sqrt(nk / 128) + 8) * 2.0**-23) * (w @ vs_) + r * of + (2.0**-25 if x.name == "f16" else 0.0))
    return out, bound


def compare(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor) -> None:
    """NaN in the same places, everything else within the bound."""
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), f"{int((got.isnan() != want.isnan()).sum())} NaN in the wrong places"
    off = torch.where(torch.isnan(want), torch.zeros_like(want), (got - want).abs())
    worst = float((off / bound).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the bound, max abs error {float(off.max()):.3g}"


def normed(x: torch.Tensor, weight: torch.Tensor | None, eps: float) -> torch.Tensor:
    """fp32 heads normalised by the definition's steps."""
    if weight is None:
        return x
    return x * (x.double().square().mean(-1, keepdim=True) + eps).pow(-0.5).float() * weight


def rotated(x: torch.Tensor, cos, sin, pos, interleaved: bool) -> torch.Tensor:
    """fp32 [n, heads, dim] rotated by rows `pos`, a rounding a step."""
    if cos is None:
        return x
    y, half = x.clone(), cos.shape[1]
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cos[pos][:, None], sin[pos][:, None]
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def workspace(x: QuantizedBatch, max_q: int, max_kv: int, window: int = 0) -> int:
    """Bytes of workspace of a call: those of plain pages are in it where values are expanded first."""
    k, s, q = x.k.codes, x.k.scales, x.q
    fields = [k.data_ptr(), x.v.codes.data_ptr(), k.shape[0], k.stride(0), k.stride(1), k.stride(2), {"f32": 0, "f16": 7, "bf16": 8}[x.name],
              k.shape[2], q.shape[2], k.shape[1], x.block_table.data_ptr(), x.block_table.stride(0), x.block_table.shape[1],
              x.kv_lens.data_ptr(), x.q_starts.data_ptr(), len(x.qs), q.shape[0], 0, q.data_ptr(), q.stride(0), q.stride(1), q.shape[1],
              q.data_ptr(), q.stride(0), q.stride(1), max_q, max_kv]
    data = struct.pack(f"={len(fields)}q", *fields) + struct.pack("=d", 0.125) + struct.pack("=4q", 1, window, 0, 0)
    data += struct.pack("=7q", x.bits, q.shape[2] // s.shape[3], s.data_ptr(), x.v.scales.data_ptr(), s.stride(0) // 2, s.stride(1) // 2,
                        s.stride(2) // 2)
    return library().mgc_cuda_paged_attention_quantized_workspace(data)


def widened(x: QuantizedBatch) -> QuantizedBatch:
    """The same batch with a block table of so many pages (none of them there) that a call without max_kv counts on long
    contexts: with many query rows values are then expanded to plain pages first."""
    width = max(1, (64 if x.q.shape[2] <= 64 else 128 if x.q.shape[2] <= 128 else 256) // 64)
    positions = 6_000_000 // (len(x.qs) * x.k.codes.shape[2] * width)
    y = copy.copy(x)
    more = -(-positions // x.page)
    y.block_table = torch.cat((x.block_table, torch.full((len(x.qs), more), -1, dtype=torch.int32, device=x.block_table.device)), 1)
    return y
