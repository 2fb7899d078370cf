"""The attention over a paged cache in 64 bits for every border of its definition (keys whose page is
missing, lengths past the block table, infinite and NaN values), with the error that a computation in
32 bits is allowed, derived term by term; and the workspace that a call would take."""

from __future__ import annotations

import math
import struct

import torch

from mgc_cuda.native import library
from paged_cases import ROUND, PagedBatch


def reference(x: PagedBatch, scale: float, causal: bool = True, window: int = 0, present=None, lens=None):
    """(output, allowed error). `present[b]`: which of the sequence's ks[b] positions can be read (all);
    `lens[b]`: its length when that is more than the ks[b] positions that its pages hold.

    Errors, N = |q o k|_2 (the root of the sum of squared products) of a score:
    * fp32, split products: h + l with l truncated to 11 bits leaves at most 2^-21 of each operand, l l'
      (2^-22) is dropped; taken as independent of mean 0, their deviation is below 0.85 2^-21 |q_c k_c| a
      channel, six deviations of the sum 6 * 0.85 * 2^-21 N. Chains of four steps truncate 2^-23 of their
      sum each, independent between chains: below 12 2^-23 N. The same for weights times values.
    * 16-bit types: products are exact, a chain of dim / 16 steps truncates 2^-22 of its sum each; the
      weight is rounded to the type (r), and what f16 cannot hold (steps of 2^-24) is at most 2^-36 of
      the largest weight.
    * every weight: the exponent's rounding, 2^-24 of its size and of the score's, and 2^-22 of exp2.
    * sums: a truncation 2^-23 per step of four to eight within a tile, a rounding 2^-24 per tile of 32 keys."""
    dev, dim = x.q.device, x.q.shape[2]
    out = torch.zeros(x.q.shape, dtype=torch.float64, device=dev)
    bound = torch.full_like(out, 1e-30)
    f32, r = x.name == "f32", ROUND[x.name]
    for b, (nq, nk) in enumerate(zip(x.qs, x.ks)):
        if not nq or not nk:
            continue
        k, v = x.k[x.slots[b]].double(), x.v[x.slots[b]].double()
        q = x.q[x.rows(b)].double()
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
            kh, vh, qh = k[:, h // x.group], v[:, h // x.group], q[:, h]
            s = (torch.where(seen[:, :, None], qh[:, None] * kh[None], 0.0).sum(-1) if not torch.isfinite(kh).all()
                 else qh @ kh.T)
            s = torch.where(seen, s * scale, -math.inf)
            w = torch.where(some, torch.softmax(s, -1), 0.0).nan_to_num(0.0)
            if torch.isfinite(vh).all():
                o = w @ vh
            else:
                o = torch.where(seen[:, :, None], w[:, :, None] * vh[None], 0.0).sum(1)
            vf = vh.nan_to_num(0.0, 0.0, 0.0).abs()
            big = (qh.square() @ kh.nan_to_num(0.0, 0.0, 0.0).square().T).sqrt() * scale
            top = s.amax(1, keepdim=True).clamp(min=-1e30)
            sf = torch.where(seen, s, 0.0)
            lin = 2.0**-24 * ((top - sf).clamp(min=0.0) + 2 * sf.abs()) + 2.0**-22
            if f32:
                rss = big * (6 * 0.85 * 2.0**-21 + 12 * 2.0**-23)
                value = 6 * 0.85 * 2.0**-21 * (w.square() @ vf.square()).sqrt()
            else:
                rss = torch.zeros_like(big)
                lin = lin + r + (dim / 16 + 2) * 2.0**-22 * (qh.abs() @ kh.nan_to_num(0.0, 0.0, 0.0).abs().T) * scale
                value = nk * 2.0**-36 * w.amax(1, keepdim=True) * vf.amax(0)[None]
            of = o.nan_to_num(0.0, 0.0, 0.0).abs()
            wl, wr = w * lin, (w * rss).square()
            out[x.rows(b), h] = o
            bound[x.rows(b), h] += (
                wl @ vf + wl.sum(1, keepdim=True) * of + 2 * (wr @ vf.square() + wr.sum(1, keepdim=True) * of.square()).sqrt()
                + value + 8 * 2.0**-23 * (w @ vf) + (3 * math.sqrt(nk / 32) + 8) * 2.0**-24 * (w @ vf) + r * of
                + (2.0**-25 if x.name == "f16" else 0.0))
    return out, bound


def compare(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor) -> None:
    """NaN and infinities in the same places, everything else within the bound."""
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), f"{int((got.isnan() != want.isnan()).sum())} NaN in the wrong places"
    inf = want.isinf()
    assert torch.equal(got.isinf(), inf) and torch.equal(got[inf], want[inf]), "infinities in the wrong places"
    off = torch.where(torch.isfinite(want), (got - want).abs(), torch.zeros_like(want))
    worst = float((off / bound).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the bound, max abs error {float(off.max()):.3g}"


def workspace(x: PagedBatch, *, max_q: int | None = None, max_kv: int | None = None, causal: bool = True, window: int = 0) -> int:
    """Bytes of workspace of a call: 0 where clusters share a row's keys, more where pieces are added by a
    second kernel."""
    k, q = x.k, x.q
    dtype = {"f32": 0, "f16": 7, "bf16": 8}[x.name]
    fields = [k.data_ptr(), x.v.data_ptr(), k.shape[0], k.stride(0), k.stride(1), k.stride(2), dtype, k.shape[2], k.shape[3],
              k.shape[1], x.block_table.data_ptr(), x.block_table.stride(0), x.block_table.shape[1], x.kv_lens.data_ptr(),
              x.q_starts.data_ptr(), len(x.qs), q.shape[0], 0, q.data_ptr(), q.stride(0), q.stride(1), q.shape[1],
              q.data_ptr(), q.stride(0), q.stride(1), max(x.qs) if max_q is None else max_q,
              max(x.ks) if max_kv is None else max_kv]
    data = struct.pack(f"={len(fields)}q", *fields) + struct.pack("=d", q.shape[2] ** -0.5) + struct.pack("=4q", causal, window, 0, 0)
    return library().mgc_cuda_paged_attention_workspace(data)
