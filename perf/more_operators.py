"""Benchmark cases of the quantised paged cache: new keys and values normalised for each head, rotated and
written (as they are or in 4 or 8 bits), read back, and attended to.

A batch is described as for the other paged-cache operators: ``block_table`` [B, P] (the pages of each
sequence, in order), ``kv_lens`` [B] (cached positions, the new tokens included) and ``q_starts`` [B + 1]
(where each sequence's new tokens begin in the packed token axis). Token t of sequence b sits at position
``kv_lens[b] - (q_starts[b + 1] - t)``.

A quantised cache is (codes, scales, bits): codes uint8 [pages, page_size, kv_heads, D * bits / 8], the lower
nibble first, and scales float16 [pages, page_size, kv_heads, groups, 2]. The D / groups channels of a group
stand for ``scale * code + offset`` with the group's two numbers; writing takes the group's least value as
the offset and the range / (2^bits - 1) as the scale, each rounded to float16, and the nearest code.

``run`` computes one pass, in plain torch operations (``own`` false) or with the framework's kernels
(``own`` true); ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
# what quantised values are read back as: the type of the sources, half for fp32 ones
READ = {"f32": "f16", "f16": "f16", "bf16": "bf16"}
EPS = 1e-6
MAX_POSITIONS = 1 << 17


def listed() -> list[dict]:
    """Two appends to plain pages, three to quantised ones (the new tokens read back after), two reads and
    five attentions; `q` and `kv` are the longest sequence's new tokens and positions, `ragged` how far the
    shortest one falls below it, `group` the channels that share a scale."""
    return [
        # a decoding step of 64 sequences of a decoder that normalises its queries and keys, plain pages
        dict(name="norm_steps_bf16", op="append", dtype="bf16", src="bf16", bits=0, group=0, batch=64, q=1, kv=4096,
             ragged=0.9, heads=32, kv_heads=8, dim=128, page=16, norm=True, rot=128, pairs="half"),
        # prompts whose projections are fp32, part of each head rotated by neighbours, pages of 24
        dict(name="norm_prompts_f16", op="append", dtype="f16", src="f32", bits=0, group=0, batch=7, q=1613, kv=2500,
             ragged=1.0, heads=20, kv_heads=4, dim=80, page=24, norm=True, rot=32, pairs="neighbour"),
        # one new token of GPT-2 small (12 heads of 64, fp32, learned positions, no norm) into 8 bits
        dict(name="write_one_q8", op="append", dtype="f32", src="f32", bits=8, group=64, batch=1, q=1, kv=128,
             ragged=0.0, heads=12, kv_heads=12, dim=64, page=16, norm=False, rot=0, pairs="half"),
        # a decoding step of 64 sequences, normalised, rotated and written in 4 bits
        dict(name="write_steps_q4", op="append", dtype="bf16", src="bf16", bits=4, group=64, batch=64, q=1, kv=4096,
             ragged=0.9, heads=32, kv_heads=8, dim=128, page=16, norm=True, rot=128, pairs="half"),
        # prompts of a few thousand tokens each, in 4 bits
        dict(name="write_prompts_q4", op="append", dtype="bf16", src="bf16", bits=4, group=64, batch=6, q=4001, kv=4001,
             ragged=0.5, heads=32, kv_heads=8, dim=128, page=64, norm=True, rot=128, pairs="half"),
        # the caches of GPT-2 small at its longest context, read back
        dict(name="read_batch_q8", op="read", dtype="f16", bits=8, group=64, batch=16, q=1024, kv=1024, ragged=0.7,
             kv_heads=12, dim=64, page=16),
        # one very long context
        dict(name="read_long_q4", op="read", dtype="bf16", bits=4, group=128, batch=1, q=131071, kv=131071, ragged=0.0,
             kv_heads=8, dim=128, page=64),
        # decoding with GPT-2 small, one sequence
        dict(name="decode_one_q8", op="attend", dtype="f32", bits=8, group=64, batch=1, q=1, kv=128, ragged=0.0,
             heads=12, kv_heads=12, dim=64, page=16, causal=True, window=0),
        # a serving batch with grouped heads and mixed contexts
        dict(name="decode_batch_q4", op="attend", dtype="bf16", bits=4, group=64, batch=64, q=1, kv=8192, ragged=0.8,
             heads=32, kv_heads=8, dim=128, page=16, causal=True, window=0),
        # one sequence with a very long context
        dict(name="decode_long_q4", op="attend", dtype="f16", bits=4, group=128, batch=1, q=1, kv=131071, ragged=0.0,
             heads=32, kv_heads=8, dim=128, page=64, causal=True, window=0),
        # five proposed tokens for each sequence, one shared key head, pages that end inside a tile
        dict(name="verify_q8", op="attend", dtype="f16", bits=8, group=96, batch=8, q=5, kv=2047, ragged=0.5,
             heads=16, kv_heads=1, dim=96, page=24, causal=True, window=0),
        # a chunk of a long prompt over what is cached already
        dict(name="chunk_q4", op="attend", dtype="bf16", bits=4, group=64, batch=1, q=2048, kv=16384, ragged=0.0,
             heads=32, kv_heads=8, dim=128, page=64, causal=True, window=0),
    ]


def draw(rng) -> dict:
    """A case of the same ranges: every length from one token to the longest, odd ones among them."""

    def spread(lo: int, hi: int) -> int:
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))

    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    share = rng.choice([1, 1, 3, 4, 8]) if kv_heads < 12 else 1
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
    bits = rng.choice([4, 4, 8])
    group = rng.choice([g for g in (64, 128, dim) if dim % g == 0])
    case = dict(dtype=dtype, bits=bits, group=group, ragged=rng.choice([0.0, 0.3, 0.7, 1.0]), kv_heads=kv_heads, dim=dim,
                page=rng.choice([8, 16, 16, 24, 32, 64, 128]))
    kind = rng.choice(["norm", "write", "write", "read", "decode", "decode", "chunk", "prompt", "verify"])
    if kind in ("norm", "write"):
        batch = spread(1, 64)
        q = spread(1, max(1, min(4001, 16000 // batch)))
        plain = kind == "norm"
        return dict(case, op="append", src=rng.choice([dtype, "f32"]) if plain else dtype, bits=0 if plain else bits,
                    group=0 if plain else group, batch=batch, q=q, kv=q + spread(1, max(2, 64000 // batch)) - 1,
                    heads=kv_heads * share, norm=plain or rng.random() < 0.6, rot=rng.choice([0, dim, dim, dim // 4 * 2]),
                    pairs=rng.choice(["half", "neighbour"]))
    if kind == "read":
        batch = spread(1, 64)
        kv = spread(1, 131071 // batch)
        return dict(case, op="read", dtype=READ[dtype], batch=batch, q=rng.choice([kv, kv, spread(1, kv)]), kv=kv)
    if kind == "decode":
        batch, q = spread(1, 64), 1
        kv = spread(1, min(131071, (64 * 8192) // batch))
    elif kind == "verify":
        batch, q = spread(1, 16), rng.randint(2, 16)
        kv = max(q, spread(16, 8192))
    elif kind == "chunk":
        batch = spread(1, 9)
        q = spread(2, max(2, 2048 // batch))
        kv = q + spread(1, min(14000, 32768 // batch))
    else:
        batch = spread(1, 16)
        q = kv = spread(2, max(2, min(2048, 8192 // batch)))
    window = rng.choice([0, 0, 0, spread(16, 4096)])
    causal = rng.random() < 0.8
    case = dict(case, op="attend", batch=batch, q=q, kv=kv, heads=kv_heads * share, causal=causal, window=window if causal else 0)
    # no dearer than the largest listed cases, in pairs of a query and a key and in cached values
    size = max(case["heads"] * dim * batch * q * kv / (32 * 128 * 2048 * 15000), kv_heads * dim * batch * kv / (8 * 128 * 64 * 5000))
    if size > 1:
        case["kv"] = max(1, int(kv / size))
        case["q"] = min(q, case["kv"])
    return case


def lengths(case: dict) -> tuple[list[int], list[int]]:
    """(new tokens, cached positions) of every sequence: the first has the longest, the others are
    spread below it; with `ragged` 1 some have no new token."""
    q, kv, ragged = case["q"], case["kv"], case["ragged"]
    below = [ragged * ((b * 0.6180339887) % 1.0) for b in range(case["batch"])]
    other = below if q == kv else [ragged * ((b * 0.7548776662) % 1.0) for b in range(case["batch"])]
    qs = [0 if ragged == 1.0 and b % 8 == 5 else 1 if q == 1 else q - int(f * q) for b, f in enumerate(below)]
    return qs, [max(n, kv - int(f * kv)) for n, f in zip(qs, other)]


def _row_bytes(case: dict) -> int:
    """Of a head's codes in the cache, rows beginning at multiples of 16 bytes."""
    return -(-(case["dim"] * case["bits"] // 8) // 16) * 16


def prepare(case: dict, seed: int) -> dict:
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 31))
    qs, ks = lengths(case)
    tokens = sum(qs)
    page, dim, kv_heads, bits = case["page"], case["dim"], case["kv_heads"], case["bits"]
    need = [-(-k // page) for k in ks]
    pages = sum(need) + 3
    order = host.permutation(pages)
    table = np.zeros((case["batch"], max(max(need), 1)), np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    s = dict(
        case=case, q_max=case["q"], kv_max=max(ks), tokens=tokens,
        block_table=torch.from_numpy(table).to(dev),
        kv_lens=torch.tensor(ks, dtype=torch.int32, device=dev),
        q_starts=torch.tensor(np.concatenate([[0], np.cumsum(qs)]), dtype=torch.int32, device=dev),
    )
    # keys have channels with an offset of their own, as trained models' keys do
    offset = normal(kv_heads, dim) * 0.5
    for name, mean in (("k_cache", offset), ("v_cache", 0.0)):
        if not bits:
            s[name] = (normal(pages, page, kv_heads, dim) + mean).to(TYPES[case["dtype"]])
            continue
        # a page holds one head's rows side by side, so that a head's tokens are contiguous
        codes = torch.zeros(pages, kv_heads, page, _row_bytes(case), dtype=torch.uint8, device=dev)
        codes = codes.transpose(1, 2)[..., : dim * bits // 8]
        scales = torch.zeros(pages, kv_heads, page, dim // case["group"], 2, dtype=torch.float16, device=dev).transpose(1, 2)
        for first in range(0, pages, max(1, (1 << 26) // (page * kv_heads * dim))):  # some pages at a time
            part = slice(first, first + max(1, (1 << 26) // (page * kv_heads * dim)))
            codes[part], scales[part] = _quantise(normal(codes[part].shape[0], page, kv_heads, dim) + mean, bits, case["group"])
        s[name] = (codes, scales, bits)
    if case["op"] == "append":
        # q, k and v as the fused projection leaves them: one row of all heads for each token
        heads = case["heads"]
        qkv = normal(max(tokens, 1), heads + 2 * kv_heads, dim)[:tokens]
        qkv[:, heads : heads + kv_heads] += offset
        qkv = qkv.to(TYPES[case["src"]])
        s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads : heads + kv_heads], qkv[:, heads + kv_heads :]
        s["q_norm"], s["k_norm"] = (1 + 0.2 * normal(dim), 1 + 0.2 * normal(dim)) if case["norm"] else (None, None)
        s["cos"] = s["sin"] = None
        if case["rot"]:
            half = case["rot"] // 2
            inv = 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
            angle = torch.arange(MAX_POSITIONS, device=dev, dtype=torch.float64)[:, None] * inv
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    elif case["op"] == "attend":
        # score rows have a spread of about 2, between flat and one-hot
        s["q"] = (normal(tokens, case["heads"], dim) * 1.75).to(TYPES[case["dtype"]])
        s["scale"] = 1.0 / math.sqrt(dim)
    return s


def run(s: dict):
    op = s["case"]["op"]
    if own:
        return _append_own(s) if op == "append" else _read_own(s, TYPES[s["case"]["dtype"]]) if op == "read" else _attend_own(s)
    return _append_plain(s) if op == "append" else _read_plain(s, TYPES[s["case"]["dtype"]]) if op == "read" else _attend_plain(s)


# ---- the framework's operators -------------------------------------------------------------------
def _paged():
    try:
        from mgc_cuda import paged
    except ImportError:
        sys.path.insert(0, str(Path.cwd() / "ml-graph-compiler_b200"))
        from mgc_cuda import paged
    return paged


def _append_own(s: dict) -> dict:
    paged = sys.modules.get("mgc_cuda.paged") or _paged()
    case = s["case"]
    q = paged.kv_append(
        s["k"], s["v"], s["k_cache"], s["v_cache"], s["block_table"], s["kv_lens"], s["q_starts"],
        q=s["q"], cos=s["cos"], sin=s["sin"], interleaved=case["pairs"] == "neighbour",
        q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
    )
    if not case["bits"]:
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return {"q": q, **_read_own(s, TYPES[READ[case["src"]]])}


def _read_own(s: dict, dtype: torch.dtype) -> dict:
    paged = sys.modules.get("mgc_cuda.paged") or _paged()
    k, v = paged.kv_read(s["k_cache"], s["v_cache"], s["block_table"], s["kv_lens"], s["q_starts"], rows=s["tokens"], dtype=dtype)
    return {"k": k, "v": v}


def _attend_own(s: dict) -> torch.Tensor:
    paged = sys.modules.get("mgc_cuda.paged") or _paged()
    case = s["case"]
    return paged.paged_attention(
        s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["kv_lens"], s["q_starts"],
        max_q=s["q_max"], max_kv=s["kv_max"], scale=s["scale"], causal=case["causal"], window=case["window"],
    )


# ---- the same in elementary torch operations -----------------------------------------------------
def _quantise(x: torch.Tensor, bits: int, group: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of fp32 x [..., D]. A code is the nearest to (x - offset) / scale, from fp32 steps in
    this order: a value on the border between two codes falls as they round."""
    top = (1 << bits) - 1
    x = x.unflatten(-1, (-1, group))
    offset = x.amin(-1, keepdim=True).half()
    scale = ((x.amax(-1, keepdim=True) - offset.float()) * (1.0 / top)).half()
    step = scale.float()
    code = torch.where(step > 0, (x - offset.float()) / step, torch.zeros_like(x))
    code = code.round_().clamp_(0, top).to(torch.uint8).flatten(-2)
    if bits == 4:
        code = code[..., 0::2] | code[..., 1::2] << 4
    return code, torch.cat((scale, offset), -1)


def _values(codes: torch.Tensor, scales: torch.Tensor, bits: int) -> torch.Tensor:
    """The fp32 values that rows of a quantised cache stand for."""
    if bits == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    x = codes.float().unflatten(-1, (scales.shape[-2], -1))
    return x.mul_(scales[..., :1].float()).add_(scales[..., 1:].float()).flatten(-2)


def _tokens(s: dict):
    """Sequence, index within it and position of every new token."""
    starts = s["q_starts"].long()
    t = torch.arange(s["tokens"], device=starts.device)
    seq = torch.searchsorted(starts[1:], t, right=True)
    return seq, t - starts[seq], s["kv_lens"].long()[seq] - (starts[seq + 1] - t)


def _normed(x: torch.Tensor, weight: torch.Tensor | None) -> torch.Tensor:
    """fp32 x over the root of its mean square, times the weight. The mean is a sum of 64-bit values: its
    last bits would move codes."""
    if weight is None:
        return x
    return x * (x.double().square().mean(-1, keepdim=True) + EPS).rsqrt().float() * weight


def _rotate(x: torch.Tensor, cos, sin, pos: torch.Tensor, neighbour: bool) -> torch.Tensor:
    if cos is None:
        return x
    half = cos.shape[1]
    c, s = cos[pos][:, None], sin[pos][:, None]
    r = x[..., : 2 * half]
    a, b = (r[..., 0::2], r[..., 1::2]) if neighbour else (r[..., :half], r[..., half:])
    ra, rb = a * c - b * s, b * c + a * s
    r = torch.stack((ra, rb), -1).flatten(-2) if neighbour else torch.cat((ra, rb), -1)
    return torch.cat((r, x[..., 2 * half :]), -1)


def _append_plain(s: dict) -> dict:
    case = s["case"]
    seq, _, pos = _tokens(s)
    page, neighbour = case["page"], case["pairs"] == "neighbour"
    q = _rotate(_normed(s["q"].float(), s["q_norm"]), s["cos"], s["sin"], pos, neighbour)
    k = _rotate(_normed(s["k"].float(), s["k_norm"]), s["cos"], s["sin"], pos, neighbour)
    at = s["block_table"].long()[seq, pos // page]
    if not case["bits"]:
        dt = s["k_cache"].dtype
        s["k_cache"][at, pos % page] = k.to(dt)
        s["v_cache"][at, pos % page] = s["v"].to(dt)
        return {"q": q.to(dt), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    k_cache, v_cache = s["k_cache"], s["v_cache"]
    k_cache[0][at, pos % page], k_cache[1][at, pos % page] = _quantise(k, case["bits"], case["group"])
    v_cache[0][at, pos % page], v_cache[1][at, pos % page] = _quantise(s["v"].float(), case["bits"], case["group"])
    return {"q": q.to(s["q"].dtype), **_read_plain(s, TYPES[READ[case["src"]]])}


def _read_plain(s: dict, dtype: torch.dtype) -> dict:
    seq, _, pos = _tokens(s)
    page = s["case"]["page"]
    at = s["block_table"].long()[seq, pos // page]
    (k, k_scales, bits), (v, v_scales, _) = s["k_cache"], s["v_cache"]
    return {"k": _values(k[at, pos % page], k_scales[at, pos % page], bits).to(dtype),
            "v": _values(v[at, pos % page], v_scales[at, pos % page], bits).to(dtype)}


def _attend_plain(s: dict) -> torch.Tensor:
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    share, nq, dev = heads // kv_heads, s["q_max"], s["q"].device
    starts, lens = s["q_starts"].long(), s["kv_lens"].long()
    batch = lens.shape[0]
    # padded copies: queries [B, Hk, nq * share, D], keys and values [B, Hk, positions, D]
    i = torch.arange(nq, device=dev)
    rows = (starts[:-1, None] + i).clamp(max=max(s["tokens"] - 1, 0))
    q = s["q"].float()[rows].reshape(batch, nq, kv_heads, share, dim).permute(0, 2, 1, 3, 4)
    q = q.reshape(batch, kv_heads, nq * share, dim)
    table = s["block_table"].long()
    (k, k_scales, bits), (v, v_scales, _) = s["k_cache"], s["v_cache"]
    k = _values(k[table], k_scales[table], bits).reshape(batch, -1, kv_heads, dim).transpose(1, 2)
    v = _values(v[table], v_scales[table], bits).reshape(batch, -1, kv_heads, dim).transpose(1, 2)
    j = torch.arange(k.shape[2], device=dev)
    seen = (j < lens[:, None])[:, None].expand(batch, nq, j.numel())
    pos = lens[:, None] - (starts[1:] - starts[:-1])[:, None] + i
    if case["causal"]:
        seen = seen & (j <= pos[..., None])
    if case["window"]:
        seen = seen & (j > pos[..., None] - case["window"])
    hidden = ~seen.repeat_interleave(share, 1)[:, None]
    p = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).masked_fill_(hidden, -math.inf)
    top = p.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.reshape(batch, kv_heads, nq, share, dim).permute(0, 2, 1, 3, 4).reshape(batch, nq, heads, dim)
    seq, at, _ = _tokens(s)
    return o[seq, at].to(s["q"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case: dict) -> dict:
    qs, ks = lengths(case)
    kv_heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    tokens = sum(qs)
    index = 4 * (2 * case["batch"] + 1)
    # bytes of one cached head of one token
    cached = dim * case["bits"] // 8 + 4 * dim // case["group"] if case["bits"] else dim * BYTES[case["dtype"]]
    spans = sum(-(-k // page) - (k - q) // page for q, k in zip(qs, ks) if q)
    if case["op"] == "read":
        return {"bytes": 2 * tokens * kv_heads * (cached + dim * BYTES[case["dtype"]]) + 4 * spans + index,
                "flops": 4 * tokens * kv_heads * dim}
    heads = case["heads"]
    if case["op"] == "append":
        positions = len(set().union(*(range(k - q, k) for q, k in zip(qs, ks))))
        back = dim * BYTES[READ[case["src"]]] if case["bits"] else 0
        out = BYTES[case["src"] if case["bits"] else case["dtype"]]
        turned = tokens * (heads + kv_heads)
        return {"bytes": tokens * (heads + 2 * kv_heads) * dim * BYTES[case["src"]] + tokens * heads * dim * out
                + 2 * tokens * kv_heads * (cached + back) + positions * case["rot"] * 4 + 4 * spans + index,
                "flops": turned * (3 * case["rot"] + 4 * dim * case["norm"]) + (10 * tokens * kv_heads * dim if case["bits"] else 0)}
    pairs = rows = 0
    for q, k in zip(qs, ks):
        if not q:
            continue
        rows += k - (max(0, k - q - case["window"] + 1) if case["window"] else 0)
        pos = np.arange(k - q, k)
        pairs += int(np.minimum(pos + 1, case["window"] or k).sum()) if case["causal"] else q * k
    return {"bytes": 2 * tokens * heads * dim * BYTES[case["dtype"]] + 2 * rows * kv_heads * cached + 4 * (rows // page) + index,
            "flops": 4 * dim * heads * pairs}


# ---- the definition in 64 bits -------------------------------------------------------------------
def _grid(x: torch.Tensor, bits: int, group: int) -> torch.Tensor:
    """What a quantised cache makes of 64-bit x [..., D]."""
    top, shape = 2**bits - 1, x.shape
    x = x.reshape(-1, group)
    low = x.min(1).values.half().double()[:, None]
    step = ((x.max(1).values[:, None] - low) / top).half().double()
    code = torch.where(step > 0, torch.round((x - low) / step.clamp(min=1e-30)), torch.zeros_like(x))
    return (code.clamp(0, top) * step + low).reshape(shape)


def _stands_for(cache: tuple, used: torch.Tensor, first: int, end: int) -> torch.Tensor:
    """64-bit values [end - first, kv_heads, D] of positions [first, end) on pages `used`."""
    codes, scales = (x[used].flatten(0, 1)[first:end] for x in cache[:2])
    per = 8 // cache[2]
    whole = torch.empty(*codes.shape[:-1], codes.shape[-1] * per, dtype=torch.float64, device=codes.device)
    for i in range(per):
        whole[..., i::per] = (codes.to(torch.int32) >> cache[2] * i & 2 ** cache[2] - 1).double()
    group = whole.shape[-1] // scales.shape[-2]
    a, b = (scales[..., i].double().repeat_interleave(group, -1) for i in (0, 1))
    return whole * a + b


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    qs, ks = lengths(case)
    table = s["block_table"].cpu().numpy()
    page, dev = case["page"], s["block_table"].device
    start = 0
    if case["op"] == "append":
        q, k, v = (s[n].double().clone() for n in ("q", "k", "v"))
        for x, weight in ((q, s["q_norm"]), (k, s["k_norm"])):
            if weight is not None:
                x /= torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS)
                x *= weight.double()
        if case["rot"]:
            a = np.arange(case["rot"] // 2)
            first, second = (2 * a, 2 * a + 1) if case["pairs"] == "neighbour" else (a, a + case["rot"] // 2)
            pos = torch.from_numpy(np.concatenate([np.arange(n - m, n) for m, n in zip(qs, ks)])).to(dev)
            turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
            for x in (q, k):
                z = torch.complex(x[..., first], x[..., second]) * turn
                x[..., first], x[..., second] = z.real, z.imag
        if case["bits"]:
            return {"q": q, "k": _grid(k, case["bits"], case["group"]), "v": _grid(v, case["bits"], case["group"])}
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        at = np.concatenate([table[b, np.arange(n - m, n) // page].astype(np.int64) * page + np.arange(n - m, n) % page
                             for b, (m, n) in enumerate(zip(qs, ks))])
        k_cache.view(-1, *k.shape[1:])[torch.from_numpy(at).to(dev)] = k
        v_cache.view(-1, *k.shape[1:])[torch.from_numpy(at).to(dev)] = v
        return {"q": q, "k_cache": k_cache, "v_cache": v_cache}
    if case["op"] == "read":
        read = []
        for cache in (s["k_cache"], s["v_cache"]):
            parts = [_stands_for(cache, torch.from_numpy(table[b, : -(-nk // page)].astype(np.int64)).to(dev), nk - nq, nk)
                     for b, (nq, nk) in enumerate(zip(qs, ks))]
            read.append(torch.cat(parts))
        return {"k": read[0], "v": read[1]}
    share = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    for b, (nq, nk) in enumerate(zip(qs, ks)):
        if not nq:
            continue
        used = torch.from_numpy(table[b, : -(-nk // page)].astype(np.int64)).to(dev)
        k, v = _stands_for(s["k_cache"], used, 0, nk), _stands_for(s["v_cache"], used, 0, nk)
        part = slice(start, start + nq)
        start += nq
        away = torch.arange(nk, device=dev)[None] - torch.arange(nk - nq, nk, device=dev)[:, None]
        hide = torch.zeros_like(away, dtype=torch.bool)
        if case["causal"]:
            hide |= away > 0
        if case["window"]:
            hide |= away <= -case["window"]
        for h in range(case["heads"]):
            score = s["q"][part, h].double() @ k[:, h // share].T * s["scale"]
            weight = torch.softmax(score.masked_fill(hide, -math.inf), -1)
            out[part, h] = weight @ v[:, h // share]
    return out
