"""Benchmark cases of the paged-cache operators: appending keys and values to a paged cache (with the
position rotation on the way) and the attention of new tokens over that cache.

A batch of sequences is described by ``block_table`` [B, P] (the pages of each sequence, in order),
``kv_lens`` [B] (cached positions, the new tokens included) and ``q_starts`` [B + 1] (where each
sequence's new tokens begin in the packed token axis). Token t of sequence b sits at position
``kv_lens[b] - (q_starts[b + 1] - t)``. The cache is two tensors [pages, page_size, kv_heads, D].

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
MAX_POSITIONS = 1 << 17


def listed() -> list[dict]:
    """Four appends, then eight attentions; `q` and `kv` are the longest sequence's new tokens and
    positions, `ragged` how far the shortest one falls below it."""
    return [
        # one new token of GPT-2 small (12 heads of 64, fp32, learned positions, nothing to rotate)
        dict(name="append_one_f32", op="append", dtype="f32", src="f32", batch=1, q=1, kv=128, ragged=0.0,
             heads=12, kv_heads=12, dim=64, page=16, rot=0, pairs="half"),
        # a decoding step of 64 sequences with grouped heads and rotated positions
        dict(name="append_steps_bf16", op="append", dtype="bf16", src="bf16", batch=64, q=1, kv=4096, ragged=0.9,
             heads=32, kv_heads=8, dim=128, page=16, rot=128, pairs="half"),
        # prompts of a few thousand tokens each
        dict(name="append_prompts_bf16", op="append", dtype="bf16", src="bf16", batch=6, q=4001, kv=4001, ragged=0.5,
             heads=32, kv_heads=8, dim=128, page=64, rot=128, pairs="half"),
        # fp32 projections into a half-precision cache, part of each head rotated by neighbours, pages of 24
        dict(name="append_ragged_f16", op="append", dtype="f16", src="f32", batch=7, q=613, kv=1500, ragged=1.0,
             heads=20, kv_heads=4, dim=80, page=24, rot=32, pairs="neighbour"),
        # decoding with GPT-2 small: one sequence, and sixteen up to its longest context
        dict(name="decode_one_f32", op="attend", dtype="f32", batch=1, q=1, kv=128, ragged=0.0,
             heads=12, kv_heads=12, dim=64, page=16, causal=True, window=0),
        dict(name="decode_batch_f32", op="attend", dtype="f32", batch=16, q=1, kv=1024, ragged=0.7,
             heads=12, kv_heads=12, dim=64, page=16, causal=True, window=0),
        # a serving batch with grouped heads and mixed contexts
        dict(name="decode_batch_bf16", op="attend", dtype="bf16", batch=64, q=1, kv=8192, ragged=0.8,
             heads=32, kv_heads=8, dim=128, page=16, causal=True, window=0),
        # one sequence with a very long context
        dict(name="decode_long_f16", op="attend", dtype="f16", batch=1, q=1, kv=131071, ragged=0.0,
             heads=32, kv_heads=8, dim=128, page=64, causal=True, window=0),
        # a chunk of a long prompt over what is cached already
        dict(name="chunk_bf16", op="attend", dtype="bf16", batch=1, q=2048, kv=16384, ragged=0.0,
             heads=32, kv_heads=8, dim=128, page=64, causal=True, window=0),
        # chunks and single tokens together, a sliding window
        dict(name="mixed_bf16", op="attend", dtype="bf16", batch=9, q=1003, kv=4100, ragged=1.0,
             heads=12, kv_heads=12, dim=64, page=16, causal=True, window=1024),
        # prompts of GPT-2 small up to its longest context
        dict(name="prompts_f32", op="attend", dtype="f32", batch=8, q=1024, kv=1024, ragged=0.6,
             heads=12, kv_heads=12, dim=64, page=16, causal=True, window=0),
        # five proposed tokens for each sequence, one shared key head, pages that end inside a tile
        dict(name="verify_f16", op="attend", dtype="f16", batch=8, q=5, kv=2047, ragged=0.5,
             heads=16, kv_heads=1, dim=96, page=24, causal=True, window=0),
    ]


def draw(rng) -> dict:
    """A case of the same ranges: every length from one token to the longest, odd ones among them."""

    def spread(lo: int, hi: int) -> int:
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))

    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    group = rng.choice([1, 1, 3, 4, 8]) if kv_heads < 12 else 1
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    ragged = rng.choice([0.0, 0.3, 0.7, 1.0])
    case = dict(dtype=dtype, ragged=ragged, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page)
    kind = rng.choice(["append", "append", "decode", "decode", "chunk", "prompt", "verify"])
    if kind == "append":
        batch = spread(1, 64)
        q = spread(1, max(1, min(4001, 16000 // batch)))
        kv = q + spread(1, max(2, 64000 // batch)) - 1
        rot = rng.choice([0, dim, dim, dim // 2])
        return dict(case, op="append", src=rng.choice([dtype, dtype, "f32"]), batch=batch, q=q, kv=kv, rot=rot,
                    pairs=rng.choice(["half", "neighbour"]))
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
    case = dict(case, op="attend", batch=batch, q=q, kv=kv, causal=causal, window=window if causal else 0)
    # no dearer than the largest listed cases, in pairs of a query and a key and in cache values
    size = max(case["heads"] * dim * batch * q * kv / (32 * 128 * 2048 * 15000),
               BYTES[dtype] * kv_heads * dim * batch * kv / (2 * 8 * 128 * 64 * 5000))
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


def prepare(case: dict, seed: int) -> dict:
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 31))
    qs, ks = lengths(case)
    tokens = sum(qs)
    page, dim, heads, kv_heads = case["page"], case["dim"], case["heads"], case["kv_heads"]
    need = [-(-k // page) for k in ks]
    pages = sum(need) + 3
    order = host.permutation(pages)
    table = np.zeros((case["batch"], max(max(need), 1)), np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    dt = TYPES[case["dtype"]]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    shape = (pages, page, kv_heads, dim)
    # keys have channels with an offset of their own, as trained models' keys do
    k_cache, v_cache = normal(*shape), normal(*shape)
    k_cache += normal(kv_heads, dim) * 0.5
    s = dict(
        case=case, q_max=case["q"], kv_max=max(ks), k_cache=k_cache, v_cache=v_cache,
        block_table=torch.from_numpy(table).to(dev),
        kv_lens=torch.tensor(ks, dtype=torch.int32, device=dev),
        q_starts=torch.tensor(np.concatenate([[0], np.cumsum(qs)]), dtype=torch.int32, device=dev),
    )
    if case["op"] == "append":
        # q, k and v as the fused projection leaves them: one row of all heads for each token
        src = TYPES[case["src"]]
        qkv = normal(max(tokens, 1), heads + 2 * kv_heads, dim, dtype=src)[:tokens]
        s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads : heads + kv_heads], qkv[:, heads + kv_heads :]
        if case["rot"]:
            half = case["rot"] // 2
            inv = 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
            angle = torch.arange(MAX_POSITIONS, device=dev, dtype=torch.float64)[:, None] * inv
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        else:
            s["cos"] = s["sin"] = None
    else:
        # score rows have a spread of about 2, between flat and one-hot
        s["q"] = normal(tokens, heads, dim) * 1.75
        s["scale"] = 1.0 / math.sqrt(dim)
    return s


def run(s: dict):
    case = s["case"]
    if case["op"] == "append":
        return _append_own(s) if own else _append_plain(s)
    return _attend_own(s) if own else _attend_plain(s)


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
    q = paged.kv_append(
        s["k"], s["v"], s["k_cache"], s["v_cache"], s["block_table"], s["kv_lens"], s["q_starts"],
        q=s["q"], cos=s["cos"], sin=s["sin"], interleaved=s["case"]["pairs"] == "neighbour",
    )
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attend_own(s: dict):
    paged = sys.modules.get("mgc_cuda.paged") or _paged()
    case = s["case"]
    return paged.paged_attention(
        s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["kv_lens"], s["q_starts"],
        max_q=s["q_max"], max_kv=s["kv_max"], scale=s["scale"], causal=case["causal"], window=case["window"],
    )


# ---- the same in elementary torch operations -----------------------------------------------------
def _tokens(s: dict):
    """Sequence, index within it and position of every new token."""
    starts, total = s["q_starts"].long(), s["q"].shape[0]
    t = torch.arange(total, device=starts.device)
    seq = (t[:, None] >= starts[None, 1:]).sum(1)
    return seq, t - starts[seq], s["kv_lens"].long()[seq] - (starts[seq + 1] - t)


def _rotate(x: torch.Tensor, cos, sin, pos: torch.Tensor, neighbour: bool) -> torch.Tensor:
    if cos is None:
        return x
    half = cos.shape[1]
    c, s = cos[pos][:, None].to(x.dtype), sin[pos][:, None].to(x.dtype)
    r = x[..., : 2 * half]
    a, b = (r[..., 0::2], r[..., 1::2]) if neighbour else (r[..., :half], r[..., half:])
    ra, rb = a * c - b * s, b * c + a * s
    r = torch.stack((ra, rb), -1).flatten(-2) if neighbour else torch.cat((ra, rb), -1)
    return torch.cat((r, x[..., 2 * half :]), -1)


def _append_plain(s: dict) -> dict:
    seq, _, pos = _tokens(s)
    page, neighbour = s["case"]["page"], s["case"]["pairs"] == "neighbour"
    dt = s["k_cache"].dtype
    q = _rotate(s["q"].float(), s["cos"], s["sin"], pos, neighbour).to(dt)
    k = _rotate(s["k"].float(), s["cos"], s["sin"], pos, neighbour).to(dt)
    at = s["block_table"].long()[seq, pos // page]
    s["k_cache"][at, pos % page] = k
    s["v_cache"][at, pos % page] = s["v"].to(dt)
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attend_plain(s: dict) -> torch.Tensor:
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    group, nq, dev = heads // kv_heads, s["q_max"], s["q"].device
    starts, lens = s["q_starts"].long(), s["kv_lens"].long()
    batch = lens.shape[0]
    # padded copies: queries [B, Hk, nq * group, D], keys and values [B, Hk, positions, D]
    i = torch.arange(nq, device=dev)
    rows = (starts[:-1, None] + i).clamp(max=max(s["q"].shape[0] - 1, 0))
    q = s["q"].float()[rows].reshape(batch, nq, kv_heads, group, dim).permute(0, 2, 1, 3, 4)
    q = q.reshape(batch, kv_heads, nq * group, dim)
    table = s["block_table"].long()
    k = s["k_cache"][table].float().reshape(batch, -1, kv_heads, dim).transpose(1, 2)
    v = s["v_cache"][table].float().reshape(batch, -1, kv_heads, dim).transpose(1, 2)
    j = torch.arange(k.shape[2], device=dev)
    seen = (j < lens[:, None])[:, None].expand(batch, nq, j.numel())
    pos = lens[:, None] - (starts[1:] - starts[:-1])[:, None] + i
    if case["causal"]:
        seen = seen & (j <= pos[..., None])
    if case["window"]:
        seen = seen & (j > pos[..., None] - case["window"])
    hidden = ~seen.repeat_interleave(group, 1)[:, None]
    p = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).masked_fill_(hidden, -math.inf)
    top = p.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.reshape(batch, kv_heads, nq, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, nq, heads, dim)
    seq, at, _ = _tokens(s)
    return o[seq, at].to(s["q"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case: dict) -> dict:
    qs, ks = lengths(case)
    heads, kv_heads, dim, es = case["heads"], case["kv_heads"], case["dim"], BYTES[case["dtype"]]
    tokens = sum(qs)
    index = 4 * (2 * case["batch"] + 1)
    if case["op"] == "append":
        values = tokens * (heads + 2 * kv_heads) * dim
        pages = sum(-(-k // case["page"]) - (k - q) // case["page"] for q, k in zip(qs, ks) if q)
        positions = len(set().union(*(range(k - q, k) for q, k in zip(qs, ks))))
        return {"bytes": values * (BYTES[case["src"]] + es) + positions * case["rot"] * 4 + 4 * pages + index,
                "flops": 3 * tokens * (heads + kv_heads) * case["rot"]}
    pairs = rows = 0
    for q, k in zip(qs, ks):
        if not q:
            continue
        first = max(0, k - q - case["window"] + 1) if case["window"] else 0
        rows += k - first
        if not case["causal"]:
            pairs += q * k
            continue
        pos = np.arange(k - q, k)
        pairs += int((pos + 1 if not case["window"] else np.minimum(pos + 1, case["window"])).sum())
    return {"bytes": 2 * tokens * heads * dim * es + 2 * rows * kv_heads * dim * es + 4 * (rows // case["page"]) + index,
            "flops": 4 * dim * heads * pairs}


# ---- the definition in 64 bits -------------------------------------------------------------------
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    qs, ks = lengths(case)
    table = s["block_table"].cpu().numpy()
    page, group = case["page"], case["heads"] // case["kv_heads"]
    start = 0
    if case["op"] == "append":
        q = s["q"].double().clone()
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        for b, (nq, nk) in enumerate(zip(qs, ks)):
            if not nq:
                continue
            at = np.arange(nk - nq, nk)
            slots = torch.from_numpy(table[b, at // page].astype(np.int64) * page + at % page).to(q.device)
            part = slice(start, start + nq)
            start += nq
            k = s["k"][part].double()
            if case["rot"]:
                half = case["rot"] // 2
                a = np.arange(half)
                first, second = (2 * a, 2 * a + 1) if case["pairs"] == "neighbour" else (a, a + half)
                turn = torch.complex(s["cos"][nk - nq : nk].double(), s["sin"][nk - nq : nk].double())[:, None]
                for x in (q[part], k):
                    z = torch.complex(x[..., first], x[..., second]) * turn
                    x[..., first], x[..., second] = z.real, z.imag
            k_cache.view(-1, *k.shape[1:])[slots] = k
            v_cache.view(-1, *k.shape[1:])[slots] = s["v"][part].double()
        return {"q": q, "k_cache": k_cache, "v_cache": v_cache}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b, (nq, nk) in enumerate(zip(qs, ks)):
        if not nq:
            continue
        used = torch.from_numpy(table[b, : -(-nk // page)].astype(np.int64)).to(out.device)
        k = s["k_cache"][used].flatten(0, 1)[:nk].double()
        v = s["v_cache"][used].flatten(0, 1)[:nk].double()
        part = slice(start, start + nq)
        start += nq
        away = torch.arange(nk, device=out.device)[None] - torch.arange(nk - nq, nk, device=out.device)[:, None]
        hide = torch.zeros_like(away, dtype=torch.bool)
        if case["causal"]:
            hide |= away > 0
        if case["window"]:
            hide |= away <= -case["window"]
        for h in range(case["heads"]):
            score = s["q"][part, h].double() @ k[:, h // group].T * s["scale"]
            weight = torch.softmax(score.masked_fill(hide, -math.inf), -1)
            out[part, h] = weight @ v[:, h // group]
    return out
