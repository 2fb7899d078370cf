"""kv_append and paged_attention against their definitions in 64 bits: every type, head layout,
page size and mask at the sizes where a kernel can go wrong."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from mgc_cuda import paged  # noqa: E402
from mgc_cuda._errors import GraphError  # noqa: E402
from paged_cases import DTYPES, ROUND, PagedBatch, angles, attention_exact, caches, rotate_exact  # noqa: E402

pytestmark = pytest.mark.gpu


def attend(x: PagedBatch, **kw):
    out = torch.full(x.q.shape, math.nan, dtype=x.q.dtype, device=x.q.device)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kw.setdefault("max_q", max(x.qs))
    kw.setdefault("max_kv", max(x.ks))
    got = paged.paged_attention(x.q, *x.operands, out=out, status=status, **kw)
    assert got is out
    paged.check_status(status)
    return out


def agree(x: PagedBatch, causal: bool = True, window: int = 0, scale: float | None = None, **kw) -> None:
    got = attend(x, causal=causal, window=window, scale=scale, **kw)
    want, bound = attention_exact(x, scale or x.q.shape[2] ** -0.5, causal, window)
    off = (got.double() - want).abs()
    worst = float((off / bound.clamp(min=1e-30)).max()) if off.numel() else 0.0
    assert torch.isfinite(got).all(), "non-finite output"
    assert worst <= 1.0, f"{worst:.3g} times the bound, max abs error {float(off.max()):.3g}"


ALL = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 1000, 4097])
def test_one_token(dtype: str, n: int) -> None:
    agree(PagedBatch([1], [n], heads=4, kv_heads=4, dim=64, page=16, dtype=dtype, seed=n))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (8, 4), (12, 4), (8, 1), (32, 8), (16, 1), (20, 1), (40, 2), (66, 2)])
def test_head_groups(dtype: str, heads: int, kv_heads: int) -> None:
    for qs, ks in (([1, 1, 1], [300, 5, 77]), ([7, 40, 1], [300, 40, 77])):
        agree(PagedBatch(qs, ks, heads=heads, kv_heads=kv_heads, dim=64, page=16, dtype=dtype, seed=heads))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("dim", [1, 4, 7, 8, 24, 32, 40, 64, 72, 80, 96, 112, 128, 160, 192, 256])
def test_head_widths(dtype: str, dim: int) -> None:
    for qs, ks in (([1, 1], [150, 33]), ([130, 3], [150, 33])):
        agree(PagedBatch(qs, ks, heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype, seed=dim))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 48, 64, 100, 128, 256, 512])
def test_page_sizes(dtype: str, page: int) -> None:
    for qs, ks in (([1, 1], [601, 130]), ([140, 70], [601, 130])):
        agree(PagedBatch(qs, ks, heads=4, kv_heads=2, dim=64, page=page, dtype=dtype, seed=page))
        agree(PagedBatch(qs, ks, heads=4, kv_heads=2, dim=128, page=page, dtype=dtype, seed=page))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("layout", ["tokens", "heads", "joint", "odd"])
def test_cache_layouts_and_query_strides(dtype: str, layout: str) -> None:
    for packed in (True, False):
        for qs in ([1, 1], [200, 30]):
            agree(PagedBatch(qs, [300, 31], heads=6, kv_heads=2, dim=64, page=16, dtype=dtype, layout=layout, packed=packed))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("qs,ks", [
    ([0, 0, 5], [0, 9, 5]),            # sequences without new tokens, without positions
    ([3, 1, 2], [1, 0, 2]),            # more new tokens than positions: rows that see nothing
    ([300, 130], [120, 0]),            # the same over whole tiles
    ([1] * 70, list(range(1, 71))),    # more sequences than a warp has lanes
    ([257, 1, 128, 64, 0, 33], [257, 900, 128, 1000, 40, 64]),
    ([513], [2000]),
])
@pytest.mark.parametrize("causal", [True, False])
def test_ragged_batches(dtype: str, qs: list[int], ks: list[int], causal: bool) -> None:
    for kv_heads, dim in ((4, 64), (1, 128)):
        agree(PagedBatch(qs, ks, heads=4, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype), causal=causal)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_short_sequences_beside_a_chunk(dtype: str, dim: int) -> None:
    """One chunk and hundreds of single tokens: a block of the tcgen05 kernel walks many units whose
    second row tile is empty, so its second warpgroup has nothing to wait for but the next unit."""
    qs = [300, *[1] * 500, 0, 129, *[2] * 100]
    ks = [400, *[1 + (37 * b) % 290 for b in range(500)], 5, 129, *[2 + (11 * b) % 40 for b in range(100)]]
    agree(PagedBatch(qs, ks, heads=2, kv_heads=2, dim=dim, page=16, dtype=dtype))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("window", [1, 2, 16, 100, 128, 1000, 5000])
def test_windows(dtype: str, window: int) -> None:
    for qs, ks in (([1, 1, 1], [700, 90, 1]), ([300, 90, 5], [700, 90, 129])):
        for dim in (64, 128):
            agree(PagedBatch(qs, ks, heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype, seed=window), window=window)


@pytest.mark.parametrize("dtype", ALL)
def test_pages_before_the_window_are_not_read(dtype: str) -> None:
    """A server may free pages that no token of a sequence sees any more: their entries say -1 and
    rows before the window hold anything."""
    for qs, ks, window in (([1, 1], [900, 333], 100), ([60, 200], [900, 333], 70)):
        x = PagedBatch(qs, ks, heads=4, kv_heads=2, dim=64, page=16, dtype=dtype)
        want, bound = attention_exact(x, 64**-0.5, True, window)
        for b, (nq, nk) in enumerate(zip(qs, ks)):
            first = max(0, nk - nq - window + 1)
            page, row = x.slots[b]
            x.k[page[:first], row[:first]] = math.nan
            x.v[page[:first], row[:first]] = math.inf
            x.block_table[b, : first // 16] = -1
        got = attend(x, window=window)
        assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("gain", [0.0, 1.0, 60.0])
def test_flat_and_peaked_rows(dtype: str, gain: float) -> None:
    """Equal scores, ordinary ones, and scores of hundreds (weights underflow, one key takes all)."""
    for qs in ([1, 1], [140, 33]):
        agree(PagedBatch(qs, [500, 200], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, gain=gain))


@pytest.mark.parametrize("dtype", ALL)
def test_rising_scores_over_many_tiles(dtype: str) -> None:
    """Scores that grow along the keys: the running maximum moves in every tile."""
    for qs in ([1], [150]):
        x = PagedBatch(qs, [1500], heads=2, kv_heads=1, dim=64, page=16, dtype=dtype)
        ramp = torch.linspace(0.05, 6.0, 1500, device="cuda")[:, None, None]
        x.k[x.slots[0]] = (torch.ones(1500, 1, 64, device="cuda") * ramp).to(x.k.dtype)
        x.q.copy_(torch.ones_like(x.q))
        agree(x)
        x.q.neg_()
        agree(x)


@pytest.mark.parametrize("dtype", ALL)
def test_minus_infinity_scores(dtype: str) -> None:
    """Keys of infinite negative score weigh nothing, as a mask added to the keys would make them;
    the first tiles hold only such keys."""
    for qs in ([1], [20]):
        x = PagedBatch(qs, [400], heads=2, kv_heads=2, dim=64, page=16, dtype=dtype)
        x.q[..., 0] = 1.0
        page, row = x.slots[0]
        x.k[page[:300], row[:300], :, 0] = -math.inf
        y = PagedBatch(qs, [400], heads=2, kv_heads=2, dim=64, page=16, dtype=dtype)
        y.q[..., 0] = 1.0
        got, (want, bound) = attend(x), attention_exact(y, 64**-0.5, True, 100 if qs == [1] else 0)
        if qs == [1]:
            assert bool(((got.double() - want).abs() <= bound).all())
        assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("max_q,max_kv", [(1, 1), (None, None), (64, 200)])
def test_bounds_only_size_the_launch(dtype: str, max_q, max_kv) -> None:
    for qs, ks in (([1, 1], [900, 40]), ([400, 40, 1], [900, 40, 300])):
        agree(PagedBatch(qs, ks, heads=4, kv_heads=2, dim=64, page=16, dtype=dtype), max_q=max_q, max_kv=max_kv)


@pytest.mark.parametrize("dtype", ALL)
def test_scales(dtype: str) -> None:
    for scale in (1e-3, 0.3, 1.0):
        agree(PagedBatch([1, 90], [200, 90], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype), scale=scale)


def test_offsets_past_32_bits() -> None:
    """Pages more than 2^31 elements apart, bytes past 2^33."""
    dim, page, heads = 64, 16, 2
    stride = 1 << 28
    flat = torch.empty(2, 17 * stride, dtype=torch.bfloat16, device="cuda")
    for qs in ([1], [150]):
        x = PagedBatch(qs, [230], heads=4, kv_heads=heads, dim=dim, page=page, dtype="bf16")
        big = [f.as_strided((x.k.shape[0], page, heads, dim), (stride, heads * dim, dim, 1)) for f in flat]
        for n, old in zip(big, (x.k, x.v)):
            n.copy_(old)
        x.k, x.v = big
        agree(x)


@pytest.mark.parametrize("dtype", ALL)
def test_a_call_repeats_its_bits_and_keeps_its_inputs(dtype: str) -> None:
    for qs, ks in (([1] * 5, [3000, 7, 900, 64, 1]), ([300, 5], [3000, 900])):
        x = PagedBatch(qs, ks, heads=8, kv_heads=2, dim=128, page=16, dtype=dtype)
        before = [t.clone() for t in (x.q, *x.operands)]
        first = attend(x)
        for _ in range(3):
            assert torch.equal(attend(x), first)
        for was, now in zip(before, (x.q, *x.operands)):
            assert torch.equal(was.nan_to_num(7.0), now.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", ALL)
def test_another_stream_and_a_cuda_graph(dtype: str) -> None:
    for qs, ks in (([1, 1], [2500, 70]), ([150, 3], [600, 70])):
        x = PagedBatch(qs, ks, heads=4, kv_heads=2, dim=64, page=16, dtype=dtype)
        want = attend(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = paged.paged_attention(x.q, *x.operands, max_q=max(qs), max_kv=max(ks))
        side.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = paged.paged_attention(x.q, *x.operands, max_q=max(qs), max_kv=max(ks))
        held.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


@pytest.mark.parametrize("dtype", ALL)
def test_bad_pages_set_the_status(dtype: str) -> None:
    for qs in ([1, 1], [200, 3]):
        x = PagedBatch(qs, [300, 20], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype)
        for bad in (-1, x.k.shape[0], 1 << 30):
            x.block_table[0, 3] = bad
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            got = paged.paged_attention(x.q, *x.operands, max_q=max(qs), max_kv=300, status=status)
            with pytest.raises(GraphError, match="out of range"):
                paged.check_status(status)
            assert torch.isfinite(got[x.rows(1)]).all()
        # a length past the block table: the positions beyond it are not read either
        x = PagedBatch(qs, [300, 20], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype)
        x.kv_lens[1] = 10_000
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        paged.paged_attention(x.q, *x.operands, max_q=max(qs), max_kv=300, status=status)
        with pytest.raises(GraphError, match="out of range"):
            paged.check_status(status)


def test_no_tokens() -> None:
    x = PagedBatch([0, 0], [5, 0], heads=4, kv_heads=2, dim=64, page=16, dtype="bf16")
    assert paged.paged_attention(x.q, *x.operands).shape == (0, 4, 64)
    assert paged.kv_append(x.q[:, :2], x.q[:, :2], *x.operands) is None


# ---- append --------------------------------------------------------------------------------------
def appended(qs, ks, *, dtype, src, heads, kv_heads, dim, page, rot, interleaved=False, layout="tokens", inplace=False,
             odd=False):
    x = PagedBatch(qs, ks, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, layout=layout)
    tokens = sum(qs)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    wide = dim + 1 if odd else dim
    qkv = torch.randn(max(tokens, 1), heads + 2 * kv_heads, wide, generator=g, device="cuda").to(DTYPES[src])[:tokens]
    qkv = qkv[..., wide - dim :]
    q, k, v = qkv[:, :heads], qkv[:, heads : heads + kv_heads], qkv[:, heads + kv_heads :]
    cos, sin = angles(max([*ks, 1]), rot) if rot else (None, None)
    want_k, want_v, want_q = x.k.double(), x.v.double(), q.double().clone()
    for b, (nq, nk) in enumerate(zip(qs, ks)):
        keep = max(0, nq - nk)  # tokens at negative positions: not cached, not rotated
        part = slice(x.rows(b).start + keep, x.rows(b).stop)
        if part.start == part.stop:
            continue
        pos = torch.arange(nk - nq + keep, nk, device="cuda")
        page_, row = x.slots[b][0][pos], x.slots[b][1][pos]
        kk = k[part].double()
        if rot:
            kk = rotate_exact(k[part], pos, cos, sin, interleaved)
            want_q[part] = rotate_exact(q[part], pos, cos, sin, interleaved)
        want_k[page_, row], want_v[page_, row] = kk, v[part].double()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = paged.kv_append(k, v, *x.operands, q=q, cos=cos, sin=sin, interleaved=interleaved,
                          q_out=q if inplace else None, status=status)
    paged.check_status(status)
    # two products and a sum in fp32 (2^-23 of their sizes, at most sqrt(2) |x|), rounded once
    for got, want in ((out, want_q), (x.k, want_k), (x.v, want_v)):
        assert got.dtype == DTYPES[dtype]
        off = (got.double() - want).abs().nan_to_num(0.0)
        bound = ROUND[dtype] * want.abs() + 2.0**-22 * 8.0 * (1.0 if rot else 0.0) + 2.0**-25 * (dtype == "f16")
        assert torch.equal(got.isnan(), want.isnan())
        assert bool((off <= bound.nan_to_num(1.0)).all()), float((off / bound.clamp(min=1e-30)).max())


@pytest.mark.parametrize("dtype,src", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("dim,rot", [(64, 0), (64, 64), (128, 128), (80, 32), (80, 40), (96, 48), (72, 72), (7, 6), (1, 0), (256, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(dtype: str, src: str, dim: int, rot: int, interleaved: bool) -> None:
    appended([1, 0, 9, 40, 2], [70, 3, 9, 100, 1], dtype=dtype, src=src, heads=6, kv_heads=2, dim=dim, page=16, rot=rot,
             interleaved=interleaved)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("layout", ["tokens", "heads", "joint", "odd"])
@pytest.mark.parametrize("page", [1, 24, 64])
def test_append_layouts(dtype: str, layout: str, page: int) -> None:
    for odd in (False, True):
        appended([5, 1, 33], [5, 100, 70], dtype=dtype, src=dtype, heads=4, kv_heads=4, dim=64, page=page, rot=32,
                 layout=layout, odd=odd)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_rotates_queries_in_place(dtype: str, interleaved: bool) -> None:
    appended([300, 1], [300, 80], dtype=dtype, src=dtype, heads=9, kv_heads=3, dim=64, page=16, rot=64,
             interleaved=interleaved, inplace=True)


def test_append_many_tokens_and_sequences() -> None:
    appended([1] * 100, list(range(1, 101)), dtype="bf16", src="bf16", heads=32, kv_heads=8, dim=128, page=16, rot=128)
    appended([2000, 1500], [2500, 1500], dtype="bf16", src="bf16", heads=8, kv_heads=2, dim=128, page=64, rot=128)


def test_append_skips_what_it_cannot_place() -> None:
    x = PagedBatch([3, 2], [40, 2], heads=4, kv_heads=2, dim=64, page=16, dtype="bf16")
    k = torch.randn(5, 2, 64, device="cuda").to(torch.bfloat16)
    before = x.k.clone()
    x.block_table[0, 2] = x.k.shape[0]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.kv_append(k, k, *x.operands, status=status)
    with pytest.raises(GraphError, match="out of range"):
        paged.check_status(status)
    page, row = x.slots[1]
    before[page, row] = k[3:]
    assert torch.equal(before.nan_to_num(7.0), x.k.nan_to_num(7.0))
    # a rotation table shorter than the positions
    cos, sin = angles(39, 64)
    x = PagedBatch([3, 2], [40, 2], heads=4, kv_heads=2, dim=64, page=16, dtype="bf16")
    status.zero_()
    q = paged.kv_append(k, k, *x.operands, q=x.q, cos=cos, sin=sin, status=status)
    with pytest.raises(GraphError, match="out of range"):
        paged.check_status(status)
    assert torch.equal(q[2], x.q[2])


def test_append_then_attend_equals_the_whole_sequence() -> None:
    """Token by token over the cache against one call over the whole sequence."""
    n, heads, kv_heads, dim, page = 75, 8, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(n, h, dim, generator=g, device="cuda") for h in (heads, kv_heads, kv_heads))
    cos, sin = angles(n, dim)
    table = torch.tensor([[4, 0, 3, 1, 2]], dtype=torch.int32, device="cuda")

    def lens(*values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    whole, single = caches("tokens", 5, page, kv_heads, dim, torch.float32, "cuda"), \
        caches("tokens", 5, page, kv_heads, dim, torch.float32, "cuda")
    rq = paged.kv_append(k, v, *whole, table, lens(n), lens(0, n), q=q, cos=cos, sin=sin)
    want = paged.paged_attention(rq, *whole, table, lens(n), lens(0, n), max_q=n, max_kv=n)
    for t in range(n):
        at = (table, lens(t + 1), lens(0, 1))
        r1 = paged.kv_append(k[t : t + 1], v[t : t + 1], *single, *at, q=q[t : t + 1], cos=cos, sin=sin)
        got = paged.paged_attention(r1, *single, *at, max_q=1, max_kv=t + 1)
        # both are within the fp32 bound of the same exact value: 1e-5 of values of a few units
        assert float((got[0] - want[t]).abs().max()) <= 1e-5 * 4
    assert torch.equal(whole[0][table[0, :4].long()], single[0][table[0, :4].long()])


# ---- refusals ------------------------------------------------------------------------------------
@pytest.mark.parametrize("change,match", [
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(window=-1), "window"), (dict(window=4, causal=False), "window"), (dict(max_q=-1), "bound"),
])
def test_refused_arguments(change: dict, match: str) -> None:
    x = PagedBatch([1], [9], heads=4, kv_heads=2, dim=64, page=16, dtype="f16")
    with pytest.raises(Exception, match=match):
        paged.paged_attention(x.q, *x.operands, **change)


def test_refused_tensors() -> None:
    x = PagedBatch([2], [9], heads=4, kv_heads=2, dim=64, page=16, dtype="f16")
    k, v, table, lens, starts = x.operands
    kv = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")
    cos, sin = angles(16, 64)
    bad = [
        lambda: paged.paged_attention(x.q.float(), k, v, table, lens, starts),
        lambda: paged.paged_attention(x.q.cpu(), k, v, table, lens, starts),
        lambda: paged.paged_attention(x.q[:, :3], k, v, table, lens, starts),
        lambda: paged.paged_attention(x.q[:, :, :32], k, v, table, lens, starts),
        lambda: paged.paged_attention(x.q, k, v.float(), table, lens, starts),
        lambda: paged.paged_attention(x.q, k, v[:1], table, lens, starts),
        lambda: paged.paged_attention(x.q, k.transpose(2, 3), v.transpose(2, 3), table, lens, starts),
        lambda: paged.paged_attention(x.q, k, v, table.long(), lens, starts),
        lambda: paged.paged_attention(x.q, k, v, table, lens, starts[:1]),
        lambda: paged.paged_attention(x.q, k, v, table, lens.cpu(), starts),
        lambda: paged.paged_attention(x.q, k, v, table, lens, starts, out=torch.empty_like(x.q, dtype=torch.float32)),
        lambda: paged.kv_append(kv, kv.float(), k, v, table, lens, starts),
        lambda: paged.kv_append(kv[:, :1], kv[:, :1], k, v, table, lens, starts),
        lambda: paged.kv_append(kv.bfloat16(), kv.bfloat16(), k, v, table, lens, starts),
        lambda: paged.kv_append(kv, kv, k, v, table, lens, starts, cos=cos),
        lambda: paged.kv_append(kv, kv, k, v, table, lens, starts, cos=cos.half(), sin=sin.half()),
        lambda: paged.kv_append(kv, kv, k, v, table, lens, starts, cos=torch.cat((cos, cos), 1), sin=torch.cat((sin, sin), 1)),
        lambda: paged.kv_append(kv.float(), kv.float(), k, v, table, lens, starts, q=x.q.float(), q_out=x.q.float()),
    ]
    for call in bad:
        with pytest.raises(Exception) as e:
            call()
        assert "paged_attention" in str(e.value) or "kv_append" in str(e.value), str(e.value)
