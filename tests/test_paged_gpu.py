"""GPU tests of the paged K/V cache against plain 64-bit formulas: attention of one token and of many, appended rows,
page bookkeeping.

Bounds of the attention outputs are derived from the arithmetic.  With A = sum_p w_p |v_p| (w the softmax weights) and
D = max_p scale sum_d |q_d k_d| over a row's visible positions, a score is off by at most e = D (2^-21 + dim 2^-24) (the
operands' pairs, the fp32 sum over the dimension, the change of base), which moves every weight by a factor within 1 +-
2e; the exponential and the running sums add (2^-20 + n / 16 2^-24).  A weight is rounded to u_w (2^-20 as an fp16
pair, 2^-16 as a bf16 pair; 2^-11 or 2^-8 where a single one of its type enters the product) and the result to u_o
(2^-23, 2^-11, 2^-8 for fp32, fp16, bf16).  So |out - exact| <= A (2e + 2 u_w + 2^-20 + n 2^-28) + |exact| u_o.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
U_OUT = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U_PAIR = {torch.float16: 2.0 ** -20, torch.bfloat16: 2.0 ** -16}
U_ONE = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -24, torch.bfloat16: 1e-37}  # an output below the normals


@pytest.fixture(scope="module")
def paged():
    from rta_b200 import paged as module
    torch.cuda.init()
    return module


def build(paged, lengths, kv_heads, dim, page, dtype, order="heads", seed=0, spare=3, slots=None, layers=1, stale=None,
          pages=None):
    """A cache whose sequences hold `lengths` positions in pages of random order; `stale` fills every place that no
    sequence holds."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare if pages is None else pages
    cache = paged.PagedCache.create(layers, pages, page, kv_heads, dim, slots or len(lengths),
                                    max(1, max(need)) * page, dtype, "cuda", order)
    perm = torch.randperm(pages, device="cuda", generator=g)[:sum(need)].to(torch.int32)
    at = 0
    for s, n in enumerate(need):
        cache.map.table[s, :n] = perm[at:at + n]
        at += n
    cache.map.refs[perm.long()] = 1
    cache.map.lengths[:len(lengths)] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for pool in (cache.k, cache.v):
        if stale is not None:
            pool.fill_(stale)
        for s, n in enumerate(lengths):
            for layer in range(layers):
                rows = torch.randn(n, kv_heads, dim, device="cuda", generator=g).to(dtype)
                put(cache, pool, layer, s, 0, rows)
    return cache


def put(cache, pool, layer, slot, first, rows):
    p = torch.arange(first, first + rows.shape[0], device="cuda")
    at = cache.map.table[slot].long()[p // cache.page_size]
    pool[layer, at, :, p % cache.page_size] = rows


def get(cache, pool, layer, slot, n, map=None):
    """[n, kv_heads, dim] of a sequence's first n positions."""
    p = torch.arange(n, device="cuda")
    at = (map or cache.map).table[slot].long()[p // cache.page_size]
    return pool[layer, at, :, p % cache.page_size]


def ints(*x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def attend(q, k, v, t, window, sinks, scale, u_w, u_out, tiny):
    """64-bit attention of rows q [m, heads, dim] at positions t over k, v [n, kv_heads, dim]: out, lse, and the bound
    of the module's docstring."""
    m, heads, dim = q.shape
    n, kv_heads = k.shape[:2]
    out = torch.zeros(m, heads, dim, dtype=torch.float64, device="cuda")
    bound, lse = torch.full_like(out, tiny), torch.full((m, heads), -math.inf, dtype=torch.float64, device="cuda")
    lse_bound = torch.zeros_like(lse)
    if n == 0 or m == 0:
        return out, lse, bound, lse_bound
    p = torch.arange(n, device="cuda")[None]
    see = p <= t[:, None]
    if window:
        see &= (p > t[:, None] - window) | (p < sinks)
    some = see.any(1)
    for h in range(heads):
        kh, vh, qh = k[:, h // (heads // kv_heads)].double(), v[:, h // (heads // kv_heads)].double(), q[:, h].double()
        s = (qh @ torch.nan_to_num(kh).T * scale).masked_fill(~see, -math.inf)
        big = (qh.abs() @ torch.nan_to_num(kh).abs().T * abs(scale)).masked_fill(~see, 0).amax(1)
        l = torch.logsumexp(s, 1)
        w = torch.exp(s - l[:, None]).masked_fill(~see, 0)
        w[~some] = 0
        o = torch.where(some[:, None], w @ torch.nan_to_num(vh), 0)
        e = big * (2.0 ** -21 + dim * 2.0 ** -24)
        a = w @ torch.nan_to_num(vh).abs()
        factor = 2 * e + 2 * u_w + 2.0 ** -20 + n * 2.0 ** -28
        out[:, h], lse[some, h] = o, l[some]
        bound[:, h] = a * factor[:, None] + o.abs() * u_out + tiny
        lse_bound[:, h] = e + 2.0 ** -18 + n * 2.0 ** -28 + l.abs().nan_to_num(posinf=0) * 2.0 ** -22
    return out, lse, bound, lse_bound


def near(got, want, bound, what):
    got = got.double()
    over = (got - want).abs() - bound
    assert torch.isfinite(got).all(), f"{what}: not finite"
    assert (over <= 0).all(), f"{what}: off by {(got - want).abs().max().item():.3g}, {over.max().item():.3g} too much"


DECODE = [
    # types, heads, kv_heads, dim, page, order, lengths, window, sinks
    (torch.float16, True, 16, 4, 256, 16, "heads", [513], 0, 0),
    (torch.float16, True, 16, 4, 256, 16, "heads", [1, 0, 15, 16, 17, 300, 4097], 0, 0),
    (torch.float16, True, 12, 12, 64, 7, "positions", [33, 1, 0, 250], 0, 0),
    (torch.float16, True, 40, 2, 128, 5, "positions", [64, 129, 2], 0, 0),
    (torch.float16, False, 16, 4, 256, 1, "heads", [3, 70, 31], 0, 0),
    (torch.float16, False, 32, 2, 256, 48, "heads", [47, 48, 49, 500], 0, 0),
    (torch.float16, False, 9, 1, 64, 100, "positions", [99, 100, 101, 777], 0, 0),
    (torch.float16, False, 28, 4, 128, 64, "heads", [0, 0, 0], 0, 0),
    (torch.bfloat16, False, 32, 8, 128, 64, "positions", [1, 64, 65, 1000, 3000], 0, 0),
    (torch.bfloat16, False, 128, 1, 128, 16, "heads", [333, 12], 0, 0),
    (torch.bfloat16, False, 8, 8, 256, 3, "positions", [8, 2, 100], 0, 0),
    (torch.bfloat16, False, 64, 4, 64, 32, "heads", [1500, 0, 31], 0, 0),
    (torch.float16, True, 16, 4, 256, 16, "heads", [5, 100, 101, 104, 1000, 0], 100, 4),
    (torch.float16, False, 32, 8, 128, 8, "positions", [5, 16, 17, 18, 33, 2000], 16, 1),
    (torch.bfloat16, False, 14, 2, 64, 6, "heads", [1, 2, 3, 700], 1, 0),
    (torch.bfloat16, False, 32, 8, 128, 64, "heads", [20, 130, 140, 1999], 128, 300),
    (torch.bfloat16, False, 16, 1, 256, 16, "heads", [90, 4000], 1000, 77),
]


@pytest.mark.parametrize("case", DECODE, ids=str)
def test_decode(paged, case):
    dtype, q32, heads, kv_heads, dim, page, order, lengths, window, sinks = case
    cache = build(paged, lengths, kv_heads, dim, page, dtype, order, seed=len(str(case)), stale=math.nan)
    q = torch.randn(len(lengths), heads, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(
        torch.float32 if q32 else dtype)
    scale = dim ** -0.5
    out, lse = cache.decode(q, window=window, sinks=sinks, lse=True)
    cache.check()
    for b, n in enumerate(lengths):
        k, v = get(cache, cache.k, 0, b, n), get(cache, cache.v, 0, b, n)
        want, want_lse, bound, lse_bound = attend(q[b:b + 1], k, v, torch.tensor([n - 1], device="cuda"), window, sinks,
                                                  scale, U_PAIR[dtype], U_OUT[q.dtype], TINY[q.dtype])
        near(out[b:b + 1], want, bound, f"sequence {b}")
        if n:
            near(lse[b:b + 1], want_lse, lse_bound, f"lse {b}")
        else:
            assert (lse[b] == -math.inf).all() and (out[b] == 0).all()


@pytest.mark.parametrize("batch,longest", [(1, 40000), (3, 20000), (300, 200), (1100, 40)])
def test_decode_many_and_long(paged, batch, longest):
    """Units that are cut over many blocks, and more sequences than a block has threads."""
    rng = np.random.default_rng(batch)
    lengths = [longest] if batch == 1 else [int(x) for x in rng.integers(0, longest + 1, batch)]
    cache = build(paged, lengths, 2, 64, 16, torch.float16, seed=batch)
    q = torch.randn(batch, 6, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    out = cache.decode(q)
    cache.check()
    for b in sorted({0, 1 % batch, batch // 2, batch - 1, int(np.argmax(lengths)), int(np.argmin(lengths))}):
        n = lengths[b]
        want, _, bound, _ = attend(q[b:b + 1], get(cache, cache.k, 0, b, n), get(cache, cache.v, 0, b, n),
                                   torch.tensor([n - 1], device="cuda"), 0, 0, 0.125, 2.0 ** -20, 2.0 ** -23, 1e-37)
        near(out[b:b + 1], want, bound, f"sequence {b}")
    assert torch.equal(out, cache.decode(q))  # the same bits again


def test_decode_slots_strides_layers_scale(paged):
    lengths = [40, 0, 77, 130]
    cache = build(paged, lengths, 2, 128, 16, torch.bfloat16, layers=3, slots=6)
    slots = torch.tensor([3, 0, 2, 3], dtype=torch.int32, device="cuda")
    wide = torch.randn(4, 24, 128, device="cuda").bfloat16()
    q = wide[:, 8:16]  # rows of a wider projection
    out = torch.empty(4, 8, 128, dtype=torch.bfloat16, device="cuda")
    got = cache.decode(q, layer=2, slots=slots, scale=-0.3, out=out)
    assert got is out
    cache.check()
    for i, s in enumerate(slots.tolist()):
        n = lengths[s]
        want, _, bound, _ = attend(q[i:i + 1], get(cache, cache.k, 2, s, n), get(cache, cache.v, 2, s, n),
                                   torch.tensor([n - 1], device="cuda"), 0, 0, -0.3, 2.0 ** -16, 2.0 ** -8, 1e-37)
        near(got[i:i + 1], want, bound, f"row {i}")


PREFILL = [
    # type, heads, kv_heads, dim, page, order, [(past, new)], window, sinks
    (torch.float16, 16, 4, 256, 16, "heads", [(0, 64)], 0, 0),
    (torch.float16, 16, 4, 256, 16, "heads", [(1984, 64)], 0, 0),
    (torch.float16, 16, 4, 256, 5, "positions", [(0, 1), (130, 3), (0, 0), (7, 200), (300, 33)], 0, 0),
    (torch.bfloat16, 32, 8, 128, 64, "positions", [(0, 129), (64, 64), (1, 1), (1000, 2)], 0, 0),
    (torch.bfloat16, 28, 4, 128, 7, "heads", [(0, 300), (50, 19)], 0, 0),
    (torch.bfloat16, 8, 8, 64, 16, "heads", [(0, 513), (2, 255)], 0, 0),
    (torch.float16, 16, 1, 64, 1, "positions", [(3, 40), (0, 17)], 0, 0),
    (torch.float16, 128, 1, 128, 32, "heads", [(10, 9), (0, 2)], 0, 0),
    (torch.float16, 12, 2, 256, 16, "heads", [(0, 700)], 100, 0),
    (torch.bfloat16, 12, 2, 256, 48, "positions", [(500, 150), (0, 90)], 64, 5),
    (torch.bfloat16, 32, 8, 128, 64, "heads", [(0, 900), (2000, 77)], 256, 16),
    (torch.float16, 28, 4, 128, 16, "heads", [(0, 400), (90, 45)], 1, 1),
    (torch.float16, 8, 8, 64, 100, "positions", [(700, 333)], 129, 200),
    (torch.bfloat16, 64, 8, 64, 16, "heads", [(0, 260)], 17, 64),
]


@pytest.mark.parametrize("case", PREFILL, ids=str)
def test_prefill(paged, case):
    dtype, heads, kv_heads, dim, page, order, parts, window, sinks = case
    lengths, new = [a + b for a, b in parts], [b for _, b in parts]
    cache = build(paged, lengths, kv_heads, dim, page, dtype, order, seed=len(str(case)), stale=math.nan)
    starts = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")
    q = torch.randn(sum(new), heads, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(dtype)
    out, lse = cache.prefill(q, starts, window=window, sinks=sinks, lse=True)
    cache.check()
    row = 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        t = torch.arange(n - m, n, device="cuda")
        want, want_lse, bound, lse_bound = attend(q[row:row + m], get(cache, cache.k, 0, b, n), get(cache, cache.v, 0, b, n),
                                                  t, window, sinks, dim ** -0.5, U_ONE[dtype], U_OUT[dtype], TINY[dtype])
        near(out[row:row + m], want, bound, f"sequence {b}")
        near(lse[row:row + m], want_lse, lse_bound, f"lse {b}")
        row += m
    assert torch.equal(out, cache.prefill(q, starts, window=window, sinks=sinks))


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,past,new", [
    (torch.float16, 16, 4, 256, 0, 3001), (torch.bfloat16, 32, 8, 128, 5000, 1111), (torch.bfloat16, 8, 8, 64, 0, 2500),
    (torch.float16, 4, 1, 128, 30000, 5)])
def test_prefill_long(paged, dtype, heads, kv_heads, dim, past, new):
    cache = build(paged, [past + new], kv_heads, dim, 16, dtype)
    starts = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    q = torch.randn(new, heads, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(dtype)
    out = cache.prefill(q, starts)
    cache.check()
    n = past + new
    want, _, bound, _ = attend(q, get(cache, cache.k, 0, 0, n), get(cache, cache.v, 0, 0, n),
                               torch.arange(past, n, device="cuda"), 0, 0, dim ** -0.5, U_ONE[dtype], U_OUT[dtype],
                               TINY[dtype])
    near(out, want, bound, "rows")


def test_growing_scores(paged):
    """Scores that rise by hundreds along the sequence: the running maximum moves at every tile, in both kernels."""
    n, dim = 1500, 128
    cache = build(paged, [n], 2, dim, 16, torch.bfloat16)
    ramp = torch.linspace(0, 60, n, device="cuda")[:, None, None].expand(n, 2, dim)
    put(cache, cache.k, 0, 0, 0, ramp.bfloat16())
    q = torch.ones(n, 8, dim, device="cuda", dtype=torch.bfloat16)
    out = cache.prefill(q, torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    want, _, bound, _ = attend(q, get(cache, cache.k, 0, 0, n), get(cache, cache.v, 0, 0, n),
                               torch.arange(n, device="cuda"), 0, 0, dim ** -0.5, 2.0 ** -8, 2.0 ** -8, 1e-37)
    near(out, want, bound, "prefill")
    one = cache.decode(q[-1:])
    near(one, want[-1:], bound[-1:], "decode")


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(torch.float16, 8, 2, 128), (torch.bfloat16, 8, 2, 256),
                                                      (torch.float16, 4, 4, 256), (torch.bfloat16, 8, 4, 64)])
@pytest.mark.parametrize("top", [-400.0, 6.0, 60.0, 900.0])
def test_scores_that_move_far(paged, dtype, heads, kv_heads, dim, top):
    """Scores that rise (or fall) by `top` along the sequence, from the first position on: the reference of the
    prefill moves, the maximum of the decode moves, weights reach both ends of their range."""
    n = 700
    cache = build(paged, [n], kv_heads, dim, 32, dtype)
    size = math.sqrt(abs(top))
    ramp = torch.linspace(0, 1, n, device="cuda")[:, None, None].expand(n, kv_heads, dim) * size
    ramp = ramp + torch.randn(n, kv_heads, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(5)) * 0.01
    put(cache, cache.k, 0, 0, 0, ramp.to(dtype))
    q = torch.full((n, heads, dim), size * math.copysign(1.0, top), device="cuda").to(dtype)
    out, lse = cache.prefill(q, ints(0, n), scale=1 / dim, lse=True)
    cache.check()
    k, v = get(cache, cache.k, 0, 0, n), get(cache, cache.v, 0, 0, n)
    want, want_lse, bound, lse_bound = attend(q, k, v, torch.arange(n, device="cuda"), 0, 0, 1 / dim, U_ONE[dtype],
                                              U_OUT[dtype], TINY[dtype])
    near(out, want, bound, "prefill")
    near(lse, want_lse, lse_bound, "lse")
    near(cache.decode(q[-1:], scale=1 / dim), want[-1:], bound[-1:], "decode")


@pytest.mark.parametrize("scale", [0.0, -0.11, 1e-6, 3.0])
@pytest.mark.parametrize("dtype,dim,page", [(torch.float16, 256, 16), (torch.bfloat16, 128, 64)])
def test_prefill_scales(paged, scale, dtype, dim, page):
    parts = [(40, 100), (0, 7)]
    lengths, new = [a + b for a, b in parts], [b for _, b in parts]
    cache = build(paged, lengths, 2, dim, page, dtype)
    starts = ints(0, *np.cumsum(new))
    q = torch.randn(sum(new), 6, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(dtype)
    out = cache.prefill(q, starts, scale=scale)
    cache.check()
    row = 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        want, _, bound, _ = attend(q[row:row + m], get(cache, cache.k, 0, b, n), get(cache, cache.v, 0, b, n),
                                   torch.arange(n - m, n, device="cuda"), 0, 0, scale, U_ONE[dtype], U_OUT[dtype],
                                   TINY[dtype])
        near(out[row:row + m], want, bound, f"sequence {b}")
        row += m


@pytest.mark.parametrize("page,order", [(128, "heads"), (256, "positions"), (96, "heads"), (224, "positions"),
                                        (65536, "heads")])
@pytest.mark.parametrize("dim,window,sinks", [(64, 0, 0), (128, 100, 33), (256, 200, 7)])
def test_prefill_page_sizes(paged, page, order, dim, window, sinks):
    """Pages that hold one box, several, or more than a block, with reads that begin inside a page."""
    parts = [(300, 260), (0, 129)] if page < 65536 else [(100, 60)]
    lengths, new = [a + b for a, b in parts], [b for _, b in parts]
    cache = build(paged, lengths, 2 if page < 65536 else 1, dim, page, torch.bfloat16, order, stale=math.nan, spare=1)
    heads = 4 * cache.kv_heads
    starts = ints(0, *np.cumsum(new))
    q = torch.randn(sum(new), heads, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).bfloat16()
    out = cache.prefill(q, starts, window=window, sinks=sinks)
    cache.check()
    row = 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        want, _, bound, _ = attend(q[row:row + m], get(cache, cache.k, 0, b, n), get(cache, cache.v, 0, b, n),
                                   torch.arange(n - m, n, device="cuda"), window, sinks, dim ** -0.5, 2.0 ** -8,
                                   2.0 ** -8, 1e-37)
        near(out[row:row + m], want, bound, f"sequence {b}")
        row += m


@pytest.mark.parametrize("batch,new,past,window,sinks", [(600, 5, 60, 0, 0), (450, 90, 10, 20, 3), (2, 1, 2 ** 14, 0, 0)])
def test_prefill_many(paged, batch, new, past, window, sinks):
    """More sequences than a block has threads, and units that are cut over many blocks."""
    rng = np.random.default_rng(batch)
    parts = [(int(rng.integers(0, past + 1)) if batch > 2 else past, int(rng.integers(0, new + 1)) if batch > 2 else 1)
             for _ in range(batch)]
    lengths, news = [a + b for a, b in parts], [b for _, b in parts]
    cache = build(paged, lengths, 2, 128, 32, torch.bfloat16, seed=batch)
    starts = ints(0, *np.cumsum(news))
    q = torch.randn(sum(news), 8, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(4)).bfloat16()
    out = cache.prefill(q, starts, window=window, sinks=sinks)
    cache.check()
    for b in sorted({0, 1, batch // 2, batch - 1, int(np.argmax(lengths)), int(np.argmax(news))}):
        n, m, row = lengths[b], news[b], sum(news[:b])
        want, _, bound, _ = attend(q[row:row + m], get(cache, cache.k, 0, b, n), get(cache, cache.v, 0, b, n),
                                   torch.arange(n - m, n, device="cuda"), window, sinks, 128 ** -0.5, 2.0 ** -8,
                                   2.0 ** -8, 1e-37)
        near(out[row:row + m], want, bound, f"sequence {b}")


@pytest.mark.parametrize("layout", ["interleaved", "one head", "one page", "padded"])
def test_pool_layouts(paged, layout):
    """Views with other strides: K and V in one tensor, dimensions of extent one, rows wider than head_dim."""
    kv_heads, page, pages, dim = (1 if layout == "one head" else 2), 64, (1 if layout == "one page" else 9), 128
    if layout == "interleaved":
        both = torch.randn(2, pages, 2, page, kv_heads, dim, device="cuda").half()
        k, v = both[:, :, 0].transpose(2, 3), both[:, :, 1].transpose(2, 3)
    elif layout == "padded":
        k, v = (torch.randn(2, pages, kv_heads, page, dim + 8, device="cuda").half()[..., :dim] for _ in range(2))
    else:
        k, v = (torch.randn(2, pages, kv_heads, page, dim, device="cuda").half() for _ in range(2))
    n = min(64, pages * page) if pages == 1 else 500
    need = -(-n // page)
    table = torch.full((1, 8), -1, dtype=torch.int32, device="cuda")
    table[0, :need] = torch.randperm(pages, device="cuda")[:need].to(torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[table[0, :need].long()] = 1
    cache = paged.PagedCache(k, v, paged.PageMap(refs, table, ints(n)))
    q = torch.randn(n, 4 * kv_heads, dim, device="cuda").half()
    out = cache.prefill(q, ints(0, n), layer=1)
    cache.check()
    want, _, bound, _ = attend(q, get(cache, k, 1, 0, n), get(cache, v, 1, 0, n), torch.arange(n, device="cuda"), 0, 0,
                               128 ** -0.5, 2.0 ** -11, 2.0 ** -11, 2.0 ** -24)
    near(out, want, bound, "prefill")
    near(cache.decode(q[-1:], layer=1), want[-1:], bound[-1:], "decode")


def test_reach_past_every_length(paged):
    """Windows and sinks larger than any sequence, up to the largest number, change nothing."""
    cache = build(paged, [300], 2, 64, 16, torch.float16)
    q = torch.randn(300, 4, 64, device="cuda").half()
    plain, one = cache.prefill(q, ints(0, 300)), cache.decode(q[-1:])
    for window, sinks in ((300, 0), (2 ** 31 + 5, 2 ** 32 - 1), (2 ** 40, 1), (7, 2 ** 32 - 1), (1, 300)):
        assert torch.equal(cache.prefill(q, ints(0, 300), window=window, sinks=sinks), plain)
        assert torch.equal(cache.decode(q[-1:], window=window, sinks=sinks), one)
    with pytest.raises(ValueError):
        cache.decode(q[-1:], window=-1)


def test_bad_pages_are_read_as_zeros(paged):
    """Table entries outside the pool, where blocks come by TMA and where rows are copied: flagged, and nothing else."""
    from rta_b200._lib import RtaError
    for page in (32, 16):
        cache = build(paged, [400, 400], 2, 128, page, torch.bfloat16)
        q = torch.randn(400, 4, 128, device="cuda").bfloat16()
        good = cache.prefill(q, ints(0, 400), slots=ints(1))
        for entry in (-1, 10 ** 6, -2 ** 31, cache.pages):
            cache.map.table[0, 3] = entry
            cache.prefill(q, ints(0, 400))
            with pytest.raises(RtaError, match="word 4$"):
                cache.check()
            cache.decode(q[-1:])
            with pytest.raises(RtaError, match="word 4$"):
                cache.check()
        assert torch.equal(cache.prefill(q, ints(0, 400), slots=ints(1)), good)
        cache.check()


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,window,sinks", [
    (torch.float16, 16, 4, 256, 0, 0), (torch.bfloat16, 8, 2, 128, 0, 0), (torch.bfloat16, 8, 8, 64, 40, 3),
    (torch.float16, 8, 2, 128, 100, 0)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_is_not_seen_does_not_reach_a_row(paged, dtype, heads, kv_heads, dim, window, sinks, value):
    """Non-finite K and V rows inside the sequence: rows that do not see them are exact, the others carry them."""
    n, bad = 300, [37, 200]
    cache = build(paged, [n], kv_heads, dim, 16, dtype, stale=math.nan)
    clean_k, clean_v = get(cache, cache.k, 0, 0, n).clone(), get(cache, cache.v, 0, 0, n).clone()
    rows = clean_v.clone()
    rows[bad] = value
    put(cache, cache.v, 0, 0, 0, rows)
    q = torch.randn(n, heads, dim, device="cuda").to(dtype)
    starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    out = cache.prefill(q, starts, window=window, sinks=sinks)
    t = torch.arange(n, device="cuda")
    want, _, bound, _ = attend(q, clean_k, clean_v, t, window, sinks, dim ** -0.5, U_ONE[dtype], U_OUT[dtype],
                               TINY[dtype])
    sees = torch.zeros(n, dtype=torch.bool, device="cuda")
    for p in bad:
        sees |= (p <= t) & ((p > t - window) | (p < sinks) if window else True)
    near(out[~sees], want[~sees], bound[~sees], "rows that do not see them")
    assert not torch.isfinite(out[sees]).any()
    # the same in K: a masked score is no score
    put(cache, cache.v, 0, 0, 0, clean_v)
    rows = clean_k.clone()
    rows[bad] = math.nan
    put(cache, cache.k, 0, 0, 0, rows)
    out = cache.prefill(q, starts, window=window, sinks=sinks)
    near(out[~sees], want[~sees], bound[~sees], "rows that do not see them (K)")
    assert torch.isnan(out[sees]).all()
    last = cache.decode(q[-1:], window=window, sinks=sinks)
    assert bool(torch.isnan(last).all()) == bool(sees[-1])
    if not sees[-1]:
        near(last, want[-1:], bound[-1:], "decode")


def test_offsets_past_32_bits(paged):
    """A pool of more than 2^32 bytes (and 2^31 elements): its last pages are reached by every call."""
    page, kv_heads, dim = 64, 4, 256
    pages = (1 << 32) // (page * kv_heads * dim * 2) + 100
    cache = paged.PagedCache.create(1, pages, page, kv_heads, dim, 3, 200, torch.float16)
    table = torch.tensor([[pages - 1, 5, pages - 2, 6], [-1] * 4, [-1] * 4], dtype=torch.int32, device="cuda")
    cache.map.table.copy_(table)
    cache.map.refs[[5, 6, pages - 1, pages - 2]] = 1
    k, v = (torch.randn(200, kv_heads, dim, device="cuda") for _ in range(2))
    cache.map.lengths[0] = 200
    starts = torch.tensor([0, 200], dtype=torch.int32, device="cuda")
    cache.append(k, v, starts)
    cache.check()
    assert torch.equal(get(cache, cache.k, 0, 0, 200), k.half()) and torch.equal(get(cache, cache.v, 0, 0, 200), v.half())
    q = torch.randn(200, 16, dim, device="cuda").half()
    want, _, bound, _ = attend(q, k.half(), v.half(), torch.arange(200, device="cuda"), 0, 0, 0.0625, 2.0 ** -11,
                               2.0 ** -11, 2.0 ** -24)
    near(cache.prefill(q, starts), want, bound, "prefill")
    near(cache.decode(q[-1:]), want[-1:], bound[-1:], "decode")
    cache.fork(torch.tensor([0], dtype=torch.int32, device="cuda"), torch.tensor([2], dtype=torch.int32, device="cuda"))
    cache.free(torch.tensor([0], dtype=torch.int32, device="cuda"))
    cache.compact()
    cache.check()
    assert cache.map.table[2].max().item() < 4 and cache.map.refs[:4].tolist() == [1] * 4
    assert torch.equal(get(cache, cache.k, 0, 2, 200), k.half()) and torch.equal(get(cache, cache.v, 0, 2, 200), v.half())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kv_heads,dim,page,order,parts", [
    (4, 256, 16, "heads", [(0, 1)]), (2, 64, 7, "positions", [(5, 9), (0, 0), (14, 1), (3, 100)]),
    (8, 128, 64, "positions", [(63, 1), (64, 1), (0, 130)]), (1, 128, 1, "heads", [(2, 33), (0, 40)])])
def test_append(paged, dtype, kv_heads, dim, page, order, parts):
    lengths = [a + b for a, b in parts]
    cache = build(paged, lengths, kv_heads, dim, page, dtype, order, layers=2, slots=len(parts) + 1)
    before = cache.k.clone(), cache.v.clone()
    new = sum(b for _, b in parts)
    starts = torch.tensor([0] + list(np.cumsum([b for _, b in parts])), dtype=torch.int32, device="cuda")
    for wide in (torch.float32, dtype):
        rows = torch.randn(new, 3 * kv_heads, dim, device="cuda").to(wide)
        k, v = rows[:, :kv_heads], rows[:, 2 * kv_heads:]  # strided rows of one projection
        cache.append(k, v, starts, layer=1)
        cache.check()
        for was, pool, x in ((before[0], cache.k, k), (before[1], cache.v, v)):
            want, row = was.clone(), 0
            for s, (a, b) in enumerate(parts):
                put(cache, want, 1, s, a, x[row:row + b].to(dtype))
                row += b
            assert torch.equal(pool, want)  # those rows, rounded once, and nothing else


class Model:
    """The bookkeeping in plain Python."""

    def __init__(self, cache):
        self.page = cache.page_size
        self.refs, self.lengths = cache.map.refs.tolist(), cache.map.lengths.tolist()
        self.table = [[x for x in row if x >= 0] for row in cache.map.table.tolist()]
        self.width = cache.map.table.shape[1]

    def free_pages(self):
        return [i for i, r in enumerate(self.refs) if r == 0]

    def reserve(self, slots, counts):
        pool = self.free_pages()
        for s, c in zip(slots, counts):
            self.lengths[s] += c
            while len(self.table[s]) * self.page < self.lengths[s]:
                self.table[s].append(pool.pop(0))
                self.refs[self.table[s][-1]] = 1

    def fork(self, src, dst):
        pool = self.free_pages()
        for a, b in zip(src, dst):
            full = self.lengths[a] // self.page
            self.table[b] = self.table[a][:full]
            for p in self.table[b]:
                self.refs[p] += 1
            if self.lengths[a] % self.page:
                self.table[b].append(pool.pop(0))
                self.refs[self.table[b][-1]] = 1
            self.lengths[b] = self.lengths[a]

    def free(self, slots):
        for s in slots:
            for p in self.table[s]:
                self.refs[p] -= 1
            self.table[s], self.lengths[s] = [], 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [i for i in range(live) if not self.refs[i]]
        movers = [i for i in range(live, len(self.refs)) if self.refs[i]]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[a], self.refs[b] = 0, self.refs[a]
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return live

    def same(self, m):
        assert m.refs.tolist() == self.refs
        assert m.lengths.tolist() == self.lengths
        assert m.table.tolist() == [row + [-1] * (self.width - len(row)) for row in self.table]


@pytest.mark.parametrize("page,order,slots,pages,width", [(16, "heads", 12, 200, 20), (5, "positions", 9, 97, 30),
                                                          (1, "heads", 40, 3000, 60), (64, "positions", 30, 9001, 300)])
def test_bookkeeping_against_plain_python(paged, page, order, slots, pages, width):
    """Random calls, in place and into another map: the same map as in Python, and every sequence keeps its rows."""
    rng = np.random.default_rng(page)
    cache = paged.PagedCache.create(3, pages, page, 2, 64, slots, width * page, torch.bfloat16, order=order)
    model, held = Model(cache), {s: torch.zeros(0, 2, 64, device="cuda", dtype=torch.bfloat16) for s in range(slots)}
    other = paged.PageMap.empty(pages, slots, width)
    for step in range(40):
        kind = rng.choice(["grow", "grow", "fork", "free", "compact"])
        before = cache.map.clone()
        into = other if rng.random() < 0.5 else None
        live = [s for s in range(slots) if model.lengths[s]]
        empty = [s for s in range(slots) if not model.lengths[s]]
        if kind == "grow":
            which = [int(s) for s in rng.permutation(slots)[:rng.integers(1, slots + 1)]]
            counts = [int(min(rng.integers(0, 3 * page + 2), width * page - model.lengths[s])) for s in which]
            need = sum(-(-(model.lengths[s] + c) // page) - len(model.table[s]) for s, c in zip(which, counts))
            if need > len(model.free_pages()):
                continue
            got = cache.reserve(ints(*counts), ints(*which), out=into)
            model.reserve(which, counts)
            total = sum(counts)
            rows = torch.randn(total, 2, 64, device="cuda").bfloat16()
            starts = ints(0, *np.cumsum(counts))
            for layer in range(3):
                cache.append(rows * (layer + 1), rows * -(layer + 1), starts, layer=layer, slots=ints(*which), map=got)
            at = 0
            for s, c in zip(which, counts):
                held[s] = torch.cat([held[s], rows[at:at + c]])
                at += c
        elif kind == "fork" and live and empty:
            n = int(rng.integers(1, len(empty) + 1))
            dst = [int(s) for s in rng.permutation(empty)[:n]]
            src = [int(s) for s in rng.choice(live, n)]
            if sum(model.lengths[s] % page > 0 for s in src) > len(model.free_pages()):
                continue
            got = cache.fork(ints(*src), ints(*dst), out=into)
            model.fork(src, dst)
            for a, b in zip(src, dst):
                held[b] = held[a]
        elif kind == "free" and live:
            gone = [int(s) for s in rng.permutation(live)[:rng.integers(1, len(live) + 1)]]
            got = cache.free(ints(*gone), out=into)
            model.free(gone)
            for s in gone:
                held[s] = held[s][:0]
        elif kind == "compact":
            count = ints(-1)
            got = cache.compact(out=into, live=count)
            assert count.item() == model.compact()
        else:
            continue
        cache.check()
        model.same(got)
        if into is not None:  # the map it was read from is as it was
            for a, b in ((before.refs, cache.map.refs), (before.table, cache.map.table),
                         (before.lengths, cache.map.lengths)):
                assert torch.equal(a, b)
            for a, b in ((got.refs, cache.map.refs), (got.table, cache.map.table), (got.lengths, cache.map.lengths)):
                b.copy_(a)
        for s in range(slots):
            for layer in range(3):
                n = model.lengths[s]
                assert torch.equal(get(cache, cache.k, layer, s, n), held[s] * (layer + 1))
                assert torch.equal(get(cache, cache.v, layer, s, n), held[s] * -(layer + 1))


def test_device_checks(paged):
    """What only the device can see is flagged, changes nothing, and the cache stays usable."""
    from rta_b200._lib import RtaError

    def flagged(bits, call, *args, **kw):
        m = cache.map.clone()
        call(*args, **kw)
        with pytest.raises(RtaError, match=f"word {bits}$"):
            cache.check()
        cache.check()
        return m

    def unchanged(m):
        assert torch.equal(m.refs, cache.map.refs) and torch.equal(m.table, cache.map.table)
        assert torch.equal(m.lengths, cache.map.lengths)

    cache = paged.PagedCache.create(1, 8, 4, 1, 64, 4, 32, torch.float16)
    cache.reserve(ints(10, 5, 0))
    cache.check()
    unchanged(flagged(8, cache.reserve, ints(4, 20, 0)))          # 1 + 5 pages of 3 left
    unchanged(flagged(16, cache.reserve, ints(-1)))
    unchanged(flagged(16, cache.reserve, ints(30)))               # past the table
    unchanged(flagged(16, cache.reserve, ints(1), ints(4)))       # no such slot
    unchanged(flagged(16, cache.fork, ints(0), ints(1)))          # not empty
    unchanged(flagged(16, cache.fork, ints(0, 1), ints(2, 2)))    # one slot twice
    unchanged(flagged(16, cache.fork, ints(0, 2), ints(2, 3)))    # a source that is a destination
    unchanged(flagged(16, cache.fork, ints(0), ints(-3)))
    unchanged(flagged(16, cache.free, ints(9)))
    cache.reserve(ints(12), ints(2))
    cache.check()
    unchanged(flagged(8, cache.fork, ints(0), ints(3)))           # no page for the rest
    q = torch.randn(2, 2, 64, device="cuda").half()
    flagged(16, cache.decode, q, slots=ints(0, 7))
    flagged(16, cache.prefill, q, ints(0, 3))                     # past the rows
    flagged(16, cache.prefill, q, ints(0, 1))                     # a row that no sequence owns
    flagged(16, cache.prefill, q, ints(1, 2))
    flagged(16, cache.append, q[:, :1], q[:, :1], ints(0, 1))     # a row that no sequence owns
    table = cache.map.table.clone()
    cache.map.table[0, 1] = 99
    flagged(4, cache.decode, q[:1])
    flagged(4, cache.prefill, q[:1], ints(0, 1))
    cache.map.table.copy_(table)
    cache.map.refs[cache.map.table[1, 0].item()] = 0
    flagged(4, cache.free, ints(1))
    flagged(4, cache.copy_pages, ints(1, 9), ints(0, 1))
    n = cache.map.lengths[0].item()
    want, _, bound, _ = attend(q[:1], get(cache, cache.k, 0, 0, n), get(cache, cache.v, 0, 0, n),
                               torch.tensor([n - 1], device="cuda"), 0, 0, 0.125, 2.0 ** -20, 2.0 ** -11, 2.0 ** -24)
    near(cache.decode(q[:1]), want, bound, "after the flags")


@pytest.mark.parametrize("slots,counts", [((0, 0), (4, 4)), ((1, 2, 1), (20, 0, 20)), (tuple([2] * 1500), tuple([1] * 1500))])
def test_reserve_of_a_slot_twice(paged, slots, counts):
    """A slot named twice is flagged whatever its sums, and the call changes nothing."""
    from rta_b200._lib import RtaError
    cache = paged.PagedCache.create(1, 1600, 4, 1, 64, 1600, 32, torch.float16)
    cache.reserve(ints(10, 5, 0))
    before = cache.map.clone()
    cache.reserve(ints(*counts), ints(*slots))
    with pytest.raises(RtaError, match="word 16$"):
        cache.check()
    for a, b in ((before.refs, cache.map.refs), (before.table, cache.map.table), (before.lengths, cache.map.lengths)):
        assert torch.equal(a, b)
    cache.reserve(ints(1, 2), ints(2, 0))
    cache.check()
    assert cache.map.lengths[:4].tolist() == [12, 5, 1, 0] and cache.map.refs.sum().item() == 3 + 2 + 1


def test_rows_before_the_sequence(paged):
    """More new rows than positions: the rows before position 0 see nothing."""
    cache = build(paged, [5], 2, 128, 16, torch.bfloat16, stale=math.nan)
    q = torch.randn(9, 4, 128, device="cuda").bfloat16()
    out, lse = cache.prefill(q, ints(0, 9), lse=True)
    cache.check()
    assert (out[:4] == 0).all() and (lse[:4] == -math.inf).all()
    want, _, bound, _ = attend(q[4:], get(cache, cache.k, 0, 0, 5), get(cache, cache.v, 0, 0, 5),
                               torch.arange(5, device="cuda"), 0, 0, 128 ** -0.5, 2.0 ** -8, 2.0 ** -8, 1e-37)
    near(out[4:], want, bound, "rows")


def test_copy_pages(paged):
    cache = paged.PagedCache.create(2, 20, 6, 3, 64, 1, 6, torch.float16, order="positions")
    for pool in (cache.k, cache.v):
        pool.copy_(torch.randn(pool.shape, device="cuda"))
    k, v = cache.k.clone(), cache.v.clone()
    cache.copy_pages(ints(3, 3, 19), ints(0, 7, 1))
    cache.check()
    for pool, was in ((cache.k, k), (cache.v, v)):
        was[:, [0, 7, 1]] = was[:, [3, 3, 19]]
        assert torch.equal(pool, was)


def test_side_stream_and_graph(paged):
    """A serving step -- grow, write, attend -- captured once as a CUDA graph on a stream of its own, replayed."""
    steps, slots = 40, 5
    cache = build(paged, [30, 7, 0, 100, 15], 2, 128, 16, torch.bfloat16, spare=40)
    wide = paged.PageMap(cache.map.refs, torch.full((slots, 16), -1, dtype=torch.int32, device="cuda"),
                         cache.map.lengths)
    wide.table[:, :cache.map.table.shape[1]] = cache.map.table
    cache = paged.PagedCache(cache.k, cache.v, wide)
    k, v = (torch.zeros(slots, 2, 128, device="cuda") for _ in range(2))
    q, out = (torch.zeros(slots, 8, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    ones, starts = ints(*[1] * slots), ints(*range(slots + 1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        cache.reserve(ones)
        cache.append(k, v, starts)
        cache.decode(q, window=50, sinks=2, out=out)

    with torch.cuda.stream(side):
        step()  # first calls set kernels up
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for _ in range(steps):
            k.normal_(), v.normal_(), q.normal_()
            graph.replay()
        cache.check()
    torch.cuda.current_stream().wait_stream(side)
    for b, n in enumerate([30, 7, 0, 100, 15]):
        n += steps + 1
        assert cache.map.lengths[b].item() == n
        want, _, bound, _ = attend(q[b:b + 1], get(cache, cache.k, 0, b, n), get(cache, cache.v, 0, b, n),
                                   torch.tensor([n - 1], device="cuda"), 50, 2, 128 ** -0.5, 2.0 ** -16, 2.0 ** -8, 1e-37)
        near(out[b:b + 1], want, bound, f"sequence {b}")


def test_refusals(paged):
    from rta_b200._lib import RtaError
    cache = paged.PagedCache.create(2, 8, 16, 2, 64, 3, 64, torch.float16)
    q = torch.zeros(3, 4, 64, device="cuda", dtype=torch.float16)
    one = ints(0, 3)
    for call in (lambda: cache.decode(q.bfloat16()), lambda: cache.decode(q, layer=2),
                 lambda: cache.decode(torch.zeros(4, 4, 64, device="cuda", dtype=torch.float16)),
                 lambda: cache.decode(torch.zeros(3, 3, 64, device="cuda", dtype=torch.float16)),
                 lambda: cache.decode(q, scale=math.nan), lambda: cache.prefill(q.float(), one),
                 lambda: cache.decode(torch.zeros(3, 4, 68, device="cuda", dtype=torch.float16)[:, :, 4:]),
                 lambda: cache.append(q[:, :2].bfloat16(), q[:, :2].bfloat16(), one), lambda: cache.reserve(ints()),
                 lambda: cache.reserve(ints(1, 1, 1, 1)), lambda: cache.fork(ints(), ints()),
                 lambda: cache.copy_pages(ints(*[0] * 9), ints(*range(9)))):
        with pytest.raises(RtaError, match="rta_page"):
            call()
    for call in (lambda: cache.decode(q.cpu()), lambda: cache.decode(q[:, :, :32]), lambda: cache.decode(q.double()),
                 lambda: cache.decode(q, slots=ints(0)), lambda: cache.decode(q, slots=torch.zeros(3, device="cuda")),
                 lambda: cache.decode(q, out=torch.zeros(3, 4, 64, device="cuda")),
                 lambda: cache.prefill(q, one.long()), lambda: cache.append(q, q, one),
                 lambda: cache.append(q[:, :2], q[:2, :2], one), lambda: cache.fork(ints(0), ints(1, 2)),
                 lambda: cache.free(ints(0), out=paged.PageMap.empty(7, 3, 4)),
                 lambda: paged.PagedCache(cache.k, cache.v.transpose(2, 3), cache.map),
                 lambda: paged.PagedCache(cache.k, cache.v, paged.PageMap.empty(9, 3, 4)),
                 lambda: paged.PagedCache.create(1, 4, 16, 1, 96, 1, 16),
                 lambda: paged.PageMap(cache.map.refs, cache.map.table, cache.map.lengths[:2])):
        with pytest.raises(ValueError):
            call()
    assert cache.decode(q[:0]).shape == (0, 4, 64)  # nothing to do


@pytest.mark.parametrize("prompt,samples,tokens", [(700, 6, 24), (33, 3, 40), (256, 2, 5)])
def test_serving_example(paged, prompt, samples, tokens):
    """Prefill in chunks, fork, decode as a graph, free, compact, decode on: the states of the model without a cache.
    bf16 activations through three layers: each rounds to 2^-9, and so do its projections, its weights and its result,
    about ten roundings a layer that add up like independent ones: 2^-9 sqrt(30) = 1.1e-2; 3e-2 is asked for."""
    from rta_b200.examples.paged_serving import serve
    said, worst, live, used, pages = serve(prompt, samples, tokens)
    assert said.shape == (samples - samples // 2, 2 * tokens)
    assert worst < 3e-2
    assert live <= used <= pages
