"""GPU tests of the paged attentions at the ends of their numbers, against 64 bits.

The bound is the one of test_paged_gpu.py -- |out - exact| <= A (2e + 2 u_w + 2^-20 + n 2^-28) + |exact| u_o -- where a
weight keeps its relative rounding u_w as long as it is not far below the largest of the positions that are weighed
together: 128 in the prefill, whose fp16 weights are multiples of 2^-32 of that largest one, 16 in the decode, whose
fp16 pairs are multiples of 2^-39 of it.  A rounding is a quarter of a multiple in the mean, so positions 2^-34 or 2^-41
max |v| are added.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_paged_gpu import TINY, U_ONE, U_OUT, U_PAIR, attend, build, get, ints, near, put  # noqa: E402


@pytest.fixture(scope="module")
def paged():
    from rta_b200 import paged as module
    torch.cuda.init()
    return module


def sink(paged, dtype, n, kv_heads, dim, gap, spread, seed=0):
    """A cache of one sequence whose position 0 scores `gap` above the others (they spread around 0) and holds zeros,
    and a query row for it; scale 1."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = build(paged, [n], kv_heads, dim, 16, dtype, seed=seed)
    k = torch.zeros(n, kv_heads, dim, device="cuda")
    k[:, :, 1] = torch.randn(n, kv_heads, device="cuda", generator=g) * spread
    k[0] = 0
    k[0, :, 0] = gap
    v = torch.randn(n, kv_heads, dim, device="cuda", generator=g) + 8
    v[0] = 0
    put(cache, cache.k, 0, 0, 0, k.to(dtype))
    put(cache, cache.v, 0, 0, 0, v.to(dtype))
    q = torch.zeros(dim, device="cuda")
    q[:2] = 1
    return cache, q


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(torch.float16, 8, 2, 128), (torch.float16, 4, 1, 256),
                                                      (torch.float16, 4, 4, 64), (torch.bfloat16, 8, 2, 128)])
@pytest.mark.parametrize("n", [120, 3000, 20000])
@pytest.mark.parametrize("gap,spread", [(10.0, 0.5), (15.0, 0.0), (16.5, 0.5), (18.0, 0.0), (21.0, 1.0), (25.0, 0.0)])
def test_prefill_behind_a_sink(paged, dtype, heads, kv_heads, dim, n, gap, spread):
    """A first position that takes nearly all the weight and holds zeros: the result is what all the others add up to."""
    cache, one = sink(paged, dtype, n, kv_heads, dim, gap, spread)
    rows = min(n, 150)
    q = one.to(dtype).expand(rows, heads, dim).contiguous()
    out, lse = cache.prefill(q, ints(0, rows), scale=1.0, lse=True)
    cache.check()
    k, v = get(cache, cache.k, 0, 0, n), get(cache, cache.v, 0, 0, n)
    want, want_lse, bound, lse_bound = attend(q, k, v, torch.arange(n - rows, n, device="cuda"), 0, 0, 1.0,
                                              U_ONE[dtype], U_OUT[dtype], TINY[dtype])
    held = 128 * 2.0 ** -34 * v.abs().max().item()
    near(out, want, bound + held, "rows")
    near(lse, want_lse, lse_bound, "lse")


def test_prefill_of_sinks_along_the_way(paged):
    """Positions of far larger scores now and then, with a window that loses sight of them: references rise and fall."""
    n, dtype, dim = 2600, torch.float16, 128
    cache, one = sink(paged, dtype, n, 2, dim, 14.0, 1.0)
    k, v = get(cache, cache.k, 0, 0, n), get(cache, cache.v, 0, 0, n)
    k[700::611, :, 0], v[700::611] = 17.0, 0.0
    put(cache, cache.k, 0, 0, 0, k)
    put(cache, cache.v, 0, 0, 0, v)
    q = one.to(dtype).expand(n, 8, dim).contiguous()
    for window, sinks in ((0, 0), (300, 2), (150, 0)):
        out, lse = cache.prefill(q, ints(0, n), window=window, sinks=sinks, scale=1.0, lse=True)
        cache.check()
        want, want_lse, bound, lse_bound = attend(q, k, v, torch.arange(n, device="cuda"), window, sinks, 1.0,
                                                  U_ONE[dtype], U_OUT[dtype], TINY[dtype])
        # each position of a large score is weighed with the others of its block
        near(out, want, bound + 128 * 2.0 ** -34 * v.abs().max().item() * 5, f"window {window}")
        near(lse, want_lse, lse_bound, f"window {window}, lse")


@pytest.mark.parametrize("q32,heads,kv_heads,dim", [(True, 8, 2, 128), (True, 16, 4, 256), (False, 24, 2, 64),
                                                    (False, 4, 4, 256)])
@pytest.mark.parametrize("n", [20, 3000, 20000])
@pytest.mark.parametrize("gap,spread", [(10.0, 0.5), (14.3, 0.0), (16.3, 0.0), (17.1, 0.0), (18.0, 0.5), (21.2, 0.0),
                                        (25.0, 1.0)])
def test_decode_behind_a_sink(paged, q32, heads, kv_heads, dim, n, gap, spread):
    """The same for one token, whose weights enter as pairs."""
    cache, one = sink(paged, torch.float16, n, kv_heads, dim, gap, spread)
    dtype = torch.float32 if q32 else torch.float16
    q = one.to(dtype).expand(1, heads, dim).contiguous()
    out, lse = cache.decode(q, scale=1.0, lse=True)
    cache.check()
    k, v = get(cache, cache.k, 0, 0, n), get(cache, cache.v, 0, 0, n)
    want, want_lse, bound, lse_bound = attend(q, k, v, torch.tensor([n - 1], device="cuda"), 0, 0, 1.0,
                                              U_PAIR[torch.float16], U_OUT[dtype], TINY[dtype])
    near(out, want, bound + 16 * 2.0 ** -41 * v.abs().max().item(), "token")
    near(lse, want_lse, lse_bound, "lse")


def test_decode_of_scores_that_jump(paged):
    """Large scores at some positions, small ones between them, both with values: maxima rise and fall tile by tile."""
    n, dim = 4000, 128
    cache = build(paged, [n], 2, dim, 16, torch.float16)
    k = torch.zeros(n, 2, dim, device="cuda")
    k[:, :, 0] = torch.randn(n, 2, device="cuda", generator=torch.Generator("cuda").manual_seed(7)) * 12
    put(cache, cache.k, 0, 0, 0, k.half())
    q = torch.zeros(1, 16, dim, device="cuda")
    q[:, :, 0] = 1
    out, lse = cache.decode(q, scale=1.0, lse=True)
    want, want_lse, bound, lse_bound = attend(q, get(cache, cache.k, 0, 0, n), get(cache, cache.v, 0, 0, n),
                                              torch.tensor([n - 1], device="cuda"), 0, 0, 1.0, U_PAIR[torch.float16],
                                              U_OUT[torch.float32], TINY[torch.float32])
    near(out, want, bound, "token")
    near(lse, want_lse, lse_bound, "lse")


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 4, 256), (6, 2, 128), (24, 2, 64)])
@pytest.mark.parametrize("size", [1e-35, 1e-20, 1e-6, 2.0 ** -7, 1.0, 1e4, 7e4, 1e6, 1e30])
def test_decode_queries_of_any_size(paged, heads, kv_heads, dim, size):
    """fp32 queries past both ends of fp16's range, the scale making up for it; each head of another size."""
    lengths = [700, 3]
    cache = build(paged, lengths, kv_heads, dim, 16, torch.float16)
    q = torch.randn(2, heads, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) * size
    q[:, ::2] *= 2.0 ** -9  # smaller by another factor, exactly
    q[1, 1] = 0
    scale = dim ** -0.5 / size
    out = cache.decode(q, scale=scale)
    cache.check()
    for b, n in enumerate(lengths):
        want, _, bound, _ = attend(q[b:b + 1], get(cache, cache.k, 0, b, n), get(cache, cache.v, 0, b, n),
                                   torch.tensor([n - 1], device="cuda"), 0, 0, scale, U_PAIR[torch.float16],
                                   U_OUT[torch.float32], 1e-37)
        near(out[b:b + 1], want, bound, f"sequence {b}")


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 1, 256), (40, 2, 64)])
@pytest.mark.parametrize("top", [0.0, 12.0, 35.0, 80.0])
def test_values_near_the_largest(paged, heads, kv_heads, dim, top):
    """bf16 values of 3e38 and scores that rise by `top`: the mean of finite values is finite."""
    n, dtype = 900, torch.bfloat16
    cache = build(paged, [n], kv_heads, dim, 32, dtype)
    k = torch.zeros(n, kv_heads, dim, device="cuda")
    k[:, :, 0] = torch.linspace(0, top, n, device="cuda")[:, None]
    put(cache, cache.k, 0, 0, 0, k.to(dtype))
    put(cache, cache.v, 0, 0, 0, torch.full((n, kv_heads, dim), 3e38, device="cuda").to(dtype))
    q = torch.zeros(n, heads, dim, device="cuda", dtype=dtype)
    q[:, :, 0] = 1
    out, lse = cache.prefill(q, ints(0, n), scale=1.0, lse=True)
    cache.check()
    want, want_lse, bound, lse_bound = attend(q, get(cache, cache.k, 0, 0, n), get(cache, cache.v, 0, 0, n),
                                              torch.arange(n, device="cuda"), 0, 0, 1.0, U_ONE[dtype], U_OUT[dtype],
                                              TINY[dtype])
    near(out, want, bound, "prefill")
    near(lse, want_lse, lse_bound, "lse")
    one, lse = cache.decode(q[-1:], scale=1.0, lse=True)
    near(one, want[-1:], bound[-1:], "decode")
    near(lse, want_lse[-1:], lse_bound[-1:], "lse of decode")


def test_values_near_the_largest_beside_nan(paged):
    """The same for rows that are computed by themselves: the last position, which they do not see, holds NaN."""
    n, dtype, dim = 300, torch.bfloat16, 128
    cache = build(paged, [n], 2, dim, 32, dtype)
    v = torch.full((n, 2, dim), 3e38, device="cuda").to(dtype)
    put(cache, cache.v, 0, 0, 0, v)
    q = torch.randn(n, 8, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(dtype)
    put(cache, cache.v, 0, 0, n - 1, torch.full((1, 2, dim), math.nan, device="cuda", dtype=dtype))
    out, lse = cache.prefill(q, ints(0, n), lse=True)
    cache.check()
    want, want_lse, bound, lse_bound = attend(q, get(cache, cache.k, 0, 0, n), v, torch.arange(n, device="cuda"), 0, 0,
                                              dim ** -0.5, U_ONE[dtype], U_OUT[dtype], TINY[dtype])
    near(out[:-1], want[:-1], bound[:-1], "rows")
    near(lse, want_lse, lse_bound, "lse")
    assert torch.isnan(out[-1]).all()


def test_a_scale_of_zero_weighs_all_alike(paged):
    """Products of 1e32 times a scale of zero are zero."""
    n, dim, dtype = 200, 64, torch.bfloat16
    cache = build(paged, [n], 2, dim, 32, dtype)
    put(cache, cache.k, 0, 0, 0, (torch.randn(n, 2, dim, device="cuda") * 1e16).to(dtype))
    q = (torch.randn(n, 4, dim, device="cuda") * 1e16).to(dtype)
    out = cache.prefill(q, ints(0, n), scale=0.0)
    cache.check()
    want, _, bound, _ = attend(q, get(cache, cache.k, 0, 0, n), get(cache, cache.v, 0, 0, n),
                               torch.arange(n, device="cuda"), 0, 0, 0.0, U_ONE[dtype], U_OUT[dtype], TINY[dtype])
    near(out, want, bound, "rows")
