"""GPU tests of prefill rows beside non-finite values that they do not see, in units that one block computes whole."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_paged_gpu import TINY, U_ONE, U_OUT, attend, build, get, ints, near, put  # noqa: E402


@pytest.fixture(scope="module")
def paged():
    from rta_b200 import paged as module
    torch.cuda.init()
    return module


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,window,sinks", [
    (torch.float16, 8, 1, 64, 0, 0), (torch.bfloat16, 6, 2, 128, 0, 0), (torch.float16, 8, 2, 256, 0, 0),
    (torch.bfloat16, 4, 4, 64, 9, 2), (torch.float16, 8, 1, 128, 30, 0)])
def test_short_sequences(paged, dtype, heads, kv_heads, dim, window, sinks):
    """Hundreds of sequences, several to a block; the last position of every third one holds a non-finite value."""
    rng = np.random.default_rng(dim)
    news = [int(x) for x in rng.integers(0, 40, 500)]
    lengths = [m + int(x) for m, x in zip(news, rng.integers(0, 60, 500))]
    cache = build(paged, lengths, kv_heads, dim, 16, dtype, seed=dim)
    clean = {}
    for b in range(0, 500, 3):
        if lengths[b]:
            clean[b] = get(cache, cache.v, 0, b, lengths[b]).clone()
            value = [math.nan, math.inf, -math.inf][b // 3 % 3]
            put(cache, cache.v, 0, b, lengths[b] - 1, torch.full_like(clean[b][:1], value))
    q = torch.randn(sum(news), heads, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(dtype)
    starts = ints(0, *np.cumsum(news))
    out, lse = cache.prefill(q, starts, window=window, sinks=sinks, lse=True)
    cache.check()
    row = 0
    for b, (n, m) in enumerate(zip(lengths, news)):
        hit = b in clean and m > 0
        if b < 60 or b > 440 or hit and b % 5 == 0:
            v = clean[b] if b in clean else get(cache, cache.v, 0, b, n)
            want, want_lse, bound, lse_bound = attend(q[row:row + m], get(cache, cache.k, 0, b, n), v,
                                                      torch.arange(n - m, n, device="cuda"), window, sinks, dim ** -0.5,
                                                      U_ONE[dtype], U_OUT[dtype], TINY[dtype])
            good = m - 1 if hit else m
            near(out[row:row + good], want[:good], bound[:good], f"sequence {b}")
            near(lse[row:row + good], want_lse[:good], lse_bound[:good], f"lse {b}")
        if hit:
            assert not torch.isfinite(out[row + m - 1]).any()
        row += m
    bits = out.view(torch.int16)  # (NaN is not equal to itself)
    assert torch.equal(bits, cache.prefill(q, starts, window=window, sinks=sinks).view(torch.int16))


def test_long_histories(paged):
    """As many sequences as there are blocks, of one long history, so that each is computed whole: rows that do not see
    the last position go over all of it by themselves, and no other part of the block waits for them."""
    n, new, heads, dim, dtype = 120000, 16, 8, 64, torch.float16
    batch = torch.cuda.get_device_properties(0).multi_processor_count
    one = build(paged, [n], 1, dim, 16, dtype)
    clean = get(one, one.v, 0, 0, n).clone()
    put(one, one.v, 0, 0, n - 1, torch.full_like(clean[:1], math.nan))
    cache = paged.PagedCache(one.k, one.v, paged.PageMap(one.map.refs, one.map.table.repeat(batch, 1),
                                                         ints(*[n] * batch)))
    q = torch.randn(batch * new, heads, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(dtype)
    out = cache.prefill(q, ints(*range(0, batch * new + 1, new)))
    cache.check()
    for b in (0, 1, batch // 2, batch - 1):
        rows = slice(b * new, b * new + new - 1)
        want, _, bound, _ = attend(q[rows], get(one, one.k, 0, 0, n), clean, torch.arange(n - new, n - 1, device="cuda"),
                                   0, 0, dim ** -0.5, U_ONE[dtype], U_OUT[dtype], TINY[dtype])
        near(out[rows], want, bound, f"sequence {b}")
    last = out.view(batch, new, heads, dim)
    assert torch.isnan(last[:, -1]).all() and torch.isfinite(last[:, :-1]).all()
