"""GPU tests of batches whose sequences with anything to do lie far apart."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_paged_gpu import U_ONE, U_OUT, U_PAIR, attend, get, ints, near  # noqa: E402


@pytest.mark.parametrize("batch,active", [(40, (0, 39)), (97, (3, 35, 36, 96)), (5000, (0, 31, 32, 2500, 4999)),
                                          (1500000, (1, 1499999))])
def test_sequences_far_apart(batch, active):
    """The blocks of an attention go from one sequence to the next over all that have nothing: 1.5 million of them must
    not run out the waits of those who wait meanwhile."""
    from rta_b200.paged import PagedCache
    heads, kv_heads, dim, dtype = 4, 2, 64, torch.bfloat16
    cache = PagedCache.create(1, 20 * len(active), 16, kv_heads, dim, batch, 320, dtype)
    counts = torch.zeros(batch, dtype=torch.int32, device="cuda")
    lengths = [300 - 7 * i for i in range(len(active))]
    counts[list(active)] = ints(*lengths)
    cache.reserve(counts)
    starts = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
    starts[1:] = counts.cumsum(0)
    k, v, q = (torch.randn(sum(lengths), h, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(h)).to(dtype)
               for h in (kv_heads, kv_heads, heads))
    cache.append(k, v, starts)
    out = cache.prefill(q, starts)
    tokens = torch.zeros(batch, heads, dim, device="cuda", dtype=dtype)
    ends = torch.tensor(lengths, device="cuda").cumsum(0) - 1
    tokens[list(active)] = q[ends]
    one = cache.decode(tokens)
    cache.check()
    row = 0
    for s, n in zip(active, lengths):
        kk, vv = get(cache, cache.k, 0, s, n), get(cache, cache.v, 0, s, n)
        want, _, bound, _ = attend(q[row:row + n], kk, vv, torch.arange(n, device="cuda"), 0, 0, 0.125, U_ONE[dtype],
                                   U_OUT[dtype], 1e-37)
        near(out[row:row + n], want, bound, f"prefill {s}")
        want, _, bound, _ = attend(q[row + n - 1:row + n], kk, vv, torch.tensor([n - 1], device="cuda"), 0, 0, 0.125,
                                   U_PAIR[dtype], U_OUT[dtype], 1e-37)
        near(one[s:s + 1], want, bound, f"decode {s}")
        row += n
    one[list(active)] = 0
    assert not one.any()


def test_a_bad_slot_gives_zeros():
    """Sequences of a slot that is none are flagged and see nothing; the others are as they were."""
    from rta_b200._lib import RtaError
    from rta_b200.paged import PagedCache
    cache = PagedCache.create(1, 8, 16, 2, 64, 3, 32, torch.float16)
    cache.reserve(ints(20, 7, 0))
    k = torch.randn(27, 2, 64, device="cuda").half()
    cache.append(k, k * 2, ints(0, 20, 27, 27))
    q = torch.randn(9, 4, 64, device="cuda").half()
    starts, slots = ints(0, 3, 5, 9), ints(0, 3, 1)
    good, good_lse = cache.prefill(q[[0, 1, 2, 5, 6, 7, 8]], ints(0, 3, 7), slots=ints(0, 1), lse=True)
    one, one_lse = cache.decode(q[:2], slots=ints(0, 1), lse=True)
    cache.check()
    for bad in (3, -1):
        slots[1] = bad
        out, lse = cache.prefill(q, starts, slots=slots, out=torch.full_like(q, 7), lse=True)
        with pytest.raises(RtaError, match="word 16$"):
            cache.check()
        assert torch.equal(out[[0, 1, 2, 5, 6, 7, 8]], good) and torch.equal(lse[[0, 1, 2, 5, 6, 7, 8]], good_lse)
        assert not out[3:5].any() and (lse[3:5] == -torch.inf).all()
        out, lse = cache.decode(q[[0, 4, 1]], slots=slots, out=torch.full_like(q[:3], 7), lse=True)
        with pytest.raises(RtaError, match="word 16$"):
            cache.check()
        assert torch.equal(out[[0, 2]], one) and torch.equal(lse[[0, 2]], one_lse)
        assert not out[1].any() and (lse[1] == -torch.inf).all()
