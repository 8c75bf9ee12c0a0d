"""GPU tests: a bookkeeping call of the paged cache that finds something wrong changes nothing."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_paged_gpu import Model, ints  # noqa: E402


@pytest.fixture(scope="module")
def paged():
    from rta_b200 import paged as module
    torch.cuda.init()
    return module


def flagged(cache, bits, call):
    """The call raises `bits` and leaves the map and the pools as they were; so it does into another map."""
    from rta_b200._lib import RtaError
    before, k, v = cache.map.clone(), cache.k.clone(), cache.v.clone()
    other = cache.map.clone()
    other.table.fill_(77)
    for into in (None, other):
        got = call(into)
        with pytest.raises(RtaError, match=f"word {bits}$"):
            cache.check()
        for m in {cache.map, got}:
            assert torch.equal(m.refs, before.refs) and torch.equal(m.table, before.table)
            assert torch.equal(m.lengths, before.lengths)
        assert torch.equal(cache.k, k) and torch.equal(cache.v, v)


def small(paged, lengths=(10, 5, 8, 0, 0), pages=12, layers=2, slots=None, width=8):
    """Pages of four positions, each filled with its own number."""
    cache = paged.PagedCache.create(layers, pages, 4, 1, 64, slots or len(lengths), 4 * width, torch.float16)
    for pool, sign in ((cache.k, 1), (cache.v, -1)):
        pool.copy_((torch.arange(pages, device="cuda") * sign).view(1, -1, 1, 1, 1).expand_as(pool))
    cache.reserve(ints(*lengths))
    cache.check()
    return cache


@pytest.mark.parametrize("slots", [(0, 9), (9, 0), (0, 1, -1), (2, 5, 0, 1), (1, 2 ** 31 - 1)])
def test_free_with_a_bad_slot_frees_none(paged, slots):
    cache = small(paged)
    flagged(cache, 16, lambda out: cache.free(ints(*slots), out=out))
    model = Model(cache)
    cache.free(ints(0, 1))
    model.free([0, 1])
    cache.check()
    model.same(cache.map)


@pytest.mark.parametrize("length", [-1, -2 ** 31, 33, 2 ** 31 - 1])
def test_free_with_a_bad_length_frees_none(paged, length):
    cache = small(paged)
    cache.map.lengths[1] = length
    flagged(cache, 16, lambda out: cache.free(ints(0, 1, 2), out=out))
    flagged(cache, 16, lambda out: cache.free(ints(1), out=out))


def test_free_of_many(paged):
    """More slots than a block has threads, and than blocks are launched; one bad one among them, then none."""
    slots, pages = 3000, 3100
    cache = paged.PagedCache.create(1, pages, 4, 1, 64, slots, 8, torch.float16)
    cache.reserve(ints(*[1 + i % 4 if i % 5 else 0 for i in range(slots)]))
    cache.check()
    for bad in (0, 1700, slots - 1):
        which = list(range(slots))
        which[bad] = slots
        flagged(cache, 16, lambda out: cache.free(ints(*which), out=out))
    model = Model(cache)
    which = list(range(0, slots, 2)) + [4, 6]  # named twice: freed once
    cache.free(ints(*which))
    model.free(which)
    cache.check()
    model.same(cache.map)


@pytest.mark.parametrize("entry", [-1, 12, 10 ** 6, -2 ** 31])
@pytest.mark.parametrize("where", [0, 1])
def test_fork_of_a_bad_page_changes_nothing(paged, entry, where):
    """A full page of the source that is no page of the pool."""
    cache = small(paged)
    cache.map.table[0, where] = entry
    flagged(cache, 4, lambda out: cache.fork(ints(1, 0), ints(3, 4), out=out))


@pytest.mark.parametrize("j", [0, 1, 2])
def test_fork_of_a_free_page_changes_nothing(paged, j):
    """A page of the source, full or the last, that nothing refers to: it could be handed out by the same call."""
    cache = small(paged)
    cache.map.refs[cache.map.table[0, j].item()] = 0
    flagged(cache, 4, lambda out: cache.fork(ints(1, 0), ints(3, 4), out=out))


def test_fork_of_long_tables(paged):
    """More full pages than the plan reads at a time; one bad one far along."""
    cache = paged.PagedCache.create(1, 5000, 1, 1, 64, 4, 4000, torch.float16)
    cache.reserve(ints(3900, 1000))
    cache.check()
    was = cache.map.table[0, 3700].item()
    cache.map.table[0, 3700] = -5
    flagged(cache, 4, lambda out: cache.fork(ints(1, 0), ints(2, 3), out=out))
    cache.map.table[0, 3700] = was
    model = Model(cache)
    cache.fork(ints(1, 0, ), ints(2, 3))
    model.fork([1, 0], [2, 3])
    cache.check()
    model.same(cache.map)


def holes(paged, **kw):
    """Slots 0 and 2 hold pages behind free ones: compact has something to move."""
    cache = small(paged, **kw)
    cache.free(ints(1))
    cache.check()
    return cache


@pytest.mark.parametrize("entry,bits", [(99, 4), (12, 4), (3, 4), (7, 4), (11, 4)])
@pytest.mark.parametrize("width", [8, 9000])
def test_compact_of_a_bad_entry_changes_nothing(paged, entry, bits, width):
    """Table entries past the pool, of the hole that another page would move to (3, 4 and the pages from 7 on are free
    once slot 1 is gone), and of a free page behind the live ones; maps that one block copies and larger ones."""
    cache = holes(paged, width=width)
    assert cache.map.refs.tolist() == [1, 1, 1, 0, 0, 1, 1, 0, 0, 0, 0, 0]
    cache.map.table[3, 1] = entry
    flagged(cache, bits, lambda out: cache.compact(out=out))
    cache.map.table[3, 1] = -1
    model = Model(cache)
    assert model.compact() == 5
    cache.compact()
    cache.check()
    model.same(cache.map)
    assert cache.k[0, :5, 0, 0, 0].tolist() == [0, 1, 2, 5, 6]


def test_compact_flagged_tells_no_count(paged):
    """The count of a call that changes nothing is the count of pages in use all the same."""
    from rta_b200._lib import RtaError
    cache, live = holes(paged), ints(-7)
    cache.map.table[3, 1] = 4
    cache.compact(live=live)
    with pytest.raises(RtaError, match="word 4$"):
        cache.check()
    assert live.item() == 5


@pytest.mark.parametrize("src,dst", [((1, 12), (0, 3)), ((-1, 1), (0, 3)), ((1, 2), (12, 3)), ((1, 2), (3, -1))])
def test_copy_with_a_bad_page_copies_none(paged, src, dst):
    cache = small(paged)
    flagged(cache, 4, lambda out: cache.copy_pages(ints(*src), ints(*dst)) or cache.map)
