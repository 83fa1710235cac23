"""Calls over a paged KV cache at its edges."""
import numpy as np
import pytest

from test_gpu_paged import NONE, be, floats, u32  # noqa: F401  (be: the module's backend)

pytestmark = pytest.mark.gpu


def test_more_key_blocks_than_the_line_of_work_counts(be):
    """2^31 key blocks and more (here one page under every table entry): OutOfRange, and nothing is computed for any request."""
    from ojas_b200 import DType, OjasError
    page, width = 1 << 24, 127
    places = width * page
    for kind, d, batch, heads, tokens in ((DType.F32, 32, 128, 1, 1), (DType.BF16, 32, 300, 1, 1), (DType.BF16, 64, 2, 1, 40000), (DType.BF16, 64, 3, 1, 3000)):
        pages = be.zeros((1, page, 1, d), kind)
        new = np.full(batch, tokens)
        cached = places - new - 5
        if batch == 3:
            cached[:2] = 100                                                   # others next to one request that is too long by itself
            new[2], heads = 40000, 1
            cached[2] = places - 40001
        n = int(new.sum())
        q, out = be.zeros((n, heads, d), kind), floats(be, np.full((n, heads, d), 7.0, np.float32), kind == DType.BF16)
        lse = be.upload(np.full((n, heads), 7.0, np.float32))
        be.paged_attention_forward(q, pages, pages, u32(be, np.zeros((batch, width))), u32(be, cached), u32(be, np.concatenate([[0], np.cumsum(new)])), out=out, lse=lse)
        with pytest.raises(OjasError) as e:
            be.sync()
        assert e.value.kind == "OutOfRange"
        assert np.all(out.numpy() == 7.0) and np.all(lse.numpy() == 7.0)
        del pages


def held_plan(cached, new, held, free, head, tables, page):
    """(slots, head, held) and the tables of one pass in which request b holds the first held[b] entries of its row."""
    slots, tables, held = [], tables.copy(), list(held)
    for b, (c, n) in enumerate(zip(cached, new)):
        while held[b] < -(-(c + n) // page):
            tables[b, held[b]] = free[head]
            held[b], head = held[b] + 1, head + 1
        slots += [int(tables[b, p // page]) * page + p % page for p in range(c, c + n)]
    return slots, head, held, tables


@pytest.mark.parametrize("page", [1, 3, 4, 16])
@pytest.mark.parametrize("batch", [1, 7, 300])
def test_pages_of_rejected_drafts_stay_with_their_request(be, page, batch):
    """Forty passes of trees of which a path is kept, from a pool that holds the kept places and one tree to a request: it never runs out, and no page has two holders."""
    rng = np.random.default_rng(page + batch)
    most, passes = 12, 40
    new = [[int(x) for x in rng.integers(0, most + 1, batch)] for _ in range(passes)]
    kept = [[int(rng.integers(0, n + 1)) if rng.random() < 0.6 else min(n, 1) for n in row] for row in new]
    ends = np.sum(kept, 0) + most
    width = int(-(-ends.max() // page))
    free = rng.permutation(int((-(-ends // page)).sum()))
    tables, head, held, cached = np.full((batch, width), 0xABCD, np.int64), 0, [0] * batch, np.zeros(batch, np.int64)
    d_free, d_head, d_held, d_tables = u32(be, free), u32(be, [0]), u32(be, held), u32(be, tables)
    for row, keep in zip(new, kept):
        n = sum(row) + 2
        want, head, held, tables = held_plan(cached, row, held, free, head, tables, page)
        got = be.paged_plan(u32(be, cached), u32(be, row), d_free, d_head, d_tables, page, tokens=n, held_pages=d_held)
        assert list(got.slots.numpy()) == want + [NONE] * 2 and list(got.held_pages.numpy()) == held and got.free_head.numpy()[0] == head
        d_head, d_held = got.free_head, got.held_pages
        cached += keep
    be.sync()
    assert np.array_equal(d_tables.numpy(), tables) and head <= len(free)
    owned = [int(p) for b in range(batch) for p in tables[b, : held[b]]]
    assert sorted(owned + [int(p) for p in free[head:]]) == list(range(len(free)))


@pytest.mark.parametrize("what,kind,held_after", [("too few held", "OutOfRange", [2, 1]), ("too many held", "OutOfRange", [9, 1]), ("free", "CapacityExceeded", [3, 0]), ("tokens", "OutOfRange", [3, 1]),
                                                  ("width", "OutOfRange", [2, 1])])
def test_held_pages_are_those_that_were_entered(be, what, kind, held_after):
    """Reported, and the count covers no entry but those of the cached places, those held before and those that the pass made."""
    from ojas_b200 import OjasError
    cached, new, held, free, tokens, width = [5, 0], [7, 3], [2, 0], [40, 41, 42], 10, 4
    if what == "too few held":
        held, new = [1, 0], [1, 3]
    if what == "too many held":
        held, new = [9, 0], [1, 3]
    if what == "free":
        free = [40]
    if what == "tokens":
        tokens = 8
    if what == "width":
        width = 2
    if what in ("too few held", "too many held"):
        tokens = 4
    tables = np.arange(2 * width).reshape(2, width)
    d_tables = u32(be, tables)
    got = be.paged_plan(u32(be, cached), u32(be, new), u32(be, free), u32(be, [0]), d_tables, 4, tokens=tokens, held_pages=u32(be, held))
    with pytest.raises(OjasError) as e:
        be.sync()
    assert e.value.kind == kind and list(got.held_pages.numpy()) == held_after
    entered = d_tables.numpy()
    for b in range(2):
        for i in range(width):
            before = max(held[b], -(-cached[b] // 4))
            assert (entered[b, i] == tables[b, i]) == (i < before or i >= held_after[b])


def test_a_free_entry_that_names_no_page_is_reported(be):
    from ojas_b200 import OjasError
    tables, free = u32(be, np.full((2, 4), 9)), u32(be, [3, NONE, 5])
    got = be.paged_plan(u32(be, [0, 0]), u32(be, [8, 3]), free, u32(be, [0]), tables, 4, tokens=11)
    with pytest.raises(OjasError) as e:
        be.sync()
    assert e.value.kind == "OutOfRange"
    assert list(got.slots.numpy()) == [12, 13, 14, 15, NONE, NONE, NONE, NONE, 20, 21, 22] and tables.numpy()[1, 0] == 5


def test_a_length_that_passes_32_bits_takes_no_page(be):
    """Request 0's lengths add up to more than 32 bits hold: none of its tokens gets a slot, request 1's page is its own."""
    from ojas_b200 import OjasError
    page = 1 << 24
    new = [page + 6, 2]
    tables = u32(be, np.zeros((2, 256)))
    got = be.paged_plan(u32(be, [(1 << 32) - page - 3, 0]), u32(be, new), u32(be, [77, 78]), u32(be, [0]), tables, page, tokens=sum(new))
    with pytest.raises(OjasError) as e:
        be.sync()
    assert e.value.kind == "OutOfRange"
    slots, entered = got.slots.numpy(), tables.numpy()
    assert np.all(slots[: new[0]] == NONE) and list(slots[new[0]:]) == [77 * page, 77 * page + 1]
    assert entered[1, 0] == 77 and not entered[0].any() and got.free_head.numpy()[0] == 1
