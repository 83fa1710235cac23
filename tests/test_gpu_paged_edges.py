"""Calls over a paged KV cache at its edges."""
import numpy as np
import pytest

from test_gpu_paged import HALF_BF16, HALF_F32, NONE, Case, be, floats, u32  # noqa: F401  (be: the module's backend)

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


# one shape for each kernel: cached, new, heads, KV heads, dim, page, BF16
KERNELS = {"rows": ([300, 77], [3, 1], 4, 2, 40, 8, True), "few f32": ([700, 90], [1, 1], 4, 2, 64, 16, False), "tiles f32": ([500, 131], [9, 4], 4, 2, 96, 8, False),
           "tiles of 16": ([900, 200], [3, 1], 8, 2, 128, 16, True), "tiles of 16, 128 keys": ([900, 200], [3, 1], 8, 2, 64, 8, True), "tiles of 32": ([500, 77], [12, 9], 4, 2, 64, 24, True),
           "tiles of 64": ([500, 77], [20, 30], 2, 1, 80, 20, True), "tiles of 192 columns": ([300, 170], [2, 9], 4, 1, 192, 16, True),
           "tcgen05": ([700, 150], [40, 35], 4, 4, 64, 16, True), "tcgen05, two tiles": ([900, 150], [150, 135], 4, 2, 128, 8, True),
           "tcgen05, large pages": ([900, 700], [60, 64], 2, 2, 128, 256, True)}


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("window", [1, 5, 70, 200])
@pytest.mark.parametrize("tree", [True, False])
def test_pages_before_the_window_may_be_released(be, kernel, window, tree):
    """Entries of pages that lie wholly before the request's first visible place, cached - window + 1, name no page any more: the same bits, no fault."""
    cached, new, h, hk, d, page, bf16 = KERNELS[kernel]
    c = Case(70 + window, cached, new, h, hk, d, page, tree, bf16)
    out, lse = c.check(be, window=window)
    for b in range(len(cached)):
        c.tables[b, : max(0, cached[b] - window + 1) // page] = NONE
    for kw in (dict(), dict(heads_first=True)):
        got = c.run(be, window=window, **kw)
        assert np.array_equal(got[0], out) and np.array_equal(got[1], lse)
    if not tree:
        got = c.run(be, window=window, use_positions=False)
        assert np.array_equal(got[0], out) and np.array_equal(got[1], lse)


def test_the_page_of_the_first_visible_place_is_still_followed(be):
    from ojas_b200 import OjasError
    for kernel in KERNELS:
        cached, new, h, hk, d, page, bf16 = KERNELS[kernel]
        c = Case(71, cached, new, h, hk, d, page, False, bf16)
        c.tables[0, (cached[0] - 40 + 1) // page] = NONE
        with pytest.raises(OjasError) as e:
            c.run(be, window=40)
        assert e.value.kind == "OutOfRange", kernel


def scored_minus_infinity(c, drop):
    """The case's reference where the places of `drop` (request 0) score -inf in every row that sees them: they weigh nothing."""
    keep_k, keep_v = c.k.copy(), c.v.copy()
    for p in drop:
        page, off = c.slot(0, p)
        c.k[page, off, :, 0] = -np.inf
    n, d, h, hk = int(c.starts[-1]), c.q.shape[2], c.q.shape[1], c.k.shape[2]
    out, lse, tol, lse_tol = np.zeros((n, h, d)), np.full((n, h), np.nan), np.zeros((n, h, d)), np.zeros((n, h))
    half, eps_p = (HALF_BF16, HALF_BF16) if c.bf16 else (HALF_F32, 0.0)
    cached, total = int(c.cached[0]), int(c.cached[0] + c.new[0])
    at = np.arange(total)
    k, v = (a[c.tables[0, at // c.page], at % c.page].astype(np.float64) for a in (keep_k, keep_v))
    for t in range(n):
        sees = at <= cached + t
        if c.masks is not None:
            sees = np.array([p < cached or bool(c.masks[t, (p - cached) // 32] >> np.uint32((p - cached) % 32) & 1) for p in at])
        sees[list(drop)] = False
        for head in range(h):
            kk, vv = k[sees, head // (h // hk)], v[sees, head // (h // hk)]
            if not len(kk):
                out[t, head] = np.nan
                continue
            s = kk @ c.q[t, head].astype(np.float64) / np.sqrt(d)
            p = np.exp(s - s.max())
            lse[t, head], out[t, head] = s.max() + np.log(p.sum()), p @ vv / p.sum()
            e_s = (d + 4) * 2.0 ** -24 * (np.abs(kk) @ np.abs(c.q[t, head])).max() / np.sqrt(d)
            e_w = e_s + 2.0 ** -20 + (total + 8) * 2.0 ** -24                      # as in paged_reference.attention
            tol[t, head] = (half + 2.0 ** -22) * np.abs(out[t, head]) + (2 * e_w + eps_p * (1 + 2.0 ** -6)) * (p @ np.abs(vv) / p.sum()) * (1 + half) + 1e-30
            lse_tol[t, head] = e_w + e_s + 2.0 ** -22 * (1 + abs(lse[t, head]))
    return out, lse, tol, lse_tol


@pytest.mark.parametrize("h,hk,d,cached,new", [(8, 1, 96, 9, 1), (4, 1, 64, 6, 2), (16, 1, 128, 7, 3), (8, 1, 32, 300, 10)])
def test_f32_operands_at_the_ends_of_the_range(be, h, hk, d, cached, new):
    """The tiles take an F32 operand apart into two of fewer bits: a key's infinity gives the infinite score, and what would round up to an infinity stays
    finite. The largest values are 2^128 - 2^116: the sums' rounding, 2^-20 of them and less, stays below the 2^-12 that are left."""
    big = np.float32(2.0 ** 128 - 2.0 ** 116)
    c = Case(73, [cached], [new], h, hk, d, 16, True, False)
    c.q[..., 0] = 1.0
    want, want_lse, tol, lse_tol = scored_minus_infinity(c, [cached])
    assert np.any(np.isinf(c.k))
    got, lse = c.run(be)
    assert np.all(np.abs(got - want) <= tol) and np.all(np.abs(lse - want_lse) <= lse_tol)
    c = Case(74, [cached], [new], h, hk, d, 16, True, False)
    c.k[..., 1], c.q[..., 1] = big, 2.0 ** -126
    first, off = c.slot(0, 0)
    c.v[first, off, :, 2], c.v[first, off, :, 3] = -0.5 * big, big              # at one place: the running sums are not normalised
    got, lse = c.check(be)
    assert np.all(np.isfinite(got))


INFINITE = [(kind, h, hk, d, cached, new, page, tree) for kind, h, hk, d, new, page, tree in [
    ("rows", 4, 2, 40, 3, 8, True), ("few f32", 4, 2, 64, 1, 16, False), ("few f32", 1, 1, 128, 3, 16, True), ("tiles f32", 8, 1, 96, 1, 16, True), ("tiles f32", 4, 1, 64, 9, 16, True),
    ("tiles", 8, 1, 128, 1, 16, True), ("tiles", 4, 1, 64, 3, 16, True), ("tiles", 4, 1, 80, 7, 16, True), ("tcgen05", 2, 1, 64, 30, 16, True), ("tcgen05", 4, 1, 128, 40, 16, True)]
    for cached in (16, 64, 5000)]


@pytest.mark.parametrize("kind,h,hk,d,cached,new,page,tree", INFINITE)
@pytest.mark.parametrize("where", ["a new token", "the first places", "all but one", "all"])
def test_scores_of_minus_infinity_weigh_nothing(be, kind, h, hk, d, cached, new, page, tree, where):
    """However the keys are shared out: places that score -inf alone in a warp or a piece, next to others, in all but one place, in all (then the formula's NaN)."""
    from ojas_b200 import OjasError
    bf16 = "f32" not in kind
    c = Case(72 + d, [cached], [new], h, hk, d, page, tree, bf16)
    c.q[..., 0] = 1.0
    drop = {"a new token": [cached], "the first places": list(range(cached - 3)), "all but one": [p for p in range(cached + new) if p != 5], "all": list(range(cached + new))}[where]
    want, want_lse, tol, lse_tol = scored_minus_infinity(c, drop)
    q, out, lse = floats(be, c.q, bf16), floats(be, np.zeros(c.q.shape), bf16), be.zeros(c.q.shape[:2])
    be.paged_attention_forward(q, floats(be, c.k, bf16), floats(be, c.v, bf16), u32(be, c.tables), u32(be, c.cached), u32(be, c.starts),
                               masks=be.upload(c.masks) if c.masks is not None else None, positions=u32(be, c.positions), out=out, lse=lse)
    if where == "all":
        with pytest.raises(OjasError) as e:
            be.sync()
        assert e.value.kind == "NonFinite"
        assert np.all(np.isnan(out.numpy())) and np.all(np.isnan(lse.numpy()))
        return
    be.sync()
    assert np.all(np.abs(out.numpy() - want) <= tol) and np.all(np.abs(lse.numpy() - want_lse) <= lse_tol)


def test_an_expired_wait_is_not_laid_to_one_kind_of_kernel(be):
    """The matrix products, the attention and the paged attention share the bounded wait and its word; the report names none of them alone."""
    import ctypes as C
    from ojas_b200 import OjasError
    from ojas_b200._lib import lib
    from ojas_b200.backend import _check
    gave_up = C.c_int32(-1)
    with pytest.raises(OjasError) as e:
        _check(lib.ojc_selftest_bounded_wait(be._handle, C.c_uint64(2_000_000), C.byref(gave_up)))
    assert e.value.kind == "WaitTimeout" and "matrix-product or attention" in str(e.value)
    be.sync()


@pytest.mark.parametrize("h,hk,d,new", [(4, 4, 64, 20), (8, 2, 64, 5), (16, 16, 128, 17), (8, 2, 128, 8)])
@pytest.mark.parametrize("requests", [1, 20])
def test_seventeen_to_thirty_two_rows_in_narrow_and_wide_tables(be, h, hk, d, new, requests):
    """Either kernel for these rows, by the number of units and (128 columns) the tables' width; at 64 columns the width has no say, so the bits are the same."""
    rng = np.random.default_rng(80)
    c = Case(81, [int(x) for x in rng.integers(1, 400, requests)], [new] * requests, h, hk, d, 16, True, True, pad=1)
    out, lse = c.check(be)
    c.tables = np.concatenate([c.tables, np.full((requests, 2100), 0x7FFFFFFF, np.int64)], 1)
    wide = c.check(be)
    if d == 64 or requests * hk <= 148:
        assert np.array_equal(wide[0], out) and np.array_equal(wide[1], lse)


def test_held_pages_with_the_largest_batch_and_many_tokens(be):
    """More lengths than the default shared memory holds, four tokens to a thread; every other request already holds a page more than its cached places need."""
    batch, page = 24000, 16
    cached, new = [int(x) for x in np.arange(batch) % 37], [int(x) for x in (np.arange(batch) * 7) % 19]
    held = [-(-c // page) + (b & 1) for b, c in enumerate(cached)]
    tables, free = np.arange(batch * 5).reshape(batch, 5), np.arange(batch * 5, batch * 8)[::-1].copy()
    want, head, held_after, entered = held_plan(cached, new, held, free, 2, tables, page)
    d_tables = u32(be, tables)
    got = be.paged_plan(u32(be, cached), u32(be, new), u32(be, free), u32(be, [2]), d_tables, page, tokens=sum(new) + 3, held_pages=u32(be, held))
    be.sync()
    assert np.array_equal(got.slots.numpy(), np.array(want + [NONE] * 3, np.uint32)) and list(got.held_pages.numpy()) == held_after and got.free_head.numpy()[0] == head
    assert np.array_equal(d_tables.numpy(), entered)


@pytest.mark.parametrize("window", [None, 300])
@pytest.mark.parametrize("h,hk,d,bf16", [(2, 1, 64, True), (2, 2, 128, True), (1, 1, 64, False)])
def test_a_long_piece_of_a_prompt(be, window, h, hk, d, bf16):
    Case(82, [0, 190], [1300, 1030], h, hk, d, 64, False, bf16).check(be, window=window)


@pytest.mark.parametrize("window", [None, 64])
@pytest.mark.parametrize("h,hk,d,bf16", [(2, 2, 64, True), (4, 1, 128, True), (2, 2, 64, False)])
def test_a_piece_of_a_prompt_among_single_tokens(be, window, h, hk, d, bf16):
    cached = [int(x) for x in np.random.default_rng(83).integers(0, 300, 64)]
    new = [1] * 64
    new[40] = 512
    Case(83, cached, new, h, hk, d, 16, False, bf16, pad=5).check(be, window=window)
