"""The paged-cache operators against their 64-bit definitions (paged_reference.py), at the sizes, masks and layouts where they can go wrong."""
import numpy as np
import pytest

import paged_reference as ref

pytestmark = pytest.mark.gpu

NONE = ref.NONE
HALF_BF16, HALF_F32 = 2.0 ** -8, 2.0 ** -24


@pytest.fixture(scope="module")
def be():
    from ojas_b200 import CudaBackend
    backend = CudaBackend(0, 32 << 30)
    yield backend
    backend.sync()
    backend.close()


def u32(be, a):
    return be.upload(np.ascontiguousarray(a).astype(np.int64).astype(np.uint32))


def floats(be, a, bf16):
    from ojas_b200 import DType
    return be.upload(np.ascontiguousarray(a, np.float32), DType.BF16 if bf16 else None)


def strided(be, a, bf16, pad, order=None):
    """A view of `a` whose storage has its axes in `order` and rows of `pad` more elements than the last axis."""
    from ojas_b200 import Tensor
    order = list(order or range(a.ndim))
    wide = np.full([a.shape[d] for d in order[:-1]] + [a.shape[order[-1]] + pad], 7.0, np.float32)
    wide[..., : a.shape[order[-1]]] = a.transpose(order)
    base = floats(be, wide, bf16)
    strides = [0] * a.ndim
    for d, s in zip(order, base.strides):
        strides[d] = s
    return Tensor(be, base.ptr, a.shape, base.dtype, strides, owner=base), base


# ---------------------------------------------------------------------------------------------------------------- plan

def tree_parents(rng, new, spread=3):
    """Per token the parent's index among the request's drafts; some roots in the middle, the first one always a root."""
    out = []
    for n in new:
        for i in range(n):
            p = i - 1 - int(rng.integers(0, spread))
            out.append(p if p >= 0 else NONE)
    return np.array(out, np.int64)


@pytest.mark.parametrize("cached,new,page,tree,pad", [
    ([0], [1], 1, False, 0), ([5], [1], 16, False, 3), ([16], [16], 16, True, 0), ([15, 16, 17, 0], [1, 1, 1, 33], 16, True, 5),
    ([0, 0, 0], [0, 0, 7], 4, True, 1), ([3, 9, 1], [4, 0, 0], 8, False, 2), ([100, 7, 31], [40, 64, 5], 20, True, 0), ([4095] * 5, [300, 1, 77, 130, 2], 64, False, 9),
    (list(range(300)), [i % 5 for i in range(300)], 7, True, 4), ([11] * 1000, [3] * 1000, 32, False, 0)])
@pytest.mark.parametrize("masked", [False, True])
def test_plan(be, cached, new, page, tree, pad, masked):
    rng = np.random.default_rng(len(cached) + page)
    n, words = sum(new), (max(new) + 31) // 32 if masked else 0
    held, total = [-(-c // page) for c in cached], [-(-(c + k) // page) for c, k in zip(cached, new)]
    pool = rng.permutation(sum(total) + 11)
    tables = np.full((len(cached), max(total) + 2), 0xABCD, np.int64)
    at = 0
    for b, k in enumerate(held):
        tables[b, :k] = pool[at:at + k]
        at += k
    free, head = np.concatenate([[0xDEAD] * 2, pool[at:]]), 2
    parents = np.concatenate([tree_parents(rng, new), np.zeros(pad, np.int64)]) if tree else None
    want = ref.plan(cached, new, free, head, tables, page, n + pad, parents, words)
    dt, dh = u32(be, tables), u32(be, [head])
    for again in range(2):                       # the same lengths once more: the same pages, nothing moves
        got = be.paged_plan(u32(be, cached), u32(be, new), u32(be, free), dh, dt, page, tokens=n + pad, parents=u32(be, parents) if tree else None, mask_words=words)
        assert np.array_equal(got.starts.numpy(), want[0]) and np.array_equal(got.slots.numpy(), want[1]) and np.array_equal(got.positions.numpy(), want[2])
        if words:
            assert np.array_equal(got.masks.numpy(), want[3])
        assert got.free_head.numpy()[0] == want[4] and np.array_equal(dt.numpy(), want[5]) and dh.numpy()[0] == head


def test_plan_with_the_largest_batch(be):
    batch = 24000
    cached, new = np.arange(batch) % 37, (np.arange(batch) * 7) % 3
    free = np.arange(batch * 2)[::-1].copy()
    tables = np.zeros((batch, 8), np.int64)
    want = ref.plan(cached, new, free, 1, tables, 16, int(new.sum()))
    dt = u32(be, tables)
    got = be.paged_plan(u32(be, cached), u32(be, new), u32(be, free), u32(be, [1]), dt, 16, tokens=int(new.sum()))
    assert np.array_equal(got.slots.numpy(), want[1]) and np.array_equal(got.starts.numpy(), want[0]) and np.array_equal(dt.numpy(), want[5])


@pytest.mark.parametrize("what,kind", [("free", "CapacityExceeded"), ("width", "OutOfRange"), ("tokens", "OutOfRange"), ("parent", "OutOfRange"), ("words", "OutOfRange"),
                                       ("entry", "OutOfRange"), ("head", "CapacityExceeded"), ("length", "OutOfRange")])
def test_plan_reports_what_only_the_device_sees(be, what, kind):
    from ojas_b200 import OjasError
    cached, new, page = [30, 8], [5, 40], 8
    free, head, width, tokens, words = np.arange(20) + 50, 0, 8, 45, 2
    tables = np.arange(2 * width).reshape(2, width)
    parents = tree_parents(np.random.default_rng(0), new)
    if what == "free":
        free = free[:3]
    if what == "width":
        tables = tables[:, :5]
    if what == "tokens":
        tokens, parents = 44, parents[:44]
    if what == "parent":
        parents[9] = 4
    if what == "words":
        words = 1
    if what == "entry":
        tables[0, 3] = NONE
    if what == "head":
        head = 25
    if what == "length":
        cached = [30, NONE - 3]
    dt = u32(be, tables)
    got = be.paged_plan(u32(be, cached), u32(be, new), u32(be, free), u32(be, [head]), dt, page, tokens=tokens, parents=u32(be, parents), mask_words=words)
    with pytest.raises(OjasError) as e:
        be.sync()
    assert e.value.kind == kind
    slots = got.slots.numpy()                    # reported once; slots that could be formed are slots of known pages
    known = set(int(p) for p in free) | set(int(p) for p in tables.ravel())
    assert all(int(s) // page in known for s in slots if s != NONE)
    if what == "free":
        assert np.sum(slots == NONE) > 0 and got.free_head.numpy()[0] == 3


# ---------------------------------------------------------------------------------------------------------------- rope

ROPE = [(1, 1, 2, 2), (5, 3, 64, 64), (7, 12, 64, 32), (130, 2, 80, 20), (33, 5, 96, 96), (9, 4, 128, 128), (3, 2, 256, 256), (17, 1, 66, 34), (65, 40, 128, 64), (2, 3, 200, 8),
        (1000, 8, 64, 64)]


def rope_bound(x, freqs, amplitude, half_out):
    """A turned pair: the angle is off by at most 2^-24 of pi where it is rounded and 2^-22 in its sine and cosine; two products and a sum of 2^-24 each."""
    size = np.abs(amplitude) * np.sqrt(2.0) * np.abs(x).max()
    return (half_out + 2.0 ** -20) * size


@pytest.mark.parametrize("n,h,d,rotary", ROPE)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("bf16", [False, True])
def test_rope_forward_and_backward(be, n, h, d, rotary, layout, bf16):
    from ojas_b200 import RopeSpec
    rng = np.random.default_rng(n + d)
    x = rng.standard_normal((n, h, d)).astype(np.float32)
    x = ref.round_bf16(x) if bf16 else x
    positions = rng.integers(0, 1 << 20, n)
    positions[0] = NONE if n % 2 else 0                 # as far as a position goes
    spec = RopeSpec(rotary, layout=layout, scaling="by_turns", factor=8.0, original_length=4096.0, amplitude=1.2)
    f = ref.frequencies(rotary, scaling="by_turns", factor=8.0, original=4096.0)
    # the reference's own angles: numpy's frequencies are good to 2^-50 or so, times the position
    angle_error = positions.max() * 2.0 ** -50
    half = HALF_BF16 if bf16 else HALF_F32
    plan = be.rope_plan(spec)
    for fn, back in ((be.rope_forward, False), (be.rope_backward, True)):
        got = fn(floats(be, x, bf16), u32(be, positions), plan).numpy()
        want = ref.rotate(x, positions, f, layout, 1.2, back)
        assert np.all(np.abs(got - want) <= rope_bound(x, f, 1.2, half) + angle_error * np.abs(x).max())
        assert np.array_equal(got[..., rotary:], x[..., rotary:])
    xs, base = strided(be, x, bf16, 6)
    inplace = be.rope_forward(xs, u32(be, positions), plan, out=xs)
    assert inplace is xs
    whole = base.numpy()
    assert np.array_equal(whole[..., :d], be.rope_forward(floats(be, x, bf16), u32(be, positions), plan).numpy()) and np.all(whole[..., d:] == 7.0)


@pytest.mark.parametrize("bf16", [False, True])
def test_rope_rank_4_broadcasts_positions_and_reads_permuted_views(be, bf16):
    from ojas_b200 import RopeSpec
    rng = np.random.default_rng(2)
    b, time, h, d = 3, 17, 4, 64
    x = ref.round_bf16(rng.standard_normal((b, time, h, d)))
    positions = rng.integers(0, 5000, time)
    plan = be.rope_plan(RopeSpec(d))
    flat = be.rope_forward(floats(be, x.reshape(b * time, h, d), bf16), u32(be, np.tile(positions, b)), plan).numpy().reshape(x.shape)
    assert np.array_equal(be.rope_forward(floats(be, x, bf16), u32(be, positions), plan).numpy(), flat)
    assert np.array_equal(be.rope_forward(floats(be, x, bf16), u32(be, np.tile(positions, (b, 1))), plan).numpy(), flat)
    heads_first = floats(be, x.transpose(0, 2, 1, 3), bf16).permuted((0, 2, 1, 3))        # [B, H, T, D] storage
    assert np.array_equal(be.rope_forward(heads_first, u32(be, positions), plan).numpy(), flat)


def test_rope_agrees_with_the_table_form(be):
    """rope_half_split_forward on tables of the same angles."""
    from ojas_b200 import RopeSpec
    rng = np.random.default_rng(3)
    b, time, h, d = 2, 50, 3, 64
    x = rng.standard_normal((b, time, h, d)).astype(np.float32)
    angle = np.arange(time)[:, None] * ref.frequencies(d)[None]
    cos, sin = np.cos(np.concatenate([angle, angle], 1)).astype(np.float32), np.sin(np.concatenate([angle, angle], 1)).astype(np.float32)
    got = be.rope_forward(be.upload(x), u32(be, np.arange(time)), be.rope_plan(RopeSpec(d))).numpy()
    want = be.rope_half_split_forward(be.upload(x), be.upload(cos), be.upload(sin)).numpy()
    assert np.abs(got - want).max() <= 2 * rope_bound(x, None, 1.0, HALF_F32)


def test_rope_gradient_is_that_of_the_forward(be):
    """Differences of <g, rope(x)>: the map is linear, so <g, rope(x + e) - rope(x)> = <rope_backward(g), e> up to f32 rounding."""
    from ojas_b200 import RopeSpec
    rng = np.random.default_rng(4)
    x, g, e = (rng.standard_normal((21, 3, 32)).astype(np.float32) for _ in range(3))
    positions, plan = u32(be, rng.integers(0, 100000, 21)), be.rope_plan(RopeSpec(24, layout="interleaved", scaling="linear", factor=3.0, amplitude=0.7))
    gx = be.rope_backward(be.upload(g), positions, plan).numpy().astype(np.float64)
    d = be.rope_forward(be.upload(x + e), positions, plan).numpy().astype(np.float64) - be.rope_forward(be.upload(x), positions, plan).numpy()
    left, right = (g.astype(np.float64) * d).sum(), (gx * e).sum()
    assert abs(left - right) <= 2.0 ** -20 * np.abs(g).astype(np.float64).ravel() @ (np.abs(d) + np.abs(x) + np.abs(e)).ravel()


# ---------------------------------------------------------------------------------------------------------------- write

@pytest.mark.parametrize("n,h,d,page,rotary,layout", [(1, 1, 8, 1, 0, "half"), (5, 2, 64, 16, 64, "half"), (67, 3, 128, 16, 64, "interleaved"), (9, 8, 80, 20, 80, "half"),
                                                      (130, 1, 66, 7, 34, "half"), (33, 12, 64, 64, 0, "half"), (300, 4, 128, 32, 128, "half")])
@pytest.mark.parametrize("src,dst", [(False, False), (False, True), (True, True), (True, False)])
@pytest.mark.parametrize("heads_first", [False, True])
def test_write(be, n, h, d, page, rotary, layout, src, dst, heads_first):
    from ojas_b200 import RopeSpec
    rng = np.random.default_rng(n + d)
    pages = -(-n // page) + 3
    k, v = (rng.standard_normal((n, h, d)).astype(np.float32) for _ in range(2))
    if src:
        k, v = ref.round_bf16(k), ref.round_bf16(v)
    slots = rng.permutation(pages * page)[:n]
    slots[n // 2] = NONE if n > 2 else slots[n // 2]
    positions = rng.integers(0, 1 << 20, n)
    old = ref.round_bf16(rng.standard_normal((2, pages, page, h, d)))
    order = (0, 2, 1, 3) if heads_first else None
    (kp, k_base), (vp, v_base) = strided(be, old[0], dst, 8 if heads_first else 0, order), strided(be, old[1], dst, 8 if heads_first else 0, order)
    fused, _ = strided(be, np.concatenate([k, v], 1), src, 0)
    from ojas_b200 import Tensor
    dk = Tensor(be, fused.ptr, k.shape, fused.dtype, fused.strides, owner=fused)
    dv = Tensor(be, fused.ptr + h * d * fused.dtype.size, v.shape, fused.dtype, fused.strides, owner=fused)
    be.paged_kv_write(kp, vp, dk, dv, u32(be, slots), rope=be.rope_plan(RopeSpec(rotary, layout=layout)) if rotary else None, positions=u32(be, positions) if rotary else None)
    live = slots != NONE
    want_k = ref.rotate(k, positions, ref.frequencies(rotary), layout) if rotary else k.astype(np.float64)
    half = HALF_BF16 if dst else HALF_F32
    for base, fill, rows, tol in ((k_base, old[0], want_k, rope_bound(k, None, 1.0, half) + 2.0 ** -30 if rotary else 0.0), (v_base, old[1], v, 0.0)):
        got = base.numpy()[..., :d]
        got = (got.transpose(0, 2, 1, 3) if heads_first else got).reshape(pages * page, h, d)
        untouched = np.setdiff1d(np.arange(pages * page), slots[live])
        assert np.array_equal(got[untouched], fill.reshape(-1, h, d)[untouched])
        want = rows[live]
        if tol == 0.0:
            assert np.array_equal(got[slots[live]], ref.round_bf16(want) if dst else want.astype(np.float32))
        else:
            assert np.all(np.abs(got[slots[live]] - want) <= tol)


def test_write_skips_and_reports_slots_outside_the_pages(be):
    from ojas_b200 import OjasError
    kp, vp = be.zeros((2, 4, 1, 8)), be.zeros((2, 4, 1, 8))
    k = be.upload(np.ones((3, 1, 8), np.float32))
    be.paged_kv_write(kp, vp, k, k, u32(be, [7, 8, NONE]))
    with pytest.raises(OjasError) as e:
        be.sync()
    assert e.value.kind == "OutOfRange"
    want = np.zeros((8, 8)); want[7] = 1
    assert np.array_equal(kp.numpy().reshape(8, 8), want) and np.array_equal(vp.numpy().reshape(8, 8), want)


# ---------------------------------------------------------------------------------------------------------------- attention

class Case:
    """Requests over a shuffled pool whose unused places hold NaN; trees of drafts unless `tree` is False."""

    def __init__(self, seed, cached, new, h, hk, d, page, tree=True, bf16=True, words_more=0, pad=0, scale=1.0):
        rng = np.random.default_rng(seed)
        self.rng, self.bf16, self.page = rng, bf16, page
        self.cached, self.new = np.array(cached), np.array(new)
        self.starts = np.concatenate([[0], np.cumsum(new)])
        n, total = int(sum(new)), -(-(self.cached + self.new) // page)
        pool = int(total.sum()) + 3
        order, self.tables, at = rng.permutation(pool), np.full((len(cached), int(total.max()) + 1), 0x7FFFFFFF, np.int64), 0
        self.k = np.full((pool, page, hk, d), np.nan, np.float32)
        self.v = np.full((pool, page, hk, d), np.nan, np.float32)
        for b, k in enumerate(total):
            self.tables[b, :k] = order[at:at + k]
            at += k
            p = np.arange(self.cached[b] + self.new[b])
            for pages in (self.k, self.v):
                pages[self.tables[b, p // page], p % page] = rng.standard_normal((len(p), hk, d))
        self.q = (scale * rng.standard_normal((n + pad, h, d))).astype(np.float32)
        if bf16:
            self.q = ref.round_bf16(self.q)
            for pages in (self.k, self.v):
                live = np.isfinite(pages)
                pages[live] = ref.round_bf16(pages[live])
        self.masks, self.positions = None, np.concatenate([c + np.arange(k) for c, k in zip(cached, new)] + [np.zeros(pad)]).astype(np.int64)
        if tree:
            words = -(-int(max(new)) // 32) + words_more
            plan = ref.plan(cached, new, np.arange(pool + 9), 0, np.zeros((len(cached), int(total.max()) + 1), np.int64), page, n + pad, tree_parents(rng, new), words)
            self.masks, self.positions = plan[3], plan[2]

    def slot(self, b, p):
        return int(self.tables[b, p // self.page]), p % self.page

    def run(self, be, window=None, use_positions=True, workspace=False, heads_first=False, order=None, q_pad=0, kp=None, vp=None):
        """(out, lse) as numpy; rows behind the last token keep 7."""
        q, _ = strided(be, self.q, self.bf16, q_pad)
        pages_order = (0, 2, 1, 3) if heads_first else None
        kp = kp or strided(be, self.k, self.bf16, 0, pages_order)[0]
        vp = vp or strided(be, self.v, self.bf16, 0, pages_order)[0]
        out, base = strided(be, np.full(self.q.shape, 7.0, np.float32), self.bf16, q_pad)
        lse = be.upload(np.full(self.q.shape[:2], 7.0, np.float32))
        be.paged_attention_forward(q, kp, vp, u32(be, self.tables), u32(be, self.cached), u32(be, self.starts), masks=be.upload(self.masks) if self.masks is not None else None,
                                   positions=u32(be, self.positions) if use_positions else None, window=window, out=out, lse=lse,
                                   workspace=be.paged_attention_workspace(q, kp) if workspace else None)
        be.sync()
        return base.numpy()[..., : self.q.shape[2]], lse.numpy()

    def check(self, be, window=None, use_positions=True, **kw):
        got, lse = self.run(be, window, use_positions, **kw)
        half = HALF_BF16 if self.bf16 else HALF_F32
        n = int(self.starts[-1])
        # unseen places are NaN: the reference looks at none of them either
        want, want_lse, tol, lse_tol = ref.attention(self.q[:n], self.k, self.v, self.tables, self.cached, self.starts, self.masks, self.positions if use_positions else None, window,
                                                     eps_out=half, eps_p=HALF_BF16 if self.bf16 else 0.0)
        assert np.all(np.abs(got[:n] - want) <= tol), float((np.abs(got[:n] - want) / tol).max())
        blank = np.isneginf(want_lse)
        assert np.array_equal(np.isneginf(lse[:n]), blank) and not got[:n][blank].any()
        assert np.all(np.abs(lse[:n][~blank] - want_lse[~blank]) <= lse_tol[~blank])
        assert np.all(got[n:] == 7.0) and np.all(lse[n:] == 7.0)
        return got, lse


SHAPES = [  # cached, new, heads, KV heads, dim, page
    ([0], [1], 1, 1, 64, 16), ([1], [1], 4, 4, 64, 16), ([776], [1], 12, 12, 64, 16), ([63, 64, 65], [1, 1, 1], 8, 2, 128, 16), ([127, 0, 300], [1, 5, 33], 4, 1, 128, 20),
    ([500, 17], [9, 16], 8, 1, 64, 64), ([250], [63], 4, 4, 128, 32), ([200, 100], [128, 70], 8, 2, 64, 8), ([90], [130], 6, 2, 128, 16), ([33, 5], [3, 4], 6, 3, 96, 7),
    ([40], [5], 2, 2, 80, 16), ([40, 2], [5, 31], 2, 1, 256, 16), ([31], [2], 3, 3, 66, 1), ([70], [6], 2, 2, 33, 5), ([1500, 1, 700], [17, 2, 0], 16, 2, 128, 64),
    ([0, 0], [40, 64], 4, 2, 64, 16), ([260], [65], 16, 2, 128, 128), ([300], [128], 16, 1, 64, 24)]


@pytest.mark.parametrize("cached,new,h,hk,d,page", SHAPES)
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("tree", [True, False])
def test_attention(be, cached, new, h, hk, d, page, bf16, tree):
    Case(len(cached) + d, cached, new, h, hk, d, page, tree, bf16, pad=2).check(be)


@pytest.mark.parametrize("window", [1, 2, 16, 100, 5000])
@pytest.mark.parametrize("cached,new,h,hk,d,page", [SHAPES[i] for i in (1, 3, 4, 6, 9, 14)])
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("tree", [True, False])
def test_attention_in_a_window(be, cached, new, h, hk, d, page, window, bf16, tree):
    Case(window, cached, new, h, hk, d, page, tree, bf16).check(be, window=window)


@pytest.mark.parametrize("cached,new,h,hk,d,page", [([4000, 2100], [63, 40], 16, 16, 128, 32), ([3000, 4100], [33, 127], 16, 16, 64, 64), ([2500, 1, 900], [100, 3, 130], 8, 4, 128, 16),
                                                    ([5000], [45], 24, 24, 128, 128), ([3900], [20], 12, 12, 64, 16), ([6000], [12], 8, 8, 96, 16)])
def test_attention_with_many_key_blocks_to_a_share(be, cached, new, h, hk, d, page):
    """Several units and key blocks to each CTA of every kernel: the rings and barriers go round more than once, warps without rows run beside others."""
    c = Case(21, cached, new, h, hk, d, page, True, True)
    out, lse = c.check(be)
    for _ in range(20):                                    # the order in which warps and copies run differs from run to run, the bits do not
        again = c.run(be)
        assert np.array_equal(again[0], out) and np.array_equal(again[1], lse)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("h,hk,d", [(8, 2, 128), (4, 4, 64), (3, 1, 40)])
def test_attention_layouts_and_workspaces_give_the_same_bits(be, bf16, h, hk, d):
    c = Case(5, [130, 7, 400], [9, 1, 20], h, hk, d, 16, True, bf16, words_more=1)
    out, lse = c.check(be)
    for kw in (dict(heads_first=True), dict(workspace=True), dict(q_pad=8, workspace=True)):
        again = c.check(be, **kw)
        assert np.array_equal(again[0], out) and np.array_equal(again[1], lse), kw


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("h,hk,d,new", [(4, 1, 64, [12, 3]), (2, 2, 128, [40, 1]), (8, 1, 128, [60, 33]), (3, 3, 48, [9, 9])])
def test_attention_rows_that_see_nothing_and_poisoned_places_that_a_row_does_not_see(be, bf16, h, hk, d, new):
    """Drafts that no row sees hold NaN and infinities; a row whose mask is empty over an empty cache is 0 with lse -inf; no fault is raised."""
    c = Case(7, [0, 50], new, h, hk, d, 16, True, bf16)
    c.masks[:] &= np.uint32(0xFFFFFFF5)                    # drafts 1 and 3 of each request drop out of every row
    c.masks[0] = 0                                         # request 0 has no cache: its row 0 sees nothing
    for b in range(2):
        for j, bad in ((1, np.nan), (3, np.inf)):
            if j < new[b]:
                p, off = c.slot(b, int(c.cached[b]) + j)
                c.k[p, off], c.v[p, off] = bad, -bad
    out, lse = c.check(be)
    assert not out[0].any() and np.all(np.isneginf(lse[0]))


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("h,hk,d,new,cached", [(4, 2, 64, 12, 20), (8, 1, 128, 40, 300), (2, 2, 48, 5, 10)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_poisoned_value_reaches_the_rows_that_see_it_and_no_other(be, bf16, h, hk, d, new, cached, bad):
    from ojas_b200 import OjasError
    c = Case(8, [cached], [new], h, hk, d, 16, True, bf16)
    clean, clean_lse = c.check(be)
    j = new // 2
    p, off = c.slot(0, cached + j)
    c.v[p, off, 0, 3] = bad
    with pytest.raises(OjasError) as e:
        c.run(be)
    assert e.value.kind == "NonFinite" and "paged_attention" in str(e.value)
    try:
        got, lse = c.run(be)
    except OjasError:
        pass
    q, _ = strided(be, c.q, bf16, 0)
    out, lse_t = be.paged_attention_forward(q, floats(be, c.k, bf16), floats(be, c.v, bf16), u32(be, c.tables), u32(be, c.cached), u32(be, c.starts), masks=be.upload(c.masks),
                                            positions=u32(be, c.positions))
    with pytest.raises(OjasError):
        be.sync()
    got, lse = out.numpy(), lse_t.numpy()
    sees = (c.masks[:, j // 32] >> np.uint32(j % 32) & 1).astype(bool)
    heads = np.arange(h) < h // hk
    assert np.array_equal(got[~sees], clean[~sees]) or np.abs(got[~sees] - clean[~sees]).max() <= (2.0 ** -7 if bf16 else 2.0 ** -18) * np.abs(clean).max()
    assert np.all(np.isfinite(got[~sees])) and np.all(np.isfinite(got[:, ~heads]))
    assert not np.any(np.isfinite(got[sees][:, heads, 3]))
    # 1 x infinity is infinity, and a weight that underflows times infinity is NaN: either is what the formula gives
    assert np.all(np.isfinite(got[sees][:, heads][..., 4:])) and np.array_equal(lse, clean_lse)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("what", ["page", "length", "starts", "order"])
def test_attention_reports_what_only_the_device_sees(be, bf16, what):
    """Entries outside the pages, lengths beyond the table and starts beyond the rows: skipped, reported once, and the other requests' rows are right."""
    from ojas_b200 import OjasError
    c = Case(9, [100, 40], [4, 4], 4, 2, 64, 16, True, bf16)
    clean, _ = c.check(be)
    saved = c.tables.copy(), c.cached.copy(), c.starts.copy()
    if what == "page":
        c.tables[0, 2] = c.k.shape[0]
    if what == "length":
        c.cached[0] = 1 << 20
    if what == "starts":
        c.starts[2] = 4000
    if what == "order":
        c.starts[1] = 4000
    q, _ = strided(be, c.q, bf16, 0)
    out, _ = be.paged_attention_forward(q, floats(be, np.nan_to_num(c.k), bf16), floats(be, np.nan_to_num(c.v), bf16), u32(be, c.tables), u32(be, c.cached), u32(be, c.starts),
                                        masks=be.upload(c.masks), positions=u32(be, c.positions))
    with pytest.raises(OjasError) as e:
        be.sync()
    assert e.value.kind == "OutOfRange"
    if what in ("page", "length"):
        assert np.array_equal(out.numpy()[4:], clean[4:]) or np.abs(out.numpy()[4:] - clean[4:]).max() <= (2.0 ** -7 if bf16 else 2.0 ** -18) * np.abs(clean).max()
    c.tables, c.cached, c.starts = saved
    c.check(be)


def test_attention_repeats_bit_for_bit(be):
    c = Case(10, [3000, 900, 10], [40, 3, 64], 8, 2, 128, 16, True, True)
    first = c.run(be)
    for _ in range(3):
        again = c.run(be)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


def test_cached_attention_agrees_with_the_paged_form(be):
    """One sequence, causal drafts: the ring cache's op on the same keys (its span is the cache's whole length)."""
    c = Case(11, [45], [3], 4, 2, 64, 16, tree=False, bf16=False)
    out, _ = c.check(be)
    p = np.arange(48)
    kc, vc = (a[c.tables[0, p // 16], p % 16][None] for a in (c.k, c.v))
    want = be.cached_attention_forward(be.upload(c.q[None]), be.upload(kc), be.upload(vc), 48).numpy()[0]
    assert np.abs(out - want).max() <= 2.0 ** -16 * np.abs(want).max()


# ---------------------------------------------------------------------------------------------------------------- together

@pytest.mark.parametrize("bf16", [True, False])
def test_a_decoding_loop_over_pages(be, bf16):
    """Prompts of different lengths, then trees of drafts of which one path is kept, then single tokens: at every pass the plan, q's rotation, the write
    with k's rotation and the attention, against attention over the kept history rebuilt in 64 bits."""
    from ojas_b200 import DType, RopeSpec
    rng = np.random.default_rng(12)
    h, hk, d, page, pool, width = 4, 2, 64, 8, 64, 16
    plan, f = be.rope_plan(RopeSpec(d, layout="interleaved", scaling="linear", factor=2.0)), ref.frequencies(d, scaling="linear", factor=2.0)
    dt = DType.BF16 if bf16 else DType.F32
    kp, vp = floats(be, np.full((pool, page, hk, d), np.nan), bf16), floats(be, np.full((pool, page, hk, d), np.nan), bf16)
    tables, free = u32(be, np.full((3, width), NONE)), u32(be, rng.permutation(pool))
    head = u32(be, [0])
    cached = np.zeros(3, np.int64)
    keys = [np.zeros((0, hk, d)) for _ in range(3)]     # the history as the cache holds it: rotated, rounded
    values = [np.zeros((0, hk, d)) for _ in range(3)]
    half = HALF_BF16 if bf16 else HALF_F32
    for new, tree in (([9, 1, 30], False), ([7, 7, 1], True), ([1, 1, 1], False), ([0, 5, 12], True), ([1, 1, 1], False)):
        n, capacity = sum(new), sum(new) + 3
        parents = np.concatenate([tree_parents(rng, new), np.zeros(3, np.int64)]) if tree else None
        q, k, v = (rng.standard_normal((capacity, x, d)).astype(np.float32) for x in (h, hk, hk))
        if bf16:
            q, k, v = ref.round_bf16(q), ref.round_bf16(k), ref.round_bf16(v)
        p = be.paged_plan(u32(be, cached), u32(be, new), free, head, tables, page, tokens=capacity, parents=u32(be, parents) if tree else None, mask_words=1 if tree else 0)
        dq = be.rope_forward(floats(be, q, bf16), p.positions, plan)
        be.paged_kv_write(kp, vp, floats(be, k, bf16), floats(be, v, bf16), p.slots, rope=plan, positions=p.positions)
        out, _ = be.paged_attention_forward(dq, kp, vp, tables, u32(be, cached), p.starts, masks=p.masks, positions=p.positions, out=be.zeros((capacity, h, d), dt))
        positions, starts = p.positions.numpy().astype(np.int64), p.starts.numpy()
        got, rq = out.numpy(), dq.numpy()
        rk = ref.rotate(k, positions, f, "interleaved")
        rk = ref.round_bf16(rk) if bf16 else rk.astype(np.float32)
        assert np.abs(rq[:n] - ref.rotate(q, positions, f, "interleaved")[:n]).max() <= rope_bound(q, None, 1.0, half)
        longest = max(len(x) for x in keys) + max(new)
        ck, cv = np.zeros((3, longest, hk, d), np.float32), np.zeros((3, longest, hk, d), np.float32)
        for b in range(3):
            s = slice(starts[b], starts[b + 1])
            ck[b, :cached[b] + new[b]] = np.concatenate([keys[b], rk[s]])
            cv[b, :cached[b] + new[b]] = np.concatenate([values[b], v[s]])
        # the keys' own rounding differs by at most one step from the device's; q is compared as the device rotated it
        want, _, tol, _ = ref.attention(rq[:n], ck, cv, np.arange(3)[:, None], cached, starts, p.masks.numpy() if tree else None, positions, None, half, HALF_BF16 if bf16 else 0.0)
        slack = (2 * half + 2.0 ** -19) * np.abs(rk).max() * np.abs(rq[:n]).sum(-1, keepdims=True) / np.sqrt(d)
        assert np.all(np.abs(got[:n] - want) <= tol + 2 * slack * np.abs(cv).max()) and not got[n:].any()
        for b in range(3):                               # keep a path: the last draft's ancestors move to the front of the new places
            kept = list(range(new[b]))
            if tree and new[b]:
                row = p.masks.numpy()[starts[b + 1] - 1, 0]
                kept = [j for j in range(new[b]) if row >> j & 1]
            slots = p.slots.numpy()[starts[b]:starts[b + 1]]
            if kept != list(range(new[b])):
                t = [starts[b] + j for j in kept]
                be.paged_kv_write(kp, vp, floats(be, k[t], bf16), floats(be, v[t], bf16), u32(be, slots[: len(kept)]), rope=plan, positions=u32(be, positions[t]))
            t = [starts[b] + j for j in kept]
            keys[b], values[b] = np.concatenate([keys[b], rk[t]]), np.concatenate([values[b], v[t]])
            cached[b] += len(kept)
        head = u32(be, [int(p.free_head.numpy()[0])])    # pages of dropped drafts stay in their request's table
    be.sync()


def test_a_pass_in_a_graph_replays_with_new_lengths_and_workspaces(be):
    """Plan, rotation, write and attention captured once from the backend's stream; replayed after the lengths, the inputs and the pages' contents changed,
    with eager calls (which may grow the library's own workspace) between. Without a workspace of its own the attention refuses to be captured."""
    from cuda.bindings import runtime as rt
    from ojas_b200 import DType, OjasError, RopeSpec
    rng = np.random.default_rng(30)
    h, hk, d, page, pool, width, capacity = 8, 2, 64, 16, 80, 40, 24

    def ok(r):
        assert r[0] == rt.cudaError_t.cudaSuccess, r[0]
        return r[1] if len(r) > 1 else None
    plan = be.rope_plan(RopeSpec(d))
    cached, new, head = u32(be, [0, 0]), u32(be, [1, 1]), u32(be, [0])
    free, tables = u32(be, rng.permutation(pool)), u32(be, np.full((2, width), NONE))
    parents = u32(be, np.full(capacity, NONE))
    q, k, v = (be.zeros((capacity, n, d), DType.F32) for n in (h, hk, hk))
    qb, out, lse = be.zeros((capacity, h, d), DType.F32), be.zeros((capacity, h, d), DType.F32), be.zeros((capacity, h))
    kp, vp = be.zeros((pool, page, hk, d)), be.zeros((pool, page, hk, d))
    work = be.paged_attention_workspace(q, kp)
    keep = {n: be.empty(s, DType.U32) for n, s in dict(starts=(3,), slots=(capacity,), positions=(capacity,), masks=(capacity, 1), free_head_out=(1,)).items()}

    def one_pass(workspace):
        p = be.paged_plan(cached, new, free, head, tables, page, parents=parents, **keep)
        be.rope_forward(q, p.positions, plan, out=qb)
        be.paged_kv_write(kp, vp, k, v, p.slots, rope=plan, positions=p.positions)
        be.paged_attention_forward(qb, kp, vp, tables, cached, p.starts, masks=p.masks, positions=p.positions, out=out, lse=lse, workspace=workspace)
    one_pass(work)                                       # what is set up once happens outside the capture
    be.sync()
    stream = be.stream()
    mode = rt.cudaStreamCaptureMode.cudaStreamCaptureModeThreadLocal
    ok(rt.cudaStreamBeginCapture(stream, mode))
    with pytest.raises(OjasError) as e:
        one_pass(None)
    assert e.value.kind == "Unsupported"
    ok(rt.cudaGraphDestroy(ok(rt.cudaStreamEndCapture(stream))))
    ok(rt.cudaStreamBeginCapture(stream, mode))
    one_pass(work)
    graph = ok(rt.cudaStreamEndCapture(stream))
    run = ok(rt.cudaGraphInstantiate(graph, 0))
    import ctypes as C
    from ojas_b200._lib import lib
    from ojas_b200.backend import _check

    def put(t, a):
        a = np.ascontiguousarray(a, np.float32 if t.dtype == DType.F32 else np.uint32)
        _check(lib.ojc_upload(be._handle, C.c_void_p(t.ptr), C.c_void_p(a.ctypes.data), C.c_uint64(a.nbytes)))
    for lens, news in (([0, 0], [3, 17]), ([100, 300], [12, 1]), ([16, 0], [20, 0]), ([500, 511], [7, 9])):
        par = np.concatenate([tree_parents(rng, news), np.zeros(capacity - sum(news), np.int64)])
        qs, ks, vs = (rng.standard_normal((capacity, n, d)).astype(np.float32) for n in (h, hk, hk))
        pages_k, pages_v = (rng.standard_normal((pool, page, hk, d)).astype(np.float32) for _ in range(2))
        order = rng.permutation(pool)
        held = [-(-c // page) for c in lens]
        tab = np.full((2, width), NONE, np.int64)
        tab[0, :held[0]], tab[1, :held[1]] = order[:held[0]], order[held[0]:sum(held)]
        rest = np.concatenate([order[sum(held):], np.full(sum(held), 7)])
        for t, a in ((cached, lens), (new, news), (parents, par), (q, qs), (k, ks), (v, vs), (kp, pages_k), (vp, pages_v), (tables, tab), (free, rest)):
            put(t, np.asarray(a))
        put(out, np.full((capacity, h, d), 7.0)); put(lse, np.full((capacity, h), 7.0))
        ok(rt.cudaGraphLaunch(run, stream))
        got, got_lse, got_k = out.numpy(), lse.numpy(), kp.numpy()
        be.sync()
        for t, a in ((kp, pages_k), (vp, pages_v), (tables, tab)):
            put(t, np.asarray(a))
        put(out, np.full((capacity, h, d), 7.0)); put(lse, np.full((capacity, h), 7.0))
        one_pass(None)                                   # eager, in the library's own workspace
        assert np.array_equal(out.numpy(), got) and np.array_equal(lse.numpy(), got_lse) and np.array_equal(kp.numpy(), got_k)
        assert np.all(got[sum(news):] == 7.0)
        starts = keep["starts"].numpy()
        want, _, tol, _ = ref.attention(qb.numpy()[:sum(news)], got_k, vp.numpy(), tables.numpy(), np.array(lens), starts, keep["masks"].numpy(), keep["positions"].numpy(), None, HALF_F32, 0.0)
        assert np.all(np.abs(got[:sum(news)] - want) <= tol)
        be.linear_forward(be.upload(rng.standard_normal((64, 64)).astype(np.float32)), be.upload(rng.standard_normal((64, 64)).astype(np.float32)))
    ok(rt.cudaGraphExecDestroy(run)); ok(rt.cudaGraphDestroy(graph))
    be.sync()


@pytest.mark.parametrize("cached,h,hk,d,new", [(60000, 4, 1, 128, 1), (30000, 2, 2, 64, 3), (40000, 16, 1, 64, 5), (25000, 8, 1, 96, 2)])
@pytest.mark.parametrize("bf16", [True, False])
def test_a_long_sequence_in_many_pieces(be, cached, h, hk, d, new, bf16):
    """One unit over most of the GPU: many pieces to join; twice with the same bits."""
    c = Case(32, [cached], [new], h, hk, d, 64, True, bf16)
    out, lse = c.check(be, workspace=True)
    again = c.run(be)
    assert np.array_equal(again[0], out) and np.array_equal(again[1], lse)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("d", [16, 24, 32, 48, 112, 160, 192])
def test_attention_at_other_head_dims(be, d, bf16):
    Case(41 + d, [130, 3, 0], [9, 1, 40], 4, 2, d, 16, True, bf16).check(be)
    Case(42 + d, [700], [1], 8, 8, d, 8, False, bf16).check(be)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("q_pad", [3, 4, 8])
def test_attention_rows_at_any_alignment(be, bf16, q_pad):
    Case(43, [100, 40], [9, 20], 4, 2, 64, 16, True, bf16, pad=1).check(be, q_pad=q_pad)


@pytest.mark.parametrize("h,hk,d,page", [(4, 2, 64, 16), (2, 2, 40, 8), (8, 1, 128, 32)])
@pytest.mark.parametrize("new", [1, 7])
def test_attention_over_more_requests_than_a_cta_has_threads(be, h, hk, d, page, new):
    """The lengths are scanned in chunks; requests without new tokens stand at the front, in the middle and at the end."""
    rng = np.random.default_rng(44)
    cached = rng.integers(0, 40, 301)
    counts = np.where(rng.random(301) < 0.3, 0, rng.integers(1, new + 1, 301))
    counts[[0, 1, 150, 299, 300]] = 0
    counts[5] = new
    Case(45, list(cached), [int(x) for x in counts], h, hk, d, page, True, True, pad=3).check(be)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("h,hk,d,new", [(4, 2, 64, [12, 3]), (8, 1, 128, [40, 33])])
@pytest.mark.parametrize("window", [3, 40])
@pytest.mark.parametrize("tree", [True, False])
def test_attention_window_without_positions(be, bf16, h, hk, d, new, window, tree):
    Case(46, [60, 0], new, h, hk, d, 16, tree, bf16).check(be, window=window, use_positions=False)


def test_attention_leaves_rows_before_the_first_start(be):
    for h, hk, d in ((4, 2, 64), (2, 2, 40), (16, 1, 128)):
        c = Case(47, [90], [20], h, hk, d, 16, False, True, pad=4)
        out, lse = c.check(be)
        c.starts = c.starts + 3                            # the same queries three rows further on
        c.q = np.concatenate([np.zeros((3, h, d), np.float32), c.q[:20], np.zeros((1, h, d), np.float32)])
        c.positions = np.concatenate([np.zeros(3, np.int64), c.positions[:20], np.zeros(1, np.int64)])
        got, got_lse = c.run(be)
        assert np.array_equal(got[3:23], out[:20]) and np.array_equal(got_lse[3:23], lse[:20])
        assert np.all(got[:3] == 7.0) and np.all(got[23:] == 7.0)


def test_attention_writes_over_its_queries(be):
    """out may be q itself: a unit's rows are written when everything that reads them has."""
    for h, hk, d, cached, new in ((4, 2, 64, 500, 1), (8, 1, 128, 3000, 40), (2, 2, 40, 50, 4), (16, 1, 64, 2000, 5)):
        c = Case(48, [cached, 30], [new, 2], h, hk, d, 16, True, True)
        out, _ = c.check(be)
        q = floats(be, c.q, True)
        be.paged_attention_forward(q, floats(be, c.k, True), floats(be, c.v, True), u32(be, c.tables), u32(be, c.cached), u32(be, c.starts), masks=be.upload(c.masks),
                                   positions=u32(be, c.positions), out=q)
        assert np.array_equal(q.numpy(), out)


def test_requests_may_share_pages_and_kv_heads_may_be_views(be):
    """A common prefix: two requests' tables name the same pages; the pages are every other head of a wider pool."""
    from ojas_b200 import Tensor
    c = Case(49, [64, 64], [5, 5], 4, 2, 64, 16, True, True)
    c.tables[1, :4] = c.tables[0, :4]
    wide = np.zeros(c.k.shape[:2] + (4, 64), np.float32)
    views = []
    for pages in (c.k, c.v):
        wide[:, :, ::2] = np.nan_to_num(pages)
        wide[:, :, 1::2] = np.nan
        base = floats(be, wide, True)
        s = base.strides
        views.append(Tensor(be, base.ptr, pages.shape, base.dtype, (s[0], s[1], 2 * s[2], 1), owner=base))
    c.check(be, kp=views[0], vp=views[1])


def test_pages_far_into_a_large_pool(be):
    """Element offsets beyond 32 bits: 2.6 GB of pages a side, the request's at the very end; attention on each kernel, and the write."""
    from ojas_b200 import DType
    pool, page, hk, d = 41000, 64, 4, 128
    for h, new, bf16 in ((8, 1, True), (32, 16, True)):
        kp, vp = be.zeros((pool, page, hk, d), DType.BF16), be.zeros((pool, page, hk, d), DType.BF16)
        c = Case(50, [200], [new], h, hk, d, page, True, bf16)
        small = c.tables.copy()
        c.tables = np.where(c.tables < 1000, pool - 1 - c.tables, c.tables)
        keep_k, keep_v = c.k, c.v
        n = 200 + new
        at = np.arange(n)
        slots = c.tables[0, at // page] * page + at % page
        rows_k, rows_v = (a[small[0, at // page], at % page] for a in (keep_k, keep_v))
        be.paged_kv_write(kp, vp, floats(be, rows_k, True), floats(be, rows_v, True), u32(be, slots))
        got, lse = c.run(be, kp=kp, vp=vp)
        tables, c.tables = c.tables, small
        want, want_lse = c.run(be)
        assert np.array_equal(got, want) and np.array_equal(lse, want_lse)
        del kp, vp


@pytest.mark.parametrize("d", [16, 32, 48, 80, 96, 112])
@pytest.mark.parametrize("new", [[20, 35], [40, 35], [200, 131]])
def test_many_rows_at_head_dims_below_the_operands(be, d, new):
    """tcgen05 operands of 64 and 128 columns with zeros behind the head's: values next to the head in memory (another head's) stay out."""
    c = Case(51 + d, [700, 90], new, 2, 1, d, 16, True, True, pad=1)
    out, lse = c.check(be)
    again = c.check(be, heads_first=True, workspace=True)
    assert np.array_equal(again[0], out) and np.array_equal(again[1], lse)
    c.masks[:, 0] &= np.uint32(0xFFFFFFF5)                  # a poisoned draft that no row sees
    p, off = c.slot(1, 90 + 1)
    c.k[p, off], c.v[p, off] = np.nan, np.inf
    c.check(be)


FEW = [([700, 90, 0], [1, 1, 1]), ([300, 64], [2, 3]), ([130, 1], [4, 4])]


@pytest.mark.parametrize("cached,new", FEW)
@pytest.mark.parametrize("h,hk", [(2, 2), (4, 2)])
@pytest.mark.parametrize("d,page", [(32, 16), (64, 5), (96, 64), (128, 24)])
@pytest.mark.parametrize("window", [None, 1, 70])
@pytest.mark.parametrize("tree", [True, False])
def test_few_rows_in_f32(be, cached, new, h, hk, d, page, window, tree):
    """One, two and four rows to a KV head (and the eight beyond them), requests with more rows than the average among them."""
    c = Case(60 + d, cached, new, h, hk, d, page, tree, False, words_more=1, pad=1)
    out, lse = c.check(be, window=window)
    again = c.run(be, window=window, workspace=True, heads_first=True)
    assert np.array_equal(again[0], out) and np.array_equal(again[1], lse)
    c.check(be, window=window, use_positions=False)


@pytest.mark.parametrize("h,hk,new", [(2, 2, [4, 1]), (4, 2, [2, 2]), (4, 1, [1, 1]), (3, 3, [4, 4])])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_few_rows_in_f32_that_see_nothing_and_places_that_hold_anything(be, h, hk, new, d):
    c = Case(61 + d, [0, 100], new, h, hk, d, 16, True, False)
    c.masks[:] &= np.uint32(0xFFFFFFFD)                    # draft 1 of each request drops out of every row
    c.masks[0] = 0                                         # request 0 has no cache: its row 0 sees nothing
    for b in range(2):
        if new[b] > 1:
            p, off = c.slot(b, int(c.cached[b]) + 1)
            c.k[p, off], c.v[p, off] = np.nan, np.inf
    out, lse = c.check(be)
    assert not out[0].any() and np.all(np.isneginf(lse[0]))


@pytest.mark.parametrize("requests,cached,h,hk,d,new", [(40, 900, 6, 6, 64, 1), (9, 3000, 2, 2, 128, 2), (150, 61, 3, 1, 96, 1)])
def test_few_rows_in_f32_with_several_units_to_a_share(be, requests, cached, h, hk, d, new):
    rng = np.random.default_rng(62)
    c = Case(62, [int(x) for x in rng.integers(0, cached, requests)], [int(x) for x in rng.integers(0, new + 1, requests - 1)] + [new], h, hk, d, 16, True, False)
    out, lse = c.check(be)
    for _ in range(3):
        again = c.run(be)
        assert np.array_equal(again[0], out) and np.array_equal(again[1], lse)


def test_few_rows_in_f32_with_infinite_scores(be):
    """Every score of a row -inf is NaN in the formula, in one piece and in many; it is reported."""
    from ojas_b200 import OjasError
    for cached in (40, 30000):
        c = Case(63, [cached], [1], 2, 2, 64, 16, False, False)
        q, k = c.q.copy(), c.k.copy()
        q[:, 0, 0], k[..., 0, 0] = -1.0, np.inf
        out, lse = be.paged_attention_forward(floats(be, q, False), floats(be, k, False), floats(be, c.v, False), u32(be, c.tables), u32(be, c.cached), u32(be, c.starts),
                                              lse=be.zeros(c.q.shape[:2]))
        with pytest.raises(OjasError) as e:
            be.sync()
        assert e.value.kind == "NonFinite"
        got = out.numpy()
        assert np.all(np.isnan(got[:, 0])) and np.all(np.isfinite(got[:, 1]))
