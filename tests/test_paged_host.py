"""Host half of the paged-cache operators, without a device: rotary frequencies, and every refusal the host makes before a launch. The refusals run
against a stand-in handle (zeroed memory of a backend's size, which the checks never look into): nothing valid is ever passed, so nothing launches."""
import ctypes as C

import numpy as np
import pytest

import paged_reference as ref
from ojas_b200 import CudaBackend, DType, OjasError, RopeSpec, Tensor
from ojas_b200._lib import lib
from ojas_b200.backend import STATUS_NAMES, _p


def kind(status):
    return STATUS_NAMES[status]


@pytest.fixture(scope="module")
def handle():
    return C.create_string_buffer(1 << 16)


def t(shape, dtype=DType.F32, strides=None, ptr=256):
    return Tensor(None, ptr, shape, dtype, strides, owner=True)


@pytest.mark.parametrize("kw", [dict(), dict(base=500000.0), dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
                                dict(scaling="by_turns", factor=8.0, original_length=4096.0), dict(scaling="by_turns", factor=32.0, original_length=8192.0, low_turns=1.0, high_turns=4.0)])
@pytest.mark.parametrize("rotary", [8, 64, 256])
def test_rope_frequencies(rotary, kw):
    rope = CudaBackend.rope_plan(RopeSpec(rotary, amplitude=1.25, layout="interleaved", **kw))
    want = ref.frequencies(rotary, kw.get("base", 10000.0), kw.get("scaling", "none"), kw.get("factor", 1.0), kw.get("original_length", 0.0), kw.get("low_turns", 1.0),
                           kw.get("high_turns", 32.0))
    got = np.array([rope.turns[i] for i in range(rotary // 2)], np.float64) * 2.0 ** -64 * 2 * np.pi
    # numpy's pow, exp and products are good to a few units of 2^-53; by_turns cancels at most a factor of 32 / 31
    assert np.all(np.abs(got - want) <= 2.0 ** -47 * want + 2.0 ** -60)
    assert rope.rotary_dim == rotary and rope.layout == 1 and rope.amplitude == 1.25 and not any(rope.turns[rotary // 2:])


@pytest.mark.parametrize("spec,want", [
    (RopeSpec(0), "Shape"), (RopeSpec(7), "Shape"), (RopeSpec(-2), "Shape"), (RopeSpec(258), "Unsupported"), (RopeSpec(8, base=0.5), "OutOfRange"),
    (RopeSpec(8, base=float("nan")), "OutOfRange"), (RopeSpec(8, amplitude=float("inf")), "OutOfRange"), (RopeSpec(8, scaling="linear", factor=0.5), "OutOfRange"),
    (RopeSpec(8, scaling="linear", factor=float("nan")), "OutOfRange"), (RopeSpec(2, scaling="base", factor=2.0), "OutOfRange"),
    (RopeSpec(8, scaling="by_turns", factor=2.0), "OutOfRange"), (RopeSpec(8, scaling="by_turns", factor=2.0, original_length=64.0, low_turns=4.0, high_turns=4.0), "OutOfRange")])
def test_rope_plan_refusals(spec, want):
    with pytest.raises(OjasError) as e:
        CudaBackend.rope_plan(spec)
    assert e.value.kind == want


def test_null_handles_and_pointers_are_errors_not_crashes():
    assert kind(lib.ojc_rope_plan(None, None)) == "Backend"
    assert kind(lib.ojc_rope_forward(None, None, None, None, None)) == "Backend"
    assert kind(lib.ojc_paged_plan(*([None] * 6), C.c_int64(16), *([None] * 6))) == "Backend"
    assert kind(lib.ojc_paged_kv_write(*([None] * 8))) == "Backend"
    assert kind(lib.ojc_paged_attention_workspace_bytes(None, None, None, None)) == "Backend"
    assert kind(lib.ojc_paged_attention_forward(*([None] * 9), C.c_int64(-1), *([None] * 3), C.c_uint64(0))) == "Backend"


def test_rope_refusals(handle):
    rope = CudaBackend.rope_plan(RopeSpec(64))
    u32 = DType.U32

    def run(x, positions, y, plan=rope, fn=lib.ojc_rope_forward):
        return kind(fn(handle, C.byref(plan) if plan is not None else None, _p(x), _p(positions), _p(y)))
    x = t((5, 2, 64))
    assert run(x, t((5,), u32), None) == "Shape"
    assert run(x, t((5,), u32), t((5, 2, 32))) == "Shape"
    assert run(t((5, 64)), t((5,), u32), t((5, 64))) == "Shape"
    assert run(x, t((5,), u32), t((5, 2, 64), DType.BF16)) == "Dtype"
    assert run(t((5, 2, 64), DType.F16), t((5,), u32), t((5, 2, 64), DType.F16)) == "Dtype"
    assert run(x, t((5,)), x) == "Dtype"
    assert run(x, t((4,), u32), x) == "Shape"
    assert run(t((2, 5, 2, 64)), t((2,), u32), t((2, 5, 2, 64))) == "Shape"          # neither T nor B * T
    assert run(t((0, 2, 64)), t((0,), u32), t((0, 2, 64))) == "Shape"
    assert run(t((5, 2, 32)), t((5,), u32), t((5, 2, 32))) == "Shape"                # rotary_dim above the head dim
    assert run(t((5, 2, 64), strides=(128, 1, 2)), t((5,), u32), x) == "Shape"
    assert run(t((5, 2, 64), ptr=0), t((5,), u32), x) == "Placement"
    assert run(x, t((5,), u32), x, plan=None) == "Backend"
    empty = type(rope)()
    assert run(x, t((5,), u32), x, plan=empty) == "Backend"
    assert run(x, t((4,), u32), x, fn=lib.ojc_rope_backward) == "Shape"


def test_paged_plan_refusals(handle):
    u32 = DType.U32
    good = dict(cached=t((3,), u32), new=t((3,), u32), parents=t((10,), u32), free=t((9,), u32), head=t((1,), u32), page=16, tables=t((3, 4), u32), starts=t((4,), u32),
                slots=t((10,), u32), positions=t((10,), u32), masks=t((10, 1), u32), out=t((1,), u32, ptr=512))

    def run(**kw):
        a = dict(good, **kw)
        return kind(lib.ojc_paged_plan(handle, _p(a["cached"]), _p(a["new"]), _p(a["parents"]), _p(a["free"]), _p(a["head"]), C.c_int64(a["page"]), _p(a["tables"]), _p(a["starts"]),
                                       _p(a["slots"]), _p(a["positions"]), _p(a["masks"]), _p(a["out"])))
    for name in ("cached", "new", "free", "head", "tables", "starts", "slots", "positions", "out"):
        assert run(**{name: None}) == "Shape", name
        g = good[name]
        assert run(**{name: t(g.shape, DType.F32)}) == "Dtype", name
        if name not in ("free",):
            assert run(**{name: t(tuple(s + 1 for s in g.shape), u32)}) == "Shape", name
    assert run(parents=t((9,), u32)) == "Shape" and run(masks=t((9, 1), u32)) == "Shape" and run(masks=t((10, 0), u32)) == "Shape" and run(masks=t((10, 1))) == "Dtype"
    assert run(page=0) == "OutOfRange" and run(page=(1 << 24) + 1) == "OutOfRange"
    assert run(out=good["head"]) == "Shape"
    assert run(tables=t((3, 4), u32, strides=(8, 1))) == "Shape"
    big = 24001
    assert run(cached=t((big,), u32), new=t((big,), u32), tables=t((big, 4), u32), starts=t((big + 1,), u32)) == "Unsupported"
    zero = dict(slots=t((0,), u32), positions=t((0,), u32), parents=None, masks=None)
    assert run(**zero) == "Shape"


def test_paged_kv_write_refusals(handle):
    u32 = DType.U32
    rope = CudaBackend.rope_plan(RopeSpec(64))
    good = dict(kp=t((8, 16, 2, 64), DType.BF16), vp=t((8, 16, 2, 64), DType.BF16), k=t((5, 2, 64)), v=t((5, 2, 64)), slots=t((5,), u32), rope=rope, positions=t((5,), u32))

    def run(**kw):
        a = dict(good, **kw)
        return kind(lib.ojc_paged_kv_write(handle, _p(a["kp"]), _p(a["vp"]), _p(a["k"]), _p(a["v"]), _p(a["slots"]), C.byref(a["rope"]) if a["rope"] else None, _p(a["positions"])))
    for name in ("kp", "vp", "k", "v", "slots", "positions"):
        assert run(**{name: None}) == "Shape", name
    assert run(vp=t((8, 16, 2, 64))) == "Dtype" and run(v=t((5, 2, 64), DType.BF16)) == "Dtype" and run(slots=t((5,))) == "Dtype"
    assert run(k=t((5, 2, 64), DType.F16), v=t((5, 2, 64), DType.F16)) == "Dtype"
    assert run(k=t((5, 3, 64)), v=t((5, 3, 64))) == "Shape" and run(k=t((5, 2, 32)), v=t((5, 2, 32))) == "Shape" and run(slots=t((4,), u32)) == "Shape"
    assert run(k=t((5, 2, 64), strides=(128, 1, 2))) == "Shape" and run(kp=t((8, 16, 2, 64), DType.BF16, strides=(2048, 128, 1, 2))) == "Shape"
    assert run(k=t((0, 2, 64)), v=t((0, 2, 64)), slots=t((0,), u32), positions=t((0,), u32)) == "Shape"
    huge = t((1 << 28, 16, 2, 64), DType.BF16)
    assert run(kp=huge, vp=huge) == "OutOfRange"
    assert run(kp=t((8, 16, 2, 32), DType.BF16), vp=t((8, 16, 2, 32), DType.BF16), k=t((5, 2, 32)), v=t((5, 2, 32))) == "Shape"   # rotary_dim above the head dim


def test_paged_attention_refusals(handle):
    u32, b16 = DType.U32, DType.BF16
    good = dict(q=t((6, 4, 64), b16), kp=t((8, 16, 2, 64), b16), vp=t((8, 16, 2, 64), b16), tables=t((3, 4), u32), cached=t((3,), u32), starts=t((4,), u32), masks=t((6, 1), u32),
                positions=t((6,), u32), window=-1, out=t((6, 4, 64), b16), lse=t((6, 4)), work=256, size=16)

    def run(**kw):
        a = dict(good, **kw)
        return kind(lib.ojc_paged_attention_forward(handle, _p(a["q"]), _p(a["kp"]), _p(a["vp"]), _p(a["tables"]), _p(a["cached"]), _p(a["starts"]), _p(a["masks"]), _p(a["positions"]),
                                                    C.c_int64(a["window"]), _p(a["out"]), _p(a["lse"]), C.c_void_p(a["work"]), C.c_uint64(a["size"])))
    for name in ("q", "kp", "vp", "tables", "cached", "starts", "out"):
        assert run(**{name: None}) == "Shape", name
    assert run() == "Shape"                                                          # a workspace of 16 bytes
    assert run(work=264, size=1 << 40) == "Shape"                                     # not 256-byte aligned
    for name in ("vp", "out"):
        assert run(**{name: t(good[name].shape, DType.F32)}) == "Dtype", name
    assert run(q=t((6, 4, 64))) == "Dtype"
    for name in ("tables", "cached", "starts", "masks", "positions"):
        assert run(**{name: t(good[name].shape, DType.F32)}) == "Dtype", name
    assert run(lse=t((6, 4), b16)) == "Shape" and run(lse=t((6, 3))) == "Shape"
    assert run(q=t((6, 3, 64), b16), out=t((6, 3, 64), b16)) == "Shape"
    assert run(tables=t((2, 4), u32)) == "Shape" and run(starts=t((3,), u32)) == "Shape" and run(masks=t((5, 1), u32)) == "Shape" and run(positions=t((5,), u32)) == "Shape"
    assert run(window=0) == "OutOfRange"
    assert run(q=t((6, 4, 64), b16, strides=(256, 1, 4))) == "Shape"
    wide = t((8, 16, 2, 264), b16)
    assert run(q=t((6, 4, 264), b16), kp=wide, vp=wide, out=t((6, 4, 264), b16)) == "UnsupportedHeadDim"
    f16 = dict(q=t((6, 4, 64), DType.F16), kp=t((8, 16, 2, 64), DType.F16), vp=t((8, 16, 2, 64), DType.F16), out=t((6, 4, 64), DType.F16))
    assert run(**f16) == "Dtype"
    assert run(q=t((0, 4, 64), b16), out=t((0, 4, 64), b16), masks=None, positions=t((0,), u32), lse=t((0, 4))) == "Shape"
    assert run(tables=t((3, 0), u32)) == "Shape"


def test_python_plan_wants_a_capacity():
    be = CudaBackend.__new__(CudaBackend)
    be._handle = None
    with pytest.raises(OjasError) as e:
        be.paged_plan(t((3,), DType.U32), t((3,), DType.U32), t((9,), DType.U32), t((1,), DType.U32), t((3, 4), DType.U32), 16)
    assert e.value.kind == "Shape"


def test_what_is_written_cannot_be_a_broadcast_view(handle):
    u32, b16, rope = DType.U32, DType.BF16, CudaBackend.rope_plan(RopeSpec(64))
    x, flat = t((5, 2, 64)), t((5, 2, 64), strides=(64, 0, 1))
    assert kind(lib.ojc_rope_forward(handle, C.byref(rope), _p(x), _p(t((5,), u32)), _p(flat))) == "Shape" and "broadcast" in lib.ojc_last_error().decode()
    pages, flat = t((8, 16, 2, 64)), t((8, 16, 2, 64), strides=(1024, 64, 0, 1))
    for kp, vp in ((flat, pages), (pages, flat)):
        assert kind(lib.ojc_paged_kv_write(handle, _p(kp), _p(vp), _p(x), _p(x), _p(t((5,), u32)), None, None)) == "Shape" and "broadcast" in lib.ojc_last_error().decode()
    got = lib.ojc_paged_attention_forward(handle, _p(t((6, 4, 64), b16)), _p(t((8, 16, 2, 64), b16)), _p(t((8, 16, 2, 64), b16)), _p(t((3, 4), u32)), _p(t((3,), u32)), _p(t((4,), u32)),
                                          None, None, C.c_int64(-1), _p(t((6, 4, 64), b16, strides=(0, 64, 1))), None, C.c_void_p(256), C.c_uint64(1 << 40))
    assert kind(got) == "Shape" and "broadcast" in lib.ojc_last_error().decode()


def test_a_changed_tensor_is_passed_as_it_is_now():
    x = t((5, 2, 64))
    assert _p(x)._obj.data == 256 and _p(x) is _p(x)
    x.ptr, x.shape, x.strides = 512, (5, 2, 32), (128, 64, 1)
    assert _p(x)._obj.data == 512 and list(_p(x)._obj.shape[:3]) == [5, 2, 32] and list(_p(x)._obj.stride[:3]) == [128, 64, 1]


def test_paged_plan_held_refusals(handle):
    u32 = DType.U32

    def run(held, out, batch=3):
        a = [t((3,), u32), t((3,), u32), held, None, t((9,), u32), t((1,), u32)]
        return kind(lib.ojc_paged_plan_held(handle, *[_p(x) for x in a], C.c_int64(16), _p(t((batch, 4), u32)), _p(out), _p(t((4,), u32)), _p(t((10,), u32)), _p(t((10,), u32)), None,
                                            _p(t((1,), u32, ptr=512))))
    good = t((3,), u32, ptr=1024)
    assert run(None, good) == "Shape" and run(good, None) == "Shape"
    assert run(t((3,)), good) == "Dtype" and run(t((3,), u32), t((3,), ptr=1024)) == "Dtype"
    assert run(t((2,), u32), t((2,), u32, ptr=1024)) == "Shape" and run(t((3,), u32), t((4,), u32, ptr=1024)) == "Shape" and run(t((3, 1), u32), good) == "Shape"
    assert run(good, t((3,), u32, ptr=1024)) == "Shape" and "another tensor" in lib.ojc_last_error().decode()
    assert run(t((3,), u32), good, batch=2) == "Shape"
    assert kind(lib.ojc_paged_plan_held(*([None] * 7), C.c_int64(16), *([None] * 7))) == "Backend"
    be = CudaBackend.__new__(CudaBackend)
    be._handle = None
    with pytest.raises(OjasError) as e:
        be.paged_plan(*[t((3,), u32)] * 4, t((3, 4), u32), 16, tokens=4, starts=t((4,), u32), slots=t((4,), u32), positions=t((4,), u32), free_head_out=t((1,), u32), held_pages_out=good)
    assert e.value.kind == "Shape"


def test_an_amplitude_that_f32_does_not_hold_is_refused():
    assert CudaBackend.rope_plan(RopeSpec(8, amplitude=3.4e38)).amplitude == np.float32(3.4e38)
    for amplitude in (1e39, -1e39, 1e300):
        with pytest.raises(OjasError) as e:
            CudaBackend.rope_plan(RopeSpec(8, amplitude=amplitude))
        assert e.value.kind == "OutOfRange"
