"""What the microscaled and row entry points refuse, before anything reaches a device (the addresses here are no memory), and the
workspaces they ask for."""
import ctypes as C

import pytest

from test_low_precision_refusals_cpu import operand, refused
from vecops_amd import capi

INVALID, NOT_APPLICABLE = 1, 2
F4, F8, E8, F32, BF16, F16, I8 = capi.F4E2M1X2, capi.F8E4M3, capi.F8E8M0, capi.F32, capi.BF16, capi.F16, capi.I8
ref = lambda o: None if o is None else C.byref(o)  # noqa: E731


@pytest.mark.parametrize("changes,code,word", [
    ({"x": operand(I8, 5, 300)}, NOT_APPLICABLE, "must be f32"),
    ({"q": operand(I8, 5, 300)}, NOT_APPLICABLE, "e2m1"),
    ({"q": operand(F4, 5, 300)}, INVALID, "shape"),
    ({"q": operand(F8, 5, 299)}, INVALID, "shape"),
    ({"q": operand(F8, 1, 5, 300)}, INVALID, "shape"),
    ({"scales": operand(E8, 5, 3)}, INVALID, "scales must be [5, 10]"),
    ({"scales": operand(F32, 5, 10)}, INVALID, "e8m0"),
    ({"x": operand(BF16, 5, 301), "q": operand(F4, 5, 150)}, INVALID, "even"),
    ({"x": operand(BF16, 300)}, INVALID, "rank"),
    ({"x": operand(BF16, 5, 300, data=None)}, INVALID, "null"),
    ({"q": operand(F8, 5, 300, data=None)}, INVALID, "null"),
    ({"scales": operand(E8, 5, 10, data=None)}, INVALID, "null"),
    ({"x": operand(BF16, 2 ** 30, 300), "q": operand(F8, 2 ** 30, 300), "scales": operand(E8, 2 ** 30, 10)}, INVALID, "too large"),
])
def test_copies(changes, code, word):
    v = {"x": operand(BF16, 5, 300), "q": operand(F8, 5, 300), "scales": operand(E8, 5, 10)} | changes
    refused(capi.lib().vecops_hip_quantize_mx(ref(v["x"]), ref(v["q"]), ref(v["scales"]), None), code, word)
    refused(capi.lib().vecops_hip_dequantize_mx(ref(v["q"]), ref(v["scales"]), ref(v["x"]), None), code, word)


def product(**changes):
    return {"a": operand(F4, 5, 320), "sa": operand(E8, 5, 20), "b": operand(F4, 200, 320), "sb": operand(E8, 200, 20), "c": operand(F32, 5, 200)} | changes


@pytest.mark.parametrize("changes,code,word", [
    ({"a": operand(I8, 5, 640)}, NOT_APPLICABLE, "e2m1"),
    ({"b": operand(F8, 200, 640)}, NOT_APPLICABLE, "b e2m1"),
    ({"c": operand(I8, 5, 200)}, NOT_APPLICABLE, "c f32"),
    ({"b": operand(F4, 200, 321)}, INVALID, "K of a"),
    ({"a": operand(F8, 5, 320)}, INVALID, "K of a (320) and b (640)"),
    ({"c": operand(F32, 5, 201)}, INVALID, "c must be"),
    ({"c": operand(F32, 1, 5, 200)}, INVALID, "ranks"),
    ({"sa": operand(E8, 5, 19)}, INVALID, "a_scales must be"),
    ({"sb": operand(E8, 7, 20)}, INVALID, "b_scales must be [N=200"),
    ({"sb": operand(F32, 200, 20)}, INVALID, "e8m0"),
    ({"a": operand(F4, 5, 320, data=None)}, INVALID, "null"),
    ({"sb": operand(E8, 200, 20, data=None)}, INVALID, "null"),
    ({"c": operand(F32, 5, 200, data=None)}, INVALID, "null"),
    ({"b": operand(F4, 200, 320, strides=(1, 200))}, INVALID, "workspace"),
    ({"sa": operand(E8, 5, 20, strides=(2 ** 20 + 1, 1))}, INVALID, "workspace"),
    ({"a": operand(F4, 5, 320, strides=(-320, 1))}, INVALID, "workspace"),
    ({"b": operand(F4, 200, 320, strides=(319, 1))}, INVALID, "workspace"),
    ({"sb": operand(E8, 200, 20, strides=(1, 1))}, INVALID, "workspace"),
])
def test_matmul(changes, code, word):
    v = product(**changes)
    refused(capi.lib().vecops_hip_matmul_mx(*(ref(v[n]) for n in ("a", "sa", "b", "sb", "c")), None, 0, None), code, word)


def test_matmul_batches_extents_and_workspace():
    f, need = capi.lib().vecops_hip_matmul_mx, capi.lib().vecops_hip_matmul_mx_workspace
    names = ("a", "sa", "b", "sb", "c")
    asked = lambda **changes: need(*(ref(product(**changes)[n]) for n in names))  # noqa: E731
    v = [operand(F4, 2, 5, 320), operand(E8, 2, 5, 20), operand(F4, 3, 200, 320), operand(E8, 2, 200, 20), operand(F32, 2, 5, 200)]
    refused(f(*map(C.byref, v), None, 0, None), INVALID, "batch")
    assert need(*map(C.byref, v)) == 0
    assert asked() == 0
    assert asked(b=operand(F4, 200, 320, strides=(353, 1))) == 0
    assert asked(b=operand(F4, 200, 320, strides=(0, 1)), sb=operand(E8, 200, 20, strides=(0, 1))) == 0
    # a single row's stride says nothing
    assert asked(a=operand(F4, 1, 320, strides=(1, 1)), sa=operand(E8, 1, 20, strides=(1 << 40, 1)), c=operand(F32, 1, 200)) == 0
    up = lambda n: -(-n // 256) * 256  # noqa: E731
    assert asked(b=operand(F4, 200, 320, strides=(1, 200))) == up(200 * 320)
    assert asked(sa=operand(E8, 5, 20, strides=(1, 5))) == up(5 * 20)
    # a K of no whole blocks: both operands padded; scales of rows apart: in place, however few
    assert asked(a=operand(F4, 5, 319), b=operand(F4, 200, 319)) == up(5 * 320) + up(200 * 320)
    assert asked(a=operand(F8, 5, 638), b=operand(F4, 200, 319)) == up(5 * 640) + up(200 * 320)
    assert asked(a=operand(F4, 5, 32), sa=operand(E8, 5, 2), b=operand(F4, 200, 32), sb=operand(E8, 200, 2)) == 0
    # the largest tiles read sixteen scales of a row at once
    assert asked(a=operand(F8, 2050, 224), sa=operand(E8, 2050, 7), b=operand(F4, 4100, 112), sb=operand(E8, 4100, 7), c=operand(BF16, 2050, 4100)) == up(2050 * 16) + up(4100 * 16)
    shared = product(a=operand(F4, 7, 5, 320), sa=operand(E8, 7, 5, 20), b=operand(F4, 7, 200, 320, strides=(0, 1, 200)),
                     sb=operand(E8, 7, 200, 20), c=operand(F32, 7, 5, 200))
    assert need(*(ref(shared[n]) for n in names)) == up(200 * 320)
    v = product(b=operand(F4, 200, 320, strides=(1, 200)))
    refused(f(*(ref(v[n]) for n in names), 0x10008, 1 << 20, None), INVALID, "16-byte aligned workspace")
    refused(f(*(ref(v[n]) for n in names), 0x10000, 100, None), INVALID, "workspace of")
    long = 1 << 26
    v = product(a=operand(F8, 300, long), sa=operand(E8, 300, long // 32), b=operand(F4, 300, long // 2), sb=operand(E8, 300, long // 32), c=operand(BF16, 300, 300))
    refused(f(*(ref(v[n]) for n in names), None, 0, None), NOT_APPLICABLE, "too long")
    v = product(b=operand(F4, 1 << 28, 320), sb=operand(E8, 1 << 28, 20), c=operand(F32, 5, 1 << 28))
    refused(f(*(ref(v[n]) for n in names), None, 0, None), INVALID, "too large")
    # nothing to do: nothing is needed
    v = product(a=operand(F4, 0, 320, data=None), sa=operand(E8, 0, 20, data=None), c=operand(F32, 0, 200, data=None))
    assert f(*(ref(v[n]) for n in names), None, 0, None) == 0


def norm(**changes):
    v = {"x": operand(BF16, 5, 300), "weight": operand(BF16, 300), "residual": None, "summed": None, "q": operand(I8, 5, 300), "scales": operand(F32, 5, 1),
         "out": None} | changes
    return capi.lib().vecops_hip_rms_norm(ref(v["x"]), ref(v["weight"]), 1e-6, *(ref(v[n]) for n in ("residual", "summed", "q", "scales", "out")), None)


@pytest.mark.parametrize("changes,code,word", [
    ({"x": operand(I8, 5, 300)}, NOT_APPLICABLE, "x must be"),
    ({"x": operand(BF16, 300)}, INVALID, "rank"),
    ({"x": operand(BF16, 5, 300, strides=(1, 5))}, NOT_APPLICABLE, "rows of x"),
    ({"weight": None}, INVALID, "weight"),
    ({"weight": operand(BF16, 299)}, INVALID, "weight must be a contiguous vector of 300"),
    ({"weight": operand(BF16, 300, strides=(2,))}, INVALID, "weight"),
    ({"weight": operand(BF16, 1, 300)}, INVALID, "weight"),
    ({"weight": operand(F16, 300)}, NOT_APPLICABLE, "weight must be of x's type"),
    ({"weight": operand(F32, 300, data=None)}, INVALID, "null"),
    ({"x": operand(BF16, 5, 300, data=None)}, INVALID, "null"),
    ({"summed": operand(BF16, 5, 300)}, INVALID, "residual"),
    ({"residual": operand(F32, 5, 300)}, NOT_APPLICABLE, "residual must be of x's type"),
    ({"residual": operand(BF16, 5, 301)}, INVALID, "residual must have x's shape"),
    ({"residual": operand(BF16, 5, 300), "summed": operand(BF16, 1, 5, 300)}, INVALID, "summed must have x's shape"),
    ({"residual": operand(BF16, 5, 300, strides=(1, 5))}, NOT_APPLICABLE, "rows of residual"),
    ({"residual": operand(BF16, 5, 300, data=None)}, INVALID, "null"),
    ({"out": operand(F32, 5, 300)}, NOT_APPLICABLE, "out must be of x's type"),
    ({"out": operand(BF16, 5, 300, strides=(600, 2))}, NOT_APPLICABLE, "rows of out"),
    ({"q": None}, INVALID, "come together"),
    ({"scales": None}, INVALID, "come together"),
    ({"q": None, "scales": None}, INVALID, "no result"),
    ({"q": operand(F4, 5, 150)}, NOT_APPLICABLE, "int8 and f32"),
    ({"scales": operand(E8, 5, 10)}, NOT_APPLICABLE, "int8 and f32"),
    ({"q": operand(I8, 5, 299)}, INVALID, "q must be [5, 300]"),
    ({"scales": operand(F32, 5, 3)}, INVALID, "scales must be [5, 1]"),
    ({"q": operand(F8, 5, 300)}, INVALID, "scales must be [5, 3]"),
    ({"q": operand(F8, 5, 300), "scales": operand(E8, 5, 3)}, INVALID, "scales must be [5, 10]"),
    ({"q": operand(I8, 1, 5, 300)}, INVALID, "rank"),
    ({"q": operand(I8, 5, 300, strides=(1, 5))}, NOT_APPLICABLE, "rows of q"),
    ({"q": operand(I8, 5, 300, data=None)}, INVALID, "null"),
    ({"scales": operand(F32, 5, 1, data=None)}, INVALID, "null"),
    ({"x": operand(BF16, 5, 301), "weight": operand(F32, 301), "q": operand(F4, 5, 150), "scales": operand(E8, 5, 10)}, INVALID, "even"),
    ({"x": operand(BF16, 2 ** 16, 2 ** 16, 8), "weight": operand(F32, 8), "q": operand(I8, 2 ** 16, 2 ** 16, 8), "scales": operand(F32, 2 ** 16, 2 ** 16, 1)},
     INVALID, "too large"),
])
def test_norm(changes, code, word):
    refused(norm(**changes), code, word)


def test_nothing_to_norm():
    empty = {"x": operand(BF16, 0, 300, data=None), "q": operand(I8, 0, 300, data=None), "scales": operand(F32, 0, 1, data=None)}
    assert norm(**empty) == 0
    assert norm(x=operand(BF16, 5, 0), weight=operand(F32, 0), q=operand(I8, 5, 0), scales=operand(F32, 5, 1)) == 0


@pytest.mark.parametrize("changes,code,word", [
    ({"x": operand(I8, 5, 600)}, NOT_APPLICABLE, "gate_up must be"),
    ({"x": operand(BF16, 5, 601)}, INVALID, "gates and as many"),
    ({"x": operand(BF16, 600)}, INVALID, "rank"),
    ({"x": operand(BF16, 5, 600, strides=(1, 5))}, NOT_APPLICABLE, "rows of gate_up"),
    ({"x": operand(BF16, 5, 600, data=None)}, INVALID, "null"),
    ({"q": operand(I8, 5, 600)}, INVALID, "q must be [5, 300]"),
    ({"q": operand(F8, 5, 300)}, INVALID, "scales must be [5, 3]"),
    ({"q": operand(F4, 5, 300)}, NOT_APPLICABLE, "int8 and f32"),
    ({"q": operand(I8, 5, 300, strides=(1, 5))}, NOT_APPLICABLE, "rows of q"),
    ({"x": operand(BF16, 5, 602), "q": operand(F4, 5, 150), "scales": operand(E8, 5, 10)}, INVALID, "even"),
    ({"q": None}, INVALID, "rank"),
])
def test_gate(changes, code, word):
    v = {"x": operand(BF16, 5, 600), "q": operand(I8, 5, 300), "scales": operand(F32, 5, 1)} | changes
    refused(capi.lib().vecops_hip_silu_mul_quantize(ref(v["x"]), ref(v["q"]), ref(v["scales"]), None), code, word)
