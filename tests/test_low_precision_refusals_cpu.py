"""What the 8-bit float and mixture-of-experts entry points refuse, before anything reaches a device (the addresses here are
no memory), and the workspaces they ask for."""
import ctypes as C

import pytest

from vecops_amd import capi

INVALID, NOT_APPLICABLE = 1, 2


def operand(dtype, *shape, strides=None, data=0x10000):
    o = capi.Operand()
    o.data, o.dtype, o.rank = data, dtype, len(shape)
    if strides is None:
        strides, step = [], 1
        for n in reversed(shape):
            strides.insert(0, step)
            step *= n
    for i, (n, s) in enumerate(zip(shape, strides)):
        o.sizes[i], o.strides[i] = n, s
    return o


def refused(rc, code, word):
    assert rc == code, (rc, capi.lib().vecops_hip_last_error())
    assert word in capi.lib().vecops_hip_last_error().decode()


F8, F32, BF16, F16, I32 = capi.F8E4M3, capi.F32, capi.BF16, capi.F16, capi.I32


@pytest.mark.parametrize("changes,code,word", [
    ({"x": operand(capi.I8, 5, 300)}, NOT_APPLICABLE, "x must be"),
    ({"q": operand(capi.I8, 5, 300)}, NOT_APPLICABLE, "q e4m3"),
    ({"q": operand(F8, 5, 299)}, INVALID, "shape"),
    ({"q": operand(F8, 1, 5, 300)}, INVALID, "shape"),
    ({"scales": operand(F32, 5, 2)}, INVALID, "scales must be [5, 3]"),
    ({"scales": operand(BF16, 5, 3)}, INVALID, "f32"),
    ({"rows": 2}, INVALID, "1 or 128"),
    ({"rows": 128}, INVALID, "scales must be [1, 3]"),
    ({"x": operand(BF16, 300)}, INVALID, "rank"),
    ({"x": operand(BF16, 5, 300, data=None)}, INVALID, "null"),
    ({"scales": operand(F32, 5, 3, data=None)}, INVALID, "null"),
    ({"x": operand(BF16, 2 ** 30, 300), "q": operand(F8, 2 ** 30, 300), "scales": operand(F32, 2 ** 30, 3)}, INVALID, "too large"),
    ({"x": operand(BF16, 2 ** 29, 2 ** 20), "q": operand(F8, 2 ** 29, 2 ** 20), "scales": operand(F32, 2 ** 22, 2 ** 13), "rows": 128}, INVALID,
     "too large"),
])
def test_quantize_refusals(changes, code, word):
    a = {"x": operand(BF16, 5, 300), "q": operand(F8, 5, 300), "scales": operand(F32, 5, 3), "rows": 1} | changes
    refused(capi.lib().vecops_hip_quantize_fp8_block(C.byref(a["x"]), a["rows"], C.byref(a["q"]), C.byref(a["scales"]), None), code, word)


@pytest.mark.parametrize("changes,code,word", [
    ({"a": operand(capi.I8, 5, 300)}, NOT_APPLICABLE, "e4m3"),
    ({"c": operand(I32, 5, 200)}, NOT_APPLICABLE, "c f32"),
    ({"b": operand(F8, 200, 301)}, INVALID, "K of a"),
    ({"c": operand(F32, 5, 201)}, INVALID, "c must be"),
    ({"c": operand(F32, 1, 5, 200)}, INVALID, "ranks"),
    ({"sa": operand(F32, 5, 2)}, INVALID, "a_scales must be"),
    ({"sb": operand(F32, 200, 3)}, INVALID, "b_scales must be [ceil(N / 128)=2"),
    ({"sb": operand(BF16, 2, 3)}, INVALID, "f32"),
    ({"sa": operand(F32, 5, 3, strides=(-3, 1))}, NOT_APPLICABLE, "row strides"),
    ({"sa": operand(F32, 5, 3, strides=(2 ** 20 + 1, 1))}, NOT_APPLICABLE, "row strides"),
    ({"a": operand(F8, 5, 300, data=None)}, INVALID, "null"),
    ({"sb": operand(F32, 2, 3, data=None)}, INVALID, "null"),
    ({"b": operand(F8, 200, 300, strides=(1, 200))}, INVALID, "workspace"),
])
def test_matmul_refusals(changes, code, word):
    v = {"a": operand(F8, 5, 300), "sa": operand(F32, 5, 3), "b": operand(F8, 200, 300), "sb": operand(F32, 2, 3), "c": operand(F32, 5, 200)} | changes
    refused(capi.lib().vecops_hip_matmul_fp8_block(*(C.byref(v[n]) for n in ("a", "sa", "b", "sb", "c")), None, 0, None), code, word)


def test_matmul_batches_and_workspace():
    f = capi.lib().vecops_hip_matmul_fp8_block
    v = [operand(F8, 2, 5, 300), operand(F32, 2, 5, 3), operand(F8, 3, 200, 300), operand(F32, 2, 2, 3), operand(F32, 2, 5, 200)]
    refused(f(*map(C.byref, v), None, 0, None), INVALID, "batch")
    def need(*operands):
        c = operand(F32, *operands[0].sizes[:operands[0].rank - 1], operands[2].sizes[operands[2].rank - 2])
        return capi.lib().vecops_hip_matmul_fp8_block_workspace(*map(C.byref, operands), C.byref(c))
    x, sx, sw = operand(F8, 5, 300), operand(F32, 5, 3), operand(F32, 2, 3)
    assert need(x, sx, operand(F8, 200, 300, strides=(333, 1)), sw) == 0
    turned = operand(F8, 200, 300, strides=(1, 200))
    assert need(x, sx, turned, sw) == -(-200 * 304 // 256) * 256
    shared = operand(F8, 7, 200, 300, strides=(0, 1, 200))
    assert need(operand(F8, 7, 5, 300), operand(F32, 7, 5, 3), shared, operand(F32, 7, 2, 3)) == -(-200 * 304 // 256) * 256
    assert need(x, operand(F32, 5, 3, strides=(1, 5)), operand(F8, 200, 300), operand(F32, 2, 3, strides=(1, 2))) == 512
    assert need(operand(F8, 5, 8), operand(F32, 5, 1), operand(F8, 200, 8), operand(F32, 2, 1)) == 256 + 3328
    # few tiles and a long K: the sums of its parts
    assert need(operand(F8, 64, 14336), operand(F32, 64, 112), operand(F8, 4096, 14336), operand(F32, 32, 112)) == 4 * 64 * 4096 * 4
    assert need(operand(F8, 4096, 4096), operand(F32, 4096, 32), operand(F8, 4096, 4096), operand(F32, 32, 32)) == 0
    v = [operand(F8, 5, 300), operand(F32, 5, 3), turned, operand(F32, 2, 3), operand(F32, 5, 200)]
    refused(f(*map(C.byref, v), 0x10008, 1 << 20, None), INVALID, "16-byte aligned workspace")
    refused(f(*map(C.byref, v), 0x10000, 100, None), INVALID, "workspace of")
    # nothing to do: nothing is needed
    v = [operand(F8, 0, 300, data=None), operand(F32, 0, 3, data=None), operand(F8, 200, 300, data=None), operand(F32, 2, 3, data=None),
         operand(F32, 0, 200, data=None)]
    assert f(*map(C.byref, v), None, 0, None) == 0


def layer(**changes):
    t, e, h, i, top = 4, 8, 256, 96, 2
    v = {"x": operand(BF16, t, h), "router": operand(BF16, e, h), "gate_up": operand(BF16, e, 2 * i, h), "gs": None, "down": operand(BF16, e, h, i),
         "ds": None, "ids": operand(I32, t, top), "weights": operand(F32, t, top), "out": operand(BF16, t, h),
         "routing": capi.MoeRouting(C.sizeof(capi.MoeRouting), 0, 1, 1.0, None), "ws": 0x10000, "size": 1 << 24} | changes
    ref = {n: C.byref(o) if isinstance(o, capi.Operand) else o for n, o in v.items()}
    names = ("gate_up", "gs", "down", "ds")
    routing = None if v["routing"] is None else C.byref(v["routing"])
    whole = capi.lib().vecops_hip_moe_layer(ref["x"], ref["router"], routing, *(ref[n] for n in names), ref["ids"], ref["weights"], ref["out"],
                                            v["ws"], v["size"], None)
    return whole


def experts(**changes):
    t, e, h, i, top = 4, 8, 256, 96, 2
    v = {"x": operand(BF16, t, h), "ids": operand(I32, t, top), "weights": operand(F32, t, top), "gate_up": operand(BF16, e, 2 * i, h), "gs": None,
         "down": operand(BF16, e, h, i), "ds": None, "out": operand(BF16, t, h), "ws": 0x10000, "size": 1 << 24} | changes
    ref = [C.byref(v[n]) if v[n] is not None else None for n in ("x", "ids", "weights", "gate_up", "gs", "down", "ds", "out")]
    return capi.lib().vecops_hip_moe_experts(*ref, v["ws"], v["size"], None)


@pytest.mark.parametrize("changes,code,word", [
    ({"x": operand(F32, 4, 256)}, NOT_APPLICABLE, "x must be bf16 or f16"),
    ({"x": operand(BF16, 1, 4, 256)}, INVALID, "rank 2"),
    ({"gate_up": operand(BF16, 16, 256)}, INVALID, "rank 3"),
    ({"gate_up": operand(BF16, 8, 96, 256)}, INVALID, "2 * inner"),
    ({"down": operand(BF16, 7, 256, 96)}, INVALID, "down"),
    ({"down": operand(F16, 8, 256, 96)}, NOT_APPLICABLE, "gate_up and down"),
    ({"gate_up": operand(F16, 8, 192, 256), "down": operand(F16, 8, 256, 96)}, NOT_APPLICABLE, "its type"),
    ({"out": operand(F16, 4, 256)}, NOT_APPLICABLE, "out of its type"),
    ({"out": operand(BF16, 4, 255)}, INVALID, "out must be"),
    ({"ids": operand(capi.I8, 4, 2)}, INVALID, "i32"),
    ({"weights": operand(BF16, 4, 2)}, INVALID, "f32"),
    ({"weights": operand(F32, 4, 3)}, INVALID, "choices"),
    ({"gate_up": operand(F8, 8, 192, 256), "down": operand(F8, 8, 256, 96)}, INVALID, "scales"),
    ({"gate_up": operand(F8, 8, 192, 256), "down": operand(F8, 8, 256, 96), "gs": operand(F32, 8, 2, 2), "ds": operand(F32, 8, 2, 2)}, INVALID,
     "scales must be"),
    ({"gs": operand(F32, 8, 2, 2)}, INVALID, "belong to e4m3"),
    ({"x": operand(BF16, 129, 256), "ids": operand(I32, 129, 2), "weights": operand(F32, 129, 2), "out": operand(BF16, 129, 256)}, NOT_APPLICABLE,
     "128 tokens"),
    ({"ids": operand(I32, 4, 17), "weights": operand(F32, 4, 17)}, NOT_APPLICABLE, "16 choices"),
    ({"gate_up": operand(BF16, 513, 192, 256), "down": operand(BF16, 513, 256, 96), "router": operand(BF16, 513, 256)}, NOT_APPLICABLE, "512 experts"),
    ({"gate_up": operand(BF16, 8, 192, 256, strides=(192 * 256, 1, 192))}, NOT_APPLICABLE, "contiguous"),
    ({"down": operand(BF16, 8, 256, 96, strides=(96 * 256, 1, 256))}, NOT_APPLICABLE, "contiguous"),
    ({"x": operand(BF16, 4, 256, strides=(1, 4))}, NOT_APPLICABLE, "contiguous"),
    ({"x": operand(BF16, 4, 256, data=None)}, INVALID, "null"),
    ({"down": operand(BF16, 8, 256, 96, data=None)}, INVALID, "null"),
    ({"ws": None}, INVALID, "workspace"),
    ({"ws": 0x10004}, INVALID, "16-byte aligned"),
    ({"size": 64}, INVALID, "workspace of"),
])
def test_experts_and_layer_refusals(changes, code, word):
    refused(layer(**changes), code, word)
    refused(experts(**{n: o for n, o in changes.items() if n != "router"}), code, word)


@pytest.mark.parametrize("changes,code,word", [
    ({"router": operand(BF16, 7, 256)}, INVALID, "router must be"),
    ({"router": operand(F16, 8, 256)}, NOT_APPLICABLE, "x's type or f32"),
    ({"router": operand(F32, 8, 256, strides=(1, 8))}, NOT_APPLICABLE, "rows of router"),
    ({"router": operand(F32, 8, 256, data=None)}, INVALID, "null"),
    ({"routing": None}, INVALID, "routing record"),
    ({"routing": capi.MoeRouting(4, 0, 1, 1.0, None)}, INVALID, "routing record"),
    ({"routing": capi.MoeRouting(C.sizeof(capi.MoeRouting), 2, 1, 1.0, None)}, INVALID, "scoring"),
    ({"ids": operand(I32, 4, 9), "weights": operand(F32, 4, 9)}, INVALID, "9 choices among 8"),
])
def test_layer_refusals(changes, code, word):
    refused(layer(**changes), code, word)


def test_nothing_to_do():
    none = {"x": operand(BF16, 0, 256, data=None), "ids": operand(I32, 0, 2, data=None), "weights": operand(F32, 0, 2, data=None),
            "out": operand(BF16, 0, 256, data=None), "ws": None, "size": 0}
    assert layer(**none) == 0 and experts(**none) == 0


def test_tensors_that_are_not_on_a_gpu():
    """The kernels read through plain addresses: the Python entry points refuse tensors in host memory, or on two devices."""
    torch = pytest.importorskip("torch")
    x, q, s = torch.zeros(4, 128), torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.zeros(4, 1)
    with pytest.raises(ValueError, match="one GPU"):
        capi.quantize_fp8_block(x, q, s)
    with pytest.raises(ValueError, match="one GPU"):
        capi.matmul_fp8_block(q, s, q, torch.zeros(1, 1), torch.zeros(4, 4))
    ids, weights, experts = torch.zeros((4, 1), dtype=torch.int32), torch.zeros(4, 1), torch.zeros(2, 16, 128)
    with pytest.raises(ValueError, match="one GPU"):
        capi.moe_experts(x.bfloat16(), ids, weights, experts.bfloat16(), torch.zeros(2, 128, 8).bfloat16(), x)
    with pytest.raises(ValueError, match="one GPU"):
        capi.moe_layer(x.bfloat16(), torch.zeros(2, 128), experts.bfloat16(), torch.zeros(2, 128, 8).bfloat16(), ids, weights, x)
    with pytest.raises(ValueError, match="bias"):
        capi.moe_layer(x.bfloat16(), torch.zeros(2, 128), experts.bfloat16(), torch.zeros(2, 128, 8).bfloat16(), ids, weights, x,
                       bias=torch.zeros(3))
