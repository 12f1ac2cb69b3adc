"""Where the 8-bit float and mixture-of-experts entry points end, before anything reaches a device (the addresses here are no
memory)."""
import ctypes as C

import pytest

from vecops_amd import capi

from test_low_precision_refusals_cpu import BF16, F8, F32, INVALID, NOT_APPLICABLE, operand, refused


def product(m, n, k, out=BF16, **strides):
    """Operands of a product of dense scales; `a` and `b` may have row strides of their own."""
    groups = -(-k // 128)
    a = operand(F8, m, k, strides=(strides.get("a", k), 1))
    b = operand(F8, n, k, strides=(strides.get("b", k), 1))
    return [a, operand(F32, m, groups), b, operand(F32, -(-n // 128), groups), operand(out, m, n)]


def multiply(operands, workspace=None, size=0):
    return capi.lib().vecops_hip_matmul_fp8_block(*map(C.byref, operands), workspace, size, None)


def need(operands):
    return capi.lib().vecops_hip_matmul_fp8_block_workspace(*map(C.byref, operands))


@pytest.mark.parametrize("m,n,k,out", [
    (17, 64, 2 ** 26, BF16), (17, 64, 2 ** 26, F32), (64, 64, 2 ** 27, BF16), (64, 64, 2 ** 25, F32),   # tiles of 64 rows
    (1024, 1024, 2 ** 24 + 100, BF16), (1024, 1024, 2 ** 24 + 100, F32),   # of 128 and more
    (2048, 2048, 2 ** 23, BF16),   # of 256
    (16, 16384, 2 ** 25, BF16), (1, 64, 2 ** 27, F32)])   # few rows of activations, 64 and 16 of weights
def test_rows_that_no_offset_spans(m, n, k, out):
    """The kernels reach a tile's rows from the first one by offsets below 2^31, and a copy of contiguous rows is as long as they
    are: such a K is refused."""
    refused(multiply(product(m, n, k, out), 0x10000, 1 << 62), NOT_APPLICABLE, "too long")


def test_rows_that_an_offset_spans_are_taken_as_they_are():
    """Up to there rows are read where they lie, however many K are: nothing but sums of parts of K needs a workspace."""
    assert need(product(1, 256, 2 ** 24)) == 0
    assert need(product(16, 64, 2 ** 26)) == 0
    assert need(product(1, 64, 4096, b=2 ** 27)) == 0   # 15 of them and a row
    # rows that lie further apart than that, but are no longer, are copied
    apart = product(1, 64, 4096, b=2 ** 28)
    assert need(apart) == 64 * 4096
    refused(multiply(apart), INVALID, "workspace of")
    apart = product(1000, 1000, 4096, a=2 ** 22, b=2 ** 62)
    assert need(apart) == 1000 * 4096
    refused(multiply(apart), INVALID, "workspace of")


I32, F16 = capi.I32, capi.F16


def moe_need(tokens=4, top=2, experts=8, hidden=256, inner=96, dtype=BF16):
    """(experts, layer): what the queries say."""
    x, ids, down = operand(dtype, tokens, hidden), operand(I32, tokens, top), operand(dtype, experts, hidden, inner)
    return (capi.lib().vecops_hip_moe_experts_workspace(C.byref(ids), C.byref(down)),
            capi.lib().vecops_hip_moe_layer_workspace(C.byref(x), C.byref(ids), C.byref(down)))


def test_nothing_is_asked_for_a_layer_that_is_refused():
    """A prompt's tokens, and whatever else the calls refuse, need no workspace: a caller that allocates what the query says
    meets the refusal and not the allocator's."""
    assert all(n > 0 for n in moe_need()) and all(n > 0 for n in moe_need(128, 16, 512))
    for refused_extent in ({"tokens": 129}, {"tokens": 65536, "top": 8, "inner": 14336}, {"top": 17}, {"experts": 513}, {"hidden": 2 ** 24 + 1},
                           {"inner": 2 ** 24 + 1}):
        assert moe_need(**refused_extent) == (0, 0), refused_extent
    assert moe_need(top=9)[1] == 0   # more choices than experts: a layer's refusal
    x, ids, down = operand(BF16, 5, 256), operand(I32, 4, 2), operand(BF16, 8, 256, 96)
    assert capi.lib().vecops_hip_moe_layer_workspace(C.byref(x), C.byref(ids), C.byref(down)) == 0
    x = operand(BF16, 4, 255)
    assert capi.lib().vecops_hip_moe_layer_workspace(C.byref(x), C.byref(ids), C.byref(down)) == 0


def test_nothing_is_asked_for_a_product_that_is_refused():
    k_strided = product(1000, 1000, 4096)
    k_strided[2] = operand(F8, 1000, 4096, strides=(1, 1000))
    assert need(k_strided) == 1000 * 4096
    for at, wrong in ((0, operand(capi.I8, 1000, 4096)), (4, operand(BF16, 1000, 999)), (1, operand(F32, 1000, 31)), (3, operand(F32, 1, 32)),
                      (0, operand(F8, 1000, 4095))):
        v = list(k_strided)
        v[at] = wrong
        assert need(v) == 0, at
    k_strided = product(64, 64, 2 ** 25)
    k_strided[2] = operand(F8, 64, 2 ** 25, strides=(1, 64))
    assert need(k_strided) == 0
