"""Results whose elements share memory, with one another or with another result: refused by the microscaled and row entry points, as
which of them stays would go by timing.  Nothing reaches a device (the addresses are no memory)."""
import ctypes as C
import itertools

import pytest

from test_low_precision_refusals_cpu import operand, refused
from test_mx_refusals_cpu import BF16, E8, F4, F8, F32, I8, INVALID, NOT_APPLICABLE, norm, product, ref
from vecops_amd import capi


def quantize(x, q, scales):
    return capi.lib().vecops_hip_quantize_mx(ref(x), ref(q), ref(scales), None)


def dequantize(q, scales, out):
    return capi.lib().vecops_hip_dequantize_mx(ref(q), ref(scales), ref(out), None)


def gate(x, q, scales):
    return capi.lib().vecops_hip_silu_mul_quantize(ref(x), ref(q), ref(scales), None)


def matmul(**changes):
    v = product(**changes)
    return capi.lib().vecops_hip_matmul_mx(*(ref(v[n]) for n in ("a", "sa", "b", "sb", "c")), None, 0, None)


RESIDUAL = operand(BF16, 5, 300)


@pytest.mark.parametrize("changes,word", [
    ({"residual": operand(BF16, 5, 300, strides=(0, 1))}, "summed"),                       # a broadcast residual, which the sum would replace
    ({"residual": operand(BF16, 5, 300, strides=(299, 1))}, "summed"),
    ({"residual": RESIDUAL, "summed": operand(BF16, 5, 300, strides=(-1, 1))}, "summed"),
    ({"out": operand(BF16, 5, 300, strides=(0, 1))}, "out"),
    ({"out": operand(BF16, 5, 300, strides=(150, 1))}, "out"),
    ({"q": operand(I8, 5, 300, strides=(0, 1))}, "q"),
    ({"scales": operand(F32, 5, 1, strides=(0, 1))}, "scales"),
    ({"q": operand(F8, 5, 300), "scales": operand(F32, 5, 3, strides=(1, 0))}, "scales"),
    ({"q": operand(F8, 5, 300), "scales": operand(E8, 5, 10, strides=(1, 4))}, "scales"),
])
def test_rows_of_the_norm(changes, word):
    refused(norm(**changes), INVALID, word + ": elements share memory")


def test_batches_of_the_norm():
    three = {"x": operand(BF16, 2, 5, 300), "q": operand(I8, 2, 5, 300), "scales": operand(F32, 2, 5, 1)}
    refused(norm(**three, out=operand(BF16, 2, 5, 300, strides=(0, 300, 1))), INVALID, "out: elements share memory")
    refused(norm(**three, out=operand(BF16, 2, 5, 300, strides=(600, 300, 1))), INVALID, "out: elements share memory")
    refused(norm(**three, residual=operand(BF16, 2, 5, 300, strides=(0, 300, 1))), INVALID, "summed: elements share memory")


def test_two_results_of_the_norm_in_one_place():
    x, residual = operand(BF16, 5, 300, data=0x100000), operand(BF16, 5, 300, data=0x200000)
    refused(norm(x=x, residual=residual, out=residual), INVALID, "out and summed")
    refused(norm(x=x, residual=residual, summed=x, out=x), INVALID, "out and summed")
    other = operand(BF16, 5, 300, data=0x300000)
    refused(norm(x=x, residual=residual, summed=other, out=other), INVALID, "out and summed")


@pytest.mark.parametrize("call,args,word", [
    (quantize, (operand(BF16, 5, 300), operand(F8, 5, 300, strides=(0, 1)), operand(E8, 5, 10)), "q"),
    (quantize, (operand(BF16, 5, 300), operand(F8, 5, 300, strides=(1, 1)), operand(E8, 5, 10)), "q"),
    (quantize, (operand(BF16, 5, 300), operand(F4, 5, 150, strides=(1, 4)), operand(E8, 5, 10)), "q"),
    (quantize, (operand(BF16, 5, 300), operand(F8, 5, 300), operand(E8, 5, 10, strides=(0, 1))), "scales"),
    (dequantize, (operand(F8, 5, 300), operand(E8, 5, 10), operand(BF16, 5, 300, strides=(0, 1))), "out"),
    (dequantize, (operand(F8, 5, 300), operand(E8, 5, 10), operand(BF16, 5, 300, strides=(2, 3))), "out"),
    (gate, (operand(BF16, 5, 600), operand(I8, 5, 300, strides=(0, 1)), operand(F32, 5, 1)), "q"),
    (gate, (operand(BF16, 5, 600), operand(I8, 5, 300), operand(F32, 5, 1, strides=(0, 1))), "scales"),
])
def test_rows_of_the_others(call, args, word):
    refused(call(*args), INVALID, word + ": elements share memory")


def test_results_of_the_product():
    for strides in ((0, 1), (199, 1), (1, 1), (1, 4), (200, 0)):
        refused(matmul(c=operand(F32, 5, 200, strides=strides)), INVALID, "c: elements share memory")
    need = capi.lib().vecops_hip_matmul_mx_workspace
    turned = product(b=operand(F4, 200, 320, strides=(1, 200)), c=operand(F32, 5, 200, strides=(0, 1)))
    assert need(*(ref(turned[n]) for n in ("a", "sa", "b", "sb", "c"))) == 0


def test_which_strides_share_memory():
    """Every small layout: refused if, and only if, two elements of its rows and columns have one address.  (What is not refused for that
    reason gets as far as the rows' own check: q of a gate has contiguous rows.)"""
    for rows, cols, rs, cs in itertools.product((1, 2, 3, 4), (2, 3, 5), range(-6, 7), range(-3, 4)):
        places = [r * rs + c * cs for r in range(rows) for c in range(cols)]
        shared = len(set(places)) < len(places)
        # a matrix without rows of scales, so that a call that is not refused has no device to reach: x is null, which is looked at last
        rc = quantize(operand(BF16, rows, cols, data=None), operand(F8, rows, cols, strides=(rs, cs)), operand(E8, rows, 1, strides=(1, 1)))
        refused(rc, INVALID, "q: elements share memory" if shared else "null")
    assert NOT_APPLICABLE == 2
