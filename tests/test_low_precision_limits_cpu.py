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
