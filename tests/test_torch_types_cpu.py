"""Describing tensors with a torch that lacks the microscaled element types, or has others than the library's."""
import pytest
import torch

from vecops_amd import capi

HERE = {torch.int8: capi.I8, torch.uint8: capi.U8, torch.int32: capi.I32, torch.float16: capi.F16, torch.bfloat16: capi.BF16, torch.float32: capi.F32,
        torch.float64: capi.F64, torch.float8_e4m3fn: capi.F8E4M3}
MICROSCALED = {"float4_e2m1fn_x2": capi.F4E2M1X2, "float8_e8m0fnu": capi.F8E8M0}


@pytest.mark.parametrize("missing", [[], *([name] for name in MICROSCALED), list(MICROSCALED)])
def test_types_of_an_older_torch(missing, monkeypatch):
    for name in missing:
        monkeypatch.delattr(torch, name)
    for dtype, code in HERE.items():
        o = capi.operand(torch.empty((3, 5), dtype=dtype))
        assert (o.dtype, o.rank, list(o.sizes[:2]), list(o.strides[:2])) == (code, 2, [3, 5], [5, 1])
    for name, code in MICROSCALED.items():
        if name not in missing:
            assert capi.operand(torch.empty((3, 5), dtype=torch.uint8).view(getattr(torch, name))).dtype == code


def test_other_types_have_no_code():
    for dtype in (torch.int64, torch.bool, torch.float8_e5m2):
        with pytest.raises(KeyError):
            capi.operand(torch.empty((3, 5), dtype=dtype))
