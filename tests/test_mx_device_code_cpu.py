"""What the compiled kernels of the microscaled product have to keep and no result shows reliably: wait states between a matrix
instruction and the use of its result along every path, read from the library as it was built here."""
import glob
import os
import re
import shutil
import subprocess

import pytest

from test_device_code_cpu import OBJDUMP, first_uses
from vecops_amd import capi


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{mangled name: [(operation, operands)], with ("label", its name) where a branch leads}."""
    if not os.path.exists(OBJDUMP) or not os.path.exists(capi.LIB_PATH):
        pytest.skip("no built library, or no llvm-objdump beside the compiler")
    here = tmp_path_factory.mktemp("device")
    shutil.copy(capi.LIB_PATH, here / "l.so")
    subprocess.run([OBJDUMP, "--offloading", "l.so"], cwd=here, check=True, capture_output=True)
    found = {}
    for part in glob.glob(str(here / "l.so.*gfx950*")):
        with open(part, "rb") as f:
            if b"mx_few_rows_kernel" not in f.read():
                continue
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", "--symbolize-operands", part], check=True,
                              capture_output=True, text=True).stdout
        code = None
        for line in text.split("\n"):
            line = line.split("//")[0].strip()
            name = re.fullmatch(r"<(.+)>:", line)
            if name and re.fullmatch(r"L\d+", name.group(1)):
                code.append(("label", name.group(1)))
            elif name:
                code = found.setdefault(name.group(1), [])
            elif line and code is not None:
                code.append(tuple((line.split(None, 1) + [""])[:2]))
    assert found
    return found


def test_matrix_results_are_not_used_too_early(kernels):
    """Four passes where both operands are of 4 bits, eight with an 8-bit one, and four more before a result may be read."""
    seen, early = 0, []
    for name, code in kernels.items():
        if not any(op.startswith("v_mfma") for op, _ in code):
            continue
        seen += 1
        for op, (states, i, j) in first_uses(code).items():
            if states < (8 if "cbsz:4 blgp:4" in code[i][1] else 12):
                early.append((name, op, states, code[i], code[j]))
    assert seen >= 4
    assert not early, f"{len(early)} kernels, the first: {early[0]}"


def test_products_stay_in_the_matrix_core(kernels):
    """Every product is the scaled instruction's, and no kernel keeps registers in memory."""
    for name, code in kernels.items():
        matrix = {op for op, _ in code if op.startswith("v_mfma")}
        assert matrix <= {"v_mfma_scale_f32_16x16x128_f8f6f4"}, (name, matrix)
        assert not any(op.startswith("scratch_") for op, _ in code), name
