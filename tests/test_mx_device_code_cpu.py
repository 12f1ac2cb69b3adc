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
            if b"mx_slim_kernel" not in f.read():
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
            elif line.startswith("v_mfma_ld_scale_b32"):   # (the first half of a scaled instruction whose name then lacks it)
                continue
            elif line and code is not None:
                code.append(tuple((line.split(None, 1) + [""])[:2]))
    assert found
    return found


def test_matrix_results_are_not_used_too_early(kernels):
    """Passes of a 16x16x128 product: four where both operands are of 4 bits, eight with an 8-bit one; of a 32x32x64 product twice as many.  Four
    more before a result may be read."""
    seen, early = 0, []
    for name, code in kernels.items():
        if not any(op.startswith("v_mfma") for op, _ in code):
            continue
        seen += 1
        for op, (states, i, j) in first_uses(code).items():
            passes = (4 if "cbsz:4 blgp:4" in code[i][1] else 8) * (2 if "32x32x64" in code[i][0] else 1)
            if states < passes + 4:
                early.append((name, op, states, code[i], code[j]))
    assert seen >= 12
    assert not early, f"{len(early)} kernels, the first: {early[0]}"


def test_products_stay_in_the_matrix_core(kernels):
    """Every product is the scaled instruction's, and no kernel keeps a register in memory but the one of 256 x 256 results, for some addresses and sizes
    between tiles."""
    for name, code in kernels.items():
        matrix = {op.replace("_scale", "") for op, _ in code if op.startswith("v_mfma")}
        assert matrix <= {"v_mfma_f32_16x16x128_f8f6f4", "v_mfma_f32_32x32x64_f8f6f4"}, (name, matrix)
        most = 40 if "mx_tile_kernelILi2ELi2ELi1ELi4ELi4E" in name else 0
        assert sum(op.startswith("scratch_") for op, _ in code) <= most, name
