"""What the compiled 8-bit float and mixture-of-experts kernels have to keep and no result shows reliably: properties of the
instructions along every path of a kernel, read from the library as it was built here."""
import glob
import os
import re
import shutil
import subprocess

import pytest

from vecops_amd import capi

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{mangled name: [(operation, operands)], with ("label", its name) where a branch leads} of both files' kernels."""
    if not os.path.exists(OBJDUMP) or not os.path.exists(capi.LIB_PATH):
        pytest.skip("no built library, or no llvm-objdump beside the compiler")
    here = tmp_path_factory.mktemp("device")
    shutil.copy(capi.LIB_PATH, here / "l.so")
    subprocess.run([OBJDUMP, "--offloading", "l.so"], cwd=here, check=True, capture_output=True)
    found = {}
    for part in glob.glob(str(here / "l.so.*gfx950*")):
        with open(part, "rb") as f:
            data = f.read()
        if b"moe_down_kernel" not in data and b"fp8_tile_kernel" not in data:
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


def walk(code, start, visit, state):
    """Follows every path behind instruction `start`.  `visit(index, operation, operands, state)` gives the state behind an
    instruction, or None where the path is done; a place is left out once a state as large has been there."""
    labels = {name: i for i, (op, name) in enumerate(code) if op == "label"}
    seen, paths = {}, [(start + 1, state)]
    while paths:
        i, state = paths.pop()
        while i < len(code) and seen.get(i, state + 1) > state:
            seen[i] = state
            op, operands = code[i]
            if op == "label":
                i += 1
                continue
            state = visit(i, op, operands, state)
            if state is None or op == "s_endpgm":
                break
            if op == "s_branch":
                i = labels[operands]
                continue
            if op.startswith("s_cbranch"):
                paths.append((labels[operands], state))
            i += 1


def test_sums_are_in_memory_before_they_are_counted(kernels):
    """A kernel whose workgroups count themselves in memory: a barrier orders wavefronts, it does not wait for what they have
    stored, and the increment's release waits for the stores of its own wavefront alone.  So no wavefront may reach the barrier
    in front of it with a store under way."""
    counting = {name: code for name, code in kernels.items() if any(op.startswith("global_atomic_add") for op, _ in code)}
    assert len([name for name in counting if "moe_down_kernel" in name]) >= 12
    early = []
    for name, code in counting.items():
        for i, (op, _) in enumerate(code):
            if not re.match(r"(global|flat|buffer)_store", op):
                continue

            def visit(j, op, operands, state, name=name, i=i):
                if op == "s_waitcnt" and "vmcnt(0)" in operands:
                    return None
                if op == "s_barrier":
                    early.append((name, i, j))
                    return None
                return state

            walk(code, i, visit, 0)
    assert not early, f"{len(early)} of a store and a barrier, the first: {early[0]}"
