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


def registers(text):
    """The vector and accumulation registers that an operand list names."""
    found = set()
    for kind, a, b in re.findall(r"\b([va])\[(\d+):(\d+)\]", text):
        found |= {(kind, r) for r in range(int(a), int(b) + 1)}
    return found | {(kind, int(r)) for kind, r in re.findall(r"\b([va])(\d+)\b", text)}


def first_uses(code):
    """For each matrix instruction the fewest wait states, over all paths, to an instruction that is no accumulation and names its
    result: {operation: (states, index of the matrix instruction, index of the use)}."""
    least = {}
    for i, (op, operands) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        result = registers(operands.split(", ")[0])

        def visit(j, other, text, states, op=op, i=i, result=result):
            if states >= 20:
                return None
            if other == "s_nop":
                return states + 1 + int(text, 0)
            if other.startswith("v_mfma"):
                to, *factors = text.split(", ")[:3]
                if result & (registers(factors[0]) | registers(factors[1])):
                    least[op] = min(least.get(op, (99,)), (states, i, j))
                    return None
                return None if result & registers(to) else states + 1
            if re.match(r"(v|ds|buffer|global|flat|scratch)_", other) and result & registers(text):
                least[op] = min(least.get(op, (99,)), (states, i, j))
                return None
            return states + 1

        walk(code, i, visit, 0)
    return least


def test_matrix_results_are_not_used_too_early(kernels):
    """The hardware does not hold back an instruction that uses a matrix instruction's result: the compiler puts wait states in
    between, for 16- and 8-bit operands four more than the passes that it takes (four for 16x16x32 and eight for 16x16x128), for
    32-bit ones two more (of eight).  Where a branch stands between the two it has been seen to count the longer path.  So they
    are counted here along every path."""
    needed = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_16x16x128_f8f6f4": 12, "v_mfma_f32_16x16x4_f32": 10}
    seen, early = set(), []
    for name, code in kernels.items():
        for op, (states, i, j) in first_uses(code).items():
            seen.add(op)
            if states < needed[op]:
                early.append((name, op, states, code[i], code[j]))
    assert seen == set(needed)
    assert not early, f"{len(early)} kernels and instructions, the first: {early[0]}"


def test_every_path_is_followed():
    """The counting itself, on a few instructions: the shorter of two paths, a loop's way back, an accumulation in between."""
    mfma = ("v_mfma_f32_16x16x32_bf16", "v[0:3], v[8:11], v[12:15], v[0:3]")
    use = ("v_add_f32_e32", "v4, v2, v4")
    skip = [mfma, ("s_cbranch_scc1", "L0"), ("s_nop", "7"), ("label", "L0"), use, ("s_endpgm", "")]
    assert first_uses(skip) == {mfma[0]: (1, 0, 4)}
    assert first_uses(skip[:1] + skip[2:]) == {mfma[0]: (8, 0, 3)}
    loop = [("label", "L0"), use, ("s_nop", "1"), mfma, ("s_nop", "0"), ("s_cbranch_scc0", "L0"), ("s_nop", "7"), use, ("s_endpgm", "")]
    assert first_uses(loop) == {mfma[0]: (2, 3, 1)}
    assert first_uses([mfma, ("v_mfma_f32_16x16x32_bf16", "v[0:3], v[16:19], v[12:15], v[0:3]"), use, ("s_endpgm", "")]) == {mfma[0]: (0, 1, 2)}
    assert first_uses([mfma, ("v_mfma_f32_16x16x32_bf16", "a[0:3], v[0:3], v[12:15], 0"), ("s_endpgm", "")]) == {mfma[0]: (0, 0, 1)}
    assert first_uses([mfma, ("v_add_f32_e32", "v4, v6, v4"), ("s_endpgm", "")]) == {}
