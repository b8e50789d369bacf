"""ISA lint of the operators' kernels in the shipped library (no GPU): no packed fp32 arithmetic, and enough wait states between a matrix instruction and whatever else
touches its result, over every path.

Why a test: hipcc once left those waits out where a branch stood between a 32x32x2 fp32 product and the first use of its registers; half a per cent of the results were wrong, and
which ones depended on the run.  diff_attention.hip keeps the products and their first use in one run of instructions since.  The counts are the documented ones for results of
8 and 16 passes: 11 wait states, and 18 for the fp32 products; an instruction is one, s_nop n is n + 1."""
import glob
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = "/opt/rocm/lib/llvm/bin/llvm-objdump"
KERNELS = ("diff_attention", "rotary_kernel", "residual_norm_kernel")


@pytest.fixture(scope="module")
def functions(tmp_path_factory):
    """{kernel: [(address, instruction, branch target or None)]}"""
    if not os.path.exists(OBJDUMP):
        pytest.skip("llvm-objdump of the ROCm toolchain not present")
    from radzero_amd import _lib
    d = tmp_path_factory.mktemp("isa")
    shutil.copy(_lib.build(), d / "lib.so")
    r = subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=d, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    found = {}
    for o in sorted(glob.glob(str(d / "lib.so.*gfx950"))):
        with open(o, "rb") as f:
            data = f.read()
        if not any(k.encode() in data for k in KERNELS):
            continue
        name, start = None, 0
        for line in subprocess.run([OBJDUMP, "-d", o], capture_output=True, text=True).stdout.splitlines():
            m = re.match(r"^([0-9a-f]+) <(\S+)>:", line)
            if m:
                name, start = (m.group(2), int(m.group(1), 16)) if any(k in m.group(2) for k in KERNELS) else (None, 0)
                if name:
                    found[name] = []
            elif name and "//" in line:
                text, rest = line.split("//")[:2]
                target = re.search(r"<\S+?(?:\+0x([0-9a-f]+))?>$", rest)
                found[name].append((int(rest.split(":")[0], 16), text.strip(), start + int(target.group(1) or "0", 16) if target else None))
    assert len(found) >= 50, "the operators' kernels are not in the library"
    return found


def registers(operands):
    out = set()
    for kind, a, b, kind1, n in re.findall(r"\b(?:([va])\[(\d+):(\d+)\]|([va])(\d+)\b)", operands):
        out.update((kind, i) for i in range(int(a), int(b) + 1)) if kind else out.add((kind1, int(n)))
    return out


def test_registers():
    assert registers("v[2:3], v7, -v208, s[40:41], a[0:1], 0") == {("v", 2), ("v", 3), ("v", 7), ("v", 208), ("a", 0), ("a", 1)}


def test_no_packed_fp32(functions):
    for name, ins in functions.items():
        assert not any(re.match(r"v_pk_(add|mul|fma)_f32", t) for _, t, _ in ins), name


def test_matrix_results_are_waited_for(functions):
    products = 0
    for name, ins in functions.items():
        at = {a: i for i, (a, _, _) in enumerate(ins)}
        touched = [registers(t.partition(" ")[2]) for _, t, _ in ins]
        for i, (_, text, _) in enumerate(ins):
            op, _, operands = text.partition(" ")
            if not op.startswith("v_mfma"):
                continue
            products += 1
            result, need = registers(operands.split(",")[0]), 18 if op == "v_mfma_f32_32x32x2_f32" else 11
            paths, seen = [(i + 1, 0)], {}
            while paths:
                j, waited = paths.pop()
                while j < len(ins) and waited < need and seen.get(j, need) > waited:
                    seen[j] = waited
                    o, _, rest = ins[j][1].partition(" ")
                    if o == "s_nop":
                        waited += int(rest) + 1
                        j += 1
                        continue
                    if re.match(r"(v_(?!mfma)|ds_|global_|buffer_|scratch_)", o) and touched[j] & result:
                        raise AssertionError(f"{name}: {waited} of {need} wait states between '{text}' and '{ins[j][1]}'")
                    if o == "s_endpgm":
                        break
                    if o.startswith("s_cbranch"):
                        paths.append((at[ins[j][2]], waited + 1))
                    j = at[ins[j][2]] if o == "s_branch" else j + 1
                    waited += 1
    assert products > 1000
