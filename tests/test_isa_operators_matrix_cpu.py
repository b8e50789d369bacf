"""ISA lint of the operators' kernels (no GPU), next to test_isa_operators_cpu.py: matrix instructions that take another one's result as an operand of the product, or accumulate
into registers that overlap it without being the same, wait for it as every other instruction does, over every path.  (Accumulating into the very same registers is what the
hardware orders by itself.)"""
import re

from test_isa_operators_cpu import functions, registers                     # noqa: F401  (a fixture)


def test_matrix_results_are_waited_for_by_matrix_instructions(functions):   # noqa: F811
    pairs = 0
    for name, ins in functions.items():
        at = {a: i for i, (a, _, _) in enumerate(ins)}
        for i, (_, text, _) in enumerate(ins):
            op, _, operands = text.partition(" ")
            if not op.startswith("v_mfma"):
                continue
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
                    if o.startswith("v_mfma"):
                        pairs += 1
                        d, a, b, c = (registers(x) for x in re.split(r",\s*", rest)[:4])
                        assert not (a | b) & result, f"{name}: {waited} of {need} wait states between '{text}' and '{ins[j][1]}'"
                        assert not c & result or c == result, f"{name}: '{text}' and '{ins[j][1]}' overlap"
                        assert not d & result or d == result, f"{name}: '{text}' and '{ins[j][1]}' overlap"
                    if o == "s_endpgm":
                        break
                    if o.startswith("s_cbranch"):
                        paths.append((at[ins[j][2]], waited + 1))
                    j = at[ins[j][2]] if o == "s_branch" else j + 1
                    waited += 1
    assert pairs > 1000
