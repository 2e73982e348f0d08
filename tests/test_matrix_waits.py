"""The hardware does not hold back an instruction that reads what a matrix instruction has not written yet: the compiler puts the wait states in between, but
none in front of inline assembly, of which it does not know what it reads.  Here the assembly of the attention over the 4-bit cache, compiled as the
build does, is walked from every matrix instruction along all paths: nothing reads its result sooner than the compiler's own rule allows.  No GPU needed."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# wait states between a matrix instruction and a vector instruction on its result, as the compiler puts them for a plain sum of two elements of it
NEEDED = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_32x32x16_bf16": 12, "v_mfma_f32_32x32x16_f16": 12}


def registers(operand):
    """Numbers of the vector registers that an operand names."""
    found = set()
    for low, high, one in re.findall(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", operand):
        found |= {int(one)} if one else set(range(int(low), int(high) + 1))
    return found


def functions(text):
    """[(name, instructions, labels)]: an instruction is (name, operands), a label the index of the one behind it."""
    out = []
    for line in text.splitlines():
        line = line.split(";")[0].strip()
        if re.match(r"_Z\w+:$", line):
            out.append((line[:-1], [], {}))
        elif out and line.endswith(":"):
            out[-1][2][line[:-1]] = len(out[-1][1])
        elif out and line and not line.startswith("."):
            name, _, operands = line.partition(" ")
            out[-1][1].append((name.strip(), [x.strip() for x in re.split(r",(?![^\[]*\])", operands)]))
    return out


def reads_and_writes(op, args):
    """Vector registers that an instruction other than a matrix one reads, and those that it writes."""
    named = [registers(x) for x in args]
    every = set().union(*named)
    if op.startswith(("ds_write", "buffer_store", "global_store", "scratch_store", "flat_store")):
        return every, set()
    if op.startswith(("v_fmac", "v_dot2c", "v_swap")) or "_swap" in op:           # the first operand, or both, are read and written
        return every, every
    return set().union(*named[1:]), named[0] if named else set()


def too_early(code, labels, start):
    """Instructions that read the result of the matrix instruction at `start` before its wait states have passed."""
    name, operands = code[start]
    found, seen = set(), {}
    todo = [(start + 1, 0, frozenset(registers(operands[0])))]
    while todo:
        at, waited, live = todo.pop()
        while at < len(code) and waited < NEEDED[name] and live:
            if seen.get((at, live), 99) <= waited:
                break
            seen[at, live] = waited
            op, args = code[at]
            if op.startswith(("v_mfma", "v_smfmac")):
                live -= registers(args[0])                                       # (its own result from here on; as an operand the hardware waits)
            elif op.startswith(("v_", "ds_", "buffer_", "global_", "scratch_", "flat_")):
                reads, writes = reads_and_writes(op, args)
                if reads & live:
                    found.add(at)
                    break
                live -= writes
            if op in ("s_endpgm", "s_setpc_b64", "s_swappc_b64"):
                break
            waited += int(args[0], 0) + 1 if op == "s_nop" else 1
            if op.startswith(("s_branch", "s_cbranch")):
                if op != "s_branch":
                    todo.append((at + 1, waited, live))
                at = labels[args[0]]
            else:
                at += 1
    return found


def test_the_walk_itself():
    text = """_Z1av:
    v_mfma_f32_16x16x32_bf16 v[2:5], v[6:9], v[10:13], v[2:5]
    s_cbranch_vccz .L1
    s_nop 6
    v_max3_f32 v1, v2, v3, v4
    s_endpgm
.L1:
    s_nop 4
    v_mov_b32_e32 v4, v7
    v_add_f32_e32 v1, v5, v6
    s_endpgm
"""
    (_, code, labels), = functions(text)
    assert too_early(code, labels, 0) == {7}                                     # one state short on the path behind the branch
    (_, code, labels), = functions(text.replace("s_nop 4", "s_nop 5"))
    assert too_early(code, labels, 0) == set()


def test_results_of_matrix_instructions_are_waited_for(tmp_path):
    build = open(os.path.join(ROOT, "kernels", "compile.sh")).read()
    flags = re.search(r"flags=\((.*?)\)", build, re.S).group(1).split()
    own = re.search(r"compile abi_kv4\.hip abi_kv4\.o(.*)", build).group(1).split()
    out = tmp_path / "abi_kv4.s"
    subprocess.run(["hipcc", *flags, *own, "--offload-device-only", "-S", os.path.join(ROOT, "ternainfer_amd", "csrc", "abi_kv4.hip"), "-o", str(out)], check=True, capture_output=True, timeout=600)
    matrix, wrong = 0, []
    for name, code, labels in functions(out.read_text()):
        for at, (op, _) in enumerate(code):
            if op.startswith(("v_mfma", "v_smfmac")):
                matrix += 1
                wrong += [(name, at, " ".join(map(str, code[i]))) for i in too_early(code, labels, at)]
    assert matrix > 100
    assert not wrong, f"{len(wrong)} too early: {wrong[:5]}"
