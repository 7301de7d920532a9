"""No kernel of the built library reads or overwrites a matrix instruction's result before its wait is over.

The hardware does not hold such an access back; the compiler puts instructions or s_nop between.
Over a branch with a side of its own it has been seen to leave them out (a result read after 3 of 8
states, different from call to call).  What it keeps within a block is taken as the wait of each
instruction, and looked for on every way out of the block."""
import collections
import os
import re
import shutil
import subprocess

import pytest

from mlx_vit_amd.build import ARCH, LIB_PATH, build

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
REG = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)")
FAR = 20   # states behind which nothing waits any more


def registers(text):
    out = set()
    for kind, lo, hi, one in REG.findall(text):
        out |= {(kind, i) for i in (range(int(lo), int(hi) + 1) if lo else (int(one),))}
    return out


def kernels(text):
    """(name, [(instruction, operands)], {label: index}) of each function of a disassembly."""
    name, code, labels = None, [], {}
    for line in text.splitlines():
        m = re.match(r"^[0-9a-f]+ <([^>]+)>:", line)
        if m:
            if re.fullmatch(r"L\d+", m[1]):
                labels[m[1]] = len(code)
                continue
            if code:
                yield name, code, labels
            name, code, labels = m[1], [], {}
        elif name and line.startswith("\t"):
            op, _, rest = line.split("//")[0].strip().partition(" ")
            if op:
                code.append((op, rest.strip()))
    if code:
        yield name, code, labels


def accesses(code, labels):
    """(matrix instruction, states between, over a border, index, index) of the first access on each way from one."""
    touched, borders = [None] * len(code), set(labels.values())
    for i, (op, rest) in enumerate(code):
        if "mfma" not in op:
            continue
        result = registers(rest.split(",")[0])
        ways, seen = [(i + 1, 0, False)], set()
        while ways:
            j, states, border = ways.pop()
            while j < len(code) and states < FAR and (j, states, border) not in seen:
                seen.add((j, states, border))
                border = border or j in borders
                o, r = code[j]
                if o == "s_endpgm":
                    break
                if o == "s_nop":
                    states, j = states + int(r, 0) + 1, j + 1
                    continue
                if o == "s_branch":
                    j, states, border = labels[r], states + 1, True
                    continue
                if o.startswith("s_cbranch"):
                    # (lanes are there again behind their return: no way that skips for want of them)
                    if not (o == "s_cbranch_execz" and code[j - 1][0] == "s_or_b64" and code[j - 1][1].startswith("exec, exec")):
                        ways.append((labels[r], states + 1, True))
                    border = True
                elif "mfma" in o:
                    a = r.split(", ")
                    if (registers(a[1]) | registers(a[2])) & result:
                        yield op, states, border, i, j, "factor"
                        break
                    if registers(r) & result:    # the sum goes on: of the unit's own order
                        break
                elif o.startswith(("v_", "ds_", "global_", "buffer_", "scratch_", "flat_")):
                    if touched[j] is None:
                        touched[j] = registers(r)
                    if touched[j] & result:
                        yield op, states, border, i, j, "other"
                        break
                states, j = states + 1, j + 1


def short(texts):
    """Accesses over a border with fewer states than within blocks."""
    least, over = collections.defaultdict(lambda: FAR), []
    for text in texts:
        for name, code, labels in kernels(text):
            for op, states, border, i, j, kind in accesses(code, labels):
                if border:
                    over.append((op, kind, states, name, code[i], code[j]))
                else:
                    least[op, kind] = min(least[op, kind], states)
    return [x for x in over if x[2] < least[x[0], x[1]] < FAR], least, len(over)


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")
def test_results_are_waited_for(tmp_path):
    if not os.path.exists(LIB_PATH):
        build()
    shutil.copy(LIB_PATH, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", os.path.basename(LIB_PATH)], cwd=tmp_path, check=True, capture_output=True)
    parts = sorted(f for f in os.listdir(tmp_path) if f.endswith(ARCH))
    assert parts
    bad, least, count = short(subprocess.run([OBJDUMP, "-d", "--symbolize-operands", "--no-show-raw-insn", f], cwd=tmp_path, check=True,
                                             capture_output=True, text=True).stdout for f in parts)
    assert least and count
    assert not bad, bad[:5]


def test_finds_what_is_missing():
    def text(side):
        return "\n".join(["0000 <k>:", "\tv_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], 0", "\ts_nop 7", "\tv_add_f32_e32 v20, v0, v0",
                          "\tv_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], 0", "\ts_cbranch_vccnz L1", *side, "0010 <L0>:",
                          "\tv_add_f32_e32 v21, v3, v3", "\ts_endpgm", "0020 <L1>:", "\tv_mov_b32_e32 v30, 0", "\ts_branch L0"])
    bad, least, _ = short([text([])])
    assert least["v_mfma_f32_16x16x32_bf16", "other"] == 8 and sorted(x[2] for x in bad) == [1, 3]
    assert [x[2] for x in short([text(["\ts_nop 7"])])[0]] == [3]     # (the way over the side is as short as before)
