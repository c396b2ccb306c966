"""CPU test of the built kernels: no instruction touches a matrix product's registers before the product is finished.

The hardware does not wait for the result of a v_mfma: the compiler keeps other instructions between it and the first that reads or
overwrites its registers, or s_nop.  Where a branch leads round a longer piece of code (`if (!full) mask`) between a product and its use, the
compiler (ROCm 7.2) has been seen to count the longer way only and to leave the wait out on the shorter one; the scores were then read
unfinished, now and then.  The remedy is in the source: no branch between products and their use.

Every path of a kernel is followed from each product for as many wait states (an instruction is one, s_nop N is N + 1) as the same compiler
puts between the product and a dependent instruction in straight code."""

import bisect
import os
import re
import shutil
import subprocess

import pytest

import build_ext

OBJDUMP = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(build_ext.HIPCC))), "llvm", "bin", "llvm-objdump")
NEEDS = {"16x16x32": 8, "32x32x16": 12}  # wait states
REGISTERS = re.compile(r"\b([av])(?:\[(\d+):(\d+)\]|(\d+)\b)")
LINE = re.compile(r"^\t(\S+)(.*?)\s*// ([0-9A-F]+): ((?:[0-9A-F]{8} ?)+)(?:<.*>)?$")


def _spans(text):
    return [(m[1], int(m[2] or m[4]), int(m[3] or m[4])) for m in REGISTERS.finditer(text)]


def _meets(a, b):
    return a[0] == b[0] and a[1] <= b[2] and b[1] <= a[2]


def _kernel(lines):
    """[(address, mnemonic, operands, branch target or None)] of a kernel's disassembled lines."""
    code = []
    for line in lines:
        m = LINE.match(line)
        if not m:
            continue
        at, words = int(m[3], 16), m[4].split()
        target = None
        if m[1].startswith(("s_branch", "s_cbranch")):
            offset = int(words[0], 16) & 0xFFFF
            target = at + 4 + 4 * (offset - 0x10000 if offset & 0x8000 else offset)
        code.append((at, m[1], m[2].strip(), target))
    return code


def too_early(lines):
    """[(address of a product, of an instruction that touches its result, wait states between them)]"""
    code = _kernel(lines)
    addresses = [c[0] for c in code]
    found = []
    for i, (at, name, operands, _) in enumerate(code):
        if not name.startswith("v_mfma"):
            continue
        need = next(n for shape, n in NEEDS.items() if shape in name)
        result = _spans(operands)[0]
        best, todo = {}, [(i + 1, 0)]
        while todo:
            j, states = todo.pop()
            while j < len(code) and states < need and states < best.get(j, need):
                best[j] = states
                _, other, args, target = code[j]
                spans = _spans(args)
                if other.startswith("v_mfma"):
                    # accumulating on is interlocked; the operands are not
                    same = len(spans) > 3 and spans[3] == result or spans[0] == result
                    touched = any(_meets(result, s) for s in spans[1:3])
                    if touched:
                        found.append((at, code[j][0], states))
                    if same or touched:
                        break
                elif any(_meets(result, s) for s in spans):
                    found.append((at, code[j][0], states))
                    break
                if other in ("s_endpgm", "s_setpc_b64", "s_swappc_b64"):
                    break
                states += int(args, 0) + 1 if other == "s_nop" else 1
                if target is not None:
                    k = bisect.bisect_left(addresses, target)
                    assert k < len(code) and addresses[k] == target
                    if other == "s_branch":
                        j = k
                        continue
                    todo.append((k, states))
                j += 1
    return found


def test_unfinished_products_are_seen():
    """The pattern itself, in the disassembler's form: the branch leads round what the straight way waits with."""
    text = """
\tv_mfma_f32_16x16x32_f16 a[0:3], v[16:19], v[84:87], a[0:3] // 000000001000: D3D48000 0402A910
\tv_mfma_f32_16x16x32_f16 a[4:7], v[0:3], v[84:87], a[4:7]  // 000000001008: D3D48004 0412A900
\ts_cbranch_vccnz 1                                          // 000000001010: BF870001 <k+0x18>
\ts_nop 7                                                    // 000000001014: BF800007
\tv_accvgpr_read_b32 v39, a3                                 // 000000001018: D3D84027 18000103
\ts_endpgm                                                   // 000000001020: BF810000"""
    assert too_early(text.split("\n")) == [(0x1000, 0x1018, 2)]
    assert too_early(text.replace("s_cbranch_vccnz 1 ", "s_cbranch_vccnz 0 ").replace("BF870001", "BF870000").split("\n")) == []
    assert too_early(text.replace("s_nop 7", "s_nop 3").replace("BF870001", "BF870000").split("\n")) == [(0x1000, 0x1018, 6)]
    assert too_early(text.replace("v39, a3", "v39, a5").split("\n")) == [(0x1008, 0x1018, 1)]


def test_no_result_is_touched_before_it_is_there(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no disassembler")
    lib = shutil.copy(build_ext.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    products, early = 0, []
    for part in sorted(p for p in os.listdir(tmp_path) if p.endswith("gfx950")):
        run = subprocess.Popen([OBJDUMP, "-d", str(tmp_path / part)], stdout=subprocess.PIPE, text=True)
        kernel, lines = None, []
        for line in [*run.stdout, "0 <end>:"]:
            if line.endswith(">:\n") or line == "0 <end>:":
                count = sum("v_mfma_f32" in x[:12] for x in lines)
                products += count
                if count:
                    early += [(kernel, *x) for x in too_early(lines)]
                kernel, lines = line.split("<")[1].split(">")[0], []
            else:
                lines.append(line.rstrip("\n"))
        assert run.wait() == 0
    assert products > 1000
    assert not early, "\n".join(f"{k}: {a:#x} is touched at {b:#x} after {n} wait states" for k, a, b, n in early[:40])
