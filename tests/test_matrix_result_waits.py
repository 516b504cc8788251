"""The built kernels leave a matrix instruction the time it needs before its result is read or overwritten, along every branch.

gfx950 does not wait for that by itself: the compiler counts instructions and fills up with ``s_nop``.  Where a branch lies
between a matrix instruction and the addition that reads its result, the compiler of ROCm 7.2 has left the branch's far side
without (``if (q < n) acc[q] += product`` in an unrolled loop, some register counts only).  The results are wrong now and then, which no test of
values shows reliably; so this one walks over the library's own code.
"""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from torchtune_amd import build

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")


def _registers(operand):
    m = re.fullmatch(r"-?\|?([va])(?:\[(\d+):(\d+)\]|(\d+))\|?", operand.strip())
    if not m:
        return frozenset()
    lo, hi = (int(m[2]), int(m[3])) if m[2] else (int(m[4]), int(m[4]))
    return frozenset((m[1], i) for i in range(lo, hi + 1))


def _passes(name, text):
    """of four cycles; the block-scaled forms take twice as long where an operand has eight bits (formats 0 and 1)"""
    size = re.search(r"_(\d+)x\d+x", name)
    base = 8 if size and size[1] == "32" else 4
    if "f8f6f4" in name and not re.search(r"cbsz:[234].*blgp:[234]", text):
        base *= 2
    return base


class _Instruction:
    __slots__ = ("name", "text", "reads", "writes", "target", "address")

    def __init__(self, line):
        code, _, note = line.partition("//")
        self.text = code.strip()
        parts = self.text.split(None, 1)
        self.name = parts[0]
        operands = re.split(r",(?![^\[]*\])", parts[1]) if len(parts) > 1 else []
        operands = [o.split()[0] if o.split() else "" for o in operands]  # modifiers stand behind the last one
        sets = [_registers(o) for o in operands]
        stores = self.name.startswith(("ds_write", "ds_bpermute")) or "store" in self.name or "atomic" in self.name
        first_is_result = not stores and self.name.startswith(("v_", "ds_", "global_load", "buffer_load", "flat_load", "scratch_load")) and not self.name.startswith("v_cmp")
        self.writes = sets[0] if first_is_result and sets else frozenset()
        self.reads = frozenset().union(*(sets[1:] if first_is_result else sets)) if sets else frozenset()
        if "swap" in self.name:  # exchanges its two operands
            self.writes = self.reads = frozenset().union(*sets)
        m = re.match(r"\s*([0-9A-Fa-f]+):", note)
        self.address = int(m[1], 16) if m else None
        m = re.search(r"<([^>+]+)(?:\+0x([0-9a-fA-F]+))?>", note)
        self.target = (m[1], int(m[2] or "0", 16)) if m and "branch" in self.name else None


def hazards(listing):
    """(kernel, matrix instruction, too early reader, waits between) in a disassembly.  Units of four cycles: an instruction takes one,
    ``s_nop n`` n + 1, and a matrix instruction is not taken before the unit is done with the passes of the one before it; a result can be
    read four units after its passes."""
    kernels, current = {}, None
    for line in listing.splitlines():
        m = re.match(r"(?:[0-9a-f]+ )?<(.+)>:$", line)
        if m:
            current = kernels.setdefault(m[1], [])
        elif current is not None and line.startswith("\t") and line.strip() and not line.strip().startswith("//"):
            current.append(_Instruction(line))
    found = []
    for kernel, code in kernels.items():
        if not code:
            continue
        base = code[0].address or 0
        at = {ins.address: i for i, ins in enumerate(code)}
        for i, ins in enumerate(code):
            if not ins.name.startswith("v_mfma"):
                continue
            need = _passes(ins.name, ins.text) + 4
            seen, todo = set(), [(i + 1, 1, need - 4)]
            while todo:
                # now: when instruction j is issued at the earliest; free: when the matrix unit takes its next instruction
                j, now, free = todo.pop()
                while j < len(code) and now <= need and (j, now, free) not in seen:
                    seen.add((j, now, free))
                    other = code[j]
                    if other.name.startswith("v_mfma"):
                        now = max(now, free)
                        a, b = re.split(r",(?![^\[]*\])", other.text.split(None, 1)[1])[1:3]
                        early = (_registers(a) | _registers(b)) & ins.writes  # sums pass from one to the next by themselves
                        free = now + _passes(other.name, other.text)
                    else:
                        early = (other.reads | other.writes) & ins.writes
                    if early and now <= need:
                        found.append((kernel, ins.text, other.text, now - 1))
                        break
                    if other.name == "s_endpgm":
                        break
                    now += int(other.text.split()[1], 0) + 1 if other.name == "s_nop" else 1
                    if other.target:
                        to = at.get(base + other.target[1]) if other.target[0] == kernel else None
                        if to is not None:
                            todo.append((to, now, free))
                        if other.name == "s_branch":
                            break
                    j += 1
    return found


_BRANCHED = """
<kernel>:
\tv_mfma_f32_16x16x32_bf16 v[4:7], v[20:23], v[24:27], 0       // 000000001000: D3B50004 02020000
\ts_andn2_b64 vcc, exec, s[38:39]                              // 000000001008: 89EA267E
\ts_cbranch_vccnz 9                                            // 00000000100C: BF870009 <kernel+0x34>
\tv_mfma_f32_16x16x32_bf16 v[8:11], v[28:31], v[24:27], 0      // 000000001010: D3B50008 02020000
\ts_nop 7                                                      // 000000001018: BF800007
\tv_add_f32_e32 v0, v8, v0                                     // 00000000101C: 02000108
\tv_add_f32_e32 v1, v9, v1                                     // 000000001020: 02020309
\tv_add_f32_e32 v2, v10, v2                                    // 000000001024: 0204050A
\tv_add_f32_e32 v3, v11, v3                                    // 000000001028: 0206070B
\ts_nop 0                                                      // 00000000102C: BF800000
\ts_nop 0                                                      // 000000001030: BF800000
\t%s
\tv_add_f32_e32 v12, v4, v12                                   // 000000001038: 02181904
\ts_endpgm                                                     // 00000000103C: BF810000
"""


def test_the_walk_finds_a_result_read_too_early():
    """In a listing written for it: the fall-through waits, the branch does not; with a wait at the branch's target both do."""
    bad = hazards(_BRANCHED % "s_mov_b32 s0, 0                                              // 000000001034: BE800080")
    assert [(k, r.split()[0], w) for k, _, r, w in bad] == [("kernel", "v_add_f32_e32", 3)]
    assert not hazards(_BRANCHED % "s_nop 7                                                      // 000000001034: BF800007")
    overwritten = _BRANCHED.replace("v_add_f32_e32 v12, v4, v12 ", "v_mov_b32_e32 v5, v12 ") % "s_mov_b32 s0, 0    // 000000001034: BE800080"
    stored = _BRANCHED.replace("v_add_f32_e32 v12, v4, v12 ", "ds_write_b128 v1, v[4:7] offset:16 ") % "s_mov_b32 s0, 0    // 000000001034: BE800080"
    multiplied = _BRANCHED.replace("v_add_f32_e32 v12, v4, v12 ", "v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[24:27], 0 ") % "s_mov_b32 s0, 0    // 000000001034: BE800080"
    assert all(len(hazards(t)) == 1 for t in (overwritten, stored, multiplied))
    summed = _BRANCHED.replace("v_add_f32_e32 v12, v4, v12 ", "v_mfma_f32_16x16x32_bf16 v[4:7], v[20:23], v[24:27], v[4:7] ") % "s_mov_b32 s0, 0    // 000000001034: BE800080"
    assert not hazards(summed)


def test_no_built_kernel_reads_a_matrix_result_too_early(tmp_path):
    if not OBJDUMP.exists():
        pytest.skip("needs the ROCm toolchain's llvm-objdump")
    lib = tmp_path / build.LIB_PATH.name
    shutil.copy(build.LIB_PATH, lib)
    subprocess.run([str(OBJDUMP), "--offloading", str(lib)], check=True, capture_output=True, cwd=tmp_path)
    products, found = 0, []
    for part in sorted(tmp_path.glob("*gfx950")):
        listing = subprocess.run([str(OBJDUMP), "-d", "--no-show-raw-insn", str(part)], check=True, capture_output=True, text=True).stdout
        products += listing.count("v_mfma")
        found += hazards(listing)
    assert products > 1000  # the listing was understood
    assert not found, f"{len(found)} results read or overwritten too early, first {found[:3]}"
