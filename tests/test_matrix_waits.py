"""Waits behind matrix instructions in the built kernels, read from the disassembly of this repository's own objects.

The result of a matrix instruction (`v_mfma_*`) is written some cycles after it was issued, and nothing in the hardware
holds back an instruction that reads or overwrites the registers before that: the compiler has to put so many others, or
`s_nop`, in between. Where two paths lead from such an instruction to a place behind a branch, the compiler of this ROCm
has counted the instructions of the longer path alone and left out up to seven of ten waits on the shorter one, and the
last row of every four came out without its last term. No test of results shows reliably where that happened, so every
path of every kernel is followed here.

Waits needed, by instruction, as the compiler itself keeps them in straight code: before a read, before an overwriting.
One instruction counts one, `s_nop n` n + 1, and a further matrix instruction is not issued before the passes of the one
in front of it are over.

The objects are built by `make -C causal-conv1d-triton_amd` (or `__graft_entry__.build()`); the tests skip when
they or the LLVM tools of the ROCm install are absent.
"""

import glob
import os
import re
import subprocess

import pytest

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(_ROOT, "causal-conv1d-triton_amd")
_LLVM = "/opt/rocm/llvm/bin"
_TARGET = "hipv4-amdgcn-amd-amdhsa--gfx950"

# opcode -> waits before a read, before an overwriting, passes
NEED = {"v_mfma_f32_16x16x32_bf16": (8, 7, 4), "v_mfma_f32_16x16x32_f16": (8, 7, 4), "v_mfma_f32_16x16x4_f32": (10, 10, 8)}

_REG = re.compile(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])")
_LINE = re.compile(r"^\s+(\S+)\s*(.*?)\s*//\s*([0-9A-F]+):")
_JUMP = re.compile(r"<[^>+]+(?:\+0x([0-9a-f]+))?>\s*$")
_READS_ALL = ("global_store", "global_atomic", "ds_write", "buffer_store", "scratch_store", "flat_store")


def _regs(text):
    out = set()
    for kind, one, lo, hi in _REG.findall(text):
        out.update((kind, i) for i in ([int(one)] if one else range(int(lo), int(hi) + 1)))
    return frozenset(out)


def _listing(obj, tmp):
    fb, co = os.path.join(tmp, "fatbin.bin"), os.path.join(tmp, "gfx950.co")
    subprocess.run([os.path.join(_LLVM, "llvm-objcopy"), "--dump-section", f".hip_fatbin={fb}", obj, os.devnull],
                   check=True, capture_output=True)
    subprocess.run([os.path.join(_LLVM, "clang-offload-bundler"), "--unbundle", "--type=o", f"--input={fb}",
                    f"--targets={_TARGET}", f"--output={co}"], check=True)
    return subprocess.run([os.path.join(_LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", co], capture_output=True,
                          text=True, check=True).stdout


def kernels_of(listing):
    """(name, address, [(opcode, operands, address, line)]) of every kernel of a listing."""
    name, at, code = None, 0, []
    for line in listing.split("\n"):
        head = re.match(r"^([0-9a-f]+) <(\S+)>:", line)
        if head:
            if code:
                yield name, at, code
            name, at, code = head.group(2), int(head.group(1), 16), []
            continue
        m = _LINE.match(line)
        if m:
            code.append((m.group(1), m.group(2), int(m.group(3), 16), line))
    if code:
        yield name, at, code


def too_early(at, code):
    """[(matrix instruction, the one that comes too early, waits, waits needed)] of a kernel, and how many matrix
    instructions it has."""
    index = {c[2]: n for n, c in enumerate(code)}
    follow = []
    for n, (op, _, _, line) in enumerate(code):
        to = [n + 1] if op not in ("s_branch", "s_endpgm") and n + 1 < len(code) else []
        if op == "s_branch" or op.startswith("s_cbranch"):
            to.append(index[at + int(_JUMP.search(line.split("//")[1]).group(1) or "0", 16)])
        assert not op.startswith(("s_setpc", "s_swappc", "s_call")), op
        follow.append(to)
    found, count = [], 0
    for n, (op, args, _, line) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        count += 1
        before_read, before_write, passes = NEED[op]
        best, todo = {}, [(k, 0, _regs(args.split(",")[0])) for k in follow[n]]
        while todo:
            k, waits, result = todo.pop()
            if waits >= before_read or best.get((k, result), 99) <= waits:
                continue
            best[k, result] = waits
            o, a, _, other = code[k]
            if o.startswith("v_mfma"):
                waits = max(waits, passes)
                to, x, y, z = (_regs(p) for p in a.split(",")[:4])
                if (x | y) & result or (z & result and z != result):
                    found.append((line, other, waits, before_read))
                left = result - to
            else:
                to = frozenset() if o.startswith(_READS_ALL) else _regs(a.split(",")[0])
                if _regs(a if o.startswith(_READS_ALL) else a.partition(",")[2]) & result:
                    found.append((line, other, waits, before_read))
                elif to & result and o.startswith("v_") and waits < before_write:  # a load's result is late itself
                    found.append((line, other, waits, before_write))
                left = result - to
            if left:
                more = waits + (int(a.split()[0], 0) + 1 if o == "s_nop" else 1)
                todo += [(t, more, left) for t in follow[k]]
    return found, count


def _sources_with_products():
    """The units whose own text or headers have matrix instructions."""
    def text(path, seen):
        if path in seen or not os.path.exists(path):
            return ""
        seen.add(path)
        with open(path) as f:
            own = f.read()
        return own + "".join(text(os.path.join(os.path.dirname(path), h), seen)
                             for h in re.findall(r'#include "([^"]+)"', own))

    csrc = os.path.join(_PKG, "csrc")
    for src in sorted(glob.glob(os.path.join(csrc, "*.hip")) + glob.glob(os.path.join(csrc, "ops", "*.hip"))):
        if "__builtin_amdgcn_mfma" in text(src, set()):
            yield os.path.basename(src)[:-len(".hip")]


@pytest.mark.parametrize("unit", list(_sources_with_products()))
def test_results_are_awaited_on_every_path(unit, tmp_path):
    if not all(os.path.exists(os.path.join(_LLVM, t)) for t in ("llvm-objcopy", "clang-offload-bundler", "llvm-objdump")):
        pytest.skip("LLVM tools of the ROCm install not found")
    obj = os.path.join(_PKG, "_build", unit + ".o")
    if not os.path.exists(obj):
        pytest.skip("library not built (make -C causal-conv1d-triton_amd)")
    bad = []
    for name, at, code in kernels_of(_listing(obj, str(tmp_path))):
        if any(c[0].startswith("v_mfma") for c in code):
            found, _ = too_early(at, code)
            bad += [f"{name}: {x.split('//')[0].strip()} -> {y.split('//')[0].strip()} after {w} of {n}"
                    for x, y, w, n in found]
    assert not bad, "\n".join(bad)


def _text(lines):
    """A listing of a kernel k; `L:` in front of a line is its label, `>L` in a branch a jump to it."""
    labels = {s.split(":")[0]: 4 * i for i, s in enumerate(lines) if ":" in s.split(" ")[0]}
    out = ["0000000000000000 <k>:"]
    for i, s in enumerate(lines):
        s = s.split(": ", 1)[1] if ":" in s.split(" ")[0] else s
        to = re.search(r">(\w+)", s)
        out.append(f"\t{s.split('>')[0].strip()} // {4 * i:012X}:" + (f" <k+0x{labels[to.group(1)]:x}>" if to else ""))
    return "\n".join(out)


F32, BF = "v_mfma_f32_16x16x4_f32", "v_mfma_f32_16x16x32_bf16"


@pytest.mark.parametrize("lines,early", [
    ([f"{BF} v[0:3], v[4:7], v[8:11], 0", "s_nop 7", "v_mul_f32_e32 v4, v9, v3", "s_endpgm"], 0),
    ([f"{BF} v[0:3], v[4:7], v[8:11], 0", "s_nop 6", "v_mul_f32_e32 v4, v9, v3", "s_endpgm"], 1),
    ([f"{BF} v[0:3], v[4:7], v[8:11], 0", "s_nop 6", "v_mov_b32_e32 v3, 0", "s_endpgm"], 0),
    ([f"{BF} v[0:3], v[4:7], v[8:11], 0", "s_nop 5", "v_mov_b32_e32 v3, 0", "s_endpgm"], 1),
    ([f"{BF} v[0:3], v[4:7], v[8:11], 0", f"{BF} v[0:3], v[4:7], v[8:11], v[0:3]", "s_nop 7",
      "global_store_dwordx4 v12, v[0:3], s[2:3]", "s_endpgm"], 0),
    ([f"{F32} a[0:3], v4, v5, 0", "s_nop 7", "s_nop 0", "v_accvgpr_read_b32 v6, a3", "s_endpgm"], 1),
    ([f"{F32} a[0:3], v4, v5, 0", f"{F32} v[6:9], v0, v1, a[0:3]", "s_nop 1", "v_accvgpr_read_b32 v16, a3",
      "s_endpgm"], 0),
    # the shorter of two paths: the branch jumps over what the other one waits with
    ([f"{F32} a[0:3], v4, v5, 0", "s_and_b64 vcc, exec, s[6:7]", "s_cbranch_vccz >L", "s_nop 7", "ds_read2_b32 a[0:1], v9",
      "L: s_waitcnt lgkmcnt(0)", "v_accvgpr_read_b32 v6, a3", "s_endpgm"], 1),
    ([f"{F32} a[0:3], v4, v5, 0", "s_and_b64 vcc, exec, s[6:7]", "s_cbranch_vccz >L", "s_nop 7", "ds_read2_b32 a[0:1], v9",
      "L: s_waitcnt lgkmcnt(0)", "s_nop 6", "v_accvgpr_read_b32 v6, a3", "s_endpgm"], 0),
])
def test_the_reading_finds_what_is_planted(lines, early):
    (_, at, code), = kernels_of(_text(lines))
    found, count = too_early(at, code)
    assert len(found) == early and count == sum("mfma" in s for s in lines), found
