"""Registers and waves of the kernels of a linear-attention layer, read from the built gfx950 code objects as
tests/test_kernel_resources.py does (which also holds every kernel to no scratch memory):

* the chains of states of the delta rule have workgroups of eight waves, two per SIMD;
* the kernel in front of them, of four waves, three in bf16 up to 128 of the keys' elements, where a CU's LDS holds
  three workgroups, else two;
* the gradients of chunks two, in fp32 and small fp16 heads one;
* the norms' forward four, their backward two.
"""

import re

from test_kernel_resources import _waves_per_simd, kernels  # noqa: F401  (fixture)


def test_delta_kernels_hold_their_waves(kernels):  # noqa: F811
    found = {}
    for _, d in kernels:
        m = re.match(r"_ZN5ccv1d3ops\d+delta_(prep|fwd|bwd|grad)_kernelI(DF16b|DF16_|f)Li(\d+)E", d["name"])
        if not m:
            continue
        kind, t, dk = m.group(1), m.group(2), int(m.group(3))
        found.setdefault(kind, []).append((t, dk))
        small = t == "f" or (t == "DF16_" and dk == 64)
        need = {"prep": 3 if t == "DF16b" and dk < 256 else 2, "fwd": 2, "bwd": 2, "grad": 1 if small else 2}[kind]
        assert _waves_per_simd(int(d["vgpr_count"])) >= need, (d["name"], d["vgpr_count"])
    # one or two tiles a workgroup where the registers hold two; with and without what the backward needs
    assert len(found["prep"]) == 3 * 3 * 2 and len(found["grad"]) == 3 * 3
    assert len(found["bwd"]) == 3 * 3 + 3 and len(found["fwd"]) == 2 * (3 * 3 + 3)


def test_norm_kernels_hold_their_waves(kernels):  # noqa: F811
    n = {"fwd": 0, "bwd": 0}
    for _, d in kernels:
        m = re.match(r"_ZN5ccv1d3ops15norm_(fwd|bwd)_kernelI", d["name"])
        if not m:
            continue
        n[m.group(1)] += 1
        assert _waves_per_simd(int(d["vgpr_count"])) >= (4 if m.group(1) == "fwd" else 2), (d["name"], d["vgpr_count"])
    assert n == {"fwd": 5 * 5 * 2, "bwd": 5 * 5 * 3 * 2}  # types, row lengths, (parts,) rows of whole eights


def test_small_kernels_are_there(kernels):  # noqa: F811
    names = " ".join(d["name"] for _, d in kernels)
    for k in ("delta_update_kernel", "delta_gates_kernel", "delta_empty_kernel", "norm_reduce_kernel"):
        assert k in names, k
