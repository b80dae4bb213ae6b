"""Registers and waves of the kernels around the convolution, read from the built gfx950 code objects as
tests/test_kernel_resources.py does (which also holds every kernel to no scratch memory):

* the recurrence's main kernels hold 4 waves per SIMD, two workgroups of 8 a CU (or one of 16), which
  their chunks are sized for, one instance of each for every combination of what a call has;
* the attention holds 2 waves per SIMD, heads of 256 in fp32 one.
"""

import re

import pytest

from test_kernel_resources import _waves_per_simd, kernels  # noqa: F401  (fixture)


def test_recurrence_kernels_hold_four_waves(kernels):  # noqa: F811
    found, bad = {}, []
    for _, d in kernels:
        m = re.match(r"_ZN5ccv1d3ops14rec_(fwd|bwd)_kernelI(DF16b|DF16_|f)Li(\d)E", d["name"])
        if not m:
            continue
        found.setdefault((m.group(1), m.group(2), int(m.group(3))), []).append(d["name"])
        if _waves_per_simd(int(d["vgpr_count"])) < 4:
            bad.append((d["name"], d["vgpr_count"]))
    assert not bad, f"fewer waves than the chunks are sized for: {bad}"
    for k, sizes in (("fwd", 2), ("bwd", 1)):
        # decay, input gate, packed, streamed; a 16-bit single channel is never streamed. The forward also
        # has workgroups of 16 waves.
        assert {t: len(found[k, t, c]) for t, c in (("DF16b", 2), ("DF16_", 2), ("f", 1))} == {
            "DF16b": 16 * sizes, "DF16_": 16 * sizes, "f": 16 * sizes}
        assert len(found[k, "DF16b", 1]) == len(found[k, "DF16_", 1]) == 8 * sizes


def test_attention_kernels_hold_two_waves(kernels):  # noqa: F811
    n = 0
    for _, d in kernels:
        m = re.match(r"_ZN5ccv1d3ops17paged_attn_kernelI(DF16b|DF16_|f)Li(\d+)E", d["name"])
        if not m:
            continue
        n += 1
        need = 1 if m.group(1) == "f" and m.group(2) == "256" else 2
        assert _waves_per_simd(int(d["vgpr_count"])) >= need, (d["name"], d["vgpr_count"])
    assert n == 3 * 5 * 3  # types, head sizes, ways that pages meet steps


def test_small_kernels_are_there(kernels):  # noqa: F811
    names = " ".join(d["name"] for _, d in kernels)
    for n in ("rec_clear_kernel", "rec_empty_kernel", "rec_reduce_kernel", "rec_update_kernel",
              "paged_plan_kernel", "paged_write_kernel", "paged_join_kernel"):
        assert n in names, n
