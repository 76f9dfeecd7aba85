"""The compiled form of attention's and the recurrent layer's kernels (CPU: hipcc cross-compiles): which of them spill, the
registers that the workgroups a CU need, and no packed FP32 instruction."""
import os
import re
import subprocess

import pytest

from apeiron_amd import build

# Bytes of scratch that a form may have: wide ones that were measured with them and are the faster for all that.
SPILLS = {"ah_state.hip": {r"delta_chain_kernelILi128ELi4E": 124},
          "ah_attn.hip": {r"attn_tile_kernelILi128E": 36, r"attn_shared_kernelILi128ELi128E": 36}, "ah_blocks.hip": {}}
# Vector registers that leave a SIMD its waves: two workgroups of 16 waves of the choice, of 8 of the preparation.
REGISTERS = {r"block_choice_kernel": 64, r"delta_prepare_kernel": 128, r"delta_step_kernelILi64E": 128, r"block_choices_kernelILi(64|128)E": 128}


@pytest.mark.parametrize("source", SPILLS)
def test_kernels_spill_no_more_than_measured(source, tmp_path):
    out = str(tmp_path / "k.s")
    flags = [f for f in build.FLAGS if f not in ("-shared",)]
    subprocess.run([build.HIPCC, *flags, "-x", "hip", "--cuda-device-only", "-S", os.path.join(build.CSRC, source), "-o", out], check=True, capture_output=True)
    asm = open(out).read()
    kernels = re.findall(r"\.amdhsa_kernel (\S+)(.*?)\.end_amdhsa_kernel", asm, re.S)
    assert len(kernels) > 5
    for name, body in kernels:
        most = max([b for pattern, b in SPILLS[source].items() if re.search(pattern, name)], default=0)
        assert int(re.search(r"private_segment_fixed_size (\d+)", body)[1]) <= most, name
        for pattern, registers in REGISTERS.items():
            if re.search(pattern, name):
                assert int(re.search(r"next_free_vgpr (\d+)", body)[1]) <= registers, name
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", asm)
