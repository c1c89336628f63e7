"""Registers of the sequence operators' kernels (device ISA metadata of a fresh hipcc -S; no GPU): none may go to scratch memory, and those that may
hold scalar registers in vector lanes are named."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))

# kernel -> scalar registers that lie in vector lanes at most: the scan's backward pass (a dozen tensors' bases and strides through its loop; more with 64 states
# and where padded ones are masked), its forward pass of more than 32 states, the convolution's backward pass, and the weight and input gradients of
# the widest gated tiles
MAY_HOLD = {
    "seq.hip": {}, "seqconv.hip": {"k_seqconv_bwd": 10}, "scan.hip": {"k_scan_bwd": 72, "k_scan_fwdIfLi16ELb0E": 8, "k_scan_fwdIDF16bLi16ELb0E": 8, "k_scan_fwdIDF16_Li16ELb0E": 8},
    "gated.hip": {"k_gated_mmaIDF16bLi1ELi256ELi256E": 44, "k_gated_mmaIDF16bLi2ELi256ELi256E": 44, "k_gated_mmaIDF16_Li1ELi256ELi256E": 44, "k_gated_mmaIDF16_Li2ELi256ELi256E": 44},
}
MUST_EXIST = {
    "seq.hip": ["k_ssm_prep", "k_seq_zero"], "seqconv.hip": ["k_seqconv_fwd", "k_seqconv_bwd", "k_seqconv_finish"],
    "scan.hip": ["k_scan_fwd", "k_scan_carry_back", "k_scan_combine", "k_scan_bwd", "k_scan_finish", "11k_scan_stepI", "k_scan_step_few"],
    "gated.hip": ["k_gated_mma", "k_gated_any", "k_gated_rows", "k_gated_grad", "k_gated_sum", "k_gated_pack"],
}


@pytest.fixture(scope="module")
def isa():
    import isa_report
    if not os.path.exists(isa_report.HIPCC):
        pytest.skip("hipcc not available")
    return isa_report.report(sorted(MAY_HOLD))


@pytest.mark.parametrize("fname", sorted(MAY_HOLD))
def test_sequence_kernels_stay_in_registers(isa, fname):
    for pat in MUST_EXIST[fname]:
        assert any(pat in name for name, _ in isa[fname]), f"no kernel of {fname} matches {pat!r}"
    for name, d in isa[fname]:
        held = max([n for pat, n in MAY_HOLD[fname].items() if pat in name], default=0)
        assert d["vgpr_spill"] == 0 and d["scratch"] == 0 and d["sgpr_spill"] <= held, (name, d)
