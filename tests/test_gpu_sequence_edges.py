"""The sequence operators on the GPU at the edges of what their documentation allows, against the 64-bit definitions of oracle/sequence.py."""
import pytest
import torch

from oracle import sequence as osq
from test_gpu_sequence import TYPES, U32, _gated_inputs, _gen, _near, _scan_call, _scan_inputs, dev, seq   # noqa: F401  (dev, seq: fixtures)

pytestmark = pytest.mark.gpu


def _norm_ratio(got, want):
    """Error's norm over that of rounding the exact values once."""
    once = (want.to(got.dtype).double() - want).norm()
    return float((got.detach().cpu().double() - want).norm() / once)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=["bf16", "f16"])
@pytest.mark.parametrize("M,D,F", [(60, 128, 136), (70, 128, 136), (300, 101, 99), (2000, 136, 200), (5000, 136, 1030), (1200, 776, 2050)])
def test_gated_gradients_round_once_at_every_size(dev, seq, M, D, F, dtype):
    """The gradients' error is that of one rounding whatever the size.  The error's mean square over n values scatters by 1 / sqrt(n) (a rounding error is
    uniform), n at least 7680 here: six of these are 7% of it, 3.5% of the norm; the float sums are off by 2^-24 sqrt(terms) of the terms' norm, at
    most 2^-18 against a rounding of 2^-9 / 2 and 2^-12 / 2 (and fp16's smallest step, 2^-24, against values near 1).  1.05 holds both.  With one part
    for d the products' terms are off by as much again: sqrt(2), within the same scatter and what fp16's subnormal numbers add."""
    x, wg, wu, _, _, dy = _gated_inputs(dev, M, D, F, dtype, False, seed=M)
    o = osq.gated_linear(x, wg, wu, None, None, "silu", dy)
    ratio = {}
    for rounded in (False, True):
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
        y = seq.gated_linear(*leaves, rounded_grads=rounded)
        grads = torch.autograd.grad(y, leaves, dy)
        ratio[rounded] = [_norm_ratio(got, o[name]) for name, got in zip(("dx", "dw_gate", "dw_up"), grads)]
    print(M, D, F, dtype, ratio)
    assert max(ratio[False]) <= 1.05, ratio
    assert max(ratio[True]) <= 1.6 and min(ratio[True]) > 1.1, ratio
