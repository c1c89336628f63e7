"""The sequence operators without a GPU: options, refusals and bookkeeping that their callers rely on at the edges."""
import ctypes as C

import pytest
import torch  # noqa: F401

from fastdeepqlearning_amd import _native as nat
from test_sequence_host import P, _gated

ROUND = 0x100      # FDQL_GATED_ROUND_GRADS


def test_gated_gradient_parts_are_the_callers_choice():
    """16-bit types hold the gradients in front of the products in two parts at every size, in one where the caller says so; float has one part."""
    lib = nat.load()
    need = lambda **kw: lib.fdql_gated_workspace_bytes(C.byref(_gated(**kw)), 1)  # noqa: E731
    for M, D, F in ((4, 8, 8), (60, 128, 136), (70, 128, 136), (5000, 136, 1032), (8192, 1024, 4096)):
        for dtype in (2, 3):
            assert need(dtype=dtype, M=M, D=D, F=F) - need(dtype=dtype, M=M, D=D, F=F, act=ROUND) == 2 * 2 * M * F     # dg and du once more
        assert need(dtype=0, M=M, D=D, F=F) == need(dtype=0, M=M, D=D, F=F, act=ROUND)
    for act in (ROUND | 3, ROUND << 1, -1):
        assert lib.fdql_gated(C.byref(_gated(act=act, x=P, w_gate=P, w_up=P, y=P)), None) == nat.FDQL_EINVAL
        assert "activation" in lib.fdql_last_error().decode()
