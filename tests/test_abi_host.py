"""Structs of include/fdql.h that another version's client hands in."""
import ctypes as C
import os
import re

import pytest

from fastdeepqlearning_amd import _native as nat
from fastdeepqlearning_amd.core import make_config

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_version_is_the_headers():
    header = open(os.path.join(ROOT, "include", "fdql.h")).read()
    assert nat.load().fdql_version() == nat.VERSION == int(re.search(r"#define FDQL_VERSION (\d+)", header).group(1)) >= 2


@pytest.mark.parametrize("T,B,kw", [(2, 1, {}), (50, 256, {}), (4, 6, dict(joiner_gru=True)), (2, 1, dict(distributional=False, bootstrap_nstep=True)), (2, 1, dict(hard_updates=True))])
def test_agent_struct_without_the_state_space_fields_is_refused(T, B, kw):
    """A client built before joiner_ssm, ssm_inner and ssm_state has every later field three places further in front: an error, not other switches."""
    old_fields = [f for f in nat.AgentConfig._fields_ if f[0] not in ("joiner_ssm", "ssm_inner", "ssm_state")]

    class Old(C.Structure):
        _fields_ = old_fields + [("behind", C.c_char * 32)]       # (what the library reads past such a struct's end)
    cfg, old = make_config(17, 6, T, B, **kw), Old()
    for name, _ in old_fields:
        setattr(old, name, getattr(cfg, name))
    lib, h = nat.load(), C.c_void_p()
    assert lib.fdql_agent_create(C.byref(h), C.cast(C.byref(old), C.POINTER(nat.AgentConfig))) == nat.FDQL_EINVAL
    assert b"version" in lib.fdql_last_error()
    assert lib.fdql_agent_create(C.byref(h), C.byref(cfg)) == nat.FDQL_OK
    lib.fdql_agent_destroy(h)
