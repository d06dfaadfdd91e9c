"""CPU tests of the gated projection's C entries: calls that are refused, with the status that the header gives for them."""
import ctypes

import pytest

from jvp_flash_attention_b200 import _lib

ERR_NULL, ERR_TOO_LARGE = -1, -10
LONG = 2**26 + 64  # terms of a 16-bit sum: one k-block more than are allowed


def _call(entry, args, workspace=None, **kw):
    a = args()
    a.struct_size = ctypes.sizeof(a)
    a.M = a.K = a.F = 64
    for name in ("x", "wg", "wu", "h", "kept", "gh", "dx"):
        if hasattr(a, name):
            setattr(a, name, 256)
    for k, v in kw.items():
        setattr(a, k, v)
    a.x_stride = a.wg_stride = a.wu_stride = a.K
    if workspace:
        a.workspace, a.workspace_bytes = 256, workspace
    lib = _lib.load()
    return getattr(lib, entry)(ctypes.byref(a), None), getattr(lib, entry + "_workspace")(ctypes.byref(a))


@pytest.mark.parametrize("workspace", [None, 1 << 40])
def test_sums_that_are_too_long(workspace):
    """Too large, whether a workspace was handed over or not (there is none to ask for)."""
    assert _call("jvpfa_gated_bwd", _lib.GatedBwdArgs, workspace, M=LONG, dx=None, dwg=256, dwu=256) == (ERR_TOO_LARGE, 0)
    assert _call("jvpfa_gated_bwd", _lib.GatedBwdArgs, workspace, M=300, F=LONG // 2) == (ERR_TOO_LARGE, 0)  # dx: two products together
    assert _call("jvpfa_gated_fwd", _lib.GatedFwdArgs, workspace, M=300, K=LONG, dtype=1) == (ERR_TOO_LARGE, 0)
    assert _call("jvpfa_gated_fwd", _lib.GatedFwdArgs, workspace, M=1, K=LONG) == (ERR_TOO_LARGE, 0)


def test_a_workspace_that_is_missing():
    status, need = _call("jvpfa_gated_bwd", _lib.GatedBwdArgs)
    assert status == ERR_NULL and need > 0
    assert _call("jvpfa_gated_bwd", _lib.GatedBwdArgs, need - 1) == (ERR_NULL, need)
    status, need = _call("jvpfa_gated_fwd", _lib.GatedFwdArgs, K=63)
    assert status == ERR_NULL and need > 0
