"""``sage_attn_direct_bwd`` checks its arguments as ``sage_attn_bwd`` does (test_training_cpu.py), under its own name."""
import ctypes

import pytest

from test_training_cpu import ALIGNMENT, FAKE, INVALID, NULL, ODD, OK, UNSUPPORTED, bwd, lib  # noqa: F401


class Direct:
    """The library with the one entry point in the place of the other."""

    def __init__(self, lib):
        self.sage_attn_bwd = lib.sage_attn_direct_bwd


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=2), INVALID, "dtype"), (dict(D=96), UNSUPPORTED, "head_dim"), (dict(Hq=3), INVALID, "multiple"),
    (dict(Sq=2 ** 31), UNSUPPORTED, "limits"), (dict(lse=NULL), INVALID, "null"), (dict(dv=NULL), INVALID, "together"),
    (dict(q=ODD), ALIGNMENT, "aligned"), (dict(stride={5: 132}), ALIGNMENT, "multiples"),
    (dict(stride={8: 64}), INVALID, "overlap"), (dict(stride={2: 2 ** 31}), UNSUPPORTED, "32-bit"),
    (dict(), INVALID, "workspace"), (dict(ws=FAKE, wsb=64), INVALID, "workspace"),
])
def test_direct_bwd_validation(lib, kw, code, msg):  # noqa: F811
    kw = dict(kw)
    assert bwd(Direct(lib), stride=kw.pop("stride", None), **kw) == code
    text = lib.sage_last_error().decode()
    assert msg in text and ("sage_attn_direct_bwd" in text or msg in ("head_dim", "multiple"))


def test_direct_bwd_nothing_to_do(lib):  # noqa: F811
    assert bwd(Direct(lib), B=0) == OK
    assert bwd(Direct(lib), Sq=0, dk=NULL, dv=NULL) == OK
    assert ctypes.string_at(lib.sage_last_error()) == b""
