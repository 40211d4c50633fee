"""wfd_sample_rows_norm refuses bad rows on the host, before anything is launched."""
from __future__ import annotations

import ctypes

import pytest

INVALID, ALIGNMENT = 1, 5
A = 0x10000


@pytest.mark.parametrize("change,status", [
    ({"xn": None}, INVALID), ({"xn": A + 8}, ALIGNMENT), ({"ld": 63}, INVALID), ({"ld": 60, "d": 56}, INVALID),
    ({"d": 0}, INVALID), ({"d": 60}, INVALID), ({"eps": -1.0}, INVALID), ({"eps": float("nan")}, INVALID),
    ({"ldx": 99}, INVALID), ({"n": -1}, INVALID), ({"u": None}, INVALID), ({"n": 0, "xn": None}, 0)])
def test_bad_calls_are_refused(change, status):
    import __graft_entry__
    __graft_entry__.build()
    from wavefront_decoding_b200 import _abi
    f = dict(x=A, out=A, u=A, err=A, ldx=100, n=4, V=100, dtype=1, n_params=4, u_stride=1, u_cols=1, seq_stride=1,
             pos_stride=1, xn=A, ld=64, d=64, eps=1e-5)
    f.update(change)
    norm = [f.pop(k) for k in ("xn", "ld", "d", "eps")]
    lib = _abi.load()
    assert lib.wfd_sample_rows_norm(ctypes.byref(_abi.wfd_sample_params(**f)), *norm, None) == status
    assert lib.wfd_sample_rows_norm(None, *norm, None) == INVALID
