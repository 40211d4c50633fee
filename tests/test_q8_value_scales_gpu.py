"""Attention over the 8-bit cache with value rows of very different scales, compared row by row and head by head."""
from __future__ import annotations

import numpy as np
import pytest

from test_q8_weights_gpu import attend, bf16, bound, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel", [0, 1])
@pytest.mark.parametrize("H,Hkv,Dh", [(4, 2, 128), (4, 4, 64), (16, 2, 128)])
@pytest.mark.parametrize("case", ["spread", "clamps", "largest value, smallest weight"])
def test_value_scales_far_apart(cuda_dev, kernel, H, Hkv, Dh, case):
    """Value rows of very different scales under moderate scores: the largest weight times scale and the largest weight
    are different keys, up to exponents of -32 and +32."""
    g = np.random.default_rng(11)
    N = 700
    q = 2.0 * g.standard_normal((1, H, Dh))
    k = g.standard_normal((N, Hkv, Dh))
    v = g.standard_normal((N, Hkv, Dh))
    v_exp = None
    if case == "spread":
        v = v * np.exp(6.0 * g.standard_normal((N, Hkv, 1)))
    elif case == "clamps":
        v_exp = g.choice([-32, 32], p=[0.95, 0.05], size=(Hkv, N))
        v_exp[0] = -32                                   # one head: all of them at the lower clamp
    else:
        s = np.einsum("hd,thd->th", q[0].reshape(Hkv, H // Hkv, Dh).sum(1), k)
        v_exp = np.clip(np.round(-6.0 * (s - s.mean(0)) / s.std(0)), -32, 32).astype(int).T
    out, ref, amp, row, smax = attend(cuda_dev, bf16(q), k, v, kernel, v_exp=v_exp)
    tol = bound(ref, amp, row, smax, N, kernel)
    assert (tol < 0.25 * np.abs(ref)).mean() > 0.75      # most outputs are really compared
    close(out, ref, tol)
