"""Gapped windows whose rows lie far apart: steps, and whole shares of a CTA, in which some rows see no key at all."""
from __future__ import annotations

import pytest

from test_q8_gpu import run_attn
from test_sample_gpu import check, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel", [0, 1])
@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("H,Hkv,Dh", [(2, 2, 128), (4, 2, 64), (16, 2, 128), (24, 4, 64)])
def test_rows_far_apart(cuda_dev, kernel, whole, H, Hkv, Dh):
    from wavefront_decoding_b200 import runtime as rt
    items = [(0, 0, 0, 5, 0), (1, 1, 255, 2, 5), (1, 0, 700, 3, 7), (0, 1, 1023, 1, 10)]
    row_pos = [0, 1, 511, 2048, 2900, 255, 2560, 700, 1535, 1536, 1023]
    with rt.batch_invariant(whole):
        run_attn(cuda_dev, H=H, Hkv=Hkv, Dh=Dh, S=2912, items=items, row_pos=row_pos, kernel=kernel, seed=2)


def test_filters_that_are_not_numbers(cuda_dev):
    """top_p NaN keeps all, min_p NaN counts as 1."""
    x, r = logits(21, 12, 3000, "f32")
    nan = float("nan")
    assert check(cuda_dev, x, r[0], k=100, p=1.0) == ids(cuda_dev, x, r[0], k=100, p=nan)
    assert check(cuda_dev, x, r[0], m=1.0) == ids(cuda_dev, x, r[0], m=nan)


def ids(dev, x, u, k=None, p=None, m=None):
    import torch
    from wavefront_decoding_b200 import fused
    n = x.shape[0]
    kw = {name: torch.full((n,), v, dtype=dt, device=dev) for name, v, dt in
          (("top_k", k, torch.int32), ("top_p", p, torch.float32), ("min_p", m, torch.float32)) if v is not None}
    return fused.sample_rows(x.to(dev), u.to(dev), **kw).tolist()
