"""write_tokens of more rows than one launch takes."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.q8 import quantise

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_past_one_launch(cuda_dev, dtype):
    """40001 rows in random order, several to some places: the last of each place is stored, and no other place."""
    from wavefront_decoding_b200 import _abi
    from wavefront_decoding_b200 import runtime as rt
    from wavefront_decoding_b200.kv_cache import QuantKVCache
    n_slots, B, S, Hkv, Dh = 3, 4, 2500, 2, 16
    n = 40001
    assert n > 2 * _abi.WFD_Q8_MAX_APPEND
    g = torch.Generator().manual_seed(1)
    where = torch.randperm(n_slots * B * S, generator=g)[:25000].repeat(2)[:n]   # a place's rows in different launches
    where[20000:20100] = where[19000:19100]                                       # ... and in one
    k, v = (torch.randn((n, Hkv, Dh), generator=g).to(dtype) for _ in range(2))
    c = QuantKVCache(n_slots, B, Hkv, Dh, S, dtype, cuda_dev)
    c.write_tokens((where // (B * S)).int(), (where // S % B).int(), (where % S).int(), k.to(cuda_dev), v.to(cuda_dev))
    assert rt.read_device_error(cuda_dev) == 0
    last = np.full(n_slots * B * S, -1)
    last[where.numpy()] = np.arange(n)       # (assignment in order: the last one stands)
    held = last >= 0
    for x, codes, exps in ((k, c.K, c.k_exp), (v, c.V, c.v_exp)):
        q, e = quantise(x.double().numpy())
        got = codes.float().cpu().double().numpy().reshape(-1, Hkv, Dh)
        got_e = exps.cpu().numpy().transpose(0, 1, 3, 2).reshape(-1, Hkv)
        assert np.array_equal(got[held], q[last[held]]) and np.array_equal(got_e[held], e[last[held]])
        assert not got[~held].any() and not got_e[~held].any()
    pos = np.where(held.reshape(n_slots * B, S), np.arange(S), -1).max(1) + 1
    assert np.array_equal(c.lens.cpu().numpy().reshape(-1), pos)
