"""Attention over the 8-bit cache where the weights of one row differ by many orders of magnitude: what the two 8-bit
pieces of a weight keep of small weights next to large ones."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.q8 import Q8CacheOracle, quantise

pytestmark = pytest.mark.gpu


def f64(t):
    return t.double().cpu().numpy()


def bf16(x):
    return torch.as_tensor(x).to(torch.bfloat16)


def attend(dev, q, k, v, kernel, k_new=None, v_new=None, v_exp=None, whole=True):
    """q (1, H, Dh) after the N rows k, v (N, Hkv, Dh) of one slot: the kernel's output, the 64-bit one, the sum of
    weights times |value|, the sum of weights times the row's largest |value|, and the largest sum of |q k| terms.
    v_exp (Hkv, N): exponents put in place of the rows' own.  whole: one CTA takes a prefix (batch-invariant mode);
    spread over the GPU, a short call gives every CTA one step."""
    from wavefront_decoding_b200 import attention as wa
    from wavefront_decoding_b200 import runtime as rt
    from wavefront_decoding_b200.kv_cache import QuantKVCache
    N, Hkv, Dh = k.shape
    H = q.shape[1]
    o = Q8CacheOracle(1, 1, Hkv, Dh, N + 1)
    c = QuantKVCache(1, 1, Hkv, Dh, N + 1, torch.bfloat16, dev)
    for x, codes, exps, ours, ours_e in ((k, o.K, o.ke, c.K, c.k_exp), (v, o.V, o.ve, c.V, c.v_exp)):
        qx, ex = quantise(np.asarray(x, dtype=np.float64))
        codes[0, 0, :N], exps[0, 0, :, :N] = qx, ex.T
        if v_exp is not None and exps is o.ve:
            exps[0, 0, :, :N] = v_exp
        ours.copy_(torch.from_numpy(codes).float().to(torch.float8_e4m3fn))
        ours_e.copy_(torch.from_numpy(exps).to(torch.int8))
    kn = bf16(np.zeros((1, Hkv, Dh)) if k_new is None else k_new)
    vn = bf16(np.zeros((1, Hkv, Dh)) if v_new is None else v_new)
    items = [(0, 0, N, 1, 0)]
    ref, amp, smax = o.wave_attn(f64(q), f64(kn), f64(vn), items)
    K, V = o.values(0, 0, N + 1)
    s = np.einsum("hgd,thd->hgt", f64(q)[0].reshape(Hkv, H // Hkv, Dh), K) / np.sqrt(Dh)
    w = np.exp(s - s.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    row = np.einsum("hgt,th->hg", w, np.abs(V).max(-1)).reshape(1, H, 1)
    with rt.batch_invariant(whole):
        out = wa.wave_attn_q8(q.to(dev), kn.to(dev), vn.to(dev), c.K, c.V, c.k_exp, c.v_exp,
                              torch.tensor(items, dtype=torch.int32, device=dev), 1, kernel=kernel)
    assert rt.read_device_error(dev) == 0
    return f64(out), ref, amp, row, smax[..., None]


def bound(ref, amp, row, smax, n_keys, kernel):
    """Scores are sums of Dh <= 128 fp32 products whose terms' absolute values sum to smax, off by 136 * 2^-24 smax;
    weights by that and their sum by it again; fp32 sums of n_keys terms (n_keys + 64) * 2^-24.  Tensor-core kernel:
    a weight's two pieces are off by 2^-4 * 2^-4 of it, or, where the low piece underflows (its step there is 2^-9,
    1/16 of that in the weight), by 2^-14 on a scale where the largest of the 256 keys of a step, value scale
    included, is 2^8: 256 * 2^-22 of that largest together.  A row's codes are at most 448, twice their 2^8 at most, so
    the steps together are off by 2^-13 of the sum of weights times each row's largest |value|.  The output is rounded
    once, to 8 significant bits: off by 2^-8 of its value."""
    t = (2 * 136 * 2.0 ** -24 * smax + (n_keys + 64) * 2.0 ** -24 + (2.0 ** -8 if kernel else 0.0)) * amp
    t = t + (2.0 ** -13 * row if kernel else 0.0)
    return t + torch.finfo(torch.bfloat16).eps / 2 * (np.abs(ref) + t)


def close(out, ref, tol):
    bad = ~(np.abs(out - ref) <= tol)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4].tolist(), (np.abs(out - ref) / tol).max())


@pytest.mark.parametrize("kernel,whole", [(0, False), (1, False), (1, True)])
@pytest.mark.parametrize("H,Hkv,Dh", [(1, 1, 128), (2, 2, 64), (16, 1, 128), (32, 1, 128)])
@pytest.mark.parametrize("N,bits,at", [(8000, 15, 0), (32768, 17, 0), (65536, 18, 30000), (32768, 22, 0),
                                       (32768, 22, 32767), (65536, 25, 40001)])
def test_the_rest_behind_a_sink_counts(cuda_dev, kernel, whole, H, Hkv, Dh, N, bits, at):
    """One key weighs 2^bits times every other: where its value is zero, the output is what the others leave."""
    q = np.zeros((1, H, Dh))
    q[..., 0] = 16.0
    k = np.zeros((N, Hkv, Dh))
    k[at, :, 0] = bits * np.log(2.0) / 16.0 * np.sqrt(Dh)
    v = np.ones((N, Hkv, Dh))
    v[at, :, Dh // 2:] = 0.0
    out, ref, amp, row, smax = attend(cuda_dev, bf16(q), k, v, kernel, v_new=np.ones((1, Hkv, Dh)), whole=whole)
    tol = bound(ref, amp, row, smax, N, kernel)
    assert (tol < 0.25 * ref).all()          # an output of zero does not pass
    close(out, ref, tol)


@pytest.mark.parametrize("kernel", [0, 1])
@pytest.mark.parametrize("H,Hkv,Dh", [(2, 2, 128), (4, 2, 64), (32, 2, 64)])
@pytest.mark.parametrize("order", [1, -1, 0])
def test_scores_over_forty_nats(cuda_dev, kernel, H, Hkv, Dh, order):
    """Scores that rise, fall or change places along the prefix by more than M may be exceeded."""
    g = np.random.default_rng(order + 5)
    N = 3000
    s = np.linspace(0.0, 40.0, N)
    s = s if order == 1 else s[::-1] if order == -1 else g.permutation(s)
    q = np.zeros((1, H, Dh))
    q[..., 0] = 16.0
    k = np.zeros((N, Hkv, Dh))
    k[:, :, 0] = s[:, None] / 16.0 * np.sqrt(Dh)
    v = 1.0 + 0.25 * g.standard_normal((N, Hkv, Dh))
    out, ref, amp, row, smax = attend(cuda_dev, bf16(q), k, v, kernel)
    tol = bound(ref, amp, row, smax, N, kernel)
    assert (tol < 0.25 * np.abs(ref)).all()
    close(out, ref, tol)
