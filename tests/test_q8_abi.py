"""The 8-bit cache's and the sampler's C entries and bindings where no GPU is needed: struct layouts, refusals (each is
made on the host, before anything is launched), and the oracles against independent forms."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import q8
from oracle.sampling import sample_row

INVALID, UNSUPPORTED, ALIGNMENT = 1, 2, 5
A = 0x10000  # an address that is never read: 16-byte aligned


@pytest.fixture(scope="module")
def abi():
    import __graft_entry__
    __graft_entry__.build()
    from wavefront_decoding_b200 import _abi
    return _abi


def cache(abi, **kw):
    f = dict(k=A, v=A, k_exp=A, v_exp=A, lens=A, n_slots=2, n_seqs=3, max_seq=40, n_kv_heads=2, head_dim=64)
    f.update(kw)
    return abi.wfd_q8_cache(**f)


def test_struct_layouts(abi):
    lib = abi.load()
    assert ctypes.sizeof(abi.wfd_q8_cache) == lib.wfd_q8_cache_bytes()
    assert ctypes.sizeof(abi.wfd_sample_params) == lib.wfd_sample_params_bytes()


BAD_CACHES = [({"k": None}, INVALID), ({"v": None}, INVALID), ({"k_exp": None}, INVALID), ({"v_exp": None}, INVALID),
              ({"n_slots": 0}, INVALID), ({"n_seqs": -1}, INVALID), ({"max_seq": 0}, INVALID),
              ({"n_kv_heads": 0}, INVALID), ({"n_kv_heads": 1025}, UNSUPPORTED), ({"head_dim": 48}, UNSUPPORTED),
              ({"head_dim": 8}, UNSUPPORTED), ({"head_dim": 512}, UNSUPPORTED), ({"k": A + 8}, ALIGNMENT),
              ({"v": A + 1}, ALIGNMENT)]


def entries(abi, c, *, n=1, k=A, v=A, slot=0, L=4, dt=1, idx=A, items=A, off=0, total=4, lens=A, mask=None, q=A, out=A,
            H=4, max_q=1, which=-1, row_pos=None, rps=0, scale=0.0, ws=A):
    lib, p = abi.load(), ctypes.byref(c)
    return {
        "append": lambda: lib.wfd_append_q8(p, k, v, idx, idx, idx, n, off, dt, A, None),
        "prefill": lambda: lib.wfd_write_prefill_q8(p, k, v, slot, L, dt, A, None),
        "gather": lambda: lib.wfd_gather_q8(p, k, v, idx, idx, idx, n, total, dt, A, None),
        "commit": lambda: lib.wfd_commit_window_q8(p, items, n, lens, mask, None, None, 0, off, A, None),
        "attn": lambda: lib.wfd_wave_attn_q8(which, p, q, k, v, out, items, n, max_q, row_pos, rps, off, 4, H, dt, scale,
                                             ws, 1 << 40, A, None),
    }


@pytest.mark.parametrize("change,status", BAD_CACHES)
def test_bad_caches_are_refused(abi, change, status):
    for name, call in entries(abi, cache(abi, **change)).items():
        assert call() == status, name


@pytest.mark.parametrize("entry,change,status", [
    ("append", {"n": -1}, INVALID), ("append", {"n": 16385}, INVALID), ("append", {"k": None}, INVALID),
    ("append", {"idx": None}, INVALID), ("append", {"dt": 7}, UNSUPPORTED), ("append", {"v": A + 2}, ALIGNMENT),
    ("append", {"n": 0}, 0),
    ("prefill", {"slot": 2}, INVALID), ("prefill", {"slot": -1}, INVALID), ("prefill", {"L": 41}, INVALID),
    ("prefill", {"L": -1}, INVALID), ("prefill", {"v": None}, INVALID), ("prefill", {"dt": 9}, UNSUPPORTED),
    ("prefill", {"k": A + 4}, ALIGNMENT), ("prefill", {"L": 0, "k": None}, 0),
    ("gather", {"n": -1}, INVALID), ("gather", {"n": 65536}, INVALID), ("gather", {"total": -1}, INVALID),
    ("gather", {"k": None}, INVALID), ("gather", {"idx": None}, INVALID), ("gather", {"dt": 5}, UNSUPPORTED),
    ("gather", {"k": A + 8}, ALIGNMENT), ("gather", {"n": 0}, 0),
    ("commit", {"n": -1}, INVALID), ("commit", {"items": None}, INVALID), ("commit", {"mask": A}, INVALID), ("commit", {"lens": None}, INVALID),
    ("commit", {"n": 0}, 0),
    ("attn", {"n": -1}, INVALID), ("attn", {"H": 3}, INVALID), ("attn", {"H": 0}, INVALID), ("attn", {"max_q": 0}, INVALID),
    ("attn", {"which": 2}, INVALID), ("attn", {"which": -2}, INVALID), ("attn", {"row_pos": A}, INVALID),
    ("attn", {"scale": -1.0}, INVALID), ("attn", {"scale": float("nan")}, INVALID),
    ("attn", {"scale": float("inf")}, INVALID), ("attn", {"dt": 4}, UNSUPPORTED), ("attn", {"q": None}, INVALID),
    ("attn", {"out": None}, INVALID), ("attn", {"items": None}, INVALID), ("attn", {"ws": None}, INVALID),
    ("attn", {"q": A + 8}, ALIGNMENT), ("attn", {"ws": A + 8}, ALIGNMENT), ("attn", {"off": 2}, INVALID),
    ("attn", {"n": 0}, 0)])
def test_bad_calls_are_refused(abi, entry, change, status):
    assert entries(abi, cache(abi), **change)[entry]() == status


@pytest.mark.parametrize("head_dim", [16, 32, 256])
def test_attention_takes_head_dims_64_and_128(abi, head_dim):
    assert entries(abi, cache(abi, head_dim=head_dim))["attn"]() == UNSUPPORTED


@pytest.mark.parametrize("change,status", [
    ({"n": -1}, INVALID), ({"V": 0}, INVALID), ({"V": (1 << 19) + 1, "ldx": 1 << 20}, INVALID), ({"ldx": 99}, INVALID),
    ({"dtype": 6}, UNSUPPORTED), ({"x": None}, INVALID), ({"out": None}, INVALID), ({"u": None}, INVALID),
    ({"err": None}, INVALID), ({"n_params": 0}, INVALID), ({"n_params": 3}, INVALID), ({"u_cols": 0}, INVALID),
    ({"u_stride": 0}, INVALID), ({"row_seq": A, "seq_stride": 0}, INVALID), ({"row_pos": A, "pos_stride": 0}, INVALID),
    ({"x": A + 1}, ALIGNMENT), ({"n": 0, "x": None}, 0)])
def test_bad_sampling_calls_are_refused(abi, change, status):
    f = dict(x=A, out=A, u=A, err=A, ldx=100, n=4, V=100, dtype=1, n_params=4, u_stride=1, u_cols=1, seq_stride=1,
             pos_stride=1)
    f.update(change)
    assert abi.load().wfd_sample_rows(ctypes.byref(abi.wfd_sample_params(**f)), None) == status
    assert abi.load().wfd_sample_rows(None, None) == INVALID


def test_python_refusals(abi):
    from wavefront_decoding_b200 import fused
    from wavefront_decoding_b200.kv_cache import QuantKVCache
    cpu = torch.device("cpu")
    with pytest.raises(ValueError, match="head_dim"):
        QuantKVCache(1, 1, 1, 48, 8, torch.bfloat16, cpu)
    with pytest.raises((TypeError, ValueError)):
        QuantKVCache(1, 1, 1, 64, 8, torch.float16, cpu)
    c = QuantKVCache(2, 1, 1, 64, 8, torch.bfloat16, cpu)
    assert c.nbytes == 2 * 2 * 8 * (64 + 1)
    with pytest.raises((TypeError, ValueError)):
        QuantKVCache.wrap(c.K, c.V, c.k_exp[:1], c.v_exp)
    with pytest.raises((TypeError, ValueError)):
        QuantKVCache.wrap(c.K.view(torch.uint8), c.V, c.k_exp, c.v_exp)
    row = torch.zeros((1, 4, 1, 64), dtype=torch.bfloat16)
    with pytest.raises((TypeError, ValueError, RuntimeError)):
        c.write_prefill(0, row, row)  # rows on the CPU
    with pytest.raises((TypeError, ValueError, RuntimeError)):
        fused.sample_rows(torch.zeros(2, 10), torch.zeros(2))


def test_rounding_of_the_oracle_is_the_type_s():
    y = torch.cat([torch.linspace(-448, 448, 20001), torch.logspace(-6, 0, 4001, base=10.0) * 0.02])
    assert np.array_equal(q8.round_e4m3(y.double().numpy()), y.to(torch.float8_e4m3fn).double().numpy())


def test_exponents_of_the_oracle():
    for top, e in ((448.0, 0), (449.0, 1), (224.0, -1), (224.1, 0), (1.0, -8), (0.0, -32), (1e30, 32), (np.inf, 32)):
        c, got = q8.quantise(np.array([[top, -top / 3 if np.isfinite(top) else 1.0]]))
        assert got[0] == e and np.abs(c).max() <= 448


def test_shares_of_the_sampling_oracle():
    """Evenly spaced numbers u give each kept id its share of the draws, to one draw either way."""
    x = np.array([1.0, -2.0, 0.5, 3.0, 2.5, -np.inf, np.nan, 3.0])
    us = (np.arange(4000) + 0.5) / 4000
    for T, k, p, m, kept in ((1.0, 0, 1.0, 0.0, [0, 1, 2, 3, 4, 7]), (0.7, 3, 1.0, 0.0, [3, 4, 7]),
                             (1.0, 0, 0.5, 0.0, [3, 7]), (1.0, 0, 1.0, 0.5, [3, 4, 7]), (1.0, 1, 1.0, 0.0, [3]),
                             (1.0, 2, 0.4, 0.0, [3])):
        ids = np.array([sample_row(x, u, T, k, p, m) for u in us])
        w = np.zeros(8)
        w[kept] = np.exp((x[kept] - 3.0) / T)
        share = 4000 * w / w.sum()
        assert (np.abs(np.bincount(ids, minlength=8) - share) <= 1.0 + 1e-9).all()
