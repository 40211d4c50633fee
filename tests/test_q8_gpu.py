"""The 8-bit KV-slot cache and the attention over it against the 64-bit oracle."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.q8 import Q8CacheOracle, quantise

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def rows(g, shape, dtype, spread=1.0):
    """Rows whose magnitudes differ by e^spread from one to the next."""
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[:-1] + (1,), generator=g))
    return x.to(DT[dtype])


def f64(t):
    return t.double().cpu().numpy()


def make_cache(n_slots, B, Hkv, Dh, S, dtype, dev, seed=0, spread=1.0, filled=True):
    """A QuantKVCache and its oracle with the same rows at every position (those past a length are stale)."""
    from wavefront_decoding_b200.kv_cache import QuantKVCache
    g = torch.Generator().manual_seed(seed)
    c = QuantKVCache(n_slots, B, Hkv, Dh, S, DT[dtype], dev)
    o = Q8CacheOracle(n_slots, B, Hkv, Dh, S)
    if filled:
        k, v = (rows(g, (n_slots, B, S, Hkv, Dh), dtype, spread) for _ in range(2))
        o.K, ke = quantise(f64(k))
        o.V, ve = quantise(f64(v))
        o.ke, o.ve = ke.transpose(0, 1, 3, 2).copy(), ve.transpose(0, 1, 3, 2).copy()
        c.K.copy_(torch.from_numpy(o.K).float().to(torch.float8_e4m3fn))
        c.V.copy_(torch.from_numpy(o.V).float().to(torch.float8_e4m3fn))
        c.k_exp.copy_(torch.from_numpy(o.ke).to(torch.int8))
        c.v_exp.copy_(torch.from_numpy(o.ve).to(torch.int8))
    return c, o, g


def same_cache(c, o):
    assert np.array_equal(f64(c.K.float()), o.K) and np.array_equal(f64(c.V.float()), o.V)
    assert np.array_equal(c.k_exp.cpu().numpy(), o.ke) and np.array_equal(c.v_exp.cpu().numpy(), o.ve)


def no_error(dev):
    from wavefront_decoding_b200 import runtime as rt
    assert rt.read_device_error(dev) == 0


def error_bits(dev):
    from wavefront_decoding_b200 import _abi
    from wavefront_decoding_b200 import runtime as rt
    with pytest.raises(_abi.WfdError) as e:
        rt.read_device_error(dev)
    return int(str(e.value).split("bits=0x")[1].rstrip(")"), 16)


def tolerance(ref, amp, smax, n_keys, dtype, tc):
    """How far an output may be.  A score is a sum of Dh <= 128 products in fp32 whose terms' absolute values sum to
    smax: off by at most 136 * 2^-24 smax with its scalings; the weights move by twice that (their sum with them).
    A weight's two e4m3 pieces are off by 2^-4 * 2^-4 of it (tensor-core kernel), or by 2^-14 of 1/256 of the
    largest weight where the low piece underflows; exp2 and the sums of up to n_keys terms in fp32 add
    (n_keys + 64) * 2^-24.  All of it scales with the output's sum taken of |v|; the output is rounded once."""
    d = 2 * 136 * 2.0 ** -24 * smax[..., None] + (n_keys + 64) * 2.0 ** -24
    vmax = amp.max()
    t = (d + (2.0 ** -8 if tc else 0.0)) * amp + (n_keys * 2.0 ** -22 * vmax if tc else 0.0)
    eps = torch.finfo(DT[dtype]).eps / 2
    return t + eps * (np.abs(ref) + t)


# ---------------------------------------------------------------------------
# rows in, rows out
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("Hkv,Dh", [(1, 16), (3, 32), (2, 64), (24, 64), (5, 128), (1, 256)])
def test_write_tokens_and_read_back(cuda_dev, dtype, Hkv, Dh):
    from wavefront_decoding_b200.kv_cache import QuantKVCache
    g = torch.Generator().manual_seed(3)
    n_slots, B, S = 3, 2, 37
    c = QuantKVCache(n_slots, B, Hkv, Dh, S, DT[dtype], cuda_dev)
    o = Q8CacheOracle(n_slots, B, Hkv, Dh, S)
    where = [(s, b, p) for s in range(n_slots) for b in range(B) for p in range(S)]
    perm = torch.randperm(len(where), generator=g).tolist()
    k, v = (rows(g, (len(where), Hkv, Dh), dtype, 4.0) for _ in range(2))
    for r, i in enumerate(perm):
        o.put(*where[i], f64(k[r]), f64(v[r]))
    sl, sq, ps = (list(t) for t in zip(*[where[i] for i in perm]))
    c.write_tokens(sl, sq, ps, k.to(cuda_dev), v.to(cuda_dev))
    same_cache(c, o)
    assert np.array_equal(c.lens.cpu().numpy(), o.lens)
    segs = [(2, 1, S - 1), (0, 0, 0), (1, 1, 31), (1, 0, 32)]
    kp, vp, cu, mx = c.gather_pack(*(list(t) for t in zip(*segs)))
    assert mx == S and cu.tolist() == [0, S, S + 1, S + 33, S + 66]
    for i, (s, b, u) in enumerate(segs):
        for got, ref in zip((kp, vp), o.values(s, b, u + 1)):
            assert np.array_equal(f64(got[cu[i]:cu[i + 1]]), ref)   # a value has 4 significant bits: exact in bf16
    no_error(cuda_dev)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("L", [1, 31, 32, 33, 70])
def test_write_prefill(cuda_dev, dtype, L):
    c, o, g = make_cache(2, 3, 3, 64, 70, dtype, cuda_dev, seed=1)
    k, v = (rows(g, (3, L, 3, 64), dtype) for _ in range(2))
    for b in range(3):
        for p in range(L):
            o.put(1, b, p, f64(k[b, p]), f64(v[b, p]))
    c.write_prefill(1, k.to(cuda_dev), v.to(cuda_dev))
    same_cache(c, o)                                        # positions past L and the other slot untouched
    assert np.array_equal(c.lens.cpu().numpy(), o.lens)
    no_error(cuda_dev)


def test_rounding_borders_and_extremes(cuda_dev):
    """Every tie and border of e4m3, scales at their clamp, infinities, subnormals, zeros."""
    from wavefront_decoding_b200.kv_cache import QuantKVCache
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mids = (codes[1:] + codes[:-1]) / 2
    near = torch.cat([mids, torch.nextafter(mids, mids + 1), torch.nextafter(mids, mids - 1), codes])
    near = torch.cat([near, -near, torch.zeros(-near.numel() * 2 % 63)])
    pool = near.view(-1, 63)
    ext = [[448.0], [448.0001], [3.4e38], [float("inf")], [1e-38], [1e-45], [0.0], [448.0 * 2.0 ** 32],
           [448.0 * 2.0 ** 33], [2.0 ** -30], [449.0 * 2.0 ** -32], [448.0 * 2.0 ** -33], [-float("inf")]]
    x = torch.zeros((pool.shape[0] + len(ext), 64))
    x[:pool.shape[0], 1:] = pool
    x[:pool.shape[0], 0] = 448.0                          # these rows have scale 1
    for i, e in enumerate(ext):
        x[pool.shape[0] + i, :] = e[0] * torch.linspace(0.0, 1.0, 64).nan_to_num() if np.isfinite(e[0]) else 1.5
        x[pool.shape[0] + i, 5] = e[0]
    n = x.shape[0]
    c = QuantKVCache(1, 1, 1, 64, n, torch.float32, cuda_dev)
    o = Q8CacheOracle(1, 1, 1, 64, n)
    for i in range(n):
        o.put(0, 0, i, f64(x[i:i + 1]), f64(-x[i:i + 1]))
    xd = x.to(cuda_dev).view(n, 1, 64)
    c.write_tokens([0] * n, [0] * n, list(range(n)), xd, -xd)
    same_cache(c, o)
    no_error(cuda_dev)


def test_nan_is_stored_as_zero_and_reported(cuda_dev):
    from wavefront_decoding_b200.kv_cache import QuantKVCache
    c = QuantKVCache(1, 1, 2, 64, 4, torch.bfloat16, cuda_dev)
    k = torch.ones((1, 2, 64), dtype=torch.bfloat16, device=cuda_dev)
    v = k.clone()
    v[0, 1, 7] = float("nan")
    c.write_tokens([0], [0], [2], k, v)
    assert error_bits(cuda_dev) == 256
    assert c.V[0, 0, 2, 1].float()[7] == 0 and c.V[0, 0, 2, 1].float()[8] != 0 and c.lens.item() == 3


def test_write_tokens_same_place_twice_stores_the_last(cuda_dev):
    from wavefront_decoding_b200.kv_cache import QuantKVCache
    g = torch.Generator().manual_seed(5)
    n = 3000
    c = QuantKVCache(1, 2, 1, 64, 8, torch.bfloat16, cuda_dev)
    o = Q8CacheOracle(1, 2, 1, 64, 8)
    k, v = (rows(g, (n, 1, 64), "bf16", 6.0) for _ in range(2))
    sq, ps = (torch.randint(0, m, (n,), generator=g).tolist() for m in (2, 8))
    for i in range(n):
        o.put(0, sq[i], ps[i], f64(k[i]), f64(v[i]))
    c.write_tokens([0] * n, sq, ps, k.to(cuda_dev), v.to(cuda_dev))
    same_cache(c, o)
    no_error(cuda_dev)


def test_bad_rows_are_left_out_and_reported(cuda_dev):
    c, o, g = make_cache(2, 2, 1, 64, 8, "bf16", cuda_dev)
    k = rows(g, (4, 1, 64), "bf16").to(cuda_dev)
    dev_pos = torch.tensor([8, -1, 0, 0], dtype=torch.int32, device=cuda_dev)
    c.write_tokens(torch.tensor([0, 0, 2, 0]), torch.tensor([0, 0, 0, -1]), dev_pos, k, k)
    assert error_bits(cuda_dev) == 2 | 4
    same_cache(c, o)
    i32 = dict(dtype=torch.int32, device=cuda_dev)
    fill = torch.full((3, 1, 64), 7.0, dtype=torch.bfloat16, device=cuda_dev)
    out = (fill.clone(), fill.clone())
    c.gather_packed(torch.tensor([0, 0, 5], **i32), torch.tensor([0, 1, 0], **i32),
                    torch.tensor([0, 2, 4, 4], **i32), 3, out=out)   # the second segment ends past the packs
    assert error_bits(cuda_dev) == 2 | 4
    assert torch.equal(out[0][2:], fill[2:]) and np.array_equal(f64(out[0][:2]), o.values(0, 0, 2)[0])


@pytest.mark.parametrize("mode", ["len", "mask"])
def test_commit_window(cuda_dev, mode):
    c, o, g = make_cache(3, 2, 3, 64, 40, "bf16", cuda_dev, seed=9)
    items = [[0, 0, 5, 6, 0], [1, 1, 30, 8, 6], [0, 1, 0, 1, 14], [1, 0, 7, 0, 15]]
    acc = torch.randint(0, 2, (15,), generator=g).tolist()
    lens = [3, 8, 0, 0]
    rows_ref, count_ref = [-1] * 15, []
    for i, (s, b, p0, ql, r0) in enumerate(items):
        keep = [j for j in range(ql) if (acc[r0 + j] if mode == "mask" else j < lens[i])]
        for n, j in enumerate(keep):
            for t in (o.K, o.V):
                t[s + 1, b, p0 + n] = t[s + 1, b, p0 + j]
            for t in (o.ke, o.ve):
                t[s + 1, b, :, p0 + n] = t[s + 1, b, :, p0 + j]
            rows_ref[r0 + n] = r0 + j
        o.lens[s + 1, b] = p0 + len(keep)
        count_ref.append(len(keep))
    kw = {"accept_mask": torch.tensor(acc)} if mode == "mask" else {"accept_len": torch.tensor(lens)}
    ar, ac = c.commit_window(torch.tensor(items), slot_offset=1, n_rows=15, **kw)
    same_cache(c, o)
    assert ar.tolist() == rows_ref and ac.tolist() == count_ref
    assert np.array_equal(c.lens.cpu().numpy(), o.lens)
    no_error(cuda_dev)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def run_attn(cuda_dev, *, n_slots=2, B=2, H=4, Hkv=2, Dh=128, S=300, dtype="bf16", items, row_pos=None, kernel=-1,
             seed=0, slot_offset=0, spread=1.0, q_scale=1.0, scale=None, max_q=None, check=True):
    c, o, g = make_cache(n_slots, B, Hkv, Dh, S, dtype, cuda_dev, seed, spread)
    n = max(i[3] + i[4] for i in items)
    q = (torch.randn((n, H, Dh), generator=g) * q_scale).to(DT[dtype])
    k, v = (rows(g, (n, Hkv, Dh), dtype, spread) for _ in range(2))
    ref, amp, smax = o.wave_attn(f64(q), f64(k), f64(v), items, row_pos, slot_offset, scale)
    it = torch.tensor(items, dtype=torch.int32, device=cuda_dev)
    rp = None if row_pos is None else torch.tensor(row_pos, dtype=torch.int32, device=cuda_dev)
    from wavefront_decoding_b200 import attention as wa
    out = wa.wave_attn_q8(q.to(cuda_dev), k.to(cuda_dev), v.to(cuda_dev), c.K, c.V, c.k_exp, c.v_exp, it,
                          max_q or max(i[3] for i in items), lens=c.lens, slot_offset=slot_offset, kernel=kernel,
                          row_pos=rp, scale=scale)
    if check:
        no_error(cuda_dev)
        same_cache(c, o)
        assert np.array_equal(c.lens.cpu().numpy(), o.lens)
        tc = kernel == 1 or (kernel < 0 and dtype == "bf16" and Hkv * Dh % 128 == 0)
        got = f64(out)
        live = ~np.isnan(ref)
        tol = tolerance(ref, np.nan_to_num(amp), smax, S, dtype, tc)
        bad = live & ~(np.abs(got - ref) <= tol)
        assert not bad.any(), (bad.sum(), np.argwhere(bad)[:5], np.abs(got - ref)[bad].max(), tol[bad].min())
    return out, c, o


# (items) windows of one token at the start of a slot, at tile borders (128, 256 keys), long, ragged, empty
WINDOWS = [
    [(0, 0, 0, 1, 0)],
    [(0, 0, 127, 1, 0), (1, 0, 128, 1, 1), (0, 1, 126, 3, 2), (1, 1, 255, 2, 5)],
    [(0, 0, 256, 1, 0), (1, 1, 200, 5, 1), (0, 1, 0, 4, 6), (1, 0, 17, 0, 10)],
    [(1, 1, 900, 11, 0), (0, 0, 640, 8, 11)],
]
SHAPES = [(1, 1, 128), (4, 1, 128), (7, 1, 128), (16, 4, 128), (2, 2, 64), (6, 2, 64), (12, 4, 64), (16, 2, 64)]


@pytest.mark.parametrize("w", range(len(WINDOWS)))
@pytest.mark.parametrize("H,Hkv,Dh", SHAPES)
@pytest.mark.parametrize("kernel", [0, 1])
def test_attn_bf16(cuda_dev, w, H, Hkv, Dh, kernel):
    run_attn(cuda_dev, H=H, Hkv=Hkv, Dh=Dh, S=913, items=WINDOWS[w], kernel=kernel, seed=w)


@pytest.mark.parametrize("w", range(len(WINDOWS)))
@pytest.mark.parametrize("H,Hkv,Dh", [(1, 1, 64), (4, 2, 128), (9, 3, 64), (8, 1, 64)])
def test_attn_f32(cuda_dev, w, H, Hkv, Dh):
    run_attn(cuda_dev, H=H, Hkv=Hkv, Dh=Dh, S=913, items=WINDOWS[w], dtype="f32", seed=w)


def test_attn_odd_kv_heads_bf16_runs_on_the_cuda_cores(cuda_dev):
    run_attn(cuda_dev, H=9, Hkv=3, Dh=64, S=300, items=WINDOWS[1], kernel=-1)


@pytest.mark.parametrize("H,Hkv,Dh", [(8, 2, 128), (6, 2, 64), (24, 24, 64)])
@pytest.mark.parametrize("kernel", [0, 1])
def test_attn_gapped_windows(cuda_dev, H, Hkv, Dh, kernel):
    items = [(0, 0, 3, 4, 0), (1, 1, 100, 5, 4), (1, 0, 0, 1, 9)]
    row_pos = [3, 5, 9, 140, 100, 129, 130, 255, 270, 0]
    run_attn(cuda_dev, H=H, Hkv=Hkv, Dh=Dh, S=290, items=items, row_pos=row_pos, kernel=kernel)


@pytest.mark.parametrize("kernel", [0, 1])
def test_attn_row_scales_far_apart(cuda_dev, kernel):
    """Value rows whose exponents reach both clamps, so that the largest weight and the largest score are different
    keys, and queries far from 1."""
    run_attn(cuda_dev, H=4, Hkv=2, Dh=128, items=[(0, 0, 280, 4, 0), (1, 1, 3, 2, 4)], kernel=kernel, spread=6.0,
             q_scale=2.0 ** -9)


@pytest.mark.parametrize("kernel", [0, 1])
def test_attn_sink(cuda_dev, kernel):
    """One key holds a weight 2^14 times every other's: the others' sum still counts."""
    from wavefront_decoding_b200 import attention as wa
    N, Dh = 8000, 128
    c, o, g = make_cache(1, 1, 1, Dh, N + 1, "bf16", cuda_dev, filled=False)
    q = torch.zeros((1, 1, Dh), dtype=torch.bfloat16)
    q[0, 0, 0] = 16.0
    k = torch.zeros((1, 1, N, 1, Dh))
    k[0, 0, 0, 0, 0] = 14 * np.log(2.0) / 16.0 * np.sqrt(Dh)
    v = rows(g, (1, 1, N, 1, Dh), "f32", 0.3) + 1.0
    c.write_prefill(0, k[0].to(cuda_dev), v[0].to(cuda_dev))
    for p in range(N):
        o.put(0, 0, p, f64(k[0, 0, p]), f64(v[0, 0, p]))
    kn, vn = torch.zeros((1, 1, Dh), dtype=torch.bfloat16), torch.ones((1, 1, Dh), dtype=torch.bfloat16)
    ref, amp, smax = o.wave_attn(f64(q), f64(kn), f64(vn), [(0, 0, N, 1, 0)])
    out = wa.wave_attn_q8(q.to(cuda_dev), kn.to(cuda_dev), vn.to(cuda_dev), c.K, c.V, c.k_exp, c.v_exp,
                          torch.tensor([[0, 0, N, 1, 0]], dtype=torch.int32, device=cuda_dev), 1, kernel=kernel)
    no_error(cuda_dev)
    # every flat key has w = 2^-6 on the tile's scale of 256: its pieces are off by 2^-10 * 2^-4 at most
    tol = (2.0 ** -8 + 2 * 136 * 2.0 ** -24 * smax[..., None] + (N + 64) * 2.0 ** -24) * amp + 2.0 ** -8 * np.abs(ref)
    assert (np.abs(f64(out) - ref) <= tol).all()


@pytest.mark.parametrize("kernel", [0, 1])
def test_attn_many_items_shared_slots_and_offset(cuda_dev, kernel):
    """More items than a CTA plans by itself (300), a slot offset, and items of one (slot, sequence) that see each
    other's rows."""
    items, r = [], 0
    for i in range(300):
        items.append((i % 3, (i // 3) % 5, 20 + 2 * (i // 15), 1 + i % 2, r))
        r += 1 + i % 2
    run_attn(cuda_dev, n_slots=5, B=5, H=4, Hkv=2, Dh=128, S=70, items=items, kernel=kernel, slot_offset=2)


@pytest.mark.parametrize("H,Hkv,Dh,q_len", [(8, 8, 64, 1), (16, 4, 128, 1), (16, 4, 128, 3), (16, 4, 128, 9)])
def test_attn_long_streams(cuda_dev, H, Hkv, Dh, q_len):
    """Enough work that every stream of every CTA goes round its rings several times and units straddle streams."""
    n_slots, B = 4, 4
    items = [(s, b, 5900 - 37 * b - 400 * s, q_len, (s * B + b) * q_len) for s in range(n_slots) for b in range(B)]
    run_attn(cuda_dev, n_slots=n_slots, B=B, H=H, Hkv=Hkv, Dh=Dh, S=6000, items=items, kernel=1)


def test_attn_two_items_on_one_position_store_the_later(cuda_dev):
    items = [(0, 0, 50, 4, 0), (0, 0, 52, 3, 4), (1, 0, 10, 1, 7), (1, 0, 10, 1, 8)]
    for kernel in (0, 1):
        run_attn(cuda_dev, items=items, kernel=kernel)
    run_attn(cuda_dev, items=items, row_pos=[50, 51, 52, 53, 52, 54, 60, 10, 10], kernel=1)


def test_attn_long_offsets_past_32_bits(cuda_dev):
    """Rows behind 2^32 code bytes, 2^31 rows not reached."""
    from wavefront_decoding_b200 import attention as wa
    from wavefront_decoding_b200.kv_cache import QuantKVCache
    S, Hkv, Dh = 40000, 8, 128
    c = QuantKVCache(110, 1, Hkv, Dh, S, torch.bfloat16, cuda_dev)   # 4.5 GB of codes each
    o = Q8CacheOracle(1, 1, Hkv, Dh, 40)
    g = torch.Generator().manual_seed(2)
    k, v = (rows(g, (1, 40, Hkv, Dh), "bf16") for _ in range(2))
    for p in range(39):
        o.put(0, 0, p, f64(k[0, p]), f64(v[0, p]))
    c.write_prefill(109, k[:, :39].to(cuda_dev), v[:, :39].to(cuda_dev))
    q = torch.randn((1, 8, Dh), generator=g).to(torch.bfloat16)
    ref, amp, smax = o.wave_attn(f64(q), f64(k[:, 39]), f64(v[:, 39]), [(0, 0, 39, 1, 0)])
    for kernel in (0, 1):
        out = wa.wave_attn_q8(q.to(cuda_dev), k[:, 39].to(cuda_dev), v[:, 39].to(cuda_dev), c.K, c.V, c.k_exp, c.v_exp,
                              torch.tensor([[109, 0, 39, 1, 0]], dtype=torch.int32, device=cuda_dev), 1, kernel=kernel,
                              lens=c.lens)
        assert (np.abs(f64(out) - ref) <= tolerance(ref, amp, smax, 40, "bf16", kernel == 1)).all()
    kp, _, _, _ = c.gather_pack([109], [0], [39])
    assert np.array_equal(f64(kp), o.values(0, 0, 40)[0])
    no_error(cuda_dev)


@pytest.mark.parametrize("kernel", [0, 1])
def test_attn_stale_and_masked_places_do_not_leak(cuda_dev, kernel):
    """Codes behind the windows are NaN: no output row changes."""
    from wavefront_decoding_b200 import attention as wa
    items = [(0, 0, 100, 3, 0), (1, 1, 255, 1, 3), (0, 1, 0, 2, 4)]
    outs = []
    for nan in (False, True):
        c, o, g = make_cache(2, 2, 2, 128, 300, "bf16", cuda_dev, seed=4)
        q = torch.randn((6, 4, 128), generator=g).to(torch.bfloat16).to(cuda_dev)
        k, v = (rows(g, (6, 2, 128), "bf16").to(cuda_dev) for _ in range(2))
        if nan:
            for s, b, p0, ql, _ in items:
                for t in (c.K, c.V):
                    t.view(torch.uint8)[s, b, p0 + ql:] = 0x7f
                for t in (c.k_exp, c.v_exp):
                    t[s, b, :, p0 + ql:] = 32
        outs.append(wa.wave_attn_q8(q, k, v, c.K, c.V, c.k_exp, c.v_exp,
                                    torch.tensor(items, dtype=torch.int32, device=cuda_dev), 3, kernel=kernel))
    assert torch.isfinite(outs[0].float()).all() and torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("kernel", [0, 1])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attn_query_that_is_not_finite_stays_alone(cuda_dev, kernel, bad):
    from wavefront_decoding_b200 import attention as wa
    c, o, g = make_cache(1, 1, 2, 64, 200, "bf16", cuda_dev, seed=4)
    q = torch.randn((2, 4, 64), generator=g).to(torch.bfloat16)
    k, v = (rows(g, (2, 2, 64), "bf16") for _ in range(2))
    ref, amp, smax = o.wave_attn(f64(q), f64(k), f64(v), [(0, 0, 150, 2, 0)])
    q[1, 2, 5] = bad
    out = f64(wa.wave_attn_q8(q.to(cuda_dev), k.to(cuda_dev), v.to(cuda_dev), c.K, c.V, c.k_exp, c.v_exp,
                              torch.tensor([[0, 0, 150, 2, 0]], dtype=torch.int32, device=cuda_dev), 2, kernel=kernel))
    assert np.isnan(out[1, 2]).all()
    ok = np.abs(out - ref) <= tolerance(ref, amp, smax, 200, "bf16", kernel == 1)
    ok[1, 2] = True
    assert ok.all()


def test_attn_scale_and_bad_items(cuda_dev):
    for kernel in (0, 1):
        run_attn(cuda_dev, items=WINDOWS[1], kernel=kernel, scale=0.031)
    # bad items are left out and reported: slot, sequence, rows, position past the slot, longer than max_q
    for kernel in (0, 1):
        items = [(0, 0, 9, 1, 0), (2, 0, 0, 1, 1), (0, 2, 0, 1, 1), (0, 1, 299, 2, 1), (1, 0, -1, 1, 1)]
        out, c, o = run_attn(cuda_dev, items=items[:1] + [(1, 1, 5, 1, 2)], kernel=kernel)
        from wavefront_decoding_b200 import attention as wa
        c2, _, g = make_cache(2, 2, 2, 128, 300, "bf16", cuda_dev, 0)
        before = c2.K.view(torch.uint8).clone()
        q = torch.ones((2, 4, 128), dtype=torch.bfloat16, device=cuda_dev)
        kv = torch.ones((2, 2, 128), dtype=torch.bfloat16, device=cuda_dev)
        res = torch.full_like(q, 7.0)
        wa.wave_attn_q8(q, kv, kv, c2.K, c2.V, c2.k_exp, c2.v_exp,
                        torch.tensor(items[1:] + [(0, 0, 0, 2, 1)], dtype=torch.int32, device=cuda_dev), 2, out=res,
                        lens=c2.lens, kernel=kernel)
        assert error_bits(cuda_dev) == 2 | 4 | 8
        assert torch.equal(c2.K.view(torch.uint8), before) and (res == 7).all() and (c2.lens == 0).all()


@pytest.mark.parametrize("kernel", [0, 1])
def test_attn_item_longer_than_max_q(cuda_dev, kernel):
    """Either computed or, where the kernel's variant has no room, reported and its rows left; the cache is written."""
    items = [(0, 0, 130, 5, 0), (1, 1, 64, 1, 5)]
    out, c, o = run_attn(cuda_dev, H=8, items=items, max_q=1, kernel=kernel, check=False)
    if kernel:
        assert error_bits(cuda_dev) == 8
    else:
        no_error(cuda_dev)
    same_cache(c, o)
    ref, _, _ = run_attn(cuda_dev, H=8, items=items, kernel=kernel)
    # the item within max_q: two results, each off by 2^-8 in its weights and 2^-8 in its rounding (2^-10 for the rest)
    vmax = np.abs(o.values(1, 1, 65)[1]).max()
    assert np.abs(f64(out[5]) - f64(ref[5])).max() <= 2 * (2.0 ** -7 + 2.0 ** -10) * vmax


def test_attn_repeats_bit_for_bit_and_captures(cuda_dev):
    """The same call twice, and a captured one replayed with new positions."""
    from wavefront_decoding_b200 import attention as wa
    from wavefront_decoding_b200 import runtime as rt
    rt.error_word(cuda_dev)
    c, o, g = make_cache(2, 3, 2, 128, 700, "bf16", cuda_dev, seed=8)
    items = torch.tensor([(s, b, 600 - 9 * b - s, 1, 3 * s + b) for s in range(2) for b in range(3)], dtype=torch.int32,
                         device=cuda_dev)
    q = torch.randn((6, 8, 128), generator=g).to(torch.bfloat16).to(cuda_dev)
    k, v = (rows(g, (6, 2, 128), "bf16").to(cuda_dev) for _ in range(2))
    out = torch.empty_like(q)

    def go(o=None):
        return wa.wave_attn_q8(q, k, v, c.K, c.V, c.k_exp, c.v_exp, items, 1, lens=c.lens, out=o)

    first = go()
    for _ in range(10):
        assert torch.equal(first, go())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go(out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(out)
    for step in range(3):
        items[:, 2] += 7
        graph.replay()
        got = out.clone()
        assert torch.equal(got, go())
    no_error(cuda_dev)


def test_attn_on_two_streams_and_two_graphs_at_once(cuda_dev):
    """Calls that overlap share no scratch: each gives what it gives alone."""
    from wavefront_decoding_b200 import attention as wa
    sides = []
    for seed in (1, 2):
        c, o, g = make_cache(2, 4, 2, 128, 3000, "bf16", cuda_dev, seed=seed)
        items = torch.tensor([(s, b, 2900 - 100 * b - s, 2, 2 * (4 * s + b)) for s in range(2) for b in range(4)],
                             dtype=torch.int32, device=cuda_dev)
        q = torch.randn((16, 8, 128), generator=g).to(torch.bfloat16).to(cuda_dev)
        k, v = (rows(g, (16, 2, 128), "bf16").to(cuda_dev) for _ in range(2))
        out = torch.empty_like(q)

        def go(q=q, k=k, v=v, c=c, items=items, out=out):
            wa.wave_attn_q8(q, k, v, c.K, c.V, c.k_exp, c.v_exp, items, 2, out=out)

        go()
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            for _ in range(4):
                go()
        sides.append((go, out, out.clone(), stream, graph))
    for eager in (True, False):
        for _, out, _, _, _ in sides:
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(20):
            for go, _, _, stream, graph in sides:
                with torch.cuda.stream(stream):
                    go() if eager else graph.replay()
        torch.cuda.synchronize()
        for _, out, alone, _, _ in sides:
            assert torch.equal(out, alone)
    no_error(cuda_dev)


def test_attn_batch_invariant(cuda_dev):
    """Batch-invariant mode: a row's output does not depend on the call's other items."""
    from wavefront_decoding_b200 import attention as wa
    from wavefront_decoding_b200 import runtime as rt
    c, o, g = make_cache(1, 6, 2, 128, 2000, "bf16", cuda_dev, seed=8)
    q = torch.randn((6, 8, 128), generator=g).to(torch.bfloat16).to(cuda_dev)
    k, v = (rows(g, (6, 2, 128), "bf16").to(cuda_dev) for _ in range(2))
    items = [(0, b, 1990 - 170 * b, 1, b) for b in range(6)]

    def go(rows_):
        it = torch.tensor([items[i] for i in rows_], dtype=torch.int32, device=cuda_dev)
        return wa.wave_attn_q8(q, k, v, c.K, c.V, c.k_exp, c.v_exp, it, 1)

    with rt.batch_invariant():
        whole = go(range(6))
        for i in range(6):
            assert torch.equal(go([i])[i], whole[i])


def test_attn_bounded_wait_gives_up_and_next_launch_is_exact(cuda_dev):
    from wavefront_decoding_b200 import _abi
    from wavefront_decoding_b200 import runtime as rt
    first, c, _ = run_attn(cuda_dev, items=WINDOWS[2], S=913, kernel=1)
    rt.test_fail_waits(True)
    try:
        run_attn(cuda_dev, items=WINDOWS[2], S=913, kernel=1, check=False)
        with pytest.raises(_abi.WfdError) as e:
            rt.read_device_error(cuda_dev)
        assert e.value.status == 16
    finally:
        rt.test_fail_waits(False)
    again, _, _ = run_attn(cuda_dev, items=WINDOWS[2], S=913, kernel=1)
    assert torch.equal(first[:10], again[:10])


def test_attn_strided_inputs_and_refusals(cuda_dev):
    from wavefront_decoding_b200 import _abi
    from wavefront_decoding_b200 import attention as wa
    c, o, g = make_cache(1, 1, 2, 64, 50, "bf16", cuda_dev)
    wide = torch.randn((3, 8, 128), generator=g).to(torch.bfloat16).to(cuda_dev)
    q, kv = wide[:, ::2, 64:], wide[:, :2, 1:65]
    it = torch.tensor([(0, 0, 10, 3, 0)], dtype=torch.int32, device=cuda_dev)
    a = wa.wave_attn_q8(q, kv, kv, c.K, c.V, c.k_exp, c.v_exp, it, 3)
    b = wa.wave_attn_q8(q.contiguous(), kv.clone(), kv.contiguous(), c.K, c.V, c.k_exp, c.v_exp, it, 3)
    assert torch.equal(a, b)
    args = (q, kv, kv, c.K, c.V, c.k_exp, c.v_exp, it, 3)
    for bad in [(q[:2],) + args[1:], args[:1] + (kv.float(),) + args[2:], args[:3] + (c.K.float(),) + args[4:],
                args[:5] + (c.k_exp[..., :49],) + args[6:], args[:7] + (it.long(), 3), args[:7] + (it[:, :4], 3),
                (q[:, :3],) + args[1:]]:
        with pytest.raises((ValueError, TypeError)):
            wa.wave_attn_q8(*bad)
    for kw in ({"scale": -1.0}, {"slot_offset": 1}, {"slot_offset": -1}, {"kernel": 2}):
        with pytest.raises(_abi.WfdError):
            wa.wave_attn_q8(*args, **kw)
    with pytest.raises(_abi.WfdError):
        wa.wave_attn_q8(*args[:8], 0)
    f = (q.float(), kv.float(), kv.float())
    with pytest.raises(_abi.WfdError):
        wa.wave_attn_q8(*f, *args[3:], kernel=1)
    no_error(cuda_dev)


def test_opcheck_and_fake(cuda_dev):
    c, o, g = make_cache(1, 1, 2, 128, 40, "bf16", cuda_dev)
    q = torch.randn((1, 4, 128), generator=g).to(torch.bfloat16).to(cuda_dev)
    kv = torch.randn((1, 2, 128), generator=g).to(torch.bfloat16).to(cuda_dev)
    it = torch.tensor([(0, 0, 10, 1, 0)], dtype=torch.int32, device=cuda_dev)
    # (opcheck's schema test compares arguments by arithmetic that float8 tensors lack)
    torch.library.opcheck(torch.ops.wfd.wave_attn_q8.default,
                          (q, kv, kv, c.K, c.V, c.k_exp, c.v_exp, it, 1, c.lens),
                          test_utils=("test_faketensor",))
    s = torch.ops.wfd.wave_attn_q8.default._schema
    assert [a.name for a in s.arguments if a.alias_info is not None and a.alias_info.is_write] == \
        ["k_cache", "v_cache", "k_exp", "v_exp", "lens"]
