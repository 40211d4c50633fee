"""fused.sample_rows against the sorted oracle, id for id."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.sampling import sample_row

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def check(dev, x, u, T=None, k=None, p=None, m=None, view=None, **kw):
    """x (n, V) on the CPU; view: how the device rows are laid out."""
    from wavefront_decoding_b200 import fused
    from wavefront_decoding_b200 import runtime as rt
    n = x.shape[0]

    def dv(t, dt):
        return None if t is None else torch.as_tensor(t, dtype=dt).expand(n).contiguous().to(dev)

    args = {"temperature": dv(T, torch.float32), "top_k": dv(k, torch.int32), "top_p": dv(p, torch.float32),
            "min_p": dv(m, torch.float32)}
    u = torch.as_tensor(u, dtype=torch.float32).expand(n).contiguous()
    xd = x.to(dev) if view is None else view(x, dev)
    out = fused.sample_rows(xd, u.to(dev), **args).tolist()
    assert rt.read_device_error(dev) == 0

    def at(a, r, d):
        return d if args[a] is None else args[a][r].item()

    rows = x.float().numpy()
    ref = [sample_row(rows[r], u[r].item(), at("temperature", r, 1.0), at("top_k", r, 0), at("top_p", r, 1.0),
                      at("min_p", r, 0.0)) for r in range(n)]
    assert out == ref
    return out


def logits(seed, n, V, dtype, spread=3.0, masked=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, V), generator=g) * spread
    if masked:
        x[torch.rand((n, V), generator=g) < masked] = float("-inf")
    return x.to(DT[dtype]), torch.rand((6, n), generator=g)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,V", [(1, 1), (3, 2), (2, 31), (5, 500), (1, 4097), (40, 32000), (150, 5003), (320, 700),
                                 (2, 131071), (1, 524288)])
@pytest.mark.parametrize("mode", ["plain", "k", "p", "m", "kpm"])
def test_against_the_oracle(cuda_dev, dtype, n, V, mode):
    x, r = logits(n + V, n, V, dtype)
    check(cuda_dev, x, r[0], T=0.3 + 1.5 * r[1],
          k=(1 + r[2] * min(V, 300)).int() if "k" in mode else None,
          p=0.3 + 0.69 * r[3] if "p" in mode else None, m=0.2 * r[4] if "m" in mode else None)


@pytest.mark.parametrize("spread,T", [(0.01, 1.0), (3.0, 50.0), (3.0, 0.02), (30.0, 1.0), (1e-30, 1e-30)])
def test_flat_and_peaked_rows(cuda_dev, spread, T):
    """Flat rows: thousands of tokens in one step of the histogram; peaked ones: one token holds the row."""
    for dtype in ("bf16", "f32"):
        x, r = logits(7, 20, 20000, dtype, spread)
        check(cuda_dev, x, r[0], T=T, p=0.05 + 0.9 * r[1])
        check(cuda_dev, x, r[0], T=T, k=(1 + r[2] * 15000).int())
        check(cuda_dev, x, r[0], T=T, k=(1 + r[2] * 15000).int(), p=0.05 + 0.9 * r[1], m=0.5 * r[3])


def test_ties_go_to_the_lowest_index(cuda_dev):
    """Rows of few distinct values: filters cut inside runs of equal tokens."""
    g = torch.Generator().manual_seed(1)
    V = 9000
    x = torch.randint(0, 3, (24, V), generator=g).float()
    x[5] = 0.25                                       # all equal
    x[6, :] = -3.0e38
    x[7, V // 2:] = -3.0e38
    r = torch.rand((4, 24), generator=g)
    for k in (1, 2, 100, 2048, 2049, 5000, 8999, 9000, 9001, 0, -5):
        check(cuda_dev, x, r[0], k=k)
        check(cuda_dev, x, r[0], k=k, p=0.7)
    check(cuda_dev, x, r[0], p=r[1])
    check(cuda_dev, x.bfloat16(), r[0], k=(1 + 8000 * r[2]).int(), p=r[1], m=r[3])
    assert check(cuda_dev, x[:6], 0.999999, k=1)[5] == 0 and check(cuda_dev, x[5:6], 0.5) == [V // 2]


def test_masked_rows(cuda_dev):
    INF = float("inf")
    V = 3001
    x, r = logits(3, 12, V, "f32", masked=0.6)
    x[0] = -INF                                       # nothing left: -1
    x[1] = float("nan")
    x[2] = -INF
    x[2, 77] = -1.0e30                                # one token left
    x[3, [5, 900, 2999]] = INF                        # infinities share the row
    x[4, ::2] = float("nan")
    x[5] = torch.finfo(torch.float32).min             # masks of the lowest value
    x[5, 10:20] = torch.arange(10.0)
    x[6, :-1], x[6, -1] = -INF, 0.5
    x[7] = -0.0
    x[7, 1::2] = 0.0                                  # the two zeros are one value
    for kw in ({}, {"k": 4}, {"p": 0.5}, {"m": 0.3}, {"k": 7, "p": 0.9, "m": 0.1}, {"T": 0.0}, {"k": 1500}):
        out = check(cuda_dev, x, r[0], **kw)
        assert out[0] == out[1] == -1 and out[2] == 77 and out[3] in (5, 900, 2999) and out[6] == V - 1
    assert check(cuda_dev, x[7:8], 0.99, k=1) == [0]


def test_borders_of_the_parameters(cuda_dev):
    x, r = logits(5, 30, 2000, "bf16")
    NAN, INF = float("nan"), float("inf")
    for T in (0.0, -1.0, NAN, INF, 1e-38, 1e-45, 3e38):
        check(cuda_dev, x, r[0], T=T)
        check(cuda_dev, x, r[0], T=T, k=50, p=0.9)
    for p in (0.0, -1.0, 1.0, 2.0, 1e-30, 0.99999994):
        check(cuda_dev, x, r[0], p=p)
    for m in (0.0, -1.0, 1.0, 5.0, 1e-30):
        check(cuda_dev, x, r[0], m=m)
    for u in (0.0, 1.0, 2.0, -1.0, NAN, 0.99999994, 1e-30):
        check(cuda_dev, x, u)
        check(cuda_dev, x, u, k=10, p=0.8)


@pytest.mark.parametrize("spread,T", [(1e37, 1e37), (8e37, 2e38), (1e38, float("inf")), (3.0, 1e30), (1e-38, 1e-40)])
def test_distances_and_temperatures_at_the_type_s_ends(cuda_dev, spread, T):
    """m0 - x, or the range of the histogram, past fp32's largest value; temperatures below its normal ones."""
    x, r = logits(11, 12, 9000, "f32", spread)
    x.clamp_(-3.4e38, 3.4e38)
    check(cuda_dev, x, r[0], T=T, p=0.05 + 0.9 * r[1])
    check(cuda_dev, x, r[0], T=T, k=(1 + r[2] * 8000).int(), p=0.05 + 0.9 * r[1], m=0.5 * r[3])


def test_shares_of_many_draws(cuda_dev):
    """u on a fine grid reproduces the probabilities: the share of each id is its weight to within one grid step."""
    from wavefront_decoding_b200 import fused
    n = 4096
    row = torch.tensor([2.0, -1.0, 0.5, 3.0, float("-inf"), 1.0])
    u = (torch.arange(n) / n).to(cuda_dev)
    ids = fused.sample_rows(row.expand(n, 6).to(cuda_dev), u)
    share = torch.bincount(ids.long(), minlength=6).cpu() / n
    assert (share - torch.softmax(row, 0)).abs().max() <= 1.0 / n + 1e-6
    assert (ids[1:] >= ids[:-1]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_padded_misaligned_and_expanded_rows(cuda_dev, dtype):
    x, r = logits(9, 7, 1003, dtype)

    def padded(x, dev):
        w = torch.full((x.shape[0], 1100), 99.0, dtype=x.dtype, device=dev)   # columns past V are not part of a row
        w[:, 5:5 + x.shape[1]] = x.to(dev)
        return w[:, 5:5 + x.shape[1]]

    for view in (padded, lambda x, dev: x.t().contiguous().to(dev).t()):
        check(cuda_dev, x, r[0], k=40, p=0.9, view=view)


def test_parameters_by_sequence_and_numbers_by_position(cuda_dev):
    """The engine's form: a tick table's columns select the parameters and the number of each row."""
    from wavefront_decoding_b200 import fused
    from wavefront_decoding_b200 import runtime as rt
    x, r = logits(11, 9, 800, "bf16")
    B, S = 4, 50
    g = torch.Generator().manual_seed(2)
    u = torch.rand((B, S), generator=g)
    T, k = torch.tensor([0.7, 0.0, 1.2, 1.0]), torch.tensor([0, 0, 9, 40], dtype=torch.int32)
    tab = torch.stack([torch.randint(0, S, (9,), generator=g), torch.randint(0, B, (9,), generator=g)], 1).int()
    td = tab.to(cuda_dev)
    out = fused.sample_rows(x.to(cuda_dev), u.to(cuda_dev), temperature=T.to(cuda_dev), top_k=k.to(cuda_dev),
                            row_seq=td[:, 1], row_pos=td[:, 0]).tolist()
    assert rt.read_device_error(cuda_dev) == 0
    ref = [sample_row(x[i].float().numpy(), u[b, c].item(), T[b].item(), k[b].item())
           for i, (c, b) in enumerate(tab.tolist())]
    assert out == ref
    # an index outside is reported, and only its row lost
    bad = td.clone()
    bad[3, 1], bad[4, 0], bad[5, 0] = B, S, -1
    out = fused.sample_rows(x.to(cuda_dev), u.to(cuda_dev), temperature=T.to(cuda_dev), top_k=k.to(cuda_dev),
                            row_seq=bad[:, 1], row_pos=bad[:, 0]).tolist()
    with pytest.raises(Exception, match="bits=0x8"):
        rt.read_device_error(cuda_dev)
    assert out[3] == out[4] == out[5] == -1 and out[:3] + out[6:] == ref[:3] + ref[6:]


def test_layout_does_not_change_an_id_and_graph_replay(cuda_dev):
    """A row gives the same id alone (8 CTAs) as among many (one CTA), and a captured call follows its inputs."""
    from wavefront_decoding_b200 import fused
    from wavefront_decoding_b200 import runtime as rt
    rt.error_word(cuda_dev)
    x, r = logits(13, 300, 50304, "bf16", spread=1.0)
    xd, u = x.to(cuda_dev), r[0].to(cuda_dev)
    kw = {"temperature": (0.5 + r[1]).to(cuda_dev), "top_p": (0.5 + 0.5 * r[2]).to(cuda_dev),
          "top_k": (1 + 20000 * r[3]).int().to(cuda_dev)}
    whole = fused.sample_rows(xd, u, **kw)
    for i in (0, 17, 299):
        one = {a: t[i:i + 1] for a, t in kw.items()}
        assert fused.sample_rows(xd[i:i + 1], u[i:i + 1], **one).item() == whole[i].item()
    out = torch.empty(300, dtype=torch.int32, device=cuda_dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fused.sample_rows(xd, u, out=out, **kw)
    u.copy_(torch.rand(300))
    g.replay()
    got = out.clone()
    assert torch.equal(got, fused.sample_rows(xd, u, **kw)) and not torch.equal(got, whole)


def test_greedy_is_argmax_rows(cuda_dev):
    from wavefront_decoding_b200 import fused
    x, r = logits(15, 65, 50304, "bf16")
    xd = x.to(cuda_dev)
    ref = fused.argmax_rows(xd, torch.empty(65, dtype=torch.int32, device=cuda_dev))
    assert torch.equal(ref, fused.sample_rows(xd, r[0].to(cuda_dev), temperature=torch.zeros(65, device=cuda_dev)))


def test_refusals(cuda_dev):
    from wavefront_decoding_b200 import _abi, fused
    x = torch.zeros((2, 10), device=cuda_dev)
    u = torch.zeros(2, device=cuda_dev)
    one = torch.ones(2, device=cuda_dev)
    for a, kw in [((x[0], u), {}), ((x, u.double()), {}), ((x, u[:1]), {}), ((x, u), {"temperature": one.double()}),
                  ((x, u), {"top_k": one}), ((x, u), {"top_p": one[:1]}), ((x, u), {"min_p": one[:, None]}),
                  ((x, u), {"row_pos": one.int()}), ((x, u), {"row_seq": one.long()}),
                  ((x, u), {"out": torch.empty(3, dtype=torch.int32, device=cuda_dev)}), ((x, u.cpu()), {})]:
        with pytest.raises((ValueError, TypeError)):
            fused.sample_rows(*a, **kw)
    with pytest.raises(TypeError):
        fused.sample_rows(x.half(), u)
    with pytest.raises(_abi.WfdError):
        fused.sample_rows(torch.zeros((1, (1 << 19) + 1), device=cuda_dev), u)
    assert fused.sample_rows(x[:0], u).shape == (0,)
