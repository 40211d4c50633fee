"""Sampling from a product whose RMSNorm is folded into its weight, and the engine's greedy rows in bf16."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.sampling import sample_row
from test_engine_gpu import _prompts, _small_cfg

pytestmark = pytest.mark.gpu


def rows(seed, n, V, d, dtype):
    g = torch.Generator().manual_seed(seed)
    xn = (torch.randn((n, d), generator=g) * torch.exp(2.0 * torch.randn((n, 1), generator=g))).to(dtype)
    rms = (xn.double().square().mean(1, keepdim=True) + 1e-5).sqrt()
    return (3.0 * rms * torch.randn((n, V), generator=g)).to(dtype), xn, rms[:, 0].numpy(), torch.rand((4, n), generator=g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,V,d", [(1, 500, 8), (7, 32000, 512), (200, 3001, 1536), (3, 50304, 4104)])
def test_against_the_oracle(cuda_dev, dtype, n, V, d):
    """Ids are the oracle's at temperature T times the RMS; where they part, the number u lies by a border: the
    fp32 RMS and its product with T are off by d * 2^-24 at most, and so is every exponent (up to 32) of a weight."""
    from wavefront_decoding_b200 import fused
    from wavefront_decoding_b200 import runtime as rt
    x, xn, rms, r = rows(n + d, n, V, d, dtype)
    T, k, p, m = 0.5 + r[0], (1 + 200 * r[1]).int(), 0.5 + 0.5 * r[2], 0.1 * r[2]
    wide = torch.zeros((n, d + 16), dtype=dtype, device=cuda_dev)       # rows with a stride
    wide[:, 8:8 + d] = xn.to(cuda_dev)
    T[n // 2] = 0.0
    out = fused.sample_rows(x.to(cuda_dev), r[3].to(cuda_dev), temperature=T.to(cuda_dev), top_k=k.to(cuda_dev),
                            top_p=p.to(cuda_dev), min_p=m.to(cuda_dev), norm_x=wide[:, 8:8 + d], norm_eps=1e-5)
    assert rt.read_device_error(cuda_dev) == 0
    near = 32 * d * 2.0 ** -24
    for i, got in enumerate(out.tolist()):
        row = x[i].float().numpy()

        def draw(du=0.0, dt=0.0):
            return sample_row(row, r[3, i].item() + du, T[i].item() * rms[i] * (1 + dt), int(k[i]), p[i].item(), m[i].item())

        if T[i] <= 0:
            assert got == int(np.argmax(row))
        elif got != draw():
            assert got in {draw(du, dt) for du in (-near, 0, near) for dt in (-d * 2.0 ** -24, 0, d * 2.0 ** -24)}


def test_greedy_and_layout(cuda_dev):
    from wavefront_decoding_b200 import fused
    x, xn, _, r = (t.to(cuda_dev) if isinstance(t, torch.Tensor) else t for t in rows(1, 300, 20000, 512, torch.bfloat16))
    ref = fused.argmax_rows(x, torch.empty(300, dtype=torch.int32, device=cuda_dev))
    assert torch.equal(ref, fused.sample_rows(x, r[3], temperature=torch.zeros(300, device=cuda_dev), norm_x=xn, norm_eps=1e-5))
    whole = fused.sample_rows(x, r[3], top_p=r[2].contiguous(), norm_x=xn, norm_eps=1e-5)
    for i in (0, 150, 299):
        one = fused.sample_rows(x[i:i + 1], r[3, i:i + 1], top_p=r[2, i:i + 1].contiguous(), norm_x=xn[i:i + 1], norm_eps=1e-5)
        assert one.item() == whole[i].item()


def test_refusals(cuda_dev):
    from wavefront_decoding_b200 import _abi, fused
    x, xn, _, r = (t.to(cuda_dev) if isinstance(t, torch.Tensor) else t for t in rows(1, 4, 100, 64, torch.bfloat16))
    for bad in (xn.float(), xn[:3], xn[:, ::2], xn[0], xn.cpu()):
        with pytest.raises((TypeError, ValueError)):
            fused.sample_rows(x, r[3], norm_x=bad)
    for bad, eps in ((xn[:, 1:9], 0.0), (xn[:, :12], 0.0), (xn, -1.0)):
        with pytest.raises(_abi.WfdError):
            fused.sample_rows(x, r[3], norm_x=bad, norm_eps=eps)


def test_temperature_zero_is_the_engine_s_greedy_decoding(cuda_dev):
    """bf16, with a vocabulary of near copies: ids drawn at temperature 0 are those of the engine without sampling,
    alone and beside requests that are drawn."""
    from wavefront_decoding_b200 import scheduler as sch
    from wavefront_decoding_b200.engine import SamplingParams, WaveEngine
    from wavefront_decoding_b200.looped_lm import LoopedLM
    cfg = _small_cfg(n_kv_heads=4)
    B, L, N = 4, 20, 24
    S = L + N + 24
    model = LoopedLM(cfg, seed=0, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(5)
    # 16 copies of each column, up to a step of bf16 here and there, so that the largest logits of a row nearly tie
    head = model.lm_head[:, :(cfg.vocab + 15) // 16].float().cpu().repeat_interleave(16, dim=1)[:, :cfg.vocab]
    head = head * (1 + 2.0 ** -8 * torch.randint(-1, 2, head.shape, generator=g))
    model.lm_head = head.to(torch.bfloat16).to(cuda_dev).contiguous()
    model._fold()
    prompts = _prompts(B, L, cfg.vocab, seed=3)
    runs = []
    for params in (None, SamplingParams(u=torch.rand((B, S), generator=g), temperature=0.0, top_k=5, top_p=0.5),
                   SamplingParams(u=torch.rand((B, S), generator=g), temperature=torch.tensor([0.0, 1.5, 0.0, 0.7]))):
        eng = WaveEngine(model, B, S)
        eng.set_sampling(params)
        runs.append([t.tokens for t in sch.ar_generate_batch(eng, prompts, N).per_seq])
    assert runs[1] == runs[0]
    assert runs[2][0] == runs[0][0] and runs[2][2] == runs[0][2] and runs[2][1] != runs[0][1]
