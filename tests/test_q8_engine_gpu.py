"""The engine on an 8-bit cache, with sampled ids: append, attention and sampling as a decode runs them."""
from __future__ import annotations

import pytest
import torch

from oracle import looped_lm as olm
from oracle import q8 as oq8
from oracle.sampling import sample_row
from test_engine_gpu import _prompts, _small_cfg

pytestmark = pytest.mark.gpu


def _engine(cfg, B, S, dtype=torch.float32, graphs=True, kv="e4m3"):
    from wavefront_decoding_b200.engine import WaveEngine
    from wavefront_decoding_b200.looped_lm import LoopedLM
    torch.backends.cuda.matmul.allow_tf32 = False
    model = LoopedLM(cfg, seed=0, dtype=dtype, device="cuda")
    return model, WaveEngine(model, B, S, use_graphs=graphs, kv_dtype=kv)


def _sampling(B, S, seed=3):
    from wavefront_decoding_b200.engine import SamplingParams
    g = torch.Generator().manual_seed(seed)
    return SamplingParams(u=torch.rand((B, S), generator=g), temperature=torch.tensor([0.9, 1.3, 0.0, 0.7])[:B],
                          top_k=torch.tensor([0, 60, 5, 20])[:B], top_p=0.95, min_p=0.01)


def _tokens(bt):
    return [t.tokens for t in bt.per_seq]


@pytest.mark.parametrize("kv", [None, "e4m3"])
def test_sampled_sequential_decoding_matches_the_oracle(cuda_dev, kv):
    """Ids drawn by the engine are those of the float64 model from the same numbers; where they part, the number
    lies within what fp32 logits (and cached elements that round the other way) can move a border by."""
    from wavefront_decoding_b200 import scheduler as sch
    cfg = _small_cfg()
    B, L, N = 3, 12, 10
    S = L + N + 16
    model, eng = _engine(cfg, B, S, kv=kv)
    sp = _sampling(B, S)
    eng.set_sampling(sp)
    prompts = _prompts(B, L, cfg.vocab)
    bt = sch.ar_generate_batch(eng, prompts, N)
    W, c = olm.weights_from(model)
    near = 1e-3 if kv is None else 2e-2
    for b in range(B):
        T, k = sp.temperature[b].item(), int(sp.top_k[b])

        def draw(lg, pos, du=0.0):
            return sample_row(lg.numpy(), sp.u[b, pos].item() + du, T, k, sp.top_p, sp.min_p)

        if kv is None:
            ids, logits = prompts[b].tolist(), []
            for _ in range(N):
                logits.append(olm.last_logits(W, c, torch.tensor(ids)))
                ids.append(draw(logits[-1], len(ids) - 1))
            want = ids[L:]
        else:
            want, logits, _ = oq8.decode(W, c, prompts[b].tolist(), N, draw)
        for i, tok in enumerate(bt.per_seq[b].tokens):
            if tok != want[i]:
                pos = L + i - 1
                if T > 0:
                    assert draw(logits[i], pos, near) != want[i] or draw(logits[i], pos, -near) != want[i], (b, i)
                else:
                    assert float(logits[i][want[i]] - logits[i][tok]) < near, (b, i)
                break
        else:
            continue
        assert i >= 2, "parted at once"
    from wavefront_decoding_b200 import runtime as rt
    assert rt.read_device_error(cuda_dev) == 0


def test_cached_rows_are_the_quantised_rows(cuda_dev):
    """Every cached value lies within the rounding of e4m3 of the row the float64 model holds there."""
    from wavefront_decoding_b200 import scheduler as sch
    cfg = _small_cfg()
    B, L, N = 2, 10, 8
    model, eng = _engine(cfg, B, L + N + 16)
    prompts = _prompts(B, L, cfg.vocab, seed=12)
    bt = sch.generate_wavefront_batch(eng, prompts, N, sch.SsdPolicy(4, 2), None)
    W, c = olm.weights_from(model)
    slots = list(range(cfg.n_slots))
    for b in range(B):
        toks = iter(bt.per_seq[b].tokens)
        _, _, rows = oq8.decode(W, c, prompts[b].tolist(), N, lambda lg, pos: next(toks))
        n = L + N - 1
        kp, vp, _, _ = eng.cache.gather_pack(slots, [b] * len(slots), [n - 1] * len(slots))
        for got, i in ((kp, 0), (vp, 1)):
            got = got.double().cpu().view(len(slots), n, cfg.n_kv_heads, cfg.head_dim)
            for s in slots:
                x = rows[s][i][:n]
                # half a step: 2^-4 of the value, or 2^-10 of a scale of at most 2 max / 448; the rows themselves
                # differ by what roundings of earlier rows that fell the other way move them
                amax = x.abs().amax(-1, keepdim=True)
                assert ((got[s] - x).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -9 / 448 * amax + 0.02 * amax).all(), (b, s, i)
    from wavefront_decoding_b200 import runtime as rt
    assert rt.read_device_error(cuda_dev) == 0


@pytest.mark.parametrize("kv", [None, "e4m3"])
@pytest.mark.parametrize("sampled", [False, True])
def test_wavefront_equals_sequential(cuda_dev, kv, sampled):
    """The same numbers give the same tokens whatever the schedule: sequential, wavefront on the host and on the
    device, draft-then-verify, eager and with graphs."""
    from wavefront_decoding_b200 import scheduler as sch
    from wavefront_decoding_b200.device_scheduler import generate_wavefront_device
    cfg = _small_cfg()
    B, L, N = 4, 10, 20
    S = L + N + 24
    prompts = _prompts(B, L, cfg.vocab, seed=6)
    runs = []
    for go, graphs in [(lambda e: sch.ar_generate_batch(e, prompts, N), True),
                       (lambda e: sch.generate_wavefront_batch(e, prompts, N, sch.SsdPolicy(4, 1)), True),
                       (lambda e: sch.generate_wavefront_batch(e, prompts, N, sch.SsdPolicy(4, 2)), False),
                       (lambda e: generate_wavefront_device(e, prompts, N, sch.SsdPolicy(4, 2)), True),
                       (lambda e: sch.generate_dtv_batch(e, prompts, N, sch.SsdPolicy(4, 2), 3), True)]:
        _, eng = _engine(cfg, B, S, graphs=graphs, kv=kv)
        if sampled:
            eng.set_sampling(_sampling(B, S))
        runs.append(_tokens(go(eng)))
    assert all(r == runs[0] for r in runs[1:])
    from wavefront_decoding_b200 import runtime as rt
    assert rt.read_device_error(cuda_dev) == 0


def test_sampling_can_be_changed_and_turned_off(cuda_dev):
    """New numbers reach captured graphs; without sampling the engine is greedy again."""
    from wavefront_decoding_b200 import scheduler as sch
    from wavefront_decoding_b200.device_scheduler import DeviceWave
    cfg = _small_cfg()
    B, L, N = 2, 8, 12
    S = L + N + 24
    prompts = _prompts(B, L, cfg.vocab, seed=7)
    _, eng = _engine(cfg, B, S)
    dw = DeviceWave(eng, N, sch.SsdPolicy(4, 2))

    def both():
        a, b = _tokens(sch.ar_generate_batch(eng, prompts, N)), _tokens(dw.generate(prompts))
        assert a == b
        return a

    greedy = both()
    seen = []
    for seed in (1, 2, 1):
        eng.set_sampling(_sampling(B, S, seed))
        seen.append(both())
    assert seen[0] == seen[2] != seen[1] and greedy not in seen
    eng.set_sampling(None)
    assert both() == greedy


def test_bf16_engine_on_8_bits(cuda_dev):
    """bf16: tensor-core attention over the 8-bit cache, KV sharing's gapped windows, emulated rejections."""
    from wavefront_decoding_b200 import runtime as rt
    from wavefront_decoding_b200 import scheduler as sch
    from wavefront_decoding_b200.device_scheduler import generate_wavefront_device
    for s in (0, 1, 2):
        cfg = _small_cfg(n_kv_heads=4, kv_budget_s=s)
        B, L, N = 4, 70, 16
        prompts = _prompts(B, L, cfg.vocab, seed=9)
        emus = [sch.EmulatedAcceptance(0.6, seed=b) for b in range(B)]
        toks = []
        for go in (lambda e: sch.generate_wavefront_batch(e, prompts, N, sch.SsdPolicy(4, 1), emus),
                   lambda e: generate_wavefront_device(e, prompts, N, sch.SsdPolicy(4, 1), emus)):
            emus = [sch.EmulatedAcceptance(0.6, seed=b) for b in range(B)]
            _, eng = _engine(cfg, B, L + N + 24, dtype=torch.bfloat16)
            toks.append(_tokens(go(eng)))
            assert all(len(t) == N for t in toks[-1])
            assert eng.cache.nbytes == 2 * cfg.n_slots * (B + 1) * (L + N + 24) * 4 * 65
        assert rt.read_device_error(cuda_dev) == 0


def test_bf16_batch_invariant_equality(cuda_dev):
    """Batch-invariant mode on the 8-bit cache: sampled wavefront decoding commits the sequential tokens in bf16."""
    from wavefront_decoding_b200 import scheduler as sch
    from wavefront_decoding_b200.device_scheduler import generate_wavefront_device
    cfg = _small_cfg(n_kv_heads=4)
    B, L, N = 3, 40, 24
    S = L + N + 24
    prompts = _prompts(B, L, cfg.vocab, seed=4)
    toks = []
    for T_draft in (4, 1, 2):
        _, eng = _engine(cfg, B, S, dtype=torch.bfloat16)
        eng.set_sampling(_sampling(B, S))
        toks.append(_tokens(generate_wavefront_device(eng, prompts, N, sch.SsdPolicy(4, T_draft),
                                                      batch_invariant=True)))
    assert toks[0] == toks[1] == toks[2]


def test_refusals(cuda_dev):
    from wavefront_decoding_b200.engine import SamplingParams
    cfg = _small_cfg()
    with pytest.raises(ValueError):
        _engine(cfg, 2, 32, kv="int4")
    _, eng = _engine(cfg, 2, 32)
    for p in (SamplingParams(u=torch.rand(2, 31)), SamplingParams(u=torch.rand(3, 32)),
              SamplingParams(u=torch.rand(2, 32), top_k=torch.ones(3)),
              SamplingParams(u=torch.rand(2, 32), top_p=torch.ones(2, 1))):
        with pytest.raises(ValueError):
            eng.set_sampling(p)
    assert not eng.sampling
