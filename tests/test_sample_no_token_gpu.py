"""A generation in which a row has no token to draw ends with an error; -1 is never a token."""
from __future__ import annotations

import pytest
import torch

from test_engine_gpu import _prompts, _small_cfg

pytestmark = pytest.mark.gpu


def runs():
    from wavefront_decoding_b200 import scheduler as sch
    from wavefront_decoding_b200.device_scheduler import generate_wavefront_device
    return {"sequential": lambda e, p, n: sch.ar_generate_batch(e, p, n),
            "wavefront": lambda e, p, n: sch.generate_wavefront_batch(e, p, n, sch.SsdPolicy(4, 2)),
            "device": lambda e, p, n: generate_wavefront_device(e, p, n, sch.SsdPolicy(4, 2)),
            "verify": lambda e, p, n: sch.generate_dtv_batch(e, p, n, sch.SsdPolicy(4, 2), 3)}


def engine(bad, B, S):
    """An engine whose logits are all `bad` from the first tick on."""
    from wavefront_decoding_b200.engine import SamplingParams, WaveEngine
    from wavefront_decoding_b200.looped_lm import LoopedLM
    model = LoopedLM(_small_cfg(), seed=0, dtype=torch.float32, device="cuda")
    eng = WaveEngine(model, B, S)
    eng.set_sampling(SamplingParams(u=torch.rand((B, S)), temperature=1.0))
    model.head = lambda x: torch.full((x.shape[0], model.cfg.vocab), bad, device=x.device)
    return model, eng


@pytest.mark.parametrize("bad", [float("nan"), -float("inf")])
def test_first_token(cuda_dev, bad):
    _, eng = engine(bad, 2, 40)
    with pytest.raises(RuntimeError, match="no token to draw"):
        runs()["sequential"](eng, _prompts(2, 8, 512), 4)


@pytest.mark.parametrize("bad", [float("nan"), -float("inf")])
@pytest.mark.parametrize("N", [2, 6])
@pytest.mark.parametrize("how", ["sequential", "wavefront", "device", "verify"])
def test_later_tokens(cuda_dev, bad, N, how):
    from wavefront_decoding_b200 import _abi
    from wavefront_decoding_b200 import runtime as rt
    _, eng = engine(bad, 2, 40)
    eng.first_ids = lambda logits, n: [3, 4]
    with pytest.raises(RuntimeError, match="no token to draw"):
        runs()[how](eng, _prompts(2, 8, 512), N)
    try:
        rt.read_device_error(cuda_dev)      # ids of -1 that went on before the host saw them are reported as well
    except _abi.WfdError as e:
        assert "bits=0x8" in str(e)
