"""Tensors of an 8-bit cache that are not all on one GPU are refused before any address of them is used."""
from __future__ import annotations

import pytest
import torch


@pytest.fixture(scope="module")
def pkg():
    import __graft_entry__
    __graft_entry__.build()
    import wavefront_decoding_b200
    return wavefront_decoding_b200


def tensors(device="cpu"):
    K = torch.zeros((2, 1, 8, 1, 64), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    e = torch.zeros((2, 1, 1, 8), dtype=torch.int8, device=device)
    return [K, K.clone(), e, e.clone(), torch.zeros((2, 1), dtype=torch.int32, device=device)]


@pytest.mark.parametrize("which", range(1, 5))
def test_a_cache_over_two_devices_is_refused(pkg, which):
    from wavefront_decoding_b200 import ops
    from wavefront_decoding_b200.kv_cache import QuantKVCache
    t = tensors()
    QuantKVCache.wrap(*t)
    t[which] = t[which].to("meta")
    with pytest.raises(ValueError, match="device"):
        QuantKVCache.wrap(*t)
    with pytest.raises(ValueError, match="device"):
        ops.q8_cache_struct(*t)


def test_every_method_of_a_cpu_cache_refuses(pkg, monkeypatch):
    """... and none gets as far as an error word, a stream or a launch."""
    from wavefront_decoding_b200 import runtime as rt
    from wavefront_decoding_b200.kv_cache import QuantKVCache

    def never(*a, **k):
        raise AssertionError("a CPU tensor got as far as the library")

    for name in ("error_word", "stream_ptr", "call"):
        monkeypatch.setattr(rt, name, never)
    c = QuantKVCache.wrap(*tensors())
    row = torch.zeros((1, 1, 64), dtype=torch.bfloat16)
    items = torch.tensor([[0, 0, 0, 1, 0]], dtype=torch.int32)
    for call in (lambda: c.write_tokens([0], [0], [0], row, row), lambda: c.write_prefill(0, row[None], row[None]),
                 lambda: c.gather_packed(torch.tensor([0]), torch.tensor([0]), torch.tensor([0, 2]), 2),
                 lambda: c.gather_pack([0], [0], [1]),
                 lambda: c.commit_window(items, accept_len=torch.tensor([1])),
                 lambda: c.wave_attn(row, row, row, items, 1),
                 lambda: c.wave_attn(row, row, row, items, 1, update_lens=False)):
        with pytest.raises(ValueError):
            call()


def test_error_word_is_a_gpu_s(pkg):
    from wavefront_decoding_b200 import runtime as rt
    before = dict(rt._err)
    for d in ("cpu", "cpu:0", "meta"):
        with pytest.raises(ValueError):
            rt.error_word(torch.device(d))
    assert rt._err == before
