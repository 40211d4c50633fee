"""An 8-bit cache's tensors are public attributes: each call works on what they are at that call, as SlotKVCache's do."""
from __future__ import annotations

import copy
import pickle

import pytest
import torch


@pytest.fixture(scope="module")
def cache_type():
    import __graft_entry__
    __graft_entry__.build()
    from wavefront_decoding_b200.kv_cache import QuantKVCache
    return QuantKVCache


def record(monkeypatch):
    """The addresses of the structs that reach the library, without a GPU."""
    from wavefront_decoding_b200 import ops as _ops
    from wavefront_decoding_b200 import runtime as rt
    seen = []

    def call(device, name, c, *args):
        c = c._obj
        seen.append((name, c.k, c.v, c.k_exp, c.v_exp, c.lens))

    monkeypatch.setattr(rt, "call", call)
    monkeypatch.setattr(rt, "require_cuda", lambda *t: t[0].device)
    monkeypatch.setattr(rt, "error_word", lambda d: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(rt, "stream_ptr", lambda d: 0)
    monkeypatch.setattr(_ops, "q8_workspace_bytes", lambda d, n: 16)
    return seen


def addresses(c):
    return tuple(t.data_ptr() for t in (c.K, c.V, c.k_exp, c.v_exp, c.lens))


def calls(c):
    row = torch.zeros((2, 1, 64), dtype=torch.bfloat16)
    i = torch.tensor([0], dtype=torch.int32)
    return {"wfd_append_q8": lambda: c.write_tokens([0], [0], [0], row[:1], row[:1]),
            "wfd_write_prefill_q8": lambda: c.write_prefill(0, row[None], row[None]),
            "wfd_gather_q8": lambda: c.gather_packed(i, i, torch.tensor([0, 2]), 2)}


@pytest.mark.parametrize("name", ["K", "V", "k_exp", "v_exp", "lens"])
def test_a_replaced_tensor_is_the_one_that_is_used(cache_type, monkeypatch, name):
    seen = record(monkeypatch)
    c = cache_type(2, 1, 1, 64, 8, torch.bfloat16, "cpu")
    old = getattr(c, name)
    setattr(c, name, old.clone())
    for entry, call in calls(c).items():
        call()
        assert seen.pop() == (entry, *addresses(c))
    # in place of a setter: an exchanged storage
    getattr(c, name).set_(old.clone())
    for entry, call in calls(c).items():
        call()
        assert seen.pop() == (entry, *addresses(c))


def test_a_tensor_that_no_longer_fits_is_refused(cache_type, monkeypatch):
    seen = record(monkeypatch)
    other = cache_type(2, 1, 1, 64, 9, torch.bfloat16, "cpu")
    for swap in (("K",), ("lens", torch.zeros((2, 2), dtype=torch.int32)), ("k_exp",),
                 ("K", "V", "k_exp", "v_exp", "lens")):
        c = cache_type(2, 1, 1, 64, 8, torch.bfloat16, "cpu")
        if len(swap) == 2 and not isinstance(swap[1], str):
            setattr(c, *swap)
        else:
            for name in swap:
                setattr(c, name, getattr(other, name))
        for call in calls(c).values():
            with pytest.raises(ValueError):
                call()
    assert not seen


def test_a_cache_can_be_copied_and_pickled(cache_type):
    c = cache_type(2, 1, 1, 64, 8, torch.bfloat16, "cpu")
    c.k_exp[0, 0, 0, 3] = 5
    c.K.view(torch.uint8)[1, 0, 2, 0, 7] = 0x38
    for d in (copy.deepcopy(c), pickle.loads(pickle.dumps(c))):
        assert d.K.dtype == d.V.dtype == torch.float8_e4m3fn and d.K[1, 0, 2, 0, 7].float() == 1
        assert torch.equal(d.k_exp, c.k_exp) and d.K.data_ptr() != c.K.data_ptr()
        assert (d.dtype, d.n_slots, d.B, d.S, d.n_kv_head, d.head_dim) == (c.dtype, 2, 1, 8, 1, 64)
