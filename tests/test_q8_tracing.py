"""The 8-bit cache's attention and commit are seen by whatever traces or dispatches on a call, as SlotKVCache's are."""
from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

import __graft_entry__

__graft_entry__.load_package()
from wavefront_decoding_b200 import ops  # noqa: E402,F401  (registers torch.ops.wfd.*)
from wavefront_decoding_b200.kv_cache import QuantKVCache, SlotKVCache  # noqa: E402


class Names(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace == "wfd":
            self.seen.append(func._schema.name.split("::")[1])
        return func(*args, **(kwargs or {}))


CASES = [(QuantKVCache, "_q8"), (SlotKVCache, "")]


@pytest.mark.parametrize("cls,suffix", CASES)
@pytest.mark.parametrize("update_lens", [True, False])
@pytest.mark.parametrize("with_out", [False, True])
def test_wave_attn_under_fake_tensors_and_a_dispatch_mode(cls, suffix, update_lens, with_out):
    with FakeTensorMode():
        c = cls(2, 3, 2, 128, 40, torch.bfloat16, "cuda")
        q = torch.empty((5, 8, 128), dtype=torch.bfloat16, device="cuda")
        kv = torch.empty((5, 2, 128), dtype=torch.bfloat16, device="cuda")
        it = torch.empty((5, 5), dtype=torch.int32, device="cuda")
        out = torch.empty_like(q) if with_out else None
        with Names() as names:
            o = c.wave_attn(q, kv, kv, it, 1, out=out, update_lens=update_lens)
        assert isinstance(o, FakeTensor) and o.shape == q.shape and o.dtype == q.dtype
        assert names.seen == ["wave_attn" + suffix + ("_out" if with_out else "")]
        if with_out:
            assert o is out


@pytest.mark.parametrize("cls,suffix", CASES)
@pytest.mark.parametrize("with_out", [False, True])
def test_commit_window_under_fake_tensors_and_a_dispatch_mode(cls, suffix, with_out):
    with FakeTensorMode():
        c = cls(2, 3, 2, 128, 40, torch.bfloat16, "cuda")
        i32 = dict(dtype=torch.int32, device="cuda")
        it, al = torch.empty((4, 5), **i32), torch.empty(4, **i32)
        out = (torch.empty(12, **i32), torch.empty(4, **i32)) if with_out else None
        with Names() as names:
            rows, count = c.commit_window(it, accept_len=al, n_rows=9, out=out)
        assert rows.shape == (9,) and count.shape == (4,) and rows.dtype == count.dtype == torch.int32
        assert names.seen == ["commit" + suffix + ("_out" if with_out else "")]


def test_the_commit_s_schema_names_what_it_writes():
    for name, more in (("commit_q8", []), ("commit_q8_out", ["acc_rows", "acc_count"])):
        s = getattr(torch.ops.wfd, name).default._schema
        assert [a.name for a in s.arguments if a.alias_info is not None and a.alias_info.is_write] == \
            ["k_cache", "v_cache", "k_exp", "v_exp", "lens"] + more
