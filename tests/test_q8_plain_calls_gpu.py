"""wave_attn_q8 past the dispatcher and through it give the same bytes."""
from __future__ import annotations

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from test_q8_gpu import make_cache, rows

pytestmark = pytest.mark.gpu


class Names(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(func._schema.name)
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("dtype,Dh", [("bf16", 128), ("f32", 64)])
@pytest.mark.parametrize("with_out", [False, True])
def test_both_ways_agree(cuda_dev, dtype, Dh, with_out):
    from wavefront_decoding_b200 import runtime as rt
    items = torch.tensor([(0, 0, 200, 3, 0), (1, 1, 7, 1, 3), (0, 1, 299, 1, 4)], dtype=torch.int32, device=cuda_dev)
    got = []
    for way in ("plain", "mode", "grad"):
        c, _, g = make_cache(2, 2, 2, Dh, 300, dtype, cuda_dev, seed=3)
        q = torch.randn((5, 4, Dh), generator=g).to(c.dtype).to(cuda_dev)
        k, v = (rows(g, (5, 2, Dh), dtype).to(cuda_dev) for _ in range(2))
        out = torch.zeros_like(q) if with_out else None
        if way == "mode":
            with Names() as names:
                o = c.wave_attn(q, k, v, items, 3, out=out)
            assert "wfd::wave_attn_q8" + ("_out" if with_out else "") in names.seen
        elif way == "grad" and not with_out:
            o = c.wave_attn(q.requires_grad_(), k, v, items, 3).detach()
        else:
            o = c.wave_attn(q, k, v, items, 3, out=out)
        got.append((o, c.K.view(torch.uint8), c.V.view(torch.uint8), c.k_exp, c.v_exp, c.lens))
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)
    assert rt.read_device_error(cuda_dev) == 0


def test_a_profile_names_the_op(cuda_dev):
    c, _, g = make_cache(1, 1, 2, 128, 40, "bf16", cuda_dev)
    q = torch.randn((1, 4, 128), generator=g).to(torch.bfloat16).to(cuda_dev)
    kv = torch.randn((1, 2, 128), generator=g).to(torch.bfloat16).to(cuda_dev)
    it = torch.tensor([(0, 0, 10, 1, 0)], dtype=torch.int32, device=cuda_dev)
    with torch.autograd.profiler.profile() as prof:
        c.wave_attn(q, kv, kv, it, 1)
    assert any("wave_attn_q8" in e.name for e in prof.function_events)


@pytest.mark.parametrize("mode", ["len", "mask"])
def test_commit_op_is_checked(cuda_dev, mode):
    c, _, _ = make_cache(2, 2, 3, 64, 40, "bf16", cuda_dev, seed=9)
    i32 = dict(dtype=torch.int32, device=cuda_dev)
    items = torch.tensor([[0, 0, 5, 6, 0], [1, 1, 30, 8, 6]], **i32)
    al = torch.tensor([3, 8], **i32) if mode == "len" else None
    am = torch.ones(14, dtype=torch.uint8, device=cuda_dev) if mode == "mask" else None
    # (opcheck's schema test compares arguments by arithmetic that float8 tensors lack)
    torch.library.opcheck(torch.ops.wfd.commit_q8.default,
                          (c.K, c.V, c.k_exp, c.v_exp, c.lens, items, al, am, 0, 14), test_utils=("test_faketensor",))
    rows_, count = torch.empty(14, **i32), torch.empty(2, **i32)
    args = dict(accept_len=al, accept_mask=am)
    c.commit_window(items, out=(rows_, count), **args)
    for bad in ((rows_.long(), count), (rows_, count[:1]), (rows_[::2], count), (rows_.cpu(), count)):
        with pytest.raises((ValueError, RuntimeError, NotImplementedError)):
            c.commit_window(items, out=bad, **args)
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.commit_window(items, out=(rows_, count), **args)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(g):
        c.commit_window(items, out=(rows_, count), **args)
    count.zero_()
    g.replay()
    assert count.tolist() == ([3, 8] if mode == "len" else [6, 8])
