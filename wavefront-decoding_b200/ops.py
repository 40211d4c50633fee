"""PyTorch custom ops over libwfd_b200: the dispatcher-level drop-in for the
reference's attention backend and KV-slot commits.

Registered in the `wfd` namespace with torch.library (schemas below), each with
a CUDA kernel (a libwfd_b200 launch on the current stream) and a fake (meta)
kernel, so the ops trace under FakeTensor / torch.compile and capture into CUDA
graphs.  Mutated arguments are declared in the schemas (`Tensor(a!)`): the KV
cache and the slot lengths.  There is no CPU kernel: a CPU tensor fails in the
dispatcher.

  wfd::attn(q, k, v, cu_q, cu_k, max_q, max_k, causal=False, scale=None) -> out
      packed varlen attention, bottom-right causal per segment.  Replaces the
      graph engine's torch.ops.aten._flash_attention_forward(q, K, V, cu_q,
      cu_k, max_q, max_k, 0.0, causal, False)[0] (graph_blocks.py:37-43) and
      fa4_attention.attn_varlen (fa4_attention.py:301-317).
  wfd::attn_out(..., Tensor(a!) out) -> ()            the same into `out`
  wfd::wave_attn(q, k_new, v_new, k_cache!, v_cache!, items, max_q,
                 lens!?=None, slot_offset=0, scale=None, kernel=-1, row_pos=None) -> out
      write_tokens + gather_pack + attn_varlen of one wavefront tick in one
      launch pair (batch_kv_cache.py:61-96, ouro_blocks_batch.py:207-231);
      row_pos (int32, one per q row, any stride) gives gapped windows their
      rows' positions (ouro_blocks_batch.py:184-205 pads such runs instead).
  wfd::wave_attn_out(..., Tensor(d!) out) -> ()
  wfd::commit(k_cache!, v_cache!, lens!, items, accept_len?, accept_mask?,
              slot_offset, n_rows) -> (acc_rows, acc_count)
      verify-window accept commit with in-place compaction
      (scheduler_batch.py:472-499 semantics, drop_positions_at_and_after
      rollback, batch_kv_cache.py:99-105).
  wfd::commit_out(..., Tensor(d!) acc_rows, Tensor(e!) acc_count) -> ()
  wfd::commit_drop(lens!, drop_pos) -> ()
      batched drop_positions_at_and_after (drop_pos[b] = -1 keeps sequence b).
  wfd::wave_attn_q8(q, k_new, v_new, k_cache!, v_cache!, k_exp!, v_exp!, items,
                    max_q, lens!?=None, slot_offset=0, scale=None, kernel=-1,
                    row_pos=None) -> out
      wave_attn over an 8-bit cache (kv_cache.QuantKVCache): the window rows are
      quantised into it, and every key is attended as the cache holds it.
  wfd::wave_attn_q8_out(..., Tensor(f!) out) -> ()
  wfd::commit_q8(k_cache!, v_cache!, k_exp!, v_exp!, lens!, items, accept_len?,
                 accept_mask?, slot_offset, n_rows) -> (acc_rows, acc_count)
  wfd::commit_q8_out(..., Tensor(f!) acc_rows, Tensor(g!) acc_count) -> ()
      commit of verify windows in an 8-bit cache: codes and exponents move as they are.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad

from . import _abi
from . import runtime as rt

_LIB = torch.library.Library("wfd", "DEF")

_SCHEMAS = {
    "attn": "attn(Tensor q, Tensor k, Tensor v, Tensor cu_q, Tensor cu_k, int max_q, int max_k, bool causal=False, "
            "float? scale=None) -> Tensor",
    "attn_out": "attn_out(Tensor q, Tensor k, Tensor v, Tensor cu_q, Tensor cu_k, int max_q, int max_k, bool causal, "
                "float? scale, Tensor(a!) out) -> ()",
    "wave_attn": "wave_attn(Tensor q, Tensor k_new, Tensor v_new, Tensor(a!) k_cache, Tensor(b!) v_cache, "
                 "Tensor items, int max_q, Tensor(c!)? lens=None, int slot_offset=0, float? scale=None, "
                 "int kernel=-1, Tensor? row_pos=None) -> Tensor",
    "wave_attn_out": "wave_attn_out(Tensor q, Tensor k_new, Tensor v_new, Tensor(a!) k_cache, Tensor(b!) v_cache, "
                     "Tensor items, int max_q, Tensor(c!)? lens, int slot_offset, float? scale, int kernel, "
                     "Tensor? row_pos, Tensor(d!) out) -> ()",
    "commit": "commit(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) lens, Tensor items, Tensor? accept_len, "
              "Tensor? accept_mask, int slot_offset, int n_rows) -> (Tensor, Tensor)",
    "commit_out": "commit_out(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) lens, Tensor items, "
                  "Tensor? accept_len, Tensor? accept_mask, int slot_offset, Tensor(d!) acc_rows, "
                  "Tensor(e!) acc_count) -> ()",
    "commit_drop": "commit_drop(Tensor(a!) lens, Tensor drop_pos) -> ()",
    "wave_attn_q8": "wave_attn_q8(Tensor q, Tensor k_new, Tensor v_new, Tensor(a!) k_cache, Tensor(b!) v_cache, "
                    "Tensor(c!) k_exp, Tensor(d!) v_exp, Tensor items, int max_q, Tensor(e!)? lens=None, "
                    "int slot_offset=0, float? scale=None, int kernel=-1, Tensor? row_pos=None) -> Tensor",
    "wave_attn_q8_out": "wave_attn_q8_out(Tensor q, Tensor k_new, Tensor v_new, Tensor(a!) k_cache, "
                        "Tensor(b!) v_cache, Tensor(c!) k_exp, Tensor(d!) v_exp, Tensor items, int max_q, "
                        "Tensor(e!)? lens, int slot_offset, float? scale, int kernel, Tensor? row_pos, "
                        "Tensor(f!) out) -> ()",
    "commit_q8": "commit_q8(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_exp, Tensor(d!) v_exp, "
                 "Tensor(e!) lens, Tensor items, Tensor? accept_len, Tensor? accept_mask, int slot_offset, int n_rows) "
                 "-> (Tensor, Tensor)",
    "commit_q8_out": "commit_q8_out(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_exp, Tensor(d!) v_exp, "
                     "Tensor(e!) lens, Tensor items, Tensor? accept_len, Tensor? accept_mask, int slot_offset, "
                     "Tensor(f!) acc_rows, Tensor(g!) acc_count) -> ()",
}
for _schema in _SCHEMAS.values():
    _LIB.define(_schema)


# ---------------------------------------------------------------------------
# argument checks shared by the kernels
# ---------------------------------------------------------------------------
def heads(q: torch.Tensor, k: torch.Tensor) -> tuple[int, int, int]:
    H, Dh = q.shape[-2], q.shape[-1]
    Hkv = k.shape[-2]
    if k.shape[-1] != Dh:
        raise ValueError(f"head_dim mismatch: q {Dh} vs k {k.shape[-1]}")
    if H % Hkv != 0:
        raise ValueError(f"query heads {H} not a multiple of kv heads {Hkv}")
    return H, Hkv, Dh


def i32(t, device) -> torch.Tensor:
    if isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.device == device and t.is_contiguous():
        return t
    t = torch.as_tensor(t)
    if t.dtype != torch.int32 or t.device != device:
        t = t.to(device=device, dtype=torch.int32)
    return t.contiguous()


def _check_varlen(q, k, v, cu_q, cu_k):
    dev = rt.require_cuda(q, k, v, cu_q, cu_k)
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape:
        raise ValueError("attn expects q (total_q, H, Dh), k/v (total_k, Hkv, Dh)")
    heads(q, k)
    if q.dtype != k.dtype or k.dtype != v.dtype:
        raise TypeError("q, k, v must share a dtype")
    if cu_q.dtype != torch.int32 or cu_k.dtype != torch.int32 or cu_q.numel() != cu_k.numel():
        raise ValueError("cu_q / cu_k must be int32 with the same number of segments + 1")
    return dev


def _check_wave(q, k_new, v_new, k_cache, v_cache, items, lens):
    dev = rt.require_cuda(q, k_new, v_new, k_cache, v_cache, items, lens)
    if k_cache.dim() != 5 or v_cache.shape != k_cache.shape:
        raise ValueError("k_cache / v_cache must be (n_slots, n_seqs, max_seq, Hkv, Dh)")
    n_slots, n_seqs, _, Hkv, Dh = k_cache.shape
    if q.dim() != 3 or q.shape[2] != Dh or k_new.shape != (q.shape[0], Hkv, Dh) or v_new.shape != k_new.shape:
        raise ValueError("q (n_rows, H, Dh) and k_new / v_new (n_rows, Hkv, Dh) must match the cache")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache / v_cache must be contiguous")
    if items.dtype != torch.int32 or items.dim() != 2 or items.shape[1] != 5 or not items.is_contiguous():
        raise ValueError("items must be a contiguous int32 (n_items, 5) device tensor")
    if lens is not None and (lens.dtype != torch.int32 or tuple(lens.shape) != (n_slots, n_seqs)):
        raise ValueError("lens must be int32 (n_slots, n_seqs)")
    return dev


def _check_commit(k_cache, v_cache, lens, items, accept_len, accept_mask):
    dev = rt.require_cuda(k_cache, v_cache, lens, items, accept_len, accept_mask)
    if (accept_len is None) == (accept_mask is None):
        raise ValueError("give exactly one of accept_len / accept_mask")
    if k_cache.dim() != 5 or v_cache.shape != k_cache.shape:
        raise ValueError("k_cache / v_cache must be (n_slots, n_seqs, max_seq, Hkv, Dh)")
    if lens.dtype != torch.int32 or tuple(lens.shape) != tuple(k_cache.shape[:2]):
        raise ValueError("lens must be int32 (n_slots, n_seqs)")
    if items.dtype != torch.int32 or items.dim() != 2 or items.shape[1] != 5 or not items.is_contiguous():
        raise ValueError("items must be a contiguous int32 (n_items, 5) device tensor")
    if accept_len is not None and accept_len.dtype != torch.int32:
        raise ValueError("accept_len must be int32")
    if accept_mask is not None and accept_mask.dtype != torch.uint8:
        raise ValueError("accept_mask must be uint8")
    return dev


def plain_eager(rows, others) -> bool:
    """Whether a call on these tensors can go to the kernel without the dispatcher, because the dispatcher would only
    hand it on: nothing compiles, traces, transforms (vmap, grad, jvp), intercepts or profiles, and every tensor is a
    plain one that needs no gradient; those of `rows` (whose type may be float32) are no views that negate.  None: an
    argument not given."""
    if torch._C._len_torch_dispatch_stack() or torch._C._len_torch_function_stack() or \
            torch.compiler.is_compiling() or torch._C._functorch.peek_interpreter_stack() is not None or \
            forward_ad._current_level >= 0 or torch.autograd._profiler_enabled() or \
            torch._C._get_tracing_state() is not None:
        return False
    for t in rows:
        if t is not None and (type(t) is not torch.Tensor or t.requires_grad or t.is_neg() or
                              torch._is_functional_tensor(t)):
            return False
    for t in others:
        if t is not None and (type(t) is not torch.Tensor or t.requires_grad):
            return False
    return True


def check_q8_cache(k, v, k_exp, v_exp, lens) -> None:
    """The shapes, types and devices of an 8-bit cache's tensors."""
    shape = k.shape
    if len(shape) != 5 or v.shape != shape or k.dtype is not torch.float8_e4m3fn or v.dtype is not k.dtype or \
            not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("K, V must be contiguous float8_e4m3fn (n_slots, n_seqs, max_seq, Hkv, Dh) tensors")
    n_slots, n_seqs, max_seq, Hkv, _ = shape
    want = (n_slots, n_seqs, Hkv, max_seq)
    for e in (k_exp, v_exp):
        if e.dtype is not torch.int8 or e.shape != want or not e.is_contiguous():
            raise ValueError("k_exp, v_exp must be contiguous int8 (n_slots, n_seqs, Hkv, max_seq) tensors")
    if lens is not None and (lens.dtype is not torch.int32 or lens.shape != (n_slots, n_seqs) or
                             not lens.is_contiguous()):
        raise ValueError("lens must be a contiguous int32 (n_slots, n_seqs) tensor")
    at = k.get_device() if k.is_cuda else None     # (an index compares faster than a device)
    for t in (v, k_exp, v_exp, lens):
        if t is not None and (t.device != k.device if at is None else t.get_device() != at):
            raise ValueError(f"an 8-bit cache's tensors must share a device: {k.device} vs {t.device}")


def q8_cache_struct(k, v, k_exp, v_exp, lens) -> "_abi.wfd_q8_cache":
    """The C view of an 8-bit cache's tensors as they are now, after their checks."""
    check_q8_cache(k, v, k_exp, v_exp, lens)
    c = _abi.wfd_q8_cache()
    c.k, c.v, c.k_exp, c.v_exp, c.lens = k.data_ptr(), v.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr(), rt.ptr(lens)
    c.n_slots, c.n_seqs, c.max_seq, c.n_kv_heads, c.head_dim = k.shape
    return c


# ---------------------------------------------------------------------------
# CUDA kernels (libwfd_b200 launches on the current stream)
# ---------------------------------------------------------------------------
def _attn_out_cuda(q, k, v, cu_q, cu_k, max_q, max_k, causal, scale, out):
    dev = _check_varlen(q, k, v, cu_q, cu_k)
    H, Hkv, Dh = heads(q, k)
    if out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor shaped like q")
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    cu_q, cu_k = cu_q.contiguous(), cu_k.contiguous()
    n = cu_q.numel() - 1
    ws, wsb = rt.workspace(dev, n, Dh)
    st = _abi.load().wfd_attn_varlen(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), cu_q.data_ptr(),
                                     cu_k.data_ptr(), n, int(max_q), q.shape[0], k.shape[0], H, Hkv, Dh,
                                     rt.dtype_code(q.dtype), 1 if causal else 0, float(scale or 0.0), ws.data_ptr(),
                                     wsb, rt.error_word(dev).data_ptr(), rt.stream_ptr(dev))
    _abi.check(st, "wfd_attn_varlen")


def _attn_cuda(q, k, v, cu_q, cu_k, max_q, max_k, causal=False, scale=None):
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _attn_out_cuda(q, k, v, cu_q, cu_k, max_q, max_k, causal, scale, out)
    return out


def _wave_attn_out_cuda(q, k_new, v_new, k_cache, v_cache, items, max_q, lens, slot_offset, scale, kernel, row_pos,
                        out):
    dev = _check_wave(q, k_new, v_new, k_cache, v_cache, items, lens)
    n_slots, n_seqs, max_seq, Hkv, Dh = k_cache.shape
    if out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor shaped like q")
    rp_stride = 1
    if row_pos is not None:
        if row_pos.dtype != torch.int32 or row_pos.dim() != 1 or row_pos.numel() < q.shape[0] or \
                row_pos.device != dev or row_pos.stride(0) < 1:
            raise ValueError("row_pos must be an int32 device vector with one position per q row")
        rp_stride = row_pos.stride(0)
    q, k_new, v_new = q.contiguous(), k_new.contiguous(), v_new.contiguous()
    n = items.shape[0]
    ws, wsb = rt.workspace(dev, n, Dh)
    st = _abi.load().wfd_wave_attn_rows(
        int(kernel), q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        out.data_ptr(), rt.ptr(lens), items.data_ptr(), n, int(max_q), rt.ptr(row_pos), rp_stride, int(slot_offset),
        q.shape[0], n_slots, n_seqs, max_seq, q.shape[1], Hkv, Dh, rt.dtype_code(q.dtype), float(scale or 0.0),
        ws.data_ptr(), wsb, rt.error_word(dev).data_ptr(), rt.stream_ptr(dev))
    _abi.check(st, "wfd_wave_attn")


def _wave_attn_cuda(q, k_new, v_new, k_cache, v_cache, items, max_q, lens=None, slot_offset=0, scale=None,
                    kernel=-1, row_pos=None):
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _wave_attn_out_cuda(q, k_new, v_new, k_cache, v_cache, items, max_q, lens, slot_offset, scale, kernel, row_pos,
                        out)
    return out


def _commit_out_cuda(k_cache, v_cache, lens, items, accept_len, accept_mask, slot_offset, acc_rows, acc_count):
    dev = _check_commit(k_cache, v_cache, lens, items, accept_len, accept_mask)
    if acc_rows.dtype != torch.int32 or acc_count.dtype != torch.int32:
        raise ValueError("acc_rows / acc_count must be int32")
    if acc_count.numel() < items.shape[0]:
        raise ValueError("acc_count needs one entry per item")
    if accept_len is not None and accept_len.numel() < items.shape[0]:
        raise ValueError("accept_len needs one entry per item")
    n_slots, n_seqs, max_seq, Hkv, Dh = k_cache.shape
    al = None if accept_len is None else accept_len.contiguous()
    am = None if accept_mask is None else accept_mask.contiguous()
    # q rows both row-indexed arrays cover: the kernel skips (and reports) windows past them
    n_rows = acc_rows.numel() if am is None else min(acc_rows.numel(), am.numel())
    st = _abi.load().wfd_commit_window(k_cache.data_ptr(), v_cache.data_ptr(), lens.data_ptr(), items.data_ptr(),
                                       items.shape[0], rt.ptr(al), rt.ptr(am), acc_rows.data_ptr(),
                                       acc_count.data_ptr(), n_rows, int(slot_offset), n_slots, n_seqs, max_seq, Hkv,
                                       Dh, rt.dtype_code(k_cache.dtype), rt.error_word(dev).data_ptr(),
                                       rt.stream_ptr(dev))
    _abi.check(st, "wfd_commit_window")


def _commit_cuda(k_cache, v_cache, lens, items, accept_len, accept_mask, slot_offset, n_rows):
    acc_rows = torch.full((int(n_rows),), -1, dtype=torch.int32, device=k_cache.device)
    acc_count = torch.zeros((items.shape[0],), dtype=torch.int32, device=k_cache.device)
    _commit_out_cuda(k_cache, v_cache, lens, items, accept_len, accept_mask, slot_offset, acc_rows, acc_count)
    return acc_rows, acc_count


def _commit_drop_cuda(lens, drop_pos):
    dev = rt.require_cuda(lens, drop_pos)
    if lens.dtype != torch.int32 or lens.dim() != 2 or drop_pos.dtype != torch.int32 or \
            drop_pos.numel() != lens.shape[1]:
        raise ValueError("lens int32 (n_slots, n_seqs), drop_pos int32 (n_seqs,)")
    st = _abi.load().wfd_commit_drop(lens.data_ptr(), drop_pos.contiguous().data_ptr(), lens.shape[0], lens.shape[1],
                                     rt.stream_ptr(dev))
    _abi.check(st, "wfd_commit_drop")


def _wave_attn_q8_out_cuda(q, k_new, v_new, k_cache, v_cache, k_exp, v_exp, items, max_q, lens, slot_offset, scale,
                           kernel, row_pos, out):
    rt.require_cuda(q, k_cache, v_cache, k_exp, v_exp, lens)
    wave_attn_q8_launch(q8_cache_struct(k_cache, v_cache, k_exp, v_exp, lens), q, k_new, v_new, items, max_q,
                        slot_offset, scale, kernel, row_pos, out)


def wave_attn_q8_launch(c, q, k_new, v_new, items, max_q, slot_offset, scale, kernel, row_pos, out) -> None:
    """wfd_wave_attn_q8 over the cache struct c (on q's device), after the checks of the other arguments."""
    dev = rt.require_cuda(q, k_new, v_new, items, row_pos, out)
    Hkv, Dh = c.n_kv_heads, c.head_dim
    if q.dim() != 3 or q.shape[2] != Dh or k_new.shape != (q.shape[0], Hkv, Dh) or v_new.shape != k_new.shape:
        raise ValueError("q (n_rows, H, Dh) and k_new / v_new (n_rows, Hkv, Dh) must match the cache")
    if q.dtype != k_new.dtype or q.dtype != v_new.dtype:
        raise TypeError("q, k_new, v_new must share a dtype")
    if q.shape[1] % Hkv != 0:
        raise ValueError(f"query heads {q.shape[1]} not a multiple of kv heads {Hkv}")
    if items.dtype != torch.int32 or items.dim() != 2 or items.shape[1] != 5 or not items.is_contiguous():
        raise ValueError("items must be a contiguous int32 (n_items, 5) device tensor")
    if out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor shaped like q")
    rp_stride = 1
    if row_pos is not None:
        if row_pos.dtype != torch.int32 or row_pos.dim() != 1 or row_pos.numel() < q.shape[0] or \
                (row_pos.numel() > 1 and row_pos.stride(0) < 1):
            raise ValueError("row_pos must be an int32 device vector with one position per q row")
        rp_stride = max(1, row_pos.stride(0))
    q, k_new, v_new = rt.rows16(q), rt.rows16(k_new), rt.rows16(v_new)
    n = items.shape[0]
    # scratch of this call alone: calls on several streams, and graphs replayed side
    # by side, share nothing
    wsb = q8_workspace_bytes(dev, n)
    ws = torch.empty(wsb, dtype=torch.uint8, device=dev)
    rt.call(dev, "wfd_wave_attn_q8", int(kernel), ctypes.byref(c), q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(),
            out.data_ptr(), items.data_ptr(), n, int(max_q), rt.ptr(row_pos), rp_stride, int(slot_offset), q.shape[0],
            q.shape[1], rt.dtype_code(q.dtype), float(scale or 0.0), ws.data_ptr(), wsb,
            rt.error_word(dev).data_ptr(), rt.stream_ptr(dev))


@functools.lru_cache(maxsize=4096)
def q8_workspace_bytes(dev: torch.device, n: int) -> int:
    with torch.cuda.device(dev):
        b = int(_abi.load().wfd_wave_attn_q8_workspace(n))
    if b <= 0:
        raise _abi.WfdError("wfd_wave_attn_q8_workspace", -1, "could not size the workspace")
    return b


def _wave_attn_q8_cuda(q, k_new, v_new, k_cache, v_cache, k_exp, v_exp, items, max_q, lens=None, slot_offset=0,
                       scale=None, kernel=-1, row_pos=None):
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _wave_attn_q8_out_cuda(q, k_new, v_new, k_cache, v_cache, k_exp, v_exp, items, max_q, lens, slot_offset, scale,
                           kernel, row_pos, out)
    return out


def _commit_q8_out_cuda(k_cache, v_cache, k_exp, v_exp, lens, items, accept_len, accept_mask, slot_offset, acc_rows,
                        acc_count):
    dev = _check_commit(k_cache, v_cache, lens, items, accept_len, accept_mask)
    n = items.shape[0]
    for t in (acc_rows, acc_count):
        if t.dtype != torch.int32 or t.device != dev or not t.is_contiguous():
            raise ValueError("acc_rows / acc_count must be contiguous int32 tensors on the cache's device")
    if acc_count.numel() < n or (accept_len is not None and accept_len.numel() < n):
        raise ValueError("acc_count and accept_len need one entry per item")
    c = q8_cache_struct(k_cache, v_cache, k_exp, v_exp, lens)
    al = None if accept_len is None else accept_len.contiguous()
    am = None if accept_mask is None else accept_mask.contiguous()
    # q rows both row-indexed arrays cover: the kernel skips (and reports) windows past them
    n_rows = acc_rows.numel() if am is None else min(acc_rows.numel(), am.numel())
    rt.call(dev, "wfd_commit_window_q8", ctypes.byref(c), items.data_ptr(), n, rt.ptr(al), rt.ptr(am),
            acc_rows.data_ptr(), acc_count.data_ptr(), n_rows, int(slot_offset), rt.error_word(dev).data_ptr(),
            rt.stream_ptr(dev))


def _commit_q8_cuda(k_cache, v_cache, k_exp, v_exp, lens, items, accept_len, accept_mask, slot_offset, n_rows):
    acc_rows = torch.full((int(n_rows),), -1, dtype=torch.int32, device=k_cache.device)
    acc_count = torch.zeros((items.shape[0],), dtype=torch.int32, device=k_cache.device)
    _commit_q8_out_cuda(k_cache, v_cache, k_exp, v_exp, lens, items, accept_len, accept_mask, slot_offset, acc_rows,
                        acc_count)
    return acc_rows, acc_count


_LIB.impl("attn", _attn_cuda, "CUDA")
_LIB.impl("attn_out", _attn_out_cuda, "CUDA")
_LIB.impl("wave_attn", _wave_attn_cuda, "CUDA")
_LIB.impl("wave_attn_out", _wave_attn_out_cuda, "CUDA")
_LIB.impl("commit", _commit_cuda, "CUDA")
_LIB.impl("commit_out", _commit_out_cuda, "CUDA")
_LIB.impl("commit_drop", _commit_drop_cuda, "CUDA")
_LIB.impl("wave_attn_q8", _wave_attn_q8_cuda, "CUDA")
_LIB.impl("wave_attn_q8_out", _wave_attn_q8_out_cuda, "CUDA")
_LIB.impl("commit_q8", _commit_q8_cuda, "CUDA")
_LIB.impl("commit_q8_out", _commit_q8_out_cuda, "CUDA")


# ---------------------------------------------------------------------------
# fake (meta) kernels: shapes and dtypes only
# ---------------------------------------------------------------------------
@torch.library.register_fake("wfd::attn")
def _attn_fake(q, k, v, cu_q, cu_k, max_q, max_k, causal=False, scale=None):
    return torch.empty_like(q)


@torch.library.register_fake("wfd::attn_out")
def _attn_out_fake(q, k, v, cu_q, cu_k, max_q, max_k, causal, scale, out):
    return None


@torch.library.register_fake("wfd::wave_attn")
def _wave_attn_fake(q, k_new, v_new, k_cache, v_cache, items, max_q, lens=None, slot_offset=0, scale=None, kernel=-1,
                    row_pos=None):
    return torch.empty_like(q)


@torch.library.register_fake("wfd::wave_attn_out")
def _wave_attn_out_fake(q, k_new, v_new, k_cache, v_cache, items, max_q, lens, slot_offset, scale, kernel, row_pos,
                        out):
    return None


@torch.library.register_fake("wfd::commit")
def _commit_fake(k_cache, v_cache, lens, items, accept_len, accept_mask, slot_offset, n_rows):
    return (k_cache.new_empty((n_rows,), dtype=torch.int32), k_cache.new_empty((items.shape[0],), dtype=torch.int32))


@torch.library.register_fake("wfd::commit_out")
def _commit_out_fake(k_cache, v_cache, lens, items, accept_len, accept_mask, slot_offset, acc_rows, acc_count):
    return None


@torch.library.register_fake("wfd::commit_drop")
def _commit_drop_fake(lens, drop_pos):
    return None


@torch.library.register_fake("wfd::wave_attn_q8")
def _wave_attn_q8_fake(q, k_new, v_new, k_cache, v_cache, k_exp, v_exp, items, max_q, lens=None, slot_offset=0,
                       scale=None, kernel=-1, row_pos=None):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


@torch.library.register_fake("wfd::wave_attn_q8_out")
def _wave_attn_q8_out_fake(q, k_new, v_new, k_cache, v_cache, k_exp, v_exp, items, max_q, lens, slot_offset, scale,
                           kernel, row_pos, out):
    return None


@torch.library.register_fake("wfd::commit_q8")
def _commit_q8_fake(k_cache, v_cache, k_exp, v_exp, lens, items, accept_len, accept_mask, slot_offset, n_rows):
    return (lens.new_empty((n_rows,)), lens.new_empty((items.shape[0],)))


@torch.library.register_fake("wfd::commit_q8_out")
def _commit_q8_out_fake(k_cache, v_cache, k_exp, v_exp, lens, items, accept_len, accept_mask, slot_offset, acc_rows,
                        acc_count):
    return None
