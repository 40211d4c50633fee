"""KV slot cache for the wavefront hot path.

Same storage contract as the reference's `BatchStaticKVCache`
(src/decoding/batch_kv_cache.py:28-105):

    K, V : (n_slots, B, max_seq_len, Hkv, Dh)     buffer index == absolute position

with the logical lengths kept ON THE DEVICE (`lens`, int32 (n_slots, B)) instead
of a host list, so appends, rollbacks and commits can run inside CUDA graphs.
`seqlen` gives the reference's host view (it synchronises).  Every mutation is
a libwfd_b200 kernel: append (write_tokens), prefill write, rollback
(drop_positions_at_and_after) and the window accept/compact commit.

`QuantKVCache` holds the same slots in 8 bits per element.
"""
from __future__ import annotations

import ctypes

import torch

from . import _abi
from . import attention as _attn
from . import ops as _ops
from . import runtime as rt


class SlotKVCache:
    def __init__(self, n_slots: int, batch_size: int, n_kv_head: int, head_dim: int, max_seq_len: int,
                 dtype: torch.dtype, device: torch.device):
        self.n_slots = n_slots
        self.B = batch_size
        self.S = max_seq_len
        self.n_kv_head = n_kv_head
        self.head_dim = head_dim
        self.dtype = dtype
        self.device = torch.device(device)
        rt.dtype_code(dtype)
        shape = (n_slots, batch_size, max_seq_len, n_kv_head, head_dim)
        self.K = torch.zeros(shape, dtype=dtype, device=self.device)
        self.V = torch.zeros(shape, dtype=dtype, device=self.device)
        self.lens = torch.zeros((n_slots, batch_size), dtype=torch.int32, device=self.device)

    @classmethod
    def wrap(cls, K: torch.Tensor, V: torch.Tensor, lens: torch.Tensor | None = None) -> "SlotKVCache":
        """Adopt existing (n_slots, B, S, Hkv, Dh) K / V tensors (e.g. a reference
        BatchStaticKVCache's .K / .V) without copying."""
        if K.dim() != 5 or V.shape != K.shape or not (K.is_contiguous() and V.is_contiguous()):
            raise ValueError("K, V must be contiguous (n_slots, B, max_seq_len, Hkv, Dh) tensors")
        rt.dtype_code(K.dtype)
        self = cls.__new__(cls)
        self.n_slots, self.B, self.S, self.n_kv_head, self.head_dim = K.shape
        self.dtype, self.device, self.K, self.V = K.dtype, K.device, K, V
        if lens is None:
            lens = torch.zeros((self.n_slots, self.B), dtype=torch.int32, device=K.device)
        if lens.dtype != torch.int32 or tuple(lens.shape) != (self.n_slots, self.B):
            raise ValueError("lens must be int32 (n_slots, B)")
        self.lens = lens
        return self

    # ------------------------------------------------------------------
    @property
    def nbytes(self) -> int:
        return (self.K.numel() + self.V.numel()) * self.K.element_size()

    @property
    def seqlen(self) -> list[list[int]]:
        """Host copy of the logical lengths, shaped like the reference's
        `seqlen[slot][b]` (batch_kv_cache.py:44).  Synchronises."""
        return self.lens.cpu().tolist()

    def _geom(self):
        return (self.n_slots, self.B, self.S, self.n_kv_head, self.head_dim, rt.dtype_code(self.dtype))

    def _stream(self) -> int:
        return rt.stream_ptr(self.device)

    # ------------------------------------------------------------------
    def write_prefill(self, slot: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """k, v: (B, L, Hkv, Dh) prompt K/V at positions [0, L) (batch_kv_cache.py:51-59)."""
        L = k.shape[1]
        assert L <= self.S
        if k.shape != (self.B, L, self.n_kv_head, self.head_dim) or v.shape != k.shape:
            raise ValueError("write_prefill expects k, v of shape (B, L, Hkv, Dh)")
        k, v = k.contiguous(), v.contiguous()
        st = _abi.load().wfd_write_prefill(k.data_ptr(), v.data_ptr(), self.K.data_ptr(), self.V.data_ptr(),
                                           self.lens.data_ptr(), int(slot), L, *self._geom(), self._stream())
        _abi.check(st, "wfd_write_prefill")

    def write_tokens(self, slots, seq_ids, positions, k: torch.Tensor, v: torch.Tensor, *, slot_offset: int = 0) -> None:
        """Scatter n rows k, v (n, Hkv, Dh) to (slots[i], seq_ids[i], positions[i])
        (batch_kv_cache.py:61-73).  Host lists are bounds-checked here with the
        reference's IndexError; device index tensors are checked in the kernel."""
        n = k.shape[0]
        if isinstance(positions, list):
            for p in positions:
                if p >= self.S:
                    raise IndexError(f"position {p} exceeds max_seq_len={self.S}")
        sl = _ops.i32(slots, self.device)
        sq = _ops.i32(seq_ids, self.device)
        ps = _ops.i32(positions, self.device)
        k, v = k.contiguous(), v.contiguous()
        st = _abi.load().wfd_append(k.data_ptr(), v.data_ptr(), self.K.data_ptr(), self.V.data_ptr(),
                                    self.lens.data_ptr(), sl.data_ptr(), sq.data_ptr(), ps.data_ptr(), n,
                                    int(slot_offset), *self._geom(), rt.error_word(self.device).data_ptr(),
                                    self._stream())
        _abi.check(st, "wfd_append")

    def gather_pack(self, slots, seq_ids, uptos):
        """Pack n prefixes [(slot, b, 0..upto)] -> (k_pack, v_pack, cu_k, max_k)
        (batch_kv_cache.py:75-96).  API parity only: the wavefront op reads the
        slots in place and never packs."""
        lengths = [u + 1 for u in uptos]
        cu_host = [0]
        for ln in lengths:
            cu_host.append(cu_host[-1] + ln)
        total = cu_host[-1]
        k_pack = torch.empty((total, self.n_kv_head, self.head_dim), dtype=self.dtype, device=self.device)
        v_pack = torch.empty_like(k_pack)
        cu_k = torch.tensor(cu_host, dtype=torch.int32, device=self.device)
        sl = _ops.i32(slots, self.device)
        sq = _ops.i32(seq_ids, self.device)
        st = _abi.load().wfd_gather_pack(self.K.data_ptr(), self.V.data_ptr(), k_pack.data_ptr(), v_pack.data_ptr(),
                                         sl.data_ptr(), sq.data_ptr(), cu_k.data_ptr(), len(lengths), *self._geom(),
                                         rt.error_word(self.device).data_ptr(), self._stream())
        _abi.check(st, "wfd_gather_pack")
        return k_pack, v_pack, cu_k, max(lengths)

    # ------------------------------------------------------------------
    def drop_positions_at_and_after(self, b: int, position: int) -> None:
        """Per-sequence rollback (batch_kv_cache.py:99-105): every slot of sequence
        b keeps min(len, position) entries; buffers are untouched."""
        drop = torch.full((self.B,), -1, dtype=torch.int32)
        drop[b] = position
        self.drop_many(drop.to(self.device))

    def drop_many(self, drop_pos: torch.Tensor) -> None:
        """Batched rollback: drop_pos (B,) int32 device tensor, -1 = keep
        (torch.ops.wfd.commit_drop)."""
        torch.ops.wfd.commit_drop(self.lens, _ops.i32(drop_pos, self.device))

    def commit_window(self, items: torch.Tensor, *, accept_len: torch.Tensor | None = None,
                      accept_mask: torch.Tensor | None = None, slot_offset: int = 0, n_rows: int | None = None,
                      out: tuple[torch.Tensor, torch.Tensor] | None = None):
        """Accept commit of verify windows.  Returns (acc_rows, acc_count):
        acc_rows[q_row0 + k] = q row of the k-th accepted row of an item (rows
        past the count are left untouched: -1 when allocated here),
        acc_count[i] = accepted rows of item i.  Accepted K/V rows are compacted
        in place to pos0, pos0+1, ...  `out` supplies preallocated (acc_rows,
        acc_count) int32 tensors (nothing is allocated then, e.g. under graph
        capture)."""
        if (accept_len is None) == (accept_mask is None):
            raise ValueError("give exactly one of accept_len / accept_mask")
        items = _ops.i32(items, self.device).reshape(-1, 5)
        n = items.shape[0]
        al = None if accept_len is None else _ops.i32(accept_len, self.device)
        am = None
        if accept_mask is not None:
            am = torch.as_tensor(accept_mask).to(device=self.device, dtype=torch.uint8).contiguous()
        if out is not None:
            acc_rows, acc_count = out
            torch.ops.wfd.commit_out(self.K, self.V, self.lens, items, al, am, int(slot_offset), acc_rows, acc_count)
            return (acc_rows if n_rows is None else acc_rows[:n_rows]), acc_count[:n]
        if n_rows is None:
            n_rows = int((items[:, 4] + items[:, 3]).max().item()) if n else 0
        return torch.ops.wfd.commit(self.K, self.V, self.lens, items, al, am, int(slot_offset), int(n_rows))

    # ------------------------------------------------------------------
    def wave_attn(self, q, k_new, v_new, items, max_q: int, *, slot_offset: int = 0, out=None, kernel: int = -1,
                  update_lens: bool = True, row_pos=None):
        """Fused append + wavefront attention over this cache's slots."""
        return _attn.wave_attn(q, k_new, v_new, self.K, self.V, items, max_q,
                               lens=self.lens if update_lens else None, slot_offset=slot_offset, out=out,
                               kernel=kernel, row_pos=row_pos)


class QuantKVCache(SlotKVCache):
    """A slot cache of 8-bit rows, quantised as they are written.

    K, V: float8_e4m3fn codes in SlotKVCache's layout; k_exp, v_exp: int8 exponents
    (n_slots, B, Hkv, max_seq_len), one per row of head_dim values.  A cached value
    is code * 2^exp, exp the smallest integer with max|row| <= 448 * 2^exp (clamped
    to [-32, 32]): the scale is a power of two, so the rounding to e4m3 (4
    significant bits) is the only one.  Per element 1 + 1/Dh bytes instead of 2 or 4.

    `dtype` is the type of the rows written and read back (bf16 or fp32); head_dim a
    power of two from 16 to 256 (64 or 128 for wave_attn).  A NaN is stored as 0 and
    reported through the device error word; an infinity saturates.  Rows given to
    the methods may have any strides.  Same methods as SlotKVCache, whose lengths
    and rollbacks it shares."""

    def __init__(self, n_slots: int, batch_size: int, n_kv_head: int, head_dim: int, max_seq_len: int,
                 dtype: torch.dtype, device: torch.device):
        dev = torch.device(device)
        shape = (n_slots, batch_size, max_seq_len, n_kv_head, head_dim)
        eshape = (n_slots, batch_size, n_kv_head, max_seq_len)
        self._adopt(torch.zeros(shape, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn),
                    torch.zeros(shape, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn),
                    torch.zeros(eshape, dtype=torch.int8, device=dev),
                    torch.zeros(eshape, dtype=torch.int8, device=dev), None, dtype)

    @classmethod
    def wrap(cls, K: torch.Tensor, V: torch.Tensor, k_exp: torch.Tensor, v_exp: torch.Tensor,
             lens: torch.Tensor | None = None, *, dtype: torch.dtype = torch.bfloat16) -> "QuantKVCache":
        """Adopt existing code and exponent tensors without copying (one device; every code finite, every exponent
        from -32 to 32)."""
        self = cls.__new__(cls)
        self._adopt(K, V, k_exp, v_exp, lens, dtype)
        return self

    def _adopt(self, K, V, k_exp, v_exp, lens, dtype) -> None:
        rt.dtype_code(dtype)
        if lens is None:
            lens = torch.zeros(K.shape[:2], dtype=torch.int32, device=K.device)
        _ops.check_q8_cache(K, V, k_exp, v_exp, lens)
        Dh = K.shape[4]
        if Dh < 16 or Dh > 256 or Dh & (Dh - 1):
            raise ValueError(f"head_dim {Dh}: an 8-bit cache takes powers of two from 16 to 256")
        self.n_slots, self.B, self.S, self.n_kv_head, self.head_dim = K.shape
        self.dtype, self.device = dtype, K.device
        self.K, self.V, self.k_exp, self.v_exp, self.lens = K, V, k_exp, v_exp, lens

    @property
    def nbytes(self) -> int:
        return self.K.numel() + self.V.numel() + self.k_exp.numel() + self.v_exp.numel()

    def __getstate__(self):   # (pickle restores no float8 storage: codes travel as bytes)
        return dict(self.__dict__, K=self.K.view(torch.uint8), V=self.V.view(torch.uint8))

    def __setstate__(self, state):
        self.__dict__.update(state, K=state["K"].view(torch.float8_e4m3fn), V=state["V"].view(torch.float8_e4m3fn))

    def _struct(self):
        """The C view of the attributes as they are at this call: any of them may have been replaced."""
        shape = (self.n_slots, self.B, self.S, self.n_kv_head, self.head_dim)
        if self.K.shape != shape or self.K.device != self.device:
            raise ValueError(f"K is {tuple(self.K.shape)} on {self.K.device}, the cache was made with {shape} on "
                             f"{self.device}")
        return _ops.q8_cache_struct(self.K, self.V, self.k_exp, self.v_exp, self.lens)

    def _call(self, name: str, *args) -> None:
        rt.require_cuda(self.K)
        rt.call(self.device, name, ctypes.byref(self._struct()), *args, rt.error_word(self.device).data_ptr(),
                self._stream())

    def _rows(self, k, v, lead: tuple):
        shape = (*lead, self.n_kv_head, self.head_dim)
        if k.shape != shape or v.shape != shape:
            raise ValueError(f"k, v must be {shape}, got {tuple(k.shape)} and {tuple(v.shape)}")
        if k.dtype != v.dtype:
            raise TypeError("k, v must share a dtype")
        if rt.require_cuda(k, v) != self.device:
            raise ValueError(f"rows on {k.device}, cache on {self.device}")
        return rt.rows16(k), rt.rows16(v), rt.dtype_code(k.dtype)

    def write_prefill(self, slot: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """k, v: (B, L, Hkv, Dh) prompt K/V, quantised to positions [0, L)."""
        L = k.shape[1]
        assert L <= self.S
        k, v, dt = self._rows(k, v, (self.B, L))
        self._call("wfd_write_prefill_q8", k.data_ptr(), v.data_ptr(), int(slot), L, dt)

    def write_tokens(self, slots, seq_ids, positions, k: torch.Tensor, v: torch.Tensor, *, slot_offset: int = 0) -> None:
        """Quantise n rows k, v (n, Hkv, Dh) to (slots[i], seq_ids[i], positions[i]);
        where two rows name one place the later one is stored.  Bounds as
        SlotKVCache.write_tokens."""
        n = k.shape[0]
        if isinstance(positions, list):
            for p in positions:
                if p >= self.S:
                    raise IndexError(f"position {p} exceeds max_seq_len={self.S}")
        sl, sq, ps = (_ops.i32(t, self.device) for t in (slots, seq_ids, positions))
        if not sl.numel() == sq.numel() == ps.numel() == n:
            raise ValueError(f"{n} rows need {n} slots, seq_ids and positions")
        k, v, dt = self._rows(k, v, (n,))
        step, row = _abi.WFD_Q8_MAX_APPEND, self.n_kv_head * self.head_dim * k.element_size()
        pk, pv, *idx = (t.data_ptr() for t in (k, v, sl, sq, ps))
        for i in range(0, n, step):
            self._call("wfd_append_q8", pk + i * row, pv + i * row, *(p + 4 * i for p in idx), min(step, n - i),
                       int(slot_offset), dt)

    def gather_packed(self, slots: torch.Tensor, seq_ids: torch.Tensor, cu_k: torch.Tensor, total: int, *, out=None):
        """Read back: segment i holds the values of positions [0, cu_k[i+1] -
        cu_k[i]) of (slots[i], seq_ids[i]) at rows cu_k[i].. of the (total, Hkv, Dh)
        packs returned.  Device int32 tensors, whose contents may change between
        CUDA-graph replays; segments that do not fit are skipped and reported.
        `out`: (k_pack, v_pack) to write into."""
        sl, sq, cu = (_ops.i32(t, self.device) for t in (slots, seq_ids, cu_k))
        n = sl.numel()
        if sq.numel() != n or cu.numel() != n + 1:
            raise ValueError("gather_packed: n slots and seq_ids need n + 1 entries of cu_k")
        shape = (int(total), self.n_kv_head, self.head_dim)
        if out is None:
            out = tuple(torch.empty(shape, dtype=self.dtype, device=self.device) for _ in range(2))
        k_pack, v_pack = out
        for t in out:
            if tuple(t.shape) != shape or t.dtype != self.dtype or t.device != self.device or not t.is_contiguous():
                raise ValueError(f"gather_packed: packs must be contiguous {self.dtype} {shape} on {self.device}")
        self._call("wfd_gather_q8", k_pack.data_ptr(), v_pack.data_ptr(), sl.data_ptr(), sq.data_ptr(), cu.data_ptr(),
                   n, int(total), rt.dtype_code(self.dtype))
        return k_pack, v_pack

    def gather_pack(self, slots, seq_ids, uptos):
        """SlotKVCache.gather_pack with the values dequantised to `dtype`."""
        lengths = [u + 1 for u in uptos]
        cu = [0]
        for ln in lengths:
            cu.append(cu[-1] + ln)
        cu_k = torch.tensor(cu, dtype=torch.int32, device=self.device)
        k_pack, v_pack = self.gather_packed(slots, seq_ids, cu_k, cu[-1])
        return k_pack, v_pack, cu_k, max(lengths)

    def commit_window(self, items: torch.Tensor, *, accept_len: torch.Tensor | None = None,
                      accept_mask: torch.Tensor | None = None, slot_offset: int = 0, n_rows: int | None = None,
                      out: tuple[torch.Tensor, torch.Tensor] | None = None):
        """SlotKVCache.commit_window: accepted rows move as they are, codes and exponents (torch.ops.wfd.commit_q8)."""
        rt.require_cuda(self.K)
        if (accept_len is None) == (accept_mask is None):
            raise ValueError("give exactly one of accept_len / accept_mask")
        items = _ops.i32(items, self.device).reshape(-1, 5)
        n = items.shape[0]
        al = None if accept_len is None else _ops.i32(accept_len, self.device)
        am = None
        if accept_mask is not None:
            am = torch.as_tensor(accept_mask).to(device=self.device, dtype=torch.uint8).contiguous()
        cache = (self.K, self.V, self.k_exp, self.v_exp, self.lens)
        if out is not None:
            acc_rows, acc_count = out
            torch.ops.wfd.commit_q8_out(*cache, items, al, am, int(slot_offset), acc_rows, acc_count)
            return (acc_rows if n_rows is None else acc_rows[:n_rows]), acc_count[:n]
        if n_rows is None:
            n_rows = int((items[:, 4] + items[:, 3]).max().item()) if n else 0
        return torch.ops.wfd.commit_q8(*cache, items, al, am, int(slot_offset), int(n_rows))

    def wave_attn(self, q, k_new, v_new, items, max_q: int, *, slot_offset: int = 0, out=None, kernel: int = -1,
                  update_lens: bool = True, row_pos=None):
        """Fused quantising append + wavefront attention over this cache's slots (attention.wave_attn_q8)."""
        return _attn.wave_attn_q8(q, k_new, v_new, self.K, self.V, self.k_exp, self.v_exp, items, max_q,
                                  lens=self.lens if update_lens else None, slot_offset=slot_offset, out=out,
                                  kernel=kernel, row_pos=row_pos)
