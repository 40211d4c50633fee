"""8-bit KV-slot cache in 64 bits, from its definition: quantised rows, the window
append, and wavefront attention over the cached values.

A row x of head_dim values is stored as e4m3 codes of x 2^-e, e the smallest
integer with max|x| <= 448 2^e, clamped to [-32, 32]; a NaN counts as 0.
"""
from __future__ import annotations

import numpy as np

E_MAX = 32


def round_e4m3(y: np.ndarray) -> np.ndarray:
    """Nearest e4m3 value (ties to even), saturating at 448."""
    a = np.abs(y)
    with np.errstate(divide="ignore"):
        ex = np.floor(np.log2(np.where((a > 0) & np.isfinite(a), a, 1.0)))
    step = 2.0 ** (np.maximum(ex, -6) - 3)
    with np.errstate(invalid="ignore"):
        r = np.where(np.isinf(y), y, np.round(np.where(np.isinf(y), 0.0, y) / step) * step)
    return np.clip(r, -448.0, 448.0)


def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """x (..., Dh) -> (code values float64 (..., Dh), exponents int (...,))."""
    x = np.where(np.isnan(x), 0.0, x.astype(np.float64))
    a = np.abs(x).max(-1)
    e = np.full(a.shape, E_MAX)
    for t in range(E_MAX - 1, -E_MAX - 1, -1):
        e = np.where(a <= 448.0 * 2.0 ** t, t, e)
    return round_e4m3(x * 2.0 ** -e[..., None].astype(np.float64)), e


class Q8CacheOracle:
    """codes K, V (n_slots, B, S, Hkv, Dh) as float64, exponents ke, ve (n_slots, B, Hkv, S)."""

    def __init__(self, n_slots: int, B: int, Hkv: int, Dh: int, S: int):
        self.K = np.zeros((n_slots, B, S, Hkv, Dh))
        self.V = np.zeros_like(self.K)
        self.ke = np.zeros((n_slots, B, Hkv, S), dtype=np.int64)
        self.ve = np.zeros_like(self.ke)
        self.lens = np.zeros((n_slots, B), dtype=np.int64)

    def put(self, slot: int, seq: int, pos: int, k: np.ndarray, v: np.ndarray) -> None:
        """One row (Hkv, Dh) of K and V at a position."""
        self.K[slot, seq, pos], self.ke[slot, seq, :, pos] = quantise(k)
        self.V[slot, seq, pos], self.ve[slot, seq, :, pos] = quantise(v)
        self.lens[slot, seq] = max(self.lens[slot, seq], pos + 1)

    def values(self, slot: int, seq: int, n: int) -> tuple[np.ndarray, np.ndarray]:
        """(n, Hkv, Dh) values of the first n positions, K and V."""
        return tuple(c[slot, seq, :n] * 2.0 ** e[slot, seq, :, :n].T[..., None].astype(np.float64)
                     for c, e in ((self.K, self.ke), (self.V, self.ve)))

    def wave_attn(self, q, k_new, v_new, items, row_pos=None, slot_offset: int = 0, scale: float | None = None):
        """Append every window row, then attend.  Returns (out, amp, smax): out (n, H, Dh) with NaN for rows no item
        names; amp the same sum with |v|, and smax (n, H) the largest sum of |q k| scale terms a row's scores hold:
        what rounding errors of weights and scores scale with."""
        n, H, Dh = q.shape
        pos = np.full(n, -1)
        for slot, seq, p0, ql, r0 in items:
            for j in range(ql):
                pos[r0 + j] = p0 + j if row_pos is None else row_pos[r0 + j]
                self.put(slot + slot_offset, seq, int(pos[r0 + j]), k_new[r0 + j], v_new[r0 + j])
        out = np.full((n, H, Dh), np.nan)
        amp, smax = out.copy(), np.zeros((n, H))
        scale = 1.0 / np.sqrt(Dh) if not scale else scale
        for slot, seq, p0, ql, r0 in items:
            if ql == 0:
                continue
            K, V = self.values(slot + slot_offset, seq, int(pos[r0:r0 + ql].max()) + 1)
            G = H // K.shape[1]
            for j in range(ql):
                N = int(pos[r0 + j]) + 1
                qj = q[r0 + j].astype(np.float64).reshape(-1, G, Dh)
                s = np.einsum("hgd,thd->hgt", qj, K[:N]) * scale
                smax[r0 + j] = (np.einsum("hgd,thd->hgt", np.abs(qj), np.abs(K[:N])) * scale).max(-1).reshape(-1)
                w = np.exp(s - s.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                out[r0 + j] = np.einsum("hgt,thd->hgd", w, V[:N]).reshape(H, Dh)
                amp[r0 + j] = np.einsum("hgt,thd->hgd", w, np.abs(V[:N])).reshape(H, Dh)
        return out, amp, smax


def decode(W: dict, cfg: dict, prompt: list[int], n_new: int, pick):
    """Sequential decoding of the looped LM (oracle.looped_lm's architecture) in float64 over an 8-bit cache: the
    prompt attends its own rows and is cached quantised; every later token attends cached values, its own row
    included.  pick(logits, position) -> id.  Returns (ids, logits, rows): the logits each id was picked from, and
    per slot the unquantised (K, V) rows of every position."""
    import torch

    from oracle import looped_lm as olm
    H, Hkv, Dh = cfg["n_heads"], cfg["n_kv_heads"], cfg["head_dim"]
    style = cfg.get("rope_style", "half")
    n_slots = len(W["prelude"]) + cfg["T_total"] * len(W["core"]) + len(W["coda"])
    held = [[] for _ in range(n_slots)]      # cached values (K, V), (T, Hkv, Dh)
    rows = [[] for _ in range(n_slots)]

    def cached(x):
        q, e = quantise(x.numpy())
        return torch.from_numpy(q * 2.0 ** e[..., None].astype(np.float64))

    def block(blk, x, slot, pos):
        T = x.shape[0]
        h = olm._rms(x, blk["norm1"], cfg["norm_eps"]) @ blk["wqkv"]
        q, k, v = torch.split(h, [H * Dh, Hkv * Dh, Hkv * Dh], dim=-1)
        q = olm._rope(q.reshape(T, H, Dh), pos, cfg["rope_theta"], style)
        k = olm._rope(k.reshape(T, Hkv, Dh), pos, cfg["rope_theta"], style)
        v = v.reshape(T, Hkv, Dh)
        rows[slot].append((k, v))
        held[slot].append((cached(k), cached(v)))
        if len(held[slot]) > 1:                                    # not the prompt
            k, v = (torch.cat([t[i] for t in held[slot]]) for i in range(2))
        k, v = (t.repeat_interleave(H // Hkv, dim=1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) / np.sqrt(Dh)
        s = s.masked_fill(torch.arange(k.shape[0])[None, :] > pos[:, None], float("-inf"))
        o = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v).reshape(T, H * Dh)
        x = x + o @ blk["wo"]
        g, u = (olm._rms(x, blk["norm2"], cfg["norm_eps"]) @ blk["wgu"]).split(cfg["d_ff"], dim=-1)
        return x + (torch.nn.functional.silu(g) * u) @ blk["wd"]

    ids, logits = list(prompt), []
    new = list(prompt)
    for _ in range(n_new):
        pos = torch.arange(len(ids) - len(new), len(ids))
        x = W["embed"][torch.tensor(new)]
        slot = 0
        for blk in W["prelude"]:
            x = block(blk, x, slot, pos)
            slot += 1
        e, h = x, torch.zeros_like(x)
        for _ in range(cfg["T_total"]):
            h = h + e
            for blk in W["core"]:
                h = block(blk, h, slot, pos)
                slot += 1
        for blk in W["coda"]:
            h = block(blk, h, slot, pos)
            slot += 1
        logits.append(olm._rms(h[-1], W["final_norm"], cfg["norm_eps"]) @ W["lm_head"])
        new = [pick(logits[-1], len(ids) - 1)]
        ids += new
    return ids[len(prompt):], logits, [tuple(torch.cat([t[i] for t in s]) for i in range(2)) for s in rows]
