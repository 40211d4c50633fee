"""Cases of the quantised-cache and sampling operators, in plain torch form and as calls of the framework.

  write   a KV slot cache quantised as it is written (e4m3 rows with a power-of-two scale), and read back
  attend  wavefront attention over the quantised slots, with the window append fused in
  sample  temperature / top-k / top-p / min-p sampling from given uniform numbers

A cached row (one position, one kv head, Dh values) holds q_i = e4m3(x_i 2^-e) and the exponent e, the smallest
integer with max|x| <= 448 2^e, clamped to [-32, 32].
"""
import math

import numpy as np
import torch

own = False

E_MAX = 32
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _attend(name, B, R, Hq, Hkv, Dh, L, q_len=1, jitter=0, gap=0, dtype="bf16", spare=64):
    """B sequences x R depth slots, one item each: window of q_len rows (ragged when odd ones are asked for by
    jitter) after L - r - (b-dependent jitter) cached positions; gap > 0: window rows gap + 1 positions apart."""
    return {"name": name, "op": "attend", "B": B, "R": R, "Hq": Hq, "Hkv": Hkv, "Dh": Dh, "L": L, "q_len": q_len,
            "jitter": jitter, "gap": gap, "dtype": dtype, "spare": spare}


def _write(name, B, R, Hkv, Dh, L, prompt, dtype="bf16"):
    """prompt: one slot's prompt rows of B sequences written and all read back; else: one row per (sequence, slot)
    scattered behind L - r positions, and the first slot's prefixes read back."""
    return {"name": name, "op": "write", "B": B, "R": R, "Hkv": Hkv, "Dh": Dh, "L": L, "prompt": prompt,
            "dtype": dtype}


def _sample(name, n, V, dtype, masked, mode):
    """n rows of V logits; masked: share of -inf logits; mode: which filters the rows ask for."""
    return {"name": name, "op": "sample", "n": n, "V": V, "dtype": dtype, "masked": masked, "mode": mode}


def listed():
    return [
        # one sequence of the small looped model (8 x 64, depth 4) shortly after its 128-token prompt
        _attend("attend_one_seq", 1, 4, 8, 8, 64, 190),
        # the isolated decode op: 8 sequences x 8 slots, GQA 16/4, one query row each
        _attend("attend_decode", 8, 8, 16, 4, 128, 4096),
        # verify windows of 8 rows, GQA 32/8
        _attend("attend_verify", 16, 8, 32, 8, 128, 8192, q_len=8),
        # the R tick of the 770M looped model: 64 sequences x 8 depths, MHA 24 x 64, ragged lengths
        _attend("attend_tick", 64, 8, 24, 24, 64, 1152, jitter=97),
        # long context, few sequences
        _attend("attend_long", 2, 16, 32, 8, 128, 32768, jitter=5),
        # KV sharing: a sequence's tokens on one slot form one window with gaps
        _attend("attend_gapped", 16, 2, 24, 24, 64, 1111, q_len=4, jitter=31, gap=1),
        # fp32 engine (exact greedy parity runs), odd lengths
        _attend("attend_f32", 8, 4, 8, 8, 64, 777, q_len=3, jitter=13, dtype="f32"),
        # a tick's rows of the 770M model into the cache, one prefix per sequence read back
        _write("write_tick", 8, 8, 24, 64, 1024, False),
        # its prompt pass, one layer: 64 prompts of 1024 tokens
        _write("write_prompt", 64, 1, 24, 64, 1024, True),
        # the C union of 64 sequences (commit and draft rows), every filter in use
        _sample("sample_union", 128, 50304, "bf16", 0.0, "mixed"),
        # one sequence of the small model, nucleus sampling
        _sample("sample_one", 1, 32000, "f32", 0.0, "top_p"),
        # a wide vocabulary with a grammar mask, temperature and min-p
        _sample("sample_masked", 32, 131071, "f32", 0.5, "mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "write", "sample", "sample"])
    if op == "attend":
        Dh = rng.choice([64, 128])
        Hkv = rng.choice([1, 2, 3, 4, 5, 8, 12, 24])
        G = rng.choice([1, 1, 2, 3, 4, 7, 8])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        q_len = rng.choice([1, 1, 2, 3, 5, 8, 11])
        gap = rng.choice([0, 0, 0, 1, 2]) if q_len > 1 else 0
        R, B = rng.randint(1, 9), _log(rng, 1, 48)
        L = _log(rng, q_len * (gap + 1) + 10, 12000)
        # no more than the largest listed case reads, or an eighth of it in fp32
        while B * R * Hkv * Dh * L > (1.0e9 if dtype == "bf16" else 0.12e9):
            if L > 600:
                L = L * 2 // 3
            elif B > 1:
                B = B // 2
            else:
                R = max(1, R // 2)
        while B * R * Hkv * G * q_len * L > 0.25e9:
            G, q_len, gap, L = max(1, G // 2), max(1, q_len // 2), gap if q_len > 3 else 0, max(64, L * 3 // 4)
        c = _attend("", B, R, Hkv * G, Hkv, Dh, L, q_len, rng.randint(0, min(40, L // 8)), gap, dtype,
                    rng.randint(1, 70))
    elif op == "write":
        c = _write("", _log(rng, 1, 48), rng.randint(1, 9), rng.choice([1, 2, 3, 5, 8, 24]), rng.choice([64, 128]),
                   _log(rng, 16, 1500), rng.choice([True, False]), rng.choice(["bf16", "bf16", "f32"]))
        while c["B"] * c["Hkv"] * c["Dh"] * c["L"] > 5e7:
            c["L"] //= 2
    else:
        V = _log(rng, 500, 131071)
        n = _log(rng, 1, 128)
        while n * V > 4194272:
            n //= 2
        c = _sample("", n, V, rng.choice(["bf16", "f32"]), rng.choice([0.0, 0.0, 0.3, 0.9]),
                    rng.choice(["mixed", "mixed", "top_p", "top_k", "plain"]))
    return {k: v for k, v in c.items() if k != "name"}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _span(c):
    return (c["q_len"] - 1) * (c["gap"] + 1) + 1


def _lengths(c):
    """Cached positions before the window, per (r, b)."""
    return [[max(0, c["L"] - r - (b * 37) % (c["jitter"] + 1)) for b in range(c["B"])] for r in range(c["R"])]


def _rows(g, shape, dtype, device):
    """Rows like a trained model's K / V: normal, with magnitudes that differ from row to row."""
    x = torch.randn(shape, generator=g, device=device)
    return (x * torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=g, device=device))).to(dtype)


def _quantise(x):
    """x (..., Dh) -> (e4m3 values, int8 exponents (...,)) in 32 bits."""
    x = x.float()
    a = torch.nan_to_num(x.abs(), nan=0.0).amax(-1)
    m, ex = torch.frexp(a)                       # a = m 2^ex, m in [0.5, 1); 448 = 0.875 2^9
    e = torch.where(m <= 0.875, ex - 9, ex - 8)
    e = torch.where(a == 0, torch.full_like(e, -E_MAX), torch.where(torch.isinf(a), torch.full_like(e, E_MAX), e))
    e = e.clamp(-E_MAX, E_MAX)
    q = (x * torch.exp2(-e.float()).unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return q, e.to(torch.int8)


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    if c["op"] == "sample":
        n, V = c["n"], c["V"]
        x = torch.randn((n, V), generator=g, device=dev)
        x *= 1.0 + 2.0 * torch.rand((n, 1), generator=g, device=dev)    # peaked and flat rows
        if c["masked"]:
            x = x.masked_fill(torch.rand((n, V), generator=g, device=dev) < c["masked"], float("-inf"))
        rnd = torch.rand((4, n), generator=g, device=dev)
        use = {"mixed": (1, 1, 1), "top_p": (0, 1, 0), "top_k": (1, 0, 0), "plain": (0, 0, 0)}[c["mode"]]
        one = torch.ones(n, device=dev)
        temp = 0.5 + rnd[0]
        if c["mode"] == "mixed":
            temp[n // 2::7] = 0.0                                       # some requests are greedy
        k = (1 + (200 * rnd[1]).to(torch.int32)) * (rnd[1] < 0.7) if use[0] else torch.zeros(n, device=dev)
        p = torch.where(rnd[2] < 0.7, 0.6 + 0.39 * rnd[2], one) if use[1] else one
        m = torch.where(rnd[3] < 0.5, 0.1 * rnd[3], 0 * one) if use[2] else 0 * one
        return {"case": c, "x": x.to(DTYPES[c["dtype"]]), "u": torch.rand(n, generator=g, device=dev),
                "temperature": temp, "top_k": k.to(torch.int32), "top_p": p, "min_p": m}
    dt = DTYPES[c["dtype"]]
    B, R, Hkv, Dh = c["B"], c["R"], c["Hkv"], c["Dh"]
    if c["op"] == "write":
        S = c["L"] + 8
    else:
        S = c["L"] + _span(c) + c["spare"]
    K = torch.empty((R, B, S, Hkv, Dh), dtype=torch.float8_e4m3fn, device=dev)
    V = torch.empty_like(K)
    k_exp = torch.empty((R, B, Hkv, S), dtype=torch.int8, device=dev)
    v_exp = torch.empty_like(k_exp)
    for r in range(R):
        for q8, ex in ((K, k_exp), (V, v_exp)):
            q, e = _quantise(_rows(g, (B, S, Hkv, Dh), torch.float32, dev))
            q8[r] = q
            ex[r] = e.transpose(1, 2)
    s = {"case": c, "K": K, "V": V, "k_exp": k_exp, "v_exp": v_exp}
    if c["op"] == "write":
        if c["prompt"]:
            s["lens"] = torch.zeros((R, B), dtype=torch.int32, device=dev)
            s["k"], s["v"] = (_rows(g, (B, c["L"], Hkv, Dh), dt, dev) for _ in range(2))
            upto = [c["L"]] * B
        else:
            s["lens"] = torch.tensor([[c["L"] - r for _ in range(B)] for r in range(R)], dtype=torch.int32, device=dev)
            s["k"], s["v"] = (_rows(g, (R * B, Hkv, Dh), dt, dev) for _ in range(2))
            at = [(r, b, c["L"] - r) for r in range(R) for b in range(B)]
            s["slots"], s["seqs"], s["pos"] = (torch.tensor(t, dtype=torch.int32, device=dev) for t in zip(*at))
            upto = [c["L"] + 1] * B
        cu = [0]
        for u in upto:
            cu.append(cu[-1] + u)
        s["r_slots"] = torch.zeros(B, dtype=torch.int32, device=dev)
        s["r_seqs"] = torch.arange(B, dtype=torch.int32, device=dev)
        s["cu_k"] = torch.tensor(cu, dtype=torch.int32, device=dev)
        s["total"] = cu[-1]
        return s
    n0 = _lengths(c)
    items, pos, row = [], [], 0
    for r in range(R):
        for b in range(B):
            items.append((r, b, n0[r][b], c["q_len"], row))
            pos += [n0[r][b] + j * (c["gap"] + 1) for j in range(c["q_len"])]
            row += c["q_len"]
    s["items"] = torch.tensor(items, dtype=torch.int32, device=dev)
    s["row_pos"] = torch.tensor(pos, dtype=torch.int32, device=dev)
    s["lens"] = torch.tensor(n0, dtype=torch.int32, device=dev)
    s["q"] = torch.randn((row, c["Hq"], Dh), generator=g, device=dev).to(dt)
    s["k"], s["v"] = (_rows(g, (row, Hkv, Dh), dt, dev) for _ in range(2))
    s["n_max"] = max(map(max, n0)) + _span(c)     # no row sees a key at or behind this position
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _store(s, slots, seqs, pos, k, v):
    """Quantise rows k, v (n, Hkv, Dh) into the cache at (slots, seqs, pos)."""
    for x, q8, ex in ((k, s["K"], s["k_exp"]), (v, s["V"], s["v_exp"])):
        q, e = _quantise(x)
        q8.view(torch.uint8)[slots, seqs, pos] = q.view(torch.uint8)
        ex[slots, seqs, :, pos] = e
    n_seqs = s["lens"].shape[1]
    s["lens"].view(-1).scatter_reduce_(0, slots * n_seqs + seqs, (pos + 1).to(torch.int32), "amax")


def _plain_write(s):
    c = s["case"]
    dev = s["K"].device
    if c["prompt"]:
        b = torch.arange(c["B"], device=dev).repeat_interleave(c["L"])
        t = torch.arange(c["L"], device=dev).repeat(c["B"])
        _store(s, torch.zeros_like(b), b, t, s["k"].flatten(0, 1), s["v"].flatten(0, 1))
    else:
        _store(s, s["slots"].long(), s["seqs"].long(), s["pos"].long(), s["k"], s["v"])
    cu = s["cu_k"].long()
    seg = torch.repeat_interleave(torch.arange(c["B"], device=dev), cu.diff(), output_size=s["total"])
    t = torch.arange(s["total"], device=dev) - cu[seg]
    sl, sq = s["r_slots"].long()[seg], s["r_seqs"].long()[seg]
    packs = []
    for q8, ex in ((s["K"], s["k_exp"]), (s["V"], s["v_exp"])):
        q = q8.view(torch.uint8)[sl, sq, t].view(torch.float8_e4m3fn).float()
        packs.append((q * torch.exp2(ex[sl, sq, :, t].float()).unsqueeze(-1)).to(DTYPES[c["dtype"]]))
    return packs


def _plain_attend(s):
    c = s["case"]
    q_len, Hq, Hkv, Dh, N = c["q_len"], c["Hq"], c["Hkv"], c["Dh"], s["n_max"]
    n = s["items"].shape[0]
    slots, seqs = s["items"][:, 0].long(), s["items"][:, 1].long()
    pos = s["row_pos"].long()
    _store(s, slots.repeat_interleave(q_len), seqs.repeat_interleave(q_len), pos, s["k"], s["v"])
    lead = (n, N, Hkv, Dh)
    k = s["K"][:, :, :N].reshape(lead).float()    # the items are every (slot, sequence), in order
    k *= torch.exp2(s["k_exp"][:, :, :, :N].reshape(n, Hkv, N).float()).transpose(1, 2).unsqueeze(-1)
    q = s["q"].float().view(n, q_len, Hkv, Hq // Hkv, Dh).permute(0, 2, 1, 3, 4).reshape(n, Hkv, -1, Dh)
    sc = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(Dh))
    del k
    hidden = torch.arange(N, device=pos.device) > pos.view(n, 1, q_len, 1)
    sc = sc.view(n, Hkv, q_len, -1).view(n, Hkv, q_len, Hq // Hkv, N).masked_fill(hidden.unsqueeze(3), float("-inf"))
    w = torch.exp(sc - sc.amax(-1, keepdim=True))
    del sc
    w /= w.sum(-1, keepdim=True)
    v = s["V"][:, :, :N].reshape(lead).float()
    v *= torch.exp2(s["v_exp"][:, :, :, :N].reshape(n, Hkv, N).float()).transpose(1, 2).unsqueeze(-1)
    o = torch.matmul(w.view(n, Hkv, -1, N), v.permute(0, 2, 1, 3))
    return o.view(n, Hkv, q_len, Hq // Hkv, Dh).permute(0, 2, 1, 3, 4).reshape(n * q_len, Hq, Dh).to(s["q"].dtype)


def _plain_sample(s):
    """In 64 bits: a sum of 1e5 weights in 32 would put u on the wrong side of a token's border."""
    x = s["x"].double()
    V = x.shape[1]
    top = x.amax(1, keepdim=True)
    T = s["temperature"].double().unsqueeze(1)
    greedy = T <= 0
    w = torch.exp((x - top) / torch.where(greedy, torch.ones_like(T), T))
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    k = s["top_k"].long().unsqueeze(1)
    rank = torch.arange(V, device=x.device).unsqueeze(0)
    ws = ws * (rank < torch.where(k <= 0, torch.full_like(k, V), k))
    cum = ws.cumsum(1)
    p = s["top_p"].double().unsqueeze(1)
    ws = ws * (((cum - ws) < p * cum[:, -1:]) | (p >= 1))
    ws = ws * (ws >= s["min_p"].double().unsqueeze(1))
    cum = torch.zeros_like(w).scatter_(1, order, ws).cumsum(1)
    ids = (cum <= s["u"].double().unsqueeze(1) * cum[:, -1:]).sum(1)
    return torch.where(greedy.squeeze(1), order[:, 0], ids).to(torch.int32)


def run(state):
    s = state
    op = s["case"]["op"]
    if op == "sample":
        if own:
            _, fused, _ = _framework()
            return fused.sample_rows(s["x"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                     min_p=s["min_p"])
        return _plain_sample(s)
    if own:
        attention, _, kv_cache = _framework()
        if op == "attend":
            out = attention.wave_attn_q8(s["q"], s["k"], s["v"], s["K"], s["V"], s["k_exp"], s["v_exp"], s["items"],
                                         s["case"]["q_len"], lens=s["lens"],
                                         row_pos=s["row_pos"] if s["case"]["gap"] else None)
        else:
            cache = kv_cache.QuantKVCache.wrap(s["K"], s["V"], s["k_exp"], s["v_exp"], s["lens"],
                                               dtype=s["k"].dtype)
            if s["case"]["prompt"]:
                cache.write_prefill(0, s["k"], s["v"])
            else:
                cache.write_tokens(s["slots"], s["seqs"], s["pos"], s["k"], s["v"])
            out = cache.gather_packed(s["r_slots"], s["r_seqs"], s["cu_k"], s["total"])
    else:
        out = _plain_attend(s) if op == "attend" else _plain_write(s)
    return {"out": out, "K": s["K"], "V": s["V"], "k_exp": s["k_exp"], "v_exp": s["v_exp"], "lens": s["lens"]}


def _framework():
    import __graft_entry__
    __graft_entry__.load_package()
    from wavefront_decoding_b200 import attention, fused, kv_cache
    return attention, fused, kv_cache


# ---------------------------------------------------------------------------
# work and exact values
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "sample":
        size = 2 if c["dtype"] == "bf16" else 4
        return {"bytes": c["n"] * (c["V"] * size + 24), "flops": 4 * c["n"] * c["V"]}
    elem = 2 if c["dtype"] == "bf16" else 4
    row = c["Hkv"] * c["Dh"]
    if c["op"] == "write":
        n_new = c["B"] * c["L"] if c["prompt"] else c["B"] * c["R"]
        n_read = c["B"] * (c["L"] if c["prompt"] else c["L"] + 1)
        # rows in, their 8-bit form out; the read-back reads what was not just written, and writes the packs
        old = 0 if c["prompt"] else n_read - c["B"]
        return {"bytes": 2 * (n_new * (row * (elem + 1) + c["Hkv"]) + old * (row + c["Hkv"]) + n_read * row * elem),
                "flops": 4 * row * (n_new + n_read)}
    rows = c["B"] * c["R"] * c["q_len"]
    keys = sum(x + _span(c) for y in _lengths(c) for x in y)
    seen = sum(x + j * (c["gap"] + 1) + 1 for y in _lengths(c) for x in y for j in range(c["q_len"]))
    return {"bytes": keys * 2 * (row + c["Hkv"]) + rows * (2 * c["Hq"] * c["Dh"] * elem + 2 * row * (elem + 1)),
            "flops": 4 * seen * c["Hq"] * c["Dh"]}


def _round_e4m3(y):
    """float64 -> nearest e4m3 value, ties to even, saturating."""
    a = y.abs()
    step = torch.exp2(torch.floor(torch.log2(torch.where(a > 0, a, torch.ones_like(a)))).clamp(min=-6.0) - 3.0)
    return (torch.round(y / step) * step).clamp(-448.0, 448.0)


def _exact_rows(x):
    """(e4m3 values, exponents) of rows x, from the definition: the smallest e with max|x| <= 448 2^e."""
    x = x.double()
    a = x.abs().amax(-1)
    e = torch.full_like(a, float(E_MAX))
    for t in range(E_MAX - 1, -E_MAX - 1, -1):
        e = torch.where(a <= 448.0 * 2.0 ** t, torch.full_like(e, float(t)), e)
    return _round_e4m3(x / torch.exp2(e).unsqueeze(-1)), e


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "sample":
        return _exact_ids(s)
    lens = s["lens"].clone()
    put = []
    if c["op"] == "write" and c["prompt"]:
        put = [(0, b, slice(0, c["L"]), s["k"][b], s["v"][b]) for b in range(c["B"])]
    elif c["op"] == "write":
        put = [(i // c["B"], i % c["B"], slice(c["L"] - i // c["B"], c["L"] - i // c["B"] + 1), s["k"][i:i + 1],
                s["v"][i:i + 1]) for i in range(c["R"] * c["B"])]
    else:
        step = c["gap"] + 1
        for slot, seq, p0, ql, row in s["items"].tolist():
            put.append((slot, seq, slice(p0, p0 + _span(c), step), s["k"][row:row + ql], s["v"][row:row + ql]))
    for slot, seq, at, k, v in put:
        for x, q8, ex in ((k, s["K"], s["k_exp"]), (v, s["V"], s["v_exp"])):
            q, e = _exact_rows(x)
            q8[slot, seq, at] = q.float().to(torch.float8_e4m3fn)
            ex[slot, seq, :, at] = e.to(torch.int8).T
        last = at.start + (at.stop - at.start - 1) // (at.step or 1) * (at.step or 1)
        lens[slot, seq] = max(int(lens[slot, seq]), last + 1)

    def value(q8, ex, slot, seq, n):
        return q8[slot, seq, :n].double() * torch.exp2(ex[slot, seq, :, :n].double()).T.unsqueeze(-1)

    if c["op"] == "write":
        n = s["cu_k"].diff().tolist()
        out = [torch.cat([value(q8, ex, 0, b, n[b]) for b in range(c["B"])])
               for q8, ex in ((s["K"], s["k_exp"]), (s["V"], s["v_exp"]))]
    else:
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        G = c["Hq"] // c["Hkv"]
        for slot, seq, p0, ql, row in s["items"].tolist():
            k = value(s["K"], s["k_exp"], slot, seq, p0 + _span(c))
            v = value(s["V"], s["v_exp"], slot, seq, p0 + _span(c))
            q = s["q"][row:row + ql].double().reshape(ql, c["Hkv"], G, -1)
            sc = torch.einsum("jhgd,thd->hjgt", q, k) / math.sqrt(c["Dh"])
            t = torch.arange(k.shape[0], device=k.device)
            see = t[None, :] <= (p0 + torch.arange(ql, device=k.device) * (c["gap"] + 1))[:, None]
            sc = torch.where(see[None, :, None, :], sc, torch.full_like(sc, -math.inf))
            out[row:row + ql] = torch.einsum("hjgt,thd->jhgd", torch.softmax(sc, -1), v).reshape(ql, c["Hq"], -1)
    return {"out": out, "K": s["K"], "V": s["V"], "k_exp": s["k_exp"], "v_exp": s["v_exp"], "lens": lens}


def _exact_ids(s):
    x = s["x"].float().cpu().numpy().astype(np.float64)
    T, K, P, M, U = (s[k].cpu().numpy() for k in ("temperature", "top_k", "top_p", "min_p", "u"))
    ids = np.zeros(len(x), dtype=np.int32)
    for r, row in enumerate(x):
        first = int(np.argmax(row))
        if T[r] <= 0:
            ids[r] = first
            continue
        w = np.exp((row - row[first]) / np.float64(T[r]))
        order = np.lexsort((np.arange(len(row)), -row))
        if 0 < K[r] < len(row):
            order = order[:K[r]]
        if P[r] < 1:
            before = np.concatenate([[0.0], np.cumsum(w[order])])
            order = order[before[:-1] < np.float64(P[r]) * before[-1]]
        order = np.sort(order[w[order] >= M[r]])
        c = np.cumsum(w[order])
        ids[r] = order[min(int(np.searchsorted(c, np.float64(U[r]) * c[-1], side="right")), len(order) - 1)]
    return torch.from_numpy(ids)
