"""Measured cases of the 4-bit KV cache: storing keys and values as they are
written, reading them back, and attention over the stored rows.

The cache
---------
Keys and values of one attention layer, ``[B, Hkv, capacity, D]`` with D = 32,
64 or 128, are held as 4-bit codes with one (scale, minimum) pair of bf16 per
group of ``group`` consecutive channels (32, 64 or 128, at most D).  For a
group with minimum m and maximum M:

    s = bf16((M - m) / 15)                       (to nearest, ties to even)
    c = min(15, rint((x - m) / s))               (0 where s is 0)
    value = m + c * s

Codes lie in uint8 ``[B, Hkv, capacity, D / 2]``.  Seen as 32-bit words, word
``t * (D / 32) + j`` of a row (t = 0..3) holds channels ``32 j + 8 t`` to
``32 j + 8 t + 7``; of those eight, channel e is the 4-bit field
``e / 2 + 4 * (e % 2)`` (field 0 lowest).  Scales lie in bf16
``[B, Hkv, capacity, D / group, 2]`` as (s, m) pairs.

Every case is one of

* ``store``:  k, v bf16 ``[B, Hkv, S, D]`` into rows ``start ..`` of the cache,
  and the stored rows read back, as a prefill in chunks does;
* ``load``:   a range of rows read back as bf16;
* ``attend``: ``softmax(q k^T * D^-1/2 + mask) v`` of bf16 q ``[B, Hq, Sq, D]``
  over the first rows of the cache, with the causal mask aligned to the last
  row when Sq > 1, returned as bf16 ``[B, Sq, Hq * D]``.
"""
from __future__ import annotations

import math

import torch

own = False

_BF16 = torch.bfloat16


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a serving batch: every sequence stores one row, each
        # at its own position (latency)
        dict(name="store_step_64", kind="store", B=64, Hkv=4, D=128, group=32, S=1, cap=512,
             start=300, ragged=True),
        # the prompt of one long request
        dict(name="store_prompt_4096", kind="store", B=1, Hkv=4, D=128, group=32, S=4096, cap=8192,
             start=0, ragged=False),
        # a ragged batch of chunks behind rows that are there already, small heads
        dict(name="store_chunk_odd", kind="store", B=7, Hkv=2, D=64, group=64, S=1531, cap=2048,
             start=77, ragged=False),
        # a batch of long prompts
        dict(name="store_batch_8x8192", kind="store", B=8, Hkv=4, D=128, group=128, S=8192,
             cap=8192, start=0, ragged=False),
        # a short range of a small-headed cache
        dict(name="load_odd", kind="load", B=3, Hkv=2, D=32, group=32, S=777, cap=1024, start=5,
             ragged=False),
        # the whole history of a batch, for a caller that works on bf16 rows
        dict(name="load_16x8192", kind="load", B=16, Hkv=4, D=128, group=32, S=8192, cap=8192,
             start=0, ragged=False),
        # one token of one short conversation (latency)
        dict(name="attend_1x500", kind="attend", B=1, Hq=32, Hkv=4, D=128, group=32, Sq=1, kv=500,
             cap=512, ragged=False),
        # one decode step of 64 sequences with 8192 positions behind them
        dict(name="attend_64x8193", kind="attend", B=64, Hq=32, Hkv=4, D=128, group=32, Sq=1,
             kv=8193, cap=8448, ragged=False),
        # one token behind a very long context
        dict(name="attend_1x131072", kind="attend", B=1, Hq=32, Hkv=4, D=128, group=64, Sq=1,
             kv=131072, cap=131072, ragged=False),
        # a serving batch whose sequences have lengths from one to the capacity
        dict(name="attend_ragged_32", kind="attend", B=32, Hq=32, Hkv=4, D=128, group=128, Sq=1,
             kv=8192, cap=8192, ragged=True),
        # four drafted tokens checked at once, small heads
        dict(name="attend_draft_4", kind="attend", B=8, Hq=8, Hkv=2, D=64, group=32, Sq=4, kv=4099,
             cap=4112, ragged=False),
        # a chunk of a prompt behind the chunks before it
        dict(name="attend_chunk_512", kind="attend", B=1, Hq=32, Hkv=4, D=128, group=32, Sq=512,
             kv=8704, cap=8704, ragged=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "load", "attend", "attend"])
    D = rng.choice([32, 64, 128, 128])
    group = rng.choice([g for g in (32, 64, 128) if g <= D])
    Hkv = rng.choice([1, 2, 4, 8])
    B = _log_int(rng, 1, 64)
    ragged = rng.random() < 0.4
    if kind != "attend":
        # at most the rows and channels of store_batch_8x8192 / load_16x8192
        most = (8 if kind == "store" else 16) * 4 * 8192 * 128 // (B * Hkv * D)
        S = _log_int(rng, 1, max(1, min(8192, most)))
        start = rng.randrange(0, 300)
        cap = -(-(S + start + rng.randrange(0, 64)) // 16) * 16
        return dict(kind=kind, B=B, Hkv=Hkv, D=D, group=group, S=S, cap=cap, start=start,
                    ragged=ragged)
    G = rng.choice([1, 2, 4, 7, 8, 16])
    # at most the stored channels of attend_64x8193 and the products of
    # attend_chunk_512
    kv = _log_int(rng, 1, max(1, min(131072, 64 * 4 * 8192 * 128 // (B * Hkv * D))))
    most = 32 * 512 * 8192 * 128 // (B * Hkv * G * D * kv)
    Sq = _log_int(rng, 1, max(1, min(kv, 1024, most))) if rng.random() < 0.5 else 1
    if ragged:
        Sq = min(Sq, max(1, 64 // G))
    cap = -(-(kv + rng.randrange(0, 64)) // 16) * 16
    return dict(kind=kind, B=B, Hq=G * Hkv, Hkv=Hkv, D=D, group=group, Sq=Sq, kv=kv, cap=cap,
                ragged=ragged)


# -------------------------------------------------------------------- inputs
def _rows(shape, gen, device):
    """Rows as an attention layer makes them: unit scale, a channel profile of
    its own per head, some channels far wider than the rest."""
    D = shape[-1]
    profile = torch.exp(0.4 * torch.randn(1, shape[1], 1, D, generator=gen, device=device))
    profile[..., ::29] *= 4.0
    x = torch.randn(shape, generator=gen, device=device, dtype=torch.float32)
    return x.mul_(profile).to(_BF16)


def prepare(case, seed):
    device = "cuda"
    gen = torch.Generator(device=device).manual_seed(seed)
    B, Hkv, D, cap, group = case["B"], case["Hkv"], case["D"], case["cap"], case["group"]
    st = dict(case=dict(case))
    cache = [torch.zeros(B, Hkv, cap, n, device=device, dtype=torch.uint8) if i % 2 == 0 else
             torch.zeros(B, Hkv, cap, n, 2, device=device, dtype=_BF16)
             for i, n in enumerate((D // 2, D // group, D // 2, D // group))]
    if case["kind"] == "store":
        st["k"] = _rows((B, Hkv, case["S"], D), gen, device)
        st["v"] = _rows((B, Hkv, case["S"], D), gen, device)
    else:
        for codes, scales in ((cache[0], cache[1]), (cache[2], cache[3])):
            for b in range(B):
                c, sm = _quantise(_rows((1, Hkv, cap, D), gen, device), group)
                codes[b], scales[b] = _pack(c)[0], sm[0]
    st["cache"] = cache
    if case["kind"] == "attend":
        st["q"] = (1.5 * torch.randn(B, case["Hq"], case["Sq"], D, generator=gen,
                                     device=device)).to(_BF16)
        if case["ragged"]:
            span = torch.rand(B, generator=gen, device=device)
            low = case["Sq"]
            lens = (low * (case["kv"] / low) ** span).round().clamp(low, case["kv"])
            lens[0], lens[-1] = low, case["kv"]
            st["kv"] = lens.to(torch.int32)
        else:
            st["kv"] = case["kv"]
    elif case["ragged"]:
        st["start"] = torch.randint(0, case["cap"] - case["S"] + 1, (B,), generator=gen,
                                    device=device, dtype=torch.int32)
    else:
        st["start"] = case["start"]
    return st


# ---------------------------------------------------------------- plain form
def _bf16_once(x):
    """float64 -> bf16 in one rounding: a value that float32 has rounded onto a
    border between two bf16 numbers is put back on its own side."""
    f = x.float()
    bits = f.view(torch.int32)
    border = (bits & 0xFFFF) == 0x8000
    away = f.double()
    bits = bits + (border & (away.abs() < x.abs())).int() - (border & (away.abs() > x.abs())).int()
    return bits.view(torch.float32).to(_BF16)


def _quantise(x, group):
    """bf16 [..., D] -> codes uint8 [..., D], (s, m) bf16 [..., D/group, 2]; in
    64 bits, since a code next to a border would flip in 32."""
    xg = x.double().unflatten(-1, (-1, group))
    m = xg.amin(-1)
    s = _bf16_once((xg.amax(-1) - m) / 15.0)
    sd = s.double().unsqueeze(-1)
    c = torch.where(sd > 0, (xg - m.unsqueeze(-1)) / sd, torch.zeros_like(xg))
    c = c.round().clamp(0, 15).to(torch.uint8).flatten(-2)
    return c, torch.stack([s, m.to(_BF16)], dim=-1)


def _pack(c):
    """codes [..., D] -> bytes [..., D/2]."""
    D = c.shape[-1]
    # channel = 32 j + 8 t + 2 i + h  ->  word (t, j), field i + 4 h
    f = c.unflatten(-1, (D // 32, 4, 4, 2))                 # j t i h
    f = f.movedim(-1, -2).movedim(-4, -3)                   # t j h i
    f = f.reshape(*c.shape[:-1], D // 2, 2)                 # byte, (low, high)
    return f[..., 0] | (f[..., 1] << 4)


def _unpack(by):
    """bytes [..., D/2] -> codes [..., D]."""
    J = by.shape[-1] // 16
    f = torch.stack([by & 15, by >> 4], dim=-1).unflatten(-2, (4, J, 2, 2)).flatten(-2)
    return f.movedim(-4, -3).movedim(-1, -2).flatten(-4)    # t j h i -> j t i h


def _values(codes, scales):
    """The float32 values that stored rows stand for."""
    c = _unpack(codes).float().unflatten(-1, (scales.shape[-2], -1))
    s, m = scales[..., 0:1].float(), scales[..., 1:2].float()
    return (m + c * s).flatten(-2)


def _row_index(start, S, B, device):
    if isinstance(start, torch.Tensor):
        return start.long()[:, None] + torch.arange(S, device=device)
    return (start + torch.arange(S, device=device)).expand(B, S)


def _gather(cache, rows):
    """Rows ``rows`` [B, S] of the four cache tensors."""
    b = torch.arange(rows.shape[0], device=rows.device)[:, None]
    return [t.transpose(1, 2)[b, rows].transpose(1, 2) for t in cache]


def _run_plain(st):
    case, cache = st["case"], st["cache"]
    B = case["B"]
    if case["kind"] != "attend":
        rows = _row_index(st["start"], case["S"], B, cache[0].device)
        if case["kind"] == "store":
            b = torch.arange(B, device=rows.device)[:, None]
            for x, codes, scales in ((st["k"], cache[0], cache[1]), (st["v"], cache[2], cache[3])):
                c, sm = _quantise(x, case["group"])
                codes.transpose(1, 2)[b, rows] = _pack(c).transpose(1, 2)
                scales.transpose(1, 2)[b, rows] = sm.transpose(1, 2)
        kc, ks, vc, vs = _gather(cache, rows)
        return _values(kc, ks).to(_BF16), _values(vc, vs).to(_BF16)
    q, kv = st["q"], st["kv"]
    Hq, Sq, D = q.shape[1:]
    Hkv = case["Hkv"]
    n = case["kv"]
    kc, ks, vc, vs = [t[:, :, :n] for t in cache]
    qg = q.float().reshape(B, Hkv, (Hq // Hkv) * Sq, D) * D ** -0.5
    s = torch.matmul(qg, _values(kc, ks).transpose(-1, -2)).reshape(B, Hkv, Hq // Hkv, Sq, n)
    lens = kv.long() if isinstance(kv, torch.Tensor) else torch.full((B,), n, device=q.device)
    # query i sees the keys up to len - Sq + i
    last = lens[:, None] - Sq + torch.arange(Sq, device=q.device)
    seen = torch.arange(n, device=q.device) <= last[..., None]
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p.reshape(B, Hkv, -1, n), _values(vc, vs))
    o = o.reshape(B, Hq, Sq, D) / p.sum(-1).reshape(B, Hq, Sq, 1)
    return o.transpose(1, 2).reshape(B, Sq, Hq * D).to(_BF16)


# ----------------------------------------------------------------- operators
def _run_own(st):
    from qwen3_5_vl_cuda_custom_b200 import kernels as K
    case, cache = st["case"], st["cache"]
    if case["kind"] == "attend":
        return K.attention_cache_q4(st["q"], *cache, st["kv"], case["D"] ** -0.5, case["Sq"] > 1)
    if case["kind"] == "store":
        K.kv_append_q4(st["k"], st["v"], *cache, st["start"])
    return K.kv_read_q4(*cache, st["start"], case["S"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------- work
def work(case):
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    row = 2 * (D // 2 + 4 * (D // case["group"]))  # stored bytes of one key and one value
    if case["kind"] != "attend":
        n = B * Hkv * case["S"]
        if case["kind"] == "store":
            return {"bytes": n * (4 * D + row + 4 * D), "flops": n * 2 * D * 8}
        return {"bytes": n * (row + 4 * D), "flops": n * 2 * D * 2}
    Hq, Sq, kv = case["Hq"], case["Sq"], case["kv"]
    if case["ragged"]:
        # lengths spread evenly over their logarithm between Sq and kv
        kv = (kv - Sq) / math.log(kv / Sq) if kv > Sq else kv
    pairs = Sq * kv - Sq * (Sq - 1) / 2
    return {"bytes": B * (Hkv * kv * row + 2 * 2 * Hq * Sq * D),
            "flops": 4.0 * B * Hq * pairs * D}


# --------------------------------------------------------------------- exact
def _exact_rows(codes, scales):
    """float64 values of stored rows, one channel's byte and shift at a time."""
    D = 2 * codes.shape[-1]
    d = torch.arange(D, device=codes.device)
    j, t, e = d // 32, (d % 32) // 8, d % 8
    field = e // 2 + 4 * (e % 2)
    byte = 4 * (t * (D // 32) + j) + field // 2
    c = (codes[..., byte].to(torch.int32) >> (4 * (field % 2)).to(torch.int32)) & 15
    pair = scales.double()[..., d // (D // scales.shape[-2]), :]
    return c.double() * pair[..., 0] + pair[..., 1]


def _exact_stored(x, group):
    """float64 values that bf16 rows are stored as."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for i in range(0, x.shape[-1], group):
        g = x[..., i:i + group].to(torch.float64)
        low, high = g.min(dim=-1, keepdim=True).values, g.max(dim=-1, keepdim=True).values
        step = (high - low) / 15
        # nearest bf16: 8 significant bits (no group here is near the subnormals)
        man, exp = torch.frexp(step)
        step = torch.ldexp(torch.round(man * 256), exp - 8)
        n = torch.where(step == 0, torch.zeros_like(g), torch.round((g - low) / step))
        out[..., i:i + group] = low + step * torch.minimum(n, torch.full_like(n, 15))
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "store":
        return _exact_stored(st["k"], case["group"]), _exact_stored(st["v"], case["group"])
    kc, ks, vc, vs = st["cache"]
    if case["kind"] == "load":
        parts = []
        for b in range(case["B"]):
            i = int(st["start"][b]) if case["ragged"] else st["start"]
            w = slice(i, i + case["S"])
            parts.append((_exact_rows(kc[b, :, w], ks[b, :, w]), _exact_rows(vc[b, :, w], vs[b, :, w])))
        return torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])
    q, Hq, Hkv, Sq, D = st["q"].double(), case["Hq"], case["Hkv"], case["Sq"], case["D"]
    out = torch.empty(case["B"], Sq, Hq * D, dtype=torch.float64, device=q.device)
    for b in range(case["B"]):
        n = int(st["kv"][b]) if case["ragged"] else case["kv"]
        for h in range(Hkv):
            key, val = _exact_rows(kc[b, h, :n], ks[b, h, :n]), _exact_rows(vc[b, h, :n], vs[b, h, :n])
            for a in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                s = q[b, a] @ key.T / math.sqrt(D)
                i = torch.arange(Sq, device=q.device)[:, None] + (n - Sq)
                s = torch.where(torch.arange(n, device=q.device) <= i, s, -torch.inf)
                out[b, :, a * D:(a + 1) * D] = torch.softmax(s, dim=-1) @ val
    return out
