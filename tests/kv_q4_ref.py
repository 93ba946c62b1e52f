"""The 4-bit KV cache in 64 bits, straight from its definition (test oracle):
one channel at a time, no code shared with the library."""
import numpy as np
import torch


def bf16_nearest(x: np.ndarray) -> np.ndarray:
    """float64 -> nearest bf16 value (ties to even), as float64; the smallest
    step is bf16's subnormal step 2^-133."""
    _, e = np.frexp(x)
    step = np.ldexp(1.0, np.maximum(e - 8, -133))
    return np.rint(x / step) * step


def quantise(x: torch.Tensor, group: int):
    """bf16 [..., D] -> (codes int [..., D], s, m float64 [..., D/group])."""
    g = x.double().cpu().numpy().reshape(*x.shape[:-1], -1, group)
    with np.errstate(all="ignore"):
        m, M = g.min(-1), g.max(-1)
        s = bf16_nearest((M - m) / 15.0)
        c = np.where(s[..., None] > 0, np.rint((g - m[..., None]) / s[..., None]), 0.0)
        c = np.minimum(c, 15.0)
    bad = ~np.isfinite(g).all(-1)
    s[bad] = m[bad] = np.nan
    c[bad] = 0
    return c.reshape(x.shape).astype(np.int64), s, m


def field_order(D: int):
    """(byte, shift) of every channel of a stored row."""
    byte, shift = [], []
    for d in range(D):
        j, t, e = d // 32, (d % 32) // 8, d % 8
        field = e // 2 + 4 * (e % 2)
        byte.append(4 * (t * (D // 32) + j) + field // 2)
        shift.append(4 * (field % 2))
    return np.array(byte), np.array(shift)


def pack(codes: np.ndarray) -> torch.Tensor:
    byte, shift = field_order(codes.shape[-1])
    out = np.zeros((*codes.shape[:-1], codes.shape[-1] // 2), dtype=np.uint8)
    for d in range(codes.shape[-1]):
        out[..., byte[d]] |= (codes[..., d] << shift[d]).astype(np.uint8)
    return torch.from_numpy(out)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 values of stored rows (codes uint8 [..., D/2], scales [..., D/group, 2])."""
    D = 2 * codes.shape[-1]
    byte, shift = field_order(D)
    by = codes.cpu().numpy().astype(np.int64)
    sm = scales.double().cpu().numpy()
    group = D // sm.shape[-2]
    out = np.empty((*by.shape[:-1], D))
    for d in range(D):
        c = (by[..., byte[d]] >> shift[d]) & 15
        out[..., d] = sm[..., d // group, 1] + c * sm[..., d // group, 0]
    return torch.from_numpy(out)


def attention(q, k, v, lens, scale: float, causal: bool):
    """q bf16 [B,Hq,Sq,D], k/v float64 [B,Hkv,n,D], lens: B ints.  Returns
    float64 out [B,Sq,Hq*D] and the same sum with |v| (the size that rounding
    errors of the weights and values go by)."""
    B, Hq, Sq, D = q.shape
    G = Hq // k.shape[1]
    out = torch.zeros(B, Sq, Hq, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for b in range(B):
        n = int(lens[b])
        for h in range(Hq):
            for i in range(Sq):
                end = min(n, n - Sq + i + 1) if causal else n
                if end <= 0:
                    continue
                kk, vv = k[b, h // G, :end], v[b, h // G, :end]
                p = torch.softmax(kk @ q[b, h, i].double().cpu() * scale, dim=0)
                out[b, i, h], mag[b, i, h] = p @ vv, p @ vv.abs()
    return out.reshape(B, Sq, Hq * D), mag.reshape(B, Sq, Hq * D)
