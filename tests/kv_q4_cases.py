"""Attention cases over a 4-bit cache in which one rounding shows by itself: two kinds
of keys whose contributions cancel, all of them with the same weight and the same value,
so that an error of the weights or the values is the same for every key and does not
average out.  Scores, and all else that is not looked at, are exact."""
import math

import numpy as np
import torch

import kv_q4_ref as R

HEADS = 2


def _cache(D, group, kinds, key_values, value_pairs):
    """cap rows; row i is of kind kinds[i]: every key channel key_values[kind], every value
    channel 15 codes of scale s above m, value_pairs[kind] = (m, s)."""
    n = len(kinds)
    cap = -(-n // 16) * 16
    kinds = np.concatenate([kinds, np.zeros(cap - n, dtype=kinds.dtype)])
    codes = [torch.zeros(1, HEADS, cap, D // 2, dtype=torch.uint8),
             torch.full((1, HEADS, cap, D // 2), 0xFF, dtype=torch.uint8)]
    pairs = [torch.zeros(1, HEADS, cap, D // group, 2, dtype=torch.float64) for _ in range(2)]
    for i in range(len(key_values)):
        rows = torch.from_numpy(kinds == i)
        pairs[0][:, :, rows] = torch.tensor([0.0, key_values[i]], dtype=torch.float64)
        pairs[1][:, :, rows] = torch.tensor([value_pairs[i][1], value_pairs[i][0]], dtype=torch.float64)
    stored = [p.bfloat16() for p in pairs]
    assert all(torch.equal(s.double(), p) for s, p in zip(stored, pairs))
    return codes[0], stored[0], codes[1], stored[1]


def bf16(x):
    return float(R.bf16_nearest(np.array(float(x))))


def weights_case(D, group, n, step):
    """Every second key weighs w = (1 + (2 step + 1) / 256) / 2 of the others, halfway
    between two bf16 numbers; its values are -bf16(1 / w), the others' 1.  Returns
    (q, cache, scale)."""
    w = (1 + (2 * step + 1) / 256) / 2
    cache = _cache(D, group, np.arange(n) % 2, (0.0, -1.0), ((1.0, 0.0), (-bf16(1 / w), 0.0)))
    return torch.full((1, 2 * HEADS, 1, D), 1.0 / D).bfloat16(), cache, -math.log(w)  # q . k = 0, -1


def values_case(D, group, n, twos):
    """Equal weights; half of the values are 1 + 3 * 2^-10 (11 bits, exact in fp16; bf16's
    next is 1) times 2^twos, half -2^twos.  Returns (q, cache, scale)."""
    cache = _cache(D, group, np.arange(n) % 2, (0.0, 0.0),
                   ((2.0 ** twos * 253 / 256, 2.0 ** (twos - 10)), (-(2.0 ** twos), 0.0)))
    return torch.ones(1, 2 * HEADS, 1, D).bfloat16(), cache, 0.25


def bounds(case, n, weights):
    """(reference, tolerance) in 64 bits.  With A = sum p |v|: the weights (or the values;
    the other is exact) rounded to 11 bits, 2^-11 A; the exponential of the kernels on
    fp16 copies 7.5e-5 < 2^-13, of one kind of key against the other, 2^-12 A (equal
    weights have equal errors); fp32 sums 2^-18 A; the output's rounding 2^-8."""
    q, cache, scale = case
    k, v = R.values(cache[0], cache[1]), R.values(cache[2], cache[3])
    ref, A = R.attention(q, k, v, [n], scale, False)
    return ref, A * (2 ** -11 + 2 ** -18 + (2 ** -12 if weights else 0)) + 2 ** -8 * ref.abs()


def with_bf16(case, n, weights):
    """The same attention with the weights (largest 1), or the values, rounded to bf16."""
    q, cache, scale = case
    k, v = R.values(cache[0], cache[1])[0, :, :n].numpy(), R.values(cache[2], cache[3])[0, :, :n].numpy()
    s = np.einsum("hd,hkd->hk", q[0, ::2, 0].double().numpy(), k) * scale
    p = np.exp(s - s.max(1, keepdims=True))
    total = p.sum(1, keepdims=True)
    p, v = (R.bf16_nearest(p), v) if weights else (p, R.bf16_nearest(v))
    out = np.einsum("hk,hkd->hd", p, v) / total
    return torch.from_numpy(np.repeat(out, 2, 0)).reshape(1, 1, -1)
