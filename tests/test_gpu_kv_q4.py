"""The 4-bit KV cache on the GPU against its definition in 64 bits: storing
rows, reading them back, attention over them, and the layer, model and captured
step that use them."""
import math

import numpy as np
import pytest
import torch

import kv_q4_ref as R

pytestmark = pytest.mark.gpu

DEV = "cuda"
SHAPES = [(32, 32), (64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


@pytest.fixture(scope="module", autouse=True)
def _ready():
    from qwen3_5_vl_cuda_custom_b200 import build
    build.build()
    yield
    from qwen3_5_vl_cuda_custom_b200 import kernels as K
    K.device_error_check()


def K():
    from qwen3_5_vl_cuda_custom_b200 import kernels
    return kernels


def rows(shape, seed, scale=1.0):
    """bf16 rows with a channel profile and a few wide channels, as keys have."""
    g = torch.Generator().manual_seed(seed)
    p = torch.exp(0.4 * torch.randn(1, shape[1], 1, shape[-1], generator=g))
    p[..., ::29] *= 4
    return (torch.randn(shape, generator=g) * p * scale).bfloat16()


def empty_cache(B, Hkv, cap, D, group, fill=0):
    mk = lambda *s, dt: torch.full(s, fill, dtype=torch.uint8, device=DEV).view(dt)
    return (mk(B, Hkv, cap, D // 2, dt=torch.uint8), mk(B, Hkv, cap, D // group, 4, dt=torch.bfloat16),
            mk(B, Hkv, cap, D // 2, dt=torch.uint8), mk(B, Hkv, cap, D // group, 4, dt=torch.bfloat16))


def filled_cache(B, Hkv, cap, D, group, seed, scale=1.0):
    """A cache with every row stored, and its float64 k, v values."""
    out, vals = [], []
    for i in range(2):
        c, s, m = R.quantise(rows((B, Hkv, cap, D), seed + i, scale), group)
        codes = R.pack(c)
        sm = torch.from_numpy(np.stack([s, m], -1)).bfloat16()
        out += [codes.to(DEV), sm.to(DEV)]
        vals.append(R.values(codes, sm))
    return tuple(out), vals[0], vals[1]


def check_stored(codes, scales, x, group):
    """Stored rows are exactly the 64-bit definition of x."""
    c, s, m = R.quantise(x, group)
    assert torch.equal(codes.cpu(), R.pack(c))
    want = torch.from_numpy(np.stack([s, m], -1))
    assert torch.equal(torch.nan_to_num(scales.double().cpu(), nan=-77.0),
                       torch.nan_to_num(want, nan=-77.0))


# ------------------------------------------------------------------ storing
@pytest.mark.parametrize("D,group", SHAPES)
@pytest.mark.parametrize("B,Hkv,S,cap,offset", [(1, 1, 1, 16, 0), (2, 3, 37, 64, 11), (5, 2, 1, 48, 47)])
def test_append_is_the_definition(D, group, B, Hkv, S, cap, offset):
    k, v = rows((B, Hkv, S, D), 1), rows((B, Hkv, S, D), 2, 3e-3)
    cache = empty_cache(B, Hkv, cap, D, group, fill=0x5A)
    before = [t.clone() for t in cache]
    K().kv_append_q4(k.to(DEV), v.to(DEV), *cache, offset)
    w = slice(offset, offset + S)
    check_stored(cache[0][:, :, w], cache[1][:, :, w], k, group)
    check_stored(cache[2][:, :, w], cache[3][:, :, w], v, group)
    for t, old in zip(cache, before):  # other rows are left as they were
        t, old = t.view(torch.uint8), old.view(torch.uint8)
        assert torch.equal(t[:, :, :offset], old[:, :, :offset])
        assert torch.equal(t[:, :, offset + S:], old[:, :, offset + S:])


@pytest.mark.parametrize("name", ["ties", "borders", "wide", "tiny", "subnormal", "huge", "constant",
                                  "signed_zero", "steps", "nonfinite"])
def test_append_where_rounding_is_delicate(name):
    """Groups whose codes or scales lie on (or a hair beside) a border, groups at
    both ends of bf16's range, and groups that hold a NaN or an infinity."""
    g = torch.Generator().manual_seed(3)
    B, Hkv, S, D, group = 2, 2, 64, 128, 32
    x = torch.randn(B, Hkv, S, D, generator=g)
    if name == "ties":  # s a power of two, every half step present
        x = torch.randint(0, 31, x.shape, generator=g) * 0.5
        x[..., 0::32], x[..., 1::32] = 0, 15
    elif name == "borders":  # the same beside a minimum that is almost 0
        x = torch.randint(0, 31, x.shape, generator=g) * 0.5
        x[..., 0::32], x[..., 1::32] = -1e-5, 15
    elif name == "wide":  # (x - m) needs more than 24 bits
        x = x.sign() * torch.exp(12 * torch.randn(x.shape, generator=g))
    elif name == "tiny":
        x = x * 1e-33
    elif name == "subnormal":
        x = x * 3e-39
    elif name == "huge":
        x = x.clamp(-3, 3) * 1e38
    elif name == "constant":
        x = x[..., :1].expand(B, Hkv, S, D)
    elif name == "signed_zero":
        x = torch.where(x > 0, 0.0, -0.0)
    elif name == "steps":  # differences of few bits: quotients near many borders
        x = torch.randint(-127, 128, x.shape, generator=g).float()
    elif name == "nonfinite":
        x[0, 0, :, 5], x[0, 1, ::2, 40], x[1, 0, 3, 127] = math.nan, math.inf, -math.inf
    x = x.bfloat16().contiguous()
    cache = empty_cache(B, Hkv, S, D, group)
    K().kv_append_q4(x.to(DEV), x.flip(2).to(DEV), *cache, 0)
    check_stored(cache[0], cache[1], x, group)
    check_stored(cache[2], cache[3], x.flip(2), group)


@pytest.mark.parametrize("exponent", [-60, 0, 60])
def test_append_halves_next_to_values_too_small_to_subtract(exponent):
    """Quotients that are a half but for a value (the channel's or the minimum) whose
    difference from the other needs more than fp32's 24 bits, and halves of every
    scale of few bits."""
    group, rows_ = 32, []
    for k in range(4, 45):
        for sign in (-1.0, 1.0):
            small = sign * 2.0 ** -k
            row = torch.arange(32) * 0.5 - 1.5             # s = 1, every half
            row[2], row[3], row[4], row[31] = small, -small, 1.5 * small, 13.5
            rows_.append(row)
            row = torch.arange(32) * 0.5                   # minimum next to 0
            row[0], row[31] = (small, 15.0) if sign < 0 else (1e-3 * small, 15.0)
            rows_.append(row)
    for n in range(1, 128):                                # s = n / 8, halves and their neighbours
        c = torch.arange(32).double() / 2
        x = ((c - 3) * n / 8).float().bfloat16().float()
        x[0], x[31] = -3 * n / 8, 12 * n / 8
        rows_.append(x)
    x = (torch.stack(rows_) * 2.0 ** exponent).bfloat16()
    x = x[:x.shape[0] // 4 * 4].view(1, 1, -1, 128).contiguous()
    S = x.shape[2]
    cache = empty_cache(1, 1, S + -S % 16, 128, group)
    K().kv_append_q4(x.to(DEV), (-x).to(DEV), *cache, 0)
    check_stored(cache[0][:, :, :S], cache[1][:, :, :S], x, group)
    check_stored(cache[2][:, :, :S], cache[3][:, :, :S], -x, group)


@pytest.mark.parametrize("D,group", SHAPES)
def test_append_of_many_random_groups(D, group):
    """Every scale, minimum and code of many groups, values of few bits
    (many quotients on a half) and of many."""
    g = torch.Generator(device=DEV).manual_seed(11)
    S = 1 << 14
    x = torch.randn(1, 2, S, D, generator=g, device=DEV)
    x[:, 1] = (x[:, 1] * torch.exp2(torch.rand(S, 1, generator=g, device=DEV) * 6)).round() * 0.25
    x = x.bfloat16()
    cache = empty_cache(1, 2, S, D, group)
    K().kv_append_q4(x, x.flip(3), *cache, 0)
    check_stored(cache[0], cache[1], x.cpu(), group)
    check_stored(cache[2], cache[3], x.flip(3).cpu(), group)


def test_append_takes_strided_rows_and_per_sequence_offsets():
    B, Hkv, S, D, cap = 3, 4, 5, 64, 64
    k = rows((B, S, Hkv, D), 5).to(DEV).transpose(1, 2)  # token-major, no copy
    v = rows((B, Hkv, S + 2, 2 * D), 6).to(DEV)[:, :, 1:S + 1, D:]
    odd = torch.empty(B * Hkv * S * D + 1, dtype=torch.bfloat16, device=DEV)[1:].view(B, Hkv, S, D)
    odd.copy_(v)  # 2-byte aligned only
    cache, other = empty_cache(B, Hkv, cap, D, 32), empty_cache(B, Hkv, cap, D, 32)
    off = torch.tensor([0, 59, 17], dtype=torch.int32, device=DEV)
    K().kv_append_q4(k, v, *cache, off)
    K().kv_append_q4(k.contiguous(), odd, *other, off)
    for b, o in enumerate(off.tolist()):
        check_stored(cache[0][b, :, o:o + S], cache[1][b, :, o:o + S], k[b].cpu(), 32)
        check_stored(cache[2][b, :, o:o + S], cache[3][b, :, o:o + S], v[b].cpu(), 32)
    for a, b in zip(cache, other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_append_takes_any_stride_of_an_axis_of_one_element():
    base = rows((1, 1, 1, 1200), 7).to(DEV).view(-1)
    for shape, strides in (((1, 4, 1, 128), (515, 128, 3, 1)), ((2, 1, 1, 128), (512, 5, 7, 1)),
                           ((1, 1, 4, 128), (1, 9, 136, 1))):
        k = base.as_strided(shape, strides)
        B, Hkv, S, D = shape
        cache = empty_cache(B, Hkv, 16, D, 32)
        K().kv_append_q4(k, k, *cache, 2)
        for i in (0, 2):
            check_stored(cache[i][:, :, 2:2 + S], cache[i + 1][:, :, 2:2 + S], k.cpu(), 32)


def test_rows_outside_the_cache_are_left_out_and_reported():
    B, Hkv, S, D, cap = 3, 2, 4, 64, 16
    k = rows((B, Hkv, S, D), 7).to(DEV)
    cache = empty_cache(B, Hkv, cap, D, 64)
    K().kv_append_q4(k, k, *cache, torch.tensor([-2, 14, 3], dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="code 2 at site 105"):
        K().device_error_check()
    for b, lo, hi, skip in ((0, 0, 2, 2), (1, 14, 16, 0), (2, 3, 7, 0)):
        check_stored(cache[0][b, :, lo:hi], cache[1][b, :, lo:hi], k[b, :, skip:skip + hi - lo].cpu(), 64)
        rest = torch.ones(cap, dtype=torch.bool)
        rest[lo:hi] = False
        assert not cache[0][b][:, rest].any() and not cache[3][b][:, rest].any()
    kr, _ = K().kv_read_q4(*cache, torch.tensor([-1, 14, 3], dtype=torch.int32, device=DEV), 4)
    with pytest.raises(RuntimeError, match="code 2 at site 106"):
        K().device_error_check()
    assert not kr[0, :, 0].any() and not kr[1, :, 2:].any() and kr[2].any()
    q = rows((B, 4, 1, D), 8).to(DEV)
    got = K().attention_cache_q4(q, *cache, torch.tensor([17, -1, 16], dtype=torch.int32, device=DEV),
                                 0.125, False)
    with pytest.raises(RuntimeError, match="code 2 at site 311"):
        K().device_error_check()
    want = K().attention_cache_q4(q, *cache, torch.tensor([16, 0, 16], dtype=torch.int32, device=DEV),
                                  0.125, False)
    assert torch.equal(got, want) and not got[1].any()


# ------------------------------------------------------------------ reading back
@pytest.mark.parametrize("D,group", SHAPES)
def test_read_rounds_each_value_once(D, group):
    B, Hkv, cap = 2, 3, 80
    cache, kv, vv = filled_cache(B, Hkv, cap, D, group, 11)
    for start, n in ((0, cap), (13, 1), (79, 1), (5, 66), (40, 0)):
        k, v = K().kv_read_q4(*cache, start, n)
        for got, want in ((k, kv), (v, vv)):
            assert got.shape == (B, Hkv, n, D)
            # code * scale is exact in fp32, so one fp32 and one bf16 rounding
            assert torch.equal(got.cpu(), want[:, :, start:start + n].float().bfloat16())
    starts = torch.tensor([60, 3], dtype=torch.int32, device=DEV)
    k, v = K().kv_read_q4(*cache, starts, 20)
    for b, s in enumerate((60, 3)):
        assert torch.equal(k[b].cpu(), kv[b, :, s:s + 20].float().bfloat16())
        assert torch.equal(v[b].cpu(), vv[b, :, s:s + 20].float().bfloat16())


# ------------------------------------------------------------------ attention
def check_attention(out, q, kv, vv, lens, scale, causal, group, chunk=False):
    """|error| of one output value, with A = sum p |v| and ref in 64 bits:
      * weights and values each rounded to bf16 (half a step, 2^-8):  2 * 2^-8 * A
      * scores off by at most d each: weights off by a factor e^(2d), so (e^(2d) - 1) * A.
        On the codes d is fp32 accumulation over T = scale sum_d |q_d| (128 s + |m|)
        (codes of up to 128 s): 2^-19 T.  A chunk also rounds the keys, 2^-8 scale
        sum_d |q_d k_d|, and its kernel's exp2 is off by up to 7.5e-5 < 2^-13.
      * the output's own rounding: 2^-8 |ref|."""
    ref, A = R.attention(q, kv, vv, lens, scale, causal)
    qa = q.double().cpu().abs().amax(dim=(0, 1, 2))
    # per key at most: values lie in [m, m + 15 s], so s <= 2/15 max|k| and |m| <= max|k|
    ka = kv.abs().amax(dim=(0, 1, 2)) if kv.numel() else torch.zeros_like(qa)
    groups = ka.view(-1, group).amax(-1).repeat_interleave(group)
    scale = abs(scale)
    d = 2.0 ** -19 * scale * float((qa * groups).sum()) * (128 * 2 / 15 + 1)
    if chunk:
        d += 2.0 ** -8 * scale * float((qa * ka).sum()) + 2.0 ** -13
    tol = A * (2 ** -7 + math.expm1(2 * d)) + 2 ** -8 * ref.abs() + 1e-30
    err = (out.double().cpu() - ref).abs()
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), f"worst {(err / tol).max():.3f} of the bound"
    return float((err / tol).max())


@pytest.mark.parametrize("D,group", SHAPES)
@pytest.mark.parametrize("Hq,Hkv,Sq,kv,causal", [
    (8, 1, 1, 1, False), (4, 4, 1, 31, False), (14, 2, 1, 33, False), (8, 2, 1, 129, True),
    (32, 2, 1, 700, False),                        # 16 rows per kv head
    (8, 2, 4, 77, True), (8, 2, 4, 3, True),       # queries that see nothing
    (6, 2, 5, 64, False), (4, 1, 24, 200, True),   # 96 rows per kv head
])
def test_attention_on_the_codes(D, group, Hq, Hkv, Sq, kv, causal):
    B, cap = 2, -(-kv // 16) * 16 + 16
    cache, kk, vv = filled_cache(B, Hkv, cap, D, group, 21)
    q = rows((B, Hq, Sq, D), 23)
    out = K().attention_cache_q4(q.to(DEV), *cache, kv, D ** -0.5, causal)
    assert out.shape == (B, Sq, Hq * D)
    check_attention(out, q, kk, vv, [kv] * B, D ** -0.5, causal, group)


@pytest.mark.parametrize("D,group", SHAPES)
@pytest.mark.parametrize("B,Hq,Hkv,Sq,kv,causal", [
    (70, 8, 8, 1, 20, False), (60, 8, 8, 3, 33, True), (130, 4, 4, 2, 1, True),
    (30, 8, 4, 10, 70, True),                      # several groups of rows per kv head
])
def test_attention_of_many_short_caches(D, group, B, Hq, Hkv, Sq, kv, causal):
    """More groups than the GPU holds at a time, of a tile or a few: with one length and
    with a length per sequence (0 among them)."""
    cap = -(-kv // 16) * 16
    cache, kk, vv = filled_cache(B, Hkv, cap, D, group, 87, 0.5)
    q = rows((B, Hq, Sq, D), 88, 0.5)
    out = K().attention_cache_q4(q.to(DEV), *cache, kv, D ** -0.5, causal)
    check_attention(out, q, kk, vv, [kv] * B, D ** -0.5, causal, group)
    lens = [(7 * b) % (kv + 1) for b in range(B)]
    got = K().attention_cache_q4(q.to(DEV), *cache, torch.tensor(lens, dtype=torch.int32, device=DEV),
                                 D ** -0.5, causal, kv)
    check_attention(got, q, kk, vv, lens, D ** -0.5, causal, group)


@pytest.mark.parametrize("D,group", SHAPES)
@pytest.mark.parametrize("Hq,Hkv,Sq,kv,causal", [(1, 1, 1, 7, False), (8, 1, 1, 300, False),
                                                 (14, 2, 3, 1000, True), (4, 4, 1, 4000, False)])
def test_attention_on_the_codes_keeps_11_bits(D, group, Hq, Hkv, Sq, kv, causal):
    """With A = sum p |v|: weights and values each rounded by 2^-11, values at most by
    2^-15 of the largest scale; scores off by d (check_attention), exp2 by 2^-21; the
    output rounded to bf16."""
    B = 2
    cache, kk, vv = filled_cache(B, Hkv, -(-kv // 16) * 16, D, group, 83, 0.5)
    q = rows((B, Hq, Sq, D), 84, 0.5)
    out = K().attention_cache_q4(q.to(DEV), *cache, kv, D ** -0.5, causal).double().cpu()
    ref, A = R.attention(q, kk, vv, [kv] * B, D ** -0.5, causal)
    qa, ka = q.double().abs().amax(dim=(0, 1, 2)), kk.abs().amax(dim=(0, 1, 2))
    groups = ka.view(-1, group).amax(-1).repeat_interleave(group)
    d = 2.0 ** -19 * D ** -0.5 * float((qa * groups).sum()) * (128 * 2 / 15 + 1)
    tol = (A * (2 ** -10 + math.expm1(2 * d + 2.0 ** -20)) + 2 ** -8 * ref.abs()
           + 2 ** -15 * float(cache[3][..., 0].max()))
    assert ((out - ref).abs() <= tol).all(), float(((out - ref).abs() / tol).max())


@pytest.mark.parametrize("D,group", SHAPES)
def test_far_larger_values_cost_the_others_nothing(D, group):
    """Rows a query does not see, whatever finite values they hold, change nothing; a
    visible row of huge values and no weight adds what it weighs and nothing else."""
    B, Hq, Hkv, kv, Sq = 1, 4, 2, 150, 4
    cache, kk, vv = filled_cache(B, Hkv, 160, D, group, 85)
    q = rows((B, Hq, Sq, D), 86, 0.3)
    want = K().attention_cache_q4(q.to(DEV), *cache, kv, 0.125, True)
    other = [t.clone() for t in cache]
    for s, m in ((0.0, 3e38), (2e37, -3e38), (4e37, -3e38), (1e-38, 1e-38)):
        other[1][:, :, kv - 3:kv, :, 0], other[1][:, :, kv - 3:kv, :, 1] = s, m
        other[3][:, :, kv - 3:kv, :, 0], other[3][:, :, kv - 3:kv, :, 1] = s, m
        got = K().attention_cache_q4(q.to(DEV), *other, kv, 0.125, True)
        assert torch.equal(got[:, :1], want[:, :1])
    q[:, :, :, 0] = 40.0  # row 9: a score of -40 * 64 * 0.125 below the rest, values of 1e5
    cache[1][:, :, 9], cache[0][:, :, 9] = 0, 0
    cache[1][:, :, 9, 0, 1] = -64
    cache[3][:, :, 9, :, 0], cache[3][:, :, 9, :, 1] = 1e4, -1e5
    kk, vv = R.values(cache[0], cache[1]), R.values(cache[2], cache[3])
    out = K().attention_cache_q4(q.to(DEV), *cache, kv, 0.125, True)
    check_attention(out, q, kk, vv, [kv], 0.125, True, group)


@pytest.mark.parametrize("D,group", [(128, 32), (64, 64)])
def test_attention_long_and_split(D, group):
    B, Hq, Hkv, kv = 1, 8, 2, 9001
    cache, kk, vv = filled_cache(B, Hkv, 9008, D, group, 31)
    q = rows((B, Hq, 2, D), 33)
    check_attention(K().attention_cache_q4(q.to(DEV), *cache, kv, D ** -0.5, True), q, kk, vv, [kv],
                    D ** -0.5, True, group)


@pytest.mark.parametrize("Hq,Hkv,D,group,Sq", [(8, 2, 128, 32, 1), (8, 1, 64, 32, 3), (20, 4, 32, 32, 2)])
def test_attention_with_a_length_per_sequence(Hq, Hkv, D, group, Sq):
    lens = [0, 1, 2, 31, 32, 33, 500, 512]
    B, cap = len(lens), 512
    cache, kk, vv = filled_cache(B, Hkv, cap, D, group, 41)
    q = rows((B, Hq, Sq, D), 43)
    t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = K().attention_cache_q4(q.to(DEV), *cache, t, D ** -0.5, True)
    check_attention(out, q, kk, vv, lens, D ** -0.5, True, group)
    assert not out[0].any()
    # the bound on the lengths only changes how the work is split
    lens2 = [min(n, 100) for n in lens]
    out = K().attention_cache_q4(q.to(DEV), *cache, t.clamp(max=100), D ** -0.5, True, max_kv_len=100)
    check_attention(out, q, kk, vv, lens2, D ** -0.5, True, group)


@pytest.mark.parametrize("Hq,Hkv,D,group,Sq,kv,causal", [
    (32, 4, 128, 32, 100, 333, True), (32, 4, 128, 128, 64, 64, True), (8, 2, 64, 64, 130, 400, True),
    (6, 2, 32, 32, 128, 100, True),                # the first 28 queries see nothing
    (32, 4, 128, 64, 40, 129, False),
])
def test_attention_of_a_chunk(Hq, Hkv, D, group, Sq, kv, causal):
    B = 2
    cache, kk, vv = filled_cache(B, Hkv, -(-kv // 16) * 16, D, group, 51, 0.5)
    q = rows((B, Hq, Sq, D), 53, 0.5)
    out = K().attention_cache_q4(q.to(DEV), *cache, kv, D ** -0.5, causal)
    check_attention(out, q, kk, vv, [kv] * B, D ** -0.5, causal, group, chunk=True)


@pytest.mark.parametrize("D,group,B,Hq,Hkv,Sq,kv,causal", [
    (128, 32, 1, 32, 4, 33, 1000, True),           # splits of the key tiles, joined
    (128, 128, 2, 6, 2, 130, 257, True),           # one head per CTA, two query blocks
    (128, 64, 1, 16, 1, 20, 5000, False),
    (64, 32, 2, 8, 2, 70, 700, True), (64, 64, 1, 8, 8, 128, 128, True),
    (32, 32, 3, 4, 2, 129, 90, True),              # queries that see nothing
    (32, 32, 1, 7, 7, 5, 1, False), (128, 32, 2, 4, 4, 1, 131, True),
])
@pytest.mark.parametrize("q_scale,k_scale,v_scale", [(1.0, 1.0, 1.0), (1e-9, 1e9, 1e30), (3e4, 2e-5, 1e-30)])
def test_attention_of_a_chunk_at_any_size_of_values(monkeypatch, D, group, B, Hq, Hkv, Sq, kv, causal,
                                                    q_scale, k_scale, v_scale):
    """The fp16 operands are scaled: values far outside fp16's range, and far apart.
    Bounds: weights and values rounded to fp16 (2^-11 each); scores off by d from the
    keys' rounding 2^-11 scale sum |q_d k_d| (bf16 queries are exact in fp16) and the
    exponential's 2^-13; the output's rounding 2^-8."""
    monkeypatch.setattr(K(), "_q4_chunk", lambda *a: True)
    cache, kk, vv = filled_cache(B, Hkv, -(-kv // 16) * 16, D, group, 55, 0.5)
    codes = list(cache)
    codes[1], codes[3] = (cache[1].double() * k_scale).bfloat16(), (cache[3].double() * v_scale).bfloat16()
    kk = R.values(codes[0], codes[1])
    vv = R.values(codes[2], codes[3])
    q = (rows((B, Hq, Sq, D), 57, 0.5).double() * q_scale).bfloat16()
    scale = D ** -0.5 / (q_scale * k_scale)
    out = K().attention_cache_q4(q.to(DEV), *codes, kv, scale, causal).double().cpu()
    ref, A = R.attention(q, kk, vv, [kv] * B, scale, causal)
    d = 2.0 ** -11 * scale * float((q.double().abs().amax((0, 1, 2)) * kk.abs().amax((0, 1, 2))).sum())
    tol = A * (2 ** -10 + math.expm1(2 * (d + 2.0 ** -13))) + 2 ** -8 * ref.abs() + 1e-38
    assert ((out - ref).abs() <= tol).all(), float(((out - ref).abs() / tol).max())


def test_which_form_a_call_takes():
    """A decode step, drafted tokens and a short chunk on the codes, long chunks by
    the tensor-memory kernels (measured times in attention_q4_chunk.cu)."""
    for B, Hq, Hkv, Sq, kv, D, chunk in ((1, 32, 4, 512, 8704, 128, True), (1, 32, 4, 16, 8192, 128, False),
                                         (64, 32, 4, 4, 8192, 128, False), (1, 8, 2, 512, 32768, 64, True),
                                         (64, 32, 4, 1, 8192, 128, False), (1, 32, 1, 1, 8192, 128, False)):
        assert K()._q4_chunk(B, Hq, Hkv, Sq, kv, D) is chunk


@pytest.mark.parametrize("q_scale,k_scale,v_scale", [(1e9, 1e-9, 1e15), (1e-12, 1e12, 1e-15), (1e3, 1e3, 1.0)])
def test_attention_on_the_codes_at_far_sizes_of_values(q_scale, k_scale, v_scale):
    B, Hq, Hkv, Sq, kv, D, group = 2, 8, 2, 2, 300, 128, 32
    cache, _, _ = filled_cache(B, Hkv, 304, D, group, 75, 0.5)
    cache = [cache[0], (cache[1].double() * k_scale).bfloat16(), cache[2], (cache[3].double() * v_scale).bfloat16()]
    kk, vv = R.values(cache[0], cache[1]), R.values(cache[2], cache[3])
    q = (rows((B, Hq, Sq, D), 77, 0.5).double() * q_scale).bfloat16()
    scale = D ** -0.5 / (q_scale * k_scale)
    out = K().attention_cache_q4(q.to(DEV), *cache, kv, scale, True)
    check_attention(out, q, kk, vv, [kv] * B, scale, True, group)


@pytest.mark.parametrize("scale", [0.0, -0.1])
@pytest.mark.parametrize("chunk", [False, True])
def test_scales_that_are_not_positive(monkeypatch, scale, chunk):
    monkeypatch.setattr(K(), "_q4_chunk", lambda *a: chunk)
    B, Hq, Hkv, Sq, kv, D = 1, 8, 2, 3, 200, 64
    cache, kk, vv = filled_cache(B, Hkv, 208, D, 64, 78)
    q = rows((B, Hq, Sq, D), 79)
    check_attention(K().attention_cache_q4(q.to(DEV), *cache, kv, scale, True), q, kk, vv, [kv], scale,
                    True, 64, chunk=chunk)


@pytest.mark.parametrize("Sq", [1, 3, 64])
def test_rows_behind_the_length_do_not_matter(Sq):
    """Unwritten rows may hold anything: NaN and infinite scales, any codes."""
    B, Hq, Hkv, D, kv, cap = 2, 32, 4, 128, 170, 272
    cache, _, _ = filled_cache(B, Hkv, cap, D, 32, 61)
    q = rows((B, Hq, Sq, D), 63).to(DEV)
    lens = torch.full((B,), kv, dtype=torch.int32, device=DEV)
    want = K().attention_cache_q4(q, *cache, kv, 0.1, True), K().attention_cache_q4(q, *cache, lens, 0.1, True)
    for t in (cache[0], cache[2]):
        t[:, :, kv:] = 255
    for t, bad in ((cache[1], math.nan), (cache[3], math.inf)):
        t[:, :, kv:] = bad
    got = K().attention_cache_q4(q, *cache, kv, 0.1, True), K().attention_cache_q4(q, *cache, lens, 0.1, True)
    assert torch.isfinite(want[0]).all()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_nonfinite_key_or_value_reaches_only_the_rows_that_see_it():
    B, Hq, Hkv, D, kv, Sq = 1, 8, 2, 64, 40, 4
    cache, _, _ = filled_cache(B, Hkv, 48, D, 32, 65)
    q = rows((B, Hq, Sq, D), 66).to(DEV)
    want = K().attention_cache_q4(q, *cache, kv, 0.125, True).view(Sq, Hkv, -1)
    cache[1][0, 0, kv - 2] = math.nan  # a key of head 0 that queries 2 and 3 see
    got = K().attention_cache_q4(q, *cache, kv, 0.125, True).view(Sq, Hkv, -1)
    assert torch.equal(got[:2], want[:2]) and torch.equal(got[:, 1], want[:, 1])
    assert got[2:, 0].isnan().all()


@pytest.mark.parametrize("D,group", SHAPES)
def test_a_nonfinite_value_reaches_only_the_rows_that_see_it(D, group):
    """A weight of 0 times NaN is NaN: a value group stored as NaN must not touch
    the queries in front of it, the other channels or the other heads."""
    B, Hq, Hkv, kv, Sq = 2, 4, 2, 150, 40  # the mask crosses more than one key tile
    cache, _, _ = filled_cache(B, Hkv, 160, D, group, 67)
    q = rows((B, Hq, Sq, D), 68).to(DEV)
    want = K().attention_cache_q4(q, *cache, kv, 0.125, True).view(B, Sq, Hkv, 2, D // group, group)
    first = D // group - 1
    for key in (112, 149):  # seen from query 2 on, and by the last query only
        cache[3][1, 0, key, first] = math.nan
    got = K().attention_cache_q4(q, *cache, kv, 0.125, True).view(B, Sq, Hkv, 2, D // group, group)
    hit = got[1, 2:, 0, :, first]
    assert hit.isnan().all()
    hit.copy_(want[1, 2:, 0, :, first])
    assert torch.equal(got, want)


@pytest.mark.parametrize("D,group,Sq,kv,causal", [(128, 32, 40, 300, True), (128, 128, 130, 130, True),
                                                  (64, 32, 33, 2000, True), (32, 32, 20, 90, False)])
def test_a_nonfinite_row_in_a_chunk_reaches_only_the_rows_that_see_it(monkeypatch, D, group, Sq, kv, causal):
    monkeypatch.setattr(K(), "_q4_chunk", lambda *a: True)
    B, Hq, Hkv = 2, 4, 2
    cache, _, vv = filled_cache(B, Hkv, -(-kv // 16) * 16, D, group, 69)
    q = rows((B, Hq, Sq, D), 70).to(DEV)
    want = K().attention_cache_q4(q, *cache, kv, 0.125, causal).view(B, Sq, Hkv, 2, D // group, group)
    v, k = kv - Sq + 7, kv - Sq + 11  # seen from query 7 on, and from 11 on
    cache[3][1, 0, v, 0] = math.nan
    cache[3][1, 0, kv - 1, 0] = math.nan
    cache[1][0, 1, k, D // group - 1] = math.nan
    got = K().attention_cache_q4(q, *cache, kv, 0.125, causal).view(B, Sq, Hkv, 2, D // group, group)
    for hit, back in ((got[1, 7 if causal else 0:, 0, :, 0], want[1, 7 if causal else 0:, 0, :, 0]),
                      (got[0, 11 if causal else 0:, 1], want[0, 11 if causal else 0:, 1])):
        assert hit.isnan().all()
        hit.copy_(back)
    # Without the NaN rows the scales of the operands may be other powers of two.  That
    # moves only numbers below 2^-14 of them, by 2^-25: values by 2^-38 of the largest,
    # scores by less than 2^-17; then an output may round to the next bf16 (2^-7).
    tol = 2 ** -7 * want.double().abs() + 2 ** -16 * float(vv.abs().max())
    assert ((got.double() - want.double()).abs() <= tol).all()


@pytest.mark.parametrize("chunk", [False, True])
@pytest.mark.parametrize("log2", [-12.0, -20.0, -24.5])
def test_many_small_weights_beside_a_large_one(monkeypatch, chunk, log2):
    """60000 keys of weight 2^log2 beside one of weight 1 whose value is 0.  Keys and
    queries are exact in bf16 and fp16, so scores are off by fp32's sums and the
    chunk's exponential alone (d = 2^-13); weights and values round to 2^-8 each, in a
    chunk to 2^-11 (weights 2^-25 of the largest and above)."""
    monkeypatch.setattr(K(), "_q4_chunk", lambda *a: chunk)
    B, Hq, Hkv, Sq, kv, D, group = 1, 2, 1, 2, 60000, 128, 32
    cache, _, _ = filled_cache(B, Hkv, kv, D, group, 91, 0.5)
    codes = [t.clone() for t in cache]
    codes[0].zero_()                      # keys: s = 0, m = -1 everywhere, 0 in row 7
    codes[1][..., 0], codes[1][..., 1] = 0, -1
    codes[1][:, :, 7, :, 1] = 0
    codes[3][:, :, 7] = 0
    q = torch.full((B, Hq, Sq, D), -log2 * math.log(2) / D).bfloat16()
    kk, vv = R.values(codes[0], codes[1]), R.values(codes[2], codes[3])
    out = K().attention_cache_q4(q.to(DEV), *codes, kv, 1.0, False).double().cpu()
    ref, A = R.attention(q, kk, vv, [kv], 1.0, False)
    tol = A * (2 ** (-10 if chunk else -7) + math.expm1(2 ** -12)) + 2 ** -8 * ref.abs()
    assert ((out - ref).abs() <= tol).all(), float(((out - ref).abs() / tol).max())


def test_large_scores_and_equal_scores():
    """Scores of thousands (one key takes all) and a row of equal scores."""
    B, Hq, Hkv, D, kv = 1, 4, 1, 128, 300
    cache, kk, vv = filled_cache(B, Hkv, 304, D, 32, 71, 8.0)
    q = rows((B, Hq, 1, D), 73, 8.0)
    q[0, 3] = 0
    out = K().attention_cache_q4(q.to(DEV), *cache, kv, 1.0, False)
    ref, A = R.attention(q, kk, vv, [kv], 1.0, False)
    top = [int((kk[0, 0, :kv] @ q[0, h, 0].double()).argmax()) for h in range(3)]
    for h in range(3):
        v = vv[0, 0, top[h]]
        assert ((out[0, 0, h * D:(h + 1) * D].cpu().double() - v).abs() <= 2 ** -7 * v.abs()).all()
    mean = vv[0, 0, :kv].mean(0)
    tol = 2 ** -7 * A[0, 0, 3 * D:] + 2 ** -8 * mean.abs()
    assert ((out[0, 0, 3 * D:].cpu().double() - mean).abs() <= tol).all()


def test_rows_past_32_bit_offsets():
    """The last head of a cache whose codes pass 4 GiB."""
    B, Hkv, D, group, cap, n = 1, 3, 128, 128, 1 << 25, 50
    assert B * Hkv * cap * D // 2 > 1 << 32
    cache = (torch.empty(B, Hkv, cap, D // 2, dtype=torch.uint8, device=DEV),
             torch.empty(B, Hkv, cap, 1, 2, dtype=torch.bfloat16, device=DEV),
             torch.empty(B, Hkv, cap, D // 2, dtype=torch.uint8, device=DEV),
             torch.empty(B, Hkv, cap, 1, 2, dtype=torch.bfloat16, device=DEV))
    k, v = rows((B, Hkv, n, D), 81), rows((B, Hkv, n, D), 82)
    K().kv_append_q4(k.to(DEV), v.to(DEV), *cache, cap - n)
    check_stored(cache[0][:, :, cap - n:], cache[1][:, :, cap - n:], k, group)
    check_stored(cache[2][:, :, cap - n:], cache[3][:, :, cap - n:], v, group)
    kr, vr = K().kv_read_q4(*cache, cap - n, n)
    K().kv_append_q4(k.to(DEV), v.to(DEV), *cache, 0)
    k0, v0 = K().kv_read_q4(*cache, 0, n)
    assert torch.equal(kr, k0) and torch.equal(vr, v0)
    q = rows((B, 6, 1, D), 83)
    out = K().attention_cache_q4(q.to(DEV), *cache, n, 0.1, False)
    small = [t[:, :, :n].contiguous() for t in cache]
    kk, vv = R.values(small[0], small[1]), R.values(small[2], small[3])
    check_attention(out, q, kk, vv, [n], 0.1, False, group)


# ------------------------------------------------------------------ streams, graphs, determinism
def test_calls_on_another_stream_and_together():
    """Two calls in flight on two streams, and the same call again, agree."""
    B, Hq, Hkv, D, kv = 4, 32, 4, 128, 3000
    cache, _, _ = filled_cache(B, Hkv, 3008, D, 64, 91)
    q = rows((B, Hq, 1, D), 93).to(DEV)
    want = K().attention_cache_q4(q, *cache, kv, 0.09, False)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(K().attention_cache_q4(q, *cache, kv, 0.09, False))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_a_captured_step_follows_the_lengths():
    """One capture of append + advance + attention, replayed as the cache grows,
    gives what eager calls give; so does a second graph captured beside it."""
    B, Hq, Hkv, D, cap = 3, 8, 2, 64, 64
    bufs = [empty_cache(B, Hkv, cap, D, 32) for _ in range(3)]
    start = torch.tensor([0, 5, 30], dtype=torch.int32, device=DEV)
    past = rows((B, Hkv, cap, D), 101).to(DEV)
    q, k, v = (torch.empty(B, h, 1, D, dtype=torch.bfloat16, device=DEV) for h in (Hq, Hkv, Hkv))
    lens = [start.clone() for _ in range(3)]
    for c in bufs:
        K().kv_append_q4(past[:, :, :30], past[:, :, :30], *c, 0)

    def step(i):
        K().kv_append_q4(k, v, *bufs[i], lens[i])
        lens[i].add_(1)
        return K().attention_cache_q4(q, *bufs[i], lens[i], 0.125, False)

    graphs, outs = [], []
    for i in range(2):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step(i)
        torch.cuda.current_stream().wait_stream(side)
        lens[i].copy_(start)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
        lens[i].copy_(start)
    for n in range(20):
        q.copy_(rows((B, Hq, 1, D), 200 + n))
        k.copy_(rows((B, Hkv, 1, D), 300 + n))
        v.copy_(rows((B, Hkv, 1, D), 400 + n))
        for g in graphs:
            g.replay()
        want = step(2)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want), n
    assert lens[0].tolist() == [20, 25, 50]
    K().device_error_check()


@pytest.mark.parametrize("S,kv0", [(1, 0), (1, 700), (40, 300)])
def test_a_captured_chain_equals_its_calls_one_by_one(S, kv0):
    """Each call is launched ahead of the one in front of it and needs its results:
    rows stored, read back and attended over, the next rows made from both."""
    B, Hq, Hkv, D, steps = 2, 8, 2, 64, 8
    x0 = rows((B, Hkv, S, D), 95).to(DEV)
    cache0 = filled_cache(B, Hkv, 1024, D, 32, 96)[0]

    def chain(x, cache, pause):
        outs = []
        for i in range(steps):
            K().kv_append_q4(x, x * 0.5, *cache, kv0 + i * S)
            pause()
            k, v = K().kv_read_q4(*cache, max(0, kv0 + i * S - 3), 3 + S if kv0 else S)
            pause()
            q = (k[:, :, -S:].repeat_interleave(Hq // Hkv, dim=1) - 0.25).contiguous()
            out = K().attention_cache_q4(q, *cache, kv0 + (i + 1) * S, 0.125, True)
            pause()
            x = (out.view(B, S, Hkv, Hq // Hkv, D).sum(3).transpose(1, 2) + v[:, :, -S:]).contiguous()
            outs += [out, x]
        return outs

    want = chain(x0, [t.clone() for t in cache0], torch.cuda.synchronize)
    cache, x = [t.clone() for t in cache0], x0.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(x, cache, lambda: None)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(x, cache, lambda: None)
    for _ in range(3):
        for t, old in zip(cache, cache0):
            t.copy_(old)
        graph.replay()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("before", ["copy", "fill", "kernel", "two streams", "nothing"])
@pytest.mark.parametrize("kv,Sq", [(40, 1), (3000, 1), (900, 200)])
def test_a_capture_behind_other_work(monkeypatch, before, kv, Sq):
    """The attention kernels are launched ahead of the work in front of them: what
    that work writes (a copy, a fill, a kernel, the join of two streams) is what they
    read, on every replay."""
    monkeypatch.setattr(K(), "_q4_chunk", lambda *a: Sq > 100)
    B, Hq, Hkv, D = 2, 8, 2, 128
    cache, _, _ = filled_cache(B, Hkv, 3008, D, 32, 121)
    q, src = (torch.zeros(B, Hq, Sq, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    big = torch.zeros(1 << 24, device=DEV)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    n = kv if Sq > 1 else lens

    def work():
        if before == "copy":
            big.add_(1)
            q.copy_(src)
        elif before == "fill":
            big.add_(1)
            q.copy_(src)
            big[:1024].zero_()
        elif before == "kernel":
            big.add_(1)
            torch.mul(src, 1.0, out=q)
        elif before == "two streams":
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                big.add_(1)
                q.copy_(src)
            lens.fill_(kv)
            torch.cuda.current_stream().wait_stream(side)
        if before != "two streams":
            lens.fill_(kv)
        if before == "nothing":
            q.copy_(src)
        return K().attention_cache_q4(q, *cache, n, 0.09, True)

    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        work()
    torch.cuda.current_stream().wait_stream(warm)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = work()
    for i in range(3):
        src.copy_(rows((B, Hq, Sq, D), 500 + i))
        q.zero_()
        lens.zero_()
        g.replay()
        want = K().attention_cache_q4(src, *cache, kv if Sq > 1 else torch.full_like(lens, kv), 0.09, True)
        assert torch.equal(out, want), i


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_a_cache_on_another_device():
    cache, kk, vv = filled_cache(1, 2, 64, 64, 32, 111)
    cache = tuple(t.to("cuda:1") for t in cache)
    q = rows((1, 4, 1, 64), 113)
    out = K().attention_cache_q4(q.to("cuda:1"), *cache, 50, 0.125, False)
    check_attention(out, q, kk, vv, [50], 0.125, False, 32)


def test_refusals():
    cache = empty_cache(2, 2, 32, 64, 32)
    x = torch.zeros(2, 2, 4, 64, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device=DEV)
    Kk = K()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    bad = [lambda: Kk.kv_append_q4(x, x, *cache, 29), lambda: Kk.kv_append_q4(x, x, *cache, -1),
           lambda: Kk.kv_append_q4(x, x[:, :, :3], *cache, 0),
           lambda: Kk.kv_append_q4(x[..., :32], x[..., :32], *cache, 0),
           lambda: Kk.kv_append_q4(x.float(), x, *cache, 0),
           lambda: Kk.kv_append_q4(x, x, *cache, i32(1)), lambda: Kk.kv_append_q4(x, x, *cache, i32(1, 2).long()),
           lambda: Kk.kv_append_q4(x, x, *cache, i32(1, 2).cpu()),
           lambda: Kk.kv_append_q4(x, x, cache[0], cache[1][..., :1, :], cache[2], cache[3], 0),
           lambda: Kk.kv_append_q4(x, x, cache[0].float(), *cache[1:], 0),
           lambda: Kk.kv_append_q4(x, x, cache[0].transpose(0, 1), *cache[1:], 0),
           lambda: Kk.kv_read_q4(*cache, 30, 3), lambda: Kk.kv_read_q4(*cache, 0, -1),
           lambda: Kk.kv_read_q4(*[t[:, :, :24].contiguous() for t in cache], 0, 1),
           lambda: Kk.attention_cache_q4(q, *cache, 33, 0.1, False),
           lambda: Kk.attention_cache_q4(q, *cache, -1, 0.1, False),
           lambda: Kk.attention_cache_q4(q[:, :3], *cache, 3, 0.1, False),
           lambda: Kk.attention_cache_q4(q[:1], *cache, 3, 0.1, False),
           lambda: Kk.attention_cache_q4(q, *cache, i32(1, 2), 0.1, False, max_kv_len=33),
           lambda: Kk.attention_cache_q4(q.float(), *cache, 3, 0.1, False)]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    # nothing to do is no error
    Kk.kv_append_q4(x[:, :, :0], x[:, :, :0], *cache, 32)
    assert Kk.attention_cache_q4(q[:, :, :0], *cache, 3, 0.1, False).shape == (2, 0, 256)
    assert not Kk.attention_cache_q4(q, *cache, 0, 0.1, False).any()
    assert not Kk.attention_cache_q4(q.expand(2, 4, 300, 64), *cache, 0, 0.1, True).any()


# ------------------------------------------------------------------ layer, model
def _layer(cfg, g):
    from qwen3_5_vl_cuda_custom_b200 import synthetic as syn
    from qwen3_5_vl_cuda_custom_b200.modules import CudaTextDecoderLayer, TextMRoPE
    layer = CudaTextDecoderLayer(cfg.hidden_size, cfg.num_heads, cfg.num_kv_heads, cfg.head_dim,
                                 cfg.intermediate_size, cfg.rms_norm_eps, use_moe=True,
                                 num_experts=cfg.num_experts, top_k=cfg.num_experts_per_tok,
                                 moe_intermediate_size=cfg.moe_intermediate_size)
    layer.load_state_dict(syn.layer_params(cfg, g))
    return (layer.to(DEV, torch.bfloat16),
            TextMRoPE(cfg.head_dim, cfg.rope_theta, cfg.mrope_section).to(DEV))


@pytest.mark.parametrize("group", [32, 128])
def test_attention_module_over_a_prompt_chunk_and_decode_steps(group):
    """Prompt (exact k/v), a second chunk (rows read back), decode steps (codes):
    every call stores its rows and matches attention over what the cache holds."""
    from qwen3_5_vl_cuda_custom_b200.configs import a3b_moe_text
    from qwen3_5_vl_cuda_custom_b200.kv_cache import Q4LayerKVCache
    cfg = a3b_moe_text(1)
    g = torch.Generator().manual_seed(5)
    layer, rot = _layer(cfg, g)
    attn, D, B = layer.self_attn, cfg.head_dim, 2
    cache = Q4LayerKVCache(B, cfg.num_kv_heads, 250, D, DEV, group_size=group)
    at = 0
    with torch.no_grad():
        for S in (100, 60, 1, 3, 1):
            x = torch.randn(B, S, cfg.hidden_size, generator=g).bfloat16().to(DEV)
            pos = torch.arange(at, at + S, device=DEV).expand(B, S)
            bound = rot.bind(torch.stack([pos] * 3))
            q, k, v = attn._project(x, bound)
            y, kept = attn(x, bound, past_kv=cache)
            at += S
            assert kept is cache and cache.length == at
            w = slice(at - S, at)
            check_stored(cache.k_codes[:, :, w], cache.k_scales[:, :, w], k.cpu(), group)
            check_stored(cache.v_codes[:, :, w], cache.v_scales[:, :, w], v.cpu(), group)
            kr, vr = cache
            assert kr.shape == (B, cfg.num_kv_heads, at, D)
            if S == 100:
                o = K().attention_tokens(q, k, v, attn.scale, True)
            else:
                o = K().attention_cache_q4(q, *cache.buffers, at, attn.scale, S > 1)
                check_attention(o, q, R.values(cache.k_codes[:, :, :at], cache.k_scales[:, :, :at]),
                                R.values(cache.v_codes[:, :, :at], cache.v_scales[:, :, :at]), [at] * B,
                                attn.scale, S > 1, group, chunk=S == 60)
            assert torch.equal(y, attn.o_proj(o))
        with pytest.raises(RuntimeError, match="KV cache full"):
            x = torch.zeros(B, 90, cfg.hidden_size, dtype=torch.bfloat16, device=DEV)
            pos = torch.arange(90, device=DEV).expand(B, 90)
            attn(x, rot.bind(torch.stack([pos] * 3)), past_kv=cache)
        assert cache.length == at


def test_graphed_layer_decodes_a_ragged_batch():
    """GraphedDecoderLayer over a cache with per-sequence lengths: one capture
    serves a decode loop and matches the eager layer step by step."""
    from qwen3_5_vl_cuda_custom_b200.configs import tiny_moe_text
    from qwen3_5_vl_cuda_custom_b200.graphs import GraphedDecoderLayer
    from qwen3_5_vl_cuda_custom_b200.kv_cache import Q4LayerKVCache
    cfg = tiny_moe_text()
    g = torch.Generator().manual_seed(9)
    layer, rot = _layer(cfg, g)
    B, S0 = 3, 20
    lens = torch.tensor([20, 7, 13])
    caches = [Q4LayerKVCache(B, cfg.num_kv_heads, 64, cfg.head_dim, DEV) for _ in range(2)]
    x = torch.randn(B, S0, cfg.hidden_size, generator=g).bfloat16().to(DEV)
    pos = torch.arange(S0, device=DEV).expand(B, S0)
    with torch.no_grad():
        for c in caches:  # right-padded prompts, then their true lengths
            layer(x, rot.bind(torch.stack([pos] * 3)), past_kv=c)
            c.set_lengths(lens)
        x1 = torch.randn(B, 1, cfg.hidden_size, generator=g).bfloat16().to(DEV)
        p = lens.to(DEV)[:, None].expand(3, B, 1).contiguous()
        gl = GraphedDecoderLayer(layer, rot, x1, p, past_kv=caches[0])
        assert caches[0].lengths.tolist() == lens.tolist()
        for i in range(6):
            x1 = torch.randn(B, 1, cfg.hidden_size, generator=g).bfloat16().to(DEV)
            got = gl(x1)[0]
            want = layer(x1, rot.bind(p + i), past_kv=caches[1])[0]
            assert torch.equal(got, want), i
            gl.static_pos.add_(1)
    assert caches[0].lengths.tolist() == (lens + 6).tolist() == caches[1].lengths.tolist()
    for a, b in zip(caches[0].buffers, caches[1].buffers):
        for s, n in enumerate((lens + 6).tolist()):
            assert torch.equal(a[s, :, :n].view(torch.uint8), b[s, :, :n].view(torch.uint8))
    K().device_error_check()


def _tiny_model():
    from qwen3_5_vl_cuda_custom_b200.configs import MoETextConfig, moe_config
    from qwen3_5_vl_cuda_custom_b200.models import CudaQwen3VLMoeModel
    t = MoETextConfig(hidden_size=256, intermediate_size=512, num_layers=2, num_heads=4,
                      num_kv_heads=2, head_dim=64, vocab_size=512, rope_theta=1e4,
                      mrope_section=[16, 8, 8], num_experts=32, num_experts_per_tok=2,
                      moe_intermediate_size=64)
    torch.manual_seed(0)
    return CudaQwen3VLMoeModel(moe_config(t), vision=False).to(DEV, torch.bfloat16)


def test_generate_with_a_4_bit_cache():
    model = _tiny_model()
    ids = torch.randint(0, 512, (2, 12), device=DEV)
    with torch.no_grad():
        cache = model.make_kv_cache(2, 20, bits=4)
        out = model.generate(ids, max_new_tokens=6, kv_cache=cache)
        assert out.shape == (2, 18) and cache.length == 17
        # the same loop through forward(); the prompt attends over its exact k/v
        step, seq = model.make_kv_cache(2, 20, bits=4), [ids]
        bf16 = model.make_kv_cache(2, 20)
        logits, _ = model(ids, past_key_values=step)
        ref, _ = model(ids, past_key_values=bf16)
        assert torch.equal(logits, ref)
        for _ in range(5):
            seq.append(logits[:, -1].argmax(-1)[:, None])
            logits, _ = model(seq[-1], past_key_values=step)
        seq.append(logits[:, -1].argmax(-1)[:, None])
    assert torch.equal(out, torch.cat(seq, dim=1))
    with pytest.raises(ValueError):
        model.make_kv_cache(2, 20, bits=8)


def test_model_decodes_ragged_prompts_like_single_ones():
    """Prompts of different lengths in one right-padded batch, then per-sequence
    lengths: each sequence's logits match its own run within the kernels' batch
    variation (other GEMM shapes round differently)."""
    model = _tiny_model()
    ids = torch.randint(0, 512, (2, 12), device=DEV)
    nxt = torch.randint(0, 512, (2, 3), device=DEV)
    lens = [12, 7]
    with torch.no_grad():
        cache = model.make_kv_cache(2, 32, bits=4)
        model(ids, past_key_values=cache)
        cache.set_lengths(torch.tensor(lens))
        got = [model(nxt[:, i:i + 1], past_key_values=cache)[0][:, 0] for i in range(3)]
        for b, n in enumerate(lens):
            one = model.make_kv_cache(1, 32, bits=4)
            model(ids[b:b + 1, :n], past_key_values=one)
            for i in range(3):
                want = model(nxt[b:b + 1, i:i + 1], past_key_values=one)[0][0, 0]
                assert (got[i][b] - want).abs().max() <= 0.05 * want.abs().max(), (b, i)
            assert one.length == n + 3 == int(cache[0].lengths[b])
