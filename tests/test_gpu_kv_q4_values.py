"""Attention over the 4-bit KV cache where the stored values are awkward: NaN keys in
every place of a key tile, values and scores at the ends of the range, and bounds as
tight as the kernels' own roundings, each form forced."""
import math

import pytest
import torch

import kv_q4_cases as C
import kv_q4_ref as R
from test_gpu_kv_q4 import DEV, SHAPES, K, filled_cache, rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _ready():
    from qwen3_5_vl_cuda_custom_b200 import build
    build.build()
    yield
    K().device_error_check()


def force(monkeypatch, chunk):
    monkeypatch.setattr(K(), "_q4_chunk", lambda *a: chunk)


# ------------------------------------------------------------------ NaN keys
@pytest.mark.parametrize("chunk", [True, False])
@pytest.mark.parametrize("Hq,Hkv", [(4, 2), (2, 2), (3, 1)])  # two heads or one per CTA
def test_a_nan_key_at_any_place_of_a_tile(monkeypatch, chunk, Hq, Hkv):
    """Both forms, every key index mod 32: the rows that see the key are NaN in all
    channels, the others and the other heads are what they were."""
    force(monkeypatch, chunk)
    B, Sq, kv, D, group = 1, 6, 140, 64, 32
    cache, _, _ = filled_cache(B, Hkv, 144, D, group, 131, 0.5)
    q = rows((B, Hq, Sq, D), 132, 0.5).to(DEV)
    cache[1][:, Hkv - 1, 96:] = 0  # what a NaN takes the place of is no largest value
    for key in range(96, 140):
        for causal in (False, True):
            want = K().attention_cache_q4(q, *cache, kv, 0.125, causal).view(Sq, Hkv, -1)
            ks = cache[1].clone()
            ks[0, Hkv - 1, key, key % 2] = math.nan
            got = K().attention_cache_q4(q, cache[0], ks, *cache[2:], kv, 0.125, causal).view(Sq, Hkv, -1)
            first = max(0, key - (kv - Sq)) if causal else 0
            assert got[first:, Hkv - 1].isnan().all(), (key, causal)
            assert torch.isfinite(want).all()
            assert torch.equal(got[:first], want[:first]), (key, causal)
            assert torch.equal(got[:, :Hkv - 1], want[:, :Hkv - 1]), (key, causal)


# ------------------------------------------------------------------ values of every size
@pytest.mark.parametrize("D,group", [(128, 32), (64, 64), (32, 32)])
@pytest.mark.parametrize("hidden", [(0.0, 3e38), (2e37, -3e38), (3e37, 0.0), (0.0, 2.0 ** 20), (0.0, 2.0 ** 116),
                                    (math.inf, 1.0), (1.0, -math.inf)])
def test_rows_a_chunk_does_not_see_hold_anything(monkeypatch, D, group, hidden):
    """Finite or not, a value reaches the queries that see it only.  A head's values share
    one power of two in this form: with e the exponent of the largest they round to
    2^(e - 39) at least, 2^-38 of the largest (at most fp32's largest).
    Other bounds as for any chunk: weights and values 2^-11 each, the keys' rounding and
    the exponential's 2^-13 in d, the output's 2^-8."""
    force(monkeypatch, True)
    B, Hq, Hkv, Sq, kv = 1, 4, 2, 40, 150
    cache, kk, vv = filled_cache(B, Hkv, 160, D, group, 133, 0.5)
    q = rows((B, Hq, Sq, D), 134, 0.5)
    seen = kv - 3  # keys 147 .. 149: the last three queries'
    cache[3][:, :, seen:kv, :, 0], cache[3][:, :, seen:kv, :, 1] = hidden
    out = K().attention_cache_q4(q.to(DEV), *cache, kv, D ** -0.5, True).double().cpu()[:, :Sq - 3]
    ref, A = R.attention(q[:, :, :Sq - 3], kk, vv, [seen], D ** -0.5, True)
    big = R.values(cache[2], cache[3])[:, :, :kv].abs()
    big = float(torch.where(torch.isfinite(big), big.clamp(max=2.0 ** 128), torch.zeros_like(big)).max())
    d = 2.0 ** -11 * D ** -0.5 * float((q.double().abs().amax((0, 1, 2)) * kk.abs().amax((0, 1, 2))).sum())
    tol = A * (2 ** -10 + math.expm1(2 * (d + 2.0 ** -13))) + 2 ** -8 * ref.abs() + 2.0 ** -38 * big
    assert torch.isfinite(out).all()
    assert ((out - ref).abs() <= tol).all(), float(((out - ref).abs() / tol).max())


@pytest.mark.parametrize("chunk", [True, False])
def test_the_largest_values_come_through(monkeypatch, chunk):
    """Values up to 2^126 (2^98 on the codes): both forms return their weighted mean."""
    force(monkeypatch, chunk)
    top = 2.0 ** (127 if chunk else 99)
    B, Hq, Hkv, Sq, kv, D, group = 1, 4, 2, 20, 150, 64, 32
    cache, kk, _ = filled_cache(B, Hkv, 160, D, group, 135, 0.5)
    q = rows((B, Hq, Sq, D), 136, 0.5)
    cache[3][..., 0], cache[3][..., 1] = top / 32, -top / 2
    vv = R.values(cache[2], cache[3])
    out = K().attention_cache_q4(q.to(DEV), *cache, kv, D ** -0.5, False).double().cpu()
    ref, A = R.attention(q, kk, vv, [kv], D ** -0.5, False)
    d = 2.0 ** -11 * D ** -0.5 * float((q.double().abs().amax((0, 1, 2)) * kk.abs().amax((0, 1, 2))).sum())
    tol = A * (2 ** -10 + math.expm1(2 * (d + 2.0 ** -13))) + 2 ** -8 * ref.abs()
    assert ((out - ref).abs() <= tol).all(), float(((out - ref).abs() / tol).max())


@pytest.mark.parametrize("chunk", [True, False])
@pytest.mark.parametrize("q_log2,k_log2", [(20, 20), (70, 40), (-60, 90), (-60, -30), (40, -90), (0, 110)])
def test_queries_and_keys_of_every_size(monkeypatch, chunk, q_log2, k_log2):
    """Powers of two on the queries and the keys that the scale takes back change nothing:
    the same call without them has the same products.  (In a chunk bit for bit; on the
    codes a product may meet fp32's smallest numbers.)"""
    force(monkeypatch, chunk)
    B, Hq, Hkv, Sq, kv, D, group = 1, 4, 2, 24, 300, 64, 32
    cache, kk, vv = filled_cache(B, Hkv, 304, D, group, 137, 0.5)
    q = rows((B, Hq, Sq, D), 138, 0.5)
    scale = 2.0 ** -3
    want = K().attention_cache_q4(q.to(DEV), *cache, kv, scale, True)
    q2 = (q.double() * 2.0 ** q_log2).bfloat16().to(DEV)
    ks = (cache[1].double() * 2.0 ** k_log2).bfloat16()
    got = K().attention_cache_q4(q2, cache[0], ks, *cache[2:], kv, scale * 2.0 ** -(q_log2 + k_log2), True)
    if chunk:
        assert torch.equal(got, want)
        return
    got, (ref, A) = got.double().cpu(), R.attention(q, kk, vv, [kv], scale, True)
    d = 2.0 ** -19 * scale * float((q.double().abs().amax((0, 1, 2)) * kk.abs().amax((0, 1, 2))).sum()) * 20
    tol = A * (2 ** -10 + math.expm1(2 * d + 2.0 ** -20)) + 2 ** -8 * ref.abs() + 2 ** -14 * float(vv.abs().max())
    assert ((got - ref).abs() <= tol).all(), float(((got - ref).abs() / tol).max())


@pytest.mark.parametrize("chunk", [True, False])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_nonfinite_query_spoils_its_own_row_only(monkeypatch, chunk, bad):
    force(monkeypatch, chunk)
    for Hq, Hkv in ((4, 2), (3, 3)):
        B, Sq, kv, D, group = 1, 9, 140, 64, 32
        cache, _, _ = filled_cache(B, Hkv, 144, D, group, 139, 0.5)
        q = rows((B, Hq, Sq, D), 140, 0.5).to(DEV)
        q[0, 1, 3, 37] = 0
        want = K().attention_cache_q4(q, *cache, kv, 0.125, True).view(Sq, Hq, D)
        q[0, 1, 3, 37] = bad
        got = K().attention_cache_q4(q, *cache, kv, 0.125, True).view(Sq, Hq, D)
        assert got[3, 1].isnan().all()
        got[3, 1] = want[3, 1]
        assert torch.equal(got, want)


@pytest.mark.parametrize("chunk,log2", [(c, x) for c in (True, False) for x in (20, 23, 24, 25, 26)]
                         + [(False, x) for x in (28, 33, 60)])
@pytest.mark.parametrize("part", [0.5, 0.625, 0.75, 0.9375])
def test_scores_of_many_millions(monkeypatch, chunk, log2, part):
    """Keys 3 and 77 have the same score, part * 2^log2, all others its negative: the
    output is the mean of their values (all operands and sums are exact)."""
    force(monkeypatch, chunk)
    B, Hq, Hkv, Sq, kv, D, group = 1, 4, 2, 3, 140, 64, 32
    cache, _, vv = filled_cache(B, Hkv, 144, D, group, 141, 0.5)
    cache[3][:, :, 77] = cache[3][:, :, 3]  # (values of one size)
    vv = R.values(cache[2], cache[3])
    cache[1][..., 0], cache[1][..., 1] = 0, -1
    cache[1][:, :, 3, :, 1] = cache[1][:, :, 77, :, 1] = 1
    q = torch.full((B, Hq, Sq, D), part * 2.0 ** (log2 - 6), dtype=torch.bfloat16, device=DEV)
    out = K().attention_cache_q4(q, *cache, kv, 1.0, False).double().cpu().view(Sq, Hkv, 2, D)
    pair = vv[0][:, [3, 77]]
    ref, A = pair.mean(1)[None, :, None], pair.abs().mean(1)[None, :, None]
    # weights and values 2^-11 each, values at most 2^-15 of the largest scale; the output
    tol = A * 2 ** -10 + 2 ** -15 * float(cache[3][:, :, 3, :, 0].max()) + 2 ** -8 * ref.abs()
    assert ((out - ref).abs() <= tol).all(), float(((out - ref).abs() / tol).max())


def test_a_chunk_at_scores_whose_steps_exceed_the_slack(monkeypatch):
    """Key 140, in the second key tile, scores 4 * 0.9 above key 3 in log2 units at about
    2^25: its weight is not rescaled for and must still fit fp16, whatever the rounding
    of the running maximum.  Operands and products are exact."""
    force(monkeypatch, True)
    B, Hq, Hkv, Sq, kv, D, group = 1, 2, 1, 103, 150, 64, 32
    cache, _, vv = filled_cache(B, Hkv, 160, D, group, 143, 0.5)
    cache[1][..., 0], cache[1][..., 1] = 0, -1
    cache[1][:, :, 3, :, 1] = cache[1][:, :, 140, :, 1] = 1
    cache[0][:, :, 140] = 0
    cache[0][:, :, 140, 0] = 1          # channel 0: code 1 of scale 1
    cache[1][:, :, 140, 0, 0] = 1
    kk = R.values(cache[0], cache[1])
    assert kk[0, 0, 140, 0] == 2 and (kk[0, 0, 140, 1:] == 1).all() and (kk[0, 0, 3] == 1).all()
    q = (2.0 ** 19 * (1 + torch.arange(18, 121) / 128)).bfloat16()[None, None, :, None].repeat(B, Hq, 1, D)
    q[..., 0] = 4
    out = K().attention_cache_q4(q.to(DEV), *cache, kv, 0.9 * math.log(2), False).double().cpu().view(Sq, Hq, D)
    w = 2.0 ** 3.6
    ref = (w * vv[0, 0, 140] + vv[0, 0, 3]) / (w + 1)
    A = (w * vv[0, 0, 140].abs() + vv[0, 0, 3].abs()) / (w + 1)
    tol = A * (2 ** -10 + math.expm1(2 ** -12)) + 2 ** -8 * ref.abs()
    assert ((out - ref).abs() <= tol).all(), float(((out - ref).abs() / tol).max())


# ------------------------------------------------------------------ precision
@pytest.mark.parametrize("chunk", [True, False])
@pytest.mark.parametrize("D,group", SHAPES)
@pytest.mark.parametrize("n", [2, 90, 1000, 9000])
def test_weights_and_values_keep_11_bits(monkeypatch, chunk, D, group, n):
    force(monkeypatch, chunk)
    for weights, xs in ((True, (0, 1, 2, 5, 17, 40, 63, 100, 127)), (False, (-50, -20, 0, 20, 36))):
        for x in xs:
            case = C.weights_case(D, group, n, x) if weights else C.values_case(D, group, n, x)
            q, cache, scale = case
            out = K().attention_cache_q4(q.to(DEV), *[t.to(DEV) for t in cache], n, scale, False)
            ref, tol = C.bounds(case, n, weights)
            err = (out.double().cpu() - ref).abs()
            assert (err <= tol).all(), (weights, x, float((err / tol).max()))


@pytest.mark.parametrize("D,group,B,Hq,Hkv,Sq,kv,causal", [
    (128, 32, 2, 32, 4, 100, 333, True), (128, 128, 2, 32, 4, 64, 64, True), (64, 64, 2, 8, 2, 130, 400, True),
    (32, 32, 2, 6, 2, 128, 100, True),             # the first 28 queries see nothing
    (128, 64, 2, 32, 4, 40, 129, False), (128, 32, 1, 5, 1, 33, 700, True), (64, 32, 1, 9, 3, 200, 2500, True),
])
def test_a_chunk_within_its_roundings(monkeypatch, D, group, B, Hq, Hkv, Sq, kv, causal):
    """The form for chunks against 64 bits, with bounds per query: keys, weights and values
    rounded to 2^-11 each, queries exact; scores off by d = (2^-11 + 2^-17) scale
    max_k sum_d |q_d k_d| (2^-17: fp32 sums of 128 products and the scale) and the
    exponential's 2^-13; the output's 2^-8.  Rows behind the length hold NaN and
    infinities."""
    force(monkeypatch, True)
    cap = -(-kv // 16) * 16 + 144
    cache, kk, vv = filled_cache(B, Hkv, cap, D, group, 145, 0.5)
    for t, bad in ((cache[0], 255), (cache[1], math.nan), (cache[2], 255), (cache[3], math.inf)):
        t[:, :, kv:] = bad
    q = rows((B, Hq, Sq, D), 146, 0.5)
    out = K().attention_cache_q4(q.to(DEV), *cache, kv, D ** -0.5, causal).double().cpu()
    ref, A = R.attention(q, kk, vv, [kv] * B, D ** -0.5, causal)
    G = Hq // Hkv
    size = torch.matmul(q.double().abs().view(B, Hkv, G * Sq, D), kk[:, :, :kv].abs().transpose(-1, -2))
    size = size.amax(-1).view(B, Hq, Sq).transpose(1, 2)[..., None]  # per query
    d = (2.0 ** -11 + 2.0 ** -17) * D ** -0.5 * size + 2.0 ** -13
    tol = A.view(B, Sq, Hq, D) * (2 ** -10 + torch.expm1(2 * d)) + 2 ** -8 * ref.abs().view(B, Sq, Hq, D)
    err = (out - ref).abs().view(B, Sq, Hq, D)
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("kv", [400, 9000])
def test_rows_of_zeros_beside_large_values(monkeypatch, kv):
    """On the codes, values of 0 weigh what others do as long as those stay below 2^40:
    every second row is 0, the rest 2^39 .. 2^40, weights 1 and 2^-20."""
    force(monkeypatch, False)
    B, Hq, Hkv, D, group = 1, 2, 1, 128, 32
    cache, _, _ = filled_cache(B, Hkv, -(-kv // 16) * 16, D, group, 147, 0.5)
    cache[0].zero_()                                   # keys: s = 0, m = 0 or -1
    cache[1][..., 0], cache[1][..., 1] = 0, 0
    cache[1][:, :, 3::4, :, 1] = -1
    cache[3][..., 0], cache[3][..., 1] = 2.0 ** 35, 2.0 ** 39
    cache[3][:, :, ::2] = 0
    q = torch.full((B, Hq, 1, D), 20 * math.log(2) / D).bfloat16()
    out = K().attention_cache_q4(q.to(DEV), *cache, kv, 1.0, False).double().cpu()
    ref, A = R.attention(q, R.values(cache[0], cache[1]), R.values(cache[2], cache[3]), [kv], 1.0, False)
    tol = A * (2 ** -10 + 2 ** -17) + 2 ** -8 * ref.abs()
    assert ((out - ref).abs() <= tol).all(), float(((out - ref).abs() / tol).max())


def test_chunks_in_flight_together_and_again(monkeypatch):
    """Two calls on two streams, replays of a captured one, a NaN key and a NaN value
    among the rows: the same bits every time."""
    force(monkeypatch, True)
    B, Hq, Hkv, Sq, kv, D, group = 2, 8, 2, 60, 3000, 128, 32
    cache, _, _ = filled_cache(B, Hkv, 3008, D, group, 148)
    cache[1][0, 1, 2970, 2] = cache[3][1, 0, 2960, 1] = math.nan
    q = rows((B, Hq, Sq, D), 149).to(DEV)
    want = K().attention_cache_q4(q, *cache, kv, 0.09, True)
    bits = want.view(torch.int16)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(K().attention_cache_q4(q, *cache, kv, 0.09, True))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs.append(K().attention_cache_q4(q, *cache, kv, 0.09, True))
    for _ in range(3):
        outs[-1].zero_()
        graph.replay()
        assert all(torch.equal(o.view(torch.int16), bits) for o in outs)
    assert want[0].isnan().any() and not want[:, :20].isnan().any()


@pytest.mark.parametrize("chunk,top", [(True, 126), (True, 100), (True, -90), (False, 98), (False, -50)])
@pytest.mark.parametrize("kv", [150, 9000])
def test_large_and_small_values_in_one_run_and_in_several(monkeypatch, chunk, top, kv):
    """Values up to 2^top: runs and splits of the keys leave partial sums in fp32, which
    have to hold them.  Equal weights (queries of 0), so the bounds are 2^-11 for values,
    2^-11 for weights, 2^-12 for the exponential and 2^-17 for sums, and the output's."""
    force(monkeypatch, chunk)
    B, Hq, Hkv, Sq, D, group = 1, 4, 2, 20, 64, 32
    cache, _, _ = filled_cache(B, Hkv, -(-kv // 16) * 16, D, group, 151, 0.5)
    cache[3][..., 0], cache[3][..., 1] = 2.0 ** (top - 4), 2.0 ** (top - 6)
    vv = R.values(cache[2], cache[3])
    q = torch.zeros(B, Hq, Sq, D, dtype=torch.bfloat16)
    out = K().attention_cache_q4(q.to(DEV), *cache, kv, D ** -0.5, False).double().cpu()
    ref = vv[:, :, :kv].mean(2).repeat_interleave(Hq // Hkv, 1).reshape(B, 1, Hq * D)
    tol = ref.abs() * (2 ** -10 + 2 ** -12 + 2 ** -17 + 2 ** -8)
    assert ((out - ref).abs() <= tol).all(), float(((out - ref).abs() / tol).max())


def test_an_infinite_query_among_sixteen_rows(monkeypatch):
    """Rows of one group, eight apart: the second's largest number lies where the first
    holds the infinity."""
    force(monkeypatch, False)
    B, Hq, Hkv, kv, D, group = 64, 64, 4, 4096, 64, 32
    cache, _, _ = filled_cache(1, Hkv, kv, D, group, 153, 0.5)
    cache = [t.repeat(B, *[1] * (t.dim() - 1)) for t in cache]
    q = rows((B, Hq, 1, D), 154, 0.5).to(DEV)
    q[:, 8::16] *= 2.0 ** -30
    q[:, 8::16, :, 0] = 2.0 ** 30
    want = K().attention_cache_q4(q, *cache, kv, 2.0 ** -27, False).view(B, Hq, D)
    q[:, ::16, :, 0] = math.inf
    got = K().attention_cache_q4(q, *cache, kv, 2.0 ** -27, False).view(B, Hq, D)
    assert got[:, ::16].isnan().all() and torch.isfinite(want).all()
    got[:, ::16] = want[:, ::16]
    assert torch.equal(got, want)
