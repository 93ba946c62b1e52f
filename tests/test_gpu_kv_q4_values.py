"""Attention over the 4-bit KV cache where the stored values are awkward: NaN keys in
every place of a key tile, values and scores at the ends of the range, and bounds as
tight as the kernels' own roundings, each form forced."""
import math

import pytest
import torch

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
