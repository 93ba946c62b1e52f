"""4-bit KV cache without a GPU: the stored form's definition, argument checks
of the C entry points, and the caches' host-side bookkeeping."""
import ctypes

import numpy as np
import pytest
import torch

import kv_q4_ref as R
from qwen3_5_vl_cuda_custom_b200 import _lib, build
from qwen3_5_vl_cuda_custom_b200 import kernels as K
from qwen3_5_vl_cuda_custom_b200.kv_cache import KVCache, LayerKVCache, Q4KVCache, Q4LayerKVCache


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


# ------------------------------------------------------------------ the oracle
@pytest.mark.parametrize("D,group", [(32, 32), (64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
def test_oracle_round_trip_is_within_half_a_step(D, group):
    x = torch.randn(3, 5, D, generator=torch.Generator().manual_seed(D + group)).bfloat16()
    c, s, m = R.quantise(x, group)
    sm = torch.from_numpy(np.stack([s, m], -1)).bfloat16()
    assert torch.equal(sm.double(), torch.from_numpy(np.stack([s, m], -1)))  # both are bf16 numbers
    y = R.values(R.pack(c), sm)
    # half a step, plus the scale's rounding (2^-8 of the scale, on at most 15 steps)
    step = torch.from_numpy(s).repeat_interleave(group, -1)
    assert ((y - x.double()).abs() <= step * (0.5 + 15 * 2.0 ** -8)).all()


def test_field_order_is_a_permutation():
    for D in (32, 64, 128):
        byte, shift = R.field_order(D)
        assert sorted(2 * b + s // 4 for b, s in zip(byte, shift)) == list(range(D))


# ------------------------------------------------------------------ C argument checks
def _strides(*v):
    return (ctypes.c_int64 * 3)(*v)


def _append(lib, B=1, Hkv=2, S=4, D=64, group=32, cap=16, offset=0, offsets=None, k=256, cache=256,
            strides=(1024, 512, 64)):
    p = ctypes.c_void_p  # never dereferenced: validation fails first
    return lib.q35_kv_append_q4(p(k), p(k), _strides(*strides), _strides(*strides), p(cache), p(cache),
                                p(cache), p(cache), B, Hkv, S, D, group, cap, offset, offsets, None)


@pytest.mark.parametrize("kw,status", [
    (dict(D=48), 4), (dict(D=256), 4), (dict(group=16), 4), (dict(group=128), 4), (dict(B=-1), 2),
    (dict(Hkv=0), 2), (dict(cap=24), 2), (dict(cap=1 << 31), 2), (dict(S=-1), 2), (dict(S=17), 2),
    (dict(offset=-1), 2), (dict(offset=13), 2), (dict(S=17, offsets=256), 2), (dict(k=None), 1),
    (dict(cache=None), 1), (dict(k=8), 3), (dict(cache=8), 3), (dict(strides=(1024, 512, 4)), 3),
])
def test_append_refusals(lib, kw, status):
    assert _append(lib, **kw) == status


def test_append_of_nothing_needs_no_gpu(lib):
    assert _append(lib, S=0, k=None) == 0
    assert _append(lib, B=0, k=None, cache=None) == 0


@pytest.mark.parametrize("kw,status", [
    (dict(n=17), 2), (dict(n=-1), 2), (dict(start=13), 2), (dict(start=-1), 2), (dict(out_cap=3), 2),
    (dict(out=None), 1), (dict(out=8), 3), (dict(group=128), 4),
])
def test_read_refusals(lib, kw, status):
    a = dict(n=4, out_cap=None, start=0, out=256, group=32)
    a.update(kw)
    p = ctypes.c_void_p
    cap = a["n"] if a["out_cap"] is None else a["out_cap"]
    assert lib.q35_kv_read_q4(p(256), p(256), p(256), p(256), p(a["out"]), p(a["out"]), 1, 2, a["n"],
                              cap, 64, a["group"], 16, a["start"], None, None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(Hq=7), 2), (dict(Hq=0), 2), (dict(Sq=-1), 2), (dict(kv_len=17), 2), (dict(kv_len=-1), 2),
    (dict(q=None), 1), (dict(q=8), 3), (dict(D=80), 4),
])
def test_attention_refusals(lib, kw, status):
    a = dict(Hq=8, Sq=1, kv_len=16, q=256, D=64)
    a.update(kw)
    p = ctypes.c_void_p
    assert lib.q35_attn_q4_fwd(p(a["q"]), p(256), p(256), p(256), p(256), p(256), 1, a["Hq"], 2, a["Sq"],
                               a["kv_len"], None, 16, a["D"], 32, 0.1, 0, p(256), None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(Hq=7), 2), (dict(Sq=-1), 2), (dict(kv_len=17), 2), (dict(kv_len=0), 2), (dict(q=None), 1),
    (dict(q=8), 3), (dict(ws=None), 1), (dict(ws=8), 3), (dict(D=80), 4), (dict(B=40000), 2),
])
def test_chunk_attention_refusals(lib, kw, status):
    a = dict(B=1, Hq=8, Sq=64, kv_len=16, q=256, D=64, ws=256)
    a.update(kw)
    p = ctypes.c_void_p
    assert lib.q35_attn_q4_chunk_fwd(p(a["q"]), p(256), p(256), p(256), p(256), p(256), a["B"], a["Hq"],
                                     2, a["Sq"], a["kv_len"], 16, a["D"], 32, 0.1, 1, p(a["ws"]), None) == status


def test_the_form_for_chunks_is_not_proposed_for_refused_shapes(lib):
    prefers = lib.q35_attn_q4_prefers_chunk
    for args in ((0, 32, 4, 4, 8192, 128), (1, 7, 2, 512, 8192, 128), (1, 8, 2, 512, 0, 128),
                 (40000, 8, 2, 512, 8192, 128)):
        assert prefers(*args) == 0
    assert not K._q4_chunk(1, 32, 4, 2, 8192, 128) and not K._q4_chunk(1, 32, 4, 512, 0, 128)


def test_workspace_covers_every_shape(lib):
    assert lib.q35_attn_q4_workspace(0, 8, 2, 1, 100, 64) >= 0
    assert lib.q35_attn_q4_workspace(64, 32, 4, 1, 8193, 128) >= 0


def test_workspace_of_refused_shapes_is_empty(lib):
    for Hq, Hkv in ((1, 4), (7, 2), (0, 4), (4, 0), (-4, 2)):
        assert lib.q35_attn_q4_workspace(2, Hq, Hkv, 1, 100, 64) == 0
        assert lib.q35_attn_q4_chunk_workspace(2, Hq, Hkv, 1, 100, 64) == 0
    assert lib.q35_attn_q4_workspace(2, 4, 2, 0, 100, 64) == 0
    assert lib.q35_attn_q4_workspace(2, 4, 2, 1, 1 << 40, 64) == 0


def test_a_cache_without_heads_is_refused():
    empty = [torch.zeros(2, 0, 16, 32, dtype=torch.uint8), torch.zeros(2, 0, 16, 2, 2, dtype=torch.bfloat16)] * 2
    with pytest.raises(RuntimeError):
        K.attention_cache_q4(torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16), *empty, 4, 1.0, False)


def test_operators_refuse_cpu_tensors():
    c = Q4LayerKVCache(1, 2, 16, 64, "cpu")
    x = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    for call in (lambda: K.kv_append_q4(x, x, *c.buffers, 0), lambda: K.kv_read_q4(*c.buffers, 0, 1),
                 lambda: K.attention_cache_q4(x, *c.buffers, 4, 0.1, True)):
        with pytest.raises(RuntimeError, match="CUDA tensor required"):
            call()


# ------------------------------------------------------------------ caches
def test_layer_cache_sizes_and_lengths():
    c = Q4LayerKVCache(3, 2, 100, 128, "cpu", group_size=64)
    assert isinstance(c, LayerKVCache) and c.capacity == 100 and c.length == 0 and len(c) == 2
    assert c.k_codes.shape == (3, 2, 112, 64) and c.v_scales.shape == (3, 2, 112, 2, 2)
    c.length = 7
    assert c.save_length() == 7
    c.restore_length(5)
    assert c.length == 5
    c.set_lengths(torch.tensor([5, 0, 100]))
    kept = c.lengths
    assert kept.dtype == torch.int32 and c.length == 100
    saved = c.save_length()
    c.lengths[1] = 9
    c.restore_length(saved)
    assert c.lengths.tolist() == [5, 0, 100]
    with pytest.raises(RuntimeError, match="length per sequence"):
        c.length = 3
    with pytest.raises(RuntimeError, match="length per sequence"):
        c.views()
    c.reset()
    assert c.length == 0 and c.lengths is None
    c.set_lengths(torch.tensor([1, 2, 3]))
    assert c.lengths is kept  # a captured graph keeps reading this tensor


@pytest.mark.parametrize("lengths", [torch.tensor([1, 2]), torch.tensor([1, 2, 101]),
                                     torch.tensor([-1, 2, 3]), torch.tensor([1.0, 2.0, 3.0])])
def test_set_lengths_refusals(lengths):
    c = Q4LayerKVCache(3, 2, 100, 64, "cpu")
    with pytest.raises(ValueError):
        c.set_lengths(lengths)


@pytest.mark.parametrize("kw", [dict(head_dim=72), dict(group_size=16), dict(group_size=128),
                                dict(capacity=0)])
def test_layer_cache_refusals(kw):
    a = dict(batch=1, num_kv_heads=2, capacity=16, head_dim=64, device="cpu")
    a.update(kw)
    with pytest.raises(ValueError):
        Q4LayerKVCache(**a)


def test_a_full_cache_refuses_rows():
    c = Q4LayerKVCache(1, 2, 16, 64, "cpu")
    c.length = 14
    x = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="KV cache full"):
        c.append_attend(x, x, x, 0.1, True)


def test_model_cache():
    cache = Q4KVCache(3, 2, 2, 32, 64, "cpu", group_size=64)
    assert isinstance(cache, KVCache) and len(cache) == 3 and cache.length == 0
    cache.set_lengths(torch.tensor([3, 4]))
    assert cache.length == 4 and all(layer.lengths.tolist() == [3, 4] for layer in cache)
    cache.reset()
    assert cache.length == 0


def test_next_positions():
    from qwen3_5_vl_cuda_custom_b200.models import _next_positions
    assert _next_positions(None, 2, 3, "cpu")[0].tolist() == [[0, 1, 2]] * 2
    kv = torch.zeros(2, 1, 5, 8)
    assert _next_positions([(kv, kv)], 2, 2, "cpu")[2].tolist() == [[5, 6]] * 2
    cache = Q4KVCache(1, 2, 2, 32, 64, "cpu")
    cache[0].length = 4
    assert _next_positions(cache, 2, 2, "cpu")[1].tolist() == [[4, 5]] * 2
    cache.set_lengths(torch.tensor([3, 9]))
    assert _next_positions(cache, 2, 2, "cpu")[1].tolist() == [[3, 4], [9, 10]]
