"""What the 4-bit cache's wrappers and caches do around a launch, on the CPU with the
library's calls replaced."""
import gc
import weakref

import pytest
import torch

from qwen3_5_vl_cuda_custom_b200 import kernels as K


@pytest.mark.parametrize("name", ["append", "read", "attention"])
def test_a_copy_of_the_positions_lives_until_the_launch(monkeypatch, name):
    """A strided tensor of positions is copied; the copy's memory must not go to the
    outputs that are allocated after it."""
    copies, seen = [], []

    def copied(t, *_):
        c = t.clone()
        copies.append(weakref.ref(c))
        return c

    def call(entry, *args):
        gc.collect()
        seen.append([r() is not None for r in copies])

    monkeypatch.setattr(K, "_per_sequence", copied)
    monkeypatch.setattr(K, "_cache_q4", lambda *a: (2, 1, 16, 32, 32))
    monkeypatch.setattr(K, "_strided_rows", lambda t, *a: (t, t.stride()))
    monkeypatch.setattr(K, "_require", lambda t, *a: t)
    monkeypatch.setattr(K, "_stream", lambda t: None)
    monkeypatch.setattr(K.torch.cuda, "current_device", lambda: None)
    monkeypatch.setattr(K._lib, "call", call)
    monkeypatch.setattr(K._lib, "query", lambda *a: 0)
    cache = [torch.zeros(2, 1, 16, 16, dtype=torch.uint8)] * 4
    x = torch.zeros(2, 1, 1, 32, dtype=torch.bfloat16)
    at = torch.zeros(2, 3, dtype=torch.int32)[:, 1]
    if name == "append":
        K.kv_append_q4(x, x, *cache, at)
    elif name == "read":
        K.kv_read_q4(*cache, at, 1)
    else:
        K.attention_cache_q4(x, *cache, at, 1.0, False)
    assert seen == [[True]]


def test_the_reference_mask_over_caches_with_lengths(monkeypatch):
    """reference_chunk_mask: causal on an empty cache, no mask behind rows; also when the
    lengths are on the device, and in the warm-up and the capture of one step."""
    from qwen3_5_vl_cuda_custom_b200.kv_cache import LayerKVCache, Q4LayerKVCache
    from qwen3_5_vl_cuda_custom_b200.modules import CudaFullAttention

    class Seen(Exception):
        pass

    attn = CudaFullAttention(64, 2, 1, 32)
    attn.reference_chunk_mask = True
    x = torch.zeros(2, 3, 64)
    monkeypatch.setattr(attn, "_project", lambda x, m: (x, x, x))

    def mask(cache):
        def append_attend(q, k, v, scale, causal):
            raise Seen(causal)
        with monkeypatch.context() as m, pytest.raises(Seen) as e:
            m.setattr(cache, "append_attend", append_attend)
            attn(x, None, past_kv=cache)
        return e.value.args[0]

    for cache in (LayerKVCache(2, 1, 16, 32, "cpu"), Q4LayerKVCache(2, 1, 16, 32, "cpu")):
        assert mask(cache) is True
        cache.length = 3
        assert mask(cache) is False
    cache.set_lengths(torch.tensor([0, 4]))
    assert mask(cache) is False
    cache.set_lengths(torch.tensor([0, 0]))
    assert mask(cache) is True
    saved = cache.save_length()
    monkeypatch.setattr(K, "kv_append_q4", lambda *a: None)
    monkeypatch.setattr(K, "attention_cache_q4", lambda *a, **k: None)
    cache.append_attend(x[:, None, :, :32], x[:, None, :, :32], x[:, None, :, :32], 1.0, True)
    assert cache.lengths.tolist() == [3, 3] and mask(cache) is False
    cache.restore_length(saved)
    assert cache.lengths.tolist() == [0, 0] and mask(cache) is True
    cache.reset()
    assert mask(cache) is True


@pytest.mark.parametrize("weights", [True, False])
@pytest.mark.parametrize("x", [0, 5, 40, 100])
def test_the_precision_cases_tell_8_bits_from_11(weights, x):
    """What the attention kernels are held to (test_gpu_kv_q4_values.py) excludes weights
    or values of bf16's 8 bits."""
    import kv_q4_cases as C
    case = C.weights_case(64, 32, 90, x) if weights else C.values_case(64, 32, 90, x - 50)
    ref, tol = C.bounds(case, 90, weights)
    assert ((C.with_bf16(case, 90, weights) - ref).abs() > 1.2 * tol).all()


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 2.0 ** 101, -(2.0 ** 120)])
def test_scales_out_of_range_are_refused(scale):
    import ctypes
    from qwen3_5_vl_cuda_custom_b200 import _lib, build
    build.build()
    lib, p = _lib.load(), ctypes.c_void_p(256)  # never dereferenced: validation fails first
    args = [p] * 6
    assert lib.q35_attn_q4_fwd(*args, 1, 8, 2, 1, 16, None, 16, 64, 32, scale, 0, p, None) == 1
    assert "scale" in lib.q35_last_error_message().decode()
    assert lib.q35_attn_q4_chunk_fwd(*args, 1, 8, 2, 64, 16, 16, 64, 32, scale, 1, p, None) == 1
    assert "scale" in lib.q35_last_error_message().decode()


HUGE = 1 << 62


def test_sizes_whose_products_overflow_are_refused():
    """Nothing wraps to an accepted size, and no plan divides by a wrapped 0."""
    import ctypes
    from qwen3_5_vl_cuda_custom_b200 import _lib, build
    build.build()
    lib, p = _lib.load(), ctypes.c_void_p(256)  # never dereferenced: validation fails first
    st = (ctypes.c_int64 * 3)(1024, 512, 64)
    for B, Sq in ((1, HUGE), (4, HUGE), (2, 1 << 32), (HUGE, 4), (1 << 31, 1)):
        for Hq, Hkv in ((8, 1), (8, 2), (8, 8)):
            assert lib.q35_attn_q4_workspace(B, Hq, Hkv, Sq, 16, 64) == 0
            assert lib.q35_attn_q4_chunk_workspace(B, Hq, Hkv, Sq, 16, 64) == 0
            assert lib.q35_attn_q4_prefers_chunk(B, Hq, Hkv, Sq, 16, 64) == 0
            assert lib.q35_attn_q4_fwd(*[p] * 6, B, Hq, Hkv, Sq, 16, None, 16, 64, 32, 0.1, 0, p, None) == 2
            assert lib.q35_attn_q4_chunk_fwd(*[p] * 6, B, Hq, Hkv, Sq, 16, 16, 64, 32, 0.1, 0, p, None) == 2
    for B, S, offset in ((1, 4, (1 << 63) - 2), (HUGE, 4, 0), (1 << 60, 16, 0), (1, HUGE, 0), (1 << 31, 1, 0)):
        assert lib.q35_kv_append_q4(p, p, st, st, p, p, p, p, B, 2, S, 64, 32, 16, offset, None, None) == 2
        assert lib.q35_kv_read_q4(p, p, p, p, p, p, B, 2, S, S, 64, 32, 16, offset, None, None) == 2
    for out_cap in (HUGE, 1 << 31):
        assert lib.q35_kv_read_q4(p, p, p, p, p, p, 4, 2, 4, out_cap, 64, 32, 16, 0, None, None) == 2


@pytest.mark.parametrize("row", [-1, 17, 1 << 32, 1 << 64, (1 << 64) + 3, -(1 << 64)])
def test_rows_that_fit_no_cache_are_refused(monkeypatch, row):
    """A Python int beyond 64 bits must not reach the library as another number."""
    monkeypatch.setattr(K, "_cache_q4", lambda *a: (2, 1, 16, 32, 32))
    monkeypatch.setattr(K, "_strided_rows", lambda t, *a: (t, t.stride()))
    monkeypatch.setattr(K, "_stream", lambda t: None)
    monkeypatch.setattr(K.torch.cuda, "current_device", lambda: None)
    monkeypatch.setattr(K._lib, "call", lambda *a: None)
    cache = [torch.zeros(2, 1, 16, 16, dtype=torch.uint8)] * 4
    x = torch.zeros(2, 1, 1, 32, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        K.kv_append_q4(x, x, *cache, row)
    with pytest.raises(RuntimeError):
        K.kv_read_q4(*cache, row, 1)
