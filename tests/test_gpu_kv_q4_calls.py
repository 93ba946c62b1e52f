"""Calls of the 4-bit cache's operators that their documentation allows: strided
positions, scratch of any SM limit, memory that does not suffice, caches past their
capacity."""
import pytest
import torch

import kv_q4_ref as R
from test_gpu_kv_q4 import DEV, K, filled_cache, rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _ready():
    from qwen3_5_vl_cuda_custom_b200 import build
    build.build()
    yield
    K().device_error_check()


def test_strided_positions():
    """Positions that are one column of a table, in calls whose outputs are as small as
    the copy that is made of them."""
    B, Hkv, D, group = 2, 1, 32, 32
    cache, kk, vv = filled_cache(B, Hkv, 64, D, group, 151)
    table = torch.tensor([[9, 60], [9, 3]], dtype=torch.int32, device=DEV)
    for _ in range(50):
        k, v = K().kv_read_q4(*cache, table[:, 1], 1)
        for b, s in enumerate((60, 3)):
            assert torch.equal(k[b].cpu(), kk[b, :, s:s + 1].float().bfloat16())
            assert torch.equal(v[b].cpu(), vv[b, :, s:s + 1].float().bfloat16())
    x = rows((B, Hkv, 1, D), 152).to(DEV)
    other = [t.clone() for t in cache]
    K().kv_append_q4(x, x, *cache, table[:, 1])
    K().kv_append_q4(x, x, *other, table[:, 1].contiguous())
    q = rows((B, 2, 1, D), 153).to(DEV)
    out = K().attention_cache_q4(q, *cache, table[:, 1], 0.2, False)
    assert torch.equal(out, K().attention_cache_q4(q, *other, table[:, 1].contiguous(), 0.2, False))
    for a, b in zip(cache, other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


class Scratch:
    """`n` bytes of scratch with a margin behind them that must stay as it is."""

    def __init__(self, n, margin=1 << 24):
        self.n = n
        self.t = torch.full((n + margin,), 0xA5, dtype=torch.uint8, device=DEV)

    def whole(self):
        return bool((self.t[self.n:] == 0xA5).all())


@pytest.mark.parametrize("asked,launched", [(100, 0), (16, 0), (0, 100), (2, 130), (147, 148)])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,kv,D,group", [
    (64, 32, 4, 1, 2049, 128, 32), (1, 32, 4, 1, 9000, 128, 64), (3, 16, 2, 2, 5000, 64, 32),
    (2, 8, 2, 4, 777, 32, 32), (1, 8, 2, 40, 3000, 64, 64),
])
def test_scratch_suffices_whatever_the_sm_limits(monkeypatch, asked, launched, B, Hq, Hkv, Sq, kv, D, group):
    """Through the C interface: scratch sized under one limit, used under another (a
    margin behind it is larger than any plan's difference)."""
    from qwen3_5_vl_cuda_custom_b200 import _lib
    cap = -(-kv // 16) * 16
    cache = [torch.randint(0, 256, (B, Hkv, cap, D // 2), dtype=torch.uint8, device=DEV) if i % 2 == 0 else
             torch.rand(B, Hkv, cap, D // group, 2, device=DEV).bfloat16() for i in range(4)]
    q = rows((B, Hq, Sq, D), 155).to(DEV)
    lens = torch.full((B,), kv, dtype=torch.int32, device=DEV)
    outs = [torch.full((B, Sq, Hq * D), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(3)]
    stream = torch.cuda.current_stream().cuda_stream
    ptrs = [q.data_ptr()] + [t.data_ptr() for t in cache]
    try:
        _lib.call("q35_set_sm_limit", asked)
        size = _lib.query("q35_attn_q4_workspace", B, Hq, Hkv, Sq, kv, D)
        chunk_size = _lib.query("q35_attn_q4_chunk_workspace", B, Hq, Hkv, Sq, kv, D)
        _lib.call("q35_set_sm_limit", launched)
        assert size == _lib.query("q35_attn_q4_workspace", B, Hq, Hkv, Sq, kv, D)
        assert chunk_size == _lib.query("q35_attn_q4_chunk_workspace", B, Hq, Hkv, Sq, kv, D)
        scratch = [Scratch(4 * size), Scratch(4 * size), Scratch(chunk_size)]
        for i, p in enumerate((None, lens.data_ptr())):
            _lib.call("q35_attn_q4_fwd", *ptrs, outs[i].data_ptr(), B, Hq, Hkv, Sq, kv, p, cap, D, group, 0.1,
                      1, scratch[i].t.data_ptr(), stream)
        _lib.call("q35_attn_q4_chunk_fwd", *ptrs, outs[2].data_ptr(), B, Hq, Hkv, Sq, kv, cap, D, group, 0.1, 1,
                  scratch[2].t.data_ptr(), stream)
    finally:
        _lib.call("q35_set_sm_limit", 0)
    assert all(s.whole() for s in scratch)
    for out, chunk, n in ((outs[0], False, kv), (outs[1], False, lens), (outs[2], True, kv)):
        monkeypatch.setattr(K(), "_q4_chunk", lambda *a: chunk)
        assert torch.isfinite(out).all()
        assert torch.equal(out, K().attention_cache_q4(q, *cache, n, 0.1, True, kv))


def test_a_chunk_without_memory_for_its_copy_runs_on_the_codes(monkeypatch):
    B, Hq, Hkv, Sq, kv, D, group = 1, 16, 8, 40, 65536, 64, 64
    monkeypatch.setattr(K(), "_q4_chunk", lambda *a: True)
    cache, _, _ = filled_cache(B, Hkv, 1024, D, group, 157)
    cache = [t.repeat(1, 1, kv // 1024, *[1] * (t.dim() - 3)) for t in cache]
    q = rows((B, Hq, Sq, D), 158).to(DEV)
    monkeypatch.setattr(K(), "_q4_chunk", lambda *a: False)
    want = K().attention_cache_q4(q, *cache, kv, 0.125, True)
    monkeypatch.setattr(K(), "_q4_chunk", lambda *a: True)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    try:  # room for 64 MB more than what is held; the copy takes 268 MB
        torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (64 << 20)) / total)
        got = K().attention_cache_q4(q, *cache, kv, 0.125, True)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert torch.equal(got, want)
    assert not torch.equal(K().attention_cache_q4(q, *cache, kv, 0.125, True), want)  # the other form


@pytest.mark.parametrize("D,group", [(64, 32), (128, 128)])
def test_a_cache_with_lengths_ends_at_its_capacity(D, group):
    """250 rows asked for (256 are held): rows behind them are reported, and queries see
    the rows within the capacity only."""
    from qwen3_5_vl_cuda_custom_b200.kv_cache import Q4LayerKVCache
    B, Hq, Hkv, cap = 3, 4, 2, 250
    cache = Q4LayerKVCache(B, Hkv, cap, D, DEV, group_size=group)
    k, v = rows((B, Hkv, cap, D), 161).to(DEV), rows((B, Hkv, cap, D), 162).to(DEV)
    K().kv_append_q4(k, v, *cache.buffers, 0)
    cache.set_lengths(torch.tensor([249, 248, 3]))
    K().device_error_check()
    for step, over in enumerate((None, 0, 1)):
        q, x = rows((B, Hq, 1, D), 163 + step).to(DEV), rows((B, Hkv, 1, D), 173 + step).to(DEV)
        out = cache.append_attend(q, x, x, D ** -0.5, False)
        if over is None:
            K().device_error_check()
        else:
            with pytest.raises(RuntimeError, match="code 2"):
                K().device_error_check()
        lens = torch.tensor([min(n + step + 1, cap) for n in (249, 248, 3)], dtype=torch.int32, device=DEV)
        assert torch.equal(out, K().attention_cache_q4(q, *cache.buffers, lens, D ** -0.5, False, cap))
    K().device_error_check()
    assert cache.length == 252
    cache.reset()
    cache.set_lengths(torch.tensor([cap, cap - 1, 0]))
    assert cache.length == cap
