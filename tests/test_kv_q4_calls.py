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
