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
