"""Operators over the paged cache and 4-bit products where calls once went wrong: caches made on side streams, page tables that name no page, scores and
activations at the ends of their range."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from flexllm_b200 import build, ops
    build.build()
    return ops


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_a_cache_made_on_a_side_stream_keeps_what_is_written_at_once(ops):
    """Pools of 4 GB each take about a millisecond to clear; the first writes come some microseconds behind their making."""
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        kv = ops.PagedKV(30000, [(8, 128, 128)], BF)
        kv.k[0][-1].fill_(1.0), kv.v[0][-1].fill_(2.0), kv.k[0][15000].fill_(3.0), kv.v[0][15000].fill_(4.0)
        plain = ops.KVCache(2, 30000, 8)
        assert not kv.k[0][0].any() and not kv.v[0][1].any()
    torch.cuda.synchronize()
    assert (kv.k[0][-1] == 1).all() and (kv.v[0][-1] == 2).all() and (kv.k[0][15000] == 3).all() and (kv.v[0][15000] == 4).all()
    assert not kv.k[0][:100].any() and not kv.v[0][-100:-1].any()
    kv.close(), plain.close()
