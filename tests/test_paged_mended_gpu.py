"""Operators over the paged cache and 4-bit products where calls once went wrong: caches made on side streams, page tables that name no page, scores and
activations at the ends of their range."""
import pytest
import torch

import paged_cases as pc

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


@pytest.mark.parametrize("dim,vdim", [(256, 256), (136, 64), (64, 200)])
def test_parts_without_keys_beside_long_sequences_with_wide_heads(ops, dim, vdim):
    """Keys are cut for the longest sequence: most parts of a short one have none, and write zeros where Q was on its way. Q's largest numbers stand in the rows
    that such a leftover would show."""
    new, ctx = [1, 2, 1, 3], [9000, 0, 70, 5]
    table, start, cx, n_pages = pc.layout(new, ctx, seed=6)
    g = torch.Generator(device="cuda").manual_seed(8)
    r = lambda *n: torch.randn(n, generator=g, device="cuda")
    k, v, q = r(n_pages, 1, 64, dim), r(n_pages, 1, vdim, 64), r(sum(new), 3, dim)
    q[3] *= 1e30                                                # the sequence behind 70: scores beyond any other, one key has all the weight
    args = (k, v, table.cuda(), start.cuda(), cx.cuda())
    want, far = pc.attention(q, k, v, table, start, cx, dim ** -0.5)
    first = ops.attn_packed(q, *args)
    for _ in range(20):
        got = ops.attn_packed(q, *args)
        assert torch.equal(got, first)
    rows = [0, 1, 2, 4, 5, 6]
    assert ((first.double() - want).abs() <= far)[rows].all()
    top = (q[3].double() @ pc.gather(k, v, table, 2, 0, 71)[0].T).argmax(-1)
    vals = pc.gather(k, v, table, 2, 0, 71)[1]
    assert torch.equal(first[3].view(3, vdim).double(), vals[top])
