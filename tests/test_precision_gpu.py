"""fp32 attention over the paged cache against the plain 32-bit form's own error, over contexts up to 80,000 keys: the 32-bit mode does 32-bit arithmetic."""
import pytest
import torch

import precision_cases as pc

pytestmark = pytest.mark.gpu
F32 = torch.float32


@pytest.fixture(scope="module")
def ops():
    from flexllm_b200 import build, ops
    build.build()
    return ops


@pytest.mark.parametrize("keys", [30, 1000, 10000, 80000])
@pytest.mark.parametrize("dim,vdim", [(64, 64), (128, 128), (80, 72), (256, 256)])
@pytest.mark.parametrize("mean,sharp", [(0.0, False), (1.0, False), (1.0, True)], ids=["centred", "offset", "sharp"])
def test_keys_cut_over_the_device(ops, keys, dim, vdim, mean, sharp):
    rows = 6                                                    # query heads of one token, one key/value head
    q, k, v = pc.inputs(rows, keys, dim, vdim, mean, sharp, seed=keys + dim, device="cuda")
    check(ops, q[None], k[:, None], v[:, None], [0])


@pytest.mark.parametrize("dim,vdim", [(64, 64), (128, 128), (96, 40), (200, 64), (136, 136)])
@pytest.mark.parametrize("keys,mean,sharp", [(1000, 1.0, False), (10000, 1.0, False), (10000, 1.0, True), (10000, 0.0, False)])
def test_keys_of_many_heads_in_one_part(ops, dim, vdim, keys, mean, sharp):
    """More heads than SMs: nobody cuts their keys."""
    G = 160
    g = torch.Generator(device="cuda").manual_seed(keys + dim)
    r = lambda *n: torch.randn(n, generator=g, device="cuda")
    check(ops, r(1, G, dim) * (8.0 if sharp else 1.0), r(keys, G, dim), r(keys, G, vdim) + mean, [0, 77, 159])


def check(ops, q, k, v, heads):
    """One token's heads q [1,H,dim] over k, v [keys,G,..]: the heads of the groups `heads` against the bound."""
    keys, G, dim = k.shape
    vdim, R, pages = v.shape[2], q.shape[1] // G, (keys + 63) // 64
    kp, vp = torch.zeros((pages * 64, G, dim), device="cuda"), torch.zeros((pages * 64, G, vdim), device="cuda")
    kp[:keys], vp[:keys] = k, v
    kp, vp = kp.view(pages, 64, G, dim).transpose(1, 2).contiguous(), vp.view(pages, 64, G, vdim).permute(0, 2, 3, 1).contiguous()
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    packed = ops.attn_packed(q, kp, vp, table, i32(0, 1), i32(keys - 1)).view(-1, vdim)
    tree = ops.attn_tree(q, torch.ones(1, dtype=torch.int64, device="cuda"), kp, vp, table, i32(0, 1), i32(keys - 1)).view(-1, vdim)
    for out in (packed, tree):
        for g in heads:
            ok, over = pc.within(out[g * R:(g + 1) * R], q[0, g * R:(g + 1) * R], k[:, g], v[:, g])
            assert ok, (g, over)


@pytest.mark.parametrize("M", [1, 4, 8, 16, 64])
@pytest.mark.parametrize("K,group", [(256, 128), (2048, 128), (2048, 64), (2048, 32), (8192, 256)])
@pytest.mark.parametrize("mean", [0.0, 1.0], ids=["centred", "offset"])
def test_four_bit_products(ops, M, K, group, mean):
    N, g = 200, torch.Generator(device="cuda").manual_seed(M + K + group)
    x = torch.randn((M, K), generator=g, device="cuda") + mean
    q = torch.randint(0, 16, (N, K), generator=g, device="cuda", dtype=torch.uint8)
    scale = torch.rand((N, K // group), generator=g, device="cuda") + 0.1
    for z in (0, 8):
        zero = torch.full(scale.shape, z, dtype=torch.uint8, device="cuda")
        ok, over = pc.linear_within(ops.linear_w4(x, (q[:, 0::2] | q[:, 1::2] << 4).contiguous(), scale, zero=zero), x, (q.double() - z) * scale.double().repeat_interleave(group, 1))
        assert ok, (z, over)
