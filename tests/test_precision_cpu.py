"""The bound of tests/test_precision_gpu.py tells 32-bit arithmetic from less."""
import pytest

import precision_cases as pc

CASES = [(4, 30, 64), (4, 1000, 128), (2, 10000, 64)]


@pytest.mark.parametrize("rows,keys,dim", CASES)
@pytest.mark.parametrize("mean", [0.0, 1.0])
@pytest.mark.parametrize("sharp", [False, True])
def test_bound_of_32_bit_attention(rows, keys, dim, mean, sharp):
    q, k, v = pc.inputs(rows, keys, dim, dim, mean, sharp, seed=keys)
    assert pc.within(pc.plain(q, k, v), q, k, v)[0]
    three = [sum(pc.cut(x, 3)) for x in (q, k, v)]
    assert all((a == b).all() for a, b in zip(three, (q, k, v)))                # three parts hold a number
    low = [x.bfloat16().float() for x in (q, k, v)]
    assert not pc.within(pc.plain(*low), q, k, v)[0]                            # bf16 operands
    if sharp:                                                                   # (many alike weights average the error of two parts away)
        assert not pc.within(pc.plain(*[sum(pc.cut(x, 2)) for x in (q, k, v)]), q, k, v)[0]
    if mean and not sharp and keys >= 1000:                                     # one long sum that is cut
        assert not pc.within(pc.one_sum(q, k, v), q, k, v)[0]


@pytest.mark.parametrize("M,K", [(1, 256), (4, 2048), (16, 8192)])
@pytest.mark.parametrize("mean", [0.0, 1.0])
def test_bound_of_32_bit_products(M, K, mean):
    import torch
    g = torch.Generator().manual_seed(K)
    x = torch.randn((M, K), generator=g) + mean
    w = torch.randint(-8, 8, (100, K), generator=g).double() * (torch.rand((100, 1), generator=g) + 0.1).double()
    assert pc.linear_within(x @ w.float().T, x, w)[0]
    for n in (1, 2) if K <= 2048 else (1,):                     # bf16 activations, activations of two parts (whose errors thousands of terms average away)
        assert not pc.linear_within((sum(pc.cut(x, n)).double() @ w.T).float(), x, w)[0]
