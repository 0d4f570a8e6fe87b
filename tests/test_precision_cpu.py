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
