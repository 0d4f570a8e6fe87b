"""Attention of a few rows over many keys in fp32: the 64-bit form, the plain 32-bit form, and what less precise forms would give.

A form is 32-bit arithmetic if its largest error is within 4 times the plain 32-bit form's on the same inputs and 2^-22 of the largest output. Scores: the plain form
rounds some dim sums of random sign, sqrt(dim) half steps together (11 at 128); a tensor core that cuts its sums once for 16 products loses dim / 16 half
steps (8). Outputs: it loses up to 4 half steps in the products with 64 keys, 2^-22 of the output, and the sums over pages are rounded in both."""
import math

import torch

F32 = torch.float32


def inputs(rows, keys, dim, vdim, mean, sharp, seed, device="cpu"):
    """q [rows,dim], k [keys,dim], v [keys,vdim] fp32; v around `mean`; sharp: scores that leave weight to a few keys."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *n: torch.randn(n, generator=g)
    return [t.to(device) for t in (r(rows, dim) * (8.0 if sharp else 1.0), r(keys, dim), r(keys, vdim) + mean)]


def exact(q, k, v):
    return torch.softmax(q.double() @ k.double().T / math.sqrt(q.shape[1]), -1) @ v.double()


def plain(q, k, v):
    s = q @ k.T * (1.0 / math.sqrt(q.shape[1]))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return p @ v / p.sum(-1, keepdim=True)


def cut(x, n):
    """n bf16 numbers whose sum is nearest to x."""
    y, rest = [], x
    for _ in range(n):
        y.append(rest.bfloat16().float())
        rest = rest - y[-1]
    return y


def one_sum(q, k, v):
    """Outputs summed over all keys in one fp32 sum, six products of bf16 parts for each 16 keys of a page, that is cut, not rounded, behind every one."""
    s = q.double() @ k.double().T / math.sqrt(q.shape[1])
    p = torch.exp(s - s.amax(-1, keepdim=True)).float()
    pp, vp = [x.double() for x in cut(p, 3)], [x.double() for x in cut(v, 3)]
    o = torch.zeros((q.shape[0], v.shape[1]), dtype=torch.float64)
    for page in range(0, k.shape[0], 64):
        for a, b in ((0, 2), (2, 0), (1, 1), (0, 1), (1, 0), (0, 0)):
            for j in range(page, min(page + 64, k.shape[0]), 16):
                o = o + pp[a][:, j:j + 16] @ vp[b][j:j + 16]
                step = torch.exp2(torch.floor(torch.log2(o.abs().clamp(min=1e-300))) - 23)
                o = torch.trunc(o / step) * step
    return (o / p.double().sum(-1, keepdim=True)).float()


def within(got, q, k, v):
    """Whether `got` is 32-bit arithmetic, and its error over the bound."""
    want = exact(q, k, v)
    bound = 4 * (plain(q, k, v).double() - want).abs().max().item() + 2.0 ** -22 * want.abs().max().item()
    over = (got.double() - want).abs().max().item() / bound
    return over <= 1.0, over


def linear_within(got, x, w):
    """The same for products got = x w^T of fp32 x with weights w in 64 bits; the plain form has the weights in fp32. A tensor core cuts the large sum of a group 8
    times at most, by half a step, 2^-24 of a sum that is half grown on average: 2^-22 of the largest result is granted."""
    want = x.double() @ w.T
    bound = 4 * ((x @ w.float().T).double() - want).abs().max().item() + 2.0 ** -22 * want.abs().max().item()
    over = (got.double() - want).abs().max().item() / bound
    return over <= 1.0, over
