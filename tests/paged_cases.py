"""Plain 64-bit forms of the operators over packed sequences and the paged cache, and inputs for them."""
import math
import random

import torch

PAGE = 64


def layout(new, ctx, seed=0, spare=2, width=None):
    """Page tables (entries behind a sequence's pages name none), row starts, contexts; CPU tensors and the number of pages."""
    used = [(n + c + PAGE - 1) // PAGE for n, c in zip(new, ctx)]
    width = max(max(used), 1) if width is None else width
    perm = torch.randperm(sum(used) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(new), width), -1, dtype=torch.int32)
    for b, u in enumerate(used):
        for i in range(u):
            table[b, i] = perm.pop()
    start = [sum(new[:b]) for b in range(len(new) + 1)]
    return table, torch.tensor(start, dtype=torch.int32), torch.tensor(ctx, dtype=torch.int32), sum(used) + spare


def gather(k, v, table, b, g, end):
    """Keys [end,dim] and values [end,vdim] of a sequence in 64 bits."""
    if end == 0:
        return k.new_zeros((0, k.shape[3]), dtype=torch.float64), v.new_zeros((0, v.shape[2]), dtype=torch.float64)
    ids = table[b, :(end + PAGE - 1) // PAGE].long().to(k.device)
    return k[ids, g].reshape(-1, k.shape[3])[:end].double(), v[ids, g].transpose(1, 2).reshape(-1, v.shape[2])[:end].double()


def attention(q, k, v, table, start, ctx, scale, mask=None):
    """[T,heads*vdim] in 64 bits, with the largest error of a kernel's output. A key that a row does not see takes no part; a row that sees none is zero.
    Largest error, with a = sum p |v| / sum p and s = the largest sum_d |q_d k_d| * scale of the row's keys: scores summed in fp32 are off by dim 2^-24 s,
    weights relatively as much and by four roundings of the exponential, numerator and denominator each, sums over the keys by keys 2^-24. bf16: weights
    are rounded to bf16 (2^-8 each) in the numerator, the output once (2^-8); a 20th more covers the products of these."""
    T, H, D = q.shape
    G, dv = k.shape[1], v.shape[2]
    out = torch.zeros((T, H, dv), dtype=torch.float64, device=q.device)
    far = torch.zeros_like(out)
    for b in range(len(ctx)):
        r0, r1, c = int(start[b]), int(start[b + 1]), int(ctx[b])
        n = r1 - r0
        if n == 0:
            continue
        for g in range(G):
            kk, vv = gather(k, v, table, b, g, c + n)
            see = torch.zeros((n, c + n), dtype=torch.bool)
            for i in range(n):
                if mask is None:
                    see[i, :c + i + 1] = True
                else:
                    see[i, :c] = True
                    m = int(mask[r0 + i]) & ((1 << 64) - 1)
                    for j in range(n):
                        see[i, c + j] = bool(m >> j & 1)
            see = see.to(q.device)
            for h in range(g * (H // G), (g + 1) * (H // G)):
                s = (q[r0:r1, h].double() @ kk.T * scale).masked_fill(~see, -math.inf)
                p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300)).masked_fill(~see, 0.0)
                total = p.sum(-1, keepdim=True)
                if bool(torch.isfinite(vv).all()):
                    o = p @ vv
                else:
                    o = torch.stack([p[i][see[i]] @ vv[see[i]] for i in range(n)])
                out[r0:r1, h] = torch.where(total > 0, o / total, torch.where(torch.isnan(total), total, 0.0))
                a = p.nan_to_num() @ vv.abs().nan_to_num() / total.clamp(min=1e-300)
                size = (q[r0:r1, h].double().abs() @ kk.abs().T * abs(scale)).masked_fill(~see, 0.0).amax(-1, keepdim=True)
                far[r0:r1, h] = a * 2.0 ** -24 * (2 * D * size + 2 * (c + n) + 16)
                if q.dtype == torch.bfloat16:
                    far[r0:r1, h] += 1.05 * 2.0 ** -8 * (a + out[r0:r1, h].abs())
    return out.reshape(T, H * dv), far.reshape(T, H * dv)


def norm_rope(proj, H, G, dim, vdim, pos, cos_t, sin_t, sections, q_gain, k_gain, eps):
    """q [T,H,dim], k [T,G,dim], v [T,G,vdim] in 64 bits, and the largest error of q and k: fp32 sums of dim squares, and a dozen roundings of the terms
    of a pair; in bf16 one rounding of the result."""
    T, half = proj.shape[0], cos_t.shape[1]
    x = proj.double()
    qk = x[:, :(H + G) * dim].reshape(T, H + G, dim).clone()
    for lo, hi, gain in ((0, H, q_gain), (H, H + G, k_gain)):
        if gain is not None:
            y = qk[:, lo:hi]
            qk[:, lo:hi] = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * gain.double()
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    turned = qk.clone()
    size = qk.abs()
    size[..., :half], size[..., half:2 * half] = size[..., :half] + size[..., half:2 * half], size[..., :half] + size[..., half:2 * half]
    for p in range(half):
        at = pos[axis[p]].long()
        c, s = cos_t[at, p].double()[:, None], sin_t[at, p].double()[:, None]
        turned[..., p] = qk[..., p] * c - qk[..., p + half] * s
        turned[..., p + half] = qk[..., p + half] * c + qk[..., p] * s
    far = size * 2.0 ** -24 * (dim + 12) + (turned.abs() * 2.0 ** -8 if proj.dtype == torch.bfloat16 else 0.0)
    return turned[:, :H], turned[:, H:], x[:, (H + G) * dim:].reshape(T, G, vdim), far[:, :H], far[:, H:]


def linear_w4(x, w, scale, zero, bias=None):
    """y in 64 bits and its largest error in fp32: sums of 16 products that may lose 2^-22 of the terms' size each, as many as a group and the groups have."""
    N, K = w.shape[0], w.shape[1] * 2
    q = torch.empty((N, K), dtype=torch.float64, device=w.device)
    q[:, 0::2], q[:, 1::2] = (w & 15).double(), (w >> 4).double()
    group = K // scale.shape[1]
    z = zero.double() if zero is not None else torch.full_like(scale, 8, dtype=torch.float64)
    W = (q - z.repeat_interleave(group, 1)) * scale.double().repeat_interleave(group, 1)
    y = x.double() @ W.T
    y = y if bias is None else y + bias.double()
    size = x.double().abs() @ W.abs().T + y.abs()
    return y, size * 2.0 ** -22 * (group / 16 + K // group + 8)


def tree_masks(new, seed=0):
    """Every token sees itself and its ancestors; parents come before their children."""
    r, masks = random.Random(seed), []
    for n in new:
        seen = []
        for i in range(n):
            parent = r.randrange(max(-1, i - 6), i)
            seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
        masks += seen
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64)
