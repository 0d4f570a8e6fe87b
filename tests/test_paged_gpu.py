"""Operators over packed sequences and the floating-point paged cache, and products with 4-bit weights, against their 64-bit forms."""
import math
import random

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


def near(got, want, far, what=""):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    ok = torch.isfinite(want)
    over = ((got - want).abs()[ok] - far[ok]).max().item() if ok.any() else 0.0
    worst = ((got - want).abs()[ok] / far[ok].clamp(min=1e-300)).max().item() if ok.any() else 0.0
    assert over <= 0, (what, "error over its bound", worst)


def inputs(new, ctx, H, G, dim, vdim, dtype, seed=0, spare=2, width=None, poison=True):
    table, start, cx, n_pages = pc.layout(new, ctx, seed, spare, width)
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = torch.randn((n_pages, G, 64, dim), generator=g, device="cuda").to(dtype)
    v = torch.randn((n_pages, G, vdim, 64), generator=g, device="cuda").to(dtype)
    if poison:                       # what no sequence has written
        used = set(table.flatten().tolist())
        for p in range(n_pages):
            if p not in used:
                k[p], v[p] = math.nan, math.inf
        for b, (n, c) in enumerate(zip(new, ctx)):
            tail = (n + c) % 64
            if tail:
                k[table[b, (n + c) // 64], :, tail:], v[table[b, (n + c) // 64], :, :, tail:] = math.nan, math.nan
    q = torch.randn((sum(new), H, dim), generator=g, device="cuda").to(dtype)
    return q, k, v, table, start, cx


CASES = [
    # new tokens, context, heads, kv heads, dim, vdim
    ([1], [0], 1, 1, 64, 64),
    ([1], [1], 4, 2, 64, 64),
    ([3, 0, 64, 65, 1], [0, 5, 0, 63, 640], 8, 2, 64, 64),
    ([128], [0], 8, 8, 128, 128),
    ([129, 127], [0, 1], 32, 8, 128, 128),
    ([500, 1, 31], [0, 1000, 200], 10, 2, 96, 96),
    ([77], [3], 7, 1, 80, 80),
    ([40, 9], [100, 64], 6, 2, 256, 256),
    ([33, 2], [64, 61], 4, 4, 72, 200),
    ([20], [11], 40, 1, 64, 64),
    ([5, 6], [60, 130], 160, 1, 64, 128),
    ([700], [0], 4, 1, 8, 8),
    ([300, 260], [64, 0], 16, 2, 128, 64),
    ([1300, 77, 1100], [0, 65, 3], 16, 16, 128, 128),
    ([700, 0, 650], [100, 0, 0], 32, 8, 64, 64),
    ([2500], [0], 40, 8, 96, 80),
    ([300, 310], [0, 70], 32, 8, 64, 64),
    ([40, 1, 64, 33, 40, 40, 0, 17, 40, 40, 40], [0, 1, 500, 63, 64, 65, 3, 127, 128, 129, 130], 32, 8, 128, 128),
    ([1, 3000, 33], [700, 128, 1], 16, 8, 72, 128),
]


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "n%s-h%dx%d-d%d-%d" % ("_".join(map(str, c[0][:4])), c[2], c[3], c[4], c[5]))
def test_packed_attention(ops, case, dtype):
    new, ctx, H, G, dim, vdim = case
    q, k, v, table, start, cx = inputs(new, ctx, H, G, dim, vdim, dtype, seed=len(new) + dim)
    got = ops.attn_packed(q, k, v, table.cuda(), start.cuda(), cx.cuda())
    want, far = pc.attention(q, k, v, table, start, cx, dim ** -0.5)
    near(got, want, far)


TREES = [
    ([1], [0], 1, 1, 64, 64),
    ([1, 1, 1], [0, 63, 64], 8, 2, 128, 128),
    ([64, 17, 0, 1, 33], [0, 100, 9, 2000, 31], 8, 2, 64, 64),
    ([26], [1000], 32, 8, 64, 64),
    ([5, 63], [700, 1], 10, 2, 96, 96),
    ([30, 64], [3000, 64], 32, 8, 128, 128),
    ([16], [5000], 4, 4, 128, 128),
    ([i % 33 for i in range(40)], [(77 * i) % 400 for i in range(40)], 32, 8, 64, 64),
    ([1] * 70, [(77 * i) % 900 for i in range(70)], 32, 8, 128, 128),
    ([12, 3], [70, 10], 6, 1, 256, 256),
    ([3], [200], 136, 1, 64, 64),
]


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", TREES, ids=lambda c: "n%s-h%dx%d-d%d-%d" % ("_".join(map(str, c[0][:4])), c[2], c[3], c[4], c[5]))
def test_tree_attention(ops, case, dtype):
    new, ctx, H, G, dim, vdim = case
    q, k, v, table, start, cx = inputs(new, ctx, H, G, dim, vdim, dtype, seed=len(new) + dim)
    mask = pc.tree_masks(new, seed=dim)
    got = ops.attn_tree(q, mask.cuda(), k, v, table.cuda(), start.cuda(), cx.cuda())
    want, far = pc.attention(q, k, v, table, start, cx, dim ** -0.5, mask)
    near(got, want, far)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
def test_rows_that_see_nothing_and_bits_of_no_token(ops, dtype):
    new, ctx = [5, 64], [0, 70]
    q, k, v, table, start, cx = inputs(new, ctx, 4, 2, 64, 64, dtype)
    mask = torch.tensor([0, 1, -1, 1 << 40, 3] + [0] * 32 + [-1] * 32)      # bits of tokens that a sequence does not have count for nothing
    got = ops.attn_tree(q, mask.cuda(), k, v, table.cuda(), start.cuda(), cx.cuda())
    want, far = pc.attention(q, k, v, table, start, cx, 0.125, mask)
    assert not got[0].any() and not got[3].any()
    near(got, want, far)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_a_row_does_not_see_do_not_reach_it(ops, dtype, bad):
    new, ctx = [90, 40], [30, 0]
    q, k, v, table, start, cx = inputs(new, ctx, 8, 2, 64, 64, dtype)
    at = 30 + 50                                                            # token 50 of the first sequence
    k[table[0, at // 64], 0, at % 64] = bad
    v[table[0, at // 64], 1, :, at % 64] = bad
    got = ops.attn_packed(q, k, v, table.cuda(), start.cuda(), cx.cuda())
    want, far = pc.attention(q, k, v, table, start, cx, 0.125)
    assert torch.isfinite(got[:50]).all() and torch.isfinite(got[90:]).all()
    near(got[:50], want[:50], far[:50])
    near(got[90:], want[90:], far[90:])
    assert not torch.isfinite(got[50:90, 4 * 64:]).any()                    # group 1 sees the value
    new = [40, 20]
    q, k, v, table, start, cx = inputs(new, [30, 70], 8, 2, 64, 64, dtype)
    mask = torch.tensor([1 << i for i in range(40)] + [1 << i for i in range(20)])
    at = 30 + 7
    k[table[0, at // 64], 0, at % 64] = bad
    v[table[0, at // 64], 1, :, at % 64] = bad
    got = ops.attn_tree(q, mask.cuda(), k, v, table.cuda(), start.cuda(), cx.cuda())
    want, far = pc.attention(q, k, v, table, start, cx, 0.125, mask)
    others = [i for i in range(60) if i != 7]
    near(got[others], want[others], far[others])


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
def test_strides_scale_and_rows_behind_the_last_sequence(ops, dtype):
    new, ctx, H, G = [70, 30], [10, 100], 8, 4
    q, k, v, table, start, cx = inputs(new, ctx, H, G, 64, 64, dtype)
    wide = torch.randn((107, H * 64 + 48), device="cuda").to(dtype)
    wide[:100, 16:16 + H * 64] = q.reshape(100, -1)
    qs = wide[:, 16:16 + H * 64].unflatten(1, (H, 64))
    out = torch.full((107, H * 64 + 24), 7.0, device="cuda").to(dtype)
    for scale in (0.5, 0.0, 1.0):
        got = ops.attn_packed(qs, k, v, table.cuda(), start.cuda(), cx.cuda(), scale=scale, out=out[:, 8:8 + H * 64])
        want, far = pc.attention(q, k, v, table, start, cx, scale)
        near(got[:100], want, far)
        assert (got[100:] == 7).all() and (out[:, :8] == 7).all() and (out[:, 8 + H * 64:] == 7).all()


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
def test_large_scores_and_growing_maxima(ops, dtype):
    new, ctx = [200], [100]
    q, k, v, table, start, cx = inputs(new, ctx, 4, 2, 64, 64, dtype)
    for i in range(300):                                                    # keys grow along the sequence: the running maximum moves in every tile
        k[table[0, i // 64], :, i % 64] *= 0.05 * i
    got = ops.attn_packed(q, k, v, table.cuda(), start.cuda(), cx.cuda())
    want, far = pc.attention(q, k, v, table, start, cx, 0.125)
    near(got, want, far)


def rope_case(ops, new, ctx, H, G, dim, vdim, rot, sections, dtype, gains=True, seed=0):
    q, k, v, table, start, cx = inputs(new, ctx, H, G, dim, vdim, dtype, seed=seed, poison=False)
    T, half = sum(new), rot // 2
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    proj = torch.randn((T + 2, (H + G) * dim + G * vdim + 8), generator=g, device="cuda").to(dtype)[:T, 8:]
    proj = torch.empty_like(proj, memory_format=torch.contiguous_format).copy_(proj) if seed % 2 else proj
    angle = torch.randn((500, half), generator=g, device="cuda") * 3
    pos = torch.randint(0, 500, (len(sections), T), generator=g, device="cuda", dtype=torch.int32)
    qg = torch.rand(dim, generator=g, device="cuda") + 0.5 if gains else None
    kg = torch.rand(dim, generator=g, device="cuda") + 0.5 if gains else None
    args = (angle.cos(), angle.sin())
    want_q, want_k, want_v, far_q, far_k = pc.norm_rope(proj, H, G, dim, vdim, pos, *args, sections, qg, kg, 1e-6)
    k0, v0 = k.clone(), v.clone()
    got = ops.qk_norm_rope(proj, H, pos if len(sections) > 1 else pos[0], *args, k, v, table.cuda(), start.cuda(), cx.cuda(), q_gain=qg, k_gain=kg,
                           sections=sections)
    near(got, want_q.reshape(T, -1), far_q.reshape(T, -1), "q")
    for b in range(len(new)):
        for i in range(new[b]):
            t, at = int(start[b]) + i, int(cx[b]) + i
            page, slot = int(table[b, at // 64]), at % 64
            near(k[page, :, slot], want_k[t], far_k[t], "k")
            assert torch.equal(v[page, :, :, slot].double(), want_v[t])
            k0[page, :, slot], v0[page, :, :, slot] = k[page, :, slot], v[page, :, :, slot]
    assert torch.equal(k0, k) and torch.equal(v0, v)                        # nothing else was written


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", [
    ([1], [0], 1, 1, 8, 8, 8, [4]),
    ([1, 1, 1, 1], [5, 63, 64, 0], 32, 8, 128, 128, 128, [64]),
    ([70, 0, 3, 130], [0, 9, 62, 1], 8, 2, 64, 64, 64, [8, 12, 12]),
    ([9, 65], [63, 10], 6, 3, 96, 96, 96, [5, 20, 23]),
    ([40], [30], 5, 1, 80, 72, 32, [3, 13]),
    ([17], [120], 4, 2, 256, 200, 256, [1, 2, 3, 122]),
    ([12], [4], 3, 3, 64, 64, 0, [0]),
], ids=lambda c: "n%s-d%d-r%d-x%d" % ("_".join(map(str, c[0])), c[4], c[6], len(c[7])))
def test_norm_rotation_and_append(ops, case, dtype):
    rope_case(ops, *case, dtype)
    rope_case(ops, *case, dtype, gains=False, seed=1)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("G,dim,vdim,layers,most", [(8, 64, 64, 3, 6), (1, 128, 128, 1, 64), (3, 96, 40, 70, 5), (2, 256, 256, 2, 64), (2, 64, 64, 1, 1)])
def test_accepted_paths(ops, dtype, G, dim, vdim, layers, most):
    new, ctx = [64, 64, 64, 64, 64], [0, 10, 63, 64, 100]
    table, _, cx, n_pages = pc.layout(new, ctx)
    r = random.Random(G)
    count = [most, 0, min(5, most), most, r.randrange(0, most + 1)]
    keep = torch.full((5, most), 99, dtype=torch.int32)                      # behind count: not looked at
    for b, c in enumerate(count):
        path = sorted(r.sample(range(64), c)) if b % 2 == 0 else [r.randrange(64) for _ in range(c)]      # any order, the same one twice
        keep[b, :c] = torch.tensor(path, dtype=torch.int32)
    kv = [(torch.randn((n_pages, G, 64, dim), device="cuda").to(dtype), torch.randn((n_pages, G, vdim, 64), device="cuda").to(dtype)) for _ in range(layers)]
    old = [(k.clone(), v.clone()) for k, v in kv]
    ops.kv_keep(kv, table.cuda(), cx.cuda(), keep.cuda(), torch.tensor(count, dtype=torch.int32).cuda())
    for (k, v), (k0, v0) in zip(kv, old):
        wk, wv = k0.clone(), v0.clone()
        for b, c in enumerate(count):
            for i in range(c):
                s, d = ctx[b] + int(keep[b, i]), ctx[b] + i
                wk[table[b, d // 64], :, d % 64] = k0[table[b, s // 64], :, s % 64]
                wv[table[b, d // 64], :, :, d % 64] = v0[table[b, s // 64], :, :, s % 64]
        assert torch.equal(k, wk) and torch.equal(v, wv)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,N,K,group", [(1, 8, 32, 32), (1, 2048, 2048, 128), (3, 1000, 96, 32), (8, 16, 64, 64), (9, 257, 1024, 64), (17, 130, 384, 128),
                                         (33, 96, 512, 256), (64, 500, 2048, 32), (65, 72, 640, 128), (200, 64, 96, 96), (5, 40, 20000, 32), (64, 48, 9088, 64),
                                         (2, 24, 32768, 32768)])
def test_four_bit_products(ops, dtype, M, N, K, group):
    g = torch.Generator(device="cuda").manual_seed(M + N)
    for zeros in (False, True):
        x = torch.randn((M, K + 8), generator=g, device="cuda").to(dtype)[:, :K] if K % 8 == 0 else None
        w = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
        scale = (torch.rand((N, K // group), generator=g, device="cuda") + 0.1).to(BF if zeros else F32)
        zero = torch.randint(0, 16, scale.shape, generator=g, device="cuda", dtype=torch.uint8) if zeros else None
        bias = torch.randn(N, generator=g, device="cuda") if zeros else None
        want, far = pc.linear_w4(x, w, scale, zero, bias)
        near(ops.linear_w4(x, w, scale, zero=zero, bias=bias, out_f32=True), want, far)
        y = torch.full((M, N + 3), 5.0, device="cuda").to(dtype)
        near(ops.linear_w4(x, w, scale, zero=zero, bias=bias, out=y[:, 1:1 + N]), want, far + (want.abs() * 2.0 ** -8 if dtype == BF else 0))
        assert (y[:, 0] == 5).all() and (y[:, 1 + N:] == 5).all()
