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


SEQUENCES = [([1], [3000]), ([40, 3], [90, 0]), ([1] * 9, [700] * 9), ([300, 500], [0, 64])]


def pages(k, v, new, ctx, seed=0):
    """k [keys,G,dim] and v [keys,G,vdim] of all sequences, one behind the other, as pages; table, start, ctx."""
    table, start, cx, n_pages = pc.layout(new, ctx, seed)
    kp = torch.zeros((n_pages, 64) + k.shape[1:], dtype=k.dtype, device="cuda")
    vp = torch.zeros((n_pages, 64) + v.shape[1:], dtype=v.dtype, device="cuda")
    at = 0
    for b, (n, c) in enumerate(zip(new, ctx)):
        for p in range((n + c + 63) // 64):
            m = min(64, n + c - 64 * p)
            kp[table[b, p], :m], vp[table[b, p], :m] = k[at:at + m], v[at:at + m]
            at += m
    return kp.transpose(1, 2).contiguous(), vp.permute(0, 2, 3, 1).contiguous(), table.cuda(), start.cuda(), cx.cuda()


def means(v, new, ctx, H, tree):
    """The mean of the values that each row sees, in 64 bits; of a tree the cached ones and the row itself."""
    out, at = [], 0
    for n, c in zip(new, ctx):
        for i in range(n):
            seen = torch.cat([v[at:at + c], v[at + c + i:at + c + i + 1]]) if tree else v[at:at + c + i + 1]
            out.append(seen.double().mean(0).repeat_interleave(H // v.shape[1], 0).reshape(-1))
        at += n + c
    return torch.stack(out)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new,ctx", SEQUENCES, ids=lambda v: "%d.%s" % (len(v), v[0]))
def test_finite_scores_below_every_start_of_a_maximum(ops, dtype, dim, new, ctx):
    """Scores of -7e31 and more: all alike, so that a row is the mean of the values it sees; and one of them higher, which has all the weight. Weights are
    one: the sums of up to 3001 values are off by as many half steps of 2^-24, a result by its rounding."""
    H, G, keys = 4, 2, sum(new) + sum(ctx)
    g = torch.Generator(device="cuda").manual_seed(dim)
    v = torch.randn((keys, G, dim), generator=g, device="cuda").to(dtype)
    k = torch.full((keys, G, dim), -3e15, device="cuda").to(dtype)
    q = torch.full((sum(new), H, dim), 3e15, device="cuda").to(dtype)
    eye = torch.cat([1 << torch.arange(min(n, 63), dtype=torch.int64) for n in new]).cuda() if max(new) < 63 else None
    for tree in (False, True):
        if tree and eye is None:
            continue
        args = pages(k, v, new, ctx)
        got = ops.attn_tree(q, eye, *args) if tree else ops.attn_packed(q, *args)
        want = means(v, new, ctx, H, tree)
        far = max(n + c for n, c in zip(new, ctx)) * 2.0 ** -24 * v.double().abs().amax() + (want.abs() * 2.0 ** -8 if dtype == BF else 0)
        assert ((got.double() - want).abs() <= far).all(), (got.double() - want).abs().max()
    up = k.clone()
    up[0] = torch.tensor(-2e15).to(dtype)                       # the first key of the first sequence
    got = ops.attn_packed(q[:new[0]], *pages(up[:new[0] + ctx[0]], v[:new[0] + ctx[0]], new[:1], ctx[:1]))
    assert torch.equal(got, v[0].repeat_interleave(H // G, 0).reshape(1, -1).expand_as(got))


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
def test_rows_that_see_nothing_stay_zero(ops, dtype):
    v = torch.randn((50, 2, 64), device="cuda").to(dtype)
    q = torch.full((50, 4, 64), 3e15, device="cuda").to(dtype)
    mask = torch.zeros(50, dtype=torch.int64, device="cuda")
    mask[7] = 1 << 3
    got = ops.attn_tree(q, mask, *pages(torch.full_like(v, -3e15), v, [50], [0]))
    assert torch.equal(got[7], v[3].repeat_interleave(2, 0).reshape(-1)) and not got[:7].any() and not got[8:].any()


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("scale", [0.0, 1e-38, 1e-44])
def test_scales_that_leave_all_weights_alike(ops, dtype, dim, scale):
    """Products of q and k from -1e38 to 1e38: a scale of 0 makes them alike, and one of 1e-38 is no other."""
    new, ctx = [70, 2], [30, 500]
    g = torch.Generator(device="cuda").manual_seed(dim)
    keys = sum(new) + sum(ctx)
    v = torch.randn((keys, 2, dim), generator=g, device="cuda").to(dtype)
    size = torch.linspace(-1.0, 1.0, keys, device="cuda")[torch.randperm(keys, generator=g, device="cuda")]
    k = (size[:, None, None] * (1e19 / dim)).expand(keys, 2, dim).to(dtype)
    q = torch.full((72, 4, dim), 1e19, device="cuda").to(dtype)
    args = pages(k, v, new, ctx)
    got = ops.attn_packed(q, *args, scale=scale)
    want, far = pc.attention(q, args[0], args[1], args[2].cpu(), args[3].cpu(), args[4].cpu(), scale)
    assert ((got.double() - want).abs() <= far).all(), ((got.double() - want).abs() / far).max()


def status():
    from flexllm_b200 import lib
    return lib().flexllm_device_status()


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("bad", [-1, 6, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_nothing_is_appended_where_the_table_names_no_page(ops, dtype, bad, many):
    """Positions 60 .. 79 of a sequence whose second page is bad: the first four are written, nothing else is, page 0 least of all."""
    H, G, dim, n = 4, 2, 64, 20
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)
    k, v, proj = r(6, G, 64, dim), r(6, G, dim, 64), r(n + 3, (H + 2 * G) * dim)
    table, cu, ctx = [[5, bad], [2, 4]], [0, n, n + 3], [60, 62]
    if many:                                                    # sequences that are searched, not looked through
        table, cu, ctx = table + [[1, 1]] * 80, cu + [n + 3] * 80, ctx + [0] * 80
    cos, sin = torch.ones((1, 32), device="cuda"), torch.zeros((1, 32), device="cuda")
    k1, v1, x = k.clone(), v.clone(), proj.view(n + 3, -1, dim)
    k1[5, :, 60:], v1[5, :, :, 60:] = x[:4, H:H + G].transpose(0, 1), x[:4, H + G:].permute(1, 2, 0)
    for i, (page, slot) in enumerate([(2, 62), (2, 63), (4, 0)]):
        k1[page, :, slot], v1[page, :, :, slot] = x[n + i, H:H + G], x[n + i, H + G:]
    assert status() == 0
    q = ops.qk_norm_rope(proj, H, torch.zeros(n + 3, dtype=torch.int32, device="cuda"), cos, sin, k, v, torch.tensor(table, dtype=torch.int32, device="cuda"), i32(*cu), i32(*ctx))
    assert status() == -7
    assert torch.equal(k, k1) and torch.equal(v, v1) and torch.equal(q.view(n + 3, H, dim), x[:, :H])


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("bad", [-1, 6, 2 ** 31 - 1])
def test_no_entry_moves_from_or_to_a_page_that_the_table_does_not_name(ops, dtype, bad):
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)
    layers = [(r(6, 2, 64, 64), r(6, 2, 64, 64)) for _ in range(3)]
    table = torch.tensor([[3, bad], [bad, 4], [1, 5]], dtype=torch.int32, device="cuda")
    # positions 60 + keep: over the border from the bad page, over it to the bad page and within the good one, good
    ctx, keep, count = i32(60, 60, 60), torch.tensor([[2, 9], [7, 1], [9, 8]], dtype=torch.int32, device="cuda"), i32(2, 2, 2)
    want = [(k.clone(), v.clone()) for k, v in layers]
    for (k, v), (k0, v0) in zip(layers, want):
        k0[3, :, 60], v0[3, :, :, 60] = k[3, :, 62], v[3, :, :, 62]             # 62 to 60; 69 is on the bad page
        for i, s in enumerate((69, 68)):
            k0[1, :, 60 + i], v0[1, :, :, 60 + i] = k[5, :, s - 64], v[5, :, :, s - 64]
    assert status() == 0
    ops.kv_keep(layers, table, ctx, keep, count)
    assert status() == -7
    for (k, v), (k0, v0) in zip(layers, want):
        assert torch.equal(k, k0) and torch.equal(v, v0)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("cu,ctx,sound", [((0, 10, 23), (-1, 3), (1,)), ((0, 10, 23), (119, 3), (1,)), ((0, 10, 23), (5, 2 ** 31 - 1), (0,)), ((0, 10, 400), (5, 3), (0,)),
                                          ((-3, 10, 23), (5, 3), (1,)), ((0, 30, 20), (5, 3), ()), ((0, 10, 5), (5, 3), (0,))], ids=str)
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_nothing_is_appended_for_a_sequence_whose_values_are_out_of_range(ops, dtype, cu, ctx, sound, many):
    """Contexts before the first position and behind the last one (128 positions), row starts that leave the 23 rows or fall: the other sequence is appended,
    nothing of the bad one is, not even at clamped positions."""
    H, G, dim, T = 4, 2, 64, 23
    g = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)
    k, v, proj = r(5, G, 64, dim), r(5, G, dim, 64), r(T, (H + 2 * G) * dim)
    table = [[1, 2], [3, 4]]
    k0, v0, k1, v1, x = k.clone(), v.clone(), k.clone(), v.clone(), proj.view(T, -1, dim)
    for b in sound:
        for t in range(cu[b], cu[b + 1]):
            at = ctx[b] + t - cu[b]
            k1[table[b][at // 64], :, at % 64], v1[table[b][at // 64], :, :, at % 64] = x[t, H:H + G], x[t, H + G:]
    if many:
        table, ctx, cu = table + [[1, 2]] * 70, list(ctx) + [0] * 70, list(cu) + [cu[2]] * 70
    cos, sin = torch.ones((1, 32), device="cuda"), torch.zeros((1, 32), device="cuda")
    assert status() == 0
    ops.qk_norm_rope(proj, H, torch.zeros(T, dtype=torch.int32, device="cuda"), cos, sin, k, v, torch.tensor(table, dtype=torch.int32, device="cuda"), i32(*cu), i32(*ctx))
    assert status() == -7
    if min(b - a for a, b in zip(cu, cu[1:])) < 0:              # where starts fall, two sequences claim a row: it may be left out
        k1, v1 = torch.where(k == k0, k0, k1), torch.where(v == v0, v0, v1)
    assert torch.equal(k, k1) and torch.equal(v, v1)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,N,K,group", [(1, 300, 512, 128), (2, 300, 512, 64), (8, 300, 512, 32), (3, 40, 480, 96), (30, 300, 512, 128), (64, 300, 512, 64), (100, 300, 512, 32), (3, 40, 8192, 256)])
def test_zero_points_of_more_than_four_bits_are_reported(ops, dtype, M, N, K, group):
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn((M, K), generator=g, device="cuda").to(dtype)
    w = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scale = (torch.rand((N, K // group), generator=g, device="cuda") + 0.1).to(BF)
    zero = torch.randint(0, 16, scale.shape, generator=g, device="cuda", dtype=torch.uint8)
    assert status() == 0
    want = ops.linear_w4(x, w, scale, zero=zero)
    assert status() == 0
    for n, k, add in ((N - 1, 0, 16), (0, K // group - 1, 128), (N // 2, (K // group) // 2, 240)):
        bad = zero.clone()
        bad[n, k] += add
        got = ops.linear_w4(x, w, scale, zero=bad)
        assert status() == -7, (n, k)
        assert torch.equal(got, want)                           # the upper bits count for nothing
    ops.linear_w4(x, w, scale)
    assert status() == 0


@pytest.mark.parametrize("M,N,K,group", [(1, 70, 256, 128), (4, 70, 128, 32), (20, 140, 256, 64), (3, 40, 4096, 128)])
def test_activations_at_the_ends_of_32_bits(ops, M, N, K, group):
    """fp32 activations up to the largest number, weights of -1, 0 and 1 and scales of 2^-60: every product and sum is in range. The error is that of sums in
    fp32 (paged_cases.linear_w4); a row with one number is exact."""
    g = torch.Generator(device="cuda").manual_seed(K)
    big = torch.finfo(F32).max
    q = torch.randint(7, 10, (N, K), generator=g, device="cuda", dtype=torch.uint8)
    w = (q[:, 0::2] | q[:, 1::2] << 4).contiguous()
    scale = torch.full((N, K // group), 2.0 ** -60, device="cuda")
    for value in (big, -big, 3.39e38, -3.395e38, 3.0e38, 2.99e38, 1e-30, 2.0 ** -100):
        x = torch.zeros((M, K), device="cuda")
        at = torch.randint(0, K, (M,), generator=g, device="cuda")
        x[torch.arange(M), at] = value
        want = (q.double() - 8)[:, at].T * x.double().amax(1, keepdim=True).where(torch.tensor(value > 0), x.double().amin(1, keepdim=True)) * 2.0 ** -60
        got = ops.linear_w4(x, w, scale)
        assert torch.equal(got, want.float()), value            # (1e-30 2^-60 is below half the smallest fp32 number)
    x = torch.randn((M, K), generator=g, device="cuda") * 2.0 ** 110
    want, far = pc.linear_w4(x, w, scale, None)
    assert ((ops.linear_w4(x, w, scale).double() - want).abs() <= far).all()
    for value in (float("inf"), -float("inf"), float("nan")):
        x[0, 5] = value
        got = ops.linear_w4(x, w, scale)
        odd = q[:, 5] != 8
        assert not torch.isfinite(got[0][odd]).any() and (torch.isnan(got[0]) if value != value else torch.isinf(got[0]) | torch.isnan(got[0])).all()
        assert torch.isfinite(got[1:]).all()
        if value == value:
            assert torch.equal(got[0][odd], (q[:, 5][odd].float() - 8) * value)
