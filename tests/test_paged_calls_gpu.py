"""The operators over packed sequences as a program calls them: together, in graphs, on several streams, through both Python paths, with device data out of range."""
import math

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


class Layer:
    """One attention block of a model with 4-bit weights over a cache of the library's."""

    def __init__(self, ops, dtype, H=8, G=2, dim=64, width=256, n_pages=9, seed=0):
        self.ops, self.dtype, self.H, self.G, self.dim = ops, dtype, H, G, dim
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.kv = ops.PagedKV(n_pages, [(G, dim, dim)], dtype)
        rnd = lambda n, k: torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        n = (H + 2 * G) * dim
        self.w_in, self.s_in = rnd(n, width), torch.rand((n, width // 64), generator=g, device="cuda") * 0.02 + 0.005
        self.w_out, self.s_out = rnd(width, H * dim), (torch.rand((width, H * dim // 32), generator=g, device="cuda") * 0.02 + 0.005).to(BF)
        self.gain = torch.rand(dim, generator=g, device="cuda") + 0.5
        angle = torch.arange(600, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64, device="cuda") / (dim // 2))
        self.cos, self.sin = angle.cos().float(), angle.sin().float()

    def __call__(self, x, pos, table, cu, ctx, mask=None):
        o = self.ops
        proj = o.linear_w4(x, self.w_in, self.s_in)
        q = o.qk_norm_rope(proj, self.H, pos, self.cos, self.sin, self.kv.k[0], self.kv.v[0], table, cu, ctx, q_gain=self.gain, k_gain=self.gain)
        q = q.view(-1, self.H, self.dim)
        a = o.attn_packed(q, self.kv.k[0], self.kv.v[0], table, cu, ctx) if mask is None else o.attn_tree(q, mask, self.kv.k[0], self.kv.v[0], table, cu, ctx)
        return o.linear_w4(a, self.w_out, self.s_out), a, q, proj


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
def test_drafted_trees_and_their_accepted_paths_leave_what_a_prompt_leaves(ops, dtype):
    """Two sequences, once as prompts; once a part of each as a prompt, then a tree of drafted tokens whose accepted path is the rest. The cache is the same to
    the bit, and so are projections and queries; outputs agree within attention's rounding."""
    lens, part, path = [150, 75], [100, 64], [[0, 2, 5, 6], [1, 3]]
    g = torch.Generator(device="cuda").manual_seed(5)
    words = [torch.randn((n, 256), generator=g, device="cuda").to(dtype) for n in lens]
    table = torch.tensor([[4, 0, 7], [2, 8, -1]], dtype=torch.int32, device="cuda")

    whole = Layer(ops, dtype)
    n = [p + len(s) for p, s in zip(part, path)]
    cu, ctx = i32(0, n[0], n[0] + n[1]), i32(0, 0)
    pos = torch.cat([torch.arange(m, dtype=torch.int32) for m in n]).cuda()
    y, a, q, _ = whole(torch.cat([w[:m] for w, m in zip(words, n)]), pos, table, cu, ctx)

    drafted = Layer(ops, dtype)
    cu0 = i32(0, part[0], part[0] + part[1])
    pos0 = torch.cat([torch.arange(m, dtype=torch.int32) for m in part]).cuda()
    drafted(torch.cat([w[:m] for w, m in zip(words, part)]), pos0, table, cu0, ctx)
    # trees: the accepted tokens at the path's places, others beside them
    T = [9, 5]
    parent = [[-1, 0, 0, 1, 2, 2, 5, 4, 5], [-1, -1, 0, 1, 3]]
    x, mask, tpos = [], [], []
    for b in range(2):
        rows = torch.randn((T[b], 256), generator=g, device="cuda").to(dtype)
        rows[path[b]] = words[b][part[b]:n[b]]
        seen, depth = [], []
        for i, p in enumerate(parent[b]):
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
            depth.append(depth[p] + 1 if p >= 0 else 0)
        x.append(rows)
        mask += seen
        tpos += [part[b] + d for d in depth]
    cut, ctxt = i32(0, T[0], T[0] + T[1]), i32(*part)
    yt, at, qt, _ = drafted(torch.cat(x), i32(*tpos), table, cut, ctxt, torch.tensor(mask, device="cuda"))
    keep = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    for b in range(2):
        keep[b, :len(path[b])] = i32(*path[b])
    ops.kv_keep([(drafted.kv.k[0], drafted.kv.v[0])], table, ctxt, keep, i32(*[len(s) for s in path]))
    for b in range(2):
        for t in range(n[b]):
            page, slot = int(table[b, t // 64]), t % 64
            assert torch.equal(drafted.kv.k[0][page, :, slot], whole.kv.k[0][page, :, slot]), (b, t)
            assert torch.equal(drafted.kv.v[0][page, :, :, slot], whole.kv.v[0][page, :, :, slot]), (b, t)
    for b in range(2):
        rows_t = [sum(T[:b]) + i for i in path[b]]
        rows_w = [sum(n[:b]) + part[b] + i for i in range(len(path[b]))]
        assert torch.equal(qt[rows_t], q[rows_w])
        # both are within the bound of the same 64-bit result
        want, far = pc.attention(q, whole.kv.k[0], whole.kv.v[0], table.cpu(), cu.cpu(), ctx.cpu(), 64 ** -0.5)
        assert ((at[rows_t].double() - want[rows_w]).abs() <= far[rows_w]).all() and ((a[rows_w].double() - want[rows_w]).abs() <= far[rows_w]).all()
    # the next step goes on from the joined path
    nx = torch.cat([w[m:] for w, m in zip(words, n)])
    rest = [l - m for l, m in zip(lens, n)]
    cu2, ctx2 = i32(0, rest[0], sum(rest)), i32(*n)
    pos2 = torch.cat([torch.arange(m, l, dtype=torch.int32) for m, l in zip(n, lens)]).cuda()
    for p, r in zip(drafted(nx, pos2, table, cu2, ctx2), whole(nx, pos2, table, cu2, ctx2)):
        assert torch.equal(p, r)
    whole.kv.close(), drafted.kv.close()
    from flexllm_b200 import lib
    assert lib().flexllm_device_status() == 0


def calls(ops, dtype, seed=0, T=37):
    """One call of each operator: name -> (function of its inputs, inputs)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *n: torch.randn(n, generator=g, device="cuda").to(dtype)
    table, cu, ctx = torch.tensor([[3, 1, -1], [0, 2, 5]], dtype=torch.int32, device="cuda"), i32(0, 20, T), i32(70, 100)
    k, v = r(6, 2, 64, 64), r(6, 2, 64, 64)
    mask = pc.tree_masks([20, T - 20], seed).cuda()
    w = torch.randint(0, 256, (200, 64), generator=g, device="cuda", dtype=torch.uint8)
    s = (torch.rand((200, 2), generator=g, device="cuda") + 0.1).to(BF)
    z = torch.randint(0, 16, (200, 2), generator=g, device="cuda", dtype=torch.uint8)
    pos = torch.randint(0, 50, (T,), generator=g, device="cuda", dtype=torch.int32)
    cos, sin, gain = torch.rand((50, 32), generator=g, device="cuda"), torch.rand((50, 32), generator=g, device="cuda"), torch.rand(64, generator=g, device="cuda")
    keep, count = torch.tensor([[1, 4, 9], [0, 3, 5]], dtype=torch.int32, device="cuda"), i32(3, 2)

    def rope(x, kk, vv):
        return ops.qk_norm_rope(x, 8, pos, cos, sin, kk, vv, table, cu, ctx, q_gain=gain, k_gain=gain, eps=1e-5, sections=[32]), kk, vv

    def kept(kk, vv):
        a, b = kk.clone(), vv.clone()
        ops.kv_keep([(a, b)], table, ctx, keep, count)
        return a, b
    return {"packed": (lambda q, kk, vv: ops.attn_packed(q, kk, vv, table, cu, ctx), [r(T, 8, 64), k, v]),
            "tree": (lambda q, kk, vv: ops.attn_tree(q, mask, kk, vv, table, cu, ctx), [r(T, 8, 64), k, v]),
            "rope": (rope, [r(T, 12 * 64), k.clone(), v.clone()]),
            "keep": (kept, [k, v]),
            "w4": (lambda x: ops.linear_w4(x, w, s, zero=z), [r(5, 128)]),
            "w4 many": (lambda x: ops.linear_w4(x, w, s, zero=z), [r(70, 128)])}


def flat(v):
    return [t.clone() for t in (v if isinstance(v, tuple) else (v,))]


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
def test_the_same_in_graphs_on_streams_and_again(ops, dtype):
    for name, (f, x) in calls(ops, dtype).items():
        want = flat(f(*x))
        for p, q in zip(want, flat(f(*x))):
            assert torch.equal(p, q), name                              # no order of arrival in a result
        other = calls(ops, dtype, seed=9)[name][1]
        want2 = flat(f(*other))
        static = [t.clone() for t in x]
        graphs = []
        for _ in range(2):                                              # two graphs of the same call, replayed in turn
            side = torch.cuda.Stream()
            with torch.cuda.stream(side):
                f(*static)
                side.synchronize()
                graph = torch.cuda.CUDAGraph()
                graph.capture_begin()
                out = f(*static)
                graph.capture_end()
            graphs.append((graph, out))
        for inputs, result in ((x, want), (other, want2), (x, want)):
            for graph, out in graphs:
                for t, s in zip(static, inputs):
                    t.copy_(s)
                graph.replay()
                torch.cuda.synchronize()
                for p, q in zip(flat(out), result):
                    assert torch.equal(p, q), name
        # two streams at once, each behind its own copies
        streams, outs = [torch.cuda.Stream() for _ in range(2)], []
        torch.cuda.synchronize()
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                mine = [torch.empty_like(t) for t in x]
                for _ in range(6):
                    for t, src in zip(mine, x if n == 0 else other):
                        t.copy_(src)
                    outs.append((n, f(*mine), mine))
        torch.cuda.synchronize()
        for n, out, _ in outs[5::6]:
            for p, q in zip(flat(out), want if n == 0 else want2):
                assert torch.equal(p, q), name


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
def test_native_and_general_python_paths(ops, dtype, monkeypatch):
    assert ops._bind_front_end()
    native = {n: flat(f(*x)) for n, (f, x) in calls(ops, dtype).items()}
    monkeypatch.setattr(ops, "_front", False)
    monkeypatch.setattr(ops, "_bind_front_end", lambda: False)
    for n, (f, x) in calls(ops, dtype).items():
        for p, q in zip(native[n], flat(f(*x))):
            assert torch.equal(p, q) and p.dtype == q.dtype, n


def test_python_checks_on_the_device(ops):
    q, k, v = torch.zeros(3, 4, 64, device="cuda"), torch.zeros(2, 2, 64, 64, device="cuda"), torch.zeros(2, 2, 64, 64, device="cuda")
    t, cu, ctx = i32(0).view(1, 1), i32(0, 3), i32(0)
    ops.attn_packed(q, k, v, t, cu, ctx)
    mask = torch.ones(3, dtype=torch.int64, device="cuda")
    for bad in (lambda: ops.attn_packed(q.half(), k, v, t, cu, ctx), lambda: ops.attn_packed(q, k.bfloat16(), v, t, cu, ctx), lambda: ops.attn_packed(q, k, v, t.long(), cu, ctx),
                lambda: ops.attn_packed(q, k, v, t, cu[:1], ctx), lambda: ops.attn_packed(q, k, v, t, cu, i32(0, 0)), lambda: ops.attn_packed(q.transpose(1, 2), k, v, t, cu, ctx),
                lambda: ops.attn_packed(q[..., :32], k, v, t, cu, ctx), lambda: ops.attn_packed(q.cpu(), k, v, t, cu, ctx), lambda: ops.attn_packed(q, k[:, :, :32], v, t, cu, ctx),
                lambda: ops.attn_packed(q, k, v, t, cu, ctx, out=torch.zeros(2, 256, device="cuda")), lambda: ops.attn_tree(q, mask[:2], k, v, t, cu, ctx),
                lambda: ops.attn_tree(q, mask.int(), k, v, t, cu, ctx), lambda: ops.linear_w4(q[0], torch.zeros(8, 32, dtype=torch.uint8, device="cuda"), torch.zeros(8, 3, device="cuda")),
                lambda: ops.kv_keep([(k, v)], t, ctx, i32(0).view(1, 1), i32(0, 0)), lambda: ops.kv_keep([(k, v.cpu())], t, ctx, i32(0).view(1, 1), i32(0))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.attn_packed(q, k, v, t, cu, ctx, scale=-1.0), lambda: ops.attn_packed(q, k, v, t, cu, ctx, max_ctx=64),
                lambda: ops.linear_w4(q[0], torch.zeros(8, 32, dtype=torch.uint8, device="cuda"), torch.zeros(8, 4, device="cuda"))):      # groups of 16
        with pytest.raises(ops.FlexLLMError):
            bad()


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
def test_empty_calls_and_sequences_without_rows(ops, dtype):
    k, v = torch.zeros(2, 2, 64, 64, device="cuda", dtype=dtype), torch.zeros(2, 2, 64, 64, device="cuda", dtype=dtype)
    table, cu, ctx = i32(0, 1).view(2, 1), i32(0, 0, 0), i32(3, 0)
    assert ops.attn_packed(torch.zeros(0, 4, 64, device="cuda", dtype=dtype), k, v, table, cu, ctx).shape == (0, 256)
    assert ops.linear_w4(torch.zeros(0, 64, device="cuda", dtype=dtype), torch.zeros(8, 32, dtype=torch.uint8, device="cuda"), torch.zeros(8, 1, device="cuda")).shape == (0, 8)
    out = torch.full((5, 256), 3.0, device="cuda", dtype=dtype)
    ops.attn_packed(torch.zeros(5, 4, 64, device="cuda", dtype=dtype), k, v, table, cu, ctx, out=out)        # no sequence has a row
    assert (out == 3).all()
    q = ops.qk_norm_rope(torch.zeros(5, 512, device="cuda", dtype=dtype), 4, i32(-1, 2, 0, 99, 0), torch.zeros(2, 32, device="cuda"), torch.zeros(2, 32, device="cuda"), k, v, table, cu,
                         ctx, out=out[:, :256])
    assert q.data_ptr() == out.data_ptr() and (out == 3).all() and not k.any() and not v.any()
    ops.kv_keep([(k, v)], table, ctx, i32(0, 0).view(2, 1), i32(0, 0))
    from flexllm_b200 import lib
    assert lib().flexllm_device_status() == 0                   # positions of rows that are no sequence's do not matter


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
def test_device_data_out_of_range_is_clamped_and_reported(ops, dtype):
    """Row starts that fall or leave the rows, contexts and pages beyond what the call says, positions behind the tables, kept indices out of their range:
    every access stays inside (index by index in paged.cuh), the status says so, and the calls behind are right."""
    from flexllm_b200 import lib
    T, g = 40, torch.Generator(device="cuda").manual_seed(1)
    r = lambda *n: torch.randn(n, generator=g, device="cuda").to(dtype)
    q, k, v = r(T, 4, 64), r(5, 2, 64, 64), r(5, 2, 64, 64)
    good = (i32(1, 2, 3, 4).view(2, 2), i32(0, 20, 40), i32(5, 60))
    bad = [(i32(1, 2, 3, 99).view(2, 2), good[1], good[2]), (i32(1, -7, 3, 4).view(2, 2), good[1], i32(60, 60)), (good[0], i32(0, 30, 20), good[2]),
           (good[0], i32(0, 20, 400), good[2]), (good[0], i32(-3, 20, 40), good[2]), (good[0], good[1], i32(5, 5000)), (good[0], good[1], i32(-1, 5))]
    want = ops.attn_packed(q, k, v, *good)
    proj, cos = r(T, 512), torch.rand((10, 32), generator=g, device="cuda")
    pos = torch.zeros(T, dtype=torch.int32, device="cuda")
    assert lib().flexllm_device_status() == 0
    for table, cu, ctx in bad:
        ops.attn_packed(q, k, v, table, cu, ctx)
        assert lib().flexllm_device_status() == -7
        ops.attn_tree(q, torch.ones(T, dtype=torch.int64, device="cuda"), k, v, table, cu, ctx)
        assert lib().flexllm_device_status() == -7
        ops.qk_norm_rope(proj, 4, pos, cos, cos, k.clone(), v.clone(), table, cu, ctx)
        assert lib().flexllm_device_status() == -7
    ops.attn_tree(r(70, 4, 64), torch.ones(70, dtype=torch.int64, device="cuda"), k, v, i32(1, 2).view(1, 2), i32(0, 70), i32(0))      # more tokens than a mask has bits
    assert lib().flexllm_device_status() == -7
    for p in (10, -1):
        ops.qk_norm_rope(proj, 4, pos + p, cos, cos, k.clone(), v.clone(), *good)
        assert lib().flexllm_device_status() == -7
    for keep, count, ctx in ((64, 1, 5), (-1, 1, 5), (3, 9, 5), (3, -2, 5), (3, 1, 126), (3, 1, -4), (63, 1, 2 ** 31 - 1), (0, 1, 2 ** 31 - 1)):
        kk, vv = k.clone(), v.clone()
        ops.kv_keep([(kk, vv)], good[0][:1], i32(ctx), i32(keep).view(1, 1), i32(count))
        assert lib().flexllm_device_status() == -7
        if count == 1:
            assert torch.equal(kk, k) and torch.equal(vv, v)
    assert torch.equal(ops.attn_packed(q, k, v, *good), want)
    assert lib().flexllm_device_status() == 0


def test_long_cache_offsets(ops):
    """Pages whose elements lie beyond 2^31: the last pages of a pool of 2.6 G elements."""
    G, dim, n_pages = 8, 128, 40000
    k = torch.empty((n_pages, G, 64, dim), dtype=BF, device="cuda")
    v = torch.empty((n_pages, G, dim, 64), dtype=BF, device="cuda")
    new, ctx = [33, 1], [150, 60]
    table = torch.tensor([[n_pages - 1, n_pages - 3, 36000], [n_pages - 2, 0, 0]], dtype=torch.int32)
    g = torch.Generator(device="cuda").manual_seed(2)
    for p in set(table.flatten().tolist()):
        k[p] = torch.randn((G, 64, dim), generator=g, device="cuda")
        v[p] = torch.randn((G, dim, 64), generator=g, device="cuda")
    q = torch.randn((34, 16, dim), generator=g, device="cuda").to(BF)
    cu, cx = torch.tensor([0, 33, 34], dtype=torch.int32), torch.tensor(ctx, dtype=torch.int32)
    got = ops.attn_packed(q, k, v, table.cuda(), cu.cuda(), cx.cuda())
    want, far = pc.attention(q, k, v, table, cu, cx, dim ** -0.5)
    assert ((got.double() - want).abs() <= far).all()
    proj = torch.randn((34, (16 + 2 * G) * dim), generator=g, device="cuda").to(BF)
    pos, one = torch.zeros(34, dtype=torch.int32, device="cuda"), torch.ones((1, 64), device="cuda")
    ops.qk_norm_rope(proj, 16, pos, one, one * 0, k, v, table.cuda(), cu.cuda(), cx.cuda())
    x = proj.view(34, -1, dim)
    assert torch.equal(v[36000, :, :, 22], x[0, 16 + G:])
    assert torch.equal(k[36000, :, 22], x[0, 16:16 + G]) and torch.equal(k[n_pages - 2, :, 60], x[33, 16:16 + G])
    ops.kv_keep([(k, v)], table.cuda(), cx.cuda(), i32(5, 0).view(2, 1), i32(1, 0))
    assert torch.equal(k[36000, :, 22], x[5, 16:16 + G]) and torch.equal(v[36000, :, :, 22], x[5, 16 + G:])


def test_library_owned_pages(ops):
    kv = ops.PagedKV(3, [(2, 64, 64), (1, 128, 96)], F32)
    assert kv.k[1].shape == (3, 1, 64, 128) and kv.v[1].shape == (3, 1, 96, 64) and kv.k[0].dtype == F32 and not kv.k[0].any()
    kv.k[0][1, 0, 5] = 2.0
    assert kv.k[0][1, 0, 5].sum() == 128
    page = kv.k[1]
    kv.close()
    page.fill_(3.0)                                             # a view keeps the memory
    assert float(page.sum()) == 3.0 * page.numel()
    with pytest.raises(ValueError):
        ops.PagedKV(2, [(1, 64, 64)], torch.float16)
    kv = ops.PagedKV(2, [(1, 64, 64)])
    assert kv.k[0].dtype == BF and math.isfinite(float(kv.v[0].float().sum()))
    kv.close()


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("H,G,dim,new,ctx", [(8, 1, 128, [1], [30000]), (8, 1, 64, [33], [12000]), (8, 2, 128, [40, 7], [3000, 10]), (12, 3, 64, [5], [5000]), (4, 4, 128, [1, 1, 0, 1], [2500, 0, 90, 700]),
                                             (16, 8, 128, [9, 2], [1500, 1501]), (10, 5, 96, [17], [20000]), (8, 8, 64, [3, 3, 3], [640, 639, 0]), (3, 1, 256, [20], [9000])],
                         ids=lambda v: str(v).replace(" ", ""))
def test_keys_cut_into_any_number_of_parts(ops, dtype, H, G, dim, new, ctx):
    table, start, cx, n_pages = pc.layout(new, ctx, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *n: torch.randn(n, generator=g, device="cuda").to(dtype)
    k, v, q = r(n_pages, G, 64, dim), r(n_pages, G, dim, 64), r(sum(new), H, dim)
    mask = pc.tree_masks(new, 7)
    for m in (None, mask):
        args = (k, v, table.cuda(), start.cuda(), cx.cuda())
        got = ops.attn_packed(q, *args) if m is None else ops.attn_tree(q, m.cuda(), *args)
        want, far = pc.attention(q, k, v, table, start, cx, dim ** -0.5, m)
        assert ((got.double() - want).abs() <= far).all()


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,most,H,G", [(65, 1, 4, 2), (300, 3, 8, 2), (130, 70, 3, 1), (1500, 2, 2, 1)])
def test_many_sequences(ops, dtype, B, most, H, G):
    """More sequences than are looked through one by one: with and without rows, over pages that are begun, full and crossed."""
    g = torch.Generator().manual_seed(B)
    new = [int(x) for x in torch.randint(0, most + 1, (B,), generator=g)] if most > 1 else [1] * B
    ctx = [int(x) for x in torch.randint(0, 130, (B,), generator=g)]
    table, start, cx, n_pages = pc.layout(new, ctx, seed=1)
    T, dim = sum(new) + 3, 64                                           # three rows that are nobody's
    gd = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *n: torch.randn(n, generator=gd, device="cuda").to(dtype)
    k, v, proj = r(n_pages, G, 64, dim), r(n_pages, G, dim, 64), r(T, (H + 2 * G) * dim)
    one = torch.ones((1, dim // 2), device="cuda")
    args = (table.cuda(), start.cuda(), cx.cuda())
    k0, v0 = k.clone(), v.clone()
    q = ops.qk_norm_rope(proj, H, torch.zeros(T, dtype=torch.int32, device="cuda"), one, one * 0, k, v, *args)
    x = proj.view(T, -1, dim)
    assert torch.equal(q[:T - 3], x[:T - 3, :H].reshape(T - 3, -1))
    row = 0
    for b in range(B):
        for i in range(new[b]):
            page, slot = int(table[b, (ctx[b] + i) // 64]), (ctx[b] + i) % 64
            k0[page, :, slot], v0[page, :, :, slot] = x[row, H:H + G], x[row, H + G:]
            row += 1
    assert torch.equal(k, k0) and torch.equal(v, v0)
    out = torch.full((T, H * dim), 7.0, device="cuda", dtype=dtype)
    ops.attn_packed(q.view(T, H, dim), k, v, *args, out=out)
    want, far = pc.attention(q.view(T, H, dim), k, v, table, start, cx, dim ** -0.5)
    assert ((out.double() - want).abs() <= far)[:T - 3].all() and (out[T - 3:] == 7).all()
    from flexllm_b200 import lib
    assert lib().flexllm_device_status() == 0
    bad = start.clone()
    bad[B // 2] = T + 40                                                # a start behind the rows, then one that falls
    ops.attn_packed(q.view(T, H, dim), k, v, args[0], bad.cuda(), args[2])
    assert lib().flexllm_device_status() == -7


def test_captured_first_and_in_many_parts(ops):
    """A call in 16 parts, captured and replayed for another context than it was captured with."""
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = torch.randn((300, 1, 64, 128), generator=g, device="cuda").to(BF), torch.randn((300, 1, 128, 64), generator=g, device="cuda").to(BF)
    q = torch.randn((1, 8, 128), generator=g, device="cuda").to(BF)
    table, cu, ctx = torch.arange(300, device="cuda", dtype=torch.int32)[None].contiguous(), i32(0, 1), i32(19000)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = ops.attn_packed(q, k, v, table, cu, ctx)
    for c in (19000, 5, 12345, 0):
        ctx.fill_(c)
        graph.replay()
        want, far = pc.attention(q, k, v, table.cpu(), cu.cpu(), ctx.cpu(), 128 ** -0.5)
        assert ((y.double() - want).abs() <= far).all()
