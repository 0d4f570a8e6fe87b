"""The operators of a speculatively decoding, weight-quantised model over the paged floating-point cache: the cases they are measured at,
and their plain forms.

  rope    norm of q and k per head, rotation (positions of one or several axes), k and v into the pages     ops.qk_norm_rope
  packed  causal attention of packed sequences of different lengths over their pages                        ops.attn_packed
  tree    attention of drafted tokens, each seeing its context and its ancestors                            ops.attn_tree
  keep    the accepted path of every tree moved together in the pages, all layers at once                    ops.kv_keep
  w4      product with 4-bit weights, one scale and zero point per group                                    ops.linear_w4

Pages hold 64 tokens: K [page][kv head][token][dim], V transposed [page][kv head][vdim][token]. Sequence b has the packed rows
cu[b] .. cu[b+1] - 1 at cache positions ctx[b] .."""
import math
import random

import torch

own = False
PAGE = 64
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one new token for each of 32 running sequences: the smallest call of every decode step, where latency counts
        {"name": "rope decode 32", "op": "rope", "type": "bf16", "seqs": 32, "tokens": 32, "ctx": 2000, "heads": 32, "kv": 8, "dim": 128, "axes": 1, "mix": 1},
        # prompts of images and video (time, height, width): 16 thousand rows in four sequences
        {"name": "rope video 16384", "op": "rope", "type": "bf16", "seqs": 4, "tokens": 16384, "ctx": 100, "heads": 16, "kv": 8, "dim": 128, "axes": 3, "mix": 2},
        # a serving step that admits eight short prompts, one of them empty
        {"name": "packed short 8", "op": "packed", "type": "bf16", "seqs": 8, "tokens": 1001, "ctx": 0, "heads": 32, "kv": 8, "dim": 64, "mix": 3},
        # two long prompts from their first token
        {"name": "packed long 2", "op": "packed", "type": "bf16", "seqs": 2, "tokens": 12291, "ctx": 0, "heads": 32, "kv": 8, "dim": 128, "mix": 4},
        # the 32-bit mode, a later portion of three prompts
        {"name": "packed f32 3", "op": "packed", "type": "f32", "seqs": 3, "tokens": 1150, "ctx": 700, "heads": 8, "kv": 2, "dim": 64, "mix": 5},
        # one user, a tree of 26 drafted tokens
        {"name": "tree one", "op": "tree", "type": "bf16", "seqs": 1, "tokens": 26, "ctx": 1000, "heads": 32, "kv": 8, "dim": 64, "mix": 6},
        # a batch of trees over long contexts: the cache is what has to be read
        {"name": "tree batch 16", "op": "tree", "type": "bf16", "seqs": 16, "tokens": 500, "ctx": 8000, "heads": 32, "kv": 8, "dim": 128, "mix": 7},
        # the 32-bit mode
        {"name": "tree f32 4", "op": "tree", "type": "f32", "seqs": 4, "tokens": 67, "ctx": 3000, "heads": 16, "kv": 4, "dim": 128, "mix": 8},
        # one token through a projection of this size: the decode step of one user
        {"name": "w4 one token", "op": "w4", "type": "bf16", "tokens": 1, "rows": 8192, "cols": 2048, "group": 128, "zeros": True},
        # a verified tree through a gate and up projection
        {"name": "w4 48 tokens", "op": "w4", "type": "bf16", "tokens": 48, "rows": 16384, "cols": 2048, "group": 64, "zeros": False},
        # one user's accepted path in 16 layers
        {"name": "keep one", "op": "keep", "type": "bf16", "seqs": 1, "tokens": 26, "ctx": 120, "kv": 8, "dim": 64, "layers": 16, "most": 6, "mix": 11},
        # a batch's accepted paths
        {"name": "keep batch 48", "op": "keep", "type": "bf16", "seqs": 48, "tokens": 1500, "ctx": 120, "kv": 8, "dim": 128, "layers": 16, "most": 8, "mix": 12},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["rope", "packed", "tree", "w4", "keep"])
    c = {"op": op, "type": rng.choice(["bf16", "bf16", "f32"])}
    small = c["type"] == "f32"
    if op == "w4":
        c["group"] = rng.choice([32, 64, 128])
        c["cols"] = c["group"] * log(2, 8192 // c["group"])
        c["rows"] = 8 * log(32, 4000)
        c["tokens"] = min(log(1, 200), (1 << 31) // (c["rows"] * c["cols"]) + 1)
        c["zeros"] = rng.random() < 0.5
        return c
    c["mix"] = rng.randrange(1, 1 << 20)
    c["kv"] = rng.choice([1, 2, 3, 4, 8])
    c["dim"] = rng.choice([64, 64, 80, 96, 128, 128])
    if op == "keep":
        c["seqs"] = log(1, 32)
        c["tokens"] = c["seqs"] * rng.randrange(8, 65)
        c["ctx"] = log(1, 300)
        c["layers"] = rng.randrange(1, 17)
        c["most"] = rng.randrange(1, 9)
        return c
    c["heads"] = c["kv"] * rng.choice([1, 2, 4, 5, 8])
    if op == "rope":
        c["axes"] = rng.choice([1, 1, 2, 3])
        c["seqs"] = log(1, 64)
        c["tokens"] = max(c["seqs"], log(1, 8000))
        c["ctx"] = log(1, 3000)
    elif op == "packed":
        c["seqs"] = log(1, 12)
        c["tokens"] = max(c["seqs"], log(1, 1500 if small else 6000))
        c["ctx"] = rng.choice([0, log(1, 1000 if small else 4000)])
    else:
        c["seqs"] = log(1, 24)
        c["tokens"] = c["seqs"] * rng.randrange(1, 65)
        c["ctx"] = log(1, 3000 if small else 12000)
    return c


def lengths(case):
    """New tokens and cached tokens of every sequence: fixed by the case."""
    r = random.Random(case["mix"])
    n, total = case["seqs"], case["tokens"]
    if case["op"] in ("tree", "keep"):
        most = 64
        new = [min(most, max(case.get("most", 1), int(total / n * r.uniform(0.5, 1.5)))) for _ in range(n)]
    elif total == n:
        new = [1] * n
    else:
        share = [r.uniform(0.3, 1.0) for _ in range(n)]
        if n >= 4:
            share[r.randrange(n - 1)] = 0.0         # an empty sequence among them
        new = [int(total * s / sum(share)) for s in share]
        new[-1] += total - sum(new)
    ctx = [int(case["ctx"] * r.uniform(0.4, 1.0)) for _ in range(n)]
    return new, ctx


def sections(case):
    """Rotated pairs per axis (time, height, width)."""
    half = case["dim"] // 2
    if case["axes"] == 1:
        return [half]
    if case["axes"] == 2:
        return [half // 2, half - half // 2]
    t = half // 4
    return [t, (half - t) // 2, half - t - (half - t) // 2]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dt)
    if case["op"] == "w4":
        M, N, K, G = case["tokens"], case["rows"], case["cols"], case["group"]
        return {"case": case, "x": normal(M, K), "w": torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8),
                "scale": (torch.rand((N, K // G), generator=g, device="cuda") * 0.02 + 0.002).to(torch.bfloat16),
                "zero": torch.randint(0, 16, (N, K // G), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None}
    new, ctx = lengths(case)
    B, T, G, D = len(new), sum(new), case["kv"], case["dim"]
    used = [(a + b + PAGE - 1) // PAGE for a, b in zip(new, ctx)]
    most, n_pages = max(max(used), 1), sum(used) + 3
    perm = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
    table = torch.full((B, most), -1, dtype=torch.int32)          # entries behind a sequence's pages name none
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = perm[at:at + u]
        at += u
    start = [sum(new[:b]) for b in range(B + 1)]
    st = {"case": case, "table": table.cuda(), "cu": torch.tensor(start, dtype=torch.int32).cuda(), "ctx": torch.tensor(ctx, dtype=torch.int32).cuda(),
          "most_new": max(new), "keys": most * PAGE}
    L = case.get("layers", 1)
    k, v = normal(L, n_pages, G, PAGE, D), normal(L, n_pages, G, D, PAGE)
    if case["op"] in ("packed", "tree"):
        st["q"] = normal(T, case["heads"], D)
        end = st["ctx"] + st["cu"].diff()
        for b, u in enumerate(used):                              # what lies behind a sequence's last token was never written
            if u and (new[b] + ctx[b]) % PAGE:
                tail = (new[b] + ctx[b]) % PAGE
                k[0, table[b, u - 1], :, tail:] = math.nan
                v[0, table[b, u - 1], :, :, tail:] = math.nan
        st["end"] = end
    if case["op"] == "tree":
        masks = []
        r = random.Random(seed)
        for n in new:                                             # every token's parent comes before it
            seen = []
            for i in range(n):
                parent = r.randrange(max(-1, i - 9), i)
                seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
            masks += seen
        st["mask"] = torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64).cuda()
    if case["op"] == "keep":
        r = random.Random(seed)
        m = case["most"]
        keep = torch.zeros((B, m), dtype=torch.int32)
        count = [r.randrange(0, m + 1) for _ in range(B)]
        for b, c in enumerate(count):                             # increasing; an entry stays or comes from behind the path
            path = sorted(r.sample(range(c, new[b]), min(c, new[b] - c)))
            stay = c - len(path) if len(path) < c else r.randrange(0, c + 1)
            keep[b, :c] = torch.tensor(list(range(stay)) + path[stay - c + len(path):] if c else [], dtype=torch.int32)
        st.update(keep=keep.cuda(), count=torch.tensor(count, dtype=torch.int32).cuda(), k=k, v=v, layers=list(zip(k.unbind(0), v.unbind(0))))
        return st
    st.update(k=k[0], v=v[0])
    if case["op"] == "rope":
        P, half = 4096 if case["axes"] == 1 else 20000, D // 2
        angle = torch.arange(P, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        pos = torch.cat([torch.arange(c, c + n, dtype=torch.int32) for n, c in zip(new, ctx)])
        pos = pos[None] if case["axes"] == 1 else torch.stack([pos // 100, pos // 10 % 10, pos % 10][3 - case["axes"]:])
        st.update(proj=normal(T, (case["heads"] + 2 * G) * D), cos=angle.cos().float(), sin=angle.sin().float(), pos=(pos % P).contiguous().cuda(),
                  q_gain=torch.rand(D, generator=g, device="cuda") + 0.5, k_gain=torch.rand(D, generator=g, device="cuda") + 0.5)
    return st


def places(st, at):
    """Page and token within it of cache positions at [B, n]."""
    return st["table"].gather(1, (at // PAGE).long()).long(), (at % PAGE).long()


def owner(st, T):
    """Sequence of every packed row, and the row's number in it."""
    t = torch.arange(T, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(st["cu"], t, right=True) - 1
    return b, t - st["cu"][b]


def plain_w4(st):
    c = st["case"]
    q = torch.stack([st["w"] & 15, st["w"] >> 4], dim=-1).view(c["rows"], -1, c["group"]).float()
    z = st["zero"].float() if c["zeros"] else torch.full_like(st["scale"], 8, dtype=torch.float32)
    w = ((q - z[..., None]) * st["scale"].float()[..., None]).view(c["rows"], c["cols"])
    return (st["x"].float() @ w.T).to(st["x"].dtype)


def plain_rope(st):
    c = st["case"]
    H, G, D = c["heads"], c["kv"], c["dim"]
    T, half, dt = st["proj"].shape[0], D // 2, st["proj"].dtype
    x = st["proj"].float().view(T, H + 2 * G, D)
    qk = x[:, :H + G]
    gain = torch.cat([st["q_gain"].expand(H, D), st["k_gain"].expand(G, D)])
    qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + 1e-6) * gain
    axis = torch.repeat_interleave(torch.arange(c["axes"], device="cuda"), torch.tensor(sections(c), device="cuda"), output_size=half)
    row = st["pos"][axis].T.long()                                                     # [T, half]
    pair = torch.arange(half, device="cuda")
    cos, sin = st["cos"][row, pair][:, None], st["sin"][row, pair][:, None]
    a, b = qk[..., :half], qk[..., half:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(dt)
    seq, i = owner(st, T)
    at = st["ctx"][seq] + i
    page, slot = st["table"][seq, (at // PAGE).long()].long(), (at % PAGE).long()
    st["k"][page, :, slot] = qk[:, H:]
    st["v"][page, :, :, slot] = st["proj"].view(T, H + 2 * G, D)[:, H + G:]
    return qk[:, :H].reshape(T, H * D), st["k"], st["v"]


def plain_attention(st):
    c = st["case"]
    H, G, D = c["heads"], c["kv"], c["dim"]
    q, T, n, K = st["q"], st["q"].shape[0], st["most_new"], st["keys"]
    B, R = st["table"].shape[0], H // G
    pages = st["table"].clamp(min=0).long()
    key = torch.arange(K, device="cuda")
    there = key < st["end"][:, None]                                                   # [B, K]
    k = st["k"][pages].permute(0, 2, 1, 3, 4).reshape(B, G, K, D).float()
    v = st["v"][pages].permute(0, 2, 1, 4, 3).reshape(B, G, K, D).float()
    k, v = k.where(there[:, None, :, None], 0.0), v.where(there[:, None, :, None], 0.0)
    i = torch.arange(n, device="cuda")
    row = (st["cu"][:-1, None] + i).clamp(max=T - 1).long()                            # [B, n]
    s = q[row].float().view(B, n, G, R, D).permute(0, 2, 3, 1, 4).reshape(B, G, R * n, D) @ k.transpose(-1, -2)
    s *= 1.0 / math.sqrt(D)
    draft = key - st["ctx"][:, None]                                                   # [B, K]: number among the new tokens
    if c["op"] == "packed":
        see = draft[:, None] <= i[:, None]
    else:
        bit = (st["mask"][row][..., None] >> draft.clamp(0, 63)[:, None]) & 1
        see = (draft < 0)[:, None] | (bit == 1) & (draft < 64)[:, None]
    see = see & there[:, None]
    s = s.view(B, G, R, n, K).masked_fill_(~see[:, None, None], -math.inf)
    s -= s.amax(-1, keepdim=True).clamp(min=-3e38)
    s = s.exp_()
    total = s.sum(-1)[..., None]
    o = s.view(B, G, R * n, K) @ v
    o = o.view(B, G, R, n, D) / total.clamp(min=1e-38)
    b, j = owner(st, T)
    return o.permute(0, 3, 1, 2, 4)[b, j.long()].reshape(T, H * D).to(q.dtype)


def plain_keep(st):
    m = st["keep"].shape[1]
    i = torch.arange(m, device="cuda", dtype=torch.int32)
    src = torch.where(i < st["count"][:, None], st["keep"], i)
    ps, ss = places(st, st["ctx"][:, None] + src)
    pd, sd = places(st, st["ctx"][:, None] + i)
    st["k"][:, pd, :, sd] = st["k"][:, ps, :, ss]
    st["v"][:, pd, :, :, sd] = st["v"][:, ps, :, :, ss]
    return st["k"], st["v"]


def run(st):
    c = st["case"]
    if own:
        from flexllm_b200 import ops
        if c["op"] == "w4":
            return ops.linear_w4(st["x"], st["w"], st["scale"], zero=st["zero"])
        if c["op"] == "rope":
            q = ops.qk_norm_rope(st["proj"], c["heads"], st["pos"], st["cos"], st["sin"], st["k"], st["v"], st["table"], st["cu"], st["ctx"],
                                 q_gain=st["q_gain"], k_gain=st["k_gain"], eps=1e-6, sections=sections(c))
            return q, st["k"], st["v"]
        if c["op"] == "packed":
            return ops.attn_packed(st["q"], st["k"], st["v"], st["table"], st["cu"], st["ctx"])
        if c["op"] == "tree":
            return ops.attn_tree(st["q"], st["mask"], st["k"], st["v"], st["table"], st["cu"], st["ctx"])
        ops.kv_keep(st["layers"], st["table"], st["ctx"], st["keep"], st["count"])
        return st["k"], st["v"]
    return {"w4": plain_w4, "rope": plain_rope, "packed": plain_attention, "tree": plain_attention, "keep": plain_keep}[c["op"]](st)


def work(case):
    e = 2 if case["type"] == "bf16" else 4
    if case["op"] == "w4":
        M, N, K, G = case["tokens"], case["rows"], case["cols"], case["group"]
        return {"bytes": N * K // 2 + N * (K // G) * (3 if case["zeros"] else 2) + M * (K + N) * e, "flops": 2 * M * N * K}
    new, ctx = lengths(case)
    T, G, D = sum(new), case["kv"], case["dim"]
    if case["op"] == "keep":
        return {"bytes": len(new) * (case["most"] / 2) * case["layers"] * G * 2 * D * e * 2, "flops": 0}
    H = case["heads"]
    if case["op"] == "rope":
        return {"bytes": 2 * T * (H + 2 * G) * D * e + min(T, 4096) * D * 4 + T * case["axes"] * 4, "flops": T * (H + G) * D * 8}
    if case["op"] == "packed":
        seen = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, ctx))
    else:
        seen = sum(n * (c + 1) for n, c in zip(new, ctx))        # a token's path in its tree is short
    return {"bytes": sum(n + c for n, c in zip(new, ctx)) * G * 2 * D * e + T * H * 2 * D * e, "flops": 4 * D * H * seen}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "w4":
        G, rows = case["group"], []
        for lo in range(0, case["rows"], 8192):
            w = st["w"][lo:lo + 8192]
            q = torch.empty((w.shape[0], case["cols"]), dtype=torch.float64, device="cuda")
            q[:, 0::2], q[:, 1::2] = w % 16, w // 16
            q -= (st["zero"][lo:lo + 8192].double() if case["zeros"] else torch.full((1, 1), 8.0, dtype=torch.float64, device="cuda").expand(
                w.shape[0], case["cols"] // G)).repeat_interleave(G, 1)
            q *= st["scale"][lo:lo + 8192].double().repeat_interleave(G, 1)
            rows.append(st["x"].double() @ q.T)
        return torch.cat(rows, 1)
    new, ctx = lengths(case)
    table = st["table"].cpu().tolist()
    G, D = case["kv"], case["dim"]
    if case["op"] == "keep":
        k, v = st["k"].double(), st["v"].double()
        keep, count = st["keep"].cpu().tolist(), st["count"].cpu().tolist()
        k0, v0 = k.clone(), v.clone()
        for b, c in enumerate(count):
            for i in range(c):
                s, d = ctx[b] + keep[b][i], ctx[b] + i
                k[:, table[b][d // PAGE], :, d % PAGE] = k0[:, table[b][s // PAGE], :, s % PAGE]
                v[:, table[b][d // PAGE], :, :, d % PAGE] = v0[:, table[b][s // PAGE], :, :, s % PAGE]
        return k, v
    H, start = case["heads"], st["cu"].cpu().tolist()
    if case["op"] == "rope":
        T, half = sum(new), D // 2
        axis = [a for a, n in enumerate(sections(case)) for _ in range(n)]
        x = st["proj"].double().view(T, H + 2 * G, D).clone()
        for lo, hi, gain in ((0, H, "q_gain"), (H, H + G, "k_gain")):
            y = x[:, lo:hi]
            y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * st[gain].double()
            z = y.clone()
            for p in range(half):
                where = st["pos"][axis[p]].long()
                co, si = st["cos"][where, p].double()[:, None], st["sin"][where, p].double()[:, None]
                z[..., p] = y[..., p] * co - y[..., p + half] * si
                z[..., p + half] = y[..., p] * si + y[..., p + half] * co
            x[:, lo:hi] = z
        k, v = st["k"].double(), st["v"].double()
        for b, n in enumerate(new):
            done = 0
            while done < n:                                       # page by page
                at = ctx[b] + done
                page, slot = table[b][at // PAGE], at % PAGE
                m = min(PAGE - slot, n - done)
                rows = x[start[b] + done:start[b] + done + m]
                k[page, :, slot:slot + m] = rows[:, H:H + G].transpose(0, 1)
                v[page, :, :, slot:slot + m] = rows[:, H + G:].permute(1, 2, 0)
                done += m
        return x[:, :H].reshape(T, H * D), k, v
    out = torch.zeros((sum(new), H, D), dtype=torch.float64, device="cuda")
    R = H // G
    for b, n in enumerate(new):
        end = ctx[b] + n
        for g in range(G if n else 0):
            ids = torch.tensor(table[b][:(end + PAGE - 1) // PAGE], device="cuda")
            k = st["k"][ids, g].reshape(-1, D)[:end].double()
            v = st["v"][ids, g].transpose(1, 2).reshape(-1, D)[:end].double()
            if case["op"] == "packed":
                see = torch.arange(end, device="cuda") <= torch.arange(ctx[b], end, device="cuda")[:, None]
            else:
                bits = [[m >> j & 1 for j in range(n)] for m in st["mask"][start[b]:start[b + 1]].tolist()]
                see = torch.cat([torch.ones((n, ctx[b]), device="cuda"), torch.tensor(bits, device="cuda", dtype=torch.float32)], 1) > 0
            for r in range(g * R, g * R + R):
                s = st["q"][start[b]:start[b + 1], r].double() @ k.T / math.sqrt(D)
                out[start[b]:start[b + 1], r] = torch.softmax(s.masked_fill(~see, -math.inf), -1) @ v
    return out.view(sum(new), H * D)
