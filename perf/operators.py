"""The operators between the QKV projection and the output projection, as `perf` measures them: the step's block
tables and slot maps, rotary positions (alone and fused with the paged cache write), and the attention of drafted
tokens over the paged cache. `own = False` computes each in elementary torch operations, `own = True` through
vllm_turing_b200."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- the cases -------------------------------------------------------------------------------------------------------
def _tables(name, B, new_lo, new_hi, ctx_lo, ctx_hi, block, tree):
    return dict(name=name, op="tables", B=B, new_lo=new_lo, new_hi=new_hi, ctx_lo=ctx_lo, ctx_hi=ctx_hi, block=block,
                tree=tree)


def _rotary(name, op, T, Hq, Hkv, D, rot, interleaved, backward, dtype, scaling, factor, far, block=16):
    return dict(name=name, op=op, T=T, Hq=Hq, Hkv=Hkv, D=D, rot=rot, interleaved=interleaved, backward=backward,
                dtype=dtype, scaling=scaling, factor=factor, far=far, block=block)


def _attn(name, B, new_lo, new_hi, tree, ctx_lo, ctx_hi, Hq, Hkv, D, block, dtype):
    return dict(name=name, op="attention", B=B, new_lo=new_lo, new_hi=new_hi, tree=tree, ctx_lo=ctx_lo, ctx_hi=ctx_hi,
                Hq=Hq, Hkv=Hkv, D=D, block=block, dtype=dtype)


def listed():
    return [
        # one decode step of a few requests, 1 + 4 drafted tokens each: once per step, latency only
        _tables("tables_decode", 8, 5, 5, 10, 8000, 16, False),
        # a large serving batch verifying draft trees
        _tables("tables_trees", 256, 1, 64, 0, 32000, 32, True),
        # a step that takes in prompts: many new blocks, chunks of ragged length
        _tables("tables_prompts", 64, 100, 2000, 0, 4000, 16, False),
        # one request's 5 rows of a decode step, 24 / 4 heads x 256, a quarter of the head rotated
        _rotary("rotary_cache_step", "rotary_cache", 5, 24, 4, 256, 64, False, False, "bf16", "none", 1.0, 30000),
        # the same layer on a prompt chunk
        _rotary("rotary_cache_prompt", "rotary_cache", 8192, 24, 4, 256, 64, False, False, "bf16", "none", 1.0, 30000),
        # interleaved pairs over the whole head at far positions of a context stretched by yarn
        _rotary("rotary_yarn", "rotary", 4099, 32, 8, 128, 128, True, False, "fp16", "yarn", 8.0, 1000000),
        # the gradient's direction, llama3 scaling, a prompt
        _rotary("rotary_backward", "rotary", 16384, 32, 8, 128, 128, False, True, "bf16", "llama3", 8.0, 131000),
        # one sequence, one token on one of four ranks, short context: latency
        _attn("attn_token", 1, 1, 1, False, 1000, 1000, 6, 1, 256, 16, "bf16"),
        # 1 + 4 drafted tokens of one sequence over a long context
        _attn("attn_verify_long", 1, 5, 5, False, 65531, 65531, 24, 4, 256, 16, "bf16"),
        # a batch of ragged sequences with draft trees
        _attn("attn_trees", 64, 5, 24, True, 100, 8000, 24, 4, 256, 32, "bf16"),
        # a large batch of single tokens, heads of 128, fp16
        _attn("attn_tokens", 256, 1, 1, False, 1, 4001, 32, 8, 128, 16, "fp16"),
        # full trees of 64 nodes, 8 query heads to a cached one: the largest products
        _attn("attn_full_trees", 8, 64, 64, True, 9000, 16000, 32, 4, 128, 64, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(("tables", "rotary", "rotary_cache", "attention", "attention"))
    dtype = rng.choice(("bf16", "fp16"))
    if op == "tables":
        tree = rng.random() < 0.5
        B = _log(rng, 1, 256)
        hi = _log(rng, 1, 64 if tree else max(1, 50000 // B))
        ctx = _log(rng, 1, 32000)
        return _tables(None, B, rng.randint(1, hi), hi, rng.randint(0, ctx), ctx, 8 * _log(rng, 1, 16), tree)
    if op in ("rotary", "rotary_cache"):
        D = rng.choice((64, 80, 96, 128, 192, 256))
        rot = rng.choice((D, D // 2, D // 4))
        Hkv = _log(rng, 1, 8)
        G = _log(rng, 1, 8)
        T = _log(rng, 1, max(1, (1 << 26) // (Hkv * (G + 2) * D)))
        scaling = rng.choice(("none", "linear", "ntk", "yarn", "llama3"))
        return _rotary(None, op, T, Hkv * G, Hkv, D, rot, rng.random() < 0.5, op == "rotary" and rng.random() < 0.5,
                       dtype, scaling, 1.0 if scaling == "none" else rng.uniform(1.5, 32.0), _log(rng, 100, 1000000))
    D = rng.choice((64, 80, 128, 128, 192, 256, 256))
    Hkv = _log(rng, 1, 8)
    G = _log(rng, 1, 12)
    hi = _log(rng, 1, 64)
    B = _log(rng, 1, 256)
    # keys * heads so that neither bytes nor products pass the largest listed case
    room = min((1 << 29) // (B * Hkv * D), (1 << 35) // (B * hi * G * Hkv * D))
    ctx = _log(rng, 1, max(1, min(100000, room)))
    return _attn(None, B, rng.randint(1, hi), hi, rng.random() < 0.5, rng.randint(0, ctx), ctx, Hkv * G, Hkv, D,
                 8 * _log(rng, 1, 32), dtype)


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _spread(lo, hi, n):
    """n whole numbers over [lo, hi], the same for every seed (work() counts them): hi first, then scattered."""
    return [hi - int((i * 0.6180339887498949 % 1.0) * (hi - lo + 1)) if hi > lo else lo for i in range(n)]


def _lengths(case):
    ctx = _spread(case["ctx_lo"], case["ctx_hi"], case["B"])
    new = _spread(case["new_lo"], case["new_hi"], case["B"])[::-1]
    return ctx, new


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _parents(new, seed):
    """A random tree for each request: node 0 hangs on the context, every other node on an earlier one."""
    T = sum(new)
    u = torch.rand(T, generator=torch.Generator().manual_seed(seed)).tolist()
    out, t = [], 0
    for n in new:
        out += [-1 if i == 0 else int(u[t + i] * i) for i in range(n)]
        t += n
    return out


def _frequencies(case):
    """64-bit angular frequencies of the rotated pairs and the factor on the rotated part, from the definitions."""
    rot, s, f = case["rot"], case["factor"], case["scaling"]
    base, orig = 10000.0, 4096
    if f == "ntk":
        base *= s ** (rot / (rot - 2))
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    w = base ** (-2.0 * i / rot)
    factor = 1.0
    if f == "linear":
        w = w / s
    elif f == "yarn":
        def dim(turns):
            return rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(dim(32)), 0), min(math.ceil(dim(1)), rot - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        w = w / s * ramp + w * (1 - ramp)
        factor = 0.1 * math.log(s) + 1.0
    elif f == "llama3":
        wave = 2 * math.pi / w
        smooth = ((orig / wave - 1.0) / 3.0).clamp(0, 1)
        w = (1 - smooth) * w / s + smooth * w
    return w, factor


def _inputs(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] == "tables":
        ctx, new = _lengths(case)
        bs, B = case["block"], case["B"]
        width = max(-(-(c + n) // bs) for c, n in zip(ctx, new)) + 1
        held = [-(-c // bs) for c in ctx]
        need = sum(-(-(c + n) // bs) - h for c, n, h in zip(ctx, new, held))
        total = sum(held) + need + 7
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        table = torch.full((B, width), -1, dtype=torch.int32)
        at = 0
        for b, h in enumerate(held):
            table[b, :h] = order[at:at + h]
            at += h
        free = torch.full((total,), -1, dtype=torch.int32)
        free[:total - at] = order[at:]
        s.update(table=table.cuda(), held=_ints(held), free=free.cuda(), count=_ints([total - at]),
                 cached=_ints(ctx), new=_ints(new), T=sum(new) + 3)
        if case["tree"]:
            s["parents"] = _ints(_parents(new, seed) + [-1] * 3)
        return s
    dt = DTYPES[case["dtype"]]
    Hq, Hkv, D, bs = case["Hq"], case["Hkv"], case["D"], case["block"]
    if case["op"] in ("rotary", "rotary_cache"):
        T = case["T"]
        # q, k and v as they leave the projection: columns of one [T, ...] result
        qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g, device="cuda").to(dt)
        q, k, v = qkv.split((Hq * D, Hkv * D, Hkv * D), dim=1)
        s.update(q=q.view(T, Hq, D), k=k.view(T, Hkv, D), v=v.view(T, Hkv, D))
        s["positions"] = torch.randint(0, case["far"] + 1, (T,), generator=g, device="cuda")
        if case["op"] == "rotary_cache":
            blocks = -(-T // bs) + 5
            s["k_cache"] = torch.zeros(blocks, bs, Hkv, D, dtype=dt, device="cuda")
            s["v_cache"] = torch.zeros_like(s["k_cache"])
            s["slots"] = torch.randperm(blocks * bs, generator=g, device="cuda")[:T].contiguous()
            if T > 4:
                s["slots"][T // 2] = -1   # a row with no place in the cache
        return s
    ctx, new = _lengths(case)
    lens = [c + n for c, n in zip(ctx, new)]
    pages = [-(-x // bs) for x in lens]
    blocks = sum(pages) + 3
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.zeros(case["B"], max(pages), dtype=torch.int32)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    parents = _parents(new, seed) if case["tree"] else None
    s.update(q=(1.5 * torch.randn(cu[-1], Hq, D, generator=g, device="cuda")).to(dt),
             k_cache=torch.empty(blocks, bs, Hkv, D, dtype=dt, device="cuda").normal_(generator=g),
             v_cache=torch.empty(blocks, bs, Hkv, D, dtype=dt, device="cuda").normal_(generator=g),
             table=table.cuda(), cu=_ints(cu), lens=_ints(lens), mask=None, host_cu=cu, host_lens=lens,
             host_parents=parents)
    if parents is not None:
        rows = []
        for a, b in zip(cu, cu[1:]):
            m = []
            for i in range(b - a):
                p = parents[a + i]
                m.append((1 << i) | (m[p] if p >= 0 else 0))
            rows += [x - (1 << 64) if x >> 63 else x for x in m]
        s["mask"] = _ints(rows, torch.int64)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if "rot" in case:
        if own:
            from vllm_turing_b200 import rotary
            s["freqs"] = rotary.rope_frequencies(case["rot"], base=10000.0, scaling=case["scaling"],
                                                 factor=case["factor"], original_length=4096, device="cuda")
        else:
            s["freqs"] = _frequencies(case)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    c = s["case"]
    if c["op"] == "tables":
        from vllm_turing_b200 import steptables
        t = steptables.step_tables(s["table"], s["held"], s["free"], s["count"], s["cached"], s["new"], c["block"],
                                   s["T"], parents=s.get("parents"))
        return [s["table"], s["held"], s["count"], t.cu, t.seq_lens, t.positions, t.slots, t.mask, t.status]
    if c["op"] == "rotary":
        from vllm_turing_b200 import rotary
        return list(rotary.rotary(s["q"], s["k"], s["positions"], s["freqs"], interleaved=c["interleaved"],
                                  transpose=c["backward"]))
    if c["op"] == "rotary_cache":
        from vllm_turing_b200 import rotary
        q = rotary.rotary_cache(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["k_cache"], s["v_cache"],
                                s["freqs"], interleaved=c["interleaved"])
        return [q, s["k_cache"], s["v_cache"]]
    from vllm_turing_b200 import treeattn
    return treeattn.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["lens"], c["new_hi"],
                                   mask=s["mask"])


def _run_plain(s):
    return {"tables": _plain_tables, "rotary": _plain_rotary, "rotary_cache": _plain_rotary_cache,
            "attention": _plain_attention}[s["case"]["op"]](s)


def _plain_tables(s):
    bs, T = s["case"]["block"], s["T"]
    table, held, cached = s["table"], s["held"], s["cached"]
    new = s["new"].clamp(min=0)
    B, width = table.shape
    want = (cached + new + bs - 1) // bs
    need = (want - held).clamp(min=0)
    fits = want <= width
    need = torch.where(fits, need, 0)
    upto = need.cumsum(0).to(torch.int32)
    served = fits & (upto <= s["count"])
    got = torch.where(served, need, 0)
    col = torch.arange(width, device="cuda", dtype=torch.int32)
    k = col[None] - held[:, None]
    fresh = (k >= 0) & (k < got[:, None])
    at = (s["count"] - 1 - (upto - need)[:, None] - k).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(fresh, s["free"][at.long()], table))
    short = (~served & fits).any() | (need.sum() > s["count"])
    held += got
    s["count"].sub_(got.sum().to(torch.int32))
    cu = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    cu[1:] = new.cumsum(0)
    status = (short.to(torch.int32) + 2 * (~fits).any().to(torch.int32) + 4 * (cu[B] > T).to(torch.int32)).reshape(1)
    t = torch.arange(T, device="cuda", dtype=torch.int32)
    live = t < cu[B]
    b = (torch.searchsorted(cu[1:].contiguous(), t, right=True)).clamp(max=B - 1)
    i = t - cu[b]
    mask = None
    depth = i
    if "parents" in s:
        mask = torch.zeros(T, dtype=torch.int64, device="cuda")
        depth = torch.full_like(i, -1)
        node = torch.where(live, i, -1)
        for _ in range(64):
            on = node >= 0
            mask = torch.where(on, mask | (torch.ones_like(mask) << node.clamp(min=0).long()), mask)
            depth = depth + on.to(torch.int32)
            up = s["parents"][(cu[b] + node.clamp(min=0)).long().clamp(max=T - 1)]
            node = torch.where(on, up, -1)
    positions = torch.where(live, (cached[b] + depth).long(), 0)
    j = cached[b] + i
    page = j // bs
    block = table[b, page.clamp(max=width - 1).long()].long()
    ok = live & (page < held[b])
    slots = torch.where(ok, block * bs + (j % bs).long(), -1)
    return [table, held, s["count"], cu, cached + new, positions, slots, mask, status]


def _rotate(x, positions, freqs, case):
    """x [T, H, D] rotated in 32 bits, angles in 64."""
    w, factor = freqs
    a = positions.double()[:, None] * w
    c, s = (a.cos() * factor).float()[:, None], (a.sin() * factor).float()[:, None]
    if case["backward"]:
        s = -s
    rot = case["rot"]
    y = x.float()
    r = y[..., :rot]
    if case["interleaved"]:
        x1, x2 = r[..., 0::2], r[..., 1::2]
        r = torch.stack((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1).flatten(-2)
    else:
        x1, x2 = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1)
    return torch.cat((r, y[..., rot:]), dim=-1).to(x.dtype)


def _plain_rotary(s):
    return [_rotate(s[n], s["positions"], s["freqs"], s["case"]) for n in ("q", "k")]


def _plain_rotary_cache(s):
    q, k = _plain_rotary(s)
    Hkv, D = k.shape[1:]
    ok = s["slots"] >= 0
    at = s["slots"][ok]
    s["k_cache"].view(-1, Hkv, D)[at] = k[ok]
    s["v_cache"].view(-1, Hkv, D)[at] = s["v"][ok]
    return [q, s["k_cache"], s["v_cache"]]


def _plain_attention(s):
    q, kc, vc = s["q"], s["k_cache"], s["v_cache"]
    T, Hq, D = q.shape
    bs, Hkv = kc.shape[1:3]
    G = Hq // Hkv
    out = torch.zeros_like(q)
    for b, L in enumerate(s["host_lens"]):
        t0, t1 = s["host_cu"][b], s["host_cu"][b + 1]
        n, ctx = t1 - t0, L - (t1 - t0)
        ids = s["table"][b, :-(-L // bs)].long()
        k = kc[ids].reshape(-1, Hkv, D)[:L].float().permute(1, 2, 0)
        v = vc[ids].reshape(-1, Hkv, D)[:L].float().permute(1, 0, 2)
        x = q[t0:t1].float().view(n, Hkv, G, D).permute(1, 0, 2, 3).reshape(Hkv, n * G, D)
        sc = torch.matmul(x, k) * D ** -0.5
        node = torch.arange(n, device="cuda")
        if s["mask"] is None:
            see = node[None] <= node[:, None]
        else:
            see = ((s["mask"][t0:t1, None] >> node[None]) & 1) == 1
        see = torch.cat((torch.ones(n, ctx, dtype=torch.bool, device="cuda"), see), dim=1)
        sc = sc.masked_fill(~see.repeat_interleave(G, dim=0)[None], float("-inf"))
        p = torch.exp(sc - sc.amax(dim=-1, keepdim=True))
        o = torch.matmul(p, v) / p.sum(dim=-1, keepdim=True)
        out[t0:t1] = o.view(Hkv, n, G, D).permute(1, 0, 2, 3).reshape(n, Hq, D).to(q.dtype)
    return out


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    if case["op"] == "tables":
        ctx, new = _lengths(case)
        bs, T = case["block"], sum(new)
        blocks = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(ctx, new))
        tree = case["tree"]
        return {"bytes": 4 * 6 * case["B"] + 8 * blocks + T * (16 + (12 if tree else 0)), "flops": 8 * T}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["op"] in ("rotary", "rotary_cache"):
        T = case["T"]
        rows = Hq + Hkv + (Hkv if case["op"] == "rotary_cache" else 0)
        return {"bytes": T * (2 * rows * D * 2 + 8 + (8 if case["op"] == "rotary_cache" else 0)),
                "flops": T * (Hq + Hkv) * case["rot"] * 3}
    ctx, new = _lengths(case)
    keys = sum(c + n for c, n in zip(ctx, new))
    pairs = sum((c + n) * n for c, n in zip(ctx, new))
    return {"bytes": keys * Hkv * D * 4 + 2 * sum(new) * Hq * D * 2, "flops": 4 * pairs * Hq * D}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    return {"tables": _exact_tables, "rotary": _exact_rotary, "rotary_cache": _exact_rotary,
            "attention": _exact_attention}[case["op"]](case, s)


def _exact_tables(case, s):
    """One request after the other, on the host."""
    bs, T = case["block"], s["T"]
    table, held, free = s["table"].tolist(), s["held"].tolist(), s["free"].tolist()
    left = s["count"].item()
    parents = s["parents"].tolist() if "parents" in s else None
    cu, lens, positions, slots, mask = [0], [], [], [], []
    for b, (c, n) in enumerate(zip(s["cached"].tolist(), s["new"].tolist())):
        while held[b] * bs < c + n:
            left -= 1
            table[b][held[b]] = free[left]
            held[b] += 1
        for i in range(n):
            j = c + i
            slots.append(table[b][j // bs] * bs + j % bs)
            seen = [i]
            if parents is None:
                positions.append(j)
                continue
            while parents[cu[-1] + seen[-1]] >= 0:
                seen.append(parents[cu[-1] + seen[-1]])
            positions.append(c + len(seen) - 1)
            word = sum(1 << x for x in seen)
            mask.append(word - (1 << 64) if word >= 1 << 63 else word)
        cu.append(cu[-1] + n)
        lens.append(c + n)
    pad = T - len(slots)
    return [_ints(table), _ints(held), _ints([left]), _ints(cu), _ints(lens), _ints(positions + [0] * pad, torch.int64),
            _ints(slots + [-1] * pad, torch.int64),
            None if parents is None else _ints(mask + [0] * pad, torch.int64), _ints([0])]


def _exact_rotary(case, s):
    """Each pair as a complex number times factor * exp(+-i position w)."""
    w, factor = _frequencies(case)
    T, rot = case["T"], case["rot"]
    angle = s["positions"].double()[:, None] * w * (-1.0 if case["backward"] else 1.0)
    turn = torch.polar(torch.full_like(angle, factor), angle)[:, None]

    def turned(x):
        y = x.double()
        first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, rot // 2),
                                                                                          slice(rot // 2, rot))
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q, k = turned(s["q"]), turned(s["k"])
    if case["op"] == "rotary":
        return [q, k]
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    bs = case["block"]
    ok = torch.nonzero(s["slots"] >= 0).flatten()
    at = s["slots"][ok]
    kc[at // bs, at % bs] = k[ok]
    vc[at // bs, at % bs] = s["v"][ok].double()
    return [q, kc, vc]


def _exact_attention(case, s):
    """One request and one cached head at a time; a node sees the context, itself and its ancestors."""
    q, table = s["q"], s["table"]
    T, Hq, D = q.shape
    bs, Hkv = case["block"], case["Hkv"]
    G = Hq // Hkv
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device="cuda")
    for b, L in enumerate(s["host_lens"]):
        t0, n = s["host_cu"][b], s["host_cu"][b + 1] - s["host_cu"][b]
        hidden = torch.zeros(n, L, dtype=torch.bool)
        hidden[:, L - n:] = True
        for i in range(n):
            if s["host_parents"] is None:
                hidden[i, L - n:L - n + i + 1] = False
                continue
            x = i
            while x >= 0:
                hidden[i, L - n + x] = False
                x = s["host_parents"][t0 + x]
        hidden = hidden.cuda()
        j = torch.arange(L, device="cuda")
        page, row = table[b].long()[j // bs], j % bs
        for h in range(Hkv):
            k, v = s["k_cache"][page, row, h].double(), s["v_cache"][page, row, h].double()
            for g in range(h * G, (h + 1) * G):
                score = q[t0:t0 + n, g].double() @ k.t() / math.sqrt(D)
                score[hidden] = float("-inf")
                out[t0:t0 + n, g] = torch.softmax(score, dim=1) @ v
    return out
