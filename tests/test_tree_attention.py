"""treeattn.tree_attention against attention in 64 bits.

Tolerance of an output value, derived before any run. With weights p_j that sum to 1 and a = sum_j p_j |v_j|:
- the result is rounded once to its type: h |out|, h = eps / 2;
- each weight may be rounded to the type once before it multiplies V: h a;
- a score is a 32-bit sum of D products (counted double, should a sum truncate): off by 2 D 2^-24 sum |q k| scale at
  most; the exponential and its argument, scaled to base 2, add less than 2^-21. A weight is off by that fraction d, and
  so is the sum that it is divided by: 2 d a;
- the 32-bit sums over L keys: 2 L 2^-24 a;
- fp16: weights are held scaled so that the largest is at least 2^4; below 2^-14 they are off by up to 2^-25: L 2^-29
  max |v| p_max in all. Results below the normal range: 2^-25.
"""
import math

import pytest
import torch

from vllm_turing_b200 import treeattn as A

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def make(lens, new, Hq, Hkv, D, bs, dt, seed=0, trees=False, layout="blocks", q_scale=1.5):
    """A cache with NaN wherever no key of any request is, a shuffled table, queries, random tree masks."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    gc = torch.Generator().manual_seed(seed)
    pages = [-(-x // bs) for x in lens]
    nb = sum(pages) + 2
    if layout == "heads":
        kv = [torch.full((nb, Hkv, bs, D), float("nan"), dtype=dt, device="cuda").transpose(1, 2) for _ in range(2)]
    elif layout == "joint":
        both = torch.full((nb, 2, bs, Hkv, D), float("nan"), dtype=dt, device="cuda")
        kv = [both[:, 0], both[:, 1]]
    else:
        kv = [torch.full((nb, bs, Hkv, D), float("nan"), dtype=dt, device="cuda") for _ in range(2)]
    order = torch.randperm(nb, generator=gc).tolist()
    table = torch.full((len(lens), max(pages + [1])), 0, dtype=torch.int32)
    at = 0
    keys = []
    for b, p in enumerate(pages):
        ids = order[at:at + p]
        at += p
        table[b, :p] = torch.tensor(ids, dtype=torch.int32)
        kb = []
        for c in kv:
            x = torch.randn(lens[b], Hkv, D, generator=g, device="cuda").to(dt)
            full = torch.full((p * bs, Hkv, D), float("nan"), dtype=dt, device="cuda")
            full[:lens[b]] = x
            c[torch.tensor(ids, device="cuda", dtype=torch.long)] = full.view(p, bs, Hkv, D)
            kb.append(x)
        keys.append(kb)
    T = sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = (q_scale * torch.randn(T, Hq, D, generator=g, device="cuda")).to(dt)
    see, words = [], []
    for n in new:
        m = torch.tril(torch.ones(n, n, dtype=torch.bool))
        if trees:
            m = torch.eye(n, dtype=torch.bool)
            for i in range(1, n):
                p = int(torch.randint(-1, i, (1,), generator=gc))
                if p >= 0:
                    m[i] |= m[p]
        see.append(m)
        for i in range(n):
            w = sum(1 << j for j in range(n) if m[i, j])
            words.append(w - (1 << 64) if w >> 63 else w)
    mask = torch.tensor(words, dtype=torch.int64, device="cuda") if trees else None
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    return dict(q=q, kc=kv[0], vc=kv[1], table=table.cuda(), cu=i32(cu), lens=i32(lens), mask=mask, keys=keys, see=see,
                host_cu=cu, max_new=max(new + [1]))


def check(case, out, hide=None, scale=None):
    """hide[b]: bool [L] of keys no row may see."""
    q = case["q"]
    T, Hq, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    h = torch.finfo(q.dtype).eps / 2
    for b, (k, v) in enumerate(case["keys"]):
        t0, t1 = case["host_cu"][b], case["host_cu"][b + 1]
        n, L = t1 - t0, k.shape[0]
        if n == 0:
            continue
        G = Hq // k.shape[1]
        see = torch.ones(n, L, dtype=torch.bool)
        m = min(n, L)
        see[:, L - m:] = case["see"][b][:, n - m:]
        if hide is not None:
            see &= ~hide[b][None]
        see = see.cuda()
        kk = k.double().repeat_interleave(G, dim=1)
        vv = v.double().repeat_interleave(G, dim=1)
        qq = q[t0:t1].double()
        # what nothing sees does not enter, whatever it is
        kk = torch.where(see.any(0)[:, None, None], kk, 0)
        vv = torch.where(see.any(0)[:, None, None], vv, 0)
        s = torch.einsum("ihd,jhd->hij", qq, kk) * scale
        mag = torch.einsum("ihd,jhd->hij", qq.abs(), kk.abs()) * scale
        s = s.masked_fill(~see[None], -math.inf)
        any_ = see.any(1)
        s[:, ~any_] = 0
        p = torch.softmax(s, dim=-1)
        p = p * see[None]
        vz = torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0)
        want = torch.einsum("hij,jhd->ihd", p, vz)
        a = torch.einsum("hij,jhd->ihd", p, vz.abs())
        d = 2 * D * 2.0 ** -24 * torch.where(see[None], mag, 0).amax(-1) + 2.0 ** -21 if L else torch.zeros(Hq, n)
        d = d.to(a.device).t()[..., None]
        tol = h * want.abs() + (h + 2 * d + 2 * L * 2.0 ** -24) * a * (1 + h) + 1e-30
        if q.dtype == torch.float16:
            tol = tol + L * 2.0 ** -29 * vz.abs().amax() * p.amax(-1).t()[..., None] + 2.0 ** -25
        got = out[t0:t1].double()
        ok = torch.isfinite(got)
        bad = ((got - want).abs() > tol) | ~ok
        # a value that is infinite or NaN where it is seen makes its column of the rows that see it so
        for j in torch.nonzero(~torch.isfinite(v).all(-1).all(-1)).flatten().tolist():
            wild = ~torch.isfinite(v[j].repeat_interleave(G, dim=0))
            rows = see[:, j]
            assert not torch.isfinite(got[rows][:, wild]).any()
            bad[rows.nonzero().flatten()[:, None, None].expand(-1, Hq, D),
                torch.arange(Hq, device="cuda")[None, :, None], torch.arange(D, device="cuda")] &= ~wild[None]
        assert not bad.any(), (f"request {b}: {int(bad.sum())} off, worst "
                               f"{((got - want).abs() - tol).nan_to_num(9e9).max().item()}, first "
                               f"{torch.nonzero(bad)[:3].tolist()}")


def run(c, **kw):
    return A.tree_attention(c["q"], c["kc"], c["vc"], c["table"], c["cu"], c["lens"], kw.pop("max_new", c["max_new"]),
                            mask=c["mask"], **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("trees", [False, True], ids=["chain", "tree"])
@pytest.mark.parametrize("Hq, Hkv, D", [(6, 1, 256), (24, 4, 256), (8, 2, 128), (4, 4, 64), (7, 1, 80), (10, 2, 192),
                                        (3, 3, 8), (16, 1, 128), (40, 1, 64), (2, 1, 248), (128, 1, 128),
                                         (200, 2, 256)])
def test_heads(Hq, Hkv, D, trees, dtype):
    c = make([1, 5, 64, 129, 300, 17], [1, 5, 3, 8, 4, 0], Hq, Hkv, D, 16, DT[dtype], seed=D + Hq, trees=trees)
    check(c, run(c))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["blocks", "heads", "joint"])
@pytest.mark.parametrize("bs", [8, 16, 24, 32, 64, 128, 256, 544])
def test_pages(bs, layout):
    c = make([5, 127, 128, 129, 700, 1023], [5, 1, 7, 64, 12, 3], 8, 2, 128, bs, torch.bfloat16, seed=bs, trees=True,
             layout=layout)
    check(c, run(c))


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 1000])
@pytest.mark.parametrize("D", [64, 256])
def test_lengths(L, D):
    for n in sorted({1, min(L, 5), min(L, 64)}):
        c = make([L], [n], 6, 2, D, 16, torch.bfloat16, seed=L, trees=n > 1)
        check(c, run(c))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 3, 5, 16, 21, 22, 33, 63, 64])
@pytest.mark.parametrize("G", [1, 6, 8, 12])
def test_rows(n, G):
    """Rows per cached head from 1 to several tiles."""
    c = make([n + 150, n, 2 * n + 700], [n, n, n], 2 * G, 2, 64, 16, torch.bfloat16, seed=n, trees=True)
    check(c, run(c))
    c = make([n + 77], [n], G, 1, 256, 32, torch.float16, seed=n)
    check(c, run(c))


@pytest.mark.gpu
@pytest.mark.parametrize("B, lo, hi, n, D, Hq, Hkv", [(1, 70000, 70000, 5, 256, 6, 1), (200, 0, 900, 1, 128, 8, 2),
                                                     (40, 0, 5000, 9, 64, 8, 4), (3, 20000, 30000, 64, 128, 16, 2),
                                                     (1000, 0, 40, 2, 64, 2, 1)])
def test_ragged_batches(B, lo, hi, n, D, Hq, Hkv):
    g = torch.Generator().manual_seed(B)
    new = torch.randint(0, n + 1, (B,), generator=g).tolist()
    lens = [int(x) + m for x, m in zip(torch.randint(lo, hi + 1, (B,), generator=g), new)]
    c = make(lens, new, Hq, Hkv, D, 16, torch.bfloat16, seed=B, trees=True)
    check(c, run(c))
    again = run(c)
    assert torch.equal(again, run(c))   # the same bits every time


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_what_is_not_seen(D):
    """NaN and infinities in keys and values that a row's mask hides, rows that see nothing, scores at the bottom."""
    n = 8
    c = make([40, n, 300], [n, n, n], 4, 2, D, 16, torch.bfloat16, seed=3, trees=True)
    words = [(1 << i) | 1 for i in range(n)] * 3      # each node sees the root and itself
    words[n], words[n + 3] = 0, 0                     # two rows of the second request see nothing
    see = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        see[i, i] = see[i, 0] = True
    c["mask"] = torch.tensor(words, dtype=torch.int64, device="cuda")
    c["see"] = [see.clone() for _ in range(3)]
    c["see"][1][0], c["see"][1][3] = False, False
    for b in range(3):   # node 2: wild keys and values; node 4: an infinity in one value
        L = c["keys"][b][0].shape[0]
        for what, (cache, x) in enumerate(zip((c["kc"], c["vc"]), c["keys"][b])):
            j = L - n + 2
            if what:
                x[j, 0, :3] = torch.tensor([float("nan"), float("inf"), -float("inf")])
                x[L - n + 4, 1, D - 1] = float("inf")
            page = c["table"][b].long()
            for jj in (j, L - n + 4):
                cache[page[jj // 16], jj % 16] = x[jj]
    out = run(c)
    check(c, out)
    for t in (n, n + 3):
        assert (out[t] == 0).all()
    # a wild key: only the rows that see it change
    b, L = 2, 300
    j = L - n + 5
    c["kc"][c["table"][b, j // 16].long(), j % 16] = float("nan")
    out2 = run(c)
    rows = torch.ones(3 * n, dtype=torch.bool)
    rows[2 * n + 5] = False
    assert torch.equal(out2[rows.cuda()].nan_to_num(3.0), out[rows.cuda()].nan_to_num(3.0))
    assert out2[2 * n + 5].isnan().all()


@pytest.mark.gpu
def test_extreme_scores():
    """Scores far apart: the running maximum jumps by hundreds from tile to tile, in both directions."""
    c = make([2000, 1500], [5, 5], 4, 2, 128, 16, torch.bfloat16, seed=9, q_scale=40.0)
    check(c, run(c))
    c = make([1200], [3], 2, 1, 64, 16, torch.float16, seed=9, q_scale=1.0)
    ramp = torch.linspace(-8, 8, 1200, device="cuda")[:, None, None]
    for sign in (1.0, -1.0):
        k = (c["q"][0, 0][None, None] * ramp * sign).to(torch.float16)
        c["keys"][0][0].copy_(k)
        for j in range(1200):
            c["kc"][c["table"][0, j // 16].long(), j % 16] = k[j]
        check(c, run(c))
    check(c, run(c, scale=0.0), scale=0.0)
    check(c, run(c, scale=-0.3), scale=-0.3)


@pytest.mark.gpu
def test_blocks_that_are_not_there():
    """Table entries outside the cache, and a length past the table's columns: those keys are not seen."""
    c = make([200, 100, 64], [4, 4, 4], 4, 2, 128, 16, torch.bfloat16, seed=4)
    hide = [torch.zeros(L, dtype=torch.bool) for L in (200, 100, 64)]
    for b, page, entry in ((0, 3, -1), (0, 8, 1 << 30), (1, 0, c["kc"].shape[0]), (2, 3, -(1 << 31))):
        c["table"][b, page] = entry
        hide[b][page * 16:(page + 1) * 16] = True
    check(c, run(c), hide)
    c["table"] = c["table"][:, :5].contiguous()   # width 5: keys from 80 on have no entry
    hide[0][80:] = True
    hide[1][80:] = True
    out = run(c)
    check(c, out, hide)
    # nothing at all to see
    c["table"].fill_(-1)
    assert (run(c) == 0).all()


@pytest.mark.gpu
def test_rows_left_alone_and_strided():
    """Rows past the last token stay; q and out are columns of wider tensors; more tokens than max_new stay too."""
    c = make([50, 0, 90], [3, 0, 6], 6, 2, 64, 16, torch.bfloat16, seed=5)
    wide = torch.randn(12, 6 * 64 + 8, device="cuda").to(torch.bfloat16)
    wide[:9, :384] = c["q"].view(9, 384)
    qv = wide[:, :384].view(12, 6, 64)
    out = torch.full((12, 6, 72), 5.0, dtype=torch.bfloat16, device="cuda")[:, :, :64]
    A.tree_attention(qv, c["kc"], c["vc"], c["table"], c["cu"], c["lens"], 6, out=out)
    check(c, out[:9])
    assert (out[9:] == 5).all()
    part = torch.full((9, 6, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    run(c, out=part, max_new=4)
    assert torch.equal(part[:7], out[:7]) and (part[7:] == 5).all()
    # an odd token stride, unaligned addresses
    odd = torch.empty(9 * 385 + 1, dtype=torch.bfloat16, device="cuda")[1:].as_strided((9, 6, 64), (385, 64, 1))
    odd.copy_(c["q"])
    out2 = torch.empty(9 * 385 + 1, dtype=torch.bfloat16, device="cuda")[1:].as_strided((9, 6, 64), (385, 64, 1))
    A.tree_attention(odd, c["kc"], c["vc"], c["table"], c["cu"], c["lens"], 6, out=out2)
    assert torch.equal(out2, out[:9])


@pytest.mark.gpu
def test_lengths_that_do_not_fit():
    """A length shorter than the request's tokens (its first ones have no key), and zero."""
    c = make([3, 0], [5, 2], 4, 2, 64, 16, torch.bfloat16, seed=6)
    out = run(c)
    check(c, out)
    assert (out[:2] == 0).all() and (out[5:] == 0).all()


@pytest.mark.gpu
def test_a_length_far_past_the_table():
    """The largest length an int holds: every key the table has is context, the step's own tokens are past it."""
    c = make([80, 40], [4, 2], 6, 2, 128, 16, torch.bfloat16, seed=12)
    c["lens"][0] = (1 << 31) - 1
    c["see"][0] = torch.ones(4, 4, dtype=torch.bool)
    check(c, run(c))


@pytest.mark.gpu
def test_graph_and_streams():
    """Captured once, replayed with other lengths, tables and masks; two captured graphs and two streams at once."""
    c = make([900, 400, 33], [5, 5, 5], 12, 2, 256, 16, torch.bfloat16, seed=7)
    d = make([100, 901, 700], [5, 5, 5], 12, 2, 256, 16, torch.bfloat16, seed=8, trees=True)
    outs = [torch.zeros_like(c["q"]) for _ in range(2)]
    run(c)
    graphs = []
    for x, o in ((c, outs[0]), (d, outs[1])):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(x, out=o)
        graphs.append(g)
    s = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(s[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    check(c, outs[0])
    check(d, outs[1])
    lens, keys = c["lens"].clone(), c["keys"]
    c["lens"].copy_(torch.tensor([800, 5, 32], dtype=torch.int32))
    c["keys"] = [[x[:L] for x in k] for k, L in zip(keys, (800, 5, 32))]
    graphs[0].replay()
    check(c, outs[0])
    c["lens"].copy_(lens)
    c["keys"] = keys
    res = []
    for i in range(2):   # eager calls on two streams at once
        with torch.cuda.stream(s[i]):
            res.append([run((c, d)[i]) for _ in range(10)])
    torch.cuda.synchronize()
    for i in range(2):
        for r in res[i]:
            assert torch.equal(r, res[i][0])
        check((c, d)[i], res[i][0])


@pytest.mark.gpu
def test_cache_past_32_bit_offsets():
    nb, bs, H, D = 32800, 64, 8, 256   # 4.3e9 elements each
    if torch.cuda.mem_get_info()[0] < 20e9:
        pytest.skip("needs 20 GB")
    kc = torch.empty(nb, bs, H, D, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    c = make([130], [5], H, H, D, bs, torch.bfloat16, seed=1)
    ids = [nb - 1, 0, nb - 2]
    for p, i in enumerate(ids):
        kc[i], vc[i] = c["kc"][c["table"][0, p].long()], c["vc"][c["table"][0, p].long()]
    c["kc"], c["vc"] = kc, vc
    c["table"] = torch.tensor([ids], dtype=torch.int32, device="cuda")
    check(c, run(c))


@pytest.mark.gpu
def test_custom_op():
    c = make([50, 70], [3, 6], 6, 2, 64, 16, torch.bfloat16, seed=5, trees=True)
    out = torch.empty_like(c["q"])
    torch.ops.vllm_turing.tree_attention_(out, c["q"], c["kc"], c["vc"], c["table"], c["cu"], c["lens"], 6, c["mask"],
                                          None)
    assert torch.equal(out, run(c))


def test_refusals():
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)   # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)   # noqa: E731
    good = dict(q=b(3, 4, 64), k_cache=b(2, 16, 2, 64), v_cache=b(2, 16, 2, 64), block_table=i(2, 5), cu=i(3),
                seq_lens=i(2), max_new=5)
    wide = b(2, 16, 2, 68)[..., :64]
    for bad in (dict(q=b(3, 4, 60), k_cache=b(2, 16, 2, 60), v_cache=b(2, 16, 2, 60)),
                dict(q=b(3, 4, 264), k_cache=b(2, 16, 2, 264), v_cache=b(2, 16, 2, 264)),
                dict(q=b(3, 3, 64)), dict(q=b(3, 64)), dict(q=b(3, 64, 4).transpose(1, 2)), dict(v_cache=b(2, 16, 1, 64)),
                dict(k_cache=b(2, 12, 2, 64), v_cache=b(2, 12, 2, 64)), dict(k_cache=wide, v_cache=wide),
                dict(k_cache=b(0, 16, 2, 64), v_cache=b(0, 16, 2, 64)), dict(max_new=0), dict(max_new=65),
                dict(cu=i(2)), dict(cu=i(3).long()), dict(seq_lens=i(2).long()), dict(block_table=i(3, 5)),
                dict(block_table=i(5, 2).t()), dict(block_table=i(2, 0)), dict(mask=i(3)),
                dict(q=b(3, 258, 64)), dict(mask=i(4).long()), dict(out=b(3, 4, 63)), {}):
        with pytest.raises(ValueError):
            A.tree_attention(**{**good, **bad})
    for bad in (dict(q=b(3, 4, 64).float()), dict(v_cache=b(2, 16, 2, 64).half()), dict(out=b(3, 4, 64).half())):
        with pytest.raises(TypeError):
            A.tree_attention(**{**good, **bad})


@pytest.mark.gpu
@pytest.mark.parametrize("G", [1, 8, 20], ids=["32 rows", "64 rows", "more"])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_every_kernel(D, G):
    """Each head size with few and many rows: other scales, several row tiles, a long context that is cut into parts,
    and what a row may not see, wild values in the step's own rows among it."""
    n = 8 if G > 1 else 16
    c = make([n + 3, 700, 9000], [n, n, n], G, 1, D, 16, torch.bfloat16, seed=G, trees=True)
    check(c, run(c))
    for scale in (0.0, -0.2, 0.5):
        check(c, run(c, scale=scale), scale=scale)
    words = c["mask"].tolist()
    for b, L in enumerate((n + 3, 700, 9000)):
        hidden = [i for i in range(n) if all(i == t or not (words[b * n + t] >> i) & 1 for t in range(n))]
        for i in hidden[:2]:   # leaves: only their own row sees them
            for what, (cache, x) in enumerate(zip((c["kc"], c["vc"]), c["keys"][b])):
                if what:
                    x[L - n + i, 0, i % D] = float("nan") if i % 2 else float("inf")
                    x[L - n + i, 0, D - 1] = -float("inf")
                    j = L - n + i
                    cache[c["table"][b, j // 16].long(), j % 16] = x[j]
    check(c, run(c))


@pytest.mark.gpu
def test_shared_blocks_and_empty_calls():
    """Requests that share a prefix's blocks; no tokens; no requests."""
    c = make([160, 0], [4, 0], 6, 2, 128, 16, torch.bfloat16, seed=11)
    d = make([160, 170], [4, 4], 6, 2, 128, 16, torch.bfloat16, seed=11)
    d["table"][1, :9] = d["table"][0, :9]   # 144 keys of the first request
    for i in range(2):
        d["keys"][1][i][:144] = d["keys"][0][i][:144]
    check(d, run(d))
    empty = c["q"][:0]
    assert A.tree_attention(empty, c["kc"], c["vc"], c["table"], c["cu"], c["lens"], 4).shape == empty.shape
    z = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    out = torch.full_like(c["q"], 3.0)
    A.tree_attention(c["q"], c["kc"], c["vc"], z, z.new_zeros(1), z[:, 0].contiguous(), 4, out=out)
    assert (out == 3).all()


@pytest.mark.gpu
def test_context_values_that_are_not_finite():
    """An infinity or NaN in the context is seen by every row of its head: the rows it reaches are not finite."""
    for Hq, D in ((2, 64), (40, 128), (8, 256)):
        c = make([300], [3], Hq, 2, D, 16, torch.bfloat16, seed=2)
        page = c["table"][0].long()
        c["vc"][page[100 // 16], 100 % 16, 0, 5] = float("inf")
        out = run(c)
        assert not torch.isfinite(out[:, :Hq // 2, 5]).any()
        assert torch.isfinite(out[:, Hq // 2:]).all() and torch.isfinite(out[:, :Hq // 2, 6]).all()
        c["kc"][page[200 // 16], 200 % 16, 1] = float("nan")
        assert run(c)[:, Hq // 2:].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("B", [400, 1100])
@pytest.mark.parametrize("Hq, Hkv, D", [(72, 1, 64), (128, 1, 128), (72, 1, 192), (128, 1, 256)])
def test_segments_of_one_tile(Hq, Hkv, D, B):
    """More than 64 rows and a few keys a request: a CTA's items are one tile each, so that its row warps go from one
    segment's "is there another" straight to the next one's."""
    lens = [1 + (7 * i) % 60 for i in range(B)]
    c = make(lens, [1] * B, Hq, Hkv, D, 16, torch.bfloat16, seed=D)
    out = run(c)
    check(c, out)
    for _ in range(20):
        assert torch.equal(run(c), out)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq", [2, 40, 160])
@pytest.mark.parametrize("masks", [False, True])
def test_far_more_tokens_than_keys(masks, Hq):
    """The largest cu an int holds, as step_tables gives it for lengths that add up past one: tokens whose keys would
    all lie before the first one see nothing; the request after them, past the rows there are, changes nothing."""
    c = make([300, 90], [3, 2], Hq, 2, 64, 16, torch.bfloat16, seed=13)
    c["mask"] = torch.full((5,), -1, dtype=torch.int64, device="cuda") if masks else None
    for n in (300 + 64, 1 << 30, (1 << 31) - 1):
        c["cu"].copy_(torch.tensor([0, n, n], dtype=torch.int32))
        assert (run(c)[:3] == 0).all(), n   # max_new is 3
    c["cu"].copy_(torch.tensor([0, 300 + 60, (1 << 31) - 1], dtype=torch.int32))   # token 60 would see the first key
    assert (run(c)[:3] == 0).all() != masks   # all bits set: the tokens see four keys


@pytest.mark.gpu
@pytest.mark.parametrize("Hq, D", [(2, 64), (100, 128), (100, 256)])
def test_segments_longer_than_the_wait_bound(Hq, D):
    """One request whose share of a CTA takes longer than a wait inside a CTA may: no wait is for a whole segment, so
    the call is as it was and no status is left."""
    from vllm_turing_b200 import _build
    L = _build.load()
    g = torch.Generator(device="cuda").manual_seed(D)
    kc, vc = [torch.randn(64, 16, 1, D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2)]
    q = torch.randn(1, Hq, D, generator=g, device="cuda").to(torch.bfloat16)
    width = 1 << 20   # 16M keys, the cache's 64 blocks over and over
    table = (torch.arange(width, device="cuda", dtype=torch.int32) % 64)[None].contiguous()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    args = (q, kc, vc, table, i32([0, 1]), i32([16 * width]), 1)
    want = A.tree_attention(*args)
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    A.tree_attention(*args)
    b.record()
    b.synchronize()
    assert a.elapsed_time(b) > 0.5   # ms
    assert L.vt_status(0) == 0
    try:
        L.vt_set_wait_bounds(0.2, 0.0)
        got = A.tree_attention(*args)
        torch.cuda.synchronize()
    finally:
        L.vt_set_wait_bounds(2000.0, 0.0)
        status = L.vt_status(1)
    assert status == 0, hex(status)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("q_scale", [1.5, 40.0], ids=["", "weights that underflow"])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("G, n", [(1, 1), (6, 5), (12, 5), (8, 16), (40, 1), (16, 20)])
@pytest.mark.parametrize("D", [64, 80, 128, 192, 256])
def test_infinities_of_the_context_stay_infinities(D, G, n, dtype, q_scale):
    """An infinite value that a row sees with any weight makes the row's value that infinity, one of either sign or a
    NaN makes it NaN, whatever the number of rows and wherever the context is cut; the rest does not change."""
    inf, nan = float("inf"), float("nan")
    c = make([n + 1, 300 + n, 20000], [n, n, n], 2 * G, 2, D, 16, DT[dtype], seed=D + G, q_scale=q_scale, trees=n > 1)
    clean = run(c)
    check(c, clean)
    puts = {0: [(0, 0, 0, inf), (0, 1, D - 1, -inf)],
            1: [(299, 0, 3, -inf), (150, 0, 3, -inf), (5, 0, 7, inf), (290, 0, 7, -inf), (130, 1, 9, nan), (299, 1, 60, inf)],
            2: [(0, 0, 0, inf), (9999, 0, 1, -inf), (19999 - n, 0, 2, inf), (3, 0, 4, inf), (19000, 0, 4, -inf),
                (12345, 0, 5, nan), (7777, 1, D - 1, inf)] + [(j, 1, 8, inf) for j in range(0, 19000, 500)]}
    want = clean.clone()
    for b, where in puts.items():
        rows = slice(c["host_cu"][b], c["host_cu"][b + 1])
        seen = {}
        for j, h, col, x in where:
            c["vc"][c["table"][b, j // 16].long(), j % 16, h, col] = x
            seen[h, col] = seen.get((h, col), 0.0) + x
        for (h, col), x in seen.items():
            want[rows, h * G:(h + 1) * G, col] = x
    out = run(c)
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.nan_to_num(7.0, inf, -inf), want.nan_to_num(7.0, inf, -inf))
    # a NaN in a query: its row alone
    c["q"][n, 0, 0] = nan
    out = run(c)
    assert out[n, 0].isnan().all()
    want[n, 0] = nan
    assert torch.equal(out.nan_to_num(7.0, inf, -inf), want.nan_to_num(7.0, inf, -inf))


def test_inputs_that_require_a_gradient():
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)   # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)   # noqa: E731
    for which in range(3):
        x = [b(3, 4, 64), b(2, 16, 2, 64), b(2, 16, 2, 64)]
        x[which].requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            A.tree_attention(*x, i(2, 5), i(3), i(2), 5)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            A.tree_attention(*x, i(2, 5), i(3), i(2), 5)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq, n, D", [(2, 1, 128), (12, 5, 80), (16, 20, 256)])
def test_a_key_whose_values_are_all_nan(Hq, n, D):
    """One key's values of one head, or of 8 columns, among infinities before and after it: NaN there and nowhere else."""
    for L in (40, 1000, 30000):
        c = make([L + n], [n], Hq, 2, D, 16, torch.bfloat16, seed=L)
        want = run(c)
        half = Hq // 2
        page, at = c["table"][0].long(), [0, L // 3, L // 2, L - 1]
        c["vc"][page[at[0] // 16], at[0] % 16, 0, 8:24] = float("inf")
        c["vc"][page[at[1] // 16], at[1] % 16, 0, 8:16] = float("nan")
        c["vc"][page[at[3] // 16], at[3] % 16, 0, 24:40] = -float("inf")
        c["vc"][page[at[2] // 16], at[2] % 16, 1] = float("nan")
        want[:, :half, 8:16], want[:, :half, 16:24], want[:, :half, 24:40] = float("nan"), float("inf"), -float("inf")
        want[:, half:] = float("nan")
        out = run(c)
        assert torch.equal(out.isnan(), want.isnan())
        assert torch.equal(out.nan_to_num(7.0, 9e9, -9e9), want.nan_to_num(7.0, 9e9, -9e9))
