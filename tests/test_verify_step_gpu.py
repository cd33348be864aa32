"""The step tables, the rotary cache write and the tree attention run together, as a decode loop with drafted trees runs
them, against a model that keeps no cache: each step drafts a tree, verifies it over the paged cache, accepts a path,
moves its rows to the front of the tree's slots and goes on from there."""
import math

import pytest
import torch

from vllm_turing_b200 import rotary as R
from vllm_turing_b200 import steptables as S
from vllm_turing_b200 import treeattn as A
from vllm_turing_b200.quantfuse import scaled_int8_quant_cuda

HQ, HKV, D, ROT, BS = 6, 2, 128, 32, 16
DT = torch.bfloat16


def rotated(x, pos, turns):
    """The rotation in 64 bits, rounded to the cache's type as the kernel's result is."""
    a = pos.double()[:, None, None] * (turns * 2 * math.pi)
    y = x.double().clone()
    x1, x2 = x.double()[..., :ROT // 2], x.double()[..., ROT // 2:ROT]
    y[..., :ROT // 2], y[..., ROT // 2:ROT] = x1 * a.cos() - x2 * a.sin(), x2 * a.cos() + x1 * a.sin()
    return y.to(DT)


def attend(q, k, v):
    """One token's attention over its keys in 64 bits, and the bound of the kernel's error (see test_tree_attention)."""
    G = HQ // HKV
    kk, vv, qq = k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1), q.double()
    s = torch.einsum("hd,jhd->hj", qq, kk) * D ** -0.5
    p = torch.softmax(s, -1)
    o, a = torch.einsum("hj,jhd->hd", p, vv), torch.einsum("hj,jhd->hd", p, vv.abs())
    mag = (torch.einsum("hd,jhd->hj", qq.abs(), kk.abs()) * D ** -0.5).amax(-1)
    h = torch.finfo(DT).eps / 2
    d = (2 * D * 2.0 ** -24 * mag + 2.0 ** -21)[:, None]
    # a rotated q or k may round to its neighbour: eps of each, which moves a score by 2 eps mag and a weight, and the
    # sum of the weights, by that
    d = d + 2 * torch.finfo(DT).eps * mag[:, None]
    return o, h * o.abs() + (h + 2 * torch.expm1(d) + 2 * len(k) * 2.0 ** -24) * a * (1 + h)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_tree_decoding(graph):
    g = torch.Generator().manual_seed(5)
    dev, B, steps, most = "cuda", 3, 6, 7
    T = B * most
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)   # noqa: E731
    blocks = 40
    table, held = torch.full((B, 12), -1, dtype=torch.int32, device=dev), ints([0] * B)
    free, count = torch.randperm(blocks, generator=g).to(torch.int32).to(dev), ints([blocks])
    kc, vc = [torch.full((blocks, BS, HKV, D), float("nan"), dtype=DT, device=dev) for _ in range(2)]
    f = R.rope_frequencies(ROT, 10000.0, device=dev)
    cached, new, par = ints([0] * B), ints([0] * B), ints([-1] * T)
    st = S.alloc_tables(B, T, True, torch.device(dev))
    q, k, v = [torch.zeros(T, h, D, dtype=DT, device=dev) for h in (HQ, HKV, HKV)]
    out = torch.zeros_like(q)

    def one_step():
        S.step_tables(table, held, free, count, cached, new, BS, T, par, st)
        qr = R.rotary_cache(q, k, v, st.positions, st.slots, kc, vc, f)
        A.tree_attention(qr, kc, vc, table, st.cu, st.seq_lens, most, mask=st.mask, out=out)
        return scaled_int8_quant_cuda(out.view(T, HQ * D))

    one_step()   # no tokens: sizes what a captured step needs
    if graph:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            quant = one_step()
    past = [([], []) for _ in range(B)]   # accepted (rotated keys, values) of each request
    lens = [0] * B
    for step in range(steps):
        n = [int(torch.randint(1, most + 1, (1,), generator=g)) for _ in range(B)]
        if step == 0:
            n = [most, 3, 1]
        parents = []
        for x in n:
            parents += [-1 if i == 0 else int(torch.randint(0, i, (1,), generator=g)) for i in range(x)]
        par.copy_(ints(parents + [-1] * (T - sum(n))))
        cached.copy_(ints(lens))
        new.copy_(ints(n))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g).to(DT))
        if graph:
            gr.replay()
        else:
            quant = one_step()
        assert st.status.item() == 0
        t = 0
        for b in range(B):
            rows, pos = [], []
            for i in range(n[b]):
                path, x = [], i
                while x >= 0:
                    path.insert(0, x)
                    x = parents[t + x]
                rows.append(path)
                pos.append(lens[b] + len(path) - 1)
            pos = torch.tensor(pos, device=dev)
            assert torch.equal(st.positions[t:t + n[b]], pos)
            kr, qr = rotated(k[t:t + n[b]], pos, f.turns), rotated(q[t:t + n[b]], pos, f.turns)
            vt = v[t:t + n[b]]
            for i, path in enumerate(rows):
                keys = torch.stack(past[b][0] + [kr[j] for j in path])
                vals = torch.stack(past[b][1] + [vt[j] for j in path])
                want, tol = attend(qr[i], keys, vals)
                assert ((out[t + i].double() - want).abs() <= tol).all(), (step, b, i)
            # accept the path to a random node: its rows go to the front of the tree's slots
            path = rows[int(torch.randint(0, n[b], (1,), generator=g))]
            slots = st.slots[t:t + n[b]]
            src, dst = slots[torch.tensor(path, device=dev)], slots[:len(path)]
            for c in (kc, vc):
                flat = c.view(-1, HKV, D)
                flat[dst] = flat[src]
            past[b] = (past[b][0] + [kr[j] for j in path], past[b][1] + [vt[j].clone() for j in path])
            lens[b] += len(path)
            t += n[b]
        # what o_proj takes: the quantiser's rows are those of the attention's output
        want_q, want_s = scaled_int8_quant_cuda(out.view(T, HQ * D))
        assert torch.equal(quant[0], want_q) and torch.equal(quant[1], want_s)


@pytest.mark.gpu
def test_a_stack_that_runs_out():
    """Requests that get no blocks, over a table whose entries past what they hold are other requests' blocks: their
    tokens see what the request holds and nothing of the others."""
    dev, bs = "cuda", 16
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)   # noqa: E731
    table = ints([[0, 1, 9, 9], [2, 3, 0, 1], [4, 5, 0, 0], [6, 7, 1, 0], [8, 9, 0, 0]])
    held, free, count = ints([2] * 5), ints([10, 11]), ints([2])
    cached, new = [20] * 5, [13, 30, 60, 6, 20]
    # blocks: 1 more, 2 more (there is one left), 3 more in a row of 4 (too narrow), none, 1 more (after one not served)
    st = S.step_tables(table, held, free, count, ints(cached), ints(new), bs, sum(new))
    assert st.status.item() == S.SHORT | S.NARROW
    assert table.tolist() == [[0, 1, 11, 9], [2, 3, -1, -1], [4, 5, -1, -1], [6, 7, 1, 0], [8, 9, -1, 0]]
    assert held.tolist() == [3, 2, 2, 2, 2] and count.item() == 1
    g = torch.Generator(device=dev).manual_seed(3)
    kc, vc = [torch.randn(12, bs, HKV, D, generator=g, device=dev).to(DT) for _ in range(2)]
    q = torch.randn(sum(new), HQ, D, generator=g, device=dev).to(DT)
    out = A.tree_attention(q, kc, vc, table, st.cu, st.seq_lens, max(new))
    t = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        keys, vals = [x[table[b].long().clamp(min=0)].flatten(0, 1) for x in (kc, vc)]
        places = int(held[b]) * bs
        for i in range(n):
            m = min(c + i + 1, places)
            want, tol = attend(q[t + i], keys[:m], vals[:m])
            assert ((out[t + i].double() - want).abs() <= tol).all(), (b, i)
            j = c + i
            assert st.slots[t + i].item() == (table[b, j // bs].item() * bs + j % bs if j < places else -1)
        t += n


@pytest.mark.parametrize("layout", ["blocks", "heads", "joint"])
def test_moving_an_accepted_path(layout):
    """The lines that the integration guide gives for it, over every layout of a cache that the operators take."""
    import os
    import textwrap
    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")) as f:
        lines = textwrap.dedent([b for b in f.read().split("```python\n") if "slots[path]" in b][0].split("```")[0]
                                .replace("\n  ", "\n").lstrip())
    nb, block_size, H, d = 5, 4, 2, 3
    if layout == "heads":
        k_cache, v_cache = [torch.randn(nb, H, block_size, d).transpose(1, 2) for _ in range(2)]
    elif layout == "joint":
        both = torch.randn(nb, 2, block_size, H, d)
        k_cache, v_cache = both[:, 0], both[:, 1]
    else:
        k_cache, v_cache = [torch.randn(nb, block_size, H, d) for _ in range(2)]
    k0, v0 = k_cache.clone(), v_cache.clone()
    slots, path = torch.tensor([18, 19, 4, 5, 6, 7, 12]), torch.tensor([0, 2, 3, 6])
    exec(lines, dict(slots=slots, path=path, k_cache=k_cache, v_cache=v_cache, block_size=block_size))
    for c, c0 in ((k_cache, k0), (v_cache, v0)):
        want = c0.reshape(-1, H, d).clone()
        want[slots[:4]] = c0.reshape(-1, H, d)[slots[path]]
        assert torch.equal(c.reshape(-1, H, d), want)


@pytest.mark.gpu
def test_the_custom_ops_in_a_traced_step():
    """The four custom ops as a traced graph holds them: traced with fake tensors, run, and compared with the calls."""
    from torch.fx.experimental.proxy_tensor import make_fx
    dev, ops = "cuda", torch.ops.vllm_turing
    g = torch.Generator(device=dev).manual_seed(9)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)   # noqa: E731
    f = R.rope_frequencies(ROT, 10000.0, device=dev)
    new, most = [3, 5, 1], 5
    T = sum(new) + 2
    parents = ints([-1, 0, 0, -1, 0, 1, 1, 0, -1, -1, -1])
    q, k, v = [torch.randn(T, h, D, generator=g, device=dev).to(DT) for h in (HQ, HKV, HKV)]

    def state():
        st = S.alloc_tables(3, T, True, torch.device(dev))
        caches = [torch.zeros(12, BS, HKV, D, dtype=DT, device=dev) for _ in range(2)]
        return [torch.full((3, 4), -1, dtype=torch.int32, device=dev), ints([0] * 3),
                torch.arange(12, dtype=torch.int32, device=dev), ints([12]), *st, *caches]

    def step(table, held, free, count, cu, seq_lens, positions, slots, mask, status, kc, vc):
        cached = torch.zeros_like(held)
        ops.step_tables_(table, held, free, count, cached, lens, BS, parents, cu, seq_lens, positions, slots, mask, status)
        qr, qk, kr = torch.empty_like(q), torch.empty_like(q), torch.empty_like(k)
        ops.rotary_cache_(qr, q, k, v, positions, slots, kc, vc, f.turns, f.factor, False)
        ops.rotary_(qk, kr, q, k, positions, f.turns, f.factor, False, False)
        out = torch.zeros_like(q)
        ops.tree_attention_(out, qr, kc, vc, table, cu, seq_lens, most, mask, None)
        return out, qr, qk, kr

    lens = ints(new)
    graph = make_fx(step, tracing_mode="fake", _allow_non_fake_inputs=True)(*state())
    names = str([n.target for n in graph.graph.nodes if n.op == "call_function"])
    for op in ("step_tables_", "rotary_cache_", "rotary_", "tree_attention_"):
        assert f"vllm_turing.{op}" in names
    traced, direct = state(), state()
    got = graph(*traced)
    table, held, free, count, *tables, kc, vc = direct
    st = S.step_tables(table, held, free, count, ints([0] * 3), lens, BS, T, parents, S.StepTables(*tables))
    qr = R.rotary_cache(q, k, v, st.positions, st.slots, kc, vc, f)
    qk, kr = R.rotary(q, k, st.positions, f)
    out = A.tree_attention(qr, kc, vc, table, st.cu, st.seq_lens, most, mask=st.mask, out=torch.zeros_like(q))
    for a, b in zip((*got, *traced), (out, qr, qk, kr, *direct)):
        assert torch.equal(a, b)
    assert st.status.item() == 0 and out[:sum(new)].any() and not out[sum(new):].any()
    # without parents: no mask
    chain = state()
    ops.step_tables_(*chain[:4], ints([0] * 3), lens, BS, None, *chain[4:8], None, chain[9])
    want = S.step_tables(*state()[:4], ints([0] * 3), lens, BS, T)
    assert want.mask is None
    for a, b in zip(chain[4:8] + [chain[9]], (want.cu, want.seq_lens, want.positions, want.slots, want.status)):
        assert torch.equal(a, b)
