"""steptables.step_tables against one request after the other in plain Python; whole numbers, so equal."""
import pytest
import torch

from vllm_turing_b200 import steptables as S


def plain(table, held, free, count, cached, new, bs, T, parents=None):
    """The documented rules, one request at a time; returns everything the call writes."""
    width, left, status = len(table[0]), count, 0
    table, held, free = [r[:] for r in table], held[:], free[:]
    wants = [0 if n < 0 else -(-(c + n) // bs) for c, n in zip(cached, new)]
    upto, stop, top = 0, False, count
    for b, w in enumerate(wants):
        if w > width:
            status |= S.NARROW
            need = 0
        else:
            need = max(0, w - held[b]) if new[b] >= 0 else 0
        upto += need
        if upto > count:
            stop = True
            status |= S.SHORT
        if not stop:
            for _ in range(need):
                top -= 1
                table[b][held[b]] = free[top]
                held[b] += 1
    for b, n in enumerate(new):
        if n < 0:
            for j in range(held[b]):
                if top < len(free):
                    free[top] = table[b][j]
                    table[b][j] = -1
                    top += 1
                else:
                    status |= S.FREE_FULL
            held[b] = 0
    cu, pos, slots, mask = [0], [], [], []
    for b, n in enumerate(new):
        n = max(n, 0)
        if parents is not None and n > 64:
            status |= S.BIG_TREE
        for i in range(n):
            t = cu[-1] + i
            word, depth = 0, i
            if parents is not None and i < 64 and t < T:
                x, depth = i, -1
                while x >= 0:
                    word |= 1 << x
                    depth += 1
                    p = parents[cu[-1] + x]
                    x = p if p < x else -1
            pos.append(cached[b] + depth)
            mask.append(word - (1 << 64) if word >> 63 else word)
            j = cached[b] + i
            blk = table[b][j // bs] if j // bs < held[b] else -1
            slots.append(blk * bs + j % bs if blk >= 0 else -1)
        cu.append(cu[-1] + n)
    if cu[-1] > T:
        status |= S.TOO_MANY
    fit = lambda x, fill: (x + [fill] * T)[:T]   # noqa: E731
    lens = [0 if n < 0 else c + n for c, n in zip(cached, new)]
    return dict(table=table, held=held, free=free, count=[top], cu=cu, seq_lens=lens, positions=fit(pos, 0),
                slots=fit(slots, -1), mask=fit(mask, 0), status=[status])


def make(cached, new, bs, width=None, spare=5, seed=0):
    g = torch.Generator().manual_seed(seed)
    held = [-(-c // bs) for c in cached]
    need = sum(max(0, -(-(c + max(n, 0)) // bs) - h) for c, n, h in zip(cached, new, held))
    total = max(1, sum(held) + need + spare)
    order = torch.randperm(total, generator=g).tolist()
    if width is None:
        width = max([1] + [-(-(c + max(n, 0)) // bs) for c, n in zip(cached, new)])
    table, at = [], 0
    for h in held:
        table.append((order[at:at + h] + [-1] * width)[:max(width, 1)])
        at += h
    free = order[at:] + [-7] * at
    return table, held, free, total - at


def tree(new, seed):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in new:
        out += [-1 if i == 0 else int(torch.randint(-1, i, (1,), generator=g)) for i in range(max(n, 0))]
    return out


def on_gpu(table, held, free, count, cached, new, bs, T, parents=None, out=None, dev="cuda"):
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)   # noqa: E731
    t, h, f, c = i(table), i(held), i(free), i([count])
    st = S.step_tables(t, h, f, c, i(cached), i(new), bs, T, i(parents) if parents is not None else None, out)
    return (t, h, f, c), st


def compare(state, st, want, tree_mask):
    t, h, f, c = state
    got = dict(table=t, held=h, free=f, count=c, cu=st.cu, seq_lens=st.seq_lens, positions=st.positions,
               slots=st.slots, status=st.status)
    if tree_mask:
        got["mask"] = st.mask
    else:
        assert st.mask is None
    for k, v in got.items():
        assert v.tolist() == want[k], k


CASES = {
    "one": ([0], [1], 16),
    "one_token_in_cache": ([15, 16, 17], [1, 1, 1], 16),
    "none_new": ([5, 0, 9], [0, 0, 0], 8),
    "ragged": ([0, 100, 7, 31, 32, 33, 1], [64, 1, 0, 33, 32, 31, 63], 32),
    "block_of_one": ([3, 0], [4, 2], 1),
    "odd_block": ([10, 543, 544, 545], [700, 1, 0, 5], 544),
    "release_between": ([40, 90, 8, 0, 17], [5, -1, 3, -1, -5], 16),
}


@pytest.mark.gpu
@pytest.mark.parametrize("trees", [False, True])
@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("name", CASES)
def test_against_plain(name, pad, trees):
    cached, new, bs = CASES[name]
    if trees:
        new = [min(n, 64) for n in new]
    T = sum(max(n, 0) for n in new) + pad
    table, held, free, count = make(cached, new, bs)
    parents = tree(new, 1) + [-1] * pad if trees else None
    want = plain(table, held, free, count, cached, new, bs, T, parents)
    state, st = on_gpu(table, held, free, count, cached, new, bs, T, parents)
    compare(state, st, want, trees)


@pytest.mark.gpu
@pytest.mark.parametrize("B, hi, bs, trees", [(256, 64, 16, True), (1025, 5, 16, False), (4096, 2, 8, True),
                                              (33, 900, 24, False), (2, 40000, 128, False),
                                              (700, 64, 16, True)])
def test_many(B, hi, bs, trees):
    g = torch.Generator().manual_seed(B)
    cached = torch.randint(0, 300, (B,), generator=g).tolist()
    new = torch.randint(-1, hi + 1, (B,), generator=g).tolist()
    T = sum(max(n, 0) for n in new) + 2
    table, held, free, count = make(cached, new, bs)
    parents = tree(new, 2) + [-1, -1] if trees else None
    want = plain(table, held, free, count, cached, new, bs, T, parents)
    state, st = on_gpu(table, held, free, count, cached, new, bs, T, parents)
    compare(state, st, want, trees)


@pytest.mark.gpu
def test_status_bits():
    # the stack runs out at the second request: it and the later ones get nothing, tokens in held blocks keep slots
    table, held, free, count = make([4, 4, 4], [8, 20, 1], 8, width=4, spare=0)
    args = (table, held, free, 2, [4, 4, 4], [8, 20, 1], 8, 29)
    want = plain(*args)
    assert want["status"] == [S.SHORT]
    state, st = on_gpu(*args)
    compare(state, st, want, False)
    # a row too narrow, and more tokens than rows
    args = (table, held, free, 2, [4, 4, 4], [8, 60, 1], 8, 29)
    want = plain(*args)
    assert want["status"] == [S.NARROW | S.TOO_MANY]
    state, st = on_gpu(*args)
    compare(state, st, want, False)
    # a tree that is too large; parents that do not come before their token count as none
    new = [70, 3]
    table, held, free, count = make([0, 1], new, 16)
    parents = [-1] + [0] * 69 + [5, 2, 1]
    args = (table, held, free, count, [0, 1], new, 16, 73, parents)
    want = plain(*args)
    assert want["status"] == [S.BIG_TREE]
    state, st = on_gpu(*args)
    compare(state, st, want, True)
    # blocks given back that the stack has no room for
    table, held, free, count = make([32, 0], [-1, 0], 8, spare=0)
    args = (table, held, free[:3], count, [32, 0], [-1, 0], 8, 1)
    want = plain(*args)
    assert want["status"] == [S.FREE_FULL]
    state, st = on_gpu(*args)
    compare(state, st, want, False)


@pytest.mark.gpu
def test_steps_in_a_graph():
    """Captured once, replayed while the lengths change (some drafts rejected, one request ended, one begun): every
    replay gives what the plain rules give, and no block is ever held twice."""
    bs, B, T = 8, 4, 24
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    table, held, free, count = [[-1] * 12 for _ in range(B)], [0] * B, list(range(40)), 40
    t, h, f, c = i(table), i(held), i(free), i([count])
    cached, new, par = i([0] * B), i([0] * B), i([-1] * T)
    st = S.alloc_tables(B, T, True, torch.device("cuda"))
    S.step_tables(t, h, f, c, cached, new, bs, T, par, st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        S.step_tables(t, h, f, c, cached, new, bs, T, par, st)
    steps = [([0, 0, 0, 0], [9, 1, 5, 0]), ([9, 1, 2, 0], [5, 5, 5, 3]), ([10, 6, 7, 1], [5, -1, 5, 5]),
             ([15, 0, 9, 2], [5, 7, 5, 5]), ([16, 7, -0, 0], [5, 5, -1, -1]), ([20, 9, 0, 0], [5, 5, 6, 1])]
    for k, (cc, nn) in enumerate(steps):
        parents = (tree(nn, k) + [-1] * T)[:T]
        want = plain(table, held, free, count, cc, nn, bs, T, parents)
        cached.copy_(i(cc))
        new.copy_(i(nn))
        par.copy_(i(parents))
        g.replay()
        compare((t, h, f, c), st, want, True)
        table, held, free, count = want["table"], want["held"], want["free"], want["count"][0]
        ids = [x for r, n in zip(table, held) for x in r[:n]] + free[:count]
        assert sorted(ids) == list(range(40))


@pytest.mark.gpu
def test_no_requests_and_strided_table():
    z = torch.zeros(0, dtype=torch.int32, device="cuda")
    st = S.step_tables(torch.zeros(0, 3, dtype=torch.int32, device="cuda"), z, z, torch.zeros(1, dtype=torch.int32,
                       device="cuda"), z, z, 16, 4)
    assert st.cu.tolist() == [0] and st.slots.tolist() == [-1] * 4 and st.status.item() == 0
    cached, new, bs = [5, 20], [30, 1], 8
    table, held, free, count = make(cached, new, bs)
    want = plain(table, held, free, count, cached, new, bs, 31)
    big = torch.full((2, 17), -9, dtype=torch.int32, device="cuda")
    w = len(table[0])
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    big[:, :w] = i(table)
    h, f, c = i(held), i(free), i([count])
    st = S.step_tables(big[:, :w], h, f, c, i(cached), i(new), bs, 31)
    compare((big[:, :w], h, f, c), st, want, False)
    assert (big[:, w:] == -9).all()


def test_refusals():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)   # noqa: E731
    good = dict(block_table=i(2, 3), held=i(2), free_blocks=i(4), free_count=i(1), cached_lens=i(2), new_lens=i(2),
                block_size=16, num_tokens=5)
    for bad in (dict(block_table=i(3, 3)), dict(block_table=i(2, 3).long()), dict(block_table=i(3, 2).t()),
                dict(held=i(2).long()), dict(cached_lens=i(3)), dict(new_lens=i(4)[::2]), dict(free_count=i(2)),
                dict(block_size=0), dict(num_tokens=-1), dict(parents=i(4)), dict(parents=i(5).long()),
                dict(out=S.alloc_tables(2, 4, False, "cpu")), dict(out=S.alloc_tables(3, 5, False, "cpu")),
                dict(parents=i(5), out=S.alloc_tables(2, 5, False, "cpu")),
                dict(free_blocks=i(4, 1)), {}):   # {}: CPU tensors
        with pytest.raises(ValueError):
            S.step_tables(**{**good, **bad})
    n = S.MAX_REQUESTS + 1
    with pytest.raises(ValueError):
        S.step_tables(i(n, 1), i(n), i(4), i(1), i(n), i(n), 16, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("trees", [False, True])
def test_lengths_whose_sums_pass_an_int(trees):
    """cu stops at the largest int (and status says that there are more tokens than rows); the rows that there are
    belong to the first request."""
    top, T, bs = (1 << 31) - 1, 40, 16
    table, held, free, count = [[4, 7, -1], [1, -1, -1], [2, -1, -1]], [2, 1, 1], [9, 8], 2
    (t, h, f, c), st = on_gpu(table, held, free, count, [5, 10, 3], [top, top, 5], bs, T, [-1] * T if trees else None)
    assert st.cu.tolist() == [0, top, top, top]
    assert st.seq_lens.tolist() == [top, top, 8]
    assert st.status.item() == S.NARROW | S.TOO_MANY | (S.BIG_TREE if trees else 0)
    assert st.positions.tolist() == [5] * T if trees else st.positions.tolist() == list(range(5, 5 + T))
    ids = [4, 7]
    assert st.slots.tolist() == [ids[j // bs] * bs + j % bs if j < 32 else -1 for j in range(5, 5 + T)]
    assert h.tolist() == held and c.item() == 2 and t.tolist() == table


@pytest.mark.gpu
def test_blocks_whose_sum_passes_an_int():
    """Requests that need 2^20 blocks each, more than 2^31 in all: the few there are go to none of them."""
    B, width = 2100, 1 << 20
    if torch.cuda.mem_get_info()[0] < 20e9:
        pytest.skip("needs 20 GB")
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")   # noqa: E731
    table, held, free, count = i(B, width), i(B), i(8) + 3, i(1) + 8
    held[:5] = width
    st = S.step_tables(table, held, free, count, i(B) + width, i(B), 1, 0)
    assert st.status.item() == S.SHORT and count.item() == 8
    assert held.tolist() == [width] * 5 + [0] * (B - 5) and free.tolist() == [3] * 8
    assert not table[:5].any() and not (table == 3).any()


@pytest.mark.gpu
def test_an_empty_stack():
    """free_blocks without an entry: what needs a block is short of it, what is given back has no room."""
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    for cached, new, status, slots in (([3, 5], [2, 3], 0, [3, 4, 13, 14, 15, -1]),
                                       ([3, 7], [2, 3], S.SHORT, [3, 4, 15, -1, -1, -1]),
                                       ([3, 5], [-1, 3], S.FREE_FULL, [13, 14, 15, -1, -1, -1])):
        table, held, free, count = i([[0, -1], [1, -1]]), i([1, 1]), i([]), i([0])
        st = S.step_tables(table, held, free, count, i(cached), i(new), 8, 6)
        assert st.status.item() == status and st.slots.tolist() == slots and count.item() == 0
        assert held.tolist() == [0 if new[0] < 0 else 1, 1]
