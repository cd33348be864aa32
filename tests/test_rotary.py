"""rotary.rotary and rotary.rotary_cache against the rotation in 64 bits.

Tolerance of a rotated value y = f (x1 c - x2 s), derived before any run: the result is rounded once to its type, at
most eps / 2 of |y|; before that everything is 32-bit: the angle's fraction of a turn rounded to 32 bits (2^-26 turns,
2 pi 2^-26 < 2^-23), the sine and cosine (2 units, 2^-23), factor times them, two products and a sum (2^-24 each): below
2^-23 + 2^-23 + 3 2^-24 < 8 2^-24 of f (|x1| + |x2|). Values passed through are equal. fp16 results below its normal
range are off by up to 2^-25."""
import math

import pytest
import torch

from vllm_turing_b200 import rotary as R

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def freqs64(rot, base, scaling, s, orig):
    """The documented scalings, written out again in 64 bits."""
    out, factor = [], 1.0
    if scaling == "ntk":
        base = base * s ** (rot / (rot - 2))
    for i in range(rot // 2):
        w = math.exp(-2 * i / rot * math.log(base))
        if scaling == "linear":
            w /= s
        elif scaling == "yarn":
            dim = lambda n: rot * math.log(orig / (n * 2 * math.pi)) / (2 * math.log(base))   # noqa: E731
            lo, hi = max(math.floor(dim(32)), 0), min(math.ceil(dim(1)), rot - 1)
            r = min(max((i - lo) / max(hi - lo, 0.001), 0), 1)
            w = (w / s) * r + w * (1 - r)
            factor = 0.1 * math.log(s) + 1
        elif scaling == "llama3":
            turns = orig * w / (2 * math.pi)
            m = min(max((turns - 1) / 3, 0), 1)
            w = (1 - m) * w / s + m * w
        out.append(w)
    return torch.tensor(out, dtype=torch.float64), factor


def rotated(x, positions, w, factor, rot, inter, transpose):
    """(y, bound) in 64 bits on x's device."""
    w = w.to(x.device)
    a = positions.double()[:, None, None] * w * (-1 if transpose else 1)
    y = x.double().clone()
    i1 = torch.arange(0, rot, 2) if inter else torch.arange(rot // 2)
    i2 = i1 + 1 if inter else i1 + rot // 2
    x1, x2 = x.double()[..., i1], x.double()[..., i2]
    y[..., i1] = factor * (x1 * a.cos() - x2 * a.sin())
    y[..., i2] = factor * (x2 * a.cos() + x1 * a.sin())
    tol = torch.zeros_like(y)
    e = 8 * 2.0 ** -24 * factor * (x1.abs() + x2.abs()) + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    h = torch.finfo(x.dtype).eps / 2
    tol[..., i1] = h * y[..., i1].abs() + e * (1 + h)
    tol[..., i2] = h * y[..., i2].abs() + e * (1 + h)
    return y, tol


def near(got, want, tol):
    d = (got.double() - want).abs()
    assert (d <= tol).all(), f"off by {d.max().item()} at {torch.nonzero(d > tol)[:4].tolist()}"


def heads(T, H, D, dt, seed, stride_pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, H * D + stride_pad, generator=g, device="cuda").to(dt)
    return x[:, :H * D].view(T, H, D) if stride_pad else x.view(T, H, D)


SHAPES = [  # T, Hq, Hkv, D, rot, pad of the token stride
    (1, 1, 1, 64, 64, 0), (5, 24, 4, 256, 64, 0), (7, 6, 1, 256, 256, 8), (3, 3, 2, 80, 40, 0), (4, 5, 1, 96, 24, 1),
    (9, 2, 2, 128, 2, 0), (2, 4, 4, 10, 6, 0), (300, 8, 2, 192, 96, 16), (6, 1, 3, 16, 0, 0), (2, 1, 1, 1024, 1024, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("inter", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rotary(shape, inter, dtype):
    T, Hq, Hkv, D, rot, pad = shape
    q, k = heads(T, Hq, D, DT[dtype], 1, pad), heads(T, Hkv, D, DT[dtype], 2, pad)
    pos = torch.randint(0, 5000, (T,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    f = R.rope_frequencies(rot)
    w, factor = freqs64(rot, 10000.0, "none", 1.0, None)
    for transpose in (False, True):
        q0, k0 = q.clone(), k.clone()
        yq, yk = R.rotary(q, k, pos, f, inter, transpose)
        near(yq, *rotated(q0, pos, w, factor, rot, inter, transpose))
        near(yk, *rotated(k0, pos, w, factor, rot, inter, transpose))
        assert torch.equal(q, q0) and torch.equal(k, k0)
        # in place, and q alone
        qi, ki = q.clone(), k.clone()
        R.rotary(qi, ki, pos, f, inter, transpose, qi, ki)
        assert torch.equal(qi, yq) and torch.equal(ki, yk)
        only, none = R.rotary(q, None, pos, f, inter, transpose)
        assert none is None and torch.equal(only, yq)


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", R.SCALINGS)
@pytest.mark.parametrize("far", [10, 131072, 1000003, (1 << 31) + 5])
def test_scalings_at_far_positions(scaling, far):
    T, rot = 33, 128
    s = 1.0 if scaling == "none" else 8.0
    q = heads(T, 2, 128, torch.float16, 5)
    pos = far - torch.arange(T, device="cuda").clamp(max=far)
    f = R.rope_frequencies(rot, 500000.0, scaling, s, 8192)
    w, factor = freqs64(rot, 500000.0, scaling, s, 8192)
    assert f.factor == pytest.approx(factor, rel=1e-15)
    assert torch.allclose(f.turns.cpu() * 2 * math.pi, w, rtol=1e-13, atol=0)
    w = f.turns.cpu() * 2 * math.pi   # the same frequencies to the last bit, so that only the rotation is tested
    y, _ = R.rotary(q, None, pos, f)
    near(y, *rotated(q, pos, w, factor, rot, False, False))


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [False, True])
def test_transpose_is_the_gradient(inter):
    """<rotary(x), g> = <x, rotary^T(g)>, and the gradient against differences of the 64-bit rotation."""
    T, H, D, rot = 6, 3, 64, 32
    f = R.rope_frequencies(rot, 10000.0, "yarn", 4.0, 2048)
    w = f.turns.cpu() * 2 * math.pi
    pos = torch.tensor([0, 1, 77, 4096, 9999, 123456], device="cuda")
    x, g = heads(T, H, D, torch.bfloat16, 7), heads(T, H, D, torch.bfloat16, 8)
    got, _ = R.rotary(g, None, pos, f, inter, transpose=True)
    near(got, *rotated(g, pos, w, f.factor, rot, inter, True))
    # differences: d/dx_i sum(g * rotated(x)) by central differences (exact up to 64-bit rounding: the map is linear)
    h = 0.5
    for i in (0, 1, rot // 2, rot - 1, rot, D - 1):
        e = torch.zeros_like(x)
        e[..., i] = h
        hi = rotated((x.double() + e.double()).to(torch.float64).float(), pos, w, f.factor, rot, inter, False)[0]
        lo = rotated((x.double() - e.double()).to(torch.float64).float(), pos, w, f.factor, rot, inter, False)[0]
        d = ((hi - lo) * g.double()).sum(-1) / (2 * h)
        _, tol = rotated(g, pos, w, f.factor, rot, inter, True)
        assert ((got[..., i].double() - d).abs() <= tol[..., i] + 1e-9).all()


LAYOUTS = ["blocks", "heads", "joint"]


def make_cache(layout, nb, bs, H, D, dt):
    fill = 7.0
    if layout == "blocks":
        return [torch.full((nb, bs, H, D), fill, dtype=dt, device="cuda") for _ in range(2)]
    if layout == "heads":
        return [torch.full((nb, H, bs, D), fill, dtype=dt, device="cuda").transpose(1, 2) for _ in range(2)]
    both = torch.full((nb, 2, bs, H, D), fill, dtype=dt, device="cuda")
    return [both[:, 0], both[:, 1]]


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("inter", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("shape", [(5, 24, 4, 256, 64, 16), (1, 6, 1, 256, 64, 16), (130, 8, 2, 80, 40, 24),
                                   (17, 2, 2, 36, 12, 1), (64, 4, 1, 128, 128, 544)], ids=str)
def test_rotary_cache(shape, inter, layout):
    T, Hq, Hkv, D, rot, bs = shape
    dt = torch.bfloat16
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, device="cuda",
                      generator=torch.Generator(device="cuda").manual_seed(T)).to(dt)
    q, k, v = [x.view(T, -1, D) for x in qkv.split((Hq * D, Hkv * D, Hkv * D), dim=1)]
    nb = -(-T // bs) + 2
    kc, vc = make_cache(layout, nb, bs, Hkv, D, dt)
    g = torch.Generator().manual_seed(1)
    slots = torch.randperm(nb * bs, generator=g)[:T]
    if T > 4:   # no place, past the cache, far outside
        slots[1], slots[3], slots[4] = -1, nb * bs, -(1 << 40)
    pos = torch.arange(T, device="cuda") * 37
    f = R.rope_frequencies(rot)
    w, factor = freqs64(rot, 10000.0, "none", 1.0, None)
    out = R.rotary_cache(q, k, v, pos, slots.cuda(), kc, vc, f, inter)
    near(out, *rotated(q, pos, w, factor, rot, inter, False))
    yk, tol = rotated(k, pos, w, factor, rot, inter, False)
    written = torch.zeros(nb * bs, dtype=torch.bool)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < nb * bs:
            written[s] = True
            near(kc[s // bs, s % bs], yk[t], tol[t])
            assert torch.equal(vc[s // bs, s % bs], v[t])
    rest = ~written.view(nb, bs).cuda()
    assert (kc[rest] == 7).all() and (vc[rest] == 7).all()
    # q in place gives the same
    q2 = q.clone()
    R.rotary_cache(q2, k, v, pos, slots.cuda(), kc, vc, f, inter, q_out=q2)
    assert torch.equal(q2, out)


@pytest.mark.gpu
def test_cache_past_32_bit_offsets():
    """A cache of more than 2^32 elements: slots of its last block."""
    nb, bs, H, D = 32800, 64, 8, 256   # 4.3e9 elements each
    if torch.cuda.mem_get_info()[0] < 20e9:
        pytest.skip("needs 20 GB")
    kc = torch.empty(nb, bs, H, D, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    kc[-1], kc[0], vc[-1], vc[0] = 0, 0, 0, 0
    T = 3
    k, v = heads(T, H, D, torch.bfloat16, 1), heads(T, H, D, torch.bfloat16, 2)
    q = heads(T, H, D, torch.bfloat16, 3)
    slots = torch.tensor([nb * bs - 1, nb * bs - 64, 5], device="cuda")
    pos = torch.zeros(T, dtype=torch.int64, device="cuda")
    R.rotary_cache(q, k, v, pos, slots, kc, vc, R.rope_frequencies(64))
    assert torch.equal(kc[-1, 63], k[0]) and torch.equal(kc[-1, 0], k[1]) and torch.equal(kc[0, 5], k[2])
    assert torch.equal(vc[-1, 63], v[0]) and torch.equal(vc[-1, 0], v[1]) and torch.equal(vc[0, 5], v[2])
    assert (kc[-1, 1:63] == 0).all() and (kc[0, :5] == 0).all()


@pytest.mark.gpu
def test_no_tokens_and_graph():
    f = R.rope_frequencies(64)
    e = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    p = torch.empty(0, dtype=torch.int64, device="cuda")
    q, k = R.rotary(e, e, p, f)
    assert q.shape == e.shape and k.shape == e.shape
    q, pos = heads(5, 4, 64, torch.bfloat16, 1), torch.arange(5, device="cuda")
    out = torch.empty_like(q)
    R.rotary(q, None, pos, f, q_out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        R.rotary(q, None, pos, f, q_out=out)
    q.copy_(heads(5, 4, 64, torch.bfloat16, 2))
    pos += 100
    g.replay()
    w, _ = freqs64(64, 10000.0, "none", 1.0, None)
    near(out, *rotated(q, pos, w, 1.0, 64, False, False))


@pytest.mark.gpu
def test_custom_ops():
    f = R.rope_frequencies(32)
    q, k = heads(5, 4, 64, torch.bfloat16, 1), heads(5, 2, 64, torch.bfloat16, 2)
    pos = torch.arange(5, device="cuda")
    want = R.rotary(q, k, pos, f, True)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    torch.ops.vllm_turing.rotary_(qo, ko, q, k, pos, f.turns, f.factor, True, False)
    assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
    kc = torch.zeros(2, 8, 2, 64, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    qo2 = torch.empty_like(q)
    torch.ops.vllm_turing.rotary_cache_(qo2, q, k, k, pos, pos, kc, vc, f.turns, f.factor, True)
    assert torch.equal(qo2, want[0]) and torch.equal(kc[0, :5], want[1]) and torch.equal(vc[0, :5], k)


def test_refusals():
    f = R.rope_frequencies(32, device="cpu")
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)   # noqa: E731
    pos = torch.zeros(3, dtype=torch.int64)
    good = dict(q=b(3, 4, 64), k=b(3, 2, 64), positions=pos, freqs=f)
    for bad in (dict(q=b(3, 256)), dict(k=b(4, 2, 64)), dict(k=b(3, 2, 32)), dict(positions=pos.int()),
                dict(positions=torch.zeros(4, dtype=torch.int64)), dict(q_out=b(3, 4, 63)), dict(freqs=f.turns),
                dict(q=b(3, 64, 4).transpose(1, 2)), dict(q=b(3, 4, 16), k=b(3, 2, 16)), dict(k_out=b(2, 2, 64)), {}):
        with pytest.raises(ValueError):
            R.rotary(**{**good, **bad})
    for bad in (dict(q=b(3, 4, 64).float()), dict(k=b(3, 2, 64).half()), dict(q_out=b(3, 4, 64).half())):
        with pytest.raises(TypeError):
            R.rotary(**{**good, **bad})
    good = dict(q=b(3, 4, 64), k=b(3, 2, 64), v=b(3, 2, 64), positions=pos, slots=pos, k_cache=b(2, 8, 2, 64),
                v_cache=b(2, 8, 2, 64), freqs=f)
    for bad in (dict(v=b(3, 1, 64)), dict(slots=pos.int()), dict(k_cache=b(2, 8, 1, 64)), dict(v_cache=b(2, 9, 2, 64)),
                dict(k_cache=b(2, 8, 64, 2).transpose(2, 3)), dict(k=b(3, 0, 64), v=b(3, 0, 64)), {}):
        with pytest.raises(ValueError):
            R.rotary_cache(**{**good, **bad})
    with pytest.raises(TypeError):
        R.rotary_cache(**{**good, "v_cache": b(2, 8, 2, 64).half()})
    for bad in (dict(rot_dim=3), dict(rot_dim=2048), dict(rot_dim=32, scaling="other"), dict(rot_dim=32, base=0.0),
                dict(rot_dim=32, scaling="yarn", factor=2.0), dict(rot_dim=2, scaling="ntk", factor=2.0),
                dict(rot_dim=32, scaling="llama3", factor=2.0, original_length=10, low_freq_factor=4.0)):
        with pytest.raises(ValueError):
            R.rope_frequencies(device="cpu", **bad)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 36])
def test_a_cache_without_blocks(D):
    """No slot is inside it: q is rotated, nothing is written."""
    q, k, pos = heads(5, 4, D, torch.bfloat16, 1), heads(5, 2, D, torch.bfloat16, 2), torch.arange(5, device="cuda")
    f = R.rope_frequencies(12)
    kc = torch.empty(0, 16, 2, D, dtype=torch.bfloat16, device="cuda")
    out = R.rotary_cache(q, k, k, pos, pos, kc, torch.empty_like(kc), f)
    assert torch.equal(out, R.rotary(q, None, pos, f)[0])


def test_inputs_that_require_a_gradient():
    """No call records one, so none takes an input that asks for it (under no_grad the next refusal is the device)."""
    f = R.rope_frequencies(32, device="cpu")
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)   # noqa: E731
    pos = torch.zeros(3, dtype=torch.int64)
    q, k, c = b(3, 4, 64), b(3, 2, 64), b(2, 8, 2, 64)
    for wanting in ((q,), (k,), (q, k)):
        for x in wanting:
            x.requires_grad_()
        for args in ((q, k, pos, f), (q, q, pos, f)) if q.requires_grad else ((q, k, pos, f),):
            with pytest.raises(ValueError, match="gradient"):
                R.rotary(*args)
        for args in ((q, k, b(3, 2, 64)), (b(3, 4, 64), b(3, 2, 64), k)) if k.requires_grad else ((q, k, k),):
            with pytest.raises(ValueError, match="gradient"):
                R.rotary_cache(*args, pos, pos, c, c, f)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            R.rotary(q, k, pos, f)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            R.rotary_cache(q, k, k, pos, pos, c, c, f)
        for x in wanting:
            x.requires_grad_(False)


@pytest.mark.gpu
def test_the_custom_ops_refuse_a_gradient_too():
    f = R.rope_frequencies(32)
    q, k, pos = heads(5, 4, 64, torch.bfloat16, 1), heads(5, 2, 64, torch.bfloat16, 2), torch.arange(5, device="cuda")
    q.requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        torch.ops.vllm_turing.rotary_(torch.empty_like(k), None, k, q, pos, f.turns, f.factor, True, False)
    with torch.no_grad():
        out, _ = R.rotary(q, k, pos, f)
    assert torch.equal(out, R.rotary(q.detach(), None, pos, f)[0])


MANY = [  # T, Hq, Hkv, D, rot, block: several shares of heads a warp, one after the other, over most of the GPU's warps
    (8193, 24, 4, 256, 64, 16), (4099, 32, 8, 128, 128, 16), (9001, 5, 1, 80, 80, 24), (6007, 20, 2, 96, 32, 8),
    (20011, 3, 1, 64, 16, 32), (5003, 64, 8, 192, 96, 64), (70001, 1, 1, 8, 0, 8), (3001, 40, 3, 256, 256, 16),
    (2500, 9, 2, 80, 20, 16), (2203, 4, 2, 96, 24, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("inter", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("shape", MANY, ids=str)
def test_prompts(shape, inter, dtype):
    """Prompt-sized calls, every row: alone in both directions and in place, and with the cache write, where some tokens
    have no place; q, k and v as columns of one wider result."""
    T, Hq, Hkv, D, rot, bs = shape
    dt = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(T)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g, device="cuda").to(dt)
    q, k, v = [x.view(T, -1, D) for x in qkv.split((Hq * D, Hkv * D, Hkv * D), dim=1)]
    pos = torch.randint(0, 200000, (T,), generator=g, device="cuda")
    f = R.rope_frequencies(rot, 500000.0, "yarn", 4.0, 32768)
    w = f.turns.cpu() * 2 * math.pi
    for transpose in (False, True):
        yq, yk = R.rotary(q, k, pos, f, inter, transpose)
        near(yq, *rotated(q, pos, w, f.factor, rot, inter, transpose))
        near(yk, *rotated(k, pos, w, f.factor, rot, inter, transpose))
        both = qkv.clone()
        qi, ki, vi = [x.view(T, -1, D) for x in both.split((Hq * D, Hkv * D, Hkv * D), dim=1)]
        R.rotary(qi, ki, pos, f, inter, transpose, qi, ki)
        assert torch.equal(qi, yq) and torch.equal(ki, yk) and torch.equal(vi, v)
    yq, yk = R.rotary(q, k, pos, f, inter)
    nb = -(-T // bs) + 1
    slots = torch.randperm(nb * bs, generator=g, device="cuda")[:T]
    slots[torch.rand(T, generator=g, device="cuda") < 0.1] = -1
    slots[T // 3] = nb * bs
    kept = (slots >= 0) & (slots < nb * bs)
    for layout in LAYOUTS:
        kc, vc = make_cache(layout, nb, bs, Hkv, D, dt)
        want_k, want_v = kc.clone(), vc.clone()
        at = slots[kept]
        want_k[at // bs, at % bs], want_v[at // bs, at % bs] = yk[kept], v[kept]
        out = R.rotary_cache(q, k, v, pos, slots, kc, vc, f, inter)
        assert torch.equal(out, yq) and torch.equal(kc, want_k) and torch.equal(vc, want_v)
