"""GPU: AdamW over many tensors with 32-bit and 8-bit states, and the squared norm of many tensors. The
32-bit step is the one-tensor step bit for bit. With 8-bit states the codes and scales are those of the
restatement below in numpy's fp32, bit for bit (every operation is rounded by itself on both sides), and the
parameter's step is within 5 * 2^-23 of itself: root (2^-23), times the rounded 1 / bc2_sqrt (2^-24) in one
operation with eps (2^-24), quotient (2 * 2^-23), times the step size (2^-24), each at most, and the same of the
restatement (5 * 2^-24); the difference is then rounded, by half a unit of p. Norms are within an ulp of the sum
in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F = np.float32
P6 = [1e-3 / (1 - 0.9 ** 7), np.sqrt(1 - 0.999 ** 7), 1 - 1e-5, 0.9, 0.999, 1e-8]
SIZES = [[1], [255], [256], [257], [2048], [2049], [5, 4096, 1, 300, 16384, 77, 0, 33], [100_003, 8]]


@pytest.fixture(scope="module")
def tc():
    import trc_cuda

    trc_cuda.lib()
    return trc_cuda


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def host(t):
    return t.cpu().numpy()


def bits(a, b):
    a, b = (np.asarray(t, dtype=F) for t in (a, b))
    nan = np.isnan(b)
    return bool(np.array_equal(np.isnan(a), nan) and np.array_equal(a.view(np.uint32)[~nan], b.view(np.uint32)[~nan]))


def tensors(sizes, seed, std, square=False):
    rng = np.random.default_rng(seed)
    got = [(rng.standard_normal(n) * std).astype(F) for n in sizes]
    return [g * g for g in got] if square else got


# ------------------------------------------------------------------ the 8-bit forms, restated

def per_block(x):
    n = x.size
    return np.concatenate([x, np.zeros(-n % 256, dtype=F)]).reshape(-1, 256)


def encode(x, which):
    with np.errstate(all="ignore"):
        x = per_block(x.astype(F))
        mag = np.abs(x) if which == "m" else np.sqrt(x)
        top = np.where(np.isfinite(mag).all(1, keepdims=True), mag.max(1, keepdims=True), F(np.nan)).astype(F)
        if which == "m":
            top = np.where(top < F(2.0 ** -100), F(0), top)
        most, unit = (F(16129), F(1) / F(16129)) if which == "m" else (F(65025), F(1) / F(65025))
        per = np.where(top > 0, most / top, F(0)).astype(F)
        code = np.where(per > 0, np.rint(np.sqrt(mag * per)), 0)
        if which == "v":
            code = np.where((per > 0) & (mag > 0), np.maximum(code, 1), code)
        else:
            code = np.where(x < 0, -code, code)
    return code.astype(np.int8 if which == "m" else np.uint8), (top * unit).astype(F)


def decode(code, scale, which, n):
    c = code.astype(np.int32)
    u = (c * np.abs(c)).astype(F) * scale
    return (u if which == "m" else u * u).astype(F).reshape(-1)[:n]


def adamw(p, g, m, v, p6):
    step, root2, decay, b1, b2, eps = (F(q) for q in p6)
    m = m + (g - m) * (F(1) - b1)
    v = v * b2 + g * g * (F(1) - b2)
    return p * decay - step * (m / (np.sqrt(v) / root2 + eps)), m, v


def step_close(got, want, old, decay):
    """p after an 8-bit step: see above; 8 * 2^-23 of the step holds both sides' errors, and each side's p is rounded."""
    got, want, old = (t.astype(np.float64) for t in (got, want, old))
    return bool((np.abs(got - want) <= 2.0 ** -20 * np.abs(want - old * decay) + 2.0 ** -23 * np.abs(want)).all())


def clip_factor(norm, max_norm, eps):
    return min(F(1), F(max_norm) / (np.sqrt(F(norm)) + F(eps)))


# ------------------------------------------------------------------ 32-bit states

@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s[:3])))
@pytest.mark.parametrize("clip", [False, True])
def test_adamw_many_is_the_one_tensor_step(tc, sizes, clip):
    host_in = [tensors(sizes, s, d, q) for s, d, q in ((1, 1.0, False), (2, 0.1, False), (3, 0.01, False), (4, 0.03, True))]
    P, G, M, V = ([dev(t) for t in part] for part in host_in)
    P2, G2, M2, V2 = ([dev(t) for t in part] for part in host_in)
    norm = torch.tensor([float(sum((g.astype(np.float64) ** 2).sum() for g in host_in[1]))], device="cuda")
    step = tc.AdamwMany(P, G, M, V)
    assert len(step) == len(sizes)
    step(P6, **({"norm": norm, "max_norm": 0.02} if clip else {}))
    for p, g, m, v in zip(P2, G2, M2, V2):
        if not p.numel():
            continue
        if clip:
            tc.clip_scale_(g, norm, 0.02, 1e-6)
        tc.opt_step_adamw_(p, g, m, v, P6)
    for got, want in zip((P, M, V), (P2, M2, V2)):
        assert all(bits(host(a), host(b)) for a, b in zip(got, want))
    assert all(np.array_equal(host(g), h) for g, h in zip(G, host_in[1]))  # gradients stay


def test_adamw_many_edge_values(tc):
    """Infinities, NaN, zeros and denormals, as the one-tensor step treats them."""
    edge = np.array([0.0, -0.0, np.inf, -np.inf, np.nan, 1e-45, 1.2e-38, 3.4e38, 1e-20, 1.0], dtype=F)
    a = np.repeat(edge, 10)
    b = np.tile(edge, 10)
    args = [dev(t.copy()) for t in (a, b, np.abs(a[::-1]), np.abs(b))]
    ref = [t.clone() for t in args]
    tc.AdamwMany(*[[t] for t in args])(P6)
    tc.opt_step_adamw_(*ref, P6)
    for got, want in zip(args, ref):
        assert bits(host(got), host(want))


@pytest.mark.parametrize("bits_", [32, 8])
def test_many_small_tensors_and_what_lies_between_them(tc, bits_):
    """1200 tensors at every alignment of one buffer: more than a launch takes; gaps keep their values."""
    rng = np.random.default_rng(5)
    sizes = rng.integers(0, 700, 1200)
    starts = np.cumsum(np.concatenate([[3], sizes[:-1] + rng.integers(1, 4, 1199)]))
    total = int(starts[-1] + sizes[-1] + 5)
    used = np.zeros(total, bool)
    for a, n in zip(starts, sizes):
        used[a:a + n] = True
    base = [dev((rng.standard_normal(total) * s).astype(F)) for s in (1.0, 0.1, 0.01)] + [dev((rng.standard_normal(total) * 0.03).astype(F) ** 2)]
    cut = lambda t: [t[a:a + n] for a, n in zip(starts.tolist(), sizes.tolist())]  # noqa: E731
    blocks = [-(-int(n) // 256) for n in sizes]
    at = np.cumsum([0] + blocks)
    extra = ()
    if bits_ == 8:
        mc, vc = torch.full((total,), 9, dtype=torch.int8, device="cuda"), torch.full((total,), 9, dtype=torch.uint8, device="cuda")
        ms, vs = (torch.full((int(at[-1]),), 5.0, device="cuda") for _ in range(2))
        scales = [[s[a:b] for a, b in zip(at[:-1].tolist(), at[1:].tolist())] for s in (ms, vs)]
        for m, v, cm, cv, sm, sv in zip(cut(base[2]), cut(base[3]), cut(mc), cut(vc), *scales):
            tc.state8_from_f32(m.clone(), cm, sm)
            tc.state8_from_f32(v.clone(), cv, sv)
        before = [t.clone() for t in (base[0], mc, vc)]
        m0 = [host(tc.state8_to_f32(c, s)) for c, s in zip(cut(mc), scales[0])]
        v0 = [host(tc.state8_to_f32(c, s)) for c, s in zip(cut(vc), scales[1])]
        p0 = [host(t) for t in cut(base[0])]
        tc.AdamwMany(cut(base[0]), cut(base[1]), cut(mc), cut(vc), *scales)(P6)
        gap = torch.from_numpy(~used).cuda()
        for t, b in zip((base[0], mc, vc), before):
            assert torch.equal(t[gap], b[gap])
        for i in range(0, 1200, 7):
            p, m, v = adamw(p0[i], host(cut(base[1])[i]), m0[i], v0[i], P6)
            assert step_close(host(cut(base[0])[i]), p, p0[i], P6[2])
            for part, scale, x, which in ((mc, scales[0], m, "m"), (vc, scales[1], v, "v")):
                code, s = encode(x, which)
                n = int(sizes[i])
                assert np.array_equal(host(cut(part)[i]), code.reshape(-1)[:n]) and bits(host(scale[i]), s.reshape(-1))
        return
    ref = [t.clone() for t in base]
    tc.AdamwMany(*[cut(t) for t in base])(P6)
    tc.opt_step_adamw_(*ref, P6)
    for got, want, old in zip(base, ref, range(4)):
        assert bits(host(got)[used], host(want)[used])
    gap = ~used
    fresh = np.random.default_rng(5)
    fresh.integers(0, 700, 1200), fresh.integers(1, 4, 1199)
    assert bits(host(base[0])[gap], (fresh.standard_normal(total) * 1.0).astype(F)[gap])


# ------------------------------------------------------------------ 8-bit states

@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s[:3])))
def test_adamw_many_8_bit(tc, sizes):
    p, g = tensors(sizes, 1, 1.0), tensors(sizes, 2, 0.1)
    M, V = zip(*[(tc.state8_empty(n, "m"), tc.state8_empty(n, "v")) for n in sizes])
    P, G = [dev(t) for t in p], [dev(t) for t in g]
    step = tc.AdamwMany(P, G, [c for c, _ in M], [c for c, _ in V], [s for _, s in M], [s for _, s in V])
    m, v = ([np.zeros(n, dtype=F) for n in sizes] for _ in range(2))
    for it in range(4):
        norm = torch.tensor([100.0 + it], device="cuda")
        step(P6, norm=norm, max_norm=5.0)
        clip = clip_factor(100.0 + it, 5.0, 1e-6)
        for i, n in enumerate(sizes):
            if n == 0:
                continue
            want, mi, vi = adamw(p[i], g[i] * clip, m[i], v[i], P6)
            (mc, ms), (vc, vs) = encode(mi, "m"), encode(vi, "v")
            assert step_close(host(P[i]), want, p[i], P6[2])
            p[i] = host(P[i])
            assert np.array_equal(host(M[i][0]), mc.reshape(-1)[:n]) and bits(host(M[i][1]), ms.reshape(-1))
            assert np.array_equal(host(V[i][0]), vc.reshape(-1)[:n]) and bits(host(V[i][1]), vs.reshape(-1))
            m[i], v[i] = decode(mc, ms, "m", n), decode(vc, vs, "v", n)
            g[i] = (g[i] * F(0.7) + F(0.01)).astype(F)
            G[i].copy_(dev(g[i]))


@pytest.mark.parametrize("which", ["m", "v"])
@pytest.mark.parametrize("n", [1, 3, 256, 300, 5000])
def test_state8_both_ways(tc, which, n):
    x = tensors([n], 3, 0.01)[0]
    x = x * np.float32(10.0) ** np.random.default_rng(1).integers(-6, 1, n).astype(F)
    x = x * x if which == "v" else x
    codes, scales = tc.state8_empty(n, which)
    tc.state8_from_f32(dev(x), codes, scales)
    wc, ws = encode(x, which)
    assert np.array_equal(host(codes), wc.reshape(-1)[:n]) and bits(host(scales), ws.reshape(-1))
    back = host(tc.state8_to_f32(codes, scales))
    assert bits(back, decode(wc, ws, which, n))
    # half a code of the square law: |x| = c^2 s is off by at most (c + 1/4) s, plus the roundings of fp32
    s = np.repeat(ws.reshape(-1), 256)[:n].astype(np.float64)
    c = np.abs(wc.reshape(-1)[:n].astype(np.float64))
    got, want = (back, x) if which == "m" else (np.sqrt(back.astype(np.float64)), np.sqrt(x.astype(np.float64)))
    assert bool((np.abs(got.astype(np.float64) - want) <= (np.maximum(c, 1) + 0.25) * s * (1 + 1e-4)).all())
    if which == "v":
        assert bool((back[x > 0] > 0).all())


@pytest.mark.parametrize("which", ["m", "v"])
def test_state8_edge_blocks(tc, which):
    """Zero, tiny, huge, infinite and NaN blocks, each with ordinary neighbours."""
    rng = np.random.default_rng(2)
    blocks = [np.abs(rng.standard_normal(256)).astype(F) for _ in range(9)]
    blocks[1][:] = 0
    blocks[2] *= F(1e-38)
    blocks[3] *= F(1e37)
    blocks[4][17] = np.inf
    blocks[5][200] = np.nan
    blocks[6][0] = F(1e-45)
    blocks[7][:] = -1.0 if which == "v" else F(1e-33)
    x = np.concatenate(blocks)
    codes, scales = tc.state8_empty(x.size, which)
    tc.state8_from_f32(dev(x), codes, scales)
    wc, ws = encode(x, which)
    assert np.array_equal(host(codes), wc.reshape(-1)) and bits(host(scales), ws.reshape(-1))
    back = host(tc.state8_to_f32(codes, scales)).reshape(9, 256)
    assert np.isnan(back[[4, 5]]).all() and (back[1] == 0).all() and np.isfinite(back[[0, 3, 6, 8]]).all()
    assert np.isnan(back[7]).all() if which == "v" else (back[7] == 0).all()


def encode_v_above_zero(x):
    """encode(x, "v") with a block's codes of values over 0 raised to the first one that reads back as more than 0."""
    code, scale = encode(x, "v")
    every = np.arange(256).astype(F)
    for row, v, s in zip(code, per_block(x), scale):
        if np.isfinite(s[0]) and s[0] > 0:
            u = every * every * s[0]
            row[v > 0] = np.maximum(row[v > 0], int(np.flatnonzero(u * u > 0)[0]))
    return code, scale


def test_a_second_moment_over_zero_never_vanishes(tc):
    """Blocks whose roots reach down to where the square of a small code's value is 0 in fp32: from the smallest float
    on, every v > 0 reads back as more than 0, codes are the restatement's, and zeros stay zeros."""
    rng = np.random.default_rng(8)
    blocks = []
    for e in range(-149, -110, 3):  # the largest v of a block: 2^e
        v = np.ldexp(1.0, e - rng.integers(0, 40, 256)) * rng.uniform(1, 2, 256)
        v[0], v[1], v[2] = np.ldexp(1.0, e), 2.0 ** -149, 0.0
        blocks.append(v.astype(F))
    x = np.concatenate(blocks + [np.full(3, 2.0 ** -149, dtype=F)])
    assert (encode(x, "v")[0] != encode_v_above_zero(x)[0]).any()  # the blocks reach that far
    codes, scales = tc.state8_empty(x.size, "v")
    tc.state8_from_f32(dev(x), codes, scales)
    back = host(tc.state8_to_f32(codes, scales))
    assert ((back > 0) == (x > 0)).all()
    wc, ws = encode_v_above_zero(x)
    assert np.array_equal(host(codes), wc.reshape(-1)[:x.size]) and bits(host(scales), ws.reshape(-1))
    assert bits(back, decode(wc, ws, "v", x.size))
    # a step from these states, its own new ones among them, without eps: no quotient by zero
    p6 = [1e-3, 1.0, 1.0, 0.9, 0.999, 0.0]
    some = x > 0
    p, g, m = np.zeros(x.size, dtype=F), np.zeros(x.size, dtype=F), np.where(some, F(2.0 ** -60), F(0))
    P, G, (MC, MS) = dev(p), dev(g), tc.state8_empty(x.size, "m")
    tc.state8_from_f32(dev(m), MC, MS)
    step = tc.AdamwMany([P], [G], [MC], [codes], [MS], [scales])
    m0, v0 = host(tc.state8_to_f32(MC, MS)), back
    for _ in range(2):
        before = host(P)
        step(p6)
        with np.errstate(all="ignore"):
            want, m1, v1 = adamw(before, g, m0, v0, p6)
        assert np.isfinite(host(P)[some]).all() and step_close(host(P)[some], want[some], before[some], F(1))
        wc, ws = encode_v_above_zero(v1)
        assert np.array_equal(host(codes), wc.reshape(-1)[:x.size]) and bits(host(scales), ws.reshape(-1))
        m0, v0 = host(tc.state8_to_f32(MC, MS)), host(tc.state8_to_f32(codes, scales))
        assert ((v0 > 0) == (v1 > 0)).all()
        P[~dev(some)] = 0.0  # 0 / 0 where nothing ever was


# ------------------------------------------------------------------ the norm

@pytest.mark.parametrize("sizes", SIZES + [[0], [], [16384, 16385], [3] * 2500], ids=lambda s: "x".join(map(str, s[:3])) or "none")
def test_sum_sqr_many(tc, sizes):
    x = tensors(sizes, 9, 3.0)
    T = [dev(t) for t in x]
    got = tc.SumSqrMany(T)()
    want = F(sum((t.astype(np.float64) ** 2).sum() for t in x))
    assert abs(int(host(got).view(np.uint32)[0]) - int(np.float32(want).view(np.uint32))) <= 1
    assert torch.equal(got, tc.SumSqrMany(T)())


def test_sum_sqr_many_unaligned_and_not_finite(tc):
    whole = torch.randn(70_001, device="cuda")
    want = F((host(whole)[1:70_000].astype(np.float64) ** 2).sum())
    got = host(tc.SumSqrMany([whole[1:30_000], whole[30_000:70_000]])())[0]
    assert abs(int(got.view(np.uint32)) - int(want.view(np.uint32))) <= 1
    whole[5] = float("inf")
    assert np.isinf(host(tc.SumSqrMany([whole])())[0])
    whole[6] = float("nan")
    assert np.isnan(host(tc.SumSqrMany([whole])())[0])
    assert host(tc.SumSqrMany([torch.full((4,), 3e38, device="cuda")])())[0] == np.inf  # beyond fp32's range


# ------------------------------------------------------------------ how they are called

def test_captured_step_reads_its_norm_on_the_device(tc):
    """Norm and step in one captured graph; the gradients and states change between replays."""
    sizes = [700, 5, 4096]
    p, g, m, v = tensors(sizes, 1, 1.0), tensors(sizes, 2, 0.1), tensors(sizes, 3, 0.01), tensors(sizes, 4, 0.03, True)
    P, G, M, V = ([dev(t) for t in part] for part in (p, g, m, v))
    step, norm = tc.AdamwMany(P, G, M, V), tc.SumSqrMany(G)
    norm()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(P6, norm=norm(), max_norm=0.5)
    for it in range(3):
        graph.replay()
        torch.cuda.synchronize()
        clip = clip_factor(F(sum((t.astype(np.float64) ** 2).sum() for t in g)), 0.5, 1e-6)
        for i in range(3):
            p[i], m[i], v[i] = adamw(p[i], g[i] * clip, m[i], v[i], P6)
            got = host(P[i]).astype(np.float64)
            # the norm may be an ulp off: a relative 2^-23 of the step
            assert bool((np.abs(got - p[i]) <= 2.0 ** -23 * np.abs(p[i]) + 2.0 ** -20 * 1e-2).all())
            p[i], m[i], v[i] = host(P[i]), host(M[i]), host(V[i])
            g[i] = (g[i] * F(0.5) + F(0.1)).astype(F)
            G[i].copy_(dev(g[i]))


def test_other_streams(tc):
    """Two handles on two streams at once, each norm's workspace its own."""
    sets = []
    for seed in (1, 2):
        sizes = [100_000, 33, 65_536]
        x = [tensors(sizes, seed + 10 * i, s, q) for i, (s, q) in enumerate(((1.0, False), (0.1, False), (0.01, False), (0.03, True)))]
        T = [[dev(t) for t in part] for part in x]
        sets.append((x, T, tc.AdamwMany(*T), tc.SumSqrMany(T[1]), torch.cuda.Stream()))
    torch.cuda.synchronize()
    norms = []
    for _, _, step, norm, s in sets:
        norms.append(norm(stream=s))
        step(P6, norm=norms[-1], max_norm=1e9, stream=s)
    torch.cuda.synchronize()
    for (x, T, *_), norm in zip(sets, norms):
        want = F(sum((t.astype(np.float64) ** 2).sum() for t in x[1]))
        assert abs(float(norm[0]) - float(want)) <= 2.0 ** -23 * float(want)
        for i in range(3):
            p, m, v = adamw(*(part[i] for part in x), P6)
            assert bits(host(T[0][i]), p) and bits(host(T[2][i]), m) and bits(host(T[3][i]), v)


def test_refusals(tc):
    err = tc.TrcCudaError
    f = lambda n: torch.zeros(n, device="cuda")  # noqa: E731
    p = f(8)
    with pytest.raises(err, match="share memory"):
        tc.AdamwMany([p, p], [f(8), f(8)], [f(8), f(8)], [f(8), f(8)])
    with pytest.raises(err, match="share memory"):
        tc.AdamwMany([p], [f(8)], [p], [f(8)])
    with pytest.raises(err, match="8 elements"):
        tc.AdamwMany([p], [f(7)], [f(8)], [f(8)])
    with pytest.raises(err, match="int8"):
        tc.AdamwMany([p], [f(8)], [f(8)], [f(8)], [f(1)], [f(1)])
    step = tc.AdamwMany([p], [f(8)], [f(8)], [f(8)])
    with pytest.raises(err, match="six"):
        step([1.0] * 5)
    with pytest.raises(err, match="norm"):
        step(P6, norm=f(2))
    with pytest.raises(err, match="scales"):
        tc.state8_to_f32(tc.state8_empty(300, "m")[0], f(1))
    tc.AdamwMany([], [], [], [])(P6)


def test_gradients_share_memory_with_one_another_only(tc):
    """One gradient for two tensors is right; a gradient in the place of what the step writes is refused."""
    err, x = tc.TrcCudaError, tensors([900] * 7, 3, 0.1)
    P, G, M, V = [dev(x[0]), dev(x[1])], dev(x[2]), [dev(x[3]), dev(x[4])], [dev(x[5] ** 2), dev(x[6] ** 2)]
    tc.AdamwMany(P, [G, G], M, V)(P6)
    for i in range(2):
        p, m, v = adamw(x[i], x[2], x[3 + i], x[5 + i] ** 2, P6)
        assert bits(host(P[i]), p) and bits(host(M[i]), m) and bits(host(V[i]), v)
    for other in (P[0], P[1], M[1], V[0]):
        with pytest.raises(err, match="one that is read"):
            tc.AdamwMany(P, [G, other], M, V)
    whole = torch.zeros(2000, device="cuda")
    with pytest.raises(err, match="one that is read"):
        tc.AdamwMany([whole[:900], P[1]], [whole[800:1700], G], M, V)
