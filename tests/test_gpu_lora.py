"""GPU: low-rank adapters beside a shared projection, forward and backward, against the formulas in 64
bits.

Bounds. With operands split into a TF32 head and tail, a product is off by at most 2.5 * 2^-21 of itself
(each tail loses at most 2^-21 of its operand, and tail * tail, 2^-22, is left out), a half-precision
factor's by less. Results are two such products one after the other, so 5 * 2^-21 of the sum of
their magnitudes' root of squares; sums in fp32 of up to 16 terms before a rounded addition add at most the
same again. 2^-18 (3.8e-6) of a tensor's 2-norm holds all of it for inputs without cancellation of whole
tensors, and the largest single error stays below 1e-5 of the largest value, the bar of the mul_mat path."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import normwise

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def tc():
    import trc_cuda

    trc_cuda.lib()
    return trc_cuda


def randn(seed, *shape, std=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def make(rows, k, n, ranks, kind="f32", order="runs", none=0, seed=1):
    dt = TYPES[kind]
    ad = [(randn(seed + 10 * i, r, k, std=k ** -0.5, dtype=dt), randn(seed + 10 * i + 1, n, r, std=r ** -0.5, dtype=dt), 0.5 + i % 3)
          for i, r in enumerate(ranks)]
    rng = np.random.default_rng(seed)
    ids = np.concatenate([np.arange(rows - none) % len(ranks), np.full(none, -1)]).astype(np.int32)
    ids = np.sort(ids) if order == "runs" else rng.permutation(ids)
    return ad, torch.from_numpy(ids).cuda(), randn(seed + 5, rows, k), randn(seed + 6, rows, n), randn(seed + 7, rows, n, std=1e-2)


def formula(ad, ids, x, base, dy=None, dx_base=None):
    """y, dx, [dA], [dB] in 64 bits."""
    ids, x = ids.cpu().long(), x.double().cpu()
    n = ad[0][1].shape[0]
    y = base.double().cpu().clone() if base is not None else torch.zeros(x.shape[0], n, dtype=torch.float64)
    dy = dy.double().cpu() if dy is not None else torch.zeros_like(y)
    dx = dx_base.double().cpu().clone() if dx_base is not None else torch.zeros_like(x)
    da, db = [], []
    for i, (a, b, c) in enumerate(ad):
        a, b, at = a.double().cpu(), b.double().cpu(), torch.nonzero(ids == i)[:, 0]
        h = c * (x[at] @ a.t())
        g = c * (dy[at] @ b)
        y[at] += h @ b.t()
        dx[at] += g @ a
        da.append(g.t() @ x[at])
        db.append(dy[at].t() @ h)
    return y, dx, da, db


def near(got, want, what=""):
    got, want = got.detach().double().cpu().numpy(), want.numpy()
    assert got.shape == want.shape, what
    norm = float(np.linalg.norm(want))
    off = float(np.linalg.norm(got - want))
    assert off <= 2.0 ** -18 * norm, f"{what}: 2-norm error {off / max(norm, 1e-300):.2e}"
    assert normwise(got, want) <= 1e-5, f"{what}: normwise {normwise(got, want):.2e}"


def grads_of(ad, fill=float("nan")):
    return [(torch.full(a.shape, fill, device="cuda"), torch.full(b.shape, fill, device="cuda")) for a, b, _ in ad]


def check_all(tc, rows, k, n, ranks, kind, order, none, seed=1):
    ad, ids, x, base, dy = make(rows, k, n, ranks, kind, order, none, seed)
    dx_base = randn(seed + 8, rows, k, std=1e-2)
    grads = grads_of(ad)
    handle = tc.LoraAdapters(ad, grads)
    h = tc.lora_h(handle, x).fill_(float("nan"))
    y = tc.lora(handle, x, ids, base=base, h=h)
    dx = tc.lora_back(handle, x, ids, dy, h, base=dx_base)
    wy, wdx, wda, wdb = formula(ad, ids, x, base, dy, dx_base)
    near(y, wy, "y")
    near(dx, wdx, "dx")
    for i in range(len(ad)):
        near(grads[i][0], wda[i], f"dA[{i}]")
        near(grads[i][1], wdb[i], f"dB[{i}]")
    assert tc.device_error() == 0
    return y, dx, grads


SIZES = [
    (1, 64, 64, (4,), "runs", 0),
    (1, 4096, 4096, (16,), "runs", 0),
    (3, 33, 17, (1,), "runs", 0),
    (2, 1, 1, (3,), "runs", 0),
    (16, 128, 96, (8, 8), "mixed", 3),
    (31, 100, 130, (5, 16), "mixed", 4),
    (32, 512, 256, (32,), "runs", 0),
    (33, 96, 160, (16, 7, 64), "runs", 1),
    (64, 1024, 320, (8, 16, 32, 64) * 4, "mixed", 8),
    (40, 256, 128, (16,) * 40, "mixed", 0),           # every row its own adapter
    (70, 128, 96, (256,), "runs", 0),
    (100, 4100, 515, (65, 130, 20), "mixed", 10),
    (257, 250, 513, (33, 8), "runs", 0),
    (300, 2048, 1088, (16, 16), "runs", 37),
    (1031, 516, 1030, (24, 3), "mixed", 0),
    (2050, 640, 416, (64,), "runs", 2),
    (128, 64, 36, (16,), "runs", 0),
    (129, 100, 164, (30,), "runs", 1),
    (200, 96, 160, (16, 7, 64), "mixed", 9),
    (400, 512, 260, (4, 8, 20, 16, 32, 3) * 4, "mixed", 17),
    (513, 1024, 2052, (40, 48, 64), "runs", 130),      # a tile of rows without an adapter
]


@pytest.mark.parametrize("rows,k,n,ranks,order,none", SIZES, ids=[f"{s[0]}x{s[1]}x{s[2]}r{max(s[3])}" for s in SIZES])
def test_forward_and_gradients_f32(tc, rows, k, n, ranks, order, none):
    check_all(tc, rows, k, n, ranks, "f32", order, none)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows,k,n,ranks,order,none", [SIZES[i] for i in (0, 1, 2, 5, 7, 8, 11, 12, 13, 17, 18, 20)],
                         ids=[f"{SIZES[i][0]}x{SIZES[i][1]}x{SIZES[i][2]}" for i in (0, 1, 2, 5, 7, 8, 11, 12, 13, 17, 18, 20)])
def test_forward_and_gradients_half_factors(tc, kind, rows, k, n, ranks, order, none):
    check_all(tc, rows, k, n, ranks, kind, order, none)


def test_256_adapters(tc):
    check_all(tc, 300, 64, 96, (2, 5, 9, 16) * 64, "f32", "mixed", 0)
    check_all(tc, 256, 64, 96, (2, 5, 9, 16) * 64, "f32", "mixed", 0)


@pytest.mark.parametrize("rows", [16, 17, 33, 256])
@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_small_batches_with_all_rows_on_one_adapter(tc, rows, kind):
    """A batch that is small for its many adapters, but only one of them (and -1) occurs: more rows than a tile."""
    ad, ids, x, base, dy = make(rows, 200, 136, (8, 20, 16, 33) * 5, kind, order="mixed")
    ids = torch.where(torch.arange(rows, device="cuda") % 9 == 4, -1, 6).int()
    handle = tc.LoraAdapters(ad)
    h = tc.lora_h(handle, x).fill_(float("nan"))
    want = formula(ad, ids, x, base)[0]
    y = tc.lora(handle, x, ids, base=base, h=h)
    near(y, want)
    assert torch.equal(tc.lora(handle, x, ids, base=base), y)  # with and without keeping h
    a, _, c = ad[6]
    near(h[ids == 6][:, :16], c * (x[ids == 6].double().cpu() @ a.double().cpu().t()))
    assert bool((h[ids == 6][:, 16:] == 0).all()) and bool((h[ids == -1] == 0).all())


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("k", [8, 36, 264, 2560])
@pytest.mark.parametrize("ranks", [(16, 16, 16, 16), (24, 32, 8, 4), (64, 40, 33, 64)], ids=lambda r: f"r{max(r)}")
def test_decode_batches_of_half_factors_again_and_again(tc, kind, k, ranks):
    """The two products of a decode batch share a warp's ring in two layouts, between which a lane's places change with
    half-precision factors: few columns of x (warps without a step), several groups of 16 rows, one call after another."""
    for rows, n in ((1, 2052), (13, 640), (61, 5000)):
        ad, ids, x, base, dy = make(rows, k, n, ranks, kind, order="mixed", none=rows // 9)
        if rows > 16:
            ids[ids >= 0] = 2  # all of them the same adapter's: one group after another
        handle = tc.LoraAdapters(ad)
        assert not tc.lib().trc_cuda_lora_needs_h(handle._arr, len(handle), rows)
        got = [tc.lora(handle, x, ids, base=base) for _ in range(25)]
        near(got[0], formula(ad, ids, x, base)[0])
        assert all(torch.equal(y, got[0]) for y in got)


@pytest.mark.parametrize("layout", ["offset", "transposed", "batched", "padded"])
@pytest.mark.parametrize("rows", [60, 192])
def test_strides_and_unaligned_rows(tc, layout, rows):
    """x, base and the outputs as parts of larger tensors; what lies between their elements stays."""
    k, n = 132, 136
    ad, ids, x, base, dy = make(rows, k, n, (16, 12), none=5, order="mixed")
    dx_base = randn(9, rows, k, std=1e-2)

    def place(t):
        r, c = t.shape
        if layout == "offset":
            whole = torch.full((r, c + 7), 7.0, device="cuda")
            part = whole[:, 3:3 + c]
        elif layout == "transposed":
            whole = torch.full((c, r + 1), 7.0, device="cuda")
            part = whole.t()[:r]
        elif layout == "batched":
            whole = torch.full((3, 5, r // 12, c + 4), 7.0, device="cuda")
            part = whole[:, :4, :, :c].transpose(0, 1)
            part = part.permute(1, 0, 2, 3)  # (3, 4, rows / 12, c), rows not one stride apart
        else:
            whole = torch.full((r, c + 8), 7.0, device="cuda")
            part = whole[:, :c]
        part.copy_(t.view(part.shape))
        return whole, part

    xs, bs, dys, dbs = (place(t)[1] for t in (x, base, dy, dx_base))
    out_whole, out = place(torch.zeros(rows, n, device="cuda"))
    dx_whole, dx = place(torch.zeros(rows, k, device="cuda"))
    grads = grads_of(ad)
    handle = tc.LoraAdapters(ad, grads)
    h = tc.lora_h(handle, xs)
    assert tc.lora(handle, xs, ids, base=bs, out=out, h=h) is out
    assert tc.lora_back(handle, xs, ids, dys, h, base=dbs, dx=dx) is dx
    wy, wdx, wda, wdb = formula(ad, ids, x, base, dy, dx_base)
    near(out.reshape(rows, n), wy, "y")
    near(dx.reshape(rows, k), wdx, "dx")
    for i in range(2):
        near(grads[i][0], wda[i])
        near(grads[i][1], wdb[i])
    for whole, part in ((out_whole, out), (dx_whole, dx)):
        part.fill_(7.0)
        assert bool((whole == 7.0).all())


@pytest.mark.parametrize("rows", [20, 200])
def test_broadcast_inputs_and_shared_factors(tc, rows):
    """One row of x, base and dy for all rows (stride 0); two adapters of the same factors with gradients of their own."""
    ad, ids, x, base, dy = make(rows, 128, 64, (16, 16))
    ad[1] = (ad[0][0], ad[0][1], 2.0)
    one = [t[:1].expand(rows, -1) for t in (x, base, dy)]
    grads = grads_of(ad)
    handle = tc.LoraAdapters(ad, grads)
    h = tc.lora_h(handle, one[0])
    y = tc.lora(handle, one[0], ids, base=one[1], h=h)
    dx = tc.lora_back(handle, one[0], ids, one[2], h, base=one[0])
    wy, wdx, wda, wdb = formula(ad, ids, *one, one[0])
    for got, want in ((y, wy), (dx, wdx), (grads[0][0], wda[0]), (grads[1][0], wda[1]), (grads[0][1], wdb[0]), (grads[1][1], wdb[1])):
        near(got, want)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_factors_at_odd_addresses(tc, kind):
    """Factors that start between 16-byte boundaries, as parts of one buffer, and widths of every remainder."""
    for rows, k, n in ((9, 128, 64), (50, 131, 66), (150, 128, 64), (150, 132, 68)):
        ad, ids, x, base, dy = make(rows, k, n, (16, 12), kind)
        moved = []
        for a, b, c in ad:
            flat = torch.zeros(a.numel() + b.numel() + 4, dtype=a.dtype, device="cuda")
            pa, pb = flat[1:1 + a.numel()].view(a.shape), flat[3 + a.numel():3 + a.numel() + b.numel()].view(b.shape)
            pa.copy_(a)
            pb.copy_(b)
            moved.append((pa, pb, c))
        grads = grads_of(ad)
        handle = tc.LoraAdapters(moved, grads)
        h = tc.lora_h(handle, x)
        wy, wdx, wda, wdb = formula(ad, ids, x, base, dy)
        near(tc.lora(handle, x, ids, base=base, h=h), wy)
        near(tc.lora_back(handle, x, ids, dy, h), wdx)
        near(grads[1][0], wda[1])
        near(grads[0][1], wdb[0])


def test_without_base_in_place_and_without_ids(tc):
    ad, ids, x, base, dy = make(37, 200, 90, (16,))
    handle = tc.LoraAdapters(ad)
    wy, wdx, _, _ = formula(ad, ids, x, None, dy)
    h = tc.lora_h(handle, x)
    near(tc.lora(handle, x, ids, h=h), wy)
    near(tc.lora(handle, x), wy)                      # one adapter for all rows
    near(tc.lora_back(handle, x, None, dy, h), wdx)
    y = base.clone()
    assert tc.lora(handle, x, ids, base=y, out=y) is y
    near(y, formula(ad, ids, x, base)[0])


def test_rows_without_an_adapter_keep_their_base(tc):
    """Ids outside the table: the base bit for bit, a NaN in x is not read, gradients know nothing of them."""
    rows, k, n = 50, 96, 72
    ad, ids, x, base, dy = make(rows, k, n, (16, 8), order="mixed")
    dx_base = randn(3, rows, k)
    out_of = torch.tensor([0, 7, 31, 32, 49], device="cuda")
    ids[out_of] = torch.tensor([-1, 2, 1000, -(2 ** 31), 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    wy, wdx, wda, wdb = formula(ad, ids, x, base, dy, dx_base)
    x[out_of], dy[out_of] = float("nan"), float("inf")
    grads = grads_of(ad)
    handle = tc.LoraAdapters(ad, grads)
    h = tc.lora_h(handle, x).fill_(float("nan"))
    y = tc.lora(handle, x, ids, base=base, h=h)
    dx = tc.lora_back(handle, x, ids, dy, h, base=dx_base)
    assert torch.equal(y[out_of], base[out_of]) and torch.equal(dx[out_of], dx_base[out_of])
    assert bool((h[out_of] == 0).all())
    near(y, wy)
    near(dx, wdx)
    for i in range(2):
        near(grads[i][0], wda[i])
        near(grads[i][1], wdb[i])
    assert bool((tc.lora(handle, x, ids, out=torch.full_like(base, 5.0))[out_of] == 0).all())  # no base: zero


@pytest.mark.parametrize("rows", [48, 100, 300])
def test_bad_values_stay_in_their_rows(tc, rows):
    """A NaN or an infinity in one row, or in one adapter's weights, reaches that row, or that adapter's rows."""
    k, n = 128, 64
    ad, ids, x, base, dy = make(rows, k, n, (16, 16, 16), order="mixed")
    clean = formula(ad, ids, x, base, dy)
    x[5, 3], x[6, 0] = float("nan"), float("inf")
    ad[1][0][2, 7] = float("inf")
    ad[1][1][3, 3] = float("nan")
    grads = grads_of(ad)
    handle = tc.LoraAdapters(ad, grads)
    h = tc.lora_h(handle, x)
    y = tc.lora(handle, x, ids, base=base, h=h)
    dx = tc.lora_back(handle, x, ids, dy, h)
    hit = (ids == 1).cpu()
    hit[5] = hit[6] = True
    near(y.cpu()[~hit], clean[0][~hit])
    assert not bool(torch.isfinite(y[5]).any()) and not bool(torch.isfinite(y[6]).any())
    mine = (ids == 1).cpu()
    near(dx.cpu()[~mine], clean[1][~mine])
    for i in {0, 1, 2} - {1, int(ids[5]), int(ids[6])}:
        near(grads[i][0], clean[2][i])
        near(grads[i][1], clean[3][i])


def test_gradients_of_an_adapter_without_rows(tc):
    ad, ids, x, base, dy = make(20, 64, 48, (8, 8, 8))
    ids[ids == 1] = 0
    grads = grads_of(ad)
    handle = tc.LoraAdapters(ad, grads)
    h = tc.lora_h(handle, x)
    tc.lora(handle, x, ids, h=h)
    assert tc.lora_back(handle, x, ids, dy, h, need_dx=False) is None
    assert bool((grads[1][0] == 0).all()) and bool((grads[1][1] == 0).all())
    first = [(a.clone(), b.clone()) for a, b in grads]
    tc.lora_back(handle, x, ids, dy, h, need_dx=False, accumulate=True)
    for (a, b), (fa, fb) in zip(grads, first):  # v + v is exact
        assert torch.equal(a, 2 * fa) and torch.equal(b, 2 * fb)
    grads[1][0].fill_(3.0)
    tc.lora_back(handle, x, ids, dy, h, need_dx=False, accumulate=True)
    assert bool((grads[1][0] == 3.0).all())


def test_frozen_adapters_and_no_rows(tc):
    ad, ids, x, base, dy = make(20, 64, 48, (8, 8))
    grads = grads_of(ad)
    handle = tc.LoraAdapters(ad, [(None, grads[0][1]), None])
    h = tc.lora_h(handle, x)
    tc.lora(handle, x, ids, h=h)
    wdb = formula(ad, ids, x, None, dy)[3]
    tc.lora_back(handle, x, ids, dy, h)
    near(grads[0][1], wdb[0])
    # no rows: outputs are empty, gradients zero
    handle = tc.LoraAdapters(ad, grads)
    e = x[:0]
    h = tc.lora_h(handle, e)
    assert tc.lora(handle, e, ids[:0], h=h).shape == (0, 48)
    assert tc.lora_back(handle, e, ids[:0], dy[:0], h).shape == (0, 64)
    assert all(bool((g == 0).all()) for pair in grads for g in pair)
    # no adapters: the base
    none = tc.LoraAdapters([])
    assert torch.equal(tc.lora(none, x, ids, base=base), base)


def test_gradients_agree_with_differences(tc):
    """L = sum dy * y is linear in A, in B and in x by itself, so a central difference along a direction is the
    slope itself, up to the rounding of two forward passes: 2 * 2^-18 |dy| |y| / 2 each."""
    rows, k, n = 90, 160, 224
    ad, ids, x, base, dy = make(rows, k, n, (12, 16), order="mixed", none=6)
    grads = grads_of(ad)
    handle = tc.LoraAdapters(ad, grads)
    h = tc.lora_h(handle, x)
    tc.lora(handle, x, ids, base=base, h=h)
    dx = tc.lora_back(handle, x, ids, dy, h)
    loss = lambda y: float((dy.double() * y.double()).sum())  # noqa: E731
    for t, slope in ((ad[0][0], grads[0][0]), (ad[1][1], grads[1][1]), (x, dx)):
        step, keep = randn(77, *t.shape, std=float(t.std())), t.clone()
        t.copy_(keep + step)
        up = tc.lora(handle, x, ids, base=base)
        moved = (t - keep).double()
        t.copy_(keep - step)
        back = (t - keep).double()
        down = tc.lora(handle, x, ids, base=base)
        t.copy_(keep)
        want = float((slope.double() * (moved - back)).sum())
        bound = 2.0 ** -18 * float(dy.norm()) * float(up.norm() + down.norm()) + 2.0 ** -18 * float(slope.norm() * (moved - back).norm())
        assert abs(loss(up) - loss(down) - want) <= bound


def test_equal_calls_give_equal_bits(tc):
    first = check_all(tc, 520, 768, 640, (16, 24, 8), "f32", "mixed", 11)
    again = check_all(tc, 520, 768, 640, (16, 24, 8), "f32", "mixed", 11)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    for a, b in zip(first[2], again[2]):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_streams_and_two_calls_at_once(tc):
    """Calls on two streams of their own, at once, with outputs and workspaces of their own."""
    sets = []
    for seed in (1, 50):
        ad, ids, x, base, dy = make(700, 1024, 1536, (16, 8), seed=seed)
        grads = grads_of(ad)
        sets.append((ad, ids, x, base, dy, grads, tc.LoraAdapters(ad, grads), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        got = []
        for ad, ids, x, base, dy, grads, handle, s in sets:
            with torch.cuda.stream(s):
                h = tc.lora_h(handle, x)
            y = tc.lora(handle, x, ids, base=base, h=h, stream=s)
            got.append((y, tc.lora_back(handle, x, ids, dy, h, stream=s), h))
    torch.cuda.synchronize()
    for (y, dx, _), (ad, ids, x, base, dy, grads, *_) in zip(got, sets):
        wy, wdx, wda, wdb = formula(ad, ids, x, base, dy)
        near(y, wy)
        near(dx, wdx)
        near(grads[0][0], wda[0])
        near(grads[1][1], wdb[1])


def test_h_on_the_stream_of_its_calls(tc):
    """h for calls on another stream: its memory is that stream's, so that dropping h while those calls are still
    running cannot hand it to the current stream's next tensor."""
    ad, ids, x, base, dy = make(700, 1024, 1536, (16, 8))
    grads, s = grads_of(ad), torch.cuda.Stream()
    handle = tc.LoraAdapters(ad, grads)
    wy, wdx, wda, wdb = formula(ad, ids, x, base, dy)
    torch.cuda.synchronize()
    for _ in range(3):
        h = tc.lora_h(handle, x, stream=s)
        y = tc.lora(handle, x, ids, base=base, h=h, stream=s)
        dx = tc.lora_back(handle, x, ids, dy, h, stream=s)
        at, size = h.data_ptr(), h.shape
        del h
        taken = [torch.full(size, float("nan"), device="cuda") for _ in range(8)]  # the current stream's, at once
        assert at not in [t.data_ptr() for t in taken]
        torch.cuda.synchronize()
        near(y, wy)
        near(dx, wdx)
        for i in range(2):
            near(grads[i][0], wda[i])
            near(grads[i][1], wdb[i])


def test_calls_follow_what_wrote_their_inputs(tc):
    """Kernels are set up while the one before drains: they must not read what it still writes. Inputs change
    between calls on one stream without a wait, and every result is that of its own inputs."""
    for rows, n, ranks in ((8, 96, (4, 8)), (100, 512, (16, 8)), (700, 2048, (16, 32)), (1500, 1024, (64,))):
        sets = [make(rows, 512, n, ranks, seed=s) for s in (1, 40, 80)]
        ad = [(a.clone(), b.clone(), c) for a, b, c in sets[0][0]]
        ids, x, base, dy = (t.clone() for t in sets[0][1:])
        grads = grads_of(ad)
        handle = tc.LoraAdapters(ad, grads)
        want, got = [], []
        for wait in (True, False):
            out = want if wait else got
            for _ in range(4):
                for s in sets:
                    for t, u in zip((ids, x, base, dy), s[1:]):
                        t.copy_(u)
                    for (a, b, _), (a2, b2, _) in zip(ad, s[0]):
                        a.copy_(a2)
                        b.copy_(b2)
                    if wait:
                        torch.cuda.synchronize()
                    h = tc.lora_h(handle, x)
                    y = tc.lora(handle, x, ids, base=base, h=h)
                    if wait:
                        torch.cuda.synchronize()
                    dx = tc.lora_back(handle, x, ids, dy, h, base=x)
                    if wait:
                        torch.cuda.synchronize()
                    out.append([y.clone(), dx.clone()] + [g.clone() for pair in grads for g in pair])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for u, v in zip(want, got) for a, b in zip(u, v))
        for (y, dx, *_), s in zip(want[:3], sets):
            wy, wdx, _, _ = formula(s[0], s[1], s[2], s[3], s[4], s[2])
            near(y, wy)
            near(dx, wdx)


def test_many_rows_of_many_adapters(tc):
    """More steps of rows than a gradient's CTA looks up at once, and more than one tile for every adapter."""
    rows, k, n, count = 26_000, 48, 40, 200
    ad, ids, x, base, dy = make(rows, k, n, (2, 3) * (count // 2), order="runs", none=70)
    grads = grads_of(ad)
    handle = tc.LoraAdapters(ad, grads)
    h = tc.lora_h(handle, x)
    y = tc.lora(handle, x, ids, base=base, h=h)
    dx = tc.lora_back(handle, x, ids, dy, h)
    wy, wdx, wda, wdb = formula(ad, ids, x, base, dy)
    near(y, wy)
    near(dx, wdx)
    for i in range(0, count, 13):
        near(grads[i][0], wda[i])
        near(grads[i][1], wdb[i])
    ids.copy_(ids[torch.randperm(rows, device="cuda")])  # mixed: every step has rows of many adapters
    tc.lora(handle, x, ids, h=h)
    tc.lora_back(handle, x, ids, dy, h, need_dx=False)
    _, _, wda, wdb = formula(ad, ids, x, None, dy)
    for i in range(0, count, 13):
        near(grads[i][0], wda[i])
        near(grads[i][1], wdb[i])


def test_one_adapter_without_ids_on_a_long_batch(tc):
    ad, _, x, base, dy = make(1000, 256, 384, (32,))
    grads = grads_of(ad)
    handle = tc.LoraAdapters(ad, grads)
    h = tc.lora_h(handle, x)
    y = tc.lora(handle, x, base=base, h=h)
    dx = tc.lora_back(handle, x, None, dy, h)
    wy, wdx, wda, wdb = formula(ad, torch.zeros(1000), x, base, dy)
    for got, want in ((y, wy), (dx, wdx), (grads[0][0], wda[0]), (grads[0][1], wdb[0])):
        near(got, want)


def test_captured_step_follows_its_inputs(tc):
    """A captured forward and backward: replayed after x, ids and the adapters changed in place."""
    rows, k, n = 130, 256, 192
    ad, ids, x, base, dy = make(rows, k, n, (16, 8, 24), order="mixed", none=9)
    grads = grads_of(ad)
    handle = tc.LoraAdapters(ad, grads)
    h = tc.lora_h(handle, x)
    tc.lora(handle, x, ids, base=base, h=h)
    tc.lora_back(handle, x, ids, dy, h)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = tc.lora(handle, x, ids, base=base, h=h)
        dx = tc.lora_back(handle, x, ids, dy, h)
    for seed in (3, 4):
        ad2, ids2, x2, base2, dy2 = make(rows, k, n, (16, 8, 24), order="mixed", none=9, seed=seed)
        for t, u in [(ids, ids2), (x, x2), (base, base2), (dy, dy2)] + [(p, q) for u, v in zip(ad, ad2) for p, q in zip(u[:2], v[:2])]:
            t.copy_(u)
        graph.replay()
        torch.cuda.synchronize()
        wy, wdx, wda, wdb = formula(ad, ids, x, base, dy)
        near(y, wy)
        near(dx, wdx)
        for i in range(3):
            near(grads[i][0], wda[i])
            near(grads[i][1], wdb[i])


def test_refusals(tc):
    ad, ids, x, base, dy = make(8, 64, 48, (8, 4))
    handle, err = tc.LoraAdapters(ad), tc.TrcCudaError
    h = tc.lora_h(handle, x)
    with pytest.raises(err, match="rows of 63"):
        tc.lora(handle, x[:, :63], ids)
    with pytest.raises(err, match="ids must be"):
        tc.lora(handle, x, ids[:7])
    with pytest.raises(err, match="ids must be"):
        tc.lora(handle, x, ids.long())
    with pytest.raises(err, match="single adapter"):
        tc.lora(handle, x)
    with pytest.raises(err, match="rows of 47"):
        tc.lora(handle, x, ids, base=base[:, :47])
    with pytest.raises(err, match="expected"):
        tc.lora(handle, x, ids, base=base[:7])
    with pytest.raises(err, match="float32"):
        tc.lora(handle, x.half(), ids)
    with pytest.raises(err, match="lora_h"):
        tc.lora_back(handle, x, ids, dy, h[:, :8])
    with pytest.raises(err, match="need_dx"):
        tc.lora_back(handle, x, ids, dy, h, dx=x.clone(), need_dx=False)
    with pytest.raises(err, match="invalid argument"):
        tc.lora(handle, x, ids, out=torch.empty(1, 48, device="cuda").expand(8, 48))
    shared = torch.empty(8, 64, device="cuda")
    with pytest.raises(err, match="share memory"):
        tc.LoraAdapters([ad[0], ad[0]], [(shared, None), (shared, None)])
    with pytest.raises(err, match="without adapters"):
        tc.lora(tc.LoraAdapters([]), x, ids)


@pytest.mark.parametrize("rows", [8, 200])
def test_outputs_apart_from_what_is_read(tc, rows):
    """Square projections invite it: the output in x's place, dx in dy's. Refused, because kernels still read these
    after the first rows are written. Halves of one buffer, and the base's place, are fine."""
    ad, ids, x, base, dy = make(rows, 64, 64, (8, 4))
    grads, err = grads_of(ad), tc.TrcCudaError
    handle = tc.LoraAdapters(ad, grads)
    h = tc.lora_h(handle, x)
    with pytest.raises(err, match="out shares memory"):
        tc.lora(handle, x, ids, base=base, out=x)
    with pytest.raises(err, match="out shares memory"):
        tc.lora(handle, x[:-1], ids[:-1], base=base[:-1], out=base[1:])
    with pytest.raises(err, match="out shares memory"):
        tc.lora(handle, x[:2], ids[:2], out=h.view(-1)[:128].view(2, 64), h=h[:2])
    for other in (x, dy, dy[:1].expand(rows, -1)):
        with pytest.raises(err, match="dx shares memory"):
            tc.lora_back(handle, x, ids, dy, h, dx=other)
    two = torch.empty(rows, 128, device="cuda")
    xs, out = two[:, :64], two[:, 64:]
    xs.copy_(x)
    wy, wdx, wda, wdb = formula(ad, ids, x, base, dy, base)
    near(tc.lora(handle, xs, ids, base=base, out=out, h=h), wy)
    out.copy_(base)
    near(tc.lora_back(handle, xs, ids, dy, h, base=out, dx=out), wdx)
    for i in range(2):
        near(grads[i][0], wda[i])
        near(grads[i][1], wdb[i])


def test_beside_a_packed_projection_through_a_training_step(tc):
    """The use they are for: y = W x + adapter from a packed weight, its gradients, the clipped AdamW step of all
    factors, and the next forward pass with them."""
    import synth

    rows, k, n = 150, 512, 384
    blocks = torch.from_numpy(synth.random_blocks(synth.TYPE_Q5_0, n * k // 32, seed=3)).cuda()
    w = tc.gguf_tensor_to_f32(synth.TYPE_Q5_0, blocks).view(n, k)
    ad, ids, x, _, dy = make(rows, k, n, (8, 16), none=10, order="mixed")
    grads = grads_of(ad)
    handle = tc.LoraAdapters(ad, grads)
    params, flat = [t for a, b, _ in ad for t in (a, b)], [g for pair in grads for g in pair]
    m, v = ([torch.zeros_like(p) for p in params] for _ in range(2))
    step, norm = tc.AdamwMany(params, flat, m, v), tc.SumSqrMany(flat)
    h = tc.lora_h(handle, x)
    y = tc.mul_mat_q(synth.TYPE_Q5_0, blocks, k, n, x)
    tc.lora(handle, x, ids, base=y, out=y, h=h)
    dx = tc.mul_mat_q(synth.TYPE_Q5_0, blocks, k, n, dy, transposed=True)
    tc.lora_back(handle, x, ids, dy, h, base=dx, dx=dx)
    wy, wdx, wda, wdb = formula(ad, ids, x, (x.double() @ w.double().t()), dy, dy.double() @ w.double())
    assert normwise(y.cpu().numpy(), wy.numpy()) <= 1e-5 and normwise(dx.cpu().numpy(), wdx.numpy()) <= 1e-5
    before = [p.double().cpu() for p in params]
    step([1e-3 / (1 - 0.9), (1 - 0.999) ** 0.5, 1.0, 0.9, 0.999, 1e-8], norm=norm(), max_norm=0.1)
    wg = [t for a, b in zip(wda, wdb) for t in (a, b)]
    total = sum(float(g.square().sum()) for g in wg) ** 0.5
    for p, b, g in zip(params, before, wg):  # the first step: lr * g / (|g| + eps) of the clipped gradient
        g = g * min(1.0, 0.1 / (total + 1e-6))
        want = b - 1e-3 * g / (g.abs() + 1e-8)
        # a gradient's relative error e moves its step by lr * e * eps / (|g| + eps)
        err = 2.0 ** -18 * g.norm() / g.numel() ** 0.5
        assert bool(((p.double().cpu() - want).abs() <= 2.0 ** -22 * b.abs() + 1e-3 * (2.0 ** -20 + 16 * err / (g.abs() + 1e-8))).all())
    after = tc.lora(handle, x, ids)
    near(after, formula(ad, ids, x, None)[0])
