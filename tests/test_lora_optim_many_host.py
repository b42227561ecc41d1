"""CPU: the adapter and many-tensor optimizer entry points refuse what they do not take before any CUDA
call (no device is needed), and their Python handles check tensors at construction."""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

import trc_cuda

HDR = (Path(__file__).resolve().parents[1] / "include" / "trc_cuda.h").read_text()
EINVAL, EUNSUPPORTED = -1, -2
F32, F16, BF16 = 0, 1, 30
A0, B0, X0, Y0, H0, W0 = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 0x60000  # never dereferenced


def view(n0, rows, data, nb0=4, nb1=None, n2=1, n3=1):
    nb1 = 4 * n0 if nb1 is None else nb1
    v = trc_cuda.View()
    v.data = data
    for i, (n, b) in enumerate(zip((n0, rows, n2, n3), (nb0, nb1, nb1 * rows, nb1 * rows * n2))):
        v.ne[i], v.nb[i] = n, b
    return v


def table(*entries):
    arr = (trc_cuda.LoraAdapter * max(1, len(entries)))()
    for e, (a, b, rank) in zip(arr, entries):
        e.a, e.b, e.rank, e.scale = a, b, rank, 1.0
    return arr, len(entries)


def lora(adapters=None, kind=F32, ids=0x100, x=None, base=None, d=None, h=H0):
    arr, n = adapters if adapters is not None else table((A0, B0, 4))
    x, d = x or view(64, 3, X0), d or view(32, 3, Y0)
    return trc_cuda.lib().trc_cuda_lora(kind, arr, n, ids, bytes(x), None if base is None else bytes(base), bytes(d), h, None)


def test_constants_match_the_header():
    for name, value in (("TRC_CUDA_LORA_MAX_ADAPTERS", trc_cuda.LORA_MAX_ADAPTERS), ("TRC_CUDA_LORA_MAX_RANK", trc_cuda.LORA_MAX_RANK),
                        ("TRC_CUDA_STATE8_BLOCK", trc_cuda.STATE8_BLOCK)):
        assert int(re.search(name + r"\s+(\d+)", HDR).group(1)) == value
    ids = dict(re.findall(r"(TRC_CUDA_TYPE_\w+)\s*=\s*(\d+)", HDR))
    assert int(ids["TRC_CUDA_TYPE_F16"]) == trc_cuda.TYPE_F16 and int(ids["TRC_CUDA_TYPE_BF16"]) == trc_cuda.TYPE_BF16


def test_h_row_length_is_the_largest_rank_rounded_up():
    L = trc_cuda.lib()
    for ranks, ld in (((1,), 16), ((16,), 16), ((17, 3), 32), ((256,), 256)):
        arr, n = table(*[(A0, B0, r) for r in ranks])
        assert L.trc_cuda_lora_h_ld(arr, n) == ld
    assert L.trc_cuda_lora_h_ld(None, 0) == 16
    assert L.trc_cuda_lora_h_ld(None, 1) == EINVAL
    assert L.trc_cuda_lora_needs_h(*table((A0, B0, 16)), 1) == 0 and L.trc_cuda_lora_needs_h(*table((A0, B0, 16)), 1000) == 1
    assert L.trc_cuda_lora_needs_h(*table((A0, B0, 256)), 1) == 1
    arr, n = table((A0, B0, 257))
    assert L.trc_cuda_lora_h_ld(arr, n) == EUNSUPPORTED and L.trc_cuda_lora_needs_h(arr, n, 1) == EUNSUPPORTED
    assert L.trc_cuda_lora_back_workspace_bytes(arr, n, 4) == 0
    assert L.trc_cuda_lora_back_workspace_bytes(*table((A0, B0, 17)), 4) >= 4 * 32 * 4


@pytest.mark.parametrize("want,kw", [
    (EUNSUPPORTED, {"kind": 8}),                                     # a quantized type
    (EINVAL, {"adapters": table((A0, B0, 0))}),                      # rank 0
    (EUNSUPPORTED, {"adapters": table((A0, B0, 257))}),
    (EINVAL, {"adapters": table((None, B0, 4))}),
    (EINVAL, {"adapters": table((A0, None, 4))}),
    (EINVAL, {"adapters": table((A0 + 2, B0, 4))}),                  # a float at half a float's address
    (EINVAL, {"adapters": table((A0 + 1, B0, 4)), "kind": BF16}),
    (EUNSUPPORTED, {"adapters": table(*[(A0, B0, 4)] * 257)}),
    (EINVAL, {"adapters": (None, 1)}),
    (EINVAL, {"adapters": (None, -1)}),
    (EINVAL, {"d": view(32, 4, Y0)}),                                # another number of rows
    (EINVAL, {"d": view(32, 3, Y0, n2=2)}),
    (EINVAL, {"base": view(33, 3, W0)}),
    (EINVAL, {"base": view(32, 2, W0)}),
    (EINVAL, {"x": view(0, 3, X0)}),                                 # no columns
    (EINVAL, {"x": view(64, 3, X0, nb1=258)}),                       # a stride between floats
    (EINVAL, {"x": view(64, 3, X0 + 2)}),
    (EINVAL, {"d": view(32, 3, Y0, nb1=0)}),                         # all rows written to one place
    (EINVAL, {"d": view(32, 3, Y0, nb0=0)}),
    (EUNSUPPORTED, {"x": view(64, 1 << 31, X0), "d": view(32, 1 << 31, Y0)}),
    (EUNSUPPORTED, {"x": view(64, 1 << 20, X0, n2=1 << 20), "d": view(32, 1 << 20, Y0, n2=1 << 20)}),
    (EINVAL, {"ids": 0x102}),
    (EINVAL, {"x": view(64, 300, X0), "d": view(32, 300, Y0), "h": None}),  # many rows: their h goes through memory
    (EINVAL, {"h": H0 + 4}),
    (0, {"x": view(64, 0, X0), "d": view(32, 0, Y0), "h": None}),    # no rows: nothing to do
])
def test_lora_checks_its_arguments(want, kw):
    assert lora(**kw) == want


@pytest.mark.parametrize("want,kw", [
    (EUNSUPPORTED, {"flags": 2}),
    (EINVAL, {"dy": view(32, 4, Y0)}),
    (EINVAL, {"dx": view(63, 3, W0)}),
    (EINVAL, {"dx": view(64, 3, W0, nb1=0)}),
    (EINVAL, {"base": view(64, 3, W0)}),                             # base without dx
    (EINVAL, {"dx": view(64, 3, W0), "base": view(64, 2, W0)}),
    (EINVAL, {"h": None}),
    (EINVAL, {"ws": None}),
    (EINVAL, {"ws": W0 + 4}),
    (EINVAL, {"ws_bytes": 16}),
])
def test_lora_back_checks_its_arguments(want, kw):
    arr, n = table((A0, B0, 4))
    k = {"flags": 0, "x": view(64, 3, X0), "dy": view(32, 3, Y0), "h": H0, "base": None, "dx": None, "ws": W0, "ws_bytes": 1 << 20, **kw}
    ref = lambda v: None if v is None else bytes(v)  # noqa: E731
    got = trc_cuda.lib().trc_cuda_lora_back(F32, arr, n, 0x100, ref(k["x"]), ref(k["dy"]), k["h"], ref(k["base"]), ref(k["dx"]),
                                            k["ws"], k["ws_bytes"], k["flags"], None)
    assert got == want


def step(bits=32, params=True, norm=None, **kw):
    job = (trc_cuda.AdamwJob * 1)()
    fields = {"param": A0, "grad": B0, "m": X0, "v": Y0, "m_scale": H0, "v_scale": W0, "n": 5, **kw}
    for name, value in fields.items():
        setattr(job[0], name, value)
    p6 = (ctypes.c_float * 6)(1, 1, 1, 0.9, 0.999, 1e-8) if params else None
    return trc_cuda.lib().trc_cuda_opt_step_adamw_many(job, 1, bits, p6, norm, 1.0, 1e-6, None)


@pytest.mark.parametrize("want,kw", [
    (EUNSUPPORTED, {"bits": 16}),
    (EINVAL, {"params": False}),
    (EINVAL, {"n": -1}),
    (EINVAL, {"n": (1 << 40) + 1}),
    (EINVAL, {"param": None}),
    (EINVAL, {"grad": None}),
    (EINVAL, {"m": None}),
    (EINVAL, {"v": None}),
    (EINVAL, {"param": A0 + 2}),
    (EINVAL, {"m": X0 + 1}),
    (EINVAL, {"bits": 8, "m_scale": None}),
    (EINVAL, {"bits": 8, "v_scale": None}),
    (EINVAL, {"bits": 8, "v_scale": W0 + 2}),
    (EINVAL, {"norm": 0x101}),
    (0, {"n": 0, "param": None, "grad": None}),
])
def test_adamw_many_checks_its_arguments(want, kw):
    assert step(**kw) == want


def test_adamw_many_checks_every_tensor_first():
    """A bad tensor behind 600 empty ones is found before anything is launched."""
    jobs = (trc_cuda.AdamwJob * 601)()
    jobs[600].n = 4
    p6 = (ctypes.c_float * 6)(*[1.0] * 6)
    assert trc_cuda.lib().trc_cuda_opt_step_adamw_many(jobs, 601, 32, p6, None, 1.0, 1e-6, None) == EINVAL
    assert trc_cuda.lib().trc_cuda_opt_step_adamw_many(jobs, 600, 32, p6, None, 1.0, 1e-6, None) == 0
    assert trc_cuda.lib().trc_cuda_opt_step_adamw_many(None, 1, 32, p6, None, 1.0, 1e-6, None) == EINVAL


def test_sum_sqr_many_checks_its_arguments():
    L = trc_cuda.lib()
    spans = (trc_cuda.Span * 2)()
    spans[0].data, spans[0].n = A0, 100
    spans[1].data, spans[1].n = B0, 70000
    need = L.trc_cuda_sum_sqr_many_workspace_bytes(spans, 2)
    assert need >= 16 and need % 8 == 0
    call = lambda n=2, out=Y0, ws=W0, size=need: L.trc_cuda_sum_sqr_many(spans, n, out, ws, size, None)  # noqa: E731
    assert call(out=None) == EINVAL and call(ws=None) == EINVAL and call(ws=W0 + 4) == EINVAL
    assert call(size=need - 8) == EINVAL and call(n=-1) == EINVAL and call(out=Y0 + 2) == EINVAL
    spans[1].data = None
    assert call() == EINVAL
    spans[1].data, spans[1].n = B0, -1
    assert call() == EINVAL


def test_state8_checks_its_arguments():
    L = trc_cuda.lib()
    for fn, args in ((L.trc_cuda_state8_to_f32, (A0, B0, X0)), (L.trc_cuda_state8_from_f32, (X0, A0, B0))):
        assert fn(2, *args, 4, None) == EUNSUPPORTED
        assert fn(0, *args, -1, None) == EINVAL
        assert fn(1, None, None, None, 0, None) == 0
        for i in range(3):
            assert fn(0, *[None if j == i else a for j, a in enumerate(args)], 4, None) == EINVAL


def test_handles_check_their_tensors():
    f = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype)  # noqa: E731
    err = trc_cuda.TrcCudaError
    with pytest.raises(err, match="CUDA"):
        trc_cuda.LoraAdapters([(f(4, 64), f(32, 4), 1.0)])
    with pytest.raises(err, match="rank"):
        trc_cuda.LoraAdapters([(f(4, 64), f(32, 5), 1.0)])
    with pytest.raises(err, match="outside"):
        trc_cuda.LoraAdapters([(f(300, 64), f(32, 300), 1.0)])
    with pytest.raises(err, match="float32, float16 or bfloat16"):
        trc_cuda.LoraAdapters([(f(4, 64), f(32, 4, dtype=torch.float16), 1.0)])
    with pytest.raises(err, match="contiguous"):
        trc_cuda.LoraAdapters([(f(64, 4).t(), f(32, 4), 1.0)])
    with pytest.raises(err, match="one entry"):
        trc_cuda.LoraAdapters([(f(4, 64), f(32, 4), 1.0)], [])
    with pytest.raises(err, match="at most"):
        trc_cuda.LoraAdapters([(f(4, 64), f(32, 4), 1.0)] * 257)
    with pytest.raises(err, match="one tensor for each"):
        trc_cuda.AdamwMany([f(4)], [], [f(4)], [f(4)])
    with pytest.raises(err, match="v_scale"):
        trc_cuda.AdamwMany([f(4)], [f(4)], [f(4)], [f(4)], [f(1)])
    with pytest.raises(err, match="CUDA"):
        trc_cuda.AdamwMany([f(4)], [f(4)], [f(4)], [f(4)])
    with pytest.raises(err, match="contiguous"):
        trc_cuda.SumSqrMany([f(4, 4).t()])
    with pytest.raises(err, match="int8"):
        trc_cuda.state8_to_f32(f(4), f(1))
    with pytest.raises(err, match="share memory"):
        trc_cuda._no_overlap([f(8), *f(16).split(8), (q := f(16))[:9], q[8:]], "x")
    trc_cuda._no_overlap([(q := f(16))[:8], q[8:], q[3:3]], "x")


def test_h_belongs_to_the_stream_of_the_calls_that_use_it(monkeypatch):
    """lora_h allocates as every other buffer of a call is allocated: on the stream that it is given."""
    asked = []
    monkeypatch.setattr(trc_cuda, "_scratch", lambda shape, dtype, device, stream: asked.append((shape, dtype, stream)) or torch.empty(shape))
    handle = type("Handle", (), {"ld": 32})()
    for x, rows in ((torch.zeros(5, 8), 5), (torch.zeros(2, 3, 8), 6), (torch.zeros(8), 1), (torch.zeros(0, 8), 0)):
        for stream in (None, object()):
            assert trc_cuda.lora_h(handle, x, stream=stream).shape == (rows, 32)
            assert asked.pop() == ((rows, 32), torch.float32, stream) and not asked


def test_shared_memory_of_strided_tensors():
    """Exactly the tensors with an element in common: against the sets of their elements' places."""
    buf = torch.zeros(600)
    views = [buf[:60], buf[59:90], buf[60:120], buf[:240].view(10, 24)[:, :12], buf[:240].view(10, 24)[:, 12:], buf[:240].view(10, 24)[:, 11:13],
             buf[:240].view(10, 24).t()[5:7], buf[:240].view(2, 5, 24)[:, :4, 2:9], buf[4:300:3], buf[5:300:3], buf[7:301:6], buf[3:3],
             buf[:24].expand(10, 24), buf[12:24].expand(4, 3, 12), buf[500], buf[:512].view(2, 4, 8, 8).permute(3, 0, 2, 1)[::2]]
    places = [set((torch.arange(600).as_strided(v.shape, v.stride(), v.storage_offset())).reshape(-1).tolist()) for v in views]
    for v, at in zip(views, places):
        for u, there in zip(views, places):
            assert trc_cuda._shares_memory(v, u) == bool(at & there)


def test_an_output_may_be_its_base_and_nothing_else():
    err, apart = trc_cuda.TrcCudaError, trc_cuda._apart
    out, x, h = torch.zeros(8, 16), torch.zeros(8, 16), torch.zeros(8, 16)
    apart(out, (x, None, h), None, "out")
    apart(out, (x, h), out, "out")
    apart(out, (x, h), out.view(1, 8, 16), "out")  # the same places
    both = torch.zeros(8, 32)
    apart(both[:, :16], (both[:, 16:],), None, "out")  # side by side
    apart(out[:0], (out,), None, "out")
    for read, base in (((out,), None), ((x, out[7:]), None), ((out.t(),), out), ((x,), out[:1].expand(8, 16))):
        with pytest.raises(err, match="out shares memory"):
            apart(out, read, base, "out")
    with pytest.raises(err, match="out shares memory"):
        apart(both[1:, :16], (x,), both[:7, :16], "out")  # a row behind


def test_what_is_written_and_what_is_read():
    """Read tensors may share memory with one another, and none with a written one, in whatever order they lie."""
    q, err, apart = torch.zeros(64), trc_cuda.TrcCudaError, trc_cuda._no_overlap
    apart([q[:8], q[24:32]], "x", read=[q[8:24], q[8:24], q[10:20], q[32:], q[3:3]])
    for written, read in (([q[8:16]], [q[:9]]), ([q[8:16]], [q[15:20]]), ([q[8:16]], [q]), ([q], [q[8:16]]), ([q[8:16]], [q[8:16]]),
                          ([q[:4], q[40:44]], [q[8:50], q[10:12]]), ([q[8:16]], [q[9:10], q[30:]])):
        with pytest.raises(err, match="one that is read"):
            apart(written, "x", read=read)
    with pytest.raises(err, match="written tensors share"):
        apart([q[:8], q[:20], q[7:9]], "x", read=[q[30:]])
