"""The adapter-training operators, as cases that can be measured: what a program does that fine-tunes
or serves low-rank adapters beside frozen (quantized) projections.

  lora          y = base + sum over the row's adapter of scale * B (A x), rows of many requests at once,
                each row with the adapter of its request (or none); `base` is the shared projection W x.
  lora_back     its gradients: dx = dx_base + scale * A^T B^T dy, dA, dB for every adapter.
  sum_sqr_many  the squared norm of the gradients of many tensors.
  adamw_many    one AdamW step over many tensors, with 32-bit states or states of 8 bits, clipped by
                that norm where the program clips.

With `own` false, run() computes them in elementary torch operations; with `own` true it makes the calls
a user makes.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 256  # elements that share a scale in an 8-bit state
UNIT_M, UNIT_V = float(np.float32(1 / 127 ** 2)), float(np.float32(1 / 255 ** 2))


def _tc():
    pkg = str(Path(__file__).resolve().parent.parent / "train.cpp_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import trc_cuda

    return trc_cuda


# ------------------------------------------------------------------ the cases

def _lora(name, rows, k, n, ranks, none, order, kind, train):
    case = {"op": "lora", "rows": rows, "k": k, "n": n, "ranks": ranks, "none": none, "order": order, "type": kind,
            "train": train}
    return {"name": name, **case} if name else case


def _adamw(name, model, layers, rank, bits, clip):
    case = {"op": "adamw", "model": model, "layers": layers, "rank": rank, "bits": bits, "clip": clip}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one request generates one token: latency
        _lora("lora 1 row r16 f16", 1, 4096, 4096, "16", 0, "runs", "f16", False),
        # a decode batch: 64 requests, each at its own token, 16 adapters of four ranks, a few without one
        _lora("lora decode 64 rows bf16", 64, 4096, 11008, "8,16,32,64,8,16,32,64,8,16,32,64,8,16,32,64", 8, "mixed",
              "bf16", False),
        # prompts of several requests in one batch, ragged lengths, odd ranks
        _lora("lora 1031 rows ragged f32", 1031, 4096, 14336, "16,5,24,8,33", 64, "runs", "f32", False),
        # a full prefill batch with the usual rank
        _lora("lora 4096 rows r16 f32", 4096, 4096, 14336, "16,16,16,16", 0, "runs", "f32", False),
        # training: one small adapter on a square projection
        _lora("train 512 rows r8", 512, 4096, 4096, "8", 0, "runs", "f32", True),
        # training: the step of the quantized Linear (4096 -> 14336, 2048 tokens) with an adapter
        _lora("train 2048 rows r16", 2048, 4096, 14336, "16", 0, "runs", "f32", True),
        # training of several adapters over one base model, larger ranks, ragged
        _lora("train 2048 rows r64,32", 2048, 4096, 11008, "64,32,64", 100, "runs", "f32", True),
        # the optimizer's step: one layer's adapters (14 small tensors), clipped: latency
        _adamw("adamw 1 layer r8", "adapters", 1, 8, 32, True),
        # all adapters of a 32-layer model (448 tensors)
        _adamw("adamw 448 tensors r16", "adapters", 32, 16, 32, True),
        _adamw("adamw 448 tensors r64 8-bit", "adapters", 32, 64, 8, True),
        # whole weights of one layer: few large tensors
        _adamw("adamw whole layer", "weights", 1, 0, 32, True),
        _adamw("adamw whole layer 8-bit", "weights", 1, 0, 8, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.65:
        train = rng.random() < 0.45
        top = 8 if train else 24
        while True:
            rows = _log(rng, 1, 4096)
            k, n = (_log(rng, 64, 14336) for _ in range(2))
            if rng.random() < 0.6:  # most widths are whole numbers of blocks
                k, n = -(-k // 32) * 32, -(-n // 32) * 32
            count = max(1, min(rows, _log(rng, 1, top)))
            ranks = [rng.choice([4, 8, 16, 16, 32, 64]) if rng.random() < 0.7 else rng.randint(1, 64) for _ in range(count)]
            order = rng.choice(["mixed", "runs"]) if rows <= 256 else "runs"
            none = rng.choice([0, 0, rows // 8])
            if rows - none < count:
                none = 0
            case = _lora(None, rows, k, n, ",".join(map(str, ranks)), none, order, rng.choice(["f32", "f32", "f16", "bf16"]), train)
            w = work(case)
            if w["bytes"] < 4e8 and rows * sum(ranks) * (k + n) * (3 if train else 1) < 1.8e10:
                return case
    bits, clip = rng.choice([8, 32]), rng.random() < 0.5
    if rng.random() < 0.7:
        return _adamw(None, "adapters", _log(rng, 1, 40), rng.choice([1, 3, 4, 8, 13, 16, 24, 32]), bits, clip)
    return _adamw(None, "odd", _log(rng, 1, 400), rng.randint(1, 5000), bits, clip)


def _shapes(case):
    """The sizes of the tensors of an optimizer's step."""
    if case["model"] == "weights":  # attention and MLP weights of one layer
        return [4096 * 4096] * 4 + [4096 * 11008] * 3 + [4096] * 2
    if case["model"] == "odd":  # tensors of unrelated, odd sizes
        return [1 + (case["rank"] * (i + 1) * 7919) % (40 * case["rank"] + 77) for i in range(case["layers"])]
    one = []
    for k, n in [(4096, 4096)] * 4 + [(4096, 11008)] * 2 + [(11008, 4096)]:
        one += [case["rank"] * k, n * case["rank"]]
    return one * case["layers"]


# ------------------------------------------------------------------ inputs

def _gen(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed) * 2654435761 % (1 << 62))
    return g


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _ids(case, seed):
    """The adapter of every row (-1: none); every adapter has a row."""
    rng = np.random.default_rng(seed)
    rows, count, none = case["rows"], len(case["ranks"].split(",")), case["none"]
    live = rows - none
    if case["order"] == "mixed":
        ids = np.concatenate([np.arange(live) % count, np.full(none, -1)])
        ids = rng.permutation(ids)
    else:
        cuts = np.sort(rng.choice(np.arange(1, live), count - 1, replace=False)) if count > 1 else np.array([], dtype=np.int64)
        ids = np.repeat(rng.permutation(count), np.diff(np.concatenate([[0], cuts, [live]])))
        ids = np.insert(ids, int(rng.integers(0, live + 1)), np.full(none, -1))
    return torch.from_numpy(ids.astype(np.int32)).cuda()


def _prepare_lora(case, seed):
    g, dt = _gen(seed), TYPES[case["type"]]
    rows, k, n = case["rows"], case["k"], case["n"]
    ranks = [int(r) for r in case["ranks"].split(",")]
    s = {"op": "lora", "train": case["train"], "ids": _ids(case, seed), "x": _randn(g, rows, k),
         "base": _randn(g, rows, n),
         # each adapter's two factors and its scale (alpha / rank)
         "adapters": [(_randn(g, r, k, std=k ** -0.5, dtype=dt), _randn(g, n, r, std=r ** -0.5, dtype=dt), 0.5 + i % 3)
                      for i, r in enumerate(ranks)]}
    if case["train"]:
        s["dy"], s["dx_base"] = _randn(g, rows, n, std=1e-2), _randn(g, rows, k, std=1e-2)
        s["grads"] = [(torch.empty(r, k, device="cuda"), torch.empty(n, r, device="cuda")) for r in ranks]
    owner = np.repeat(np.arange(len(ranks)), ranks)  # the adapter of every one of all the ranks
    s["owner"] = torch.from_numpy(owner.astype(np.int32)).cuda()
    s["scale"] = torch.tensor([s["adapters"][i][2] for i in owner], device="cuda")
    if own:  # the program's handle on its adapters
        s["handle"] = _tc().LoraAdapters(s["adapters"], s.get("grads"))
    return s


def _arena(sizes, dtype=torch.float32):
    """One buffer with a tensor of each size in it, each at a multiple of 256 elements, and the tensors."""
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    whole = torch.zeros(at, dtype=dtype, device="cuda")
    return whole, [whole[a:a + n] for a, n in zip(starts, sizes)]


def _live(sizes):
    whole, parts = _arena(sizes)
    torch._foreach_add_(parts, 1.0)
    return whole


HYPER = {"lr": 1e-3, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "decay": 0.01, "step": 100, "max_norm": 1.0, "clip_eps": 1e-6}


def _params6():
    h = HYPER
    return [h["lr"] / (1 - h["beta1"] ** h["step"]), math.sqrt(1 - h["beta2"] ** h["step"]), 1 - h["lr"] * h["decay"],
            h["beta1"], h["beta2"], h["eps"]]


def _encode_m(m):
    """Signed 8-bit codes with a square law: |m| ~ c * c * scale, one scale for 256 elements."""
    top = m.abs().amax(1, keepdim=True)
    top = torch.where(top < 2.0 ** -100, torch.zeros_like(top), top)
    per = torch.where(top > 0, torch.full_like(top, 16129.0) / top, torch.zeros_like(top))
    return (torch.sign(m) * torch.round(torch.sqrt(m.abs() * per))).to(torch.int8), top * UNIT_M


def _encode_v(v):
    """Unsigned 8-bit codes of the root with a square law: sqrt(v) ~ c * c * scale; no v > 0 gets the code 0."""
    u = torch.sqrt(v)
    top = u.amax(1, keepdim=True)
    per = torch.where(top > 0, torch.full_like(top, 65025.0) / top, torch.zeros_like(top))
    code = torch.maximum(torch.round(torch.sqrt(u * per)), (u > 0).float())
    return code.to(torch.uint8), top * UNIT_V


def _decode_m(codes, scale):
    c = codes.float()
    return (c * c.abs()) * scale


def _decode_v(codes, scale):
    c = codes.float()
    u = (c * c) * scale
    return u * u


def _prepare_adamw(case, seed):
    g, sizes = _gen(seed), _shapes(case)
    live = _live(sizes)
    flat = lambda std: _randn(g, live.numel(), std=std).mul_(live)  # noqa: E731
    p, grad, m = flat(0.02), flat(1e-3), flat(3e-4)
    v = flat(1e-3).square_()
    s = {"op": "adamw", "bits": case["bits"], "clip": case["clip"], "p": p, "g": grad, "params6": _params6(),
         "root2": torch.tensor(_params6()[1], device="cuda")}
    if case["bits"] == 8:
        (mc, ms), (vc, vs) = _encode_m(m.view(-1, BLOCK)), _encode_v(v.view(-1, BLOCK))
        s |= {"m": mc.view(-1), "v": vc.view(-1), "m_scale": ms.view(-1), "v_scale": vs.view(-1)}
    else:
        s |= {"m": m, "v": v}
    if own:  # the optimizer's handle: its tensors, each a part of the buffers
        tc, cut = _tc(), {}
        for key in ("p", "g", "m", "v", "m_scale", "v_scale"):
            if key in s:
                at, cut[key] = 0, []
                for n in sizes:
                    blocks = -(-n // BLOCK)
                    cut[key].append(s[key][at:at + blocks] if key.endswith("scale") else s[key][at * BLOCK:at * BLOCK + n])
                    at += blocks
        s["step"] = tc.AdamwMany(cut["p"], cut["g"], cut["m"], cut["v"], cut.get("m_scale"), cut.get("v_scale"))
        if case["clip"]:
            s["norm"] = tc.SumSqrMany(cut["g"])
    return s


def prepare(case, seed):
    return _prepare_lora(case, seed) if case["op"] == "lora" else _prepare_adamw(case, seed)


# ------------------------------------------------------------------ one pass

def _plain_lora(s):
    a = torch.cat([a for a, _, _ in s["adapters"]]).float()                       # [all ranks, k]
    b = torch.cat([b.t() for _, b, _ in s["adapters"]]).float()                   # [all ranks, n]
    ranks = [x.shape[0] for x, _, _ in s["adapters"]]
    mine = s["ids"][:, None] == s["owner"][None, :]
    zero = torch.zeros((), device="cuda")
    h = torch.where(mine, (s["x"] @ a.t()) * s["scale"], zero)
    y = s["base"] + h @ b
    if not s["train"]:
        return y
    g = torch.where(mine, (s["dy"] @ b.t()) * s["scale"], zero)
    dx = s["dx_base"] + g @ a
    da, db = (g.t() @ s["x"]).split(ranks), (s["dy"].t() @ h).split(ranks, dim=1)
    return {"y": y, "dx": dx, "da": list(da), "db": [d.contiguous() for d in db]}


def _own_lora(s):
    tc = _tc()
    if not s["train"]:
        return tc.lora(s["handle"], s["x"], s["ids"], base=s["base"])
    h = tc.lora_h(s["handle"], s["x"])
    y = tc.lora(s["handle"], s["x"], s["ids"], base=s["base"], h=h)
    dx = tc.lora_back(s["handle"], s["x"], s["ids"], s["dy"], h, base=s["dx_base"])
    return {"y": y, "dx": dx, "da": [a for a, _ in s["grads"]], "db": [b for _, b in s["grads"]]}


def _plain_adamw(s):
    step, _, decay, beta1, beta2, eps = (float(np.float32(q)) for q in s["params6"])
    g = s["g"]
    if s["clip"]:
        norm = g.double().square().sum().float()
        g = g * torch.clamp(HYPER["max_norm"] / (torch.sqrt(norm) + HYPER["clip_eps"]), max=1.0)
    if s["bits"] == 8:
        m = _decode_m(s["m"].view(-1, BLOCK), s["m_scale"].view(-1, 1)).view(-1)
        v = _decode_v(s["v"].view(-1, BLOCK), s["v_scale"].view(-1, 1)).view(-1)
    else:
        m, v = s["m"], s["v"]
    one1, one2 = float(np.float32(1) - np.float32(beta1)), float(np.float32(1) - np.float32(beta2))
    m = m + (g - m) * one1
    v = v * beta2 + (g * g) * one2
    denom = torch.sqrt(v) / s["root2"] + eps
    s["p"].copy_(s["p"] * decay - step * (m / denom))
    if s["bits"] == 8:
        (mc, ms), (vc, vs) = _encode_m(m.view(-1, BLOCK)), _encode_v(v.view(-1, BLOCK))
        for key, new in (("m", mc), ("m_scale", ms), ("v", vc), ("v_scale", vs)):
            s[key].copy_(new.view(-1))
        m, v = _decode_m(mc, ms).view(-1), _decode_v(vc, vs).view(-1)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
        m, v = s["m"], s["v"]
    out = {"p": s["p"], "m": m, "v": v}
    return {**out, "norm": norm} if s["clip"] else out


def _own_adamw(s):
    tc, norm = _tc(), None
    if s["clip"]:
        norm = s["norm"]()
        s["step"](s["params6"], norm=norm, max_norm=HYPER["max_norm"], clip_eps=HYPER["clip_eps"])
    else:
        s["step"](s["params6"])
    m, v = s["m"], s["v"]
    if s["bits"] == 8:  # the states as a checkpoint holds them
        m, v = tc.state8_to_f32(m, s["m_scale"]), tc.state8_to_f32(v, s["v_scale"])
    out = {"p": s["p"], "m": m, "v": v}
    return {**out, "norm": norm.view(())} if s["clip"] else out


def run(state):
    if state["op"] == "lora":
        return _own_lora(state) if own else _plain_lora(state)
    return _own_adamw(state) if own else _plain_adamw(state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if case["op"] == "lora":
        rows, k, n, ranks = case["rows"], case["k"], case["n"], [int(r) for r in case["ranks"].split(",")]
        live, total, item = rows - case["none"], sum(ranks), 4 if case["type"] == "f32" else 2
        # x of the rows with an adapter, their adapters, all rows of base and y
        nbytes = 4 * live * k + item * total * (k + n) + 8 * rows * n + 4 * rows
        flops = 2 * live * (total / len(ranks)) * (k + n)
        if case["train"]:  # dy, dx_base and dx, the gradients
            nbytes += 4 * live * n + 8 * rows * k + 4 * total * (k + n)
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    n = sum(_shapes(case))
    # p and the gradient read, p written; states of 32 bits read and written, or of 8 bits with a scale for
    # 256, read, written and given back as the values that they stand for
    states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8
    return {"bytes": n * (12 + states), "flops": n * (15 + (2 if case["clip"] else 0))}


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_lora(case, seed):
    s = _prepare_lora(case, seed)
    x, y, ids = s["x"].double(), s["base"].double(), s["ids"].long()
    dx = s["dx_base"].double() if case["train"] else None
    da, db = [], []
    for i, (a, b, c) in enumerate(s["adapters"]):
        rows = (ids == i).nonzero()[:, 0]
        a, b, xi = a.double(), b.double(), x[rows]
        h = c * (xi @ a.t())
        y[rows] += h @ b.t()
        if case["train"]:
            dy = s["dy"][rows].double()
            g = c * (dy @ b)
            dx[rows] += g @ a
            da.append(g.t() @ xi)
            db.append(dy.t() @ h)
    return {"y": y, "dx": dx, "da": da, "db": db} if case["train"] else y


def _exact_adamw(case, seed):
    s, h = _prepare_adamw(case, seed), HYPER
    step, root2, decay, beta1, beta2, eps = (float(np.float32(q)) for q in s["params6"])
    g = s["g"].double()
    if case["bits"] == 8:  # square law: code^2 and code^4
        c, unit = s["m"].double(), s["m_scale"].double().repeat_interleave(BLOCK)
        m = c.sign() * c.pow(2) * unit
        v = (s["v"].double().pow(2) * s["v_scale"].double().repeat_interleave(BLOCK)).pow(2)
    else:
        m, v = s["m"].double(), s["v"].double()
    norm = g.pow(2).sum()
    if case["clip"]:
        g = g * min(1.0, h["max_norm"] / (float(norm.sqrt()) + h["clip_eps"]))
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g.pow(2)
    p = decay * s["p"].double() - step * m / (v.sqrt() / root2 + eps)
    # a state of 8 bits is a rounded value: next to a border 64 bits may round to the other side
    out = {"p": p, "m": m if case["bits"] == 32 else None, "v": v if case["bits"] == 32 else None}
    return {**out, "norm": norm} if case["clip"] else out


def exact(case, seed):
    return _exact_lora(case, seed) if case["op"] == "lora" else _exact_adamw(case, seed)
