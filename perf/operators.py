"""The operators that train a gated feed-forward block of its own: what is measured.

Beside the LoRA steps, whose base weights stay frozen, a program may train a
block's own weights.  The operators are the block's normalisation (layer or
root mean square) forward and backward with the reduction of its weight's
gradient, the gated feed-forward block forward and backward, and an AdamW step
over a group of tensors with moments in 32 or in 8 bits.

``listed()`` are the fixed cases, ``draw(rng)`` more of the same ranges,
``prepare`` / ``run`` what a program holds and calls, ``work`` what a pass
cannot do without, ``exact`` the same results in 64 bits.
"""
from __future__ import annotations

import ctypes
import functools
import importlib
import math

import numpy as np
import torch

own = False

F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
TYPES = {"f32": F32, "bf16": BF16}
EPS = 1e-5


# --- the cases ------------------------------------------------------------------------------------

def listed():
    return [
        # One sequence's next token through a layer norm: latency.
        {"name": "norm_token", "op": "norm_fwd", "kind": "layer", "dtype": "bf16", "rows": 1,
         "cols": 768},
        # The larger decoder's root-mean-square norm over a step's 8192 tokens.
        {"name": "norm_fwd", "op": "norm_fwd", "kind": "rms", "dtype": "bf16", "rows": 8192,
         "cols": 2048},
        # The same step's backward pass, the weight's and the bias's gradients
        # reduced over the tokens.
        {"name": "norm_bwd", "op": "norm_bwd", "kind": "layer", "dtype": "bf16", "rows": 8192,
         "cols": 2048},
        # A ragged batch in f32, rows off every vector width.
        {"name": "norm_bwd_odd", "op": "norm_bwd", "kind": "layer", "dtype": "f32", "rows": 3001,
         "cols": 1023},
        # One token, and the tokens of 24 sequences, through a block that is served.
        {"name": "ffn_token", "op": "ffn_fwd", "dtype": "bf16", "act": "silu", "rows": 1,
         "dim": 2048, "ffn": 5632, "train": False},
        {"name": "ffn_decode", "op": "ffn_fwd", "dtype": "bf16", "act": "silu", "rows": 24,
         "dim": 2048, "ffn": 5632, "train": False},
        # A training step's tokens: forward with what the backward needs, and
        # the backward with all three weights' gradients.
        {"name": "ffn_fwd", "op": "ffn_fwd", "dtype": "bf16", "act": "silu", "rows": 8192,
         "dim": 2048, "ffn": 5632, "train": True},
        {"name": "ffn_bwd", "op": "ffn_bwd", "dtype": "bf16", "act": "silu", "rows": 8192,
         "dim": 2048, "ffn": 5632},
        # A ragged batch of a small f32 block, widths off every tile.
        {"name": "ffn_bwd_odd", "op": "ffn_bwd", "dtype": "f32", "act": "gelu", "rows": 1001,
         "dim": 777, "ffn": 2050},
        # The adapters of a 12-layer decoder: many small tensors, moments in 32 bits.
        {"name": "adamw_adapters", "op": "adamw", "states": 32, "grads": "f32", "copy": False,
         "tensors": 96, "most": 6144, "total": 589824},
        # A trained block of the larger decoder: few large tensors, bf16
        # gradients and a bf16 copy of the weights, moments in 32 and in 8 bits.
        {"name": "adamw_block", "op": "adamw", "states": 32, "grads": "bf16", "copy": True,
         "tensors": 5, "most": 11534336, "total": 34605056},
        {"name": "adamw_block_8bit", "op": "adamw", "states": 8, "grads": "bf16", "copy": True,
         "tensors": 5, "most": 11534336, "total": 34605056},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Model widths are multiples of 64 as often as not."""
    n = _spread(rng, lo, hi)
    return max(lo, n // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "ffn_fwd", "ffn_bwd", "adamw"])
    dtype = rng.choice(["f32", "bf16"])
    if op.startswith("norm"):
        while True:
            c = {"op": op, "kind": rng.choice(["layer", "rms"]), "dtype": dtype,
                 "rows": _spread(rng, 1, 32768), "cols": _width(rng, 16, 8192)}
            if c["rows"] * c["cols"] <= 8192 * 2048:
                return c
    if op.startswith("ffn"):
        while True:
            c = {"op": op, "dtype": dtype, "act": rng.choice(["silu", "gelu", "relu"]),
                 "rows": _spread(rng, 1, 8192), "dim": _width(rng, 64, 4096),
                 "ffn": _width(rng, 128, 8192)}
            if op == "ffn_fwd":
                c["train"] = rng.random() < 0.5
            if c["rows"] * c["dim"] * c["ffn"] <= 8192 * 2048 * 5632 // (4 if dtype == "f32" else 1):
                return c
    tensors = _spread(rng, 1, 200)
    most = _spread(rng, 64, 8000000)
    return {"op": op, "states": rng.choice([8, 32]), "grads": dtype, "copy": rng.random() < 0.5,
            "tensors": tensors, "most": most, "total": min(tensors * most, 34605056)}


# --- what a program holds -------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


BLOCK = 128  # elements under one scale of an 8-bit moment
STEP = {"lr": 1e-3, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "wd": 0.01, "step": 40}


def _sizes(case):
    """The group's tensor sizes, each at most `most`, and where each begins:
    end to end, every one from a multiple of BLOCK."""
    rng = np.random.default_rng(case["tensors"] * 1000003 + case["most"])
    n = np.full(case["tensors"], case["most"], np.int64)
    if case["tensors"] >= 2 and case["tensors"] < 8:  # three weights and their small companions
        n[-2:] = np.minimum(n[-2:], 1024)
    elif case["tensors"] >= 8:
        n = np.maximum(1, n - rng.integers(0, max(1, case["most"] // 8), case["tensors"]))
    while n.sum() > case["total"]:
        n[np.argmax(n)] -= int(min(n.sum() - case["total"], n.max() - 1))
    at = np.concatenate([[0], np.cumsum((n + BLOCK - 1) // BLOCK * BLOCK)])
    return [int(x) for x in n], [int(x) for x in at]


def _inputs(case, seed):
    g = _gen(seed)
    t = TYPES[case.get("dtype", "f32")]
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    if case["op"].startswith("norm"):
        R, C = case["rows"], case["cols"]
        x = {"x": (rnd(R, C) * (0.5 + torch.rand(R, 1, device="cuda", generator=g))
                   + 0.5 * rnd(R, 1)).to(t),
             "w": 1.0 + 0.1 * rnd(C), "b": 0.1 * rnd(C) if case["kind"] == "layer" else None}
        if case["op"] == "norm_bwd":  # with the statistics that the forward pass saved
            x["dy"] = rnd(R, C).to(t)
            x64 = x["x"].to(F64)
            mean = x64.mean(1, keepdim=True) if case["kind"] == "layer" else torch.zeros_like(x64[:, :1])
            x["mean"] = mean[:, 0].to(F32)
            x["rstd"] = ((x64 - mean).square().mean(1) + EPS).rsqrt().to(F32)
        return x
    if case["op"].startswith("ffn"):
        M, D, F = case["rows"], case["dim"], case["ffn"]
        x = {"x": rnd(M, D).to(t), "wg": (rnd(D, F) * D ** -0.5).to(t),
             "wu": (rnd(D, F) * D ** -0.5).to(t), "wd": (rnd(F, D) * F ** -0.5).to(t)}
        if case["op"] == "ffn_bwd":  # with the projections that the forward pass saved
            x["gate"] = (x["x"].to(F32) @ x["wg"].to(F32)).to(t)
            x["up"] = (x["x"].to(F32) @ x["wu"].to(F32)).to(t)
            x["dy"] = rnd(M, D).to(t)
        return x
    sizes, at = _sizes(case)
    total = at[-1]
    held = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"),
                                   torch.tensor([b - a for a, b in zip(at, at[1:])], device="cuda"))
    inside = (torch.arange(total, device="cuda") - torch.tensor(at[:-1], device="cuda")[held]
              < torch.tensor(sizes, device="cuda")[held])
    flat = lambda v: torch.where(inside, v, torch.zeros((), device="cuda"))  # noqa: E731
    size = 1e-3 * torch.exp(rnd(total // BLOCK)).repeat_interleave(BLOCK)  # gradients differ by rows
    x = {"p": flat(0.02 * rnd(total)), "g": flat(size * rnd(total)).to(TYPES[case["grads"]]),
         "m": flat(0.3 * size * rnd(total)), "v": flat(size.square() * (0.01 + 0.06 * torch.rand(
             total, device="cuda", generator=g)))}
    # Small tensors (norm weights and biases) are not decayed.
    x["decays"] = [0.0 if n <= 4096 and len(sizes) < 8 else 1.0 for n in sizes]
    x["decay"] = torch.tensor(x["decays"], device="cuda")[held]
    if case["states"] == 8:
        for k, v in (("m", x["m"]), ("v", x["v"].sqrt())):
            s = _scales(v)
            q = v / s.repeat_interleave(BLOCK)
            x[k], x[k + "s"] = q.to(torch.float8_e4m3fn).view(torch.uint8), s
    if case["copy"]:
        x["p16"] = torch.zeros(total, dtype=BF16, device="cuda")
    return x


@functools.lru_cache(maxsize=1)
def _framework():
    """The binding and one backend context for the whole program, on torch's stream."""
    hip = importlib.import_module("see-ai_amd.hip")
    ctx = hip.Context(0)
    ctx.use_torch_stream()
    return hip, ctx


def prepare(case, seed):
    x = _inputs(case, seed)
    if not own:
        return case, x
    hip, ctx = _framework()
    if case["op"] == "norm_bwd":
        n = hip.lib().seeai_norm_bwd_workspace(case["rows"], case["cols"])
        x["ws"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    elif case["op"].startswith("ffn"):
        n = hip.lib().seeai_ffn_workspace(int(case["dtype"] == "bf16"), case["rows"], case["dim"],
                                          case["ffn"], int(case["op"] == "ffn_bwd"))
        x["ws"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    elif case["op"] == "adamw":
        sizes, at = _sizes(case)
        tensors = []
        for n, a, decay in zip(sizes, at, x["decays"]):
            t = {"p": x["p"][a:], "g": x["g"][a:], "m": x["m"][a:], "v": x["v"][a:], "n": n,
                 "decay": decay}
            if case["states"] == 8:
                t["m_scale"], t["v_scale"] = x["ms"][a // BLOCK:], x["vs"][a // BLOCK:]
            if case["copy"]:
                t["p_bf16"] = x["p16"][a:]
            tensors.append(t)
        x["group"] = hip.AdamWGroup(ctx, tensors, state_bits=case["states"],
                                    grads=case["grads"], seed=SEED)
        x["params"] = hip.StepParams(STEP["lr"], STEP["beta1"], STEP["beta2"], STEP["eps"],
                                     STEP["wd"], 0, STEP["step"])
    return case, x


# --- one pass -------------------------------------------------------------------------------------

def run(state):
    case, x = state
    if own:
        return _own(case, x)
    with torch.no_grad():
        return {"norm_fwd": _norm_fwd, "norm_bwd": _norm_bwd, "ffn_fwd": _ffn_fwd,
                "ffn_bwd": _ffn_bwd, "adamw": _adamw}[case["op"]](case, x)


def _own(case, x):
    hip, ctx = _framework()
    p, bf16 = hip.ptr, int(case.get("dtype") == "bf16")
    new, new32 = torch.empty_like, lambda *s: torch.empty(s, dtype=F32, device="cuda")
    if case["op"].startswith("norm"):
        R, C, rms = case["rows"], case["cols"], int(case["kind"] == "rms")
        if case["op"] == "norm_fwd":
            y, mean, rstd = new(x["x"]), None if rms else new32(R), new32(R)
            ctx.call("seeai_norm_fwd", rms, bf16, p(x["x"]), p(x["w"]), p(x["b"]), p(y), p(mean),
                     p(rstd), R, C, EPS)
            return {"y": y, "mean": mean, "rstd": rstd}
        dx, dw, db = new(x["x"]), new32(C), None if rms else new32(C)
        ctx.call("seeai_norm_bwd", rms, bf16, p(x["dy"]), p(x["x"]), p(x["w"]),
                 None if rms else p(x["mean"]), p(x["rstd"]), p(dx), p(dw), p(db), R, C, p(x["ws"]),
                 x["ws"].numel())
        return {"dx": dx, "dw": dw, "db": db}
    if case["op"].startswith("ffn"):
        M, D, F = case["rows"], case["dim"], case["ffn"]
        act = {"relu": 1, "gelu": 2, "silu": 3}[case["act"]]
        if case["op"] == "ffn_fwd":
            saved = [torch.empty(M, F, dtype=x["x"].dtype, device="cuda") if case["train"] else None
                     for _ in range(2)]
            y = new(x["x"])
            ctx.call("seeai_ffn_fwd", bf16, act, p(x["x"]), p(x["wg"]), p(x["wu"]), p(x["wd"]),
                     p(saved[0]), p(saved[1]), p(y), M, D, F, p(x["ws"]), x["ws"].numel())
            return {"y": y, "gate": saved[0], "up": saved[1]}
        d = {"dx": new(x["x"]), "dwg": new(x["wg"]), "dwu": new(x["wu"]), "dwd": new(x["wd"])}
        ctx.call("seeai_ffn_bwd", bf16, act, p(x["x"]), p(x["wg"]), p(x["wu"]), p(x["wd"]),
                 p(x["gate"]), p(x["up"]), p(x["dy"]), p(d["dx"]), p(d["dwg"]), p(d["dwu"]),
                 p(d["dwd"]), M, D, F, p(x["ws"]), x["ws"].numel())
        return d
    x["group"].step(x["params"])
    out = {"p": x["p"]}
    if case["copy"]:
        out["p16"] = x["p16"]
    if case["states"] == 32:
        return out | {"m": x["m"], "v": x["v"]}
    for k, which in (("m", 0), ("v", 1)):  # the moments that the codes stand for
        out[k] = torch.empty(x["p"].shape, dtype=BF16, device="cuda")
        ctx.call("seeai_adamw_state_values", which, 1, p(x[k]), p(x[k + "s"]), x["p"].numel(),
                 p(out[k]))
    return out


def _norm_fwd(case, x):
    t, layer = x["x"].dtype, case["kind"] == "layer"
    x32 = x["x"].to(F32)
    mean = x32.mean(1, keepdim=True) if layer else 0.0
    c = x32 - mean
    rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    y = c * rstd * x["w"]
    if layer:
        y = y + x["b"]
    return {"y": y.to(t), "mean": mean[:, 0] if layer else None, "rstd": rstd[:, 0]}


def _norm_bwd(case, x):
    t, layer = x["x"].dtype, case["kind"] == "layer"
    dy, rstd = x["dy"].to(F32), x["rstd"][:, None]
    xhat = (x["x"].to(F32) - x["mean"][:, None]) * rstd
    d = dy * x["w"]
    dx = d - xhat * (d * xhat).mean(1, keepdim=True)
    if layer:
        dx = dx - d.mean(1, keepdim=True)
    return {"dx": (dx * rstd).to(t), "dw": (dy * xhat).sum(0), "db": dy.sum(0) if layer else None}


def _act(name, a):
    """The activation and its derivative."""
    if name == "relu":
        return a * (a > 0), (a > 0).to(a.dtype)
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-a))
        return a * s, s * (1.0 + a * (1.0 - s))
    k, c = 0.7978845608028654, 0.044715
    th = torch.tanh(k * (a + c * a * a * a))
    return (0.5 * a * (1.0 + th),
            0.5 * (1.0 + th) + 0.5 * a * (1.0 - th * th) * k * (1.0 + 3.0 * c * a * a))


def _ffn_fwd(case, x):
    t, x32 = x["x"].dtype, x["x"].to(F32)
    gate, up = x32 @ x["wg"].to(F32), x32 @ x["wu"].to(F32)
    y = (_act(case["act"], gate)[0] * up) @ x["wd"].to(F32)
    keep = (lambda v: v.to(t)) if case["train"] else lambda v: None
    return {"y": y.to(t), "gate": keep(gate), "up": keep(up)}


def _ffn_bwd(case, x):
    t = x["x"].dtype
    x32, dy = x["x"].to(F32), x["dy"].to(F32)
    up = x["up"].to(F32)
    a, da = _act(case["act"], x["gate"].to(F32))
    dh = dy @ x["wd"].to(F32).t()
    dgate, dup = dh * up * da, dh * a
    dx = dgate @ x["wg"].to(F32).t() + dup @ x["wu"].to(F32).t()
    return {"dx": dx.to(t), "dwg": (x32.t() @ dgate).to(t), "dwu": (x32.t() @ dup).to(t),
            "dwd": ((a * up).t() @ dy).to(t)}


# The 8-bit moments.  A block of 128 elements holds 8-bit floats of four
# significant bits (e4m3) under one scale, the power of two that brings the
# block's largest magnitude into (224, 448]; the first moment is held as it is,
# the second as its square root.  A value is rounded up or down with the
# chances that make it right on average, by 16 bits drawn from the group's
# seed, the step and the element's number, so that an average that moves by
# less than half a code a step still moves.
SEED = 20260


def _scales(v):
    """Each block's scale, for values laid out block after block."""
    big = v.reshape(-1, BLOCK).abs()
    big = torch.where(big.isfinite(), big, torch.zeros_like(big)).amax(1)
    f, e = torch.frexp(big)  # big = f 2^e, f in [1/2, 1): 448 = 7/8 2^9
    e = torch.where(f > 0.875, e - 8, e - 9).clamp(-126, 120)
    e = torch.where(big > 0, e, -126).to(torch.int32)
    return ((e + 127) << 23).view(F32)


def _mix(h):
    """32 well-mixed bits of 32 bits, in 64-bit integers."""
    h = ((h ^ (h >> 15)) * 0x6C8E9CF5) & 0xFFFFFFFF
    h = ((h ^ (h >> 13)) * 0x3A5D2B97) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _draws(total):
    """The 32 bits of every element of this step: the low half rounds the
    first moment, the high half the second."""
    i = torch.arange(total, device="cuda")
    key = _mix(_mix(torch.tensor([SEED], device="cuda")) ^ STEP["step"])
    return _mix((i & 0xFFFFFFFF) ^ _mix(key ^ (i >> 32)))


def _encode(v, bits, least):
    """Codes and scales of values, rounded by their 16 bits; with `least`, a
    value above zero keeps the smallest code at least."""
    s = _scales(v)
    q = v.abs() / s.repeat_interleave(BLOCK)
    small = q < 2.0 ** -6
    b = torch.where(small, q + 2.0 ** -6, q).view(torch.int32)
    b = (b + (bits << 4).to(torch.int32)) >> 20
    code = b - torch.where(small, 968, 960).to(torch.int32)
    if least:
        code = torch.where(q > 0, code.clamp(min=1), code)
    code = torch.where(q.isfinite(), code, torch.full_like(code, 0x7F))
    return (code | ((v < 0).to(torch.int32) << 7)).to(torch.uint8), s


def _decode(codes, s):
    return codes.view(torch.float8_e4m3fn).to(F32) * s.repeat_interleave(BLOCK)


def _adamw(case, x):
    f = np.float32
    b1, b2, t = f(STEP["beta1"]), f(STEP["beta2"]), f(STEP["step"])
    c1, c2 = f(1) / (f(1) - np.power(b1, t)), f(1) / (f(1) - np.power(b2, t))
    g, small = x["g"].to(F32), case["states"] == 8
    m = _decode(x["m"], x["ms"]) if small else x["m"]
    v = _decode(x["v"], x["vs"]).square() if small else x["v"]
    m = m * float(b1) + g * float(f(1) - b1)
    v = v * float(b2) + g * float(f(1) - b2) * g
    p = x["p"]
    wd = x["decay"] * float(f(STEP["wd"]))
    new = p - float(f(STEP["lr"])) * ((m * float(c1)) / (torch.sqrt(v * float(c2)) + float(f(STEP["eps"])))
                                      + wd * p)
    x["p"].copy_(new)
    out = {"p": x["p"]}
    if case["copy"]:
        x["p16"].copy_(new.to(BF16))
        out["p16"] = x["p16"]
    if not small:
        x["m"].copy_(m)
        x["v"].copy_(v)
        return out | {"m": x["m"], "v": x["v"]}
    draws = _draws(p.numel())
    mc, ms = _encode(m, draws & 0xFFFF, False)
    vc, vs = _encode(torch.sqrt(v), draws >> 16, True)
    x["m"].copy_(mc), x["ms"].copy_(ms), x["v"].copy_(vc), x["vs"].copy_(vs)
    return out | {"m": _decode(mc, ms).to(BF16), "v": _decode(vc, vs).square().to(BF16)}


# --- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    size = 4 if case.get("dtype") == "f32" else 2
    if case["op"].startswith("norm"):
        R, C, layer = case["rows"], case["cols"], case["kind"] == "layer"
        bwd = case["op"] == "norm_bwd"
        vectors = (1 + layer) * (4 * C + 4 * R) + bwd * 4 * C
        return {"bytes": (3 if bwd else 2) * R * C * size + vectors, "flops": (14 if bwd else 8) * R * C}
    if case["op"].startswith("ffn"):
        M, D, F = case["rows"], case["dim"], case["ffn"]
        weights = 3 * D * F
        if case["op"] == "ffn_fwd":
            return {"bytes": size * (2 * M * D + weights + 2 * M * F * case["train"]),
                    "flops": 6 * M * D * F}
        return {"bytes": size * (3 * M * D + 2 * M * F + 2 * weights), "flops": 12 * M * D * F}
    n = sum(_sizes(case)[0])
    # 8-bit moments: read, written, and the values they stand for come back.
    states = 16 if case["states"] == 32 else 4 + 2 * 8 / BLOCK + 4
    return {"bytes": n * (8 + (4 if case["grads"] == "f32" else 2) + 2 * case["copy"] + states),
            "flops": 16 * n}


# --- the same in 64 bits --------------------------------------------------------------------------

def _sum(v, dims):
    return v.sum(dims, keepdim=True)


def _gelu64(u):
    return 0.5 * u * (1 + torch.tanh(math.sqrt(2 / math.pi) * (u + 0.044715 * u ** 3)))


GATES = {"relu": torch.relu, "silu": lambda u: u / (1 + torch.exp(-u)),
         "gelu": _gelu64}


def exact(case, seed):
    x = {k: v.to(F64) if isinstance(v, torch.Tensor) and v.is_floating_point() else v
         for k, v in _inputs(case, seed).items()}
    return {"norm_fwd": _exact_norm_fwd, "norm_bwd": _exact_norm_bwd, "ffn_fwd": _exact_ffn_fwd,
            "ffn_bwd": _exact_ffn_bwd, "adamw": _exact_adamw}[case["op"]](case, x)


def _exact_norm_fwd(case, x):
    n = case["cols"]
    mean = _sum(x["x"], 1) / n if case["kind"] == "layer" else torch.zeros_like(x["x"][:, :1])
    std = torch.sqrt(_sum((x["x"] - mean) ** 2, 1) / n + EPS)
    y = (x["x"] - mean) / std * x["w"] + (x["b"] if case["kind"] == "layer" else 0)
    return {"y": y, "mean": mean[:, 0] if case["kind"] == "layer" else None, "rstd": 1 / std[:, 0]}


def _exact_norm_bwd(case, x):
    """The Jacobian of the normalisation, (I - [1 1'/n] - xhat xhat'/n) / std, at
    the saved statistics, applied to w dy."""
    n, s = case["cols"], x["rstd"][:, None]
    xhat = x["x"] * s - x["mean"][:, None] * s
    up = x["w"][None] * x["dy"]
    inner = _sum(up * xhat, 1) / n
    level = _sum(up, 1) / n if case["kind"] == "layer" else 0
    return {"dx": s * (up - level - xhat * inner), "dw": _sum(x["dy"] * xhat, 0)[0],
            "db": _sum(x["dy"], 0)[0] if case["kind"] == "layer" else None}


def _exact_ffn_fwd(case, x):
    gate, up = torch.mm(x["x"], x["wg"]), torch.mm(x["x"], x["wu"])
    y = torch.mm(GATES[case["act"]](gate) * up, x["wd"])
    return {"y": y, "gate": gate if case["train"] else None, "up": up if case["train"] else None}


def _exact_ffn_bwd(case, x):
    """Differentiated by torch from the block's product at the saved projections."""
    gate, up = x["gate"].requires_grad_(), x["up"].requires_grad_()
    with torch.enable_grad():
        h = GATES[case["act"]](gate) * up
        dgate, dup = torch.autograd.grad(h, (gate, up), torch.mm(x["dy"], x["wd"].t().contiguous()))
    xt = x["x"].t().contiguous()
    return {"dx": torch.mm(dgate, x["wg"].t().contiguous()) + torch.mm(dup, x["wu"].t().contiguous()),
            "dwg": torch.mm(xt, dgate), "dwu": torch.mm(xt, dup),
            "dwd": torch.mm(h.detach().t().contiguous(), x["dy"])}


def _held64(codes, scale):
    """What codes stand for, from their bits: sign, four bits of exponent, three of fraction."""
    c = codes.to(torch.int64)
    e, f = (c >> 3) & 15, (c & 7).to(F64)
    mag = torch.where(e == 0, f * 2.0 ** -9, (8 + f) * torch.ldexp(torch.ones_like(f), e - 10))
    return mag * (1 - 2 * (c >> 7)) * scale[:, None].expand(-1, BLOCK).reshape(-1)


def _round64(v, u):
    """The nearest codes' values below and above, chosen by u in [0, 1)."""
    blocks = v.reshape(-1, BLOCK)
    big = blocks.abs().amax(1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2((big / 448).clamp(min=2.0 ** -126))))
    q = blocks / scale
    grid = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.sign(q) * torch.floor(q.abs() / grid + u.reshape(-1, BLOCK)) * grid, scale)


def _exact_adamw(case, x):
    s = {k: float(np.float32(v)) for k, v in STEP.items()}
    g, small = x["g"], case["states"] == 8
    m = _held64(x["m"], x["ms"]) if small else x["m"]
    v = _held64(x["v"], x["vs"]) ** 2 if small else x["v"]
    m = s["beta1"] * m + (1 - s["beta1"]) * g
    v = s["beta2"] * v + (1 - s["beta2"]) * g ** 2
    step = (m / (1 - s["beta1"] ** s["step"])) / (torch.sqrt(v / (1 - s["beta2"] ** s["step"])) + s["eps"])
    p = x["p"] - s["lr"] * (step + s["wd"] * x["decay"] * x["p"])
    out = {"p": p, **({"p16": p} if case["copy"] else {})}
    if not small:
        return out | {"m": m, "v": v}
    draws = _draws(p.numel())
    mq, ms = _round64(m, (draws & 0xFFFF).to(F64) / 65536)
    vq, vs = _round64(torch.sqrt(v), (draws >> 16).to(F64) / 65536)
    vq = torch.where(v.reshape(-1, BLOCK) > 0, vq.clamp(min=2.0 ** -9), vq)
    return out | {"m": (mq * ms).reshape(-1), "v": ((vq * vs) ** 2).reshape(-1)}
