"""The operators of a training step on preferences: what is measured.

Beside cross-entropy a model may learn from preferences: from pairs of answers,
one chosen and one rejected (a logistic loss of the pair's log ratios against a
reference model), or from rewarded answers (a clipped policy loss with a KL
term).  The operators are the labels' log-probabilities from logits, forward and
backward, the two losses with their gradients, the norm of a step's gradients
with the clipped optimizer step, and what stands between two trained blocks: the
norm after a block, its gate, the residual and the norm before the next, forward
and backward.

``listed()`` are the fixed cases, ``draw(rng)`` more of the same ranges,
``prepare`` / ``run`` what a program holds and calls, ``work`` what a pass
cannot do without, ``exact`` the same results in 64 bits.
"""
from __future__ import annotations

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
        # One sequence's newest token against a vocabulary: latency.
        {"name": "logp_token", "op": "logp", "dtype": "bf16", "rows": 1, "vocab": 32000, "ld": 32000,
         "seqs": 1, "prompt": 0.0},
        # The reference model's log-probabilities of a step's answers; prompts are not judged.
        {"name": "logp_reference", "op": "logp", "dtype": "bf16", "rows": 8192, "vocab": 32000,
         "ld": 32000, "seqs": 16, "prompt": 0.3},
        # Four short pairs in f32, rows off every vector width in a padded buffer.
        {"name": "pref_odd", "op": "pref", "dtype": "f32", "rows": 701, "vocab": 4001, "ld": 4003,
         "seqs": 8, "prompt": 0.5, "average": True},
        # A preference step of the larger decoder: eight pairs, forward and backward.
        {"name": "pref", "op": "pref", "dtype": "bf16", "rows": 8192, "vocab": 32000, "ld": 32000,
         "seqs": 16, "prompt": 0.3, "average": False},
        # A small policy step in f32 without a reference model.
        {"name": "policy_small", "op": "policy", "dtype": "f32", "rows": 300, "vocab": 4000, "ld": 4000,
         "seqs": 3, "prompt": 0.2, "kl": 0.0},
        # A policy step of the larger decoder with its KL term.
        {"name": "policy", "op": "policy", "dtype": "bf16", "rows": 8192, "vocab": 32000, "ld": 32000,
         "seqs": 32, "prompt": 0.3, "kl": 0.05},
        # The norm of a 12-layer decoder's adapter gradients: many small tensors.
        {"name": "clip_adapters", "op": "clip", "grads": "f32", "tensors": 96, "most": 6144,
         "total": 589824, "step": False},
        # The clipped step of a trained block of the larger decoder.
        {"name": "clip_block", "op": "clip", "grads": "bf16", "tensors": 5, "most": 11534336,
         "total": 34605056, "step": True},
        # One sequence's newest token between two blocks: latency.
        {"name": "join_token", "op": "join_fwd", "kind": "rms", "dtype": "bf16", "rows": 1, "cols": 768,
         "post": True, "pre": True, "gate_rows": 0},
        # The larger decoder's tokens between two blocks, a learned gate a channel.
        {"name": "join_fwd", "op": "join_fwd", "kind": "rms", "dtype": "bf16", "rows": 8192, "cols": 2048,
         "post": True, "pre": True, "gate_rows": 8192},
        # The same step's backward pass.
        {"name": "join_bwd", "op": "join_bwd", "kind": "rms", "dtype": "bf16", "rows": 8192, "cols": 2048,
         "post": True, "pre": True, "gate_rows": 8192},
        # A ragged f32 batch, rows off every vector width, a gate a sequence.
        {"name": "join_bwd_odd", "op": "join_bwd", "kind": "layer", "dtype": "f32", "rows": 3001,
         "cols": 1023, "post": True, "pre": True, "gate_rows": 500},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Widths are multiples of 64 as often as not."""
    n = _spread(rng, lo, hi)
    return max(lo, n // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["logp", "pref", "policy", "clip", "join_fwd", "join_bwd"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "clip":
        tensors, most = _spread(rng, 1, 200), _spread(rng, 64, 8000000)
        return {"op": op, "grads": dtype, "tensors": tensors, "most": most,
                "total": min(tensors * most, 34605056), "step": rng.random() < 0.5}
    if op.startswith("join"):
        while True:
            c = {"op": op, "kind": rng.choice(["layer", "rms"]), "dtype": dtype,
                 "rows": _spread(rng, 1, 32768), "cols": _width(rng, 16, 8192)}
            c["post"] = rng.random() < 0.75
            c["pre"] = not c["post"] or rng.random() < 0.75
            c["gate_rows"] = rng.choice([0, c["rows"], _spread(rng, 16, 4096)])
            if c["rows"] * c["cols"] <= 8192 * 2048 // (2 if dtype == "f32" else 1):
                return c
    while True:
        c = {"op": op, "dtype": dtype, "rows": _spread(rng, 1 if op == "logp" else 2, 16384),
             "vocab": _width(rng, 64, 131072)}
        c["ld"] = c["vocab"] if rng.random() < 0.5 else (c["vocab"] + 63) // 64 * 64
        c["seqs"] = min(c["rows"], _spread(rng, 1, 64))
        if op == "pref":
            c["seqs"] = max(2, c["seqs"] // 2 * 2)
            c["average"] = rng.random() < 0.5
        if op == "policy":
            c["kl"] = rng.choice([0.0, 0.05])
        c["prompt"] = rng.choice([0.0, 0.3, 0.6])
        if c["rows"] * c["ld"] <= 8192 * 32000 // (2 if dtype == "f32" else 1):
            return c


# --- what a program holds -------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _tokens(case):
    """Where each sequence begins (and the last ends), and which rows are judged:
    a sequence opens with its prompt, whose rows are not."""
    R, Q = case["rows"], case["seqs"]
    rng = np.random.default_rng(R * 1000003 + case["vocab"])
    share = rng.uniform(0.5, 1.5, Q)
    cuts = np.floor(np.cumsum(share) / share.sum() * (R - Q) + 1e-9).astype(np.int64)
    starts = np.concatenate([[0], cuts + np.arange(1, Q + 1)])
    starts[-1] = R
    seq = np.repeat(np.arange(Q), np.diff(starts))
    within = np.arange(R) - starts[seq]
    prompt = np.floor(case["prompt"] * np.diff(starts))[seq]
    return starts, seq, within >= prompt


STEP = {"lr": 1e-3, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "wd": 0.01, "step": 40}
PREF = {"beta": 0.1, "smoothing": 0.05}
CLIP = {"low": 0.2, "high": 0.28}
MAX_NORM = 1.0


def _sizes(case):
    """The group's tensor sizes, each at most `most`, and where each begins: end
    to end, every one from a multiple of 128."""
    rng = np.random.default_rng(case["tensors"] * 1000003 + case["most"])
    n = np.full(case["tensors"], case["most"], np.int64)
    if 2 <= case["tensors"] < 8:  # three weights and their small companions
        n[-2:] = np.minimum(n[-2:], 1024)
    elif case["tensors"] >= 8:
        n = np.maximum(1, n - rng.integers(0, max(1, case["most"] // 8), case["tensors"]))
    while n.sum() > case["total"]:
        n[np.argmax(n)] -= int(min(n.sum() - case["total"], n.max() - 1))
    at = np.concatenate([[0], np.cumsum((n + 127) // 128 * 128)])
    return [int(x) for x in n], [int(x) for x in at]


def _label_logp64(logits, labels, vocab):
    """The labels' log-probabilities in 64 bits, some rows at a time."""
    parts = []
    for at in range(0, logits.shape[0], 1024):
        z = logits[at:at + 1024, :vocab].to(F64)
        picked = z.gather(1, labels[at:at + 1024].clamp(min=0).to(torch.int64)[:, None])[:, 0]
        parts.append(picked - z.logsumexp(1))
    return torch.cat(parts)


def _inputs(case, seed):
    g = _gen(seed)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    rand = lambda *s: torch.rand(s, device="cuda", generator=g)  # noqa: E731
    if case["op"] in ("logp", "pref", "policy"):
        R, V = case["rows"], case["vocab"]
        starts, seq, judged = _tokens(case)
        labels = torch.randint(0, V, (R,), device="cuda", generator=g)
        z = 2.0 * rnd(R, case["ld"])
        # A trained model's own answers: most labels stand out from the rest.
        sure = math.log(V) + 2.0 + 3.0 * rnd(R)
        z.scatter_(1, labels[:, None], torch.where(rand(R) < 0.8, sure, 2.0 * rnd(R))[:, None])
        z += 3.0 * rnd(R, 1)
        x = {"logits": z.to(TYPES[case["dtype"]]),
             "labels": torch.where(torch.tensor(judged, device="cuda"), labels, -1).to(torch.int32)}
        if case["op"] == "logp":
            return x
        now = _label_logp64(x["logits"], x["labels"], V)
        x["ref"] = (now + 0.3 * rnd(R)).to(F32)
        if case["op"] == "pref":
            x["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
            x["seq"] = torch.tensor(seq, device="cuda")
            return x
        # The policy has moved since the answers were sampled; no ratio lies so
        # near a bound that its side is a matter of rounding.
        moved = 0.25 * rnd(R)
        for bound in (math.log(1 - CLIP["low"]), math.log(1 + CLIP["high"])):
            moved = torch.where((moved - bound).abs() < 1e-3, bound + 2e-3, moved)
        x["old"] = (now - moved).to(F32)
        # An answer's advantage is its tokens'; each answer weighs the same.
        x["adv"] = rnd(case["seqs"])[torch.tensor(seq, device="cuda")]
        counted = np.maximum(np.bincount(seq, judged, case["seqs"]), 1)
        x["weight"] = torch.tensor((1.0 / counted)[seq], dtype=F32, device="cuda")
        return x
    if case["op"].startswith("join"):
        t, R, C, layer = TYPES[case["dtype"]], case["rows"], case["cols"], case["kind"] == "layer"
        G = -(-R // case["gate_rows"]) if case["gate_rows"] else 0
        vec = lambda on, at, by: at + by * rnd(C) if on else None  # noqa: E731
        x = {"o": (rnd(R, C) * (0.5 + rand(R, 1))).to(t), "x": (2.0 * rnd(R, C) + 0.5 * rnd(R, 1)).to(t),
             "post_w": vec(case["post"], 1.0, 0.1), "post_b": vec(case["post"] and layer, 0.0, 0.1),
             "gate": 0.5 + 0.2 * rnd(G, C) if G else None,
             "pre_w": vec(case["pre"], 1.0, 0.1), "pre_b": vec(case["pre"] and layer, 0.0, 0.1)}
        if case["op"] == "join_bwd":  # with what the forward pass left
            x["dy"] = rnd(R, C).to(t)
            x["dh"] = rnd(R, C).to(t) if case["pre"] else None
            out = _join64(case, {k: v.to(F64) if v is not None else None for k, v in x.items()})
            x["y"], x["stats"] = out["y"].to(t), out["stats"].to(F32)
        return x
    sizes, at = _sizes(case)
    total = at[-1]
    held = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"),
                                   torch.tensor([b - a for a, b in zip(at, at[1:])], device="cuda"))
    inside = (torch.arange(total, device="cuda") - torch.tensor(at[:-1], device="cuda")[held]
              < torch.tensor(sizes, device="cuda")[held])
    flat = lambda v: torch.where(inside, v, torch.zeros((), device="cuda"))  # noqa: E731
    size = torch.exp(rnd(total // 128)).repeat_interleave(128)  # gradients differ by rows
    size *= (1.0 + 2.0 * rand(1)) * 0.5 / math.sqrt(sum(sizes))  # norms on either side of the cap
    x = {"g": flat(size * rnd(total)).to(TYPES[case["grads"]])}
    if case["step"]:
        x["p"], x["m"] = flat(0.02 * rnd(total)), flat(0.3 * size * rnd(total))
        x["v"] = flat(size.square() * (0.01 + 0.06 * rand(total)))
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
    lib, byte = hip.lib(), lambda n: torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    if case["op"] == "pref":
        x["ws"] = byte(lib.seeai_pref_workspace(case["seqs"] // 2))
    elif case["op"] == "policy":
        x["ws"] = byte(lib.seeai_policy_workspace(case["rows"], case["vocab"]))
    elif case["op"].startswith("join"):
        p = hip.ptr
        x["join"] = hip.BlockJoin(
            p(x["o"]), p(x["x"]), p(x["post_w"]), p(x["post_b"]), p(x["gate"]), p(x["pre_w"]),
            p(x["pre_b"]), case["rows"], case["cols"], case["gate_rows"], int(case["kind"] == "rms"),
            int(case["dtype"] == "bf16"), RES, EPS)
        if case["op"] == "join_bwd":
            x["ws"] = byte(lib.seeai_block_join_workspace(case["rows"], case["cols"], case["gate_rows"]))
    elif case["op"] == "clip":
        sizes, at = _sizes(case)
        x["grads"] = hip.GradGroup(ctx, [x["g"][a:a + n] for n, a in zip(sizes, at)])
        if case["step"]:
            x["group"] = hip.AdamWGroup(ctx, [{k: x[k][a:a + n] for k in ("p", "g", "m", "v")}
                                              for n, a in zip(sizes, at)], 32, case["grads"])
            x["params"] = hip.StepParams(STEP["lr"], STEP["beta1"], STEP["beta2"], STEP["eps"],
                                         STEP["wd"], 0, STEP["step"])
    return case, x


# --- one pass -------------------------------------------------------------------------------------

RES = 0.75  # the residual's scale


def run(state):
    case, x = state
    if own:
        return _own(case, x)
    with torch.no_grad():
        return {"logp": _logp, "pref": _pref, "policy": _policy, "clip": _clip, "join_fwd": _join_fwd,
                "join_bwd": _join_bwd}[case["op"]](case, x)


def _own(case, x):
    hip, ctx = _framework()
    p, bf16 = hip.ptr, int(case.get("dtype") == "bf16")
    new, new32 = torch.empty_like, lambda *s: torch.empty(s, dtype=F32, device="cuda")
    if case["op"] in ("logp", "pref"):
        R, V, ld = case["rows"], case["vocab"], case["ld"]
        logp, stats = new32(R), new32(R, 2)
        ctx.call("seeai_token_logp_fwd", bf16, p(x["logits"]), ld, p(x["labels"]), p(logp), p(stats),
                 R, V)
        if case["op"] == "logp":
            return {"logp": logp}
        pairs = case["seqs"] // 2
        loss, margin, dlogp, dlogits = new32(1), new32(pairs), new32(R), new(x["logits"])
        ctx.call("seeai_pref_loss", p(logp), p(x["ref"]), p(x["labels"]), p(x["starts"]), R, pairs,
                 PREF["beta"], 0.0, PREF["smoothing"], int(case["average"]), 1.0 / pairs, p(loss),
                 p(margin), p(dlogp), p(x["ws"]), x["ws"].numel())
        ctx.call("seeai_token_logp_bwd", bf16, p(x["logits"]), ld, p(x["labels"]), p(stats), p(dlogp),
                 p(dlogits), R, V)
        return {"loss": loss, "logp": logp, "margin": margin, "dlogits": dlogits[:, :V]}
    if case["op"] == "policy":
        R, V, ld = case["rows"], case["vocab"], case["ld"]
        loss, logp, dlogits = new32(1), new32(R), new(x["logits"])
        ctx.call("seeai_policy_loss", bf16, p(x["logits"]), ld, p(x["labels"]), p(x["old"]),
                 p(x["ref"]) if case["kl"] else None, p(x["adv"]), p(x["weight"]), R, V, CLIP["low"],
                 CLIP["high"], case["kl"], 1.0 / case["seqs"], p(loss), p(logp), p(dlogits), p(x["ws"]),
                 x["ws"].numel())
        return {"loss": loss, "logp": logp, "dlogits": dlogits[:, :V]}
    if case["op"] == "join_fwd":
        y, h = new(x["x"]), new(x["x"]) if case["pre"] else None
        stats = new32(case["rows"], 4)
        ctx.call("seeai_block_join_fwd", x["join"], p(y), p(h), p(stats))
        return {"y": y, "h": h, "stats": _given(case, stats)}
    if case["op"] == "join_bwd":
        C = case["cols"]
        d = {"dx": new(x["o"]), "do": new(x["o"]),
             "dpost_w": new32(C) if x["post_w"] is not None else None,
             "dpost_b": new32(C) if x["post_b"] is not None else None,
             "dgate": new(x["gate"]) if x["gate"] is not None else None,
             "dpre_w": new32(C) if x["pre_w"] is not None else None,
             "dpre_b": new32(C) if x["pre_b"] is not None else None}
        ctx.call("seeai_block_join_bwd", x["join"], p(x["y"]), p(x["stats"]), p(x["dh"]), p(x["dy"]),
                 hip.BlockJoinGrads(*(p(v) for v in d.values())), p(x["ws"]), x["ws"].numel())
        return d
    norm, factor = new32(1), new32(1)
    x["grads"].norm(MAX_NORM, norm, factor)
    out = {"norm": norm, "factor": factor}
    if case["step"]:
        x["group"].step(x["params"], factor)
        out |= {k: x[k] for k in ("p", "m", "v")}
    return out


# The labels' log-probabilities and what the losses take of them.

def _softmax(case, x):
    """Probabilities of every row and its label's log-probability, 32 bits."""
    z = x["logits"][:, :case["vocab"]].to(F32)
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    at = x["labels"].clamp(min=0).to(torch.int64)[:, None]
    logp = (z.gather(1, at) - top - torch.log(total))[:, 0]
    return e / total, torch.where(x["labels"] >= 0, logp, torch.zeros_like(logp))


def _logits_grad(x, probs, dlogp):
    dlogp = torch.where(x["labels"] >= 0, dlogp, torch.zeros_like(dlogp))[:, None]
    d = -dlogp * probs
    return d.scatter_add(1, x["labels"].clamp(min=0).to(torch.int64)[:, None], dlogp).to(x["logits"].dtype)


def _logp(case, x):
    return {"logp": _softmax(case, x)[1]}


def _pref(case, x):
    probs, logp = _softmax(case, x)
    pairs, judged = case["seqs"] // 2, (x["labels"] >= 0).to(F64)
    per = torch.zeros(case["seqs"], dtype=F64, device="cuda")
    ratio = per.index_add(0, x["seq"], (logp.to(F64) - x["ref"].to(F64)) * judged)
    share = torch.ones_like(ratio)
    if case["average"]:
        share = 1.0 / per.index_add(0, x["seq"], judged).clamp(min=1.0)
    ratio = (ratio * share).view(pairs, 2)
    margin = PREF["beta"] * (ratio[:, 0] - ratio[:, 1])
    won = 1.0 / (1.0 + torch.exp(-margin))
    eps = PREF["smoothing"]
    loss = (-(1.0 - eps) * torch.log(won) - eps * torch.log(1.0 - won)).mean()
    dmargin = (won - (1.0 - eps)) / pairs * PREF["beta"]
    dseq = torch.stack([dmargin, -dmargin], 1).view(-1) * share
    dlogits = _logits_grad(x, probs, dseq[x["seq"]].to(F32))
    return {"loss": loss.to(F32).view(1), "logp": logp, "margin": margin.to(F32), "dlogits": dlogits}


def _policy(case, x):
    probs, logp = _softmax(case, x)
    judged = x["labels"] >= 0
    moved = logp - x["old"]
    ratio = torch.exp(moved)
    held = ratio.clamp(1.0 - CLIP["low"], 1.0 + CLIP["high"])
    free, clipped = ratio * x["adv"], held * x["adv"]
    loss = -torch.minimum(free, clipped)
    d = torch.where(clipped < free, torch.zeros_like(free), -free)
    if case["kl"]:
        back = x["ref"] - logp
        e = torch.exp(back)
        loss = loss + case["kl"] * (e - back - 1.0)
        d = d + case["kl"] * (1.0 - e)
    w = torch.where(judged, x["weight"] / case["seqs"], torch.zeros_like(loss))
    loss = torch.where(judged, loss, torch.zeros_like(loss)).to(F64) * w.to(F64)
    return {"loss": loss.sum().to(F32).view(1), "logp": logp, "dlogits": _logits_grad(x, probs, d * w)}


# The gradients' norm and the clipped step.

def _clip(case, x):
    norm = x["g"].to(F64).square().sum().sqrt()
    factor = torch.where(norm > MAX_NORM, MAX_NORM / norm, torch.ones_like(norm)).to(F32)
    out = {"norm": norm.to(F32).view(1), "factor": factor.view(1)}
    if not case["step"]:
        return out
    f = np.float32
    b1, b2, t = f(STEP["beta1"]), f(STEP["beta2"]), f(STEP["step"])
    c1, c2 = f(1) / (f(1) - np.power(b1, t)), f(1) / (f(1) - np.power(b2, t))
    g = x["g"].to(F32) * factor
    m = x["m"] * float(b1) + g * float(f(1) - b1)
    v = x["v"] * float(b2) + g * float(f(1) - b2) * g
    p = x["p"]
    new = p - float(f(STEP["lr"])) * ((m * float(c1)) / (torch.sqrt(v * float(c2)) + float(f(STEP["eps"])))
                                      + float(f(STEP["wd"])) * p)
    x["p"].copy_(new), x["m"].copy_(m), x["v"].copy_(v)
    return out | {k: x[k] for k in ("p", "m", "v")}


# Between two blocks: y = RES x + gate norm(o), h = norm(y).

def _given(case, stats):
    """The statistics that the case's norms have: the means of a layer norm alone."""
    layer = case["kind"] == "layer"
    return {"post_mean": stats[:, 0] if case["post"] and layer else None,
            "post_rstd": stats[:, 1] if case["post"] else None,
            "pre_mean": stats[:, 2] if case["pre"] and layer else None,
            "pre_rstd": stats[:, 3] if case["pre"] else None}


def _normalised(case, v):
    mean = v.mean(1, keepdim=True) if case["kind"] == "layer" else torch.zeros_like(v[:, :1])
    c = v - mean
    rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    return c * rstd, mean, rstd


def _gates(case, gate, rows):
    """Each row's gate."""
    return gate[torch.arange(rows, device="cuda") // case["gate_rows"]]


def _scaled(v, w, b):
    return v * w if b is None else v * w + b


def _join_fwd(case, x):
    t, rows = x["o"].dtype, case["rows"]
    n, none = x["o"].to(F32), torch.zeros(rows, 1, device="cuda")
    stats, h = [none, none, none, none], None
    if case["post"]:
        n, stats[0], stats[1] = _normalised(case, n)
        n = _scaled(n, x["post_w"], x["post_b"])
    if x["gate"] is not None:
        n = n * _gates(case, x["gate"], rows)
    y = RES * x["x"].to(F32) + n
    if case["pre"]:
        h, stats[2], stats[3] = _normalised(case, y)
        h = _scaled(h, x["pre_w"], x["pre_b"]).to(t)
    return {"y": y.to(t), "h": h, "stats": _given(case, torch.cat(stats, 1))}


def _norm_grad(case, d, hat, rstd):
    """Back through a normalisation whose output was `hat`."""
    back = d - hat * (d * hat).mean(1, keepdim=True)
    if case["kind"] == "layer":
        back = back - d.mean(1, keepdim=True)
    return back * rstd


def _join_bwd(case, x):
    t, s, out = x["o"].dtype, x["stats"], dict.fromkeys(
        ("dx", "do", "dpost_w", "dpost_b", "dgate", "dpre_w", "dpre_b"))
    dy = x["dy"].to(F32)
    if case["pre"]:
        hat, dh = (x["y"].to(F32) - s[:, 2:3]) * s[:, 3:4], x["dh"].to(F32)
        out["dpre_w"] = (dh * hat).sum(0)
        out["dpre_b"] = dh.sum(0) if x["pre_b"] is not None else None
        dy = dy + _norm_grad(case, dh * x["pre_w"], hat, s[:, 3:4])
    out["dx"] = (RES * dy).to(t)
    n = hat = x["o"].to(F32)
    if case["post"]:
        hat = (n - s[:, 0:1]) * s[:, 1:2]
        n = _scaled(hat, x["post_w"], x["post_b"])
    if x["gate"] is not None:
        group = torch.arange(case["rows"], device="cuda") // case["gate_rows"]
        out["dgate"] = torch.zeros_like(x["gate"]).index_add(0, group, dy * n)
        dy = dy * x["gate"][group]
    if case["post"]:
        out["dpost_w"] = (dy * hat).sum(0)
        out["dpost_b"] = dy.sum(0) if x["post_b"] is not None else None
        dy = _norm_grad(case, dy * x["post_w"], hat, s[:, 1:2])
    out["do"] = dy.to(t)
    return out


# --- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    size = 4 if case.get("dtype") == "f32" else 2
    if case["op"] in ("logp", "pref", "policy"):
        R, V = case["rows"], case["vocab"]
        judged = int(_tokens(case)[2].sum())
        read = judged * V * size  # rows that are not judged need not be read
        if case["op"] == "logp":
            return {"bytes": read + 8 * R, "flops": 4 * judged * V}
        write = R * V * size
        if case["op"] == "policy":
            return {"bytes": read + write + 28 * R, "flops": 6 * judged * V}
        # (a row's gradient needs its whole sequence's sum: the logits come twice)
        return {"bytes": 2 * read + write + 24 * R, "flops": 8 * judged * V}
    if case["op"].startswith("join"):
        R, C, bwd = case["rows"], case["cols"], case["op"] == "join_bwd"
        post, pre, gate = case["post"], case["pre"], case["gate_rows"] > 0
        vectors = 4 * C * (2 * post + 2 * pre) * (1 + bwd) + 16 * R
        vectors += 4 * C * (-(-R // case["gate_rows"]) if gate else 0) * (1 + bwd)
        if not bwd:
            return {"bytes": (3 + pre) * R * C * size + vectors, "flops": (2 + 6 * post + 6 * pre) * R * C}
        tensors = 3 + 2 * pre + (post or gate)  # dy, dx, do; dh and y; o
        return {"bytes": tensors * R * C * size + vectors, "flops": (3 + 12 * post + 12 * pre) * R * C}
    n, size = sum(_sizes(case)[0]), 4 if case["grads"] == "f32" else 2
    if not case["step"]:
        return {"bytes": n * size, "flops": 2 * n}
    # (the step needs the norm of all gradients first: they come twice)
    return {"bytes": n * (2 * size + 24), "flops": 18 * n}


# --- the same in 64 bits --------------------------------------------------------------------------

def exact(case, seed):
    x = {k: v.to(F64) if isinstance(v, torch.Tensor) and v.is_floating_point() else v
         for k, v in _inputs(case, seed).items()}
    if case["op"] in ("logp", "pref", "policy"):
        return _exact_loss(case, x)
    if case["op"] == "join_fwd":
        out = _join64(case, x)
        return {"y": out["y"], "h": out["h"], "stats": _given(case, out["stats"])}
    return {"clip": _exact_clip, "join_bwd": _exact_join_bwd}[case["op"]](case, x)


def _exact_loss(case, x):
    """The losses from torch's log-softmax, their gradients by differentiating the
    per-token expressions."""
    V, judged = case["vocab"], x["labels"] >= 0
    lp = torch.log_softmax(x["logits"][:, :V], 1)
    at = x["labels"].clamp(min=0).to(torch.int64)[:, None]
    logp = torch.where(judged, lp.gather(1, at)[:, 0], torch.zeros((), dtype=F64, device="cuda"))
    if case["op"] == "logp":
        return {"logp": logp}
    leaf, out = logp.clone().requires_grad_(), {}
    with torch.enable_grad():
        if case["op"] == "pref":
            which = torch.nn.functional.one_hot(x["seq"], case["seqs"]).to(F64) * judged[:, None]
            sums = (leaf - x["ref"]) @ which
            if case["average"]:
                sums = sums / which.sum(0).clamp(min=1)
            margin = PREF["beta"] * (sums[0::2] - sums[1::2])
            ls = torch.nn.functional.logsigmoid
            loss = -((1 - PREF["smoothing"]) * ls(margin) + PREF["smoothing"] * ls(-margin)).mean()
            out["margin"] = margin.detach()
        else:
            ratio = (leaf - x["old"]).exp()
            adv = x["adv"]
            worst = torch.where(adv >= 0, torch.minimum(ratio, ratio.new_tensor(1 + CLIP["high"])) * adv,
                                torch.maximum(ratio, ratio.new_tensor(1 - CLIP["low"])) * adv)
            gap = x["ref"] - leaf
            loss = (((case["kl"] * (torch.expm1(gap) - gap) - worst) * x["weight"])[judged]).sum() / case["seqs"]
        d, = torch.autograd.grad(loss, leaf)
    d = torch.where(judged, d, torch.zeros_like(d))[:, None]
    dlogits = lp.exp_().mul_(-d)
    dlogits.scatter_add_(1, at, d)
    return {"loss": loss.detach().view(1), "logp": logp, **out, "dlogits": dlogits}


def _exact_clip(case, x):
    norm = torch.linalg.vector_norm(x["g"])
    factor = (MAX_NORM / norm).clamp(max=1.0)
    out = {"norm": norm.view(1), "factor": factor.view(1)}
    if not case["step"]:
        return out
    s = {k: float(np.float32(v)) for k, v in STEP.items()}
    g = x["g"] * factor
    m = s["beta1"] * x["m"] + (1 - s["beta1"]) * g
    v = s["beta2"] * x["v"] + (1 - s["beta2"]) * g ** 2
    step = (m / (1 - s["beta1"] ** s["step"])) / (torch.sqrt(v / (1 - s["beta2"] ** s["step"])) + s["eps"])
    return out | {"p": x["p"] - s["lr"] * (step + s["wd"] * x["p"]), "m": m, "v": v}


def _norm64(case, v, w, b):
    mu = v.sum(1, keepdim=True) / v.shape[1] if case["kind"] == "layer" else torch.zeros_like(v[:, :1])
    std = torch.sqrt(((v - mu) ** 2).sum(1, keepdim=True) / v.shape[1] + EPS)
    out = (v - mu) / std * w
    return out + b if b is not None else out, mu, 1 / std


def _join64(case, x):
    n, none = x["o"], torch.zeros_like(x["o"][:, :1])
    stats, h = [none] * 4, None
    if case["post"]:
        n, stats[0], stats[1] = _norm64(case, n, x["post_w"], x["post_b"])
    if x["gate"] is not None:
        n = n * x["gate"].repeat_interleave(case["gate_rows"], 0)[:case["rows"]]
    y = n + RES * x["x"]
    if case["pre"]:
        h, stats[2], stats[3] = _norm64(case, y, x["pre_w"], x["pre_b"])
    return {"y": y, "h": h, "stats": torch.cat(stats, 1)}


def _jacobian64(case, up, hat, rstd):
    """The normalisation's Jacobian, (I - [1 1'/n] - hat hat'/n) rstd, at the saved
    statistics, applied to `up`."""
    n = up.shape[1]
    inner = (up * hat).sum(1, keepdim=True) / n
    level = up.sum(1, keepdim=True) / n if case["kind"] == "layer" else 0
    return rstd * (up - level - hat * inner)


def _exact_join_bwd(case, x):
    s, total, out = x["stats"], x["dy"], dict.fromkeys(
        ("dx", "do", "dpost_w", "dpost_b", "dgate", "dpre_w", "dpre_b"))
    if case["pre"]:
        hat = x["y"] * s[:, 3:4] - s[:, 2:3] * s[:, 3:4]
        total = total + _jacobian64(case, x["dh"] * x["pre_w"], hat, s[:, 3:4])
        out["dpre_w"] = (x["dh"] * hat).sum(0)
        out["dpre_b"] = x["dh"].sum(0) if x["pre_b"] is not None else None
    out["dx"] = RES * total
    n = hat = x["o"]
    if case["post"]:
        hat = x["o"] * s[:, 1:2] - s[:, 0:1] * s[:, 1:2]
        n = hat * x["post_w"] + (x["post_b"] if x["post_b"] is not None else 0)
    if x["gate"] is not None:
        each = torch.split(total * n, case["gate_rows"])
        out["dgate"] = torch.stack([e.sum(0) for e in each])
        total = total * x["gate"].repeat_interleave(case["gate_rows"], 0)[:case["rows"]]
    out["do"] = total
    if case["post"]:
        out["dpost_w"] = (total * hat).sum(0)
        out["dpost_b"] = total.sum(0) if x["post_b"] is not None else None
        out["do"] = _jacobian64(case, total * x["post_w"], hat, s[:, 1:2])
    return out
