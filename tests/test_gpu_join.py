"""GPU: what stands between two blocks -- seeai_block_join_fwd / _bwd -- against
plain float64, and a whole training step on preferences: joins, feed-forward
block, head, paired loss, clip and optimizer, eagerly and as captured graphs.

Tolerances are bounds on what the kernels' own roundings may add up to, u = 2^-24
for each f32 operation and 2^-8 of the value for a rounding to bf16 (half a step),
carried through the formulas."""
from __future__ import annotations

import pytest

from tests.test_gpu_block import DEPTH, EPS, U, Guarded, ctx, gen, put, types, within  # noqa: F401

pytestmark = pytest.mark.gpu

# rows, cols, gate_rows (0: no gate): rows of a wave to sixteen, registers of 8
# and 16, odd widths, gates of one row, a few, a part of a band, all rows.
SHAPES = [(1, 1, 0), (1, 768, 1), (3, 7, 2), (5, 64, 5), (70, 512, 7), (9, 513, 1), (130, 1000, 50),
          (33, 1023, 0), (2100, 1024, 700), (2100, 96, 3), (64, 1030, 64), (40, 2048, 11), (7, 2050, 2), (37, 128, 5), (70, 130, 9), (300, 255, 100), (41, 256, 0), (9, 126, 2),
          (600, 4096, 1000), (5, 5001, 3), (3, 8192, 2), (4, 8193, 0), (3, 16384, 1), (35, 511, 6), (20, 1025, 0), (11, 4097, 3), (2, 16383, 2),
          (4100, 320, 1025), (5000, 40, 1), (5000, 17, 33), (129, 6, 4), (6000, 202, 1500), (2049, 2048, 1)]
# kind, post norm, pre norm, biases
FORMS = [(0, 1, 1, 1), (1, 1, 1, 0), (0, 1, 0, 0), (1, 0, 1, 0), (0, 0, 1, 1), (1, 1, 0, 0)]


def inputs(torch, kind, post, pre, bias, rows, cols, gate_rows, t, off):
    rnd = gen(torch, rows * 31 + cols)
    vec = lambda at, by: put(torch, at + by * rnd(cols), torch.float32, off)  # noqa: E731
    G = -(-rows // gate_rows) if gate_rows else 0
    return {"o": put(torch, rnd(rows, cols) * 2 + rnd(rows, 1), t, off),
            "x": put(torch, 2 * rnd(rows, cols) + 0.5, t, off),
            "post_w": vec(1.0, 0.3) if post else None, "post_b": vec(0.0, 0.5) if post and bias else None,
            "gate": put(torch, 0.5 + 0.5 * rnd(G, cols), torch.float32, off) if G else None,
            "pre_w": vec(1.0, 0.3) if pre else None, "pre_b": vec(0.0, 0.5) if pre and bias else None}


RES = 0.75


def struct(hip, kind, bf16, d, rows, cols, gate_rows):
    p = hip.ptr
    return hip.BlockJoin(*(p(d[k]) for k in ("o", "x", "post_w", "post_b", "gate", "pre_w", "pre_b")), rows, cols,
                         gate_rows, kind, bf16, RES, EPS)


def forward(hip, ctx, torch, kind, bf16, d, rows, cols, gate_rows, off=0, y=None, stats=True):
    t, _ = types(torch, bf16)
    gy, gh = Guarded(torch, (rows, cols), t, off), Guarded(torch, (rows, cols), t, off)
    st = Guarded(torch, (rows, 4), torch.float32)
    at = gy.t if y is None else y
    ctx.call("seeai_block_join_fwd", struct(hip, kind, bf16, d, rows, cols, gate_rows), at.data_ptr(),
             gh.t.data_ptr() if d["pre_w"] is not None else None, st.t.data_ptr() if stats else None)
    assert gy.intact() and gh.intact() and st.intact()
    return at, gh.t, st.t


def norm64(torch, kind, v, e_v, w, b):
    """A norm of v known within e_v: mean, 1 / deviation, result and their bounds."""
    mu = v.mean(1, keepdim=True) if kind == 0 else torch.zeros_like(v[:, :1])
    e_mu = (DEPTH * U * v.abs().mean(1, keepdim=True) + e_v.mean(1, keepdim=True)) * (kind == 0)
    c = v - mu
    rs = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    e_c = e_v + e_mu + U * (v.abs() + mu.abs())
    # d(rs) = -rs^3 mean(c dc), the squares' sum within DEPTH u of itself
    e_rs = rs * (DEPTH * U + 4 * U + rs ** 2 * ((c.abs() + e_c) * e_c).mean(1, keepdim=True))
    xh = c * rs
    e_xh = (e_c * rs + c.abs() * e_rs + e_c * e_rs) + U * xh.abs()
    out = xh * w + (b if b is not None else 0)
    return mu, e_mu + U * mu.abs(), rs, e_rs, out, e_xh * w.abs() + 4 * U * ((xh * w).abs() + out.abs())


def gates64(torch, gate, gate_rows, rows):
    return gate.double().repeat_interleave(gate_rows, 0)[:rows]


def check_forward(torch, kind, step, d, gate_rows, y, h, st):
    dd = {k: v.double() if v is not None else None for k, v in d.items()}
    rows = d["o"].shape[0]
    n, e = dd["o"], torch.zeros_like(dd["o"])
    if d["post_w"] is not None:
        mu, e_mu, rs, e_rs, n, e = norm64(torch, kind, n, e, dd["post_w"], dd["post_b"])
        within(torch, st[:, 0:1], mu, e_mu)
        within(torch, st[:, 1:2], rs, e_rs)
    else:
        assert not st[:, :2].any()
    if d["gate"] is not None:
        g = gates64(torch, d["gate"], gate_rows, rows)
        n, e = n * g, e * g.abs() + U * (n * g).abs()
    want = RES * dd["x"] + n
    e = e + U * ((RES * dd["x"]).abs() + want.abs())
    within(torch, y, want, e + step * (want.abs() + e))
    if d["pre_w"] is not None:
        mu, e_mu, rs, e_rs, H, e_h = norm64(torch, kind, want, e, dd["pre_w"], dd["pre_b"])
        within(torch, st[:, 2:3], mu, e_mu)
        within(torch, st[:, 3:4], rs, e_rs)
        within(torch, h, H, e_h + step * (H.abs() + e_h))
    else:
        assert not st[:, 2:].any()


def back64(torch, kind, up, e_up, hat, e_hat, rs):
    """A norm's backward pass from `up` known within e_up."""
    c1 = up.mean(1, keepdim=True) if kind == 0 else torch.zeros_like(rs)
    c2 = (up * hat).mean(1, keepdim=True)
    e_c1 = DEPTH * U * up.abs().mean(1, keepdim=True) + e_up.mean(1, keepdim=True)
    e_c2 = (DEPTH * U * (up * hat).abs().mean(1, keepdim=True)
            + (up.abs() * e_hat + e_up * (hat.abs() + e_hat)).mean(1, keepdim=True))
    e = rs * (e_up + e_c1 + (hat.abs() + e_hat) * e_c2 + e_hat * c2.abs()
              + 6 * U * (up.abs() + c1.abs() + (hat * c2).abs()))
    return rs * (up - c1 - hat * c2), e


def check_backward(torch, kind, step, d, gate_rows, y, st, dh, dy, got):
    dd = {k: v.double() if v is not None else None for k, v in d.items()}
    rows, cols = d["o"].shape
    s = st.double()
    t, e = torch.zeros(rows, cols, dtype=torch.float64, device="cuda"), 0.0
    if d["pre_w"] is not None:
        rs, mu, H = s[:, 3:4], s[:, 2:3], dh.double()
        hat = (y.double() - mu) * rs
        e_hat = 3 * U * (y.double().abs() + mu.abs()) * rs
        up = H * dd["pre_w"]
        t, e = back64(torch, kind, up, U * up.abs(), hat, e_hat, rs)
        within(torch, got["dpre_w"], (H * hat).sum(0), DEPTH * U * (H * hat).abs().sum(0) + (H.abs() * e_hat).sum(0))
        if got["dpre_b"] is not None:
            within(torch, got["dpre_b"], H.sum(0), DEPTH * U * H.abs().sum(0))
    if dy is not None:
        t = t + dy.double()
        e = e + U * t.abs()
    e = e + torch.zeros_like(t)
    within(torch, got["dx"], RES * t, RES * e + 2 * U * t.abs() + step * RES * (t.abs() + e))
    v, hat, e_hat = dd["o"], dd["o"], torch.zeros_like(t)
    post, g = d["post_w"] is not None, 1.0
    if post:
        rs, mu = s[:, 1:2], s[:, 0:1]
        hat = (v - mu) * rs
        e_hat = 3 * U * (v.abs() + mu.abs()) * rs
    e_prod = e * (hat.abs() + e_hat) + t.abs() * e_hat
    if d["gate"] is not None:
        G, w, b = d["gate"].shape[0], dd["post_w"] if post else 1.0, dd["post_b"]
        g = gates64(torch, d["gate"], gate_rows, rows)
        which = torch.arange(rows, device="cuda") // gate_rows
        by = lambda z: torch.zeros(G, cols, dtype=torch.float64, device="cuda").index_add(0, which, z)  # noqa: E731
        S1, S0 = by(t * hat), by(t)
        e1 = by(e_prod) + (DEPTH + 8) * U * by((t * hat).abs())
        e0 = by(e) + (DEPTH + 8) * U * by(t.abs())
        aw = w.abs() if post else 1.0
        want, bound = S1 * w, e1 * aw
        if b is not None:
            want, bound = want + S0 * b, bound + e0 * b.abs()
        if got["dgate"] is not None:
            within(torch, got["dgate"], want, bound + 4 * U * (want.abs() + bound))
        e = e * g.abs() + U * (t * g).abs()
        t = t * g
        e_prod = e_prod * g.abs()
    if post:
        # (a gate's sums may be formed before the gate multiplies them)
        P = (DEPTH + 16) * U
        within(torch, got["dpost_w"], (t * hat).sum(0), P * (t * hat).abs().sum(0) + e_prod.sum(0)
               + (U * t.abs() * hat.abs()).sum(0))
        if got["dpost_b"] is not None:
            within(torch, got["dpost_b"], t.sum(0), P * t.abs().sum(0) + e.sum(0))
        up = t * dd["post_w"]
        t, e = back64(torch, kind, up, e * dd["post_w"].abs() + U * up.abs(), hat, e_hat, rs)
    within(torch, got["do"], t, e + step * (t.abs() + e))


NAMES = ("dx", "do", "dpost_w", "dpost_b", "dgate", "dpre_w", "dpre_b")


def backward(hip, ctx, torch, kind, bf16, d, gate_rows, y, st, dh, dy, off=0, without=(), dx=None):
    rows, cols = d["o"].shape
    t, _ = types(torch, bf16)
    G = d["gate"].shape[0] if d["gate"] is not None else 0
    out = {"dx": Guarded(torch, (rows, cols), t, off), "do": Guarded(torch, (rows, cols), t, off)}
    for name, of in (("dpost_w", "post_w"), ("dpost_b", "post_b"), ("dgate", "gate"), ("dpre_w", "pre_w"),
                     ("dpre_b", "pre_b")):
        there = d[of] is not None and name not in without
        out[name] = Guarded(torch, (G, cols) if name == "dgate" else (cols,), torch.float32, off) if there else None
    n = hip.lib().seeai_block_join_workspace(rows, cols, gate_rows if G else 0)
    ws, p = Guarded(torch, (n,), torch.uint8), hip.ptr
    at = {k: p(v.t) if v is not None else None for k, v in out.items()}
    if dx is not None:
        at["dx"] = p(dx)
    j = struct(hip, kind, bf16, d, rows, cols, gate_rows)
    j.x = None
    ctx.call("seeai_block_join_bwd", j, p(y) if d["pre_w"] is not None else None, p(st), p(dh), p(dy),
             hip.BlockJoinGrads(*(at[k] for k in NAMES)), p(ws.t) if n else None, n)
    assert ws.intact() and all(v is None or v.intact() for v in out.values())
    res = {k: v.t if v is not None else None for k, v in out.items()}
    if dx is not None:
        res["dx"] = dx
    return res


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("form", FORMS)
def test_block_join(hip, ctx, torch_cuda, form, bf16, off):
    torch = torch_cuda
    kind, post, pre, bias = form
    t, step = types(torch, bf16)
    for rows, cols, gate_rows in SHAPES:
        print(f"join form={form} bf16={bf16} off={off} {rows}x{cols} gates of {gate_rows}", flush=True)
        d = inputs(torch, kind, post, pre, bias, rows, cols, gate_rows, t, off)
        y, h, st = forward(hip, ctx, torch, kind, bf16, d, rows, cols, gate_rows, off)
        check_forward(torch, kind, step, d, gate_rows, y, h, st)
        rnd = gen(torch, rows + cols)
        dh = put(torch, rnd(rows, cols), t, off) if pre else None
        dy = put(torch, rnd(rows, cols), t, off)
        got = backward(hip, ctx, torch, kind, bf16, d, gate_rows, y, st, dh, dy, off)
        check_backward(torch, kind, step, d, gate_rows, y, st, dh, dy, got)
        # In place, and the same bits again.
        again = backward(hip, ctx, torch, kind, bf16, d, gate_rows, y, st, dh, dy, off, dx=dy)
        assert all(got[k] is None or torch.equal(got[k], again[k]) for k in NAMES)
        x = d["x"]
        y2, h2, _ = forward(hip, ctx, torch, kind, bf16, d, rows, cols, gate_rows, off, y=x, stats=False)
        assert torch.equal(y2, y) and (not pre or torch.equal(h2, h))


@pytest.mark.parametrize("which", [("o",), ("y", "h"), ("dx",), ("dh", "do")])
def test_block_join_of_tensors_that_lie_differently(hip, ctx, torch_cuda, which):
    """Some operands off a dword, the others on it: the bits of operands all on 16 bytes."""
    torch = torch_cuda
    t = torch.bfloat16
    for rows, cols in ((40, 128), (37, 514), (9, 4098), (300, 30)):
        d = inputs(torch, 0, 1, 1, 1, rows, cols, 7, t, 0)
        y, h, st = forward(hip, ctx, torch, 0, 1, d, rows, cols, 7)
        dh, dy = put(torch, gen(torch, 1)(rows, cols), t), put(torch, gen(torch, 2)(rows, cols), t)
        want = backward(hip, ctx, torch, 0, 1, d, 7, y, st, dh, dy)
        at = lambda name: Guarded(torch, (rows, cols), t, int(name in which))  # noqa: E731
        o, gy, gh, gdx, gdo, gdh = (at(k) for k in ("o", "y", "h", "dx", "do", "dh"))
        o.t.copy_(d["o"]), gdh.t.copy_(dh)
        j = struct(hip, 0, 1, d | {"o": o.t}, rows, cols, 7)
        p = hip.ptr
        ctx.call("seeai_block_join_fwd", j, p(gy.t), p(gh.t), p(st))
        assert torch.equal(gy.t, y) and torch.equal(gh.t, h) and gy.intact() and gh.intact()
        n = hip.lib().seeai_block_join_workspace(rows, cols, 7)
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
        grads = {k: torch.empty_like(want[k]) for k in NAMES[2:]}
        ctx.call("seeai_block_join_bwd", j, p(gy.t), p(st), p(gdh.t), p(dy),
                 hip.BlockJoinGrads(p(gdx.t), p(gdo.t), *(p(grads[k]) for k in NAMES[2:])), p(ws), n)
        assert torch.equal(gdx.t, want["dx"]) and torch.equal(gdo.t, want["do"]) and gdx.intact() and gdo.intact()
        assert all(torch.equal(grads[k], want[k]) for k in NAMES[2:])


def test_block_join_without_some_gradients(hip, ctx, torch_cuda):
    torch = torch_cuda
    for rows, cols, gate_rows in ((300, 264, 100), (300, 264, 2), (5, 64, 5)):
        d = inputs(torch, 0, 1, 1, 1, rows, cols, gate_rows, torch.float32, 0)
        y, _, st = forward(hip, ctx, torch, 0, 0, d, rows, cols, gate_rows)
        dh, dy = gen(torch, 1)(rows, cols), gen(torch, 2)(rows, cols)
        whole = backward(hip, ctx, torch, 0, 0, d, gate_rows, y, st, dh, dy)
        some = backward(hip, ctx, torch, 0, 0, d, gate_rows, y, st, dh, dy, without=("dgate", "dpost_b", "dpre_b"))
        assert some["dgate"] is None
        assert all(torch.equal(whole[k], v) for k, v in some.items() if v is not None)
        none = backward(hip, ctx, torch, 0, 0, d, gate_rows, y, st, dh, None)  # nothing reaches y past h
        check_backward(torch, 0, U, d, gate_rows, y, st, dh, None, none)


def test_block_join_of_no_rows_and_odd_values(hip, ctx, torch_cuda):
    torch = torch_cuda
    w = torch.ones(24, device="cuda")
    g = [torch.full((24,), 3.0, device="cuda") for _ in range(4)]
    p = hip.ptr
    j = hip.BlockJoin(None, None, p(w), p(w), None, p(w), p(w), 0, 24, 0, 0, 0, 1.0, EPS)
    ctx.call("seeai_block_join_fwd", j, None, None, None)
    grads = hip.BlockJoinGrads(None, None, p(g[0]), p(g[1]), None, p(g[2]), p(g[3]))
    ctx.call("seeai_block_join_bwd", j, None, None, None, None, grads, None, 0)
    assert not any(v.any() for v in g)
    # A NaN or an infinity stays in its row; its columns' sums take it.
    d = inputs(torch, 0, 1, 1, 1, 7, 40, 3, torch.float32, 0)
    d["o"][1, 3], d["x"][2, 5], d["o"][4], d["x"][4] = float("nan"), float("inf"), 2.5, 0.0
    y, h, st = forward(hip, ctx, torch, 0, 0, d, 7, 40, 3)
    assert y[1].isnan().all() and h[2].isnan().any() and torch.isfinite(y[[0, 3, 4, 5, 6]]).all()
    assert torch.isfinite(h[[0, 3, 4, 5, 6]]).all()
    dh, dy = gen(torch, 1)(7, 40), gen(torch, 2)(7, 40)
    got = backward(hip, ctx, torch, 0, 0, d, 3, y, st, dh, dy)
    assert torch.isfinite(got["dx"][[0, 3, 4, 5, 6]]).all() and torch.isfinite(got["do"][[0, 3, 4, 5, 6]]).all()
    assert got["dpost_w"].isnan().all() and torch.isfinite(got["dgate"][1:]).all()


def test_block_join_past_32_bit_offsets(hip, ctx, torch_cuda):
    """Over 2^32 bytes and 2^31 elements: the last rows are the formulas'."""
    torch = torch_cuda
    rows, cols, gate_rows = 1_060_000, 2048, 400_000
    rnd = gen(torch, 1)
    t = torch.bfloat16
    o = torch.empty(rows, cols, dtype=t, device="cuda").normal_()
    x = torch.empty(rows, cols, dtype=t, device="cuda").normal_()
    d = {"o": o, "x": x, "post_w": 1 + 0.1 * rnd(cols), "post_b": None, "gate": rnd(3, cols), "pre_w": 1 + rnd(cols),
         "pre_b": None}
    y, h, st = torch.empty_like(o), torch.empty_like(o), torch.empty(rows, 4, device="cuda")
    j = struct(hip, 1, 1, d, rows, cols, gate_rows)
    ctx.call("seeai_block_join_fwd", j, y.data_ptr(), h.data_ptr(), st.data_ptr())
    cuts = [(slice(0, 5), 0), (slice(rows - 5, rows), 2), (slice(399_998, 400_000), 0), (slice(400_000, 400_003), 1)]
    for s, g in cuts:
        part = {k: v[s] if k in ("o", "x") else v[g:g + 1] if k == "gate" else v for k, v in d.items()}
        check_forward(torch, 1, 2.0 ** -8, part, 10, y[s], h[s], st[s])
    dx = torch.empty_like(o)
    grads = {"dx": dx, "do": x, "dpost_w": torch.empty(cols, device="cuda"), "dpost_b": None,
             "dgate": torch.empty(3, cols, device="cuda"), "dpre_w": torch.empty(cols, device="cuda"), "dpre_b": None}
    n = hip.lib().seeai_block_join_workspace(rows, cols, gate_rows)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    j.x = None
    ctx.call("seeai_block_join_bwd", j, y.data_ptr(), st.data_ptr(), h.data_ptr(), None,
             hip.BlockJoinGrads(*(hip.ptr(grads[k]) for k in NAMES)), ws.data_ptr(), n)
    for s, g in cuts:
        part = {k: v[s] if k in ("o", "x") else v[g:g + 1] if k == "gate" else v for k, v in d.items()}
        got = {"dx": dx[s], "do": x[s], "dgate": None}
        dd = {k: v.double() if v is not None else None for k, v in part.items()}
        sd, H = st[s].double(), h[s].double()
        hat = (y[s].double() - 0) * sd[:, 3:4]
        e_hat = 3 * U * y[s].double().abs() * sd[:, 3:4]
        up = H * dd["pre_w"]
        T, e = back64(torch, 1, up, U * up.abs(), hat, e_hat, sd[:, 3:4])
        within(torch, got["dx"], RES * T, RES * e + 2 * U * T.abs() + 2.0 ** -8 * RES * (T.abs() + e))
        up = T * dd["gate"] * dd["post_w"]
        e_up = e * (dd["gate"] * dd["post_w"]).abs() + 2 * U * up.abs()
        ohat = dd["o"] * sd[:, 1:2]
        D, e = back64(torch, 1, up, e_up, ohat, 3 * U * ohat.abs(), sd[:, 1:2])
        within(torch, got["do"], D, e + 2.0 ** -8 * (D.abs() + e))


# --- together -------------------------------------------------------------------------------------

class Step:
    """A training step on preferences: a block's output o and the residual x, the
    join (norm after, gate, norm before), a feed-forward block, the last join, a
    head over V tokens, the paired loss, every gradient, the clip and AdamW."""

    KEYS = ("post1", "post1_b", "gate1", "pre1", "pre1_b", "wg", "wu", "wd", "post2", "post2_b", "gate2", "pre2",
            "pre2_b", "head")

    def __init__(self, hip, ctx, torch, seqs, D, F, V, seed=0):
        self.hip, self.ctx, self.torch = hip, ctx, torch
        rnd = gen(torch, seed)
        M = sum(seqs)
        self.M, self.D, self.F, self.V, self.Q = M, D, F, V, len(seqs)
        self.gate_rows = 7
        G = -(-M // 7)
        new = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
        self.o, self.x = rnd(M, D), rnd(M, D)
        shapes = {"wg": (D, F), "wu": (D, F), "wd": (F, D), "head": (D, V)}
        self.w = {}
        for k in self.KEYS:
            if k in shapes:
                self.w[k] = rnd(*shapes[k]) * shapes[k][0] ** -0.5
            elif k == "gate1":
                self.w[k] = 0.5 + 0.2 * rnd(G, D)
            elif k.startswith("gate"):
                self.w[k] = 0.5 + 0.2 * rnd(1, D)
            else:
                self.w[k] = (0.0 if k.endswith("_b") else 1.0) + 0.2 * rnd(D)
        self.g = {k: torch.empty_like(v) for k, v in self.w.items()}
        self.starts = torch.tensor([0, *torch.tensor(seqs).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
        lab = torch.randint(0, V, (M,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + 1))
        self.labels = torch.where(rnd(M) < 0.7, lab, -1).to(torch.int32)
        self.ref = -rnd(M).abs() - 1
        self.a = {k: new(M, D) for k in ("y1", "h1", "f", "y2", "h2", "dh2", "dy1", "df", "dh1", "dx", "do")}
        self.a |= {k: new(M, F) for k in ("G", "U")} | {"z": new(M, V), "st1": new(M, 4), "st2": new(M, 4)}
        self.a |= {"logp": new(M), "stats": new(M, 2), "dlogp": new(M), "loss": new(1), "margin": new(self.Q // 2),
                   "norm": new(1), "factor": new(1)}
        lib = hip.lib()
        byte = lambda n: torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")  # noqa: E731
        self.ws_f = byte(max(lib.seeai_ffn_workspace(0, M, D, F, b) for b in (0, 1)))
        self.ws_1 = byte(lib.seeai_block_join_workspace(M, D, 7))
        self.ws_2 = byte(lib.seeai_block_join_workspace(M, D, M))
        self.ws_p = byte(lib.seeai_pref_workspace(self.Q // 2))
        self.state = {k: {"p": v, "g": self.g[k], "m": torch.zeros_like(v), "v": torch.zeros_like(v)}
                      for k, v in self.w.items()}
        self.clip = hip.GradGroup(ctx, list(self.g.values()))
        self.group = hip.AdamWGroup(ctx, list(self.state.values()), 32, "f32", seed=3)

    def joins(self):
        p, w, a = self.hip.ptr, self.w, self.a
        one = self.hip.BlockJoin(p(self.o), p(self.x), p(w["post1"]), p(w["post1_b"]), p(w["gate1"]), p(w["pre1"]),
                                 p(w["pre1_b"]), self.M, self.D, self.gate_rows, 0, 0, 1.0, EPS)
        two = self.hip.BlockJoin(p(a["f"]), p(a["y1"]), p(w["post2"]), p(w["post2_b"]), p(w["gate2"]), p(w["pre2"]),
                                 p(w["pre2_b"]), self.M, self.D, self.M, 0, 0, 1.0, EPS)
        return one, two

    def gradients(self):
        p, w, a, g, c = self.hip.ptr, self.w, self.a, self.g, self.ctx
        M, D, F, V = self.M, self.D, self.F, self.V
        one, two = self.joins()
        c.call("seeai_block_join_fwd", one, p(a["y1"]), p(a["h1"]), p(a["st1"]))
        c.call("seeai_ffn_fwd", 0, 3, p(a["h1"]), p(w["wg"]), p(w["wu"]), p(w["wd"]), p(a["G"]), p(a["U"]), p(a["f"]),
               M, D, F, p(self.ws_f), self.ws_f.numel())
        c.call("seeai_block_join_fwd", two, p(a["y2"]), p(a["h2"]), p(a["st2"]))
        c.call("seeai_gemm_f32", 0, p(a["h2"]), p(w["head"]), p(a["z"]), M, V, D, None, 0, None, 1.0, 0)
        c.call("seeai_token_logp_fwd", 0, p(a["z"]), V, p(self.labels), p(a["logp"]), p(a["stats"]), M, V)
        c.call("seeai_pref_loss", p(a["logp"]), p(self.ref), p(self.labels), p(self.starts), M, self.Q // 2, 0.5, 0.0,
               0.1, 0, 2.0 / self.Q, p(a["loss"]), p(a["margin"]), p(a["dlogp"]), p(self.ws_p), self.ws_p.numel())
        c.call("seeai_token_logp_bwd", 0, p(a["z"]), V, p(self.labels), p(a["stats"]), p(a["dlogp"]), p(a["z"]), M, V)
        c.call("seeai_gemm_f32", 1, p(a["z"]), p(w["head"]), p(a["dh2"]), M, D, V, None, 0, None, 1.0, 0)
        c.call("seeai_gemm_f32", 2, p(a["h2"]), p(a["z"]), p(g["head"]), D, V, M, None, 0, None, 1.0, 0)
        c.call("seeai_block_join_bwd", two, p(a["y2"]), p(a["st2"]), p(a["dh2"]), None,
               self.hip.BlockJoinGrads(p(a["dy1"]), p(a["df"]), p(g["post2"]), p(g["post2_b"]), p(g["gate2"]),
                                       p(g["pre2"]), p(g["pre2_b"])), p(self.ws_2), self.ws_2.numel())
        c.call("seeai_ffn_bwd", 0, 3, p(a["h1"]), p(w["wg"]), p(w["wu"]), p(w["wd"]), p(a["G"]), p(a["U"]), p(a["df"]),
               p(a["dh1"]), p(g["wg"]), p(g["wu"]), p(g["wd"]), M, D, F, p(self.ws_f), self.ws_f.numel())
        c.call("seeai_block_join_bwd", one, p(a["y1"]), p(a["st1"]), p(a["dh1"]), p(a["dy1"]),
               self.hip.BlockJoinGrads(p(a["dx"]), p(a["do"]), p(g["post1"]), p(g["post1_b"]), p(g["gate1"]),
                                       p(g["pre1"]), p(g["pre1_b"])), p(self.ws_1), self.ws_1.numel())

    def params(self, n):
        return self.hip.StepParams(1e-2, 0.9, 0.999, 1e-8, 0.05, 0, n)

    def step(self, n, held=False):
        self.gradients()
        self.clip.norm(0.5, self.a["norm"], self.a["factor"])
        self.group.step(None if held else self.params(n), self.a["factor"])

    def tensors(self):
        return [*self.a.values(), *self.g.values(), *(v for s in self.state.values() for v in s.values())]


def step_loss64(torch, s, o, x, w):
    """The step's loss in float64, from the definitions."""
    def norm(v, weight, bias):
        mu = v.mean(1, keepdim=True)
        return (v - mu) / torch.sqrt(((v - mu) ** 2).mean(1, keepdim=True) + EPS) * weight + bias
    y1 = x + w["gate1"].repeat_interleave(s.gate_rows, 0)[:s.M] * norm(o, w["post1"], w["post1_b"])
    h1 = norm(y1, w["pre1"], w["pre1_b"])
    gate = h1 @ w["wg"]
    f = (gate * torch.sigmoid(gate) * (h1 @ w["wu"])) @ w["wd"]
    h2 = norm(y1 + w["gate2"] * norm(f, w["post2"], w["post2_b"]), w["pre2"], w["pre2_b"])
    lp = torch.log_softmax(h2 @ w["head"], 1).gather(1, s.labels.clamp(min=0).long()[:, None])[:, 0]
    diff = torch.where(s.labels >= 0, lp - s.ref.double(), 0.0)
    at = s.starts.tolist()
    sums = torch.stack([diff[a:b].sum() for a, b in zip(at, at[1:])])
    margin = 0.5 * (sums[0::2] - sums[1::2])
    ls = torch.nn.functional.logsigmoid
    eps = float(torch.tensor(0.1))
    return (-(1 - eps) * ls(margin) - eps * ls(-margin)).mean()


def test_preference_step_gradients_against_differences(hip, ctx, torch_cuda):
    torch = torch_cuda
    s = Step(hip, ctx, torch, [5, 9, 3, 6], 48, 80, 70)
    s.gradients()
    w = {k: v.double() for k, v in s.w.items()}
    o, x = s.o.double(), s.x.double()
    want = float(step_loss64(torch, s, o, x, w))
    assert abs(float(s.a["loss"]) - want) <= 1e-5 * abs(want)
    h = 2.0 ** -13
    for i, (k, grad) in enumerate([*s.g.items(), ("o", s.a["do"]), ("x", s.a["dx"])]):
        d = gen(torch, 40 + i)(*grad.shape).double()
        d /= d.norm()
        at = []
        for sign in (h, -h):
            w2 = w | {k: w[k] + sign * d} if k in w else w
            at.append(float(step_loss64(torch, s, o + sign * d if k == "o" else o,
                                        x + sign * d if k == "x" else x, w2)))
        got = float((grad.double() * d).sum())
        # f32's and the difference's own error, relative to the gradient's size
        assert abs((at[0] - at[1]) / (2 * h) - got) <= 2e-5 * float(grad.double().norm()) + 1e-9, k


def test_preference_steps_captured_and_replayed(hip, torch_cuda):
    """A step captured once and replayed, eager work in between, against the same
    steps run eagerly; two graphs with workspaces of their own on two streams."""
    torch = torch_cuda
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ctxs = []
    for st in streams:
        c = hip.Context(0)
        with torch.cuda.stream(st):
            c.use_torch_stream()
        ctxs.append(c)
    ce = hip.Context(0)
    ce.use_torch_stream()
    size = ([30, 41, 7, 64], 136, 264, 1000)
    eager, warm = Step(hip, ce, torch, *size), None
    steps = [Step(hip, c, torch, *size) for c in ctxs]
    torch.cuda.synchronize()
    for c, st in zip(ctxs, streams):  # the products' scratch is taken at their first use
        warm = Step(hip, c, torch, *size, seed=9)
        warm.step(1)
        st.synchronize()
    graphs = []
    for s, st in zip(steps, streams):
        s.group.hold(s.params(1))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            s.step(1, held=True)
            with pytest.raises(hip.BackendError, match="held params"):
                s.group.step(s.params(1), s.a["factor"])
            with pytest.raises(hip.BackendError, match="captured"):
                hip.GradGroup(s.ctx, [s.o])
        graphs.append(g)
    for n in range(1, 6):
        for s in steps:
            s.group.hold(s.params(n))
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        eager.step(n)
        junk = torch.randn(512, 512, device="cuda") @ torch.randn(512, 512, device="cuda")
        torch.cuda.synchronize()
        for s in steps:
            for got, want in zip(s.tensors(), eager.tensors()):
                assert torch.equal(got, want), n
    assert torch.isfinite(junk).all() and torch.isfinite(eager.a["loss"]).all()


def test_join_refuses_on_the_context(hip, ctx, torch_cuda):
    torch = torch_cuda
    x, w = torch.zeros(4, 8, device="cuda"), torch.ones(8, device="cuda")
    p = hip.ptr
    j = hip.BlockJoin(p(x), p(x), p(w), None, None, None, None, 4, 8, 0, 1, 0, 1.0, EPS)
    with pytest.raises(hip.BackendError, match="block_join_fwd: an output overlaps"):
        ctx.call("seeai_block_join_fwd", j, p(x), None, None)  # y over o
    with pytest.raises(hip.BackendError, match="block_join_bwd: null operand"):
        ctx.call("seeai_block_join_bwd", j, None, None, None, None, hip.BlockJoinGrads(), None, 0)
    with pytest.raises(hip.BackendError, match="null argument"):
        ctx.call("seeai_block_join_fwd", None, p(x), None, None)
    assert hip.lib().seeai_block_join_fwd(None, j, None, None, None) == 2
