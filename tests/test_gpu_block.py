"""GPU: the operators that train a block's own weights -- seeai_norm_fwd / _bwd,
seeai_ffn_fwd / _bwd, seeai_adamw_group_* -- against plain float64.

Tolerances are bounds, element by element, on what the kernels' own roundings
may add up to: u = 2^-24 for each f32 operation, 2^-8 of the value for each
rounding to bf16 (half a step), carried through the formulas below.  A sum of n
f32 terms in any order is within n u of its terms' magnitudes."""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5


@pytest.fixture(scope="module")
def ctx(hip, torch_cuda):
    c = hip.Context(0)
    c.use_torch_stream()
    yield c
    torch_cuda.cuda.synchronize()


def types(torch, bf16):
    """The element type, and half its rounding step relative to the value."""
    return (torch.bfloat16, 2.0 ** -8) if bf16 else (torch.float32, U)


def gen(torch, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s: torch.randn(s, device="cuda", generator=g)


class Guarded:
    """A tensor with a guard behind it that a kernel must leave alone, and,
    `off` elements from a 256-byte boundary."""

    def __init__(self, torch, shape, dtype, off=0):
        n = math.prod(shape)
        self.raw = torch.full((n + off + 64,), 7.0, device="cuda").to(dtype)
        self.t = self.raw[off:off + n].view(shape)
        self.off, self.n = off, n

    def intact(self):
        return bool((self.raw[:self.off] == 7).all() and (self.raw[self.off + self.n:] == 7).all())


def put(torch, src, dtype, off=0):
    g = Guarded(torch, tuple(src.shape), dtype, off)
    g.t.copy_(src)
    return g.t


def within(torch, got, want, bound):
    got = got.to(torch.float64)
    bad = ~((got - want).abs() <= bound) & ~(got == want)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} past their bound, worst "
                           f"{float(((got - want).abs() / bound)[bad].max()):.3g} times it")


# --- the norms ------------------------------------------------------------------------------------

NORM_SHAPES = [(1, 1), (3, 7), (1, 768), (5, 64), (70, 512), (9, 513), (130, 1000), (33, 1023),
               (2100, 1024), (64, 1030), (40, 2048), (7, 2050), (600, 4096), (5, 5001), (3, 8192),
               (4, 8193), (3, 16384), (2, 16385), (130, 20000), (6, 2051), (4, 6143), (3, 257),
               (2, 12289)]
DEPTH = 260  # f32 additions behind one sum over a row's or a column's partials


def norm_reference(torch, kind, x, w, b, dy):
    """float64 results and their bounds, forward and backward."""
    x, w, dy = x.double(), w.double(), dy.double()
    n = x.shape[1]
    mu = x.mean(1, keepdim=True) if kind == 0 else torch.zeros_like(x[:, :1])
    rs = 1 / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + EPS)
    ax = x.abs().mean(1, keepdim=True)
    e_mu = DEPTH * U * ax * (kind == 0)
    xh = (x - mu) * rs
    y = xh * w + (b.double() if b is not None else 0)
    # rs from a sum of squares about a mean that is e_mu off.
    e_rs = rs * (DEPTH * U + rs * e_mu * 2)
    e_xh = 4 * U * (x.abs() + mu.abs()) * rs + e_mu * rs + xh.abs() * (e_rs / rs)
    e_y = e_xh * w.abs() + 4 * U * ((xh * w).abs() + y.abs())
    return {"mu": mu, "rs": rs, "y": y, "e_mu": e_mu + U * mu.abs(), "e_rs": e_rs + 4 * U * rs,
            "e_y": e_y}


def norm_backward_reference(torch, kind, x, w, dy, mean, rstd):
    x, w, dy = x.double(), w.double(), dy.double()
    mu = mean.double()[:, None] if kind == 0 else torch.zeros_like(x[:, :1])
    rs = rstd.double()[:, None]
    xh = (x - mu) * rs
    e_xh = 3 * U * (x.abs() + mu.abs()) * rs
    d = dy * w
    c1 = d.mean(1, keepdim=True) if kind == 0 else torch.zeros_like(mu)
    c2 = (d * xh).mean(1, keepdim=True)
    e_c1 = DEPTH * U * d.abs().mean(1, keepdim=True)
    e_c2 = DEPTH * U * (d * xh).abs().mean(1, keepdim=True) + (d.abs() * e_xh).mean(1, keepdim=True)
    dx = rs * (d - c1 - xh * c2)
    e_dx = rs * (e_c1 + xh.abs() * e_c2 + e_xh * c2.abs()
                 + 6 * U * (d.abs() + c1.abs() + (xh * c2).abs()))
    dw, db = (dy * xh).sum(0), dy.sum(0)
    e_dw = DEPTH * U * (dy * xh).abs().sum(0) + (dy.abs() * e_xh).sum(0)
    e_db = DEPTH * U * dy.abs().sum(0)
    return dx, e_dx, dw, e_dw, db, e_db


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("kind", [0, 1])
def test_norm(ctx, torch_cuda, kind, bf16, off):
    torch = torch_cuda
    t, step = types(torch, bf16)
    for rows, cols in NORM_SHAPES:
        print(f"norm kind={kind} bf16={bf16} off={off} {rows}x{cols}", flush=True)
        rnd = gen(torch, rows * 31 + cols)
        x = put(torch, rnd(rows, cols) * 2 + rnd(rows, 1) * 3, t, off)
        w = put(torch, 1 + 0.3 * rnd(cols), torch.float32, off)
        b = put(torch, 0.5 * rnd(cols), torch.float32, off) if kind == 0 else None
        dy = put(torch, rnd(rows, cols), t, off)
        y, dx = Guarded(torch, (rows, cols), t, off), Guarded(torch, (rows, cols), t, off)
        mean, rstd = (Guarded(torch, (rows,), torch.float32) for _ in range(2))
        dw, db = (Guarded(torch, (cols,), torch.float32) for _ in range(2))
        call_norm_fwd(ctx, kind, bf16, x, w, b, y.t, mean.t if kind == 0 else None, rstd.t)
        ref = norm_reference(torch, kind, x, w, b, dy)
        within(torch, y.t, ref["y"], ref["e_y"] + step * ref["y"].abs())
        within(torch, rstd.t, ref["rs"][:, 0], ref["e_rs"][:, 0])
        if kind == 0:
            within(torch, mean.t, ref["mu"][:, 0], ref["e_mu"][:, 0])
        ws = norm_bwd(ctx, kind, bf16, dy, x, w, mean.t if kind == 0 else None, rstd.t, dx.t, dw.t,
                      db.t if kind == 0 else None)
        r = norm_backward_reference(torch, kind, x, w, dy, mean.t, rstd.t)
        within(torch, dx.t, r[0], r[1] + step * r[0].abs())
        within(torch, dw.t, r[2], r[3])
        if kind == 0:
            within(torch, db.t, r[4], r[5])
        assert all(g.intact() for g in (y, dx, mean, rstd, dw, db)) and ws.intact()
        again = Guarded(torch, (cols,), torch.float32)
        norm_bwd(ctx, kind, bf16, dy, x, w, mean.t if kind == 0 else None, rstd.t, dx.t, again.t, None)
        assert torch.equal(again.t, dw.t), "the weight's gradient differs run to run"


@pytest.mark.parametrize("rows,cols,off", [(8192, 1024, 0), (8199, 1023, 1), (16411, 520, 0),
                                           (8203, 2048, 0)])
@pytest.mark.parametrize("bf16", [0, 1])
def test_norm_backward_over_two_workgroups_a_cu(ctx, torch_cuda, bf16, rows, cols, off):
    """Rows enough for 512 workgroups' partial sums, the last of them without a full share."""
    torch = torch_cuda
    t, step = types(torch, bf16)
    rnd = gen(torch, rows + cols)
    x = put(torch, rnd(rows, cols) * 2 + rnd(rows, 1) * 3, t, off)
    w, dy = put(torch, 1 + 0.3 * rnd(cols), torch.float32, off), put(torch, rnd(rows, cols), t, off)
    mean = x.double().mean(1).float()
    rstd = (x.double().var(1, unbiased=False) + EPS).rsqrt().float()
    dx = Guarded(torch, (rows, cols), t, off)
    dw, db = (Guarded(torch, (cols,), torch.float32) for _ in range(2))
    ws = norm_bwd(ctx, 0, bf16, dy, x, w, mean, rstd, dx.t, dw.t, db.t)
    r = norm_backward_reference(torch, 0, x, w, dy, mean, rstd)
    within(torch, dx.t, r[0], r[1] + step * r[0].abs())
    within(torch, dw.t, r[2], r[3])
    within(torch, db.t, r[4], r[5])
    assert all(g.intact() for g in (dx, dw, db, ws))


def call_norm_fwd(ctx, kind, bf16, x, w, b, y, mean, rstd, eps=EPS):
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    ctx.call("seeai_norm_fwd", kind, bf16, p(x), p(w), p(b), p(y), p(mean), p(rstd), *x.shape, eps)


def norm_bwd(ctx, kind, bf16, dy, x, w, mean, rstd, dx, dw, db):
    import importlib
    import torch
    hip = importlib.import_module("see-ai_amd.hip")
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    n = hip.lib().seeai_norm_bwd_workspace(*x.shape)
    ws = Guarded(torch, (n,), torch.uint8)
    ctx.call("seeai_norm_bwd", kind, bf16, p(dy), p(x), p(w), p(mean), p(rstd), p(dx), p(dw), p(db),
             *x.shape, p(ws.t) if n else None, n)
    return ws


def test_norm_of_no_rows_and_odd_values(ctx, torch_cuda):
    torch = torch_cuda
    x, w = torch.zeros(0, 24, device="cuda"), torch.ones(24, device="cuda")
    none = torch.zeros(0, device="cuda")
    dw, db = torch.full((24,), 3.0, device="cuda"), torch.full((24,), 3.0, device="cuda")
    # A tensor of no elements has no address: any will do.
    ctx.call("seeai_norm_fwd", 0, 0, None, w.data_ptr(), w.data_ptr(), None, None, None, 0, 24, EPS)
    ctx.call("seeai_norm_bwd", 0, 0, None, None, w.data_ptr(), None, None, None, dw.data_ptr(),
             db.data_ptr(), 0, 24, None, 0)
    assert not dw.any() and not db.any() and x.numel() == none.numel() == 0
    # A NaN or an infinity stays in its row; a constant row has xhat = 0.
    x = torch.randn(6, 40, device="cuda")
    x[1, 3], x[2, 5], x[4] = float("nan"), float("inf"), 2.5
    y, rstd = torch.empty_like(x), torch.empty(6, device="cuda")
    w = torch.ones(40, device="cuda")
    call_norm_fwd(ctx, 0, 0, x, w, w, y, None, rstd)
    assert y[1].isnan().all() and y[2].isnan().any() and torch.isfinite(y[[0, 3, 4, 5]]).all()
    assert (y[4] == 1).all()


def test_norm_past_32_bit_offsets(ctx, torch_cuda):
    """Over 2^32 bytes and 2^31 elements: the last rows are the formula's."""
    torch = torch_cuda
    rows, cols = 1_060_000, 2048
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    x.normal_()
    w, b = torch.randn(cols, device="cuda"), torch.randn(cols, device="cuda")
    y, rstd = torch.empty_like(x), torch.empty(rows, device="cuda")
    call_norm_fwd(ctx, 0, 1, x, w, b, y, None, rstd)
    for s in (slice(0, 5), slice(rows - 5, rows)):
        ref = norm_reference(torch, 0, x[s], w, b, x[s])
        within(torch, y[s], ref["y"], ref["e_y"] + 2.0 ** -8 * ref["y"].abs())


# --- the gated feed-forward block -----------------------------------------------------------------

ACTS = {0: "none", 1: "relu", 2: "gelu", 3: "silu"}
FFN_SHAPES = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (2, 64, 128), (1, 520, 1032), (5, 257, 300),
              (16, 96, 96), (17, 128, 65), (24, 512, 640), (33, 200, 136), (64, 72, 264),
              (65, 129, 257), (130, 256, 128), (257, 264, 520), (300, 90, 1000), (1100, 160, 224)]


def act_of(torch, act, g):
    """The activation and its derivative, float64."""
    if act == 0:
        return g, torch.ones_like(g)
    if act == 1:
        return g.clamp(min=0), (g > 0).double()
    if act == 3:
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    k, c = math.sqrt(2 / math.pi), 0.044715
    th = torch.tanh(k * (g + c * g ** 3))
    return (0.5 * g * (1 + th),
            0.5 * (1 + th) + 0.5 * g * (1 - th * th) * k * (1 + 3 * c * g * g))


def gamma(n):
    """f32 sums of n products, each within a few roundings of the exact one."""
    return (n + 24) * U


def ffn_inputs(torch, M, D, F, t, off, seed):
    rnd = gen(torch, seed)
    return [put(torch, v, t, off) for v in
            (rnd(M, D), rnd(D, F) * D ** -0.5, rnd(D, F) * D ** -0.5, rnd(F, D) * F ** -0.5)]


def ffn_fwd(hip, ctx, torch, bf16, act, x, wg, wu, wd, keep, off=0):
    M, D, F = x.shape[0], x.shape[1], wg.shape[1]
    outs = [Guarded(torch, (M, n), x.dtype, off) for n in (F, F, D)]
    n = hip.lib().seeai_ffn_workspace(bf16, M, D, F, 0)
    ws = Guarded(torch, (n,), torch.uint8)
    p = lambda v: v.data_ptr()  # noqa: E731
    ctx.call("seeai_ffn_fwd", bf16, act, p(x), p(wg), p(wu), p(wd), p(outs[0].t) if keep else None,
             p(outs[1].t) if keep else None, p(outs[2].t), M, D, F, p(ws.t), n)
    assert all(o.intact() for o in outs) and ws.intact()
    return [o.t for o in outs]


def ffn_bwd(hip, ctx, torch, bf16, act, x, wg, wu, wd, gate, up, dy, off=0):
    M, D, F = x.shape[0], x.shape[1], wg.shape[1]
    outs = [Guarded(torch, s, x.dtype, off) for s in ((M, D), (D, F), (D, F), (F, D))]
    n = hip.lib().seeai_ffn_workspace(bf16, M, D, F, 1)
    ws = Guarded(torch, (n,), torch.uint8)
    p = lambda v: v.data_ptr()  # noqa: E731
    ctx.call("seeai_ffn_bwd", bf16, act, p(x), p(wg), p(wu), p(wd), p(gate), p(up), p(dy),
             *(p(o.t) for o in outs), M, D, F, p(ws.t), n)
    assert all(o.intact() for o in outs) and ws.intact()
    return [o.t for o in outs]


def check_ffn_fwd(torch, act, step, x, wg, wu, wd, gate, up, y):
    D, F = wg.shape
    x, wg, wu, wd = (v.double() for v in (x, wg, wu, wd))
    G, Up = x @ wg, x @ wu
    eG, eU = gamma(D) * (x.abs() @ wg.abs()), gamma(D) * (x.abs() @ wu.abs())
    if gate is not None:
        within(torch, gate, G, eG + step * G.abs())
        within(torch, up, Up, eU + step * Up.abs())
    a, _ = act_of(torch, act, G)
    H = a * Up
    # |act'| <= 1.13; the activation's own expression within 16 roundings of |G|.
    eA = 1.13 * eG + 16 * U * G.abs()
    eH = eA * (Up.abs() + eU) + a.abs() * eU + step * (H.abs() + eA * Up.abs()) + U * H.abs()
    Y = H @ wd
    eY = eH @ wd.abs() + gamma(F) * ((H.abs() + eH) @ wd.abs())
    within(torch, y, Y, eY + step * (Y.abs() + eY))


def check_ffn_bwd(torch, act, step, x, wg, wu, wd, gate, up, dy, dx, dwg, dwu, dwd):
    M, D, F = x.shape[0], *wg.shape
    x, wg, wu, wd, G, Up, dy = (v.double() for v in (x, wg, wu, wd, gate, up, dy))
    a, da = act_of(torch, act, G)
    dH = dy @ wd.t().contiguous()
    eH = gamma(D) * (dy.abs() @ wd.t().contiguous().abs())
    ops = 32 * U  # the activation's and its derivative's expressions
    dG, dU, H = dH * Up * da, dH * a, a * Up
    # GELU's derivative is a sum of terms that may cancel: its error is of their size.
    eG = eH * (Up * da).abs() + ops * (dH.abs() + eH) * Up.abs() * (1.2 + G.abs())
    eU = eH * a.abs() + ops * (dH.abs() + eH) * G.abs()
    eHh = ops * (G * Up).abs()
    eG, eU, eHh = (e + step * (v.abs() + e) for e, v in ((eG, dG), (eU, dU), (eHh, H)))
    wgt, wut, xt, ht = (v.t().contiguous() for v in (wg, wu, x, H))
    dX = dG @ wgt + dU @ wut
    eX = (eG @ wgt.abs() + eU @ wut.abs()
          + gamma(2 * F) * ((dG.abs() + eG) @ wgt.abs() + (dU.abs() + eU) @ wut.abs()))
    within(torch, dx, dX, eX + step * (dX.abs() + eX))
    for got, e, v in ((dwg, eG, dG), (dwu, eU, dU)):
        W, eW = xt @ v, xt.abs() @ e + gamma(M) * (xt.abs() @ (v.abs() + e))
        within(torch, got, W, eW + step * (W.abs() + eW))
    W = ht @ dy
    eW = eHh.t().contiguous() @ dy.abs() + gamma(M) * ((ht.abs() + eHh.t()) @ dy.abs())
    within(torch, dwd, W, eW + step * (W.abs() + eW))


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("act", [3, 2, 1, 0])
@pytest.mark.parametrize("bf16", [0, 1])
def test_ffn(hip, ctx, torch_cuda, bf16, act, off):
    torch = torch_cuda
    t, step = types(torch, bf16)
    shapes = FFN_SHAPES if act == 3 else FFN_SHAPES[2:14:3]
    for M, D, F in shapes:
        print(f"ffn bf16={bf16} act={ACTS[act]} off={off} M={M} D={D} F={F}", flush=True)
        ins = ffn_inputs(torch, M, D, F, t, off, M * 7 + D * 3 + F)
        gate, up, y = ffn_fwd(hip, ctx, torch, bf16, act, *ins, True, off)
        check_ffn_fwd(torch, act, step, *ins, gate, up, y)
        _, _, served = ffn_fwd(hip, ctx, torch, bf16, act, *ins, False, off)
        assert torch.equal(served, y), "y depends on whether the projections are kept"
        dy = put(torch, gen(torch, 5)(M, D), t, off)
        grads = ffn_bwd(hip, ctx, torch, bf16, act, *ins, gate, up, dy, off)
        check_ffn_bwd(torch, act, step, *ins, gate, up, dy, *grads)
        for a, b in zip(grads, ffn_bwd(hip, ctx, torch, bf16, act, *ins, gate, up, dy, off)):
            assert torch.equal(a, b), "a gradient differs run to run"


@pytest.mark.parametrize("bf16,M,D,F", [
    # the largest tile on every side of an f32 backward; few f32 rows (they take the weights as
    # they are) about where that ends, K long enough to be shared out, rows on and off 16 bytes
    (0, 4096, 64, 4096), (1, 4096, 64, 4096), (0, 1, 2048, 640), (0, 33, 1001, 1538),
    (0, 64, 700, 2052), (0, 65, 700, 2052), (0, 128, 700, 2052), (0, 129, 700, 2052),
    (0, 64, 4100, 36), (0, 7, 36, 9000)])
def test_ffn_sizes_a_rule_turns_at(hip, ctx, torch_cuda, bf16, M, D, F):
    torch = torch_cuda
    t, step = types(torch, bf16)
    ins = ffn_inputs(torch, M, D, F, t, 0, M + D + F)
    gate, up, y = ffn_fwd(hip, ctx, torch, bf16, 3, *ins, True)
    check_ffn_fwd(torch, 3, step, *ins, gate, up, y)
    dy = put(torch, gen(torch, 5)(M, D), t, 0)
    grads = ffn_bwd(hip, ctx, torch, bf16, 3, *ins, gate, up, dy)
    check_ffn_bwd(torch, 3, step, *ins, gate, up, dy, *grads)


# Sizes that between them take every tile the block's products can run on, with several stages of K,
# rows on and off 16 bytes, K whole, shared out, and shared out for the tiles past whole rounds alone
# (tests/test_ffn_plan.py holds the list to that).
TILE_SHAPES = [(300, 260, 515), (512, 1024, 4096), (700, 1000, 1500), (1001, 776, 2056),
               (1001, 777, 2050), (1500, 1033, 4107), (3000, 1000, 3000), (1024, 2048, 5632),
               (4096, 2048, 1408), (4097, 1030, 2055), (4000, 2050, 4100), (8190, 2050, 5630),
               (8192, 2048, 5632)]


@pytest.mark.parametrize("bf16", [1, 0])
@pytest.mark.parametrize("M,D,F", TILE_SHAPES)
def test_ffn_on_every_tile(hip, ctx, torch_cuda, M, D, F, bf16):
    torch = torch_cuda
    t, step = types(torch, bf16)
    for off in (0, 1) if M < 4000 else (0,):
        print(f"ffn tiles bf16={bf16} off={off} M={M} D={D} F={F}", flush=True)
        ins = ffn_inputs(torch, M, D, F, t, off, M + D + F)
        gate, up, y = ffn_fwd(hip, ctx, torch, bf16, 3, *ins, True, off)
        check_ffn_fwd(torch, 3, step, *ins, gate, up, y)
        dy = put(torch, gen(torch, 5)(M, D), t, off)
        grads = ffn_bwd(hip, ctx, torch, bf16, 3, *ins, gate, up, dy, off)
        check_ffn_bwd(torch, 3, step, *ins, gate, up, dy, *grads)
        for a, b in zip(ffn_fwd(hip, ctx, torch, bf16, 3, *ins, True, off)
                        + ffn_bwd(hip, ctx, torch, bf16, 3, *ins, gate, up, dy, off),
                        [gate, up, y, *grads]):
            assert torch.equal(a, b), "an output differs run to run"


@pytest.mark.parametrize("bf16", [1, 0])
def test_ffn_packing_past_a_row_of_workgroups(hip, ctx, torch_cuda, bf16):
    """Operands off 16 bytes of more than 2^27 elements together: packed by several rows of workgroups."""
    torch = torch_cuda
    t, step = types(torch, bf16)
    M, D, F = 70001, 2050, 9
    ins = ffn_inputs(torch, M, D, F, t, 0, 1)
    gate, up, y = ffn_fwd(hip, ctx, torch, bf16, 3, *ins, True)
    check_ffn_fwd(torch, 3, step, *ins, gate, up, y)
    dy = put(torch, gen(torch, 5)(M, D), t)
    grads = ffn_bwd(hip, ctx, torch, bf16, 3, *ins, gate, up, dy)
    check_ffn_bwd(torch, 3, step, *ins, gate, up, dy, *grads)


@pytest.mark.parametrize("e", [0, -110, -120])
@pytest.mark.parametrize("M", [100, 200])
def test_ffn_f32_products_leave_out_less_than_2_to_the_minus_21(hip, ctx, torch_cuda, M, e):
    """Past 128 tokens a term loses less than 2^-21 of itself, towards zero (here 7.8 2^-24, about the
    most there is), and an operand its bits below 2^-133, bf16's last; up to 128 tokens nothing.  The
    sum of D equal terms adds (D + 1) U for its own roundings."""
    torch = torch_cuda
    D, F, v = 16, 24, 1 + 2.0 ** -7 - 2.0 ** -23
    x, wg, wu, wd = (torch.full(s, v, device="cuda") for s in ((M, D), (D, F), (D, F), (F, D)))
    x *= 2.0 ** e
    x[1::2] *= -1
    gate, up, _ = ffn_fwd(hip, ctx, torch, 0, 0, x, wg, wu, wd, True)
    want = D * v * v * 2.0 ** e
    for got in (gate.double(), up.double()):
        assert (got[0::2] > 0).all() and (got[1::2] < 0).all()
        short = want - got.abs()  # (towards zero)
        assert (short >= -(D + 1) * U * want).all()
        left_out = (M > 128) * (2.0 ** -21 * want + D * v * 2.0 ** -133)
        assert (short <= left_out + (D + 1) * U * want).all()


def test_ffn_gradients_against_differences(hip, ctx, torch_cuda):
    """Central differences of the block's own forward, f32: the loss sum(y c) along random
    directions of x and of each weight.  A difference at h is off by h^2 of the third
    derivative (about 1 here) and by the loss's roundings over h."""
    torch = torch_cuda
    M, D, F, h = 6, 40, 56, 2.0 ** -7
    ins = ffn_inputs(torch, M, D, F, torch.float32, 0, 11)
    c = gen(torch, 12)(M, D)
    for act in (2, 3):
        gate, up, _ = ffn_fwd(hip, ctx, torch, 0, act, *ins, True)
        grads = ffn_bwd(hip, ctx, torch, 0, act, *ins, gate, up, c)
        for i in range(4):
            d = gen(torch, 20 + i)(*ins[i].shape)
            d /= d.norm()
            loss = []
            for s in (h, -h):
                moved = list(ins)
                moved[i] = ins[i] + s * d
                y = ffn_fwd(hip, ctx, torch, 0, act, *moved, False)[2]
                loss.append(float((y.double() * c.double()).sum()))
            want = float((grads[i].double() * d.double()).sum())
            size = float(grads[i].double().norm())
            assert abs((loss[0] - loss[1]) / (2 * h) - want) <= 1e-3 * size, (act, i)


def test_ffn_of_no_rows(hip, ctx, torch_cuda):
    torch = torch_cuda
    w = torch.randn(8, 16, device="cuda")
    wd = torch.randn(16, 8, device="cuda")
    d = [torch.full_like(v, 5.0) for v in (w, w, wd)]
    p = lambda v: v.data_ptr()  # noqa: E731
    ctx.call("seeai_ffn_fwd", 0, 3, None, p(w), p(w), p(wd), None, None, None, 0, 8, 16, None, 0)
    n = hip.lib().seeai_ffn_workspace(0, 0, 8, 16, 1)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    ctx.call("seeai_ffn_bwd", 0, 3, None, p(w), p(w), p(wd), None, None, None, None, *map(p, d), 0, 8,
             16, p(ws), n)
    assert not any(v.any() for v in d)


def test_ffn_values_that_are_not_finite(hip, ctx, torch_cuda):
    """What a NaN or an infinity in a token reaches is not finite; other tokens are as before."""
    torch = torch_cuda
    for bf16 in (0, 1):
        for M in (4, 40, 300):
            t, _ = types(torch, bf16)
            ins = ffn_inputs(torch, M, 128, 192, t, 0, 3)
            clean = ffn_fwd(hip, ctx, torch, bf16, 3, *ins, False)[2]
            ins[0][1, 5], ins[0][3, 7] = float("nan"), float("inf")
            y = ffn_fwd(hip, ctx, torch, bf16, 3, *ins, False)[2]
            keep = [i for i in range(M) if i not in (1, 3)]
            assert torch.equal(y[keep], clean[keep])
            assert y[1].isnan().all() and not torch.isfinite(y[3]).any()


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("bf16", [0, 1])
def test_ffn_nan_gates_reach_every_result(hip, ctx, torch_cuda, bf16, act):
    """A NaN in the gate's weights reaches y of every token, with every activation; one in a saved
    gate reaches the gradients that depend on it and no others.  (The derivative without an
    activation is 1 whatever the gate, so there the gate's weights' gradient stays finite.)"""
    torch = torch_cuda
    t, _ = types(torch, bf16)
    for M in (4, 40, 300):
        x, wg, wu, wd = ffn_inputs(torch, M, 128, 192, t, 0, 3)
        gate, up, _ = ffn_fwd(hip, ctx, torch, bf16, act, x, wg, wu, wd, True)
        dy = put(torch, gen(torch, 5)(M, 128), t)
        gate[2, 7] = float("nan")
        dx, dwg, dwu, dwd = ffn_bwd(hip, ctx, torch, bf16, act, x, wg, wu, wd, gate, up, dy)
        keep = [i for i in range(M) if i != 2]
        assert dx[2].isnan().all() and torch.isfinite(dx[keep]).all()
        cols = [i for i in range(192) if i != 7]
        assert act == 0 or dwg[:, 7].isnan().all()
        assert dwu[:, 7].isnan().all() and dwd[7].isnan().all()
        assert all(torch.isfinite(v).all() for v in (dwg[:, cols], dwu[:, cols], dwd[cols]))
        wg[5, 7] = float("nan")
        y = ffn_fwd(hip, ctx, torch, bf16, act, x, wg, wu, wd, False)[2]
        assert y.isnan().all()


@pytest.mark.parametrize("act", [1, 2, 3])
@pytest.mark.parametrize("bf16", [0, 1])
def test_ffn_gradients_at_large_gates(hip, ctx, torch_cuda, bf16, act):
    """Finite gates have finite derivatives, 0 or 1 far out, also where the gate's square is past
    f32."""
    torch = torch_cuda
    t, step = types(torch, bf16)
    for M in (4, 40, 300):
        ins = ffn_inputs(torch, M, 128, 192, t, 0, 3)
        gate, up = (put(torch, gen(torch, i)(M, 192), t) for i in (8, 9))
        gate[0, 1], gate[1, 3], gate[2, 5], gate[3, 2] = 1e25, 1e20, -1e20, -3e37
        dy = put(torch, gen(torch, 5)(M, 128), t)
        grads = ffn_bwd(hip, ctx, torch, bf16, act, *ins, gate, up, dy)
        check_ffn_bwd(torch, act, step, *ins, gate, up, dy, *grads)


# --- AdamW over a group ---------------------------------------------------------------------------

PARAMS = dict(lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, wd=0.05)


def params(hip, step, **over):
    q = PARAMS | over
    return hip.StepParams(q["lr"], q["beta1"], q["beta2"], q["eps"], q["wd"], 0, step)


def tensors(torch, sizes, bits, grads, copy, off=0, seed=1):
    rnd, out = gen(torch, seed), []
    g16 = torch.bfloat16 if grads == "bf16" else torch.float32
    for i, n in enumerate(sizes):
        t = {"p": put(torch, rnd(n), torch.float32, off), "g": put(torch, 0.1 * rnd(n), g16, off),
             "decay": float(i % 2)}
        if bits == 32:
            t["m"] = put(torch, torch.zeros(n, device="cuda"), torch.float32, off)
            t["v"] = put(torch, torch.zeros(n, device="cuda"), torch.float32, off)
        else:
            t["m"], t["v"] = (put(torch, torch.zeros(n, device="cuda"), torch.uint8, off)
                              for _ in range(2))
            t["m_scale"], t["v_scale"] = (torch.zeros((n + 127) // 128, device="cuda")
                                          for _ in range(2))
        if copy:
            t["p_bf16"] = put(torch, rnd(n), torch.bfloat16, off)
        out.append(t)
    return out


SIZES = [1, 5, 128, 0, 127, 129, 2048, 4100, 10000, 3]


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("grads", ["f32", "bf16"])
def test_group_with_32_bit_moments_leaves_the_single_step_bytes(hip, ctx, torch_cuda, grads, off):
    torch = torch_cuda
    ts = tensors(torch, SIZES, 32, grads, True, off)
    twins = [{k: v.clone().float() if k == "g" else v.clone() for k, v in t.items() if k != "decay"}
             for t in ts]
    group = hip.AdamWGroup(ctx, ts, 32, grads)
    for step in (1, 2, 7):
        group.step(params(hip, step))
        for t, w in zip(ts, twins):
            if w["p"].numel():
                q = params(hip, step, wd=np.float32(PARAMS["wd"]) * t["decay"])
                ctx.call("seeai_adamw_step", *(w[k].data_ptr() for k in ("p", "g", "m", "v")),
                         w["p"].numel(), q, 0.0)
    for t, w in zip(ts, twins):
        assert all(torch.equal(t[k], w[k]) for k in ("p", "m", "v"))
        assert torch.equal(t["p_bf16"], w["p"].to(torch.bfloat16))
    group.close()


def mix(h):
    h = ((h ^ (h >> 15)) * 0x6C8E9CF5) & 0xFFFFFFFF
    h = ((h ^ (h >> 13)) * 0x3A5D2B97) & 0xFFFFFFFF
    return h ^ (h >> 16)


def code_values():
    """What the 256 codes stand for."""
    c = np.arange(256)
    e, f = (c >> 3) & 15, c & 7
    v = np.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * 2.0 ** (e - 7.0))
    v[[0x7F, 0xFF]] = np.nan
    return np.where(c >> 7, -v, v)


def encode64(v, u, least, seen):
    """Codes and scales of float64 values from their definition: q = |v| / scale
    rounded up with the chance of its remainder.  Also how far q / grid + u is
    from the whole number where the choice turns.  `seen`: the kernel's scales,
    taken where f32 roundings decide -- the scale doubles where the block's
    largest magnitude passes 448 2^k, and that magnitude is within 4 u of the
    exact one, so where the exact one is within 8 u = 2^-21 of such a turn."""
    n = len(v)
    pad = np.zeros((n + 127) // 128 * 128)
    pad[:n] = np.where(np.isfinite(v), np.abs(v), 0)
    big = np.maximum(pad.reshape(-1, 128).max(1), 2.0 ** -126)
    turn = np.log2(big / 448)
    scale = 2.0 ** np.maximum(np.ceil(turn), -126.0)
    near = np.abs(2.0 ** (turn - np.round(turn)) - 1) < 2.0 ** -21
    scale = np.where(near & ((seen == 2 * scale) | (seen == scale / 2)), seen, scale)
    q = np.abs(v) / np.repeat(scale, 128)[:n]
    grid = 2.0 ** (np.floor(np.log2(np.maximum(q, 2.0 ** -6))) - 3)
    t = q / grid + u
    val = np.floor(t) * grid
    if least:
        val = np.where((q > 0) & (val == 0), 2.0 ** -9, val)
    return np.copysign(val, v), scale, np.abs(t - np.round(t))


@pytest.mark.parametrize("off", [0, 3])
@pytest.mark.parametrize("grads", ["f32", "bf16"])
def test_group_with_8_bit_moments(hip, ctx, torch_cuda, grads, off):
    """Codes, scales and weights against float64 from the state before the
    step.  A code may be its neighbour only where f32 roundings decide: m' and
    sqrt(v') are within 4 u of the exact ones and t = q / grid is at most 16,
    so where t + u' is within 16 * 4 u < 2^-17 of a whole number."""
    torch = torch_cuda
    table = code_values()
    ts = tensors(torch, SIZES, 8, grads, True, off, seed=4)
    ts[7]["g"][130:140] = 0
    ts[8]["g"][5000:5200] *= 1e-4
    group = hip.AdamWGroup(ctx, ts, 8, grads, seed=99)
    f = np.float32
    for step in (1, 2, 3, 40):
        before = [{k: v.double().cpu().numpy() if k in ("p", "g", "m_scale", "v_scale")
                   else v.cpu().numpy() for k, v in t.items() if k not in ("decay", "p_bf16")}
                  for t in ts]
        group.step(params(hip, step))
        number = 0
        b1, b2 = float(f(0.9)), float(f(0.999))
        for t, w in zip(ts, before):
            n = len(w["p"])
            i = np.arange(number, number + n, dtype=np.int64)
            number += (n + 127) // 128 * 128
            if n == 0:
                continue
            bits = mix((i & 0xFFFFFFFF) ^ mix(mix(mix(99) ^ step) ^ (i >> 32)))
            blk = np.arange(n) // 128
            m = b1 * table[w["m"]] * w["m_scale"][blk] + (1 - b1) * w["g"]
            v = b2 * (table[w["v"]] * w["v_scale"][blk]) ** 2 + (1 - b2) * w["g"] ** 2
            for name, val, u, least in (("m", m, (bits & 0xFFFF) / 65536.0, False),
                                        ("v", np.sqrt(v), (bits >> 16) / 65536.0, True)):
                seen = t[name + "_scale"].double().cpu().numpy()
                want, scale, edge = encode64(val, u, least, seen)
                got = table[t[name].cpu().numpy()]
                assert np.array_equal(seen, scale), name
                off_by = got != want
                assert (edge[off_by] < 2.0 ** -17).all(), (name, step, int(off_by.sum()))
                # (0.1 % of elements at most lie that near a turn)
                assert off_by.sum() <= max(2, 2e-3 * n)
                out = torch.empty(n, device="cuda")
                ctx.call("seeai_adamw_state_values", int(least), 0, t[name].data_ptr(),
                         t[name + "_scale"].data_ptr(), n, out.data_ptr())
                stands = (got * scale[blk]) ** (2 if least else 1)
                assert np.array_equal(out.double().cpu().numpy(), stands)
                half = torch.empty(n, dtype=torch.bfloat16, device="cuda")
                ctx.call("seeai_adamw_state_values", int(least), 1, t[name].data_ptr(),
                         t[name + "_scale"].data_ptr(), n, half.data_ptr())
                assert torch.equal(half.float(), out)
            c1, c2 = 1 - b1 ** step, 1 - b2 ** step
            move = float(f(1e-2)) * ((m / c1) / (np.sqrt(v / c2) + float(f(1e-8)))
                                     + float(f(0.05)) * t["decay"] * w["p"])
            p = w["p"] - move
            # 1 - beta^t in f32 loses up to u / (1 - beta^t) of itself.
            slack = (24 + 4 / c1 + 4 / c2) * U * np.abs(move) + 2 * U * np.abs(p)
            # (m may cancel: its error is of its terms' size)
            slack += 8 * U * float(f(1e-2)) * (np.abs(w["g"]) + np.abs(m)) / c1 / (np.sqrt(v / c2) + 1e-8)
            assert (np.abs(t["p"].double().cpu().numpy() - p) <= slack).all(), step
            assert torch.equal(t["p_bf16"], t["p"].to(torch.bfloat16))
    group.close()


def test_8_bit_moments_are_right_on_average(hip, ctx, torch_cuda):
    """One gradient step after step: beta2's average climbs by less than a code a
    step and must still reach the gradient's square.  Codes are at most d = 1/8 of
    their value apart; elements round independently.
    m: roundings of variance d^2 / 6 at most, decaying by 0.9 a step, leave a spread
    of d / sqrt(6 (1 - 0.81)) = 12 % an element, 0.2 % over the 4064: within 1 %.
    v: r = sqrt(v) is right on average, and v = r^2 gains r's variance.  A step that
    moves r by a fraction f of the gap d r adds f (1 - f) (d r)^2 <= move d r, an exact
    one 2 r move: a surplus of at most d / 2 = 1/16 of what v climbs.  An element's
    spread is under 40 %, 0.6 % over them: from -2 % to 1/16 + 2 %."""
    torch = torch_cuda
    n = 4096
    t = {"p": torch.zeros(n, device="cuda"), "g": torch.full((n,), 0.25, device="cuda"),
         "m": torch.zeros(n, dtype=torch.uint8, device="cuda"),
         "v": torch.zeros(n, dtype=torch.uint8, device="cuda"),
         "m_scale": torch.zeros(n // 128, device="cuda"),
         "v_scale": torch.zeros(n // 128, device="cuda")}
    t["g"][::128] = 0.3  # the scales are not the common value's own
    group = hip.AdamWGroup(ctx, [t], 8, "f32", seed=5)
    for step in range(1, 401):
        group.step(params(hip, step))
    out = torch.empty(n, device="cuda")
    for which, name, want, least, most in (
            (0, "m", 0.25 * (1 - 0.9 ** 400), -0.01, 0.01),
            (1, "v", 0.0625 * (1 - 0.999 ** 400), -0.02, 1 / 16 + 0.02)):
        ctx.call("seeai_adamw_state_values", which, 0, t[name].data_ptr(),
                 t[name + "_scale"].data_ptr(), n, out.data_ptr())
        rest = out.view(-1, 128)[:, 1:].double()
        assert least < float(rest.mean()) / want - 1 < most, name


def test_8_bit_moments_near_the_smallest_code(hip, ctx, torch_cuda):
    """From the smallest code on r = sqrt(v) is right on average and v high by its variance; below it
    every r > 0 is that code.  From zero moments one step leaves r = sqrt(1 - beta2) |g|; a block's
    largest, 300, is the scale's 300, so the others, in smallest codes of 2^-9, are q.  N = 8128
    elements a q, each off by up to half a code at a spread of one half: means within 5 / (2 sqrt(N))
    = 0.028 codes, v's within (2 q + 1) times that."""
    torch = torch_cuda
    blocks, qs = 64 * 5, (0.3, 0.9, 1.5, 3.3, 7.5)
    n = 128 * blocks
    root = math.sqrt(1.0 - float(np.float32(0.999)))
    q = torch.tensor(qs, device="cuda").repeat_interleave(64)
    r = (q / 512)[:, None].repeat(1, 128)
    r[:, 0] = 300.0
    t = {"p": torch.zeros(n, device="cuda"), "g": (r / root).flatten().contiguous(),
         "m": torch.zeros(n, dtype=torch.uint8, device="cuda"),
         "v": torch.zeros(n, dtype=torch.uint8, device="cuda"),
         "m_scale": torch.zeros(blocks, device="cuda"), "v_scale": torch.zeros(blocks, device="cuda")}
    hip.AdamWGroup(ctx, [t], 8, "f32", seed=6).step(params(hip, 1))
    assert (t["v_scale"] == 1).all()
    out = torch.empty(n, device="cuda")
    ctx.call("seeai_adamw_state_values", 1, 0, t["v"].data_ptr(), t["v_scale"].data_ptr(), n, out.data_ptr())
    v = out.view(5, 64, 128)[:, :, 1:].double() * 512 ** 2  # in smallest codes, squared
    for i, want in enumerate(qs):
        if want < 1:
            assert (v[i] == 1).all()
            continue
        f, slack = want - math.floor(want), 2.5 / math.sqrt(64 * 127)
        assert abs(float(v[i].sqrt().mean()) - want) < slack
        assert abs(float(v[i].mean()) - (want ** 2 + f * (1 - f))) < (2 * want + 1) * slack


def test_8_bit_moments_with_values_that_are_not_finite(hip, ctx, torch_cuda):
    torch = torch_cuda
    ts = tensors(torch, [300], 8, "f32", False)
    t = ts[0]
    t["g"][4], t["g"][200], t["g"][201] = float("nan"), float("inf"), -float("inf")
    p0 = t["p"].clone()
    group = hip.AdamWGroup(ctx, ts, 8, "f32")
    for step in (1, 2):
        group.step(params(hip, step))
    bad = [4, 200, 201]
    keep = [i for i in range(300) if i not in bad]
    assert (t["m"][bad] & 0x7F == 0x7F).all() and (t["v"][bad] & 0x7F == 0x7F).all()
    assert not (t["m"][keep] & 0x7F == 0x7F).any() and torch.isfinite(t["m_scale"]).all()
    assert torch.isfinite(t["p"][keep]).all() and not torch.equal(t["p"][keep], p0[keep])
    assert t["p"][bad].isnan().all()


def test_group_refusals_and_held_params(hip, ctx, torch_cuda):
    torch = torch_cuda
    ts = tensors(torch, [3000, 200], 8, "f32", True)
    group = hip.AdamWGroup(ctx, ts, 8, "f32", seed=1)
    with pytest.raises(hip.BackendError, match="none held"):
        group.step()
    with pytest.raises(hip.BackendError, match="from 1"):
        group.step(params(hip, 0))
    with pytest.raises(hip.BackendError, match="overlaps"):
        hip.AdamWGroup(ctx, [ts[0], ts[0]], 8, "f32")
    twins = [{k: v.clone() if torch.is_tensor(v) else v for k, v in t.items()} for t in ts]
    twin = hip.AdamWGroup(ctx, twins, 8, "f32", seed=1)
    for step in (1, 2, 3):
        group.hold(params(hip, step))
        group.step()
        twin.step(params(hip, step))
    for t, w in zip(ts, twins):
        assert all(torch.equal(v, w[k]) for k, v in t.items() if torch.is_tensor(v))


# --- together -------------------------------------------------------------------------------------

class Block:
    """x + ffn(norm(x)) with its own weights, trained by the operators alone."""

    def __init__(self, hip, ctx, torch, M, D, F, bf16, bits, seed=0):
        self.hip, self.ctx, self.torch, self.bf16 = hip, ctx, torch, bf16
        self.t, _ = types(torch, bf16)
        rnd = gen(torch, seed)
        self.M, self.D, self.F = M, D, F
        master = [1 + 0.1 * rnd(D), 0.1 * rnd(D), rnd(D, F) * D ** -0.5, rnd(D, F) * D ** -0.5,
                  rnd(F, D) * F ** -0.5]
        new = lambda *s: torch.empty(s, dtype=self.t, device="cuda")  # noqa: E731
        self.master = [m.contiguous() for m in master]
        self.w = [m.to(self.t) if i >= 2 and bf16 else m for i, m in enumerate(self.master)]
        self.grads = [torch.empty(D, device="cuda") for _ in range(2)] + [new(D, F), new(D, F), new(F, D)]
        self.x, self.dy = rnd(M, D).to(self.t), rnd(M, D).to(self.t)
        self.xn, self.y, self.dxn, self.dx = new(M, D), new(M, D), new(M, D), new(M, D)
        self.gate, self.up = new(M, F), new(M, F)
        self.mean, self.rstd = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
        lib = hip.lib()
        byte = lambda n: torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")  # noqa: E731
        self.ws_n = byte(lib.seeai_norm_bwd_workspace(M, D))
        self.ws_f = byte(max(lib.seeai_ffn_workspace(bf16, M, D, F, b) for b in (0, 1)))

        def state(i):
            n = self.master[i].numel()
            s = {"p": self.master[i], "g": self.grads[i], "decay": float(i >= 2)}
            if bits == 32:
                s["m"], s["v"] = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
            else:
                s["m"], s["v"] = (torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2))
                s["m_scale"], s["v_scale"] = (torch.zeros((n + 127) // 128, device="cuda")
                                              for _ in range(2))
            if i >= 2 and bf16:
                s["p_bf16"] = self.w[i]
            return s
        self.state = [state(i) for i in range(5)]
        self.groups = [hip.AdamWGroup(ctx, self.state[:2], bits, "f32", seed=3),
                       hip.AdamWGroup(ctx, self.state[2:], bits, "bf16" if bf16 else "f32", seed=4)]

    def gradients(self):
        p, c, b = self.hip.ptr, self.ctx, self.bf16
        M, D, F = self.M, self.D, self.F
        c.call("seeai_norm_fwd", 0, b, p(self.x), p(self.w[0]), p(self.w[1]), p(self.xn), p(self.mean),
               p(self.rstd), M, D, EPS)
        c.call("seeai_ffn_fwd", b, 3, p(self.xn), *map(p, self.w[2:]), p(self.gate), p(self.up),
               p(self.y), M, D, F, p(self.ws_f), self.ws_f.numel())
        c.call("seeai_ffn_bwd", b, 3, p(self.xn), *map(p, self.w[2:]), p(self.gate), p(self.up),
               p(self.dy), p(self.dxn), *map(p, self.grads[2:]), M, D, F, p(self.ws_f),
               self.ws_f.numel())
        c.call("seeai_norm_bwd", 0, b, p(self.dxn), p(self.x), p(self.w[0]), p(self.mean), p(self.rstd),
               p(self.dx), p(self.grads[0]), p(self.grads[1]), M, D, p(self.ws_n), self.ws_n.numel())

    def step(self, n, held=False):
        self.gradients()
        for g in self.groups:
            g.step(None if held else params(self.hip, n))

    def hold(self, n):
        for g in self.groups:
            g.hold(params(self.hip, n))

    def tensors(self):
        return ([self.y, self.dx, *self.master, *self.w]
                + [v for s in self.state for k, v in s.items() if k in ("m", "v", "m_scale", "v_scale")])


def test_block_gradients_against_differences(hip, ctx, torch_cuda):
    """The whole block's gradients, f32, against central differences of float64."""
    torch = torch_cuda
    b = Block(hip, ctx, torch, 9, 48, 80, 0, 32)
    b.gradients()
    ws = [w.double() for w in b.master]
    x, c = b.x.double(), b.dy.double()

    def loss(x, w):
        mu = x.mean(1, keepdim=True)
        xn = (x - mu) / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + EPS) * w[0] + w[1]
        g = xn @ w[2]
        return float((((g * torch.sigmoid(g)) * (xn @ w[3])) @ w[4] * c).sum())
    h = 2.0 ** -13
    for i, grad in enumerate([*b.grads, b.dx]):
        d = gen(torch, 40 + i)(*grad.shape).double()
        d /= d.norm()
        at = []
        for s in (h, -h):
            w = list(ws)
            if i < 5:
                w[i] = ws[i] + s * d
            at.append(loss(x + s * d if i == 5 else x, w))
        want = float((grad.double() * d).sum())
        assert abs((at[0] - at[1]) / (2 * h) - want) <= 2e-5 * float(grad.double().norm()), i


@pytest.mark.parametrize("bf16,bits,M", [(1, 8, 200), (1, 32, 3), (0, 8, 65)])
def test_block_steps_captured_and_replayed(hip, torch_cuda, bf16, bits, M):
    """A training step captured once (held params) and replayed, eager work in
    between, against the same steps run eagerly; two graphs with workspaces of
    their own on two streams at once."""
    torch = torch_cuda
    stream = torch.cuda.Stream()
    c1, c2, ce = hip.Context(0), hip.Context(0), hip.Context(0)
    with torch.cuda.stream(stream):
        c1.use_torch_stream()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        c2.use_torch_stream()
    ce.use_torch_stream()
    blocks = [Block(hip, c, torch, M, 136, 264, bf16, bits) for c in (c1, c2)]
    eager = Block(hip, ce, torch, M, 136, 264, bf16, bits)
    torch.cuda.synchronize()
    graphs = []
    for b, s in zip(blocks, (stream, other)):
        b.hold(1)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            b.step(1, held=True)
            with pytest.raises(hip.BackendError, match="held params"):
                b.groups[0].step(params(hip, 1))
            with pytest.raises(hip.BackendError, match="captured"):
                b.groups[0].hold(params(hip, 1))
        graphs.append(g)
    for n in range(1, 6):
        for b in blocks:
            b.hold(n)
        torch.cuda.synchronize()
        for g, s in zip(graphs, (stream, other)):
            with torch.cuda.stream(s):
                g.replay()
        eager.step(n)
        junk = torch.randn(512, 512, device="cuda") @ torch.randn(512, 512, device="cuda")
        torch.cuda.synchronize()
        for b in blocks:
            for got, want in zip(b.tensors(), eager.tensors()):
                assert torch.equal(got, want), n
    assert torch.isfinite(junk).all()


def test_entry_points_refuse_on_the_context(hip, ctx, torch_cuda):
    torch = torch_cuda
    x = torch.zeros(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    with pytest.raises(hip.BackendError, match="norm_fwd: an output overlaps"):
        call_norm_fwd(ctx, 0, 0, x, w, w, x, None, None)
    with pytest.raises(hip.BackendError, match="ffn_fwd: workspace too small"):
        ctx.call("seeai_ffn_fwd", 0, 3, *[w.data_ptr()] * 4, None, None, x.data_ptr(), 1, 8, 1, None, 0)
    assert hip.lib().seeai_norm_fwd(None, 0, 0, None, None, None, None, None, None, 1, 1, EPS) == 2
