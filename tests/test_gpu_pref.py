"""GPU: learning from preferences -- seeai_token_logp_fwd / _bwd, seeai_pref_loss,
seeai_policy_loss -- and the clip of a step's gradients -- seeai_grad_group_*,
seeai_adamw_group_step_scaled -- against plain float64.

Tolerances are bounds on what the kernels' own roundings may add up to: u = 2^-24
for each f32 operation, 2^-8 of the value for a rounding to bf16 (half a step).
An exponential exp(x) as 2^(x log2 e) is within (3 |x| + 2) u of itself: x, log2 e
and their product each rounded, the hardware's exp2 good to one unit in the last
place, 2 u.  A sum of n terms one after another is within n u of them."""
from __future__ import annotations

import math

import numpy as np
import pytest

from tests.test_gpu_block import U, Guarded, ctx, gen, put, types, within  # noqa: F401

pytestmark = pytest.mark.gpu

TINY = 2.0 ** -120  # what exp2 may flush to zero


def token_inputs(torch, N, V, ld, bf16, seed, skip=0.3, off=0, spread=3.0):
    """Logits in a buffer of rows ld apart with NaNs between them, and labels."""
    rnd = gen(torch, seed)
    t, _ = types(torch, bf16)
    buf = Guarded(torch, (N, ld), t, off)
    buf.t.fill_(float("nan"))
    z = spread * rnd(N, V) + 4.0 * rnd(N, 1)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    labels = torch.randint(0, V, (N,), device="cuda", generator=g)
    z[torch.arange(N), labels] += 4.0
    labels[torch.rand(N, device="cuda", generator=g) < skip] = -1
    buf.t[:, :V] = z.to(t)
    buf.t[labels < 0] = float("nan")  # rows that are not judged are not read
    return buf, labels.to(torch.int32)


def softmax64(torch, z, labels):
    """Each judged row's label's log-probability and its bound, the probabilities
    and theirs."""
    z = z.double()
    V = z.shape[1]
    m = z.amax(1, keepdim=True)
    d = z - m
    s = torch.exp(d).sum(1, keepdim=True)
    p = torch.exp(d) / s
    far = d.abs().clamp(max=1e3)  # (from there on p is zero)
    # The terms' own errors, twice for the rescaling of what came before a new
    # maximum; the longest run of additions is a 64th of the row and the joins.
    e_s = U * (V / 64 + 80 + 8 * (p * far).sum(1, keepdim=True))
    picked = d.gather(1, labels.clamp(min=0).long()[:, None])
    logp = picked - torch.log(s)
    e = U * picked.abs() + e_s + 3 * U * torch.log(s).abs() + U * logp.abs()
    e_p = p * (e_s + U * (3 * far + 8)) + TINY
    return logp[:, 0], e[:, 0], p, e_p


def token_logp(ctx, torch, z, ld, labels, V, stats=True):
    N = labels.numel()
    logp, st = Guarded(torch, (N,), torch.float32), Guarded(torch, (N, 2), torch.float32)
    ctx.call("seeai_token_logp_fwd", int(z.dtype == torch.bfloat16), z.data_ptr(), ld, labels.data_ptr(),
             logp.t.data_ptr(), st.t.data_ptr() if stats else None, N, V)
    assert logp.intact() and st.intact()
    return logp.t, st.t


def token_logp_bwd(ctx, torch, z, ld, labels, stats, dlogp, V, out):
    ctx.call("seeai_token_logp_bwd", int(z.dtype == torch.bfloat16), z.data_ptr(), ld, labels.data_ptr(),
             stats.data_ptr(), dlogp.data_ptr(), out.data_ptr(), labels.numel(), V)


def check_logits_grad(torch, got, z, labels, d, e_d, p, e_p, step):
    """dz = d (1[c = l] - p), from d within e_d and p within e_p."""
    hot = torch.zeros_like(p)
    hot.scatter_(1, labels.clamp(min=0).long()[:, None], 1.0)
    d, e_d = d.double()[:, None], e_d[:, None]
    want = d * (hot - p)
    bound = e_d * (hot - p).abs() + (d.abs() + e_d) * (e_p + 4 * U * p + U * hot)
    live = (labels >= 0)[:, None]
    want, bound = torch.where(live, want, 0.0), torch.where(live, bound, 0.0)
    within(torch, got, want, bound + step * (want.abs() + bound) + TINY)
    assert not got[labels < 0].any()


# Rows of a wave, of four waves and of sixteen; odd widths and paddings.
LOGITS = [(1, 1, 1), (3, 2, 5), (1, 64, 64), (7, 511, 511), (70, 513, 520), (5, 2047, 2050), (9, 2048, 2048),
          (4, 2049, 2049), (33, 4001, 4003), (2, 8192, 8192), (3, 8193, 8200), (2100, 2112, 2112),
          (2, 32000, 32000), (2049, 2051, 2051), (3, 32769, 32770), (2, 65537, 65540), (1, 128000, 128000),
          (2, 131073, 131080), (600, 9001, 9001), (520, 17000, 17000), (513, 29999, 30002), (1, 40000, 40000)]


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("bf16", [0, 1])
def test_token_logp(ctx, torch_cuda, bf16, off):
    torch = torch_cuda
    t, step = types(torch, bf16)
    for N, V, ld in LOGITS:
        print(f"token_logp bf16={bf16} off={off} {N}x{V} ld {ld}", flush=True)
        buf, labels = token_inputs(torch, N, V, ld, bf16, N * 7 + V, off=off)
        z = buf.t[:, :V]
        logp, stats = token_logp(ctx, torch, buf.t, ld, labels, V)
        want, e, p, e_p = softmax64(torch, z, labels)
        live = labels >= 0
        within(torch, logp[live], want[live], e[live])
        assert not logp[~live].any() and not stats[~live].any()
        assert torch.equal(stats[live, 0], z[live].float().amax(1))
        again, _ = token_logp(ctx, torch, buf.t, ld, labels, V, stats=False)
        assert torch.equal(again, logp)
        dlogp = gen(torch, 5)(N)
        out = Guarded(torch, (N, ld), t, off)
        token_logp_bwd(ctx, torch, buf.t, ld, labels, stats, dlogp, V, out.t)
        check_logits_grad(torch, out.t[:, :V], z, labels, dlogp, torch.zeros_like(dlogp, dtype=torch.float64),
                          p, e_p, step)
        assert out.intact() and (out.t[:, V:] == 7).all()  # between the rows: left alone
        keep = out.t[:, :V].clone()
        token_logp_bwd(ctx, torch, buf.t, ld, labels, stats, dlogp, V, buf.t)  # in place
        assert torch.equal(buf.t[:, :V], keep) and buf.t[:, V:].isnan().all()


@pytest.mark.parametrize("bf16", [0, 1])
def test_gradients_where_the_logits_lie_otherwise(hip, ctx, torch_cuda, bf16):
    """A gradient buffer whose rows begin elsewhere within 16 bytes than the logits', and
    gradients too large for the last cache."""
    torch = torch_cuda
    t, step = types(torch, bf16)
    cases = [(5, 1000, 1000), (3, 9001, 9003), (4, 70000, 70000), (2, 7, 9), (9, 33, 33)]
    for N, V, ld in cases + ([(4400, 16001, 16001)] if bf16 else [(2200, 16000, 16000)]):
        buf, labels, old, ref, adv, weight = policy_inputs(torch, N, V, ld, bf16, V)
        same, other = Guarded(torch, (N, ld), t), Guarded(torch, (N, ld), t, 3)
        _, stats = token_logp(ctx, torch, buf.t, ld, labels, V)
        dlogp = gen(torch, 5)(N)
        for out in (same, other):
            token_logp_bwd(ctx, torch, buf.t, ld, labels, stats, dlogp, V, out.t)
            assert out.intact() and (out.t[:, V:] == 7).all()
        assert torch.equal(same.t, other.t)
        if N > 1000:
            rows = list(range(0, N, N // 20))
            _, _, p, e_p = softmax64(torch, buf.t[rows, :V], labels[rows])
            check_logits_grad(torch, same.t[rows, :V], buf.t[rows, :V], labels[rows], dlogp[rows],
                              torch.zeros(len(rows), dtype=torch.float64, device="cuda"), p, e_p, step)
        for out in (same, other):
            policy_loss(hip, ctx, torch, buf.t, ld, labels, old, ref, adv, weight, V, 0.1, 1.0, out.t)
            assert out.intact() and (out.t[:, V:] == 7).all()
        assert torch.equal(same.t, other.t)


def test_token_logp_of_masked_and_odd_logits(ctx, torch_cuda):
    """Tokens ruled out by -inf or the type's lowest value, whole rows of either,
    infinities, NaNs, labels past the vocabulary: as log_softmax has them, each in
    its own row."""
    torch = torch_cuda
    for bf16 in (0, 1):
        t, step = types(torch, bf16)
        for V in (40, 3000, 33001):
            N, inf, low = 14, float("inf"), torch.finfo(t).min
            z = gen(torch, V)(N, V)
            labels = torch.full((N,), 7, dtype=torch.int32, device="cuda")
            z[1, ::2] = -inf  # the label is left
            z[2, ::2] = low
            z[3, 7] = -inf  # the label is ruled out
            z[4] = -inf
            z[5] = low
            z[6, 9] = inf
            z[7, 9] = float("nan")
            z[8] = float("nan")
            labels[9], labels[10], labels[11] = V, 2 ** 31 - 1, -2 ** 31
            z[12, :-1], labels[12] = -inf, V - 1  # one token is left
            z[13] = 3e4
            z = z.to(t).contiguous()
            logp, stats = token_logp(ctx, torch, z, V, labels, V)
            want = torch.log_softmax(z.double(), 1)
            at = labels.clamp(0, V - 1).long()[:, None]
            want = want.gather(1, at)[:, 0]
            want[[9, 10]], want[11] = float("nan"), 0.0
            assert torch.equal(logp.isnan(), want.isnan()), (logp, want)
            assert logp[3] == -inf and logp[12] == 0 and logp[11] == 0
            fine = [0, 1, 2, 5, 13]
            _, e, p, e_p = softmax64(torch, z[fine], labels[fine])
            within(torch, logp[fine], want[fine], e)
            dlogp = torch.full((N,), 0.5, device="cuda")
            out = Guarded(torch, (N, V), t)
            token_logp_bwd(ctx, torch, z, V, labels, stats, dlogp, V, out.t)
            check_logits_grad(torch, out.t[fine], z[fine], labels[fine], dlogp[fine],
                              torch.zeros(len(fine), dtype=torch.float64, device="cuda"), p, e_p, step)
            assert not out.t[11].any() and not out.t[1, ::2].any() and out.t[[9, 10]].isnan().all()
            assert torch.isfinite(out.t[[0, 1, 2, 3, 5, 11, 12, 13]]).all() and out.intact()
            assert out.t[12, -1] == 0  # a sure token has no gradient


@pytest.mark.parametrize("bf16", [0, 1])
def test_token_logp_of_a_nearly_sure_token(ctx, torch_cuda, bf16):
    """The sum is 1 and a little: its small logarithm keeps its own digits.  The group that holds
    the 1 rounds three times, the other terms and their rescalings (to a thread's, a wave's and a
    row's maximum) by (3 |d| + 2) u each, all else is f64."""
    torch = torch_cuda
    t, _ = types(torch, bf16)
    for N, V in ((64, 40), (64, 4000), (700, 32000), (3, 131000), (64, 32001)):
        z = (gen(torch, V)(N, V) - math.log(V) - 4.0).to(t)
        labels = torch.randint(0, V, (N,), device="cuda").to(torch.int32)
        z[torch.arange(N), labels.long()] = 1.0
        logp, _ = token_logp(ctx, torch, z, V, labels, V)
        d = z.double() - 1.0
        p = torch.exp(d).scatter(1, labels.long()[:, None], 0.0)
        want = -torch.log1p(p.sum(1))
        bound = U * (3.5 + (p * (12 * d.abs() + 10)).sum(1) + 6 * want.abs())
        assert float(bound.max()) < 0.05 * float(want.abs().min())
        within(torch, logp, want, bound)


def test_token_logp_past_32_bit_offsets(ctx, torch_cuda):
    """Over 2^32 bytes and 2^31 elements: the last rows are the formula's."""
    torch = torch_cuda
    N, V, ld = 70000, 32000, 32064
    z = torch.empty(N, ld, dtype=torch.bfloat16, device="cuda")
    z.normal_()
    labels = torch.full((N,), -1, dtype=torch.int32, device="cuda")
    rows = [0, 1, N // 2, 66977, 66978, N - 1]
    labels[rows] = torch.tensor([5, V - 1, 77, 0, 31999, 12345], dtype=torch.int32, device="cuda")
    logp, stats = token_logp(ctx, torch, z, ld, labels, V)
    want, e, p, e_p = softmax64(torch, z[rows][:, :V], labels[rows])
    within(torch, logp[rows], want, e)
    dlogp = torch.ones(N, device="cuda")
    keep = z[rows].clone()
    token_logp_bwd(ctx, torch, z, ld, labels, stats, dlogp, V, z)
    check_logits_grad(torch, z[rows][:, :V], keep, labels[rows], dlogp[rows],
                      torch.zeros(len(rows), dtype=torch.float64, device="cuda"), p, e_p, 2.0 ** -8)
    assert torch.equal(z[rows][:, V:], keep[:, V:])
    others = torch.arange(0, N, 997, device="cuda")
    assert not z[others[labels[others] < 0], :V].any()


def test_no_tokens(hip, ctx, torch_cuda):
    torch = torch_cuda
    ctx.call("seeai_token_logp_fwd", 0, None, 9, None, None, None, 0, 9)
    ctx.call("seeai_token_logp_bwd", 0, None, 9, None, None, None, None, 0, 9)
    loss = torch.full((1,), 5.0, device="cuda")
    ctx.call("seeai_policy_loss", 0, None, 9, None, None, None, None, None, 0, 9, 0.2, 0.2, 0.1, 1.0,
             loss.data_ptr(), None, None, None, 0)
    assert float(loss) == 0
    loss.fill_(5.0)
    d = torch.full((6,), 3.0, device="cuda")
    ctx.call("seeai_pref_loss", None, None, None, None, 6, 0, 0.1, 0.0, 0.0, 0, 1.0, loss.data_ptr(), None,
             d.data_ptr(), None, 0)
    assert float(loss) == 0 and not d.any()


# --- the paired loss ------------------------------------------------------------------------------

def pref_loss(hip, ctx, torch, logp, ref, labels, starts, beta, offset, eps, average, scale, grad=True):
    N, pairs = logp.numel(), (starts.numel() - 1) // 2
    loss, margin = Guarded(torch, (1,), torch.float32), Guarded(torch, (pairs,), torch.float32)
    d = Guarded(torch, (N,), torch.float32)
    n = hip.lib().seeai_pref_workspace(pairs)
    ws = Guarded(torch, (n,), torch.uint8)
    p = hip.ptr
    ctx.call("seeai_pref_loss", p(logp), p(ref), p(labels), p(starts), N, pairs, beta, offset, eps, average,
             scale, p(loss.t), p(margin.t) if grad else None, p(d.t) if grad else None, p(ws.t), n)
    assert loss.intact() and margin.intact() and d.intact() and ws.intact()
    return loss.t, margin.t, d.t


def pref64(torch, logp, ref, labels, starts, beta, offset, eps, average, scale):
    f = lambda v: float(np.float32(v))  # noqa: E731
    beta, offset, eps, scale = f(beta), f(offset), f(eps), f(scale)
    lp = logp.double().cpu().requires_grad_()
    diff = lp - (ref.double().cpu() if ref is not None else 0.0)
    live = (labels >= 0).cpu()
    s = starts.tolist()
    sums = []
    for a, b in zip(s, s[1:]):
        picked = diff[a:b][live[a:b]]
        sums.append(picked.sum() / (max(picked.numel(), 1) if average else 1))
    sums = torch.stack(sums) if sums else torch.zeros(0, dtype=torch.float64)
    margin = beta * (sums[0::2] - sums[1::2]) - offset
    ls = torch.nn.functional.logsigmoid
    loss = scale * (-(1 - eps) * ls(margin) - eps * ls(-margin)).sum()
    d, = torch.autograd.grad(loss, lp)
    return loss.detach().cuda(), margin.detach().cuda(), d.cuda(), float(diff.detach().abs().sum())


# Sequences' lengths: pairs of one token, none, long ones; rows before and behind.
PAIRS = [([1, 1], 0, 0), ([5, 0], 2, 3), ([0, 0], 1, 0), ([64, 65, 511, 513], 0, 7),
         ([1000, 3000, 1, 2, 0, 9], 11, 70), ([7] * 130, 0, 0), ([40000, 20000], 5, 1), ([3] * 600, 2, 1),
         ([511] * 4, 1, 3), ([600, 500, 400, 300, 200, 40], 0, 8), ([90] * 22, 0, 9)]


@pytest.mark.parametrize("average", [0, 1])
@pytest.mark.parametrize("with_ref", [True, False])
def test_pref_loss(hip, ctx, torch_cuda, with_ref, average):
    torch = torch_cuda
    for lengths, before, behind in PAIRS:
        print(f"pref {lengths[:6]} ref={with_ref} average={average}", flush=True)
        rnd = gen(torch, sum(lengths) + before)
        N = sum(lengths) + before + behind
        starts = torch.tensor(np.cumsum([before, *lengths]), dtype=torch.int32, device="cuda")
        logp, ref = -rnd(N).abs() - 0.01, -rnd(N).abs() if with_ref else None
        labels = torch.where(rnd(N) < 0.5, 3, -1).to(torch.int32)
        for beta, offset, eps, scale in ((0.1, 0.0, 0.0, 1.0), (2.5, 0.5, 0.1, 0.25), (-0.3, -1.0, 1.0, -2.0)):
            got = pref_loss(hip, ctx, torch, logp, ref, labels, starts, beta, offset, eps, average, scale)
            loss, margin, d, size = pref64(torch, logp, ref, labels, starts, beta, offset, eps, average, scale)
            # f64 throughout, each result rounded once.
            slack = 1e-13 * (1 + abs(beta)) * (1 + size)
            within(torch, got[0], loss.view(1), U * loss.abs() + slack)
            within(torch, got[1], margin, U * margin.abs() + slack)
            within(torch, got[2], d, U * d.abs() + abs(scale) * slack)
            outside = torch.ones(N, dtype=torch.bool, device="cuda")
            outside[before:before + sum(lengths)] = False
            assert not got[2][outside | (labels < 0)].any()
        alone = pref_loss(hip, ctx, torch, logp, ref, labels, starts, -0.3, -1.0, 1.0, average, -2.0, grad=False)
        assert torch.equal(alone[0], got[0])


def test_pref_loss_against_differences(hip, ctx, torch_cuda):
    torch = torch_cuda
    starts = torch.tensor([0, 5, 9, 12, 20], dtype=torch.int32, device="cuda")
    logp, ref = -gen(torch, 1)(20).abs(), -gen(torch, 2)(20).abs()
    labels = torch.arange(20, device="cuda", dtype=torch.int32) - 1
    args = (0.7, 0.2, 0.05, 1, 0.5)
    _, _, d = pref_loss(hip, ctx, torch, logp, ref, labels, starts, *args)
    way = gen(torch, 3)(20)
    h = 2.0 ** -10
    at = [float(pref64(torch, logp.double() + s * way.double(), ref, labels, starts, *args)[0]) for s in (h, -h)]
    assert abs((at[0] - at[1]) / (2 * h) - float((d.double() * way.double()).sum())) < 1e-6


def test_pref_loss_of_far_margins_and_bad_starts(hip, ctx, torch_cuda):
    torch = torch_cuda
    inf = float("inf")
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    labels = torch.zeros(2, dtype=torch.int32, device="cuda")
    for chosen, rejected, loss, d in ((1e6, 0.0, 0.0, 0.0), (-1e6, 0.0, 1e6, -1.0), (0.0, -inf, 0.0, 0.0),
                                      (-inf, 0.0, inf, -1.0)):
        lp = torch.tensor([chosen, rejected], device="cuda")
        got = pref_loss(hip, ctx, torch, lp, None, labels, starts, 1.0, 0.0, 0.0, 0, 1.0)
        assert float(got[0]) == loss and got[2].tolist() == [d, -d]
    lp = torch.tensor([float("nan"), 0.0], device="cuda")
    got = pref_loss(hip, ctx, torch, lp, None, labels, starts, 1.0, 0.0, 0.1, 0, 1.0)
    assert all(v.isnan().all() for v in got)
    # Starts outside the rows, or falling, are kept within them.
    lp = torch.zeros(6, device="cuda")
    labels = torch.zeros(6, dtype=torch.int32, device="cuda")
    for bad in ([-7, 3, 900], [6, 2, 4], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1]):
        s = torch.tensor(bad, dtype=torch.int32, device="cuda")
        got = pref_loss(hip, ctx, torch, lp, None, labels, s, 1.0, 0.0, 0.0, 0, 1.0)
        assert abs(float(got[0]) - math.log(2)) < 1e-6


# --- the policy loss ------------------------------------------------------------------------------

LOW, HIGH = 0.2, 0.28


def policy_inputs(torch, N, V, ld, bf16, seed, off=0):
    buf, labels = token_inputs(torch, N, V, ld, bf16, seed, off=off)
    rnd = gen(torch, seed + 9)
    now = softmax64(torch, buf.t[:, :V], labels)[0]
    moved = 0.3 * rnd(N).double()
    for bound in (math.log(1 - LOW), math.log(1 + HIGH)):  # no ratio near a bound
        moved = torch.where((moved - bound).abs() < 1e-2, bound + 2e-2, moved)
    old = torch.where(labels >= 0, now - moved, float("nan")).float()
    ref = torch.where(labels >= 0, now + 0.3 * rnd(N).double(), float("nan")).float()
    adv = torch.where(labels >= 0, rnd(N), float("nan"))
    weight = torch.where(labels >= 0, rnd(N).abs() + 0.1, float("nan"))
    return buf, labels, old, ref, adv, weight


def policy_loss(hip, ctx, torch, z, ld, labels, old, ref, adv, weight, V, kl, scale, out=None, logp=True):
    N = labels.numel()
    loss, lp = Guarded(torch, (1,), torch.float32), Guarded(torch, (N,), torch.float32)
    n = hip.lib().seeai_policy_workspace(N, V)
    ws, p = Guarded(torch, (n,), torch.uint8), hip.ptr
    ctx.call("seeai_policy_loss", int(z.dtype == torch.bfloat16), p(z), ld, p(labels), p(old), p(ref), p(adv),
             p(weight), N, V, LOW, HIGH, kl, scale, p(loss.t), p(lp.t) if logp else None, p(out), p(ws.t), n)
    assert loss.intact() and lp.intact() and ws.intact()
    return loss.t, lp.t


def policy64(torch, logp, e_logp, labels, old, ref, adv, weight, kl, scale):
    """The loss, each token's derivative, and their bounds, from log-probabilities
    within e_logp."""
    f = lambda v: float(np.float32(v))  # noqa: E731
    low, high = float(np.float32(1) - np.float32(LOW)), float(np.float32(1) + np.float32(HIGH))
    live = labels >= 0
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    x = lambda v: torch.where(live, v.double(), zero)  # noqa: E731
    lp, A, w = x(logp), x(adv), (x(weight) if weight is not None else live.double()) * f(scale)
    moved = lp - x(old)
    r = moved.exp()
    e_r = r * (e_logp + U * (moved.abs() + 6))
    free, cut = r * A, r.clamp(low, high) * A
    took = cut < free
    val = torch.where(took, -cut, -free)
    d = torch.where(took, zero, -free)
    e_v = A.abs() * (e_r + 3 * U * r)
    e_d = torch.where(took, zero, e_v)
    if ref is not None:
        back = x(ref) - lp
        e = back.exp()
        e_e = e * (e_logp + U * (back.abs() + 6))
        val, d = val + f(kl) * (e - back - 1), d + f(kl) * (1 - e)
        e_v = e_v + f(kl) * (e_e + e_logp + 4 * U * (e + back.abs() + 1)) + 2 * U * val.abs()
        e_d = e_d + f(kl) * (e_e + 4 * U * (1 + e)) + 2 * U * d.abs()
    loss, e_loss = (w * val).sum(), (w.abs() * (e_v + 3 * U * val.abs())).sum()
    return loss, e_loss + 2 * U * loss.abs(), w * d, w.abs() * (e_d + 3 * U * d.abs())


@pytest.mark.parametrize("kl", [0.0, 0.3])
@pytest.mark.parametrize("bf16,off", [(0, 0), (0, 1), (1, 0), (1, 1)])
def test_policy_loss(hip, ctx, torch_cuda, bf16, off, kl):
    torch = torch_cuda
    t, step = types(torch, bf16)
    for N, V, ld in LOGITS:
        print(f"policy bf16={bf16} off={off} kl={kl} {N}x{V} ld {ld}", flush=True)
        buf, labels, old, ref, adv, weight = policy_inputs(torch, N, V, ld, bf16, N * 7 + V, off)
        if kl == 0.0:
            ref, weight = None, None
        z = buf.t[:, :V]
        out = Guarded(torch, (N, ld), t, off)
        loss, logp = policy_loss(hip, ctx, torch, buf.t, ld, labels, old, ref, adv, weight, V, kl, 0.7, out.t)
        want, e, p, e_p = softmax64(torch, z, labels)
        live = labels >= 0
        within(torch, logp[live], want[live], e[live])
        assert not logp[~live].any()
        # (the log-probabilities that the call gave are the ones it went on with)
        L, e_L, d, e_d = policy64(torch, logp, torch.zeros_like(e), labels, old, ref, adv, weight, kl, 0.7)
        within(torch, loss, L.view(1), e_L.view(1))
        check_logits_grad(torch, out.t[:, :V], z, labels, d, e_d, p, e_p, step)
        assert out.intact() and (out.t[:, V:] == 7).all()
        alone, _ = policy_loss(hip, ctx, torch, buf.t, ld, labels, old, ref, adv, weight, V, kl, 0.7, None, False)
        assert torch.equal(alone, loss)
        again, lp2 = policy_loss(hip, ctx, torch, buf.t, ld, labels, old, ref, adv, weight, V, kl, 0.7, buf.t)
        assert torch.equal(again, loss) and torch.equal(lp2, logp)
        assert torch.equal(buf.t[:, :V], out.t[:, :V]) and buf.t[:, V:].isnan().all()


def test_policy_loss_against_differences(hip, ctx, torch_cuda):
    """The whole gradient against central differences of the float64 loss."""
    torch = torch_cuda
    N, V = 12, 50
    buf, labels, old, ref, adv, weight = policy_inputs(torch, N, V, V, 0, 3)
    z = torch.where((labels >= 0)[:, None], buf.t, 0.0).double()
    out = torch.empty_like(buf.t)
    policy_loss(hip, ctx, torch, buf.t, V, labels, old, ref, adv, weight, V, 0.3, 1.0, out)
    way, h = gen(torch, 4)(N, V).double(), 2.0 ** -12
    at = []
    for s in (h, -h):
        lp = softmax64(torch, z + s * way, labels)[0]
        at.append(float(policy64(torch, lp, torch.zeros_like(lp), labels, old, ref, adv, weight, 0.3, 1.0)[0]))
    assert abs((at[0] - at[1]) / (2 * h) - float((out.double() * way).sum())) < 2e-5


def test_policy_sides_of_the_clip(hip, ctx, torch_cuda):
    """Ratios inside, past and on the bounds, for advantages of either sign: where
    the unclipped term is the smaller or equal its gradient stays.  Two equal logits
    give log 1/2 to the bit, so a ratio of 1 is exact."""
    torch = torch_cuda
    half = float(np.float32(-math.log(2.0)))
    z = torch.zeros(8, 2, device="cuda")
    labels = torch.zeros(8, dtype=torch.int32, device="cuda")
    moved = torch.tensor([0.0, 0.0, 1.0, 1.0, -1.0, -1.0, 0.1, -0.1], device="cuda")
    old = half - moved
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0, 1.0, -1.0, 2.0, 2.0], device="cuda")
    out = torch.empty_like(z)
    loss, logp = policy_loss(hip, ctx, torch, z, 2, labels, old, None, adv, None, 2, 0.0, 1.0, out)
    assert ((logp - half).abs() <= 2 * U).all()
    r = torch.exp((logp - old).double())
    live = torch.tensor([1, 1, 0, 1, 1, 0, 1, 1], device="cuda")  # past the bound on the worse side: no gradient
    want = -(r * adv * live)[:, None] * torch.tensor([0.5, -0.5], device="cuda")
    within(torch, out, want, 16 * U * want.abs())
    held = torch.where(live == 1, r, r.clamp(1 - LOW, 1 + HIGH))
    assert abs(float(loss) + float((held * adv).sum())) < 32 * U * float((held * adv).abs().sum())


def test_policy_near_the_reference(hip, ctx, torch_cuda):
    """A KL term is about half the square of a small difference of log-probabilities:
    it keeps its digits.  The difference is rounded once (twice that in its square),
    the square twice, the series' end once and its steps by a twelfth of theirs, off
    by 2^-26 = U / 4, the sum once: within 8 U of the loss; the derivative, the
    difference and a part of at most a seventh of that, within 4 U."""
    torch = torch_cuda
    N, V = 64, 40
    buf, labels = token_inputs(torch, N, V, V, 0, 77)
    live, zeros = labels >= 0, torch.zeros(N, device="cuda")
    call = lambda old, ref, out: policy_loss(hip, ctx, torch, buf.t, V, labels, old, ref, zeros, None,  # noqa: E731
                                             V, 1.0, 1.0, out)
    lp = call(zeros, zeros, None)[1]
    _, _, p, e_p = softmax64(torch, buf.t, labels)
    for far in (1e-5, 1e-3, 0.1, 0.2499):
        print(f"policy near the reference {far}", flush=True)
        ref, out = lp + far * torch.linspace(-1, 1, N, device="cuda"), torch.empty_like(buf.t)
        loss, again = call(lp, ref, out)
        assert torch.equal(again, lp)
        back = torch.where(live, ref.double() - lp.double(), 0.0)
        L, d = (torch.expm1(back) - back).sum().view(1), -torch.expm1(back)
        within(torch, loss, L, 8 * U * L)
        check_logits_grad(torch, out, buf.t, labels, d, 4 * U * d.abs(), p, e_p, U)


def test_policy_with_odd_values(hip, ctx, torch_cuda):
    """A NaN or an infinity stays in its row, though not out of the loss."""
    torch = torch_cuda
    for V in (30, 5000):
        z = gen(torch, V)(9, V)
        labels = torch.full((9,), 4, dtype=torch.int32, device="cuda")
        lp, _ = token_logp(ctx, torch, z, V, labels, V)
        old, ref, adv = lp.clone(), lp.clone(), torch.ones(9, device="cuda")
        z[1, 2], old[2], adv[3], labels[4], ref[5] = float("nan"), float("nan"), float("inf"), V, float("nan")
        z[6, 1::2], z[6, 4] = -float("inf"), 1.0
        labels[7] = -5
        out = torch.empty_like(z)
        loss, got = policy_loss(hip, ctx, torch, z, V, labels, old, ref, adv, None, V, 0.1, 1.0, out)
        assert loss.isnan().all() and got[[1, 4]].isnan().all() and torch.isfinite(got[[0, 2, 3, 5, 6, 7, 8]]).all()
        assert out[[1, 2, 4, 5]].isnan().all() and not torch.isfinite(out[3]).any()
        assert torch.isfinite(out[[0, 6, 7, 8]]).all() and not out[7].any()


# --- the clip -------------------------------------------------------------------------------------

def grad_tensors(torch, sizes, kinds, seed=0, off=0):
    rnd = gen(torch, seed)
    return [put(torch, rnd(n) * (10.0 ** (i % 5 - 3)), torch.bfloat16 if k else torch.float32, off)
            for i, (n, k) in enumerate(zip(sizes, kinds))]


def norm64(torch, tensors):
    return math.sqrt(sum(float(t.double().square().sum()) for t in tensors))


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("sizes", [[1], [0, 7, 0], [2048, 2049, 1, 4096, 0, 5], [300] * 100,
                                   [3, 5_000_001, 17], [2047 * 4096]])
def test_grad_norm(hip, ctx, torch_cuda, sizes, off):
    torch = torch_cuda
    for kinds in ([0] * len(sizes), [1] * len(sizes), [i % 2 for i in range(len(sizes))]):
        ts = grad_tensors(torch, sizes, kinds, len(sizes), off)
        group = hip.GradGroup(ctx, ts)
        norm, factor = Guarded(torch, (1,), torch.float32), Guarded(torch, (1,), torch.float32)
        want = norm64(torch, ts)
        group.norm(0.0, norm.t)
        # f64 sums of f64 squares, rounded once.
        assert abs(float(norm.t) - want) <= (U + 1e-12) * want and float(factor.t) == 7
        for cap in (want / 3, want * 3):
            cap = float(np.float32(cap))
            norm.t.fill_(0)
            group.norm(cap, norm.t, factor.t)
            f = min(1.0, cap / want)
            assert abs(float(norm.t) - want) <= (U + 1e-12) * want
            assert abs(float(factor.t) - f) <= (U + 1e-12) * f
            group.norm(cap, None, factor.t)
            assert abs(float(factor.t) - f) <= (U + 1e-12) * f
        assert norm.intact() and factor.intact()
        ctx.call("seeai_flush")
        # in place
        factor.t.fill_(0.3)
        before = [t.clone() for t in ts]
        group.scale(factor.t)
        for t, b in zip(ts, before):
            assert torch.equal(t, (b.float() * factor.t).to(t.dtype))
        factor.t.fill_(1.0)
        before = [t.clone() for t in ts]
        group.scale(factor.t)
        assert all(torch.equal(t, b) for t, b in zip(ts, before))
        group.close()


def test_grad_norm_of_nothing_zeros_and_large_values(hip, ctx, torch_cuda):
    torch = torch_cuda
    norm, factor = torch.full((1,), 3.0, device="cuda"), torch.full((1,), 3.0, device="cuda")
    for ts in ([], [torch.zeros(0, device="cuda")], [torch.zeros(5000, device="cuda")]):
        hip.GradGroup(ctx, ts).norm(1.0, norm, factor)
        assert float(norm) == 0 and float(factor) == 1
    big = torch.full((4,), 2e30, device="cuda")  # their squares are past f32
    hip.GradGroup(ctx, [big]).norm(1.0, norm, factor)
    assert abs(float(norm) - 4e30) < 1e24 and abs(float(factor) - 2.5e-31) < 1e-37
    small = torch.full((4,), 2e-30, device="cuda")
    hip.GradGroup(ctx, [small]).norm(1.0, norm, factor)
    assert abs(float(norm) / 4e-30 - 1) < 1e-6 and float(factor) == 1
    with pytest.raises(hip.BackendError) as e:
        hip.GradGroup(ctx, [big]).norm(-1.0, norm, factor)
    assert e.value.status == hip.REFUSED and str(e.value) == hip.CLIP_THRESHOLD_REFUSAL
    for cap in (float("inf"), float("nan")):
        with pytest.raises(hip.BackendError):
            hip.GradGroup(ctx, [big]).norm(cap, norm, factor)
    with pytest.raises(hip.BackendError, match="needs a max_norm"):
        hip.GradGroup(ctx, [big]).norm(0.0, norm, factor)
    with pytest.raises(hip.BackendError, match="null operand"):
        hip.GradGroup(ctx, [big]).norm(1.0, norm)
    with pytest.raises(hip.BackendError, match="null operand"):
        hip.GradGroup(ctx, [big]).norm()
    with pytest.raises(hip.BackendError, match="share memory"):
        hip.GradGroup(ctx, [big, big])


def states(torch, sizes, bits, seed):
    rnd = gen(torch, seed)
    out = []
    for n in sizes:
        t = {"p": 0.1 * rnd(n)}
        if bits == 32:
            t["m"], t["v"] = 0.1 * rnd(n), 0.01 * rnd(n).abs()
        else:
            t["m"], t["v"] = (torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2))
            t["m_scale"], t["v_scale"] = (torch.zeros((n + 127) // 128, device="cuda") for _ in range(2))
        out.append(t)
    return out


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bf16", [0, 1])
def test_scaled_step_is_the_step_on_scaled_gradients(hip, ctx, torch_cuda, bf16, bits):
    """Bit for bit, the product rounded to f32."""
    torch = torch_cuda
    sizes = [1, 300, 2048, 5001]
    ts, twins = states(torch, sizes, bits, 1), states(torch, sizes, bits, 1)
    grads = grad_tensors(torch, sizes, [bf16] * len(sizes))
    factor = torch.tensor([0.37], device="cuda")
    group = hip.AdamWGroup(ctx, [t | {"g": g} for t, g in zip(ts, grads)], bits, "bf16" if bf16 else "f32", seed=2)
    scaled = hip.AdamWGroup(ctx, [t | {"g": g.float() * factor} for t, g in zip(twins, grads)], bits, "f32", seed=2)
    for step in (1, 2, 3):
        pr = hip.StepParams(1e-2, 0.9, 0.999, 1e-8, 0.05, 0, step)
        if step == 3:  # the same through values held on the device
            group.hold(pr)
            group.step(None, factor)
        else:
            group.step(pr, factor)
        scaled.step(pr)
    for t, w in zip(ts, twins):
        assert all(torch.equal(v, w[k]) for k, v in t.items())
    with pytest.raises(hip.BackendError, match="from 1"):
        group.step(hip.StepParams(), factor)


def test_a_norm_that_is_not_finite_refuses_the_step(hip, torch_cuda):
    torch = torch_cuda
    ctx = hip.Context(0)
    ctx.use_torch_stream()
    sizes = [5, 3000]
    for bad in (float("nan"), float("inf")):
        ts = states(torch, sizes, 32, 3)
        grads = grad_tensors(torch, sizes, [0, 0])
        grads[1][2999] = bad
        keep = [{k: v.clone() for k, v in t.items()} for t in ts]
        kept = [g.clone() for g in grads]
        group = hip.AdamWGroup(ctx, [t | {"g": g} for t, g in zip(ts, grads)])
        clip = hip.GradGroup(ctx, grads)
        norm, factor = torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda")
        clip.norm(0.0, norm)  # the norm alone refuses nothing
        ctx.call("seeai_flush")
        assert not torch.isfinite(norm).any()
        clip.norm(1.0, norm, factor)
        clip.scale(factor)
        group.step(hip.StepParams(1e-2, 0.9, 0.999, 1e-8, 0.05, 0, 1), factor)
        with pytest.raises(hip.BackendError) as e:
            ctx.call("seeai_flush")
        assert e.value.status == hip.REFUSED and str(e.value) == hip.NON_FINITE_NORM_REFUSAL
        assert float(factor) == 1
        for t, w in zip(ts, keep):
            assert all(torch.equal(v, w[k]) for k, v in t.items())
        for g, w in zip(grads, kept):
            assert torch.equal(g.view(torch.int32), w.view(torch.int32))
        grads[1][2999] = 0.5  # the refusal was for that step
        clip.norm(1.0, norm, factor)
        group.step(hip.StepParams(1e-2, 0.9, 0.999, 1e-8, 0.05, 0, 1), factor)
        ctx.call("seeai_flush")
        assert not torch.equal(ts[0]["p"], keep[0]["p"])


def test_entry_points_refuse_on_the_context(hip, ctx, torch_cuda):
    torch = torch_cuda
    z = torch.zeros(4, 8, device="cuda")
    labels = torch.zeros(4, dtype=torch.int32, device="cuda")
    p, lib = hip.ptr, hip.lib()
    with pytest.raises(hip.BackendError, match="token_logp_fwd: rows are at least C apart"):
        ctx.call("seeai_token_logp_fwd", 0, p(z), 7, p(labels), p(z), None, 4, 8)
    with pytest.raises(hip.BackendError, match="token_logp_bwd: null operand"):
        ctx.call("seeai_token_logp_bwd", 0, p(z), 8, p(labels), None, p(z), p(z), 4, 8)
    with pytest.raises(hip.BackendError, match="pref_loss: workspace too small"):
        ctx.call("seeai_pref_loss", p(z), None, p(labels), p(labels), 4, 1, 0.1, 0.0, 0.0, 0, 1.0, p(z), None,
                 None, None, 0)
    with pytest.raises(hip.BackendError, match="policy_loss: a KL term"):
        ctx.call("seeai_policy_loss", 0, p(z), 8, p(labels), p(z), None, p(z), None, 4, 8, 0.2, 0.2, 0.1, 1.0,
                 p(z), None, None, None, 0)
    assert lib.seeai_token_logp_fwd(None, 0, None, 1, None, None, None, 0, 1) == 2
    assert lib.seeai_grad_group_norm(None, 1.0, None, None) == 2
    assert lib.seeai_grad_group_scale(None, None) == 2
    assert lib.seeai_adamw_group_step_scaled(None, None, None) == 2
    lib.seeai_grad_group_destroy(None)
