"""GPU: where the losses from logits come to the ends of their ranges -- nearly sure
labels, far margins, coefficients of zero, ratios and KL terms past f32 -- and the
joins' column sums past 32-bit offsets, against plain float64.

Tolerances are bounds on what the kernels' own roundings may add up to, as in
test_gpu_pref.py and test_gpu_join.py: u = 2^-24 for each f32 operation, 2^-8 of the
value for a rounding to bf16, exp(x) within (3 |x| + 2) u of itself."""
from __future__ import annotations

import math

import pytest

from tests.test_gpu_block import U, Guarded, ctx, gen, types, within  # noqa: F401
from tests.test_gpu_join import DEPTH, NAMES, back64, backward, forward, inputs, struct
from tests.test_gpu_pref import (policy64, policy_loss, pref_loss, softmax64, token_inputs, token_logp,
                                 token_logp_bwd)

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


# --- nearly sure labels ---------------------------------------------------------------------------

# Rows of a wave, of four and sixteen waves, walked and in registers; the label's
# neighbours within 16 bytes are terms like all others, wherever the row begins.
SURE = [(64, 3, 3, 0), (64, 40, 40, 0), (64, 41, 43, 1), (64, 2000, 2000, 0), (700, 2113, 2113, 1),
        (64, 4000, 4000, 0), (3, 32001, 32003, 1), (700, 32000, 32000, 0), (520, 50001, 50001, 1),
        (3, 131000, 131000, 0), (2, 131073, 131080, 1)]


def sure_inputs(torch, N, V, ld, off, bf16, gap):
    """Rows whose labels, anywhere in them, are sure but for about exp(-gap)."""
    t, step = types(torch, bf16)
    buf = Guarded(torch, (N, ld), t, off)
    buf.t.fill_(NAN)
    z = 0.5 * gen(torch, V + ld)(N, V) - math.log(V) - gap + 1.0
    labels = torch.randint(0, V, (N,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(V))
    labels[0], labels[-1] = 0, V - 1
    z[torch.arange(N), labels] = 1.0
    buf.t[:, :V] = z.to(t)
    d = buf.t[:, :V].double() - 1.0
    e = torch.exp(d).scatter(1, labels[:, None], 0.0)  # the others, beside the label's 1
    return buf, labels.to(torch.int32), d, e, step


def sure_logp(d, e):
    """-log(1 + the others' sum), and its bound: each of the others' terms within
    (3 |d| + 2) u, the rescalings to higher maxima on their way (together as far, 2 u
    for each of at most 11), three additions within 16 bytes, then f64; a rounding of the
    sum and a logarithm good to 4 u."""
    want = -e.sum(1).log1p()
    return want, U * ((e * (6 * d.abs() + 30)).sum(1) + 6 * want.abs())


@pytest.mark.parametrize("gap", [6.0, 14.0, 21.0])
@pytest.mark.parametrize("bf16", [0, 1])
def test_a_nearly_sure_label_beside_its_neighbours(hip, ctx, torch_cuda, bf16, gap):
    """However little is left beside the label, and wherever it lies, the
    log-probability keeps its own digits."""
    torch = torch_cuda
    for N, V, ld, off in SURE:
        buf, labels, d, e, _ = sure_inputs(torch, N, V, ld, off, bf16, gap)
        want, bound = sure_logp(d, e)
        logp, stats = token_logp(ctx, torch, buf.t, ld, labels, V)
        within(torch, logp, want, bound)
        assert (stats[:, 0] == 1).all()
        within(torch, stats[:, 1], 1 + e.sum(1), bound + 2 * U)
        zeros = torch.zeros(N, device="cuda")
        _, again = policy_loss(hip, ctx, torch, buf.t, ld, labels, zeros, None, zeros, None, V, 0.0, 1.0)
        within(torch, again, want, bound)


@pytest.mark.parametrize("gap", [6.0, 14.0, 21.0])
@pytest.mark.parametrize("bf16", [0, 1])
def test_a_nearly_sure_label_keeps_its_gradient(hip, ctx, torch_cuda, bf16, gap):
    """The label's element is d (1 - p): small beside d, but as near to itself as the
    others' d p, whose sum it is.  Those are within (3 |d| + 2) u, the row's sum and
    the division 2 u each, a product, three additions within 16 bytes."""
    torch = torch_cuda
    t, _ = types(torch, bf16)
    for N, V, ld, off in SURE:
        buf, labels, d, e, step = sure_inputs(torch, N, V, ld, off, bf16, gap)
        row = torch.arange(N, device="cuda")
        p = e / (1 + e.sum(1, keepdim=True))
        rest, e_rest = p.sum(1), U * (p * (3 * d.abs() + 12)).sum(1)
        _, stats = token_logp(ctx, torch, buf.t, ld, labels, V)
        dlogp = gen(torch, 5)(N)
        out = Guarded(torch, (N, ld), t, off)
        token_logp_bwd(ctx, torch, buf.t, ld, labels, stats, dlogp, V, out.t)
        got, dd = out.t[row, labels.long()], dlogp.double()
        within(torch, got, dd * rest, dd.abs() * (e_rest + step * (rest + e_rest)))
        assert out.intact() and (out.t[:, V:] == 7).all()
        # The policy loss, from the log-probabilities that it gives itself.
        adv, old = gen(torch, 6)(N), torch.full((N,), -0.05, device="cuda")
        _, lp = policy_loss(hip, ctx, torch, buf.t, ld, labels, old, None, adv, None, V, 0.0, 1.0, out.t)
        _, _, dd, e_d = policy64(torch, lp, torch.zeros_like(dd), labels, old, None, adv, None, 0.0, 1.0)
        rest = -torch.expm1(lp.double())
        bound = e_d * rest + dd.abs() * 8 * U * rest
        within(torch, out.t[row, labels.long()], dd * rest, bound + step * ((dd * rest).abs() + bound))
        keep = out.t.clone()
        policy_loss(hip, ctx, torch, buf.t, ld, labels, old, None, adv, None, V, 0.0, 1.0, buf.t)
        assert torch.equal(buf.t[:, :V], keep[:, :V])


@pytest.mark.parametrize("bf16", [0, 1])
def test_wide_rows_add_up_in_64_bits(ctx, torch_cuda, bf16):
    """Of a sum's roundings only the exponentials' own count, and three additions
    within 16 bytes, however wide the row is."""
    torch = torch_cuda
    for N, V, ld, off in ((600, 9001, 9001, 1), (520, 50001, 50001, 0), (2, 131073, 131080, 1), (1, 262144, 262144, 0)):
        buf, labels = token_inputs(torch, N, V, ld, bf16, V, skip=0.0, off=off)
        logp, _ = token_logp(ctx, torch, buf.t, ld, labels, V)
        want, _, p, _ = softmax64(torch, buf.t[:, :V], labels)
        z = buf.t[:, :V].double()
        d = (z - z.amax(1, keepdim=True)).abs()
        picked, log_s = d.gather(1, labels.long()[:, None])[:, 0], d.gather(1, labels.long()[:, None])[:, 0] + want
        within(torch, logp, want, U * ((p * (6 * d + 30)).sum(1) + picked + 4 * log_s.abs() + 2 * want.abs() + 2))


@pytest.mark.parametrize("bf16", [0, 1])
def test_log_probabilities_are_rounded_once(hip, ctx, torch_cuda, bf16):
    """Equal logits but the label's, so that the others' sum is a whole number: what is
    left is a logarithm of at most 0.35, good to 4 u of itself, and the result's own
    rounding."""
    torch = torch_cuda
    t, _ = types(torch, bf16)
    N = 64
    for V in range(300, 40000, 1237):
        below = torch.linspace(0.0, 16.0, N, device="cuda").to(t)
        z = torch.zeros(N, V, dtype=t, device="cuda")
        labels = torch.randint(0, V, (N,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(V))
        z[torch.arange(N), labels] = -below
        labels, zeros = labels.to(torch.int32), torch.zeros(N, device="cuda")
        want = -below.double() - torch.log(V - 1 + torch.exp(-below.double()))
        logp, _ = token_logp(ctx, torch, z, V, labels, V)
        within(torch, logp, want, U * (want.abs() + 2))
        _, again = policy_loss(hip, ctx, torch, z, V, labels, zeros, None, zeros, None, V, 0.0, 1.0)
        within(torch, again, want, U * (want.abs() + 2))


# --- far margins ----------------------------------------------------------------------------------

def test_pairs_of_far_margins_keep_their_gradient(hip, ctx, torch_cuda):
    """scale beta (eps - sigmoid(-margin)) is exp(-margin) where the chosen answer is far
    ahead and nothing is smoothed: its digits are its own, not those of a difference
    from 1."""
    torch = torch_cuda
    for lengths in ([1, 1] * 9, [700, 700] * 9):  # one workgroup for all pairs, and one a pair
        margins = torch.tensor([-80.0, -40.0, -20.0, -3.0, 0.0, 3.0, 20.0, 40.0, 80.0], dtype=torch.float64)
        N = sum(lengths)
        starts = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
        logp = torch.zeros(N, device="cuda")
        logp[starts[0:-1:2].long()] = margins.float().cuda()  # the chosen answers' first tokens
        labels = torch.zeros(N, dtype=torch.int32, device="cuda")
        for eps, sign in ((0.0, 1.0), (1.0, -1.0)):
            got = pref_loss(hip, ctx, torch, logp, None, labels, starts, 1.0, 0.0, eps, 0, 1.0)
            want = -sign * torch.sigmoid(-sign * margins).cuda()
            d = got[2][starts[0:-1:2].long()]
            within(torch, d, want, (U + 1e-14) * want.abs())
            assert torch.equal(got[2][starts[1::2].long()], -d)


# --- coefficients of zero, and terms past f32 -----------------------------------------------------

def rows_of_tokens(hip, ctx, torch, V, N=12):
    z = gen(torch, V)(N, V)
    labels = torch.full((N,), 4, dtype=torch.int32, device="cuda")
    lp, _ = token_logp(ctx, torch, z, V, labels, V)
    return z, labels, lp, gen(torch, 1)(N), gen(torch, 2)(N).abs() + 0.1


def call_policy(hip, ctx, torch, z, labels, old, ref, adv, weight, kl):
    out = torch.empty_like(z)
    loss, lp = policy_loss(hip, ctx, torch, z, z.shape[1], labels, old, ref, adv, weight, z.shape[1], kl, 1.0, out)
    return loss, lp, out


@pytest.mark.parametrize("V", [30, 5000, 40000])
def test_a_kl_coefficient_of_zero_takes_the_reference_out(hip, ctx, torch_cuda, V):
    """Tokens that the reference rules out, or has far above the policy, and a NaN: the
    bits of the call without a reference."""
    torch = torch_cuda
    z, labels, lp, adv, weight = rows_of_tokens(hip, ctx, torch, V)
    old, ref = lp + 0.01, lp.clone()
    ref[1], ref[2], ref[3], ref[4] = -INF, lp[2] + 200, NAN, INF
    z[5, 4] = -INF  # the policy rules the label out
    want = call_policy(hip, ctx, torch, z, labels, old, None, adv, weight, 0.0)
    got = call_policy(hip, ctx, torch, z, labels, old, ref, adv, weight, 0.0)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.isfinite(v).all() for v in (got[0], got[2]))


@pytest.mark.parametrize("V", [30, 5000])
def test_an_advantage_of_zero_beside_a_far_ratio(hip, ctx, torch_cuda, V):
    """Answers no better and no worse than the rest of their group: no term, however far
    the policy has moved (a ratio past f32)."""
    torch = torch_cuda
    z, labels, lp, adv, weight = rows_of_tokens(hip, ctx, torch, V)
    old = lp + 0.01
    adv[3], adv[5] = 0.0, -0.0
    want = call_policy(hip, ctx, torch, z, labels, old, None, adv, weight, 0.0)
    old[3], old[5] = lp[3] - 100, lp[5] - 1e4
    got = call_policy(hip, ctx, torch, z, labels, old, None, adv, weight, 0.0)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.isfinite(got[2]).all()
    assert not got[2][[3, 5]].any()


@pytest.mark.parametrize("V", [30, 5000])
def test_a_weight_of_zero_takes_its_row_out(hip, ctx, torch_cuda, V):
    """Whatever its other numbers are; its log-probability is given all the same."""
    torch = torch_cuda
    z, labels, lp, adv, weight = rows_of_tokens(hip, ctx, torch, V)
    old, ref = lp + 0.01, lp + 0.02
    off = [2, 3, 4, 5, 6]
    weight[off] = 0.0
    old[2], adv[2] = lp[2] - 100, -1.0  # a term past f32
    ref[3] = lp[3] + 200
    old[4], adv[5], ref[6] = NAN, INF, NAN
    out = call_policy(hip, ctx, torch, z, labels, old, ref, adv, weight, 0.1)
    labels[off] = -1
    want = call_policy(hip, ctx, torch, z, labels, old, ref, adv, weight, 0.1)
    assert torch.equal(out[0], want[0]) and torch.equal(out[2], want[2]) and torch.isfinite(out[2]).all()
    within(torch, out[1], lp, U * lp.abs())


@pytest.mark.parametrize("V", [30, 5000])
def test_the_kl_term_of_a_token_that_the_policy_rules_out(hip, ctx, torch_cuda, V):
    """exp(back) - back - 1 is an infinity where back is, on either side."""
    torch = torch_cuda
    for side in (0, 1):
        z, labels, lp, adv, weight = rows_of_tokens(hip, ctx, torch, V)
        old, ref = lp + 0.01, lp + 0.02
        if side:
            ref[3] = -INF
        else:
            z[3, 4] = -INF
        loss, got, out = call_policy(hip, ctx, torch, z, labels, old, ref, adv, weight, 0.1)
        assert float(loss) == INF and bool(got[3] == -INF) == (side == 0)
        others = [i for i in range(12) if i != 3]
        assert torch.isfinite(out[others]).all() and (side == 0 or torch.isfinite(out[3]).all())


# --- the joins ------------------------------------------------------------------------------------

@pytest.mark.parametrize("bf16", [0, 1])
def test_block_join_of_one_gate_for_more_rows_than_there_are(hip, ctx, torch_cuda, bf16):
    """The bits of a gate for exactly these rows."""
    torch = torch_cuda
    t, _ = types(torch, bf16)
    for rows, cols in ((5, 96), (300, 257), (300, 512), (2100, 130)):
        d = inputs(torch, 0, 1, 1, 1, rows, cols, rows, t, 0)
        dh, dy = gen(torch, 1)(rows, cols).to(t), gen(torch, 2)(rows, cols).to(t)
        y, h, st = forward(hip, ctx, torch, 0, bf16, d, rows, cols, rows)
        want = backward(hip, ctx, torch, 0, bf16, d, rows, y, st, dh, dy)
        for gate_rows in (rows + 1, 2 ** 31, 2 ** 61):
            got = forward(hip, ctx, torch, 0, bf16, d, rows, cols, gate_rows)
            assert all(torch.equal(a, b) for a, b in zip(got, (y, h, st)))
            got = backward(hip, ctx, torch, 0, bf16, d, gate_rows, y, st, dh, dy)
            assert all(torch.equal(got[k], want[k]) for k in NAMES)


def test_block_join_column_sums_past_32_bit_offsets(hip, ctx, torch_cuda):
    """Over 2^32 bytes and 2^31 elements, the last gate's rows few: the vectors' gradients
    against float64 sums.  A band's rows add up one after another, two rows at a time:
    512 bands, so up to 1,040 roundings, and the joins'."""
    torch = torch_cuda
    rows, cols, gate_rows, chunk = 1_060_000, 2048, 400_000, 20_000
    assert gate_rows % chunk == 0 and rows % chunk == 0
    t, rnd = torch.bfloat16, gen(torch, 1)
    o, x = (torch.empty(rows, cols, dtype=t, device="cuda").normal_(generator=torch.Generator(device="cuda")
                                                                   .manual_seed(s)) for s in (2, 3))
    d = {"o": o, "x": x, "post_w": 1 + 0.1 * rnd(cols), "post_b": None, "gate": rnd(3, cols), "pre_w": 1 + rnd(cols),
         "pre_b": None}
    y, h, st = torch.empty_like(o), torch.empty_like(o), torch.empty(rows, 4, device="cuda")
    j = struct(hip, 1, 1, d, rows, cols, gate_rows)
    ctx.call("seeai_block_join_fwd", j, y.data_ptr(), h.data_ptr(), st.data_ptr())
    grads = {"dx": torch.empty_like(o), "do": x, "dpost_w": torch.empty(cols, device="cuda"), "dpost_b": None,
             "dgate": torch.empty(3, cols, device="cuda"), "dpre_w": torch.empty(cols, device="cuda"), "dpre_b": None}
    n = hip.lib().seeai_block_join_workspace(rows, cols, gate_rows)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    ctx.call("seeai_block_join_bwd", j, y.data_ptr(), st.data_ptr(), h.data_ptr(), None,
             hip.BlockJoinGrads(*(hip.ptr(grads[k]) for k in NAMES)), ws.data_ptr(), n)
    run = 1100 + DEPTH  # a band's rows, the fold
    sums = lambda *s: torch.zeros(*s, cols, dtype=torch.float64, device="cuda")  # noqa: E731
    pre, e_pre, S1, e1 = sums(), sums(), sums(3), sums(3)
    w, w2, gate = d["post_w"].double(), d["pre_w"].double(), d["gate"].double()
    for at in range(0, rows, chunk):
        s, g = slice(at, at + chunk), at // gate_rows
        sd, H = st[s].double(), h[s].double()
        hat = y[s].double() * sd[:, 3:4]
        pre += (H * hat).sum(0)
        e_pre += (run + 3) * U * (H * hat).abs().sum(0)
        up = H * w2
        T, e = back64(torch, 1, up, U * up.abs(), hat, 3 * U * hat.abs(), sd[:, 3:4])
        ohat = o[s].double() * sd[:, 1:2]
        S1[g] += (T * ohat).sum(0)
        e1[g] += (run + 3) * U * (T * ohat).abs().sum(0) + (e * ohat.abs()).sum(0)
    within(torch, grads["dpre_w"], pre, e_pre)
    within(torch, grads["dgate"], S1 * w, (e1 + 4 * U * S1.abs()) * w.abs())
    within(torch, grads["dpost_w"], (S1 * gate).sum(0), ((e1 + 8 * U * S1.abs()) * gate.abs()).sum(0))
    # (a band left out or counted twice would show)
    assert float((e_pre / pre.abs()).max()) < 1e-3
