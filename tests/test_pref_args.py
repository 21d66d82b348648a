"""CPU: the refusals of seeai_token_logp_*, seeai_pref_loss, seeai_policy_loss,
seeai_block_join_* and seeai_grad_group_*, and their workspaces.  The checks are
plain C++ (csrc/pref_args.h, csrc/block_args.h), built here with g++ behind one C
function a check; operands are made-up addresses that nothing reads."""
from __future__ import annotations

import ctypes as C
import subprocess

import pytest

from tests.conftest import ROOT

HARNESS = r"""
#include "see-ai_amd/csrc/pref_args.h"
using namespace seeai;
static const float* f(uint64_t p) { return reinterpret_cast<const float*>(p); }
static const int32_t* i(uint64_t p) { return reinterpret_cast<const int32_t*>(p); }
static const void* v(uint64_t p) { return reinterpret_cast<const void*>(p); }
extern "C" {
const char* logp_fwd(int dt, const uint64_t* p, uint64_t ld, uint64_t N, uint64_t C) {
  return CheckTokenLogpFwd(dt, v(p[0]), ld, i(p[1]), f(p[2]), f(p[3]), N, C);
}
const char* logp_bwd(int dt, const uint64_t* p, uint64_t ld, uint64_t N, uint64_t C) {
  return CheckTokenLogpBwd(dt, v(p[0]), ld, i(p[1]), f(p[2]), f(p[3]), v(p[4]), N, C);
}
const char* pref(const uint64_t* p, uint64_t N, uint64_t pairs, float beta, float off, float eps, int avg, float scale, uint64_t wsb, uint64_t need) {
  return CheckPrefLoss(f(p[0]), f(p[1]), i(p[2]), i(p[3]), N, pairs, beta, off, eps, avg, scale, f(p[4]), f(p[5]), f(p[6]), v(p[7]), wsb, need);
}
const char* policy(int dt, const uint64_t* p, uint64_t ld, uint64_t N, uint64_t C, float low, float high, float kl, float scale, uint64_t wsb, uint64_t need) {
  return CheckPolicyLoss(dt, v(p[0]), ld, i(p[1]), f(p[2]), f(p[3]), f(p[4]), f(p[5]), N, C, low, high, kl, scale, f(p[6]), f(p[7]), v(p[8]), v(p[9]), wsb, need);
}
const char* join_fwd(const seeai_block_join* j, const uint64_t* p) { return CheckJoinFwd(*j, v(p[0]), v(p[1]), f(p[2])); }
const char* join_bwd(const seeai_block_join* j, const uint64_t* p, const seeai_block_join_grads* g, uint64_t ws, uint64_t wsb, uint64_t need) {
  return CheckJoinBwd(*j, v(p[0]), f(p[1]), v(p[2]), v(p[3]), *g, v(ws), wsb, need);
}
const char* grads(const seeai_grad_tensor* t, uint64_t n) { return CheckGradGroup(t, n); }
}
"""
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    d = tmp_path_factory.mktemp("pref_args")
    src, lib = d / "h.cc", d / "h.so"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", f"-I{ROOT}", str(src), "-o", str(lib)], check=True)
    h = C.CDLL(str(lib))

    def call(name, *args):
        fn = getattr(h, name)
        fn.restype = C.c_char_p
        return fn(*[(C.c_uint64 * len(a))(*a) if isinstance(a, list) else C.c_float(a)
                    if isinstance(a, float) else a for a in args])
    return call


def spread(n, step=1 << 30):
    return [(i + 1) * step for i in range(n)]


def u(x):
    return C.c_uint64(x)


def test_token_logp_refusals(checks):
    fwd = lambda dt=0, p=None, ld=10, N=4, V=8: checks("logp_fwd", dt, p or spread(4), u(ld), u(N), u(V))  # noqa: E731
    assert fwd() is None and fwd(1) is None and fwd(N=0) is None and fwd(N=0, p=[0] * 4) is None
    assert fwd(p=[*spread(3), 0]) is None  # no statistics wanted
    assert b"dtype" in fwd(2) and b"dtype" in fwd(-1)
    assert b"shape" in fwd(V=0, ld=0) and b"shape" in fwd(V=1 << 31, ld=1 << 31) and b"shape" in fwd(N=1 << 31)
    assert b"apart" in fwd(ld=7)
    assert b"large" in fwd(ld=1 << 40, N=1 << 22) and b"large" in fwd(ld=(1 << 64) - 1)
    for i in range(3):
        p = spread(4)
        p[i] = 0
        assert b"null" in fwd(p=p), i
    p = spread(4)
    p[0] += 2
    assert b"alignment" in fwd(p=p) and fwd(1, p=p) is None
    p = spread(4)
    p[2] = p[0] + 4 * (3 * 10 + 8) - 4  # logp on the last logit
    assert b"overlaps" in fwd(p=p)
    p[2] += 4
    assert fwd(p=p) is None
    bwd = lambda dt=0, p=None, ld=10, N=4, V=8: checks("logp_bwd", dt, p or spread(5), u(ld), u(N), u(V))  # noqa: E731
    assert bwd() is None and bwd(N=0, p=[0] * 5) is None
    for i in range(5):
        p = spread(5)
        p[i] = 0
        assert b"null" in bwd(p=p), i
    p = spread(5)
    p[4] = p[0]  # in place
    assert bwd(p=p) is None
    p[4] = p[0] + 8
    assert b"overlaps" in bwd(p=p)
    p[4] = p[3] = p[0]
    assert b"overlaps" in bwd(p=p)


def test_pref_refusals(checks):
    def ask(p=None, N=9, pairs=2, beta=0.1, off=0.0, eps=0.1, avg=0, scale=0.5, wsb=16, need=16):
        return checks("pref", p or spread(8), u(N), u(pairs), beta, off, eps, avg, scale, u(wsb), u(need))
    assert ask() is None and ask(eps=0.0) is None and ask(eps=1.0) is None and ask(beta=-1.0) is None
    assert ask(pairs=0, need=0, wsb=0, p=[0, 0, 0, 0, 1 << 30, 0, 2 << 30, 0]) is None
    for i in (1, 5, 6):  # without a reference, margins, a gradient
        p = spread(8)
        p[i] = 0
        assert ask(p=p) is None, i
    for i in (0, 2, 3, 4, 7):
        p = spread(8)
        p[i] = 0
        assert b"null" in ask(p=p), i
    assert b"shape" in ask(N=1 << 31) and b"shape" in ask(pairs=(1 << 20) + 1) and ask(pairs=1 << 20) is None
    assert b"average" in ask(avg=2)
    for bad in (-0.1, 1.1, NAN):
        assert b"smoothing" in ask(eps=bad)
    for bad in (INF, -INF, NAN):
        assert all(b"finite" in ask(**{k: bad}) for k in ("beta", "off", "scale"))
    assert b"workspace" in ask(wsb=15)
    p = spread(8)
    p[6] = p[0]  # the gradient over the log-probabilities
    assert b"overlaps" in ask(p=p)


def test_policy_refusals(checks):
    def ask(p=None, dt=1, ld=8, N=4, V=8, low=0.2, high=0.2, kl=0.1, scale=1.0, wsb=32, need=32):
        return checks("policy", dt, p or spread(10), u(ld), u(N), u(V), low, high, kl, scale, u(wsb), u(need))
    assert ask() is None and ask(low=0.0, high=0.0) is None and ask(low=1.0, high=1e30) is None
    assert ask(N=0, need=0, wsb=0, p=[0] * 6 + [1 << 30, 0, 0, 0]) is None
    for i in (5, 7, 8):  # without weights, log-probabilities, a gradient
        p = spread(10)
        p[i] = 0
        assert ask(p=p) is None, i
    p = spread(10)
    p[3] = 0
    assert b"KL" in ask(p=p) and ask(p=p, kl=0.0) is None
    for i in (0, 1, 2, 4, 6, 9):
        p = spread(10)
        p[i] = 0
        assert b"null" in ask(p=p), i
    for bad in (-0.1, 1.1, NAN):
        assert b"clip_low" in ask(low=bad)
    for bad in (-0.1, INF, NAN):
        assert b"clip_high" in ask(high=bad)
    for bad in (INF, NAN):
        assert b"finite" in ask(kl=bad) and b"finite" in ask(scale=bad)
    assert b"workspace" in ask(wsb=31) and b"apart" in ask(ld=7) and b"dtype" in ask(dt=2)
    p = spread(10)
    p[8] = p[0]  # in place
    assert ask(p=p) is None
    p[7] = p[2]
    assert b"overlaps" in ask(p=p)


def make_join(hip, **over):
    names = ("o", "x", "post_w", "post_b", "gate", "pre_w", "pre_b")
    j = hip.BlockJoin(*spread(7), 6, 32, 4, 0, 0, 1.0, 1e-5)
    for k, v in over.items():
        assert k in names or hasattr(j, k)
        setattr(j, k, v)
    return j


def test_join_refusals(checks, hip):
    y = [8 << 30, 9 << 30, 10 << 30]
    fwd = lambda p=None, **over: checks("join_fwd", C.byref(make_join(hip, **over)), p or y)  # noqa: E731
    assert fwd() is None and fwd(dtype=1) is None and fwd(gate=0, gate_rows=0) is None
    assert fwd(kind=1, post_b=0, pre_b=0) is None and fwd(post_b=0) is None
    assert fwd(p=[y[0], y[1], 0]) is None
    assert fwd(p=[2 << 30, y[1], y[2]]) is None  # y in x's place
    assert b"overlaps" in fwd(p=[1 << 30, y[1], y[2]])  # not in o's
    assert fwd(p=[y[0], 0, y[2]], pre_w=0, pre_b=0) is None
    assert b"no norm" in fwd(pre_w=0, pre_b=0)
    assert b"neither" in fwd(pre_w=0, pre_b=0, post_w=0, post_b=0)
    assert b"without its norm" in fwd(post_w=0) and b"without its norm" in fwd(pre_w=0, p=[y[0], 0, y[2]])
    assert b"has no bias" in fwd(kind=1) and b"kind" in fwd(kind=2) and b"dtype" in fwd(dtype=2)
    assert b"shape" in fwd(cols=0) and b"shape" in fwd(cols=16385) and b"shape" in fwd(rows=1 << 31)
    assert fwd(cols=16384) is None and fwd(rows=0, o=0, x=0, p=[0, 0, 0]) is None
    assert b"eps" in fwd(eps=-1.0) and b"eps" in fwd(eps=NAN) and b"res_scale" in fwd(res_scale=INF)
    assert b"gate_rows" in fwd(gate_rows=0) and fwd(gate_rows=1 << 40) is None
    for name in ("o", "x"):
        assert b"null" in fwd(**{name: 0})
    for k in range(2):
        assert b"null" in fwd(p=[0 if i == k else a for i, a in enumerate(y)])
    assert b"alignment" in fwd(pre_w=(6 << 30) + 2)
    # the gate's rows are ceil(6 / 4) = 2
    assert b"overlaps" in fwd(p=[(5 << 30) + 2 * 32 * 4 - 4, y[1], y[2]])
    assert fwd(p=[(5 << 30) + 2 * 32 * 4, y[1], y[2]]) is None

    def bwd(p=None, g=None, ws=30 << 30, wsb=64, need=64, **over):
        grads = hip.BlockJoinGrads(*(g or [(20 + i) << 30 for i in range(7)]))
        return checks("join_bwd", C.byref(make_join(hip, **over)), p or spread(4, 1 << 36), C.byref(grads), u(ws),
                      u(wsb), u(need))
    g = [(20 + i) << 30 for i in range(7)]
    assert bwd() is None and bwd(x=0) is None and b"workspace" in bwd(wsb=63)
    some = lambda **at: [at.get(f"g{i}", a) for i, a in enumerate(g)]  # noqa: E731
    for i in (3, 4, 6):  # gradients that are not wanted
        assert bwd(g=some(**{f"g{i}": 0})) is None, i
    for i in (0, 1, 2, 5):
        assert b"null" in bwd(g=some(**{f"g{i}": 0})), i
    for i in (0, 1, 2):
        p = spread(4, 1 << 36)
        p[i] = 0
        assert b"null" in bwd(p=p), i
    p = spread(4, 1 << 36)
    p[3] = 0
    assert bwd(p=p) is None  # nothing reaches y past h
    p[3] = g[0]
    assert bwd(p=p) is None  # dx in dy's place
    assert b"overlaps" in bwd(g=some(g1=p[2]), p=p)
    rms = dict(kind=1, post_b=0, pre_b=0)
    assert b"absent" in bwd(**rms) and bwd(g=some(g3=0, g6=0), **rms) is None
    assert b"absent" in bwd(gate=0) and bwd(gate=0, g=some(g4=0)) is None
    assert b"no norm that gave" in bwd(pre_w=0, pre_b=0, g=some(g5=0, g6=0))
    p = spread(4, 1 << 36)
    p[0] = p[2] = 0
    assert bwd(p=p, pre_w=0, pre_b=0, g=some(g5=0, g6=0)) is None


def test_grad_group_refusals(checks, hip):
    def ask(**over):
        t = (hip.GradTensor * 2)()
        for i in range(2):
            t[i].g, t[i].n, t[i].dtype = (i + 1) << 30, 1000, i
        for k, v in over.items():
            setattr(t[1], k, v)
        return checks("grads", t, u(2))
    assert ask() is None and checks("grads", None, u(0)) is None and b"null" in checks("grads", None, u(1))
    assert b"dtype" in ask(dtype=2) and b"null" in ask(g=0) and ask(g=0, n=0, dtype=7) is None
    assert b"alignment" in ask(g=(2 << 30) + 1) and ask(g=(2 << 30) + 2) is None
    assert b"alignment" in ask(g=(2 << 30) + 2, dtype=0)
    assert b"share" in ask(g=(1 << 30) + 3998) and ask(g=(1 << 30) + 4000) is None
    assert b"large" in ask(n=1 << 36) and b"large" in ask(n=1 << 35, g=1 << 50)


def test_workspaces(hip):
    lib = hip.lib()
    assert lib.seeai_pref_workspace(0) == 0 and lib.seeai_pref_workspace(10) == 80
    assert lib.seeai_pref_workspace(1 << 21) == 0
    assert lib.seeai_policy_workspace(0, 100) == 0 and 0 < lib.seeai_policy_workspace(1 << 20, 32000) <= 1 << 20
    assert lib.seeai_policy_workspace(5, 0) == 0
    assert lib.seeai_block_join_workspace(8192, 0, 0) == 0
    for rows, cols, gate in ((8192, 2048, 8192), (8192, 2048, 0), (8192, 2048, 1), (100000, 64, 7),
                             (3001, 1023, 500), (1, 16384, 1)):
        n = lib.seeai_block_join_workspace(rows, cols, gate)
        assert n <= 4 * 4 * cols * 1100, (rows, cols, gate, n)
        assert n == 0 or n >= 2 * 16 * cols


class Fake:
    """What the group's own checks ask of a tensor."""

    def __init__(self, dtype="float32", n=300, contiguous=True, device=True):
        self.dtype, self.n, self.contiguous, self.is_cuda = "torch." + dtype, n, contiguous, device

    def numel(self):
        return self.n

    def is_contiguous(self):
        return self.contiguous

    def data_ptr(self):
        return 1 << 20


class Accepting:
    h = None

    def call(self, name, *args):
        return None

    def check(self, rc):
        return None


def test_grad_group_wrapper(hip):
    make = lambda *ts: hip.GradGroup(Accepting(), ts)  # noqa: E731
    held = make(Fake(), Fake("bfloat16"), Fake("int16"), Fake("uint16"))
    assert len(held.tensors) == 4
    for t in (Fake("float16"), Fake("int32"), Fake(contiguous=False), Fake(device=False)):
        with pytest.raises(ValueError):
            make(Fake(), t)

    class At:
        index = 0
    ctx = Accepting()
    ctx.device_index = 1
    t = Fake()
    t.device = At()
    with pytest.raises(ValueError, match="device 1"):
        hip.GradGroup(ctx, [t])
    group = hip.GradGroup.__new__(hip.GradGroup)
    group.h, group.ctx = None, Accepting()
    for call in (lambda: group.norm(1.0, Fake(n=1), Fake(n=1)), lambda: group.scale(Fake(n=1))):
        with pytest.raises(hip.BackendError, match="closed"):
            call()
    for bad in (Fake(n=2), Fake("bfloat16", 1), Fake(n=1, device=False)):
        with pytest.raises(ValueError, match="factor"):
            group.scale(bad)
        with pytest.raises(ValueError, match="norm"):
            group.norm(0.0, bad)
    step = hip.AdamWGroup.__new__(hip.AdamWGroup)
    step.h, step.ctx = 1 << 20, Accepting()
    step.ctx.h = 1
    with pytest.raises(ValueError, match="factor"):
        step.step(hip.StepParams(), Fake(n=2))
    step.h = None


def test_policy_logits_are_there_without_a_gradient(checks):
    """No gradient wanted is not a gradient in the logits' place."""
    def ask(p, N=4):
        return checks("policy", 1, p, u(8), u(N), u(8), 0.2, 0.2, 0.1, 1.0, u(32), u(32))
    p = spread(10)
    p[0] = p[8] = 0
    assert b"null" in ask(p)
    assert ask([0] * 6 + [1 << 30, 0, 0, 2 << 30], N=0) is None
    p = spread(10)
    p[8] = 0
    assert ask(p) is None
    p[8] = p[0]
    assert ask(p) is None
