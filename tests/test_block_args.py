"""CPU: the refusals of the trained-block entry points (seeai_norm_*,
seeai_ffn_*, seeai_adamw_group_create) and their workspace sizes.  The checks
are plain C++ (csrc/block_args.h), built here with g++ behind one C function a
check; operands are made-up addresses that nothing reads."""
from __future__ import annotations

import ctypes as C
import os
import subprocess

import pytest

from tests.conftest import ROOT

HARNESS = r"""
#include "see-ai_amd/csrc/block_args.h"
using namespace seeai;
static const float* f(uint64_t p) { return reinterpret_cast<const float*>(p); }
static const void* v(uint64_t p) { return reinterpret_cast<const void*>(p); }
extern "C" {
const char* norm_fwd(int kind, int dt, const uint64_t* p, uint64_t r, uint64_t c, float eps) {
  return CheckNormFwd(kind, dt, v(p[0]), f(p[1]), f(p[2]), v(p[3]), f(p[4]), f(p[5]), r, c, eps);
}
const char* norm_bwd(int kind, int dt, const uint64_t* p, uint64_t r, uint64_t c, uint64_t wsb, uint64_t need) {
  return CheckNormBwd(kind, dt, v(p[0]), v(p[1]), f(p[2]), f(p[3]), f(p[4]), v(p[5]), f(p[6]), f(p[7]), r, c, v(p[8]), wsb, need);
}
const char* ffn_fwd(int dt, int act, const uint64_t* p, uint64_t M, uint64_t D, uint64_t F, uint64_t wsb, uint64_t need) {
  return CheckFfnFwd(dt, act, v(p[0]), v(p[1]), v(p[2]), v(p[3]), v(p[4]), v(p[5]), v(p[6]), M, D, F, v(p[7]), wsb, need);
}
const char* ffn_bwd(int dt, int act, const uint64_t* p, uint64_t M, uint64_t D, uint64_t F, uint64_t wsb, uint64_t need) {
  return CheckFfnBwd(dt, act, v(p[0]), v(p[1]), v(p[2]), v(p[3]), v(p[4]), v(p[5]), v(p[6]), v(p[7]), v(p[8]), v(p[9]), v(p[10]), M, D, F, v(p[11]), wsb, need);
}
const char* group(const seeai_adamw_tensor* t, uint64_t n, int bits, int g) { return CheckAdamWGroup(t, n, bits, g); }
}
"""


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    d = tmp_path_factory.mktemp("block_args")
    src, lib = d / "h.cc", d / "h.so"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", f"-I{ROOT}", str(src), "-o", str(lib)],
                   check=True)
    h = C.CDLL(str(lib))
    for name in ("norm_fwd", "norm_bwd", "ffn_fwd", "ffn_bwd", "group"):
        getattr(h, name).restype = C.c_char_p
    u64 = C.c_uint64

    def call(name, *args):
        conv = []
        for a in args:
            if isinstance(a, list):
                conv.append((u64 * len(a))(*a))
            elif isinstance(a, float):
                conv.append(C.c_float(a))
            else:
                conv.append(a)
        return getattr(h, name)(*conv)
    return call


def spread(n, step=1 << 24):
    return [(i + 1) * step for i in range(n)]


def u(x):
    return C.c_uint64(x)


def test_norm_refusals(checks):
    fwd = lambda kind=0, dt=0, p=None, r=4, c=8, eps=1e-5: checks(  # noqa: E731
        "norm_fwd", kind, dt, p or spread(6), u(r), u(c), eps)
    assert fwd() is None and fwd(dt=1) is None and fwd(r=0) is None
    rms = spread(6)
    rms[2] = rms[4] = 0
    assert fwd(1, p=rms) is None
    assert b"no bias" in fwd(1)
    assert b"kind" in fwd(2) and b"dtype" in fwd(dt=2) and b"shape" in fwd(c=0)
    assert b"shape" in fwd(r=1 << 31)
    assert b"eps" in fwd(eps=-1.0) and b"eps" in fwd(eps=float("nan")) and b"eps" in fwd(eps=float("inf"))
    for i in (0, 1, 3):
        p = spread(6)
        p[i] = 0
        assert b"null" in fwd(p=p)
    p = spread(6)
    p[0] += 2
    assert b"alignment" in fwd(p=p) and fwd(dt=1, p=p) is None
    p = spread(6)
    p[3] = p[0] + 4 * 8 * 4 - 4  # y begins on x's last element
    assert b"overlaps" in fwd(p=p)
    p[3] = p[0] + 4 * 8 * 4
    assert fwd(p=p) is None
    bwd = lambda kind=0, dt=0, p=None, r=4, c=8, wsb=256, need=256: checks(  # noqa: E731
        "norm_bwd", kind, dt, p or spread(9), u(r), u(c), u(wsb), u(need))
    assert bwd() is None and b"workspace" in bwd(wsb=255)
    assert b"no bias" in bwd(1)
    for i in (0, 1, 2, 3, 4, 5, 6, 8):
        p = spread(9)
        p[i] = 0
        assert b"null" in bwd(p=p), i
    p = spread(9)
    p[7] = 0  # no bias gradient
    assert bwd(p=p) is None
    p[8] += 8
    assert b"alignment" in bwd(p=p)
    p = spread(9)
    p[5] = p[0]  # dx over dy
    assert b"overlaps" in bwd(p=p)
    p = spread(9)
    p[0] = p[1]  # inputs may be one tensor
    assert bwd(p=p) is None


def test_ffn_refusals(checks):
    fwd = lambda dt=1, act=3, p=None, M=2, D=8, F=16, wsb=64, need=64: checks(  # noqa: E731
        "ffn_fwd", dt, act, p or spread(8), u(M), u(D), u(F), u(wsb), u(need))
    assert fwd() is None and fwd(M=0) is None
    p = spread(8)
    p[4] = p[5] = 0
    assert fwd(p=p) is None
    p[5] = 1 << 20
    assert b"both or neither" in fwd(p=p)
    assert b"act" in fwd(act=4) and b"dtype" in fwd(dt=-1)
    for bad in (dict(D=0), dict(F=0), dict(D=(1 << 20) + 1), dict(F=1 << 21), dict(M=1 << 31),
                dict(M=(1 << 29) + 1)):
        assert b"shape" in fwd(**bad)
    assert b"workspace" in fwd(wsb=63)
    for i in (0, 1, 2, 3, 6, 7):
        p = spread(8)
        p[i] = 0
        assert b"null" in fwd(p=p), i
    p = spread(8)
    p[6] = p[0]
    assert b"overlaps" in fwd(p=p)
    bwd = lambda dt=1, act=3, p=None, M=2, D=8, F=16, wsb=64, need=64: checks(  # noqa: E731
        "ffn_bwd", dt, act, p or spread(12), u(M), u(D), u(F), u(wsb), u(need))
    assert bwd() is None and b"workspace" in bwd(wsb=0)
    for i in range(12):
        p = spread(12)
        p[i] = 0
        assert b"null" in bwd(p=p), i
    p = spread(12)
    p[8] = p[9]
    assert b"overlaps" in bwd(p=p)
    p = spread(12)
    p[7] = p[6]  # dx over dy
    assert b"overlaps" in bwd(p=p)


def test_group_refusals(checks, hip):
    def table(**over):
        t = (hip.AdamWTensor * 2)()
        for i in range(2):
            for k, name in enumerate(("p", "g", "m", "v", "m_scale", "v_scale", "p_bf16")):
                setattr(t[i], name, ((i * 8 + k + 1) << 20))
            t[i].n, t[i].decay = 1000, 1.0
        for name, value in over.items():
            setattr(t[1], name, value)
        return t

    def ask(t, bits=32, g=0):
        return checks("group", t, u(len(t)), bits, g)
    assert ask(table()) is None and ask(table(), 8, 1) is None
    assert checks("group", None, u(0), 32, 0) is None
    assert b"state_bits" in ask(table(), 16) and b"grad_dtype" in ask(table(), 32, 2)
    assert b"null" in checks("group", None, u(1), 32, 0)
    for name in ("p", "g", "m", "v"):
        assert b"null" in ask(table(**{name: 0}))
        assert ask(table(**{name: 0, "n": 0})) is None
    assert ask(table(m_scale=0)) is None and b"null" in ask(table(m_scale=0), 8)
    assert ask(table(p_bf16=0), 8) is None
    assert b"alignment" in ask(table(p=(9 << 20) + 2))
    assert ask(table(m=(11 << 20) + 1), 8) is None
    assert b"decay" in ask(table(decay=float("nan"))) and b"decay" in ask(table(decay=-1.0))
    assert b"overlaps" in ask(table(p=1 << 20))  # the other tensor's p
    assert b"overlaps" in ask(table(g=3 << 20))  # reads what the other writes
    assert ask(table(g=2 << 20)) is None  # one gradient for both
    assert b"overlaps" in ask(table(v=(3 << 20) + 3996))
    assert ask(table(v=(3 << 20) + 4000)) is None
    assert b"large" in ask(table(n=1 << 36))


def test_workspace_sizes(hip):
    lib = hip.lib()
    assert lib.seeai_norm_bwd_workspace(0, 64) == 0
    assert 0 < lib.seeai_norm_bwd_workspace(8192, 2048) <= 16 << 20
    assert lib.seeai_norm_bwd_workspace(1, 0) == 0
    for dtype, size in ((0, 4), (1, 2)):
        for backward in (0, 1):
            assert lib.seeai_ffn_workspace(dtype, 64, 96, 160, backward) >= 64 * 160 * size
    assert lib.seeai_ffn_workspace(1, 4, 0, 8, 0) == 0
    assert lib.seeai_ffn_workspace(2, 4, 8, 8, 0) == 0


class Fake:
    """What the group's own checks ask of a tensor."""

    def __init__(self, n, size, contiguous=True, device=True):
        self.n, self.size, self.contiguous, self.is_cuda = n, size, contiguous, device

    def numel(self):
        return self.n

    def element_size(self):
        return self.size

    def is_contiguous(self):
        return self.contiguous

    def data_ptr(self):
        return 1 << 20


class Recorder:
    h = None

    def call(self, name, *args):
        raise LookupError(name)

    check = call


def test_group_wrapper_refuses_short_and_mistyped_tensors(hip):
    def make(bits=8, grads="f32", **over):
        t = {"p": Fake(300, 4), "g": Fake(300, 4), "m": Fake(300, 1), "v": Fake(300, 1),
             "m_scale": Fake(3, 4), "v_scale": Fake(3, 4), "p_bf16": Fake(300, 2)} | over
        return hip.AdamWGroup(Recorder(), [t], bits, grads)

    with pytest.raises(LookupError):  # complete: the call is made
        make()
    with pytest.raises(LookupError):
        make(g=Fake(300, 2), grads="bf16")
    with pytest.raises(LookupError):
        make(bits=32, m=Fake(300, 4), v=Fake(300, 4), m_scale=None, v_scale=None, p_bf16=None)
    for over in (dict(n=301), dict(g=Fake(299, 4)), dict(g=Fake(300, 2)), dict(m=Fake(300, 4)),
                 dict(v_scale=Fake(2, 4)), dict(p_bf16=Fake(300, 4)), dict(p=Fake(300, 4, False)),
                 dict(v=Fake(300, 1, True, False))):
        with pytest.raises(ValueError):
            make(**over)
    for over in (dict(bits=16), dict(grads="f16")):
        with pytest.raises(ValueError):
            make(**over)


def test_a_closed_group_refuses(hip):
    group = hip.AdamWGroup.__new__(hip.AdamWGroup)
    group.h, group.ctx = None, Recorder()
    for call in (group.step, lambda: group.hold(hip.StepParams())):
        with pytest.raises(hip.BackendError, match="closed"):
            call()


class Accepting(Recorder):
    """A context whose calls succeed."""

    def call(self, name, *args):
        return None


def test_a_group_keeps_the_tensors_it_was_made_of(hip):
    """The device's table holds addresses: what the caller does to its dicts afterwards must not
    free the memory behind them."""
    t = {"p": Fake(300, 4), "g": Fake(300, 4), "m": Fake(300, 4), "v": Fake(300, 4), "decay": 0.5}
    given = [t]
    group = hip.AdamWGroup(Accepting(), given, 32, "f32")
    p, g, m = t["p"], t["g"], t["m"]
    t["g"] = Fake(300, 4)
    del t["m"]
    given.clear()
    held = list(group.tensors[0].values())
    assert all(any(x is y for y in held) for x in (p, g, m, t["v"]))


class Typed(Fake):
    """A tensor that says its type, as a device tensor does."""

    def __init__(self, n, dtype):
        super().__init__(n, {"32": 4, "16": 2, "t8": 1, "fn": 1}[dtype[-2:]])
        self.dtype = "torch." + dtype


def test_group_wrapper_refuses_wrong_types_of_the_right_size(hip):
    def make(bits=8, grads="f32", **over):
        code = "uint8" if bits == 8 else "float32"
        types = {"p": "float32", "g": "float32" if grads == "f32" else "bfloat16", "m": code, "v": code,
                 "m_scale": "float32", "v_scale": "float32", "p_bf16": "bfloat16"} | over
        return hip.AdamWGroup(Accepting(), [{k: Typed(300, t) for k, t in types.items()}], bits, grads)

    for bits in (8, 32):
        for grads in ("f32", "bf16"):
            make(bits, grads)
    make(m="float8_e4m3fn", v="float8_e4m3fn")  # what the codes are
    make(g="int16", p_bf16="uint16", grads="bf16")  # bf16 bits
    for over in (dict(p="int32"), dict(g="int32"), dict(g="float16", grads="bf16"), dict(m="int8"),
                 dict(v="int8"), dict(m_scale="int32"), dict(v_scale="int32"), dict(p_bf16="float16"),
                 dict(m="int32", bits=32), dict(v="int32", bits=32)):
        with pytest.raises(ValueError, match=next(k for k in over if k not in ("grads", "bits"))):
            make(**over)


def test_group_wrapper_refuses_tensors_of_another_device(hip):
    """A step runs on its context's device; another device's memory may be out of its reach."""
    class At:
        def __init__(self, index):
            self.index = index

    def make(**over):
        t = {k: Typed(300, "float32") for k in ("p", "g", "m", "v")}
        for k, x in t.items():
            x.device = At(over.get(k, 1))
        ctx = Accepting()
        ctx.device_index = 1
        return hip.AdamWGroup(ctx, [t], 32, "f32")

    make()
    for name in ("p", "g", "m", "v"):
        with pytest.raises(ValueError, match=f"{name}: .*device 1"):
            make(**{name: 0})


def test_values_refusals(tmp_path):
    """As many values as one launch takes: a workgroup of 256 threads to 2048, below 2^32 threads."""
    src, lib = tmp_path / "v.cc", tmp_path / "v.so"
    src.write_text(r"""
#include "see-ai_amd/csrc/block_args.h"
extern "C" const char* values(int which, int dt, const uint64_t* p, uint64_t n) {
  return seeai::CheckAdamWValues(which, dt, reinterpret_cast<const void*>(p[0]),
                                 reinterpret_cast<const float*>(p[1]), n, reinterpret_cast<const void*>(p[2]));
}
""")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", f"-I{ROOT}", str(src), "-o", str(lib)], check=True)
    h = C.CDLL(str(lib))
    h.values.restype = C.c_char_p

    def ask(which=0, dt=0, p=(1 << 40, 2 << 40, 3 << 40), n=300):
        return h.values(which, dt, (C.c_uint64 * 3)(*p), u(n))
    assert ask() is None and ask(1, 1) is None and ask(n=0, p=(0, 0, 0)) is None
    assert b"which" in ask(2) and b"dtype" in ask(dt=2)
    most = ((1 << 24) - 1) * 2048
    assert ask(n=most) is None and most // 2048 * 256 < 1 << 32
    assert all(b"large" in ask(n=n) for n in (most + 1, (1 << 35) - 1, 1 << 35, 1 << 63, (1 << 64) - 1))
    for i in range(3):
        p = [1 << 40, 2 << 40, 3 << 40]
        p[i] = 0
        assert b"null" in ask(p=p)
    assert b"alignment" in ask(p=(1 << 40, (2 << 40) + 2, 3 << 40))
    assert b"overlaps" in ask(p=(1 << 40, 2 << 40, (1 << 40) + 256))
