"""C ABI of the gated delta rule and the group norm on the CPU: arguments are refused on the host,
before any HIP call, and workspaces are what the layouts add up to."""
import ctypes
import os
import re

import pytest

from conftest import ROOT

HEADER = os.path.join(ROOT, "include", "fpscan_hip.h")
LIB = os.path.join(ROOT, "fpscan_amd", "libfpscan_hip.so")
vp, i64, c_int, size_t = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t
FAKE = 1 << 20
BIG = 1 << 60


class Heads(ctypes.Structure):
    _fields_ = [("data", vp), ("stride_b", i64), ("stride_t", i64), ("stride_h", i64)]


class Delta(ctypes.Structure):
    _fields_ = [(n, i64) for n in ("batch", "seqlen", "key_heads", "heads", "key_dim", "value_dim")] + [
        ("dtype", c_int), ("scale", ctypes.c_float)] + [
        (n, Heads) for n in ("q", "k", "v", "log_decay", "beta")]


class Norm(ctypes.Structure):
    _fields_ = [(n, i64) for n in ("batch", "seqlen", "dim", "groups")] + [
        ("dtype", c_int), ("activation", c_int), ("eps", ctypes.c_float)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB)
    pd, pn, ph = ctypes.POINTER(Delta), ctypes.POINTER(Norm), ctypes.POINTER(Heads)
    lib.fpscan_delta_workspace_bytes.argtypes = [pd, c_int]
    lib.fpscan_delta_workspace_bytes.restype = size_t
    lib.fpscan_delta_fwd.argtypes = [pd, vp, vp, vp, size_t, vp]
    lib.fpscan_delta_fwd_saved.argtypes = [pd, vp, vp, size_t, vp]
    lib.fpscan_delta_bwd.argtypes = [pd, ph, vp, size_t, vp, vp, vp, vp, vp, vp, size_t, vp]
    lib.fpscan_delta_step.argtypes = [pd, vp, vp, vp, i64, vp]
    lib.fpscan_norm_workspace_bytes.argtypes = [pn, c_int]
    lib.fpscan_norm_workspace_bytes.restype = size_t
    lib.fpscan_norm_fwd.argtypes = [pn, vp, vp, vp, vp, vp, vp, vp, size_t, vp]
    lib.fpscan_norm_bwd.argtypes = [pn] + [vp] * 11 + [size_t, vp]
    return lib


@pytest.fixture(scope="module")
def d():
    text = open(HEADER).read()
    return {m.group(1): int(m.group(2)) for m in re.finditer(r"#define\s+(FPSCAN_\w+)\s+(\d+)", text)}


def delta(batch=2, seqlen=100, key_heads=2, heads=4, key_dim=64, value_dim=64, dtype=2, **change):
    p = Delta(batch, seqlen, key_heads, heads, key_dim, value_dim, dtype, 0.125)
    for n, h, dim in (("q", key_heads, key_dim), ("k", key_heads, key_dim), ("v", heads, value_dim),
                      ("log_decay", heads, 1), ("beta", heads, 1)):
        setattr(p, n, Heads(FAKE, seqlen * h * dim, h * dim, dim))
    for n, v in change.items():
        name, field = n.split("__")
        setattr(getattr(p, name), field, v)
    return p


def calls(lib, p):
    go = ctypes.byref(Heads(FAKE, 64 * 400, 64 * 4, 64))
    return [lib.fpscan_delta_fwd(p, FAKE, FAKE, FAKE, BIG, None),
            lib.fpscan_delta_fwd_saved(p, FAKE, FAKE, BIG, None),
            lib.fpscan_delta_bwd(p, go, FAKE, BIG, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, BIG, None),
            lib.fpscan_delta_step(p, FAKE, FAKE, None, 1 << 20, None)]


@pytest.mark.parametrize("change, error", [
    (dict(dtype=3), "DTYPE"), (dict(batch=-1), "SHAPE"), (dict(key_heads=3), "SHAPE"),
    (dict(key_dim=60), "SHAPE"), (dict(key_dim=136), "SHAPE"), (dict(key_dim=0), "SHAPE"),
    (dict(value_dim=4), "SHAPE"), (dict(value_dim=4104), "SHAPE"), (dict(key_heads=0), "SHAPE"),
    (dict(batch=1 << 20, seqlen=1 << 30), "SHAPE"), (dict(q__data=None), "NULL"),
    (dict(v__data=FAKE + 8), "ALIGN"), (dict(k__stride_t=132), "ALIGN"), (dict(k__stride_t=32), "SHAPE"),
    (dict(q__stride_b=-8), "SHAPE"), (dict(v__stride_t=1 << 24), "SHAPE"),
    (dict(beta__data=FAKE + 1), "ALIGN"), (dict(v__stride_b=1 << 47), "SHAPE"),
])
def test_delta_refuses(lib, d, change, error):
    assert calls(lib, ctypes.byref(delta(**change))) == [d["FPSCAN_ERR_" + error]] * 4


def test_delta_refuses_null_misaligned_and_short_workspaces(lib, d):
    p = ctypes.byref(delta())
    null, align, short = (d["FPSCAN_ERR_" + n] for n in ("NULL", "ALIGN", "WORKSPACE"))
    assert lib.fpscan_delta_fwd(None, FAKE, FAKE, FAKE, BIG, None) == null
    assert lib.fpscan_delta_fwd(p, None, FAKE, FAKE, BIG, None) == null
    assert lib.fpscan_delta_fwd(p, FAKE, FAKE + 4, FAKE, BIG, None) == align
    for op, call in ((0, lambda n: lib.fpscan_delta_fwd(p, FAKE, FAKE, FAKE, n, None)),
                     (2, lambda n: lib.fpscan_delta_fwd_saved(p, FAKE, FAKE, n, None))):
        assert call(lib.fpscan_delta_workspace_bytes(p, op) - 1) == short
    go = Heads(FAKE, 64 * 400, 64 * 4, 64)
    bwd = lambda h, s, w: lib.fpscan_delta_bwd(p, ctypes.byref(h), FAKE, s, FAKE, FAKE, FAKE, FAKE, FAKE,
                                               FAKE, w, None)  # noqa: E731
    assert bwd(go, lib.fpscan_delta_workspace_bytes(p, 2) - 1, BIG) == short
    assert bwd(go, BIG, lib.fpscan_delta_workspace_bytes(p, 1) - 1) == short
    assert bwd(Heads(FAKE + 2, 64 * 400, 64 * 4, 64), BIG, BIG) == align
    assert bwd(Heads(FAKE, 0, 0, 0), BIG, BIG) == d["FPSCAN_ERR_SHAPE"]
    assert lib.fpscan_delta_step(p, FAKE, FAKE, None, 1, None) == d["FPSCAN_ERR_SHAPE"]
    assert lib.fpscan_delta_step(p, FAKE, FAKE, FAKE + 2, 9, None) == align
    assert lib.fpscan_delta_step(p, FAKE, None, None, 9, None) == null


def test_delta_with_nothing_to_do(lib):
    for change in (dict(batch=0), dict(seqlen=0), dict(heads=0, key_heads=0)):
        p = ctypes.byref(delta(**change))
        assert calls(lib, p) == [0] * 4
        assert [lib.fpscan_delta_workspace_bytes(p, op) for op in (0, 1, 2)] == [0] * 3


def norm(batch=2, seqlen=100, dim=64, groups=4, dtype=2, activation=1, eps=1e-5):
    return ctypes.byref(Norm(batch, seqlen, dim, groups, dtype, activation, eps))


@pytest.mark.parametrize("change, error", [
    (dict(dtype=3), "DTYPE"), (dict(batch=-1), "SHAPE"), (dict(groups=5), "SHAPE"),
    (dict(groups=0), "SHAPE"), (dict(dim=60), "SHAPE"), (dict(dim=8200, groups=1), "SHAPE"),
    (dict(activation=2), "SHAPE"), (dict(batch=1 << 45), "SHAPE"),
])
def test_norm_refuses(lib, d, change, error):
    p = norm(**change)
    assert lib.fpscan_norm_fwd(p, FAKE, None, None, None, FAKE, None, FAKE, BIG, None) == \
        d["FPSCAN_ERR_" + error]
    assert lib.fpscan_norm_bwd(p, FAKE, None, None, None, FAKE, FAKE, FAKE, None, None, None, FAKE, BIG,
                               None) == d["FPSCAN_ERR_" + error]


def test_norm_refuses_pointers_and_short_workspaces(lib, d):
    null, align, short = (d["FPSCAN_ERR_" + n] for n in ("NULL", "ALIGN", "WORKSPACE"))
    for p in (norm(seqlen=5000), norm(seqlen=1)):
        fwd = lambda x=FAKE, w=None, out=FAKE, n=BIG: lib.fpscan_norm_fwd(  # noqa: E731
            p, x, w, None, None, out, None, FAKE, n, None)
        bwd = lambda stats=FAKE, gate=None, gx=FAKE, n=BIG: lib.fpscan_norm_bwd(  # noqa: E731
            p, FAKE, None, None, gate, stats, FAKE, gx, None, None, None, FAKE, n, None)
        assert fwd(x=None) == null and fwd(out=None) == null and bwd(stats=None) == null
        assert bwd(gate=FAKE) == null  # no place for the gate's gradient
        assert fwd(x=FAKE + 8) == align and fwd(w=FAKE + 2) == align and bwd(gx=FAKE + 4) == align
        assert bwd(n=lib.fpscan_norm_workspace_bytes(p, 1) - 1) == short
    p = norm(seqlen=5000)
    assert lib.fpscan_norm_fwd(p, FAKE, None, None, None, FAKE, None, FAKE,
                               lib.fpscan_norm_workspace_bytes(p, 0) - 1, None) == short
    for p in (norm(batch=0), norm(seqlen=0), norm(dim=0)):
        assert lib.fpscan_norm_workspace_bytes(p, 0) == lib.fpscan_norm_workspace_bytes(p, 1) == 0
        assert lib.fpscan_norm_fwd(p, None, None, None, None, None, None, None, 0, None) == 0
