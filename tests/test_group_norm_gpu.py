"""group_norm_channel_last against its definition in float64 on the CPU, gradients by autograd through
it and by differences.

Tolerances are relative in the 2-norm: a result's rounding is at most 2^-8 (bf16), 2^-11 (fp16) or
2^-24 (fp32) of each value; statistics and sums in fp32 add a few 2^-24 times the square root of the
terms' number of a thread, and the activation's exponential a few 2^-23.
"""
import math

import pytest
import torch

import fpscan_amd

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device (MI355X)"),
]

DEVICE = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
TOL = {torch.float32: 2e-6, torch.float16: 2.0 ** -11 + 1e-5, torch.bfloat16: 2.0 ** -8 + 1e-5}
PARAM_TOL = 4e-6


def inputs(B, L, D, dtype, gate, seed=0):
    gen = torch.Generator().manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=gen)

    t = {"x": (randn(B, L, D) + 0.5 * randn(D)).to(dtype), "weight": 1 + 0.2 * randn(D),
         "bias": 0.2 * randn(D)}
    if gate:
        t["gate"] = randn(B, L, D).to(dtype)
    return t, randn(B, L, D).to(dtype)


def norm(t, groups, activation="silu", eps=1e-5):
    x = t["x"].double()
    B, L, D = x.shape
    x = x.view(B, L, groups, -1)
    x = x - x.mean((1, 3), keepdim=True)
    y = (x / torch.sqrt(x.square().mean((1, 3), keepdim=True) + eps)).reshape(B, L, D)
    y = y * t["weight"].double() if "weight" in t else y
    y = y + t["bias"].double() if "bias" in t else y
    z = t["gate"].double() if "gate" in t else y
    act = z * torch.sigmoid(z) if activation else z
    return y * act if "gate" in t else act


def call(t, groups, activation="silu", eps=1e-5):
    return fpscan_amd.group_norm_channel_last(t["x"], groups, t.get("weight"), t.get("bias"),
                                              gate=t.get("gate"), activation=activation, eps=eps)


def check(got, want, tol, what):
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape, what
    norm = want.norm()
    err = (got - want).norm() / norm if norm > 0 else got.norm()
    assert err <= tol, f"{what}: {err:.3e} > {tol:.3e}"


def gradients(t, go, groups, activation="silu", dtype=None):
    names = list(t)
    ref = {n: x.double().requires_grad_() for n, x in t.items()}
    want = norm(ref, groups, activation)
    grads = torch.autograd.grad(want, [ref[n] for n in names], go.double())
    on = {n: x.to(DEVICE).requires_grad_() for n, x in t.items()}
    out = call(on, groups, activation)
    got = torch.autograd.grad(out, [on[n] for n in names], go.to(DEVICE))
    dtype = t["x"].dtype
    with torch.no_grad():
        check(call(on, groups, activation), want, TOL[dtype], "out without gradients")
    check(out, want, TOL[dtype], "out")
    for n, a, b in zip(names, got, grads):
        assert a.dtype == on[n].dtype
        check(a, b, PARAM_TOL if n in ("weight", "bias") else TOL[dtype], "grad_" + n)


SHAPES = [  # batch, seqlen, dim, groups
    (1, 1, 8, 1), (5, 1, 64, 4), (300, 1, 1024, 8), (70, 1, 776, 8), (33, 1, 96, 3), (9, 1, 4096, 1),
    (2, 2, 32, 4), (3, 100, 776, 8), (2, 1000, 64, 64), (1, 5000, 128, 1), (4, 257, 2048, 32),
    (2100, 3, 16, 2), (2, 777, 40, 5),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(shape, gate, dtype):
    *sizes, groups = shape
    t, go = inputs(*sizes, dtype, gate)
    gradients(t, go, groups)


@pytest.mark.parametrize("seqlen", [1, 90])
@pytest.mark.parametrize("left_out", [("weight",), ("bias",), ("weight", "bias")])
def test_without_parameters_or_activation(left_out, seqlen):
    for gate in (False, True):
        t, go = inputs(4, seqlen, 128, torch.float32, gate, seed=1)
        for n in left_out:
            del t[n]
        gradients(t, go, 4, None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_8192_half_or_4096_single_values(dtype):
    t, go = inputs(3, 1, 16384 // torch.empty((), dtype=dtype).element_size(), dtype, True, seed=2)
    gradients(t, go, 16)
    t, go = inputs(2, 20, 16384 // torch.empty((), dtype=dtype).element_size(), dtype, False, seed=2)
    gradients(t, go, 64)


@pytest.mark.parametrize("seqlen", [1, 3000])
def test_large_means_and_outliers_keep_the_variance(seqlen):
    """Means a thousand deviations from 0, and first values far from all others: the variance is
    of differences. A mean near 1000 is held to 2^-15 (half a spacing), 3e-5 of a deviation."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(2, seqlen, 256, generator=gen)
    for y in (x + 1000.0, torch.where(torch.arange(256) % 64 == 0, x + 3000.0, x)):
        t = {"x": y}
        check(call({"x": y.to(DEVICE)}, 4, None), norm(t, 4, None), 5e-5, "out")


@pytest.mark.parametrize("seqlen", [1, 64])
def test_constant_groups_give_the_bias(seqlen):
    t, _ = inputs(2, seqlen, 64, torch.bfloat16, False, seed=4)
    t["x"][:] = 3.0
    out = call({n: x.to(DEVICE) for n, x in t.items()}, 4, None)
    assert torch.equal(out.cpu(), t["bias"].to(torch.bfloat16).expand_as(out))


@pytest.mark.parametrize("seqlen", [1, 200])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_nan_stays_in_its_sequence_and_group(seqlen, bad):
    t, _ = inputs(3, seqlen, 64, torch.float32, False, seed=5)
    want = norm(t, 4)
    t["x"][1, seqlen // 2, 20] = bad
    out = call({n: x.to(DEVICE) for n, x in t.items()}, 4).cpu()
    touched = torch.zeros(3, 1, 64, dtype=torch.bool)
    touched[1, 0, 16:32] = True
    touched = touched.expand_as(out)
    assert torch.isnan(out[touched]).all()
    check(out[~touched], want[~touched], TOL[torch.float32], "the others")


def test_activation_at_its_ends():
    """A gate of +-100 and beyond: z / (1 + exp(-z)) is z or 0, with slopes 1 and 0."""
    t, go = inputs(2, 1, 64, torch.float32, True, seed=6)
    t["gate"][..., ::4] = 100.0
    t["gate"][..., 1::4] = -100.0
    t["gate"][..., 2::4] = -1e30
    gradients(t, go, 4)


def test_gradients_against_differences():
    t, go = inputs(2, 30, 32, torch.float32, True, seed=7)
    on = {n: x.to(DEVICE).requires_grad_() for n, x in t.items()}
    got = torch.autograd.grad(call(on, 4), list(on.values()), go.to(DEVICE))
    for i, n in enumerate(t):
        d = torch.randn(t[n].shape, generator=torch.Generator().manual_seed(8 + i), dtype=torch.float64)
        f = [(norm({**t, n: t[n].double() + s * 1e-5 * d}, 4) * go).sum() for s in (1, -1)]
        want, terms = float((f[0] - f[1]) / 2e-5), got[i].double().cpu() * d
        assert abs(float(terms.sum()) - want) <= 1e-4 * float(terms.norm()), n


@pytest.mark.parametrize("shape", [(300, 1, 256), (2, 700, 256)])
def test_repeats_bit_for_bit_and_other_streams(shape):
    t, go = inputs(*shape, torch.bfloat16, True, seed=9)
    on = {n: x.to(DEVICE).requires_grad_() for n, x in t.items()}
    go = go.to(DEVICE)

    def step():
        out = call(on, 8)
        return (out, *torch.autograd.grad(out, list(on.values()), go))

    first = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = step()
    torch.cuda.synchronize()
    for a, b, c in zip(first, step(), other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_expanded_gradient_and_empty():
    t, _ = inputs(2, 50, 64, torch.float32, False, seed=10)
    ref = t["x"].double().requires_grad_()
    want = torch.autograd.grad(norm({**t, "x": ref}, 4).sum(), ref)[0]
    on = {n: x.to(DEVICE).requires_grad_() for n, x in t.items()}
    check(torch.autograd.grad(call(on, 4).sum(), on["x"])[0], want, 2 * TOL[torch.float32], "grad_x")
    for shape in [(0, 5, 64), (2, 0, 64)]:
        x = torch.zeros(shape, device=DEVICE, requires_grad=True)
        w = torch.ones(64, device=DEVICE, requires_grad=True)
        out = fpscan_amd.group_norm_channel_last(x, 4, w)
        gx, gw = torch.autograd.grad(out.sum(), (x, w))
        assert gx.shape == x.shape and (gw == 0).all()


def test_refusals():
    x = torch.zeros(2, 3, 64, device=DEVICE)
    f = fpscan_amd.group_norm_channel_last
    for bad, match in [((x.cpu(), 4), "CUDA tensor"), ((x.double(), 4), "float16 or bfloat16"),
                       ((x[0], 4), "3-d"), ((x.transpose(1, 2), 3), "contiguous"), ((x, 5), "divide"),
                       ((x, 0), "divide"), ((x[..., :62].contiguous(), 2), "multiple of 4"),
                       ((x, 4, torch.ones(64, device=DEVICE).half()), "float32"),
                       ((x, 4, torch.ones(32, device=DEVICE)), "one value per channel"),
                       ((torch.zeros(1, 1, 8192, device=DEVICE), 1), "at most 4096")]:
        with pytest.raises(RuntimeError, match=match):
            f(*bad)
    with pytest.raises(RuntimeError, match="shape of x"):
        f(x, 4, gate=x[:1])
    with pytest.raises(RuntimeError, match="activation"):
        f(x, 4, activation="relu6")
    with pytest.raises(RuntimeError, match="eps"):
        f(x, 4, eps=-1.0)
