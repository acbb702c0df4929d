"""Group norms of so many short sequences that one workgroup for each sequence's sums would pass the 2^32
threads of a launch, against the definition in float64.

Tolerances, relative in the 2-norm: the rounding to fp16 is at most 2^-11 of each value; a parameter's
gradient is an fp32 sum of 2^19 sequences, 2^13 terms in a row to a thread, whose errors add up like
their square root: 2^-24 * 2^6.5, taken four times.
"""
import pytest
import torch

import fpscan_amd

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device (MI355X)"),
]

TOL = 2.0 ** -11 + 1e-5


def norm(x, groups, weight):
    B, L, D = x.shape
    x = x.view(B, L, groups, -1)
    x = x - x.mean((1, 3), keepdim=True)
    y = (x / torch.sqrt(x.square().mean((1, 3), keepdim=True) + 1e-5)).reshape(B, L, D) * weight
    return y * torch.sigmoid(y)


def error(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


def test_gradients():
    torch.manual_seed(3)
    x = torch.randn((1 << 19) + 3, 2, 64, device="cuda").half().requires_grad_()
    weight = (1 + 0.2 * torch.randn(64, device="cuda")).requires_grad_()
    go = torch.randn_like(x)
    out = fpscan_amd.group_norm_channel_last(x, 4, weight)
    gx, gw = torch.autograd.grad(out, [x, weight], go)
    x64, w64 = x.detach().double().requires_grad_(), weight.detach().double().requires_grad_()
    want = norm(x64, 4, w64)
    wx, ww = torch.autograd.grad(want, [x64, w64], go.double())
    assert error(out.detach(), want.detach()) <= TOL
    assert error(gx, wx) <= TOL
    assert error(gw, ww) <= 4 * 2.0 ** -17.5


def test_a_group_per_channel():
    torch.manual_seed(4)
    x = torch.randn((1 << 20) + 3, 2, 64, device="cuda").half()
    weight = 1 + 0.2 * torch.randn(64, device="cuda")
    out = fpscan_amd.group_norm_channel_last(x, 64, weight)
    for part in (slice(0, 1 << 15), slice((1 << 19) - 5, (1 << 19) + 5), slice(1 << 20, None)):
        assert error(out[part], norm(x[part].double(), 64, weight.double())) <= TOL
