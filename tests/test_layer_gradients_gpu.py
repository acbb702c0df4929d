"""Gradients of the layer operators: with parameters left out, and those that arrive at addresses which
are no whole vector, as a result gets that is joined with something of another size: a slice of the
joined tensor's gradient.

A copy changes no value, so the gradients are those of the same gradient at an aligned address, bit
for bit.
"""
import pytest
import torch

import fpscan_amd

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device (MI355X)"),
]

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def both(leaves, call):
    """The gradients of `leaves` for a slice from the second element on, and for its copy."""
    out = call()
    joined = torch.randn(out.numel() + 1, device="cuda").to(out.dtype)
    go = joined[1:].view(out.shape)
    assert go.is_contiguous() and go.data_ptr() % 16 != 0
    got = torch.autograd.grad(out, leaves, go)
    return got, torch.autograd.grad(call(), leaves, go.clone())


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_delta_gradient_of_a_slice(dtype):
    torch.manual_seed(1)
    B, L, Hk, H, D = 2, 70, 1, 2, 64
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)
    q, k = (unit(torch.randn(B, L, Hk, D, device="cuda")).to(dtype) for _ in range(2))
    v = torch.randn(B, L, H, D, device="cuda").to(dtype)
    g, beta = (s * torch.rand(B, L, H, device="cuda").to(dtype) for s in (-0.1, 1.0))
    leaves = [x.requires_grad_() for x in (q, k, v, g, beta)]
    for got, want in zip(*both(leaves, lambda: fpscan_amd.gated_delta(*leaves))):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seqlen", [1, 90])
def test_norm_gradient_of_a_slice(seqlen, dtype):
    torch.manual_seed(2)
    x, gate = (torch.randn(3, seqlen, 64, device="cuda").to(dtype).requires_grad_() for _ in range(2))
    weight = torch.randn(64, device="cuda").requires_grad_()
    call = lambda: fpscan_amd.group_norm_channel_last(x, 4, weight, gate=gate)
    for got, want in zip(*both([x, gate, weight], call)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("batch", [2, 16, 17])
def test_norm_parameters_left_out(batch):
    """A weight of ones and a bias of zeros change no value: the other one's gradient stays as it is."""
    torch.manual_seed(3)
    x = torch.randn(batch, 3000, 256, device="cuda").requires_grad_()
    weight = torch.randn(256, device="cuda").requires_grad_()
    bias = torch.randn(256, device="cuda").requires_grad_()
    ones, zeros = torch.ones(256, device="cuda"), torch.zeros(256, device="cuda")
    go = torch.randn_like(x)

    def grads(w, b, *leaves):
        return torch.autograd.grad(fpscan_amd.group_norm_channel_last(x, 4, w, b), leaves, go)

    for alone, both in ((grads(weight, None, x, weight), grads(weight, zeros, x, weight)),
                        (grads(None, bias, x, bias), grads(ones, bias, x, bias)),
                        (grads(None, None, x), grads(ones, zeros, x))):
        for got, want in zip(alone, both):
            assert torch.equal(got, want)
    x64 = x.detach().double().view(batch, 3000, 4, 64)
    h = x64 - x64.mean((1, 3), keepdim=True)
    h = (h / torch.sqrt(h.square().mean((1, 3), keepdim=True) + 1e-5)).view(x.shape)
    y = h * weight.detach().double() + bias.detach().double()
    s = torch.sigmoid(y)
    dy = go.double() * s * (1 + y * (1 - s))
    gw, gb = grads(weight, bias, weight, bias)
    # fp32 sums of up to 51000 terms, in parts whose errors add up like the square root of 2^8 terms a
    # thread, chunk or sequence, and the terms' own few 2^-23
    for got, want in ((gw, (dy * h).sum((0, 1))), (gb, dy.sum((0, 1)))):
        assert (got.double() - want).norm() <= 2.0 ** -18 * want.norm()
