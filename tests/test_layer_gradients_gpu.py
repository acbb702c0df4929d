"""Gradients of the layer operators that arrive at addresses which are no whole vector: a result that
is joined with something of another size gets a slice of the joined tensor's gradient.

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
