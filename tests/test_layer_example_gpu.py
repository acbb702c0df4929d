"""examples/gated_delta_layer.py: the gated delta rule and the group norm together, trained and served."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device (MI355X)"),
]


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location(
        "gated_delta_layer", os.path.join(ROOT, "examples", "gated_delta_layer.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_recall_is_learned_and_decoding_agrees(example):
    """Eight values: a guess costs log 8 = 2.08. Prompt and decoding run the same rule in other chunks
    and with other operand roundings, each output rounded to bf16 three times on its way: a few 2^-8."""
    model, losses = example.train(steps=150, verbose=False)
    assert losses[0] > 1.8 and sum(losses[-10:]) / 10 < 1.0
    assert example.decode_difference(model) < 4 * 2.0 ** -8


def test_shared_key_heads_in_fp32(example):
    """The layer with keys shared by two heads: its gradient along a direction against a difference."""
    torch.manual_seed(0)
    layer = example.GatedDeltaLayer(64, 4, 32, key_heads=2, dtype=torch.float32)
    x = torch.randn(2, 100, 64, device="cuda", requires_grad=True)
    go, d = torch.randn(2, 100, 64, device="cuda"), torch.randn(2, 100, 64, device="cuda")
    grad = torch.autograd.grad(layer(x), x, go)[0]
    with torch.no_grad():
        h = 1e-2  # the difference's own error is of order h^2 = 1e-4, fp32's 1e-7 / h = 1e-5
        want = ((layer(x + h * d) - layer(x - h * d)).double() * go).sum() / (2 * h)
    terms = grad.double() * d
    assert abs(float(terms.sum() - want)) < 5e-3 * float(terms.norm())
