"""The example layer: gradients against the same layer in elementary 64-bit
operations, training that lowers the loss, and serving with 4-bit experts."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parents[1] / "examples" / "moe_layer.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("moe_layer_example", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain(layer, x):
    """The layer token by token over the chosen experts, in 64 bits."""
    logits = x @ layer["router"].T
    top, idx = torch.sort(logits, dim=1, descending=True, stable=True)
    k = layer["top_k"]
    w, idx = torch.softmax(top[:, :k], 1), idx[:, :k]
    out = torch.zeros_like(x)
    for e in range(layer["up"].shape[0]):
        gate, up = (x @ layer["up"][e].T).split(layer["hidden"], 1)
        y = (torch.nn.functional.silu(gate) * up) @ layer["down"][e].T
        out = out + y * torch.where(idx == e, w, 0).sum(1, keepdim=True)
    return out


def test_gradients_of_the_layer(example):
    torch.manual_seed(1)
    layer = example.MoELayer(128, 192, 8, 2)
    x = torch.randn(75, 128, device="cuda").bfloat16().requires_grad_(True)
    c = torch.randn(75, 128, device="cuda").bfloat16()
    got = torch.autograd.grad((layer(x) * c).sum(), (x, layer.router, layer.up, layer.down))
    wide = {n: getattr(layer, n).detach().double().requires_grad_(True)
            for n in ("router", "up", "down")}
    xd = x.detach().double().requires_grad_(True)
    out = plain({**wide, "top_k": 2, "hidden": 192}, xd)
    want = torch.autograd.grad((out * c.double()).sum(), (xd, *wide.values()))
    # each of the chain's about ten 16-bit roundings is within 2^-8 of its value
    for g, v in zip(got, want):
        assert float((g.double() - v).norm() / v.norm()) <= 10 * 2.0 ** -8


def test_training_and_serving(example):
    got = example.main(width=256, hidden=256, experts=8, top_k=2, tokens=512, steps=6)
    assert got["losses"][-1] < got["losses"][0]
    assert got["device_status"] == 0
    # 4-bit weights: 7 steps each way, off by up to half of one; rms 1/sqrt(12)
    # of a step against weights of rms about 7/3 steps (normal, 128 to a
    # group), over two products in a row: well within a quarter
    assert got["w4_off"] < 0.25
    # one token alone: the same sums in another order, rounded to bf16 per product
    assert got["single_off"] <= 4 * 2.0 ** -8
