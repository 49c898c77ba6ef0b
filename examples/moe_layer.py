"""A mixture-of-experts layer, trained for a few steps and then served.

    python examples/moe_layer.py

Training: route -> dispatch -> grouped products -> combine, with gradients in
the experts, the router and the input.  Serving: the experts' weights are
quantised to 4 bits and laid out once; single tokens go through the same
route, dispatch and combine, and the 4-bit products.  Prints the loss of each
step and how far the served answers are from the 16-bit layer's.
"""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import blackwell_gemm_b200 as bg  # noqa: E402


class MoELayer(torch.nn.Module):
    """out = sum over a token's top_k experts of w * down(silu(gate x) * up x)."""

    def __init__(self, width: int, hidden: int, experts: int, top_k: int,
                 dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        kw = dict(dtype=dtype, device=device)
        self.top_k, self.hidden = top_k, hidden
        self.router = torch.nn.Parameter(torch.randn(experts, width, **kw) * width ** -0.5)
        # gate and up projections of an expert in one matrix: one grouped product
        self.up = torch.nn.Parameter(torch.randn(experts, 2 * hidden, width, **kw) * width ** -0.5)
        self.down = torch.nn.Parameter(torch.randn(experts, width, hidden, **kw) * hidden ** -0.5)
        self.up4 = self.down4 = None

    def quantize(self, group: int = 128) -> None:
        """Lay the experts out in 4 bits; forward without gradients uses them."""
        self.up4 = bg.pack_w4(*bg.quantize_w4(self.up.detach(), group))
        self.down4 = bg.pack_w4(*bg.quantize_w4(self.down.detach(), group))

    def experts(self, x, offsets):
        serve = self.up4 is not None and not torch.is_grad_enabled()
        h = (bg.matmul_b200_w4(x, self.up4, offsets) if serve else
             bg.matmul_b200_grouped(x, self.up.transpose(1, 2), offsets))
        gate, up = h.split(self.hidden, dim=1)
        h = torch.nn.functional.silu(gate) * up
        return (bg.matmul_b200_w4(h, self.down4, offsets) if serve else
                bg.matmul_b200_grouped(h, self.down.transpose(1, 2), offsets))

    def forward(self, x):
        routing = bg.route_b200(x.float() @ self.router.float().T, self.top_k)
        y = self.experts(bg.dispatch_b200(x, routing), routing.offsets)
        return bg.combine_b200(y, routing)


def main(width=1024, hidden=2048, experts=16, top_k=2, tokens=2048, steps=8) -> dict:
    torch.manual_seed(0)
    layer = MoELayer(width, hidden, experts, top_k)
    optimizer = torch.optim.SGD(layer.parameters(), lr=0.5)
    x = torch.randn(tokens, width, device="cuda").bfloat16()
    target = torch.tanh(x.roll(1, dims=1))
    losses = []
    for _ in range(steps):
        optimizer.zero_grad(set_to_none=True)
        loss = torch.nn.functional.mse_loss(layer(x).float(), target.float(), reduction="sum") / tokens
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    losses = [float(v) for v in losses]
    with torch.no_grad():
        full = layer(x[:64])
        layer.quantize()
        batch = layer(x[:64])
        single = torch.cat([layer(x[i:i + 1]) for i in range(8)])   # a token at a time
    return {"losses": losses,
            "w4_off": float((batch.float() - full.float()).norm() / full.float().norm()),
            "single_off": float((single.float() - batch[:8].float()).norm() /
                                batch[:8].float().norm()),
            "device_status": bg.capi.device_status(True)}


if __name__ == "__main__":
    got = main()
    for i, v in enumerate(got["losses"]):
        print(f"step {i}: loss {v:.4f}")
    print(f"4-bit experts: relative distance {got['w4_off']:.3f} from the 16-bit layer; "
          f"one token at a time {got['single_off']:.2e} from the batch; "
          f"device error word {got['device_status']:#x}")
