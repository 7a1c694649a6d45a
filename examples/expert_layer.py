"""A mixture-of-experts layer on the grouped products: training steps, then the same weights in 8 bits, integer and
floating point.

Each token goes to ``topk`` of the experts; an expert is a gated feed-forward block,
``(silu(x gate^T) * (x up^T)) down^T``.  The tokens' rows are sorted by expert on the device, and nothing
waits for the number of rows that an expert gets.

    python examples/expert_layer.py            # on a B200
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from cumpsgemm_b200 import api, experts  # noqa: E402


def route(logits, topk):
    """The rows of the experts' products: the token of each, sorted by expert, the weight it comes back with,
    and the running total of rows after each expert."""
    weight, expert = torch.softmax(logits.float(), -1).topk(topk, -1)
    weight = weight / weight.sum(-1, keepdim=True)
    expert, order = torch.sort(expert.flatten(), stable=True)
    ends = torch.searchsorted(expert, torch.arange(logits.shape[1], device=logits.device), right=True)
    return order // topk, weight.flatten()[order], ends.to(torch.int32)


class ExpertLayer(torch.nn.Module):
    def __init__(self, handle, width, hidden, num_experts, topk, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.handle, self.topk = handle, topk
        new = lambda *shape, fan: torch.nn.Parameter(  # noqa: E731
            torch.randn(*shape, device=device, dtype=torch.float32).mul_(fan ** -0.5).to(dtype))
        self.router = new(num_experts, width, fan=width)
        self.gate_up = new(num_experts, 2 * hidden, width, fan=width)
        self.down = new(num_experts, width, hidden, fan=hidden)

    def forward(self, x):
        tokens, weight, ends = route(x @ self.router.t(), self.topk)
        y = experts.gated_feed_forward(self.handle, x[tokens], self.gate_up, self.down, ends)
        return torch.zeros_like(x).index_add_(0, tokens, y * weight[:, None].to(y.dtype))

    @torch.no_grad()
    def quantised_f8(self):
        """The layer's forward pass in 8-bit floating point: weights with a scale for each 128 x 128, activations with
        one for each 128 columns of a row."""
        gate_up, down = (experts.quantize_weight_blocks(self.handle, w) for w in (self.gate_up, self.down))
        router, topk, handle = self.router.detach().clone(), self.topk, self.handle

        @torch.no_grad()
        def forward(x):
            tokens, weight, ends = route(x @ router.t(), topk)
            q, scale = experts.quantize_blocks(handle, x, row_index=tokens.to(torch.int32))
            q, scale = experts.f8_gated_matmul(handle, q, scale, *gate_up, ends)
            y = experts.f8_matmul(handle, q, scale, *down, ends, out_dtype=x.dtype)
            return torch.zeros_like(x).index_add_(0, tokens, y * weight[:, None].to(y.dtype))

        return forward

    @torch.no_grad()
    def quantised(self):
        """The layer's forward pass with 8-bit integer weights and activations."""
        def channels(w):
            q, scale = experts.quantize_rows(self.handle, w.flatten(0, 1))
            return q.unflatten(0, w.shape[:2]), scale.view(w.shape[:2])

        gate_up, gate_up_scale = channels(self.gate_up)
        down, down_scale = channels(self.down)
        router, topk, handle = self.router.detach().clone(), self.topk, self.handle

        @torch.no_grad()
        def forward(x):
            tokens, weight, ends = route(x @ router.t(), topk)
            q, scale = experts.quantize_rows(handle, x, row_index=tokens.to(torch.int32))
            h = experts.i8_matmul(handle, q, scale, gate_up, gate_up_scale, ends, out_dtype=x.dtype)
            gate, up = h.chunk(2, -1)
            q, scale = experts.quantize_rows(handle, torch.nn.functional.silu(gate) * up)
            y = experts.i8_matmul(handle, q, scale, down, down_scale, ends, out_dtype=x.dtype)
            return torch.zeros_like(x).index_add_(0, tokens, y * weight[:, None].to(y.dtype))

        return forward


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=4096)
    ap.add_argument("--width", type=int, default=1024)
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--experts", type=int, default=16)
    ap.add_argument("--topk", type=int, default=2)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    torch.manual_seed(0)
    with api.Handle() as handle:
        handle.use_current_torch_stream()
        teacher = ExpertLayer(handle, a.width, a.hidden, a.experts, a.topk)
        layer = ExpertLayer(handle, a.width, a.hidden, a.experts, a.topk)
        layer.load_state_dict(teacher.state_dict())
        with torch.no_grad():
            for w in (layer.gate_up, layer.down):
                w.add_(torch.randn_like(w), alpha=0.3 * w.float().std().item())
        optimiser = torch.optim.AdamW(layer.parameters(), lr=1e-3, weight_decay=0.0)
        for step in range(a.steps):
            x = torch.randn(a.tokens, a.width, device="cuda", dtype=torch.bfloat16)
            with torch.no_grad():
                target = teacher(x)
            loss = (layer(x) - target).float().square().mean()
            optimiser.zero_grad()
            loss.backward()
            optimiser.step()
            if step % 5 == 0 or step == a.steps - 1:
                print(f"step {step:3d}  loss {loss.item():.5f}")
        x = torch.randn(a.tokens, a.width, device="cuda", dtype=torch.bfloat16)
        with torch.no_grad():
            full = layer(x).float()
        for name, serve in (("integer", layer.quantised()), ("floating-point", layer.quantised_f8())):
            off = (serve(x).float() - full).norm() / full.norm()
            print(f"8-bit {name} layer against bfloat16: relative difference {off.item():.4f}")
        if handle.kernel_status() != 0:
            raise SystemExit("a kernel gave up waiting")


if __name__ == "__main__":
    main()
