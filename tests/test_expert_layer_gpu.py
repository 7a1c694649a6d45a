"""The example layer: the products as they are used together, against the layer written out in 64 bits."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def example():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    spec = importlib.util.spec_from_file_location("expert_layer", ROOT / "examples" / "expert_layer.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _written_out(torch, layer, x, topk):
    """The same layer, every expert on its own rows, in 64 bits (the routing as the layer has it: a
    different rounding of the router's logits may send a token elsewhere)."""
    with torch.no_grad():
        logits = (x @ layer.router.t()).float()
    weight, expert = torch.softmax(logits, -1).topk(topk, -1)
    weight = weight / weight.sum(-1, keepdim=True)
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for e in range(layer.gate_up.shape[0]):
        token, slot = (expert == e).nonzero(as_tuple=True)
        gate, up = (x[token].double() @ layer.gate_up[e].double().t()).chunk(2, -1)
        y = (torch.nn.functional.silu(gate) * up) @ layer.down[e].double().t()
        out = out.index_add(0, token, y * weight[token, slot][:, None].double())
    return out


def test_forward_backward_and_8_bits(handle, example):
    """FP32 weights, so that the layer is known to FP32 accuracy: five roundings in a row, each below 2^-22
    of sums whose terms cancel by no more than a factor of 2^6 in norm.  In 8 bits, steps of 1 / 127 of the
    largest of a row: about 1 % of noise for each of four operands."""
    import torch

    torch.manual_seed(1)
    layer = example.ExpertLayer(handle, 128, 192, 8, 2, dtype=torch.float32)
    x = torch.randn(301, 128, device="cuda", requires_grad=True)
    want = _written_out(torch, layer, x, 2)
    y = layer(x)
    assert (y.double() - want).norm() <= 5 * 2.0 ** -16 * want.norm()
    dy = torch.randn_like(y)
    params = [layer.gate_up, layer.down, x]
    got = torch.autograd.grad(y, params, dy)
    # (in `want` the router's weights are constants; x's gradient through them is left out on both sides)
    y = layer_with_fixed_routing(example, layer, x)
    got_x = torch.autograd.grad(y, x, dy)[0]
    exact = torch.autograd.grad(want, params, dy.double())
    for g, e in ((got[0], exact[0]), (got[1], exact[1]), (got_x, exact[2])):
        assert (g.double() - e).norm() <= 5 * 2.0 ** -16 * e.norm()
    serve = layer.quantised()
    assert (serve(x.detach()).double() - want).norm() <= 0.05 * want.norm()


def layer_with_fixed_routing(example, layer, x):
    import torch

    with torch.no_grad():
        fixed = example.route(x @ layer.router.t(), layer.topk)
    route, example.route = example.route, lambda logits, topk: fixed
    try:
        return layer(x)
    finally:
        example.route = route


def test_a_token_whose_experts_are_all_one_and_experts_without_tokens(handle, example):
    import torch

    torch.manual_seed(2)
    layer = example.ExpertLayer(handle, 64, 64, 16, 1, dtype=torch.bfloat16)
    x = torch.randn(1, 64, device="cuda", dtype=torch.bfloat16)
    y = layer(x)
    assert (y.double() - _written_out(torch, layer, x, 1)).norm() <= 0.02 * y.double().norm()
    y.float().sum().backward()
    used = layer.down.grad.flatten(1).abs().sum(1) > 0
    assert int(used.sum()) == 1
