"""The example layer served in 8-bit floating point: the calls as they are used together, against the layer itself."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


def test_served_in_8_bit_floating_point(handle):
    """Five operands of 8 bits (tokens, two weights on the gate's side, what is between, the weights behind), each off by
    at most 2^-4 of an element and some half of that in the mean; the errors of a sum's terms are independent: 5^(1/2)
    2^-5 of the norm at most.  Sizes that are and that are not multiples of 128."""
    import torch

    spec = importlib.util.spec_from_file_location("expert_layer", ROOT / "examples" / "expert_layer.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(3)
    for width, hidden in ((256, 384), (200, 150)):
        layer = example.ExpertLayer(handle, width, hidden, 8, 2)
        x = torch.randn(301, width, device="cuda", dtype=torch.bfloat16)
        with torch.no_grad():
            full = layer(x).double()
        off = (layer.quantised_f8()(x).double() - full).norm() / full.norm()
        assert float(off) < 5 ** 0.5 * 2.0 ** -5
