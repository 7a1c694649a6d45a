"""Quantised rows against the formula as the header states it, each step rounded to FP32."""
import pytest

pytestmark = pytest.mark.gpu


def _formula(torch, x):
    """(q, scale) of rows with a normal, finite scale.  (Divisions of tensors: one rounding each.)"""
    x = x.float()
    top = x.abs().amax(1)
    c = torch.full_like(top, 127.0)
    return torch.round(x * (c / top)[:, None]).to(torch.int8), top / c


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,k", [(40, 900), (2000, 512), (700, 2048), (700, 8192), (30, 9000)])
def test_every_integer_is_the_formula_s(handle, dtype, rows, k):
    """Whole numbers: they have to be equal.  (Every kernel: a warp for a row, a block, rows read twice.)"""
    import torch

    from cumpsgemm_b200 import experts

    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(rows + k)
    x = torch.randn(rows, k, generator=g, device="cuda").to(dt)
    x[:, ::7] = x.abs().amax(1, keepdim=True) / 2  # halves: 63.5 of 127
    x[:, 1::7] = -x.abs().amax(1, keepdim=True) / 2
    q, scale = experts.quantize_rows(handle, x)
    want, want_scale = _formula(torch, x)
    assert torch.equal(q, want), int((q != want).sum())
    assert torch.equal(scale, want_scale)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_halves_go_to_the_even_neighbour(handle, dtype):
    """top = 381: 127 / top is 1 / 3, which FP32 rounds up, and 3 j + 1.5 is the half j + 0.5."""
    import torch

    from cumpsgemm_b200 import experts

    j = torch.arange(-126, 126, device="cuda", dtype=torch.float32)
    x = torch.cat([3 * j + 1.5, torch.tensor([381.0], device="cuda")])[None].to(getattr(torch, dtype))
    q, _ = experts.quantize_rows(handle, x)
    assert torch.equal(q[0, :-1].float(), torch.round(j + 0.5)) and q[0, -1] == 127


def test_rows_at_the_bottom_of_the_range(handle):
    """scale * q is the row to half a step, and where the scale is subnormal to 127 / 2 of its smallest unit
    more.  A row whose scale rounds to zero has zeros."""
    import torch

    from cumpsgemm_b200 import experts

    tops = [2.0 ** e * f for e in range(-149, -110) for f in (1.0, 1.5)]
    g = torch.Generator(device="cuda").manual_seed(9)
    part = torch.rand(len(tops), 300, generator=g, device="cuda") * 2 - 1
    part[:, 11] = 1
    x = (part.double() * torch.tensor(tops, dtype=torch.float64, device="cuda")[:, None]).float()
    q, scale = experts.quantize_rows(handle, x)
    back = scale.double()[:, None] * q.double()
    step = x.double().abs().amax(1, keepdim=True) / 127
    tol = step * (0.5 + 2.0 ** -16) + torch.where(step < 2.0 ** -126, 127 * 2.0 ** -150, 127 * 2.0 ** -24 * step)
    # (without a scale all that is left is the row itself, of at most 63 * 2^-149)
    assert ((back - x.double()).abs() <= torch.where(scale[:, None] == 0, x.double().abs(), tol)).all()
    assert (q[scale == 0] == 0).all() and (scale == 0).any() and (q[scale > 0][:, 11] == 127).all()
