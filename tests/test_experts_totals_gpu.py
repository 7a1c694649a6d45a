"""Running totals that fall back, where the operands are scaled by their largest element."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups", [4, 300])
@pytest.mark.parametrize("transpose_w", [False, True])
def test_weights_of_a_group_that_a_falling_total_empties_do_not_scale(handle, groups, transpose_w):
    """Group 2 of totals 100, 50, 80 is empty: its weights, 1e30, are not the largest there are.  Bit for bit
    what the totals say that it is taken as."""
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from cumpsgemm_b200 import api, experts

    rows, n, k = 7 * groups + 200, 40, 64
    g = torch.Generator(device="cuda").manual_seed(groups)
    x = torch.randn(rows, k, generator=g, device="cuda")
    w = torch.randn(groups, *((n, k) if transpose_w else (k, n)), generator=g, device="cuda")
    w[1:3] = 1e30
    good = [100, 100, 100] + [100 + i + 1 for i in range(groups - 3)]
    bad = [100, 50, 80] + good[3:]
    dy = torch.randn(rows, n, generator=g, device="cuda")
    x[good[-1]:] = 1e25  # rows of no group scale nothing either
    results = []
    for totals in (good, bad):
        ends = torch.tensor(totals, dtype=torch.int32, device="cuda")
        mode = api.ComputeMode.FP16TCEC_SCALING
        results.append((experts.grouped_matmul(handle, x, w, ends, transpose_w, mode=mode),
                        experts.grouped_matmul_wgrad(handle, x, dy, ends, transpose_w, mode=mode)))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    first = x[:100].double() @ (w[0].double().t() if transpose_w else w[0].double())
    assert ((results[1][0][:100].double() - first).norm() <= 2.0 ** -16 * first.norm())
