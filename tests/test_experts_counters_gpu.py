"""What grouped products count tiles and slices with: zero behind every call, and again once a raised status
word has been read."""
import pytest

pytestmark = pytest.mark.gpu


def test_a_raised_status_word_takes_the_counts_with_it(handle):
    """The words filled as a kernel that gave up may leave them (by a copy: none gives up here): reading the
    status word sets them to zero, and the next product, few tiles cut into slices, is the same bit for bit."""
    import torch

    from cumpsgemm_b200 import experts

    x = torch.randn(70, 5000, device="cuda").to(torch.bfloat16)
    w = torch.randn(2, 5000, 200, device="cuda").to(torch.bfloat16)
    ends = torch.tensor([30, 70], dtype=torch.int32, device="cuda")
    product = lambda: experts.grouped_matmul(handle, x, w, ends)  # noqa: E731
    first = product()
    assert handle.selftest_grouped_counters() == 0
    assert torch.equal(first, product())
    assert handle.selftest_grouped_counters(1) == 0
    assert handle.selftest_grouped_counters() > 1000  # all of them, for 16 warps of every pair of CTAs
    assert handle.kernel_status() == 8
    assert handle.selftest_grouped_counters() == 0
    assert torch.equal(first, product())
    assert handle.kernel_status() == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("counts", [[1], [0, 700, 3], [40] * 30, [0, 0]])
def test_every_call_leaves_the_counts_at_zero(handle, dtype, counts):
    import torch

    from cumpsgemm_b200 import experts

    dt = getattr(torch, dtype)
    rows = sum(counts) + 70  # more than the kernel for few FP32 rows takes, and some of no expert
    x, dy = torch.randn(rows, 4200, device="cuda").to(dt), torch.randn(rows, 130, device="cuda").to(dt)
    w = torch.randn(len(counts), 4200, 130, device="cuda").to(dt)
    ends = torch.tensor(counts).cumsum(0).to(torch.int32).cuda()
    for call in (lambda: experts.grouped_matmul(handle, x, w, ends),
                 lambda: experts.grouped_matmul_wgrad(handle, x, dy, ends)):
        call()
        assert handle.selftest_grouped_counters() == 0
