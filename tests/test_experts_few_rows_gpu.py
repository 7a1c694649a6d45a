"""FP32 products with few rows for each group on average, and very differently many in fact: groups of more rows
than a block takes at a time.  FP32 arithmetic, k + 16 roundings of at most 2^-24 of the sum of magnitudes."""
import pytest

pytestmark = pytest.mark.gpu

UNEVEN = [
    [384] + [0] * 63,                       # all in one group, the first or the last
    [0] * 63 + [384],
    [100, 0, 9, 8, 17, 16, 1] + [2] * 57,   # more chunks than groups with rows
    [0] * 255 + [1000, 1] + [0] * 43,       # groups that share a thread
    [7] * 500 + [0] * 300 + [15] * 150 + [1] * 74,
    [9, 9],                                 # (six rows on average with the rows of no group left out)
]


@pytest.mark.parametrize("transpose_w", [False, True])
@pytest.mark.parametrize("counts", UNEVEN)
@pytest.mark.parametrize("n,k", [(70, 90), (300, 64)])
def test_uneven_groups(handle, transpose_w, counts, n, k):
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from cumpsgemm_b200 import experts

    groups = max(len(counts), -(-(sum(counts) + 20) // 6))
    counts = counts + [0] * (groups - len(counts))
    rows = sum(counts) + 20  # twenty rows of no group
    assert rows <= 6 * groups and groups <= 1024
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(rows, k, generator=g, device="cuda")
    x[sum(counts):] = float("nan")
    w = torch.randn(groups, *((n, k) if transpose_w else (k, n)), generator=g, device="cuda")
    w[torch.tensor(counts, device="cuda") == 0] = float("nan")
    y0 = torch.randn(rows, n, generator=g, device="cuda")
    ends = torch.tensor(counts).cumsum(0)
    falling = ends.clone()  # totals that fall back behind a group count as the one in front of it
    empty = (torch.tensor(counts) == 0).nonzero()[:, 0]
    falling[empty] = falling[empty] // 2 - 3
    want, size = torch.zeros(2, rows, n, dtype=torch.float64, device="cuda")
    at = 0
    for e, c in enumerate(counts):
        if c:
            we = w[e].double().t() if transpose_w else w[e].double()
            want[at:at + c] = x[at:at + c].double() @ we
            size[at:at + c] = x[at:at + c].double().abs() @ we.abs()
        at += c
    for totals in (ends, falling):
        totals = totals.to(torch.int32).cuda()
        y = experts.grouped_matmul(handle, x, w, totals, transpose_w)
        assert ((y.double() - want).abs() <= (k + 16) * 2.0 ** -24 * size).all()
        assert (y[sum(counts):] == 0).all()
    y = y0.clone()
    experts.grouped_matmul(handle, x, w, totals, transpose_w, alpha=2.0, beta=-0.5, out=y)
    tol = (k + 18) * 2.0 ** -24 * (2.0 * size + 0.5 * y0.double().abs())
    assert ((y.double() - (2.0 * want - 0.5 * y0.double())).abs() <= tol).all()


@pytest.mark.parametrize("transpose_w", [False, True])
def test_rows_in_one_group_take_no_longer_than_the_same_rows_in_all(handle, transpose_w):
    """Less has to be read for them.  (Several times as long where one group's rows queue up; half as long
    where they are spread.)"""
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from cumpsgemm_b200 import experts

    groups, each, n, k = 128, 4, 512, 1024
    x = torch.randn(groups * each, k, device="cuda")
    w = torch.randn(groups, *((n, k) if transpose_w else (k, n)), device="cuda")

    def best(counts):
        ends = torch.tensor(counts).cumsum(0).to(torch.int32).cuda()
        times = []
        for _ in range(8):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            for _ in range(5):
                experts.grouped_matmul(handle, x, w, ends, transpose_w)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    assert best([0] * 77 + [groups * each] + [0] * 50) <= 1.5 * best([each] * groups)
