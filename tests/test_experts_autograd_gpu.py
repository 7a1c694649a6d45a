"""The grouped products under autograd, on the kernels: against the same expression in 64 bits."""
import pytest

pytestmark = pytest.mark.gpu

COUNTS = [30, 0, 77, 1]
SPARE = 5  # rows of no expert


def _case(dtype, transpose_w, n=64, k=96):
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from cumpsgemm_b200 import experts

    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(sum(COUNTS) + SPARE, k, generator=g, device="cuda").to(dtype).requires_grad_()
    shape = (n, k) if transpose_w else (k, n)
    w = torch.randn(len(COUNTS), *shape, generator=g, device="cuda").to(dtype).requires_grad_()
    return torch, experts, x, w, torch.tensor(COUNTS).cumsum(0).to(torch.int32).cuda()


def _in_64_bits(torch, x, w, transpose_w):
    """(x, w, y): copies in 64 bits and the product of them as autograd knows it."""
    x, w = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    parts, at = [], 0
    for e, c in enumerate(COUNTS):
        parts.append(x[at:at + c] @ (w[e].t() if transpose_w else w[e]))
        at += c
    parts.append(x.new_zeros(x.shape[0] - at, parts[0].shape[1]))
    return x, w, torch.cat(parts)


def _near(got, want, limit):
    off = (got.double() - want).norm() / want.norm()
    assert off <= limit, float(off)


@pytest.mark.parametrize("dtype,limit", [("float32", 2.0 ** -12), ("bfloat16", 0.1)])
@pytest.mark.parametrize("transpose_w", [False, True])
def test_a_penalty_on_the_gradients(handle, dtype, limit, transpose_w):
    """Three products in a row.  FP32: 14 * 2^-22 of the sum of magnitudes for each, which in norm is at most 16
    times the sum here.  bfloat16: six roundings of 2^-9, terms cancelling by no more than a factor of 8."""
    import torch

    _, experts, x, w, ends = _case(getattr(torch, dtype), transpose_w)
    y = experts.grouped_linear(handle, x, w, ends, transpose_w)
    dx, dw = torch.autograd.grad(y.sum(), (x, w), create_graph=True)
    # (the sum over the experts sends each of them one and the same matrix)
    loss = dx.float().square().sum() + dw.float().square().sum() + dw.float().sum(0).square().sum()
    got = torch.autograd.grad(loss, (x, w))
    xd, wd, yd = _in_64_bits(torch, x, w, transpose_w)
    dx, dw = torch.autograd.grad(yd.sum(), (xd, wd), create_graph=True)
    want = torch.autograd.grad(dx.square().sum() + dw.square().sum() + dw.sum(0).square().sum(), (xd, wd))
    _near(got[0], want[0], limit)
    _near(got[1], want[1], limit)
    assert (got[0][sum(COUNTS):] == 0).all() and (got[1][1] == 0).all()


@pytest.mark.parametrize("magnitude", [1.0, 1e-6, 1e-9, 1e-20, 1e8])
@pytest.mark.parametrize("counts", [COUNTS, [300, 0, 5, 40]])
@pytest.mark.parametrize("transpose_w", [False, True])
def test_fp32_gradients_of_any_magnitude(handle, magnitude, counts, transpose_w):
    """Operands scaled by their largest element: each is hi + lo to 2^-22 of itself or 2^-50 of the largest.
    Sums as in test_experts_gpu.py, (12 + terms / 512 + 1) * 2^-22 of the sum of magnitudes."""
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from cumpsgemm_b200 import experts

    n, k, rows = 64, 96, sum(counts) + SPARE
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(rows, k, generator=g, device="cuda").requires_grad_()
    w = torch.randn(len(counts), *((n, k) if transpose_w else (k, n)), generator=g, device="cuda").requires_grad_()
    dy = torch.randn(rows, n, generator=g, device="cuda") * magnitude
    ends = torch.tensor(counts).cumsum(0).to(torch.int32).cuda()
    experts.grouped_linear(handle, x, w, ends, transpose_w).backward(dy)
    xd, wd, dyd = x.detach().double(), w.detach().double(), dy.double()
    at = 0
    for e, c in enumerate(counts):
        r, we = slice(at, at + c), wd[e] if transpose_w else wd[e].t()  # n x k
        at += c
        for got, a, b in ((x.grad[r], dyd[r], we),
                          (w.grad[e] if transpose_w else w.grad[e].t(), dyd[r].t(), xd[r])):
            terms = a.shape[1]
            tol = (12 + terms / 512 + 1) * 2.0 ** -22 * (a.abs() @ b.abs())
            tol = tol + 2.0 ** -50 * terms * float(dyd.abs().max()) * float(max(xd.abs().max(), wd.abs().max()))
            assert ((got.double() - a @ b).abs() <= tol).all()


@pytest.mark.parametrize("transpose_w", [False, True])
def test_the_products_themselves_have_gradients(handle, transpose_w):
    """grouped_matmul and grouped_matmul_wgrad of tensors that require gradients, alpha included; a result in
    `out` has none to give and is refused.  Bounds as in the first test."""
    import torch

    _, experts, x, w, ends = _case(torch.float32, transpose_w)
    y = experts.grouped_matmul(handle, x, w, ends, transpose_w, alpha=-0.5)
    dw = experts.grouped_matmul_wgrad(handle, x, y, ends, transpose_w, alpha=3.0)  # x_e^T y_e
    got = torch.autograd.grad(dw.sum() + y.square().sum(), (x, w))
    xd, wd, yd = _in_64_bits(torch, x, w, transpose_w)
    yd, at, total = -0.5 * yd, 0, 0.0
    for c in COUNTS:
        total = total + 3.0 * (xd[at:at + c].t() @ yd[at:at + c]).sum()
        at += c
    want = torch.autograd.grad(total + yd.square().sum(), (xd, wd))
    _near(got[0], want[0], 2.0 ** -12)
    _near(got[1], want[1], 2.0 ** -12)
    with pytest.raises(ValueError, match="no_grad"):
        experts.grouped_matmul(handle, x, w, ends, transpose_w, out=y.detach())
    with pytest.raises(ValueError, match="no_grad"):
        experts.grouped_matmul_wgrad(handle, x, y, ends, transpose_w, out=dw.detach())
    with torch.no_grad():
        assert not experts.grouped_matmul(handle, x, w, ends, transpose_w, out=y.detach()).requires_grad


def test_a_result_in_out_is_seen_by_autograd(handle):
    """What a graph has kept and a product overwrites is refused by the backward pass, not used."""
    import torch

    _, experts, x, w, ends = _case(torch.bfloat16, False)
    x, w = x.detach(), w.detach()
    xq, sx = experts.quantize_rows(handle, x)
    wq, sw = experts.quantize_rows(handle, w.transpose(1, 2).reshape(-1, w.shape[1]))
    wq = wq.unflatten(0, (len(COUNTS), w.shape[2]))
    y, dw = x.new_zeros(x.shape[0], w.shape[2]), torch.zeros_like(w)
    for out, call in ((y, lambda out: experts.grouped_matmul(handle, x, w, ends, out=out)),
                      (dw, lambda out: experts.grouped_matmul_wgrad(handle, x, y, ends, out=out)),
                      (y, lambda out: experts.i8_matmul(handle, xq, sx, wq, sw, ends, out=out))):
        factor = torch.ones_like(out, requires_grad=True)
        loss = (factor * out).sum()
        call(out)
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
        with pytest.raises(ValueError, match="no_grad"):
            call(factor)
        with torch.no_grad():
            call(factor)
