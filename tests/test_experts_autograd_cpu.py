"""What autograd makes of the grouped products, without a GPU: stand-ins for the two products, which like the
kernels leave no graph behind, and every derivative against differences in 64 bits."""
import pytest
import torch

COUNTS, N, K = [3, 0, 2], 3, 4
ROWS = sum(COUNTS) + 2  # two rows of no expert


def _spans(group_ends, rows):
    ends = [rows] if group_ends is None else group_ends.tolist()
    return list(zip([0] + ends[:-1], ends))


@pytest.fixture()
def experts(monkeypatch):
    from cumpsgemm_b200 import experts

    calls = []

    @torch.no_grad()
    def matmul(handle, x, w, group_ends=None, transpose_w=False, *, mode=None, alpha=1.0):
        calls.append(("matmul", mode))
        experts._rows_of(x, "x"), experts._matrices_of(w, "w")
        y = x.new_zeros(x.shape[0], w.shape[1] if transpose_w else w.shape[2])
        for e, (a, b) in enumerate(_spans(group_ends, x.shape[0])):
            y[a:b] = alpha * x[a:b] @ (w[e].t() if transpose_w else w[e])
        return y

    @torch.no_grad()
    def wgrad(handle, x, dy, group_ends=None, transpose_w=False, *, mode=None, alpha=1.0):
        calls.append(("wgrad", mode))
        experts._rows_of(x, "x"), experts._rows_of(dy, "dy")
        parts = [alpha * x[a:b].t() @ dy[a:b] for a, b in _spans(group_ends, x.shape[0])]
        return torch.stack([p.t() if transpose_w else p for p in parts]).contiguous()

    monkeypatch.setattr(experts, "grouped_matmul", matmul)
    monkeypatch.setattr(experts, "grouped_matmul_wgrad", wgrad)
    return experts, calls


def _operands(transpose_w, dtype=torch.float64):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(ROWS, K, generator=g, dtype=dtype).requires_grad_()
    w = torch.randn(len(COUNTS), *((N, K) if transpose_w else (K, N)), generator=g, dtype=dtype).requires_grad_()
    return x, w, torch.tensor(COUNTS).cumsum(0).to(torch.int32)


@pytest.mark.parametrize("transpose_w", [False, True])
def test_first_second_and_third_derivatives(experts, transpose_w):
    module, _ = experts
    x, w, ends = _operands(transpose_w)
    f = lambda x, w: module.grouped_linear(None, x, w, ends, transpose_w)  # noqa: E731
    assert torch.autograd.gradcheck(f, (x, w))
    assert torch.autograd.gradgradcheck(f, (x, w))
    dx = lambda x, w: torch.autograd.grad(f(x, w).pow(3).sum(), x, create_graph=True)[0]  # noqa: E731
    assert torch.autograd.gradgradcheck(dx, (x, w))


@pytest.mark.parametrize("transpose_w", [False, True])
def test_a_penalty_on_the_gradient_counts(experts, transpose_w):
    """y.sum() has a gradient by y that needs none itself: that of x depends on w all the same."""
    module, _ = experts
    x, w, ends = _operands(transpose_w)
    y = module.grouped_linear(None, x, w, ends, transpose_w)
    dx, dw = torch.autograd.grad(y.sum(), (x, w), create_graph=True)
    (dx.square().sum() + dw.square().sum()).backward()
    xd, wd = x.detach().requires_grad_(), w.detach().requires_grad_()
    parts = [xd[a:b] @ (wd[e].t() if transpose_w else wd[e]) for e, (a, b) in enumerate(_spans(ends, ROWS))]
    want = torch.autograd.grad(torch.cat(parts).sum(), (xd, wd), create_graph=True)
    (want[0].square().sum() + want[1].square().sum()).backward()
    assert torch.allclose(x.grad, xd.grad, rtol=1e-12, atol=0) and torch.allclose(w.grad, wd.grad, rtol=1e-12, atol=0)


def test_a_gradient_that_is_one_value_for_several_experts(experts):
    """The sum over the experts sends each of them the same matrix, at a distance of zero."""
    module, _ = experts
    x, w, ends = _operands(False)
    y = module.grouped_linear(None, x, w, ends)
    dw, = torch.autograd.grad(y.square().sum(), w, create_graph=True)
    got = torch.autograd.grad((dw.sum(0) ** 2).sum(), (x, w))
    xd, wd = x.detach().requires_grad_(), w.detach().requires_grad_()
    yd = torch.cat([xd[a:b] @ wd[e] for e, (a, b) in enumerate(_spans(ends, ROWS))])
    dw, = torch.autograd.grad(yd.square().sum(), wd, create_graph=True)
    want = torch.autograd.grad((dw.sum(0) ** 2).sum(), (xd, wd))
    for g, e in zip(got, want):
        assert torch.allclose(g, e, rtol=1e-10, atol=1e-10)


def test_gradients_are_multiplied_at_any_magnitude(experts):
    """Each product of a backward pass, of a second one too, has its operands scaled; the forward pass does not."""
    from cumpsgemm_b200.api import ComputeMode

    module, calls = experts
    x, w, ends = _operands(False)
    y = module.grouped_linear(None, x, w, ends)
    assert calls == [("matmul", ComputeMode.FP16TCEC)]
    dx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    dx.square().sum().backward()
    assert len(calls) > 4 and all(mode == ComputeMode.FP16TCEC_SCALING for _, mode in calls[1:])
    del calls[:]
    module.grouped_linear(None, x, w, ends, mode=ComputeMode.FP16TCEC_SCALING,
                          backward_mode=ComputeMode.FP16TCEC).sum().backward()
    assert [mode for _, mode in calls] == [ComputeMode.FP16TCEC_SCALING] + 2 * [ComputeMode.FP16TCEC]


@pytest.mark.parametrize("transpose_w", [False, True])
def test_no_rows_at_all(experts, transpose_w):
    """The gradient of a sum over no rows: an empty tensor whose strides, 0 and 0, say nothing."""
    module, _ = experts
    _, w, _ = _operands(transpose_w)
    x = torch.zeros(0, K, dtype=torch.float64, requires_grad=True)
    ends = torch.zeros(len(COUNTS), dtype=torch.int32)
    for create_graph in (False, True):
        y = module.grouped_linear(None, x, w, ends, transpose_w)
        dx, dw = torch.autograd.grad(y.sum(), (x, w), create_graph=create_graph)
        assert dx.shape == (0, K) and dw.shape == w.shape and not dw.any()
    assert module._rows_of(torch.zeros(()).expand(0, 5), "x", 5) == (0, 5, 5)
    with pytest.raises(ValueError, match="columns"):
        module._rows_of(torch.zeros(0, 4), "x", 5)
