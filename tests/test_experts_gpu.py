"""Products of rows grouped by expert against their definitions in 64 bits.

Tolerances, element by element, with S = sum |x| |w| over the terms of that element:
* 16-bit types: one rounding of the result (2^-8 bfloat16, 2^-11 float16, plus half the smallest
  subnormal of float16), and FP32 sums to which the tensor core adds 16 products at a time.  It
  truncates, so each of the k / 16 + 1 additions is off by at most 2^-22 S.
* FP32: an operand is hi + lo / 2^11 to 2^-22 of itself (2^-36 where lo is subnormal), lo * lo is left
  out: 3 * 2^-22 S.  Eight additions of the tensor core between drains, 9 * 2^-22 S; FP32 additions of the
  drained sums and the corrections, (k / 512 + 1) * 2^-22 S.
  (Few rows are multiplied in FP32 arithmetic, k roundings of at most 2^-24 S, which with the random signs
  here come to their square root: they are held to the same bound.)
* 8 bits: the sums are exact; three FP32 roundings for conversion and scales, one for the bias, one
  for the result.
"""
import pytest

pytestmark = pytest.mark.gpu


def _setup():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from cumpsgemm_b200 import api, experts

    return torch, api, experts


def _matrix(torch, values, ld, offset):
    """The values in rows `ld` apart, `offset` elements into their allocation, NaN in between."""
    *batch, rows, cols = values.shape
    count = rows * ld
    for b in batch:
        count *= b
    fill = float("nan") if values.dtype.is_floating_point else 77
    buf = torch.full((offset + count,), fill, dtype=values.dtype, device="cuda")
    view = buf[offset:].view(*batch, rows, ld)[..., :cols]
    view.copy_(values)
    return view


def _ends(torch, counts):
    return torch.tensor(counts).cumsum(0).to(torch.int32).cuda()


def _spans(counts):
    at = 0
    for c in counts:
        yield at, at + c
        at += c


def _unit(torch, dtype):
    return {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]


def _tolerance(torch, dtype, k, want, size, spread):
    """size: S; spread: the sum of |x| and |w| over the terms."""
    if dtype == torch.float32:
        return (12 + k / 512 + 1) * 2.0 ** -22 * size + 2.0 ** -36 * spread
    return (_unit(torch, dtype) * want.abs() + (k / 16 + 1) * 2.0 ** -22 * size +
            (2.0 ** -25 if dtype == torch.float16 else 0.0))


def _close(got, want, tol, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((off / tol.clamp(min=1e-300)).max()))


def _product(torch, x, w, counts, transpose_w):
    rows, n = x.shape[0], w.shape[1] if transpose_w else w.shape[2]
    y, size, spread = (torch.zeros(rows, n, dtype=torch.float64, device="cuda") for _ in range(3))
    for e, (a, b) in enumerate(_spans(counts)):
        xe, we = x[a:b].double(), w[e].double()
        we = we.t() if transpose_w else we
        y[a:b] = xe @ we
        size[a:b] = xe.abs() @ we.abs()
        spread[a:b] = xe.abs().sum(1, keepdim=True) + we.abs().sum(0, keepdim=True)
    return y, size, spread


def _wgrad(torch, x, dy, counts, transpose_w):
    out = []
    for a, b in _spans(counts):
        xe, de = x[a:b].double(), dy[a:b].double()
        t = (xe.t() @ de, xe.t().abs() @ de.abs(),
             xe.abs().sum(0)[:, None] + de.abs().sum(0)[None, :])
        out.append([v.t() if transpose_w else v for v in t])
    return [torch.stack([o[i] for o in out]) for i in range(3)]


# rows of each expert: none at all, one, less than a step of 16 or 32, whole tiles, more than a tile
COUNTS = [
    [1],
    [0, 3, 0],
    [16, 17, 1, 31, 0, 33, 64, 63, 65],
    [256, 0, 257, 300, 128, 5],
    [0, 0, 700],
]
# n, k: a single element, less than a step, odd, whole tiles and one past them
SIZES = [(1, 1), (8, 16), (33, 65), (256, 64), (257, 129), (512, 1000), (100, 640)]
DTYPES = ["bfloat16", "float16", "float32"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("transpose_w", [False, True])
@pytest.mark.parametrize("n,k", SIZES)
def test_product_and_wgrad(handle, dtype, transpose_w, n, k):
    torch, api, experts = _setup()
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(n * 7 + k)
    for counts in COUNTS:
        rows = sum(counts)
        x = torch.randn(rows, k, generator=g, device="cuda").to(dt)
        dy = torch.randn(rows, n, generator=g, device="cuda").to(dt)
        w = torch.randn(len(counts), *((n, k) if transpose_w else (k, n)), generator=g, device="cuda").to(dt)
        ends = _ends(torch, counts)
        y = experts.grouped_matmul(handle, x, w, ends, transpose_w)
        want, size, spread = _product(torch, x, w, counts, transpose_w)
        _close(y, want, _tolerance(torch, dt, k, want, size, spread), ("product", counts))
        dw = experts.grouped_matmul_wgrad(handle, x, dy, ends, transpose_w)
        want, size, spread = _wgrad(torch, x, dy, counts, transpose_w)
        _close(dw, want, _tolerance(torch, dt, max(counts), want, size, spread), ("wgrad", counts))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pads,offset", [((0, 0, 0), 1), ((1, 3, 2), 0), ((8, 16, 24), 8), ((5, 8, 7), 3)])
def test_strides_alignment_alpha_and_beta(handle, dtype, pads, offset):
    torch, api, experts = _setup()
    dt = getattr(torch, dtype)
    counts, n, k = [40, 0, 90, 1], 70, 200
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    rows, e = sum(counts) + 4, len(counts)  # four rows of no expert
    x0, w0, y0, dy0, dw0 = rnd(rows, k), rnd(e, k, n), rnd(rows, n), rnd(rows, n), rnd(e, k, n)
    x, w = _matrix(torch, x0, k + pads[0], offset), _matrix(torch, w0, n + pads[1], offset)
    y, dy = _matrix(torch, y0, n + pads[2], offset), _matrix(torch, dy0, n + pads[2], offset)
    dw = _matrix(torch, dw0, n + pads[1], offset)
    ends = _ends(torch, counts)
    alpha, beta = -0.75, 0.5
    experts.grouped_matmul(handle, x, w, ends, alpha=alpha, beta=beta, out=y)
    want, size, spread = _product(torch, x0, w0, counts, False)
    want = alpha * want + beta * y0.double()
    size = abs(alpha) * size + abs(beta) * y0.double().abs()
    _close(y, want, _tolerance(torch, dt, k, want, size, spread))
    experts.grouped_matmul_wgrad(handle, x, dy, ends, alpha=alpha, beta=beta, out=dw)
    want, size, spread = _wgrad(torch, x0, dy0, counts, False)
    want = alpha * want + beta * dw0.double()
    size = abs(alpha) * size + abs(beta) * dw0.double().abs()
    _close(dw, want, _tolerance(torch, dt, max(counts), want, size, spread))
    # what lies between the rows of the outputs is left alone
    for t in (y, dw):
        whole = torch.as_strided(t, (t.numel() // t.shape[-1], t.stride(-2)), (t.stride(-2), 1))
        assert whole[:, t.shape[-1]:].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mode", ["FP16TCEC", "FP16TCEC_SCALING"])
def test_nan_in_other_groups_and_in_no_group_does_not_count(handle, dtype, mode):
    """Every other expert's rows are NaN or infinite, and so are the rows behind the last."""
    torch, api, experts = _setup()
    if dtype != "float32" and mode != "FP16TCEC":
        pytest.skip("16-bit types do not look at the mode")
    dt, m = getattr(torch, dtype), api.ComputeMode[mode]
    counts, n, k = [5, 7, 66, 100, 1, 30], 96, 80
    g = torch.Generator(device="cuda").manual_seed(5)
    rows = sum(counts) + 9
    x = torch.randn(rows, k, generator=g, device="cuda").to(dt)
    dy = torch.randn(rows, n, generator=g, device="cuda").to(dt)
    w = torch.randn(len(counts), k, n, generator=g, device="cuda").to(dt)
    ends = _ends(torch, counts)
    clean = [e % 2 == 0 for e in range(len(counts))]
    xp, dyp = x.clone(), dy.clone()
    for e, (a, b) in enumerate(_spans(counts)):
        if not clean[e]:
            xp[a:b], dyp[a:b] = float("nan"), float("inf")
    xp[sum(counts):], dyp[sum(counts):] = float("inf"), float("nan")
    y = experts.grouped_matmul(handle, xp, w, ends, mode=m)
    dw = experts.grouped_matmul_wgrad(handle, xp, dyp, ends, mode=m)
    want, size, spread = _product(torch, x, w, counts, False)
    want_w, size_w, spread_w = _wgrad(torch, x, dy, counts, False)
    for e, (a, b) in enumerate(_spans(counts)):
        if clean[e]:
            _close(y[a:b], want[a:b], _tolerance(torch, dt, k, want, size, spread)[a:b])
            _close(dw[e], want_w[e], _tolerance(torch, dt, 100, want_w, size_w, spread_w)[e])
        else:
            assert y[a:b].isnan().all() and dw[e].isnan().all()
    assert (y[sum(counts):] == 0).all()


def test_totals_are_not_trusted(handle):
    """Falling, negative and too large totals: taken as the one in front, or as the rows there are."""
    torch, api, experts = _setup()
    x = torch.randn(100, 64, device="cuda").to(torch.bfloat16)
    w = torch.randn(5, 64, 40, device="cuda").to(torch.bfloat16)
    bad = torch.tensor([-7, 30, 12, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    good = torch.tensor([0, 30, 30, 100, 100], dtype=torch.int32, device="cuda")
    assert torch.equal(experts.grouped_matmul(handle, x, w, bad), experts.grouped_matmul(handle, x, w, good))
    dy = torch.randn(100, 40, device="cuda").to(torch.bfloat16)
    assert torch.equal(experts.grouped_matmul_wgrad(handle, x, dy, bad),
                       experts.grouped_matmul_wgrad(handle, x, dy, good))
    f = lambda t: t.float()  # noqa: E731
    for xf in (f(x), f(x)[:30]):  # on the tensor core, and in FP32 arithmetic
        good30 = good.clamp(max=xf.shape[0])
        assert torch.equal(experts.grouped_matmul(handle, xf, f(w), bad),
                           experts.grouped_matmul(handle, xf, f(w), good30))


def test_no_rows_at_all(handle):
    torch, api, experts = _setup()
    for dt in (torch.bfloat16, torch.float32):
        x, w = torch.empty(0, 48, device="cuda", dtype=dt), torch.ones(3, 48, 24, device="cuda", dtype=dt)
        ends = torch.zeros(3, dtype=torch.int32, device="cuda")
        assert experts.grouped_matmul(handle, x, w, ends).shape == (0, 24)
        dw = torch.full((3, 48, 24), 3.0, device="cuda", dtype=dt)
        experts.grouped_matmul_wgrad(handle, x, x.new_empty(0, 24), ends, beta=0.5, out=dw)
        assert (dw == 1.5).all()
        # rows, but none of them of any group
        x = torch.full((70, 48), float("nan"), device="cuda", dtype=dt)
        assert (experts.grouped_matmul(handle, x, w, ends) == 0).all()
        assert (experts.grouped_matmul_wgrad(handle, x, x[:, :24], ends) == 0).all()


@pytest.mark.parametrize("groups", [31, 32, 33, 1000, 1024])
def test_many_groups(handle, groups):
    torch, api, experts = _setup()
    g = torch.Generator().manual_seed(groups)
    counts = torch.randint(0, 5, (groups,), generator=g).tolist()
    counts[groups // 2] = 400
    x = torch.randn(sum(counts), 64, device="cuda").to(torch.bfloat16)
    w = torch.randn(groups, 64, 48, device="cuda").to(torch.bfloat16)
    y = experts.grouped_matmul(handle, x, w, _ends(torch, counts))
    want, size, spread = _product(torch, x, w, counts, False)
    _close(y, want, _tolerance(torch, torch.bfloat16, 64, want, size, spread))


@pytest.mark.parametrize("magnitude", [1e-6, 1e6, 1e-30])
def test_fp32_scaling(handle, magnitude):
    """Operands that FP16 cannot hold: brought into its range, and back out of it.  An operand is then
    exact to 2^-22 of itself or 2^-36 of 2^-14 of its largest element."""
    torch, api, experts = _setup()
    counts, n, k = [60, 0, 141], 130, 260
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(sum(counts), k, generator=g, device="cuda") * magnitude
    dy = torch.randn(sum(counts), n, generator=g, device="cuda") / magnitude
    w = torch.randn(3, n, k, generator=g, device="cuda")
    ends = _ends(torch, counts)
    m = api.ComputeMode.FP16TCEC_SCALING
    y = experts.grouped_matmul(handle, x, w, ends, True, mode=m)
    want, size, _ = _product(torch, x, w, counts, True)
    floor = 2.0 ** -50 * k * (x.abs().max() * w.abs().max()).double()
    _close(y, want, _tolerance(torch, torch.float32, k, want, size, 0.0) + floor)
    dw = experts.grouped_matmul_wgrad(handle, x, dy, ends, True, mode=m)
    want, size, _ = _wgrad(torch, x, dy, counts, True)
    floor = 2.0 ** -50 * 141 * (x.abs().max().double() * dy.abs().max().double())
    _close(dw, want, _tolerance(torch, torch.float32, 141, want, size, 0.0) + floor)


def _quantised(torch, x):
    """q before rounding, and the scale, in 64 bits."""
    top = x.double().abs().amax(1, keepdim=True)
    return torch.where(top > 0, x.double() * 127 / top.clamp(min=1e-320), 0.0), top[:, 0] / 127


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [1, 7, 64, 1000, 1024, 1025, 2048, 4096, 8192, 8200, 20000])
def test_quantize_rows(handle, dtype, k):
    torch, api, experts = _setup()
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn(37, k, generator=g, device="cuda")
    x[:, 0] *= 30
    x[3] = 0
    x[4] *= 1e-4
    x = x.to(dt)
    for pad, offset in ((0, 0), (3, 1), (8, 8)):
        xs = _matrix(torch, x, k + pad, offset)
        q, scale = experts.quantize_rows(handle, xs)
        want, want_scale = _quantised(torch, x)
        # x * (127 / top): two roundings of a value of at most 127
        assert ((q.double() - want).abs() <= 0.5 + 127 * 2.0 ** -22).all()
        assert ((scale.double() - want_scale).abs() <= 2.0 ** -24 * want_scale).all()
        index = torch.tensor([36, 0, 0, -1, 37, 5, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
        qi, si = experts.quantize_rows(handle, xs, row_index=index)
        for r, i in enumerate(index.tolist()):
            if 0 <= i < 37:
                assert torch.equal(qi[r], q[i]) and si[r] == scale[i]
            else:
                assert (qi[r] == 0).all() and si[r] == 0


def test_quantize_rows_at_the_ends_of_the_range(handle):
    torch, api, experts = _setup()
    x = torch.ones(6, 300, device="cuda")
    x[0, 17] = float("inf")
    x[1, 18] = float("nan")
    x[2] *= 2.0 ** -140
    x[2, 5] = -2.0 ** -133
    x[3] *= 3e38
    x[4] = -x[4]
    x[5] = float("-inf")
    q, scale = experts.quantize_rows(handle, x)
    for r in (0, 1, 5):
        assert scale[r].isnan() and (q[r] == 0).all()
    assert q[2, 5] == -127 and (q[2, :5] == 1).all()
    assert (q[3] == 127).all() and (q[4] == -127).all() and scale[3].isfinite()


@pytest.mark.parametrize("n,k", [(1, 1), (33, 65), (256, 128), (257, 129), (100, 1000), (300, 4096)])
@pytest.mark.parametrize("out_dtype", DTYPES)
def test_i8_product(handle, n, k, out_dtype):
    torch, api, experts = _setup()
    dt = getattr(torch, out_dtype)
    g = torch.Generator(device="cuda").manual_seed(n + k)
    rnd = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device="cuda", dtype=torch.int32).to(torch.int8)  # noqa: E731
    for counts in COUNTS:
        rows, e = sum(counts) + 3, len(counts)
        xq, wq = rnd(-128, 128, rows, k), rnd(-128, 128, e, n, k)
        sx = torch.rand(rows, generator=g, device="cuda") * 1e-2
        sw = torch.rand(e, n, generator=g, device="cuda") * 1e-2
        bias = torch.randn(e, n, generator=g, device="cuda")
        sx[sum(counts):] = float("nan")  # of no expert: their results are zero
        for b in (None, bias):
            y = experts.i8_matmul(handle, xq, sx, wq, sw, _ends(torch, counts), bias=b, out_dtype=dt)
            for i, (lo, hi) in enumerate(_spans(counts)):
                want = (xq[lo:hi].double() @ wq[i].double().t()) * sx[lo:hi, None].double() * sw[i].double()
                tol = 3 * 2.0 ** -24 * want.abs()
                want = want + (b[i].double() if b is not None else 0.0)
                tol = tol + (_unit(torch, dt) + 2.0 ** -24) * want.abs() + 2.0 ** -25
                _close(y[lo:hi], want, tol, counts)
            assert (y[sum(counts):] == 0).all()


def test_i8_sums_are_exact(handle):
    """The largest sums there are: every product 2^14, k the most that is taken."""
    torch, api, experts = _setup()
    k = 131071
    xq = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
    wq = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    wq[1] = 127
    wq[2, 1:] = 0
    one = torch.ones(3, device="cuda")
    y = experts.i8_matmul(handle, xq, one[:2], wq, one, out_dtype=torch.float32)
    want = torch.tensor([float(2 ** 14 * k), float(-128 * 127 * k), 2.0 ** 14], dtype=torch.float64)
    assert torch.equal(y.cpu(), want.float().expand(2, 3))


@pytest.mark.parametrize("pads,offset", [((1, 3), 0), ((16, 32), 16), ((0, 0), 5)])
def test_i8_strides(handle, pads, offset):
    torch, api, experts = _setup()
    counts, n, k = [20, 0, 41], 50, 144
    xq = torch.randint(-127, 128, (61, k), device="cuda", dtype=torch.int32).to(torch.int8)
    wq = torch.randint(-127, 128, (3, n, k), device="cuda", dtype=torch.int32).to(torch.int8)
    sx, sw = torch.rand(61, device="cuda"), torch.rand(3, n, device="cuda")
    ends = _ends(torch, counts)
    plain = experts.i8_matmul(handle, xq, sx, wq, sw, ends)
    got = experts.i8_matmul(handle, _matrix(torch, xq, k + pads[0], offset), sx,
                            _matrix(torch, wq, k + pads[1], offset), sw, ends)
    assert torch.equal(plain, got)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("transpose_w", [False, True])
def test_backward(handle, dtype, transpose_w):
    """Gradients against the formula's in 64 bits, and in FP32 against differences of the forward pass."""
    torch, api, experts = _setup()
    dt = getattr(torch, dtype)
    counts, n, k = [30, 0, 77, 1], 64, 96
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(sum(counts) + 5, k, generator=g, device="cuda").to(dt).requires_grad_()
    w = torch.randn(4, *((n, k) if transpose_w else (k, n)), generator=g, device="cuda").to(dt).requires_grad_()
    dy = torch.randn(sum(counts) + 5, n, generator=g, device="cuda").to(dt)
    ends = _ends(torch, counts)
    experts.grouped_linear(handle, x, w, ends, transpose_w).backward(dy)
    want, size, spread = _product(torch, dy, w.detach(), counts, not transpose_w)
    _close(x.grad, want, _tolerance(torch, dt, n, want, size, spread))
    assert (x.grad[sum(counts):] == 0).all()
    want, size, spread = _wgrad(torch, x.detach(), dy, counts, transpose_w)
    _close(w.grad, want, _tolerance(torch, dt, 77, want, size, spread))
    assert (w.grad[1] == 0).all()
    # the gradient of a sum arrives as one value for all elements
    x.grad = None
    experts.grouped_linear(handle, x, w, ends, transpose_w).sum().backward()
    want, size, spread = _product(torch, torch.ones_like(dy), w.detach(), counts, not transpose_w)
    _close(x.grad, want, _tolerance(torch, dt, n, want, size, spread))
    if dt == torch.float32:
        # y is linear in x and in w: the difference quotient along a direction is the gradient's product
        # with it, but for the rounding of both forward passes
        for t in (x, w):
            t.grad = None
        y0 = experts.grouped_linear(handle, x, w, ends, transpose_w)
        y0.backward(dy)
        for t, other in ((x, w), (w, x)):
            step = torch.randn(t.shape, generator=g, device="cuda")
            with torch.no_grad():
                moved = t + step
                step = moved - t  # what was added, exactly
                y1 = (experts.grouped_matmul(handle, moved, other, ends, transpose_w) if t is x else
                      experts.grouped_matmul(handle, other, moved, ends, transpose_w))
            slope = ((y1.double() - y0.double()) * dy.double()).sum()
            along = (t.grad.double() * step.double()).sum()
            terms = (t.grad.double() * step.double()).abs().sum()
            assert abs(slope - along) <= 2.0 ** -16 * terms, (float(slope), float(along), float(terms))


def test_runs_repeat_bit_for_bit_on_another_stream_and_in_a_graph(handle):
    torch, api, experts = _setup()
    counts, n, k = [100, 3, 0, 500], 300, 512
    x = torch.randn(603, k, device="cuda").to(torch.bfloat16)
    w = torch.randn(4, k, n, device="cuda").to(torch.bfloat16)
    ends = _ends(torch, counts)
    first = experts.grouped_matmul(handle, x, w, ends)
    first32 = experts.grouped_matmul(handle, x.float(), w.float(), ends)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    handle.set_stream(side)
    with torch.cuda.stream(side):
        again = experts.grouped_matmul(handle, x, w, ends)
    side.synchronize()
    assert torch.equal(first, again)
    y, y32, xf, wf = torch.empty_like(first), torch.empty_like(first32), x.float(), w.float()
    graph = torch.cuda.CUDAGraph()
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        experts.grouped_matmul(handle, x, w, ends, out=y)
        experts.grouped_matmul(handle, xf, wf, ends, out=y32)
    ends.copy_(_ends(torch, [3, 100, 500, 0]))  # the sizes are read at every replay
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(y, first)
    ends.copy_(_ends(torch, counts))
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, first) and torch.equal(y32, first32)
    handle.set_stream(torch.cuda.current_stream())


def test_offsets_beyond_32_bits(handle):
    """An output of more than 2^32 bytes, and a row index far into x."""
    torch, api, experts = _setup()
    rows, n, k = 600000, 4096, 16
    x = torch.randn(rows, k, device="cuda").to(torch.bfloat16)
    w = torch.randn(2, k, n, device="cuda").to(torch.bfloat16)
    ends = torch.tensor([rows - 300, rows], dtype=torch.int32, device="cuda")
    y = experts.grouped_matmul(handle, x, w, ends)
    tail = x[-300:].double() @ w[1].double()
    size = x[-300:].double().abs() @ w[1].double().abs()
    _close(y[-300:], tail, _tolerance(torch, torch.bfloat16, k, tail, size, 0.0))
    q, s = experts.quantize_rows(handle, y, row_index=torch.tensor([rows - 1], dtype=torch.int32, device="cuda"))
    want, _ = _quantised(torch, y[-1:])
    assert ((q.double() - want).abs() <= 0.5 + 127 * 2.0 ** -22).all()


def test_refusals(handle):
    torch, api, experts = _setup()
    bf = dict(device="cuda", dtype=torch.bfloat16)
    x, w = torch.zeros(8, 16, **bf), torch.zeros(2, 16, 24, **bf)
    ends = torch.tensor([4, 8], dtype=torch.int32, device="cuda")
    for call in (lambda: experts.grouped_matmul(handle, x, w),                      # which rows go where?
                 lambda: experts.grouped_matmul(handle, x, w, ends.long()),
                 lambda: experts.grouped_matmul(handle, x, w, ends[:1]),
                 lambda: experts.grouped_matmul(handle, x, w, ends.cpu()),
                 lambda: experts.grouped_matmul(handle, x, w, ends, True),            # k does not match
                 lambda: experts.grouped_matmul(handle, x.float(), w, ends),
                 lambda: experts.grouped_matmul(handle, x.double(), w.double(), ends),
                 lambda: experts.grouped_matmul(handle, x.t().contiguous().t(), w, ends),
                 lambda: experts.grouped_matmul(handle, x[:1].expand(8, 16), w, ends),
                 lambda: experts.grouped_matmul(handle, x.cpu(), w, ends),
                 lambda: experts.grouped_matmul(handle, x, w, ends, beta=1.0),
                 lambda: experts.grouped_matmul(handle, x, w, ends, out=torch.zeros(8, 24, device="cuda")),
                 lambda: experts.grouped_matmul_wgrad(handle, x, x[:4], ends),
                 lambda: experts.quantize_rows(handle, x, row_index=ends.long()),
                 lambda: experts.i8_matmul(handle, x, x[:, 0].float(), w, w[0].float(), ends)):
        with pytest.raises(ValueError):
            call()
    f = x.float(), w.float()
    for mode in (api.ComputeMode.TF32TCEC, api.ComputeMode.AUTO, api.ComputeMode.CUBLAS):
        with pytest.raises(api.CuMpSGEMMError) as e:
            experts.grouped_matmul(handle, *f, ends, mode=mode)
        assert e.value.status == api.CUBLAS_STATUS_NOT_SUPPORTED
    y = torch.zeros(8, 24, **bf)
    good = dict(op_W=0, rows=8, n=24, k=16, num_groups=2, group_ends=ends, alpha=1.0, X=x, ldx=16, W=w,
                ldw=24, stridew=384, beta=0.0, Y=y, ldy=24, data_type=api.CUDA_R_16BF)
    assert handle.grouped_gemm(**good) == 0
    for change in (dict(op_W=3), dict(n=0), dict(k=0), dict(num_groups=0), dict(num_groups=1025), dict(ldx=15),
                   dict(ldw=23), dict(ldy=23), dict(stridew=383), dict(data_type=1), dict(group_ends=None),
                   dict(rows=1 << 31), dict(X=0), dict(W=0), dict(Y=0)):
        assert handle.grouped_gemm(**{**good, **change}, check=False) == api.CUBLAS_STATUS_INVALID_VALUE, change
    assert handle.i8_grouped_gemm(8, 24, 131072, 1, None, x, 131072, x, w, 131072, 0, w, None, y, 24,
                                  api.CUDA_R_16BF, check=False) == api.CUBLAS_STATUS_INVALID_VALUE
    assert handle.quantize_rows_i8(8, 16, x, 16, api.CUDA_R_16BF, None, 7, y, 16, y,
                                   check=False) == api.CUBLAS_STATUS_INVALID_VALUE
    handle.set_workspace_limit(1 << 10)
    with pytest.raises(api.CuMpSGEMMError) as e:  # (few rows need none)
        experts.grouped_matmul(handle, torch.zeros(80, 16, device="cuda"), f[1], ends)
    assert e.value.status == api.CUBLAS_STATUS_ALLOC_FAILED
    handle.set_workspace_limit(0)
    # results are allocated on the current stream and written on the handle's
    with torch.cuda.stream(torch.cuda.Stream()), pytest.raises(ValueError, match="stream"):
        experts.grouped_matmul(handle, x, w, ends)
    # and the handle goes on working
    assert handle.grouped_gemm(**good) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", [[1], [20, 0, 300], [256]])
def test_few_tiles_with_a_long_sum(handle, dtype, counts):
    """Tiles fewer than half the pairs of SMs are cut along K and their sums added in a fixed order: at
    most 15 more FP32 additions, 4 * 2^-22 S.  Without memory for the sums they stay whole."""
    torch, api, experts = _setup()
    dt = getattr(torch, dtype)
    n, k, rows = 200, 5000, sum(counts)
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, k, generator=g, device="cuda").to(dt)
    w = torch.randn(len(counts), n, k, generator=g, device="cuda").to(dt)
    want, size, spread = _product(torch, x, w, counts, True)
    tol = _tolerance(torch, dt, k, want, size, spread) + 2.0 ** -20 * size
    y = experts.grouped_matmul(handle, x, w, _ends(torch, counts), True)
    _close(y, want, tol)
    for _ in range(3):
        assert torch.equal(y, experts.grouped_matmul(handle, x, w, _ends(torch, counts), True))
    if dt != torch.float32:
        handle.set_workspace_limit(1 << 10)
        _close(experts.grouped_matmul(handle, x, w, _ends(torch, counts), True), want, tol)
        handle.set_workspace_limit(0)
    # the gradient of the weights, over rows that end inside a block
    x = torch.randn(5000 + rows, 90, generator=g, device="cuda").to(dt)
    dy = torch.randn(5000 + rows, n, generator=g, device="cuda").to(dt)
    counts = [rows, 5000]
    dw = experts.grouped_matmul_wgrad(handle, x, dy, _ends(torch, counts))
    want, size, spread = _wgrad(torch, x, dy, counts, False)
    _close(dw, want, _tolerance(torch, dt, 5000, want, size, spread) + 2.0 ** -20 * size)


def test_few_tiles_with_a_long_integer_sum(handle):
    torch, api, experts = _setup()
    rows, n, k = 70, 130, 20000
    xq = torch.randint(-128, 128, (rows, k), device="cuda", dtype=torch.int32).to(torch.int8)
    wq = torch.randint(-128, 128, (n, k), device="cuda", dtype=torch.int32).to(torch.int8)
    one = torch.ones(n, device="cuda")
    y = experts.i8_matmul(handle, xq, one[:rows], wq, one, out_dtype=torch.float32)
    assert torch.equal(y.double(), (xq.double() @ wq.double().t()).float().double())


@pytest.mark.parametrize("transpose_w", [False, True])
@pytest.mark.parametrize("counts", [[1], [6], [2, 0, 3, 1], [0] * 20 + [60, 1, 0, 9, 8, 7, 17], [1] * 40])
@pytest.mark.parametrize("n,k,pad,offset", [(1, 1, 0, 0), (130, 4100, 0, 0), (300, 70, 3, 1), (1024, 2048, 0, 0)])
def test_fp32_with_few_rows(handle, transpose_w, counts, n, k, pad, offset):
    """At most six rows for each group on average: FP32 arithmetic, k + 16 roundings of at most 2^-24 S."""
    torch, api, experts = _setup()
    rows, e = sum(counts) + (1 if len(counts) > 3 else 0), len(counts)
    assert rows <= 6 * e
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    x0 = torch.randn(rows, k, generator=g, device="cuda") * 1e-6
    w0 = torch.randn(e, *((n, k) if transpose_w else (k, n)), generator=g, device="cuda") * 1e6
    y0 = torch.randn(rows, n, generator=g, device="cuda")
    for i, c in enumerate(counts):  # weights of experts without rows never count
        if c == 0:
            w0[i] = float("nan")
    x0[sum(counts):] = float("nan")  # nor do rows of no expert
    x, w = _matrix(torch, x0, k + pad, offset), _matrix(torch, w0, w0.shape[2] + pad, offset)
    y = _matrix(torch, y0, n + pad, offset)
    ends = _ends(torch, counts)
    want, size, _ = _product(torch, x0, w0, counts, transpose_w)
    for mode in (api.ComputeMode.FP16TCEC, api.ComputeMode.FP16TCEC_SCALING):
        got = experts.grouped_matmul(handle, x, w, ends, transpose_w, mode=mode)
        _close(got, want, (k + 16) * 2.0 ** -24 * size)
        assert (got[sum(counts):] == 0).all()
        assert torch.equal(got, experts.grouped_matmul(handle, x, w, ends, transpose_w, mode=mode))
    experts.grouped_matmul(handle, x, w, ends, transpose_w, alpha=-2.0, beta=0.5, out=y)
    want = -2.0 * want + 0.5 * y0.double()
    _close(y, want, (k + 18) * 2.0 ** -24 * (2.0 * size + 0.5 * y0.double().abs()))


def test_a_wait_that_gave_up_leaves_the_handle_usable(handle):
    """The status word raised (by the self-test's wait, which runs out): clearing it clears what the grouped
    kernel counts with, and the next products are right."""
    torch, api, experts = _setup()
    x = torch.randn(90, 64, device="cuda").to(torch.bfloat16)
    w = torch.randn(3, 64, 40, device="cuda").to(torch.bfloat16)
    ends = _ends(torch, [30, 0, 60])
    first = experts.grouped_matmul(handle, x, w, ends)
    status, _ = handle.selftest_bounded_wait(50)
    assert status != 0
    assert torch.equal(first, experts.grouped_matmul(handle, x, w, ends))
    assert handle.kernel_status() == 0
