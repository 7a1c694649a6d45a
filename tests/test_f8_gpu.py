"""Products in 8-bit floating point with a scale for each block of 128, and what brings operands there, against their
definitions.

Tolerances:
* quantisation of 16-bit values: none.  x M has at most 14 bits and is exact in FP32, its quotient by the largest
  magnitude is rounded once, and so is that in the oracle; the same for scales.  FP32 values: half a step of the
  8-bit type (2^-4 e4m3, 2^-3 e5m2 of the value, or half its smallest subnormal, 2^-10 and 2^-17, of the scale), and
  2^-22 of the value for the roundings in front of it.
* products, with S = sum |x| |w| over the terms of an element (x and w as their 8-bit values and scales stand for
  them): the tensor core adds 32 products at a time and truncates, 5 such additions a block of 128, each off by at
  most 2^-22 S; two FP32 roundings of a scale and one for each of the blocks' additions, 2^-24 S each.
  Together (6 + blocks / 4) 2^-22 S, and the rounding of the result.
* a gated product: what its two products are off by, through the activation (slope at most 1.13) and the product; the
  activation's own error as in the tests of the 16-bit blocks, (8 + 6 |g| + 2 g^2 + |g|^3) 2^-23; then half a step.
"""
import pytest

pytestmark = pytest.mark.gpu

MOST = {"float8_e4m3fn": 448.0, "float8_e5m2": 57344.0}
UNIT = {"float8_e4m3fn": 2.0 ** -4, "float8_e5m2": 2.0 ** -3}  # half a step, of the value
TINY = {"float8_e4m3fn": 2.0 ** -10, "float8_e5m2": 2.0 ** -17}  # half of the smallest subnormal


def _setup():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from cumpsgemm_b200 import api, experts

    return torch, api, experts


def _ends(torch, counts):
    return torch.tensor(counts).cumsum(0).to(torch.int32).cuda()


def _spans(counts):
    at = 0
    for c in counts:
        yield at, at + c
        at += c


def _rows_quantised(torch, x, name):
    """(q, scale) of rows by elementary operations in FP32."""
    rows, k = x.shape
    kb = (k + 127) // 128
    t = torch.nn.functional.pad(x.float(), (0, kb * 128 - k)).view(rows, kb, 128)
    top = t.abs().amax(2, keepdim=True)
    most = torch.full_like(top, MOST[name])
    q = torch.where(top > 0, t * most / top, t).reshape(rows, kb * 128)[:, :k]
    return q.to(getattr(torch, name)), (top / most)[..., 0]


def _spread(scale, rows, cols, by_rows):
    """Scales of blocks as one for each element."""
    s = scale.double()
    if by_rows:
        s = s.repeat_interleave(128, -2)[..., :rows, :]
    return s.repeat_interleave(128, -1)[..., :cols]


def _same_values(torch, a, b):
    return torch.equal(a.float(), b.float())


@pytest.mark.parametrize("name", ["float8_e4m3fn", "float8_e5m2"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,k,pad,offset", [(1, 1, 0, 0), (3, 127, 1, 1), (5, 128, 0, 0), (7, 129, 0, 3), (130, 1000, 8, 8),
                                               (2, 2050, 0, 0), (2049, 264, 0, 0), (4, 8192, 0, 0), (33, 1160, 5, 2)])
def test_rows_exactly(handle, name, dtype, rows, k, pad, offset):
    torch, api, experts = _setup()
    dtype, f8 = getattr(torch, dtype), getattr(torch, name)
    x = torch.randn(rows, k, device="cuda")
    x[:, torch.rand(k, device="cuda") < 0.02] *= 50
    buf = torch.full((offset + rows * (k + pad),), float("nan"), dtype=dtype, device="cuda")
    view = buf[offset:].view(rows, k + pad)[:, :k]
    view.copy_(x)
    want_q, want_s = _rows_quantised(torch, view, name)
    q, scale = experts.quantize_blocks(handle, view, dtype=f8)
    assert q.dtype == f8 and q.shape == (rows, k) and scale.shape == (rows, (k + 127) // 128)
    assert torch.equal(scale, want_s) and _same_values(torch, q, want_q)
    index = torch.randint(-1, rows + 1, (2 * rows + 3,), device="cuda").to(torch.int32)
    q, scale = experts.quantize_blocks(handle, view, index, dtype=f8)
    real = (index >= 0) & (index < rows)
    at = index.long().clamp(0, rows - 1)
    assert torch.equal(scale, torch.where(real[:, None], want_s[at], 0.0))
    assert torch.equal(q.float(), torch.where(real[:, None], want_q.float()[at], 0.0))


@pytest.mark.parametrize("name", ["float8_e4m3fn", "float8_e5m2"])
def test_fp32_rows(handle, name):
    torch, api, experts = _setup()
    for rows, k in ((1, 5), (9, 300), (64, 2048)):
        for magnitude in (1.0, 1e-30, 1e30):
            x = torch.randn(rows, k, device="cuda") * magnitude
            q, scale = experts.quantize_blocks(handle, x, dtype=getattr(torch, name))
            each = _spread(scale, rows, k, False)
            off = (q.double() * each - x.double()).abs()
            assert (off <= (UNIT[name] + 2.0 ** -22) * x.double().abs() + TINY[name] * each).all()
            assert torch.equal(scale, _rows_quantised(torch, x, name)[1])


def test_special_blocks(handle):
    """Zeros, infinities, NaN, the largest and the smallest: of their block alone."""
    torch, api, experts = _setup()
    x = torch.randn(6, 400, device="cuda")
    x[0, 128:256] = 0
    x[1, 5] = float("inf")
    x[2, 399] = float("nan")
    x[3, 256:384] = torch.randn(128, device="cuda").sign() * 3.4028234663852886e38
    x[4, :128] = 2.0 ** -140
    x[5, 128:256] *= 2.0 ** -130
    clean = _rows_quantised(torch, x, "float8_e4m3fn")
    q, scale = experts.quantize_blocks(handle, x)
    value = q.float()
    assert scale[0, 1] == 0 and not value[0, 128:256].any()
    assert torch.isnan(scale[1, 0]) and not value[1, :128].any()
    assert torch.isnan(scale[2, 3]) and not value[2, 384:].any()
    assert (value[3, 256:384].abs() == 448).all()
    assert (value[4, :128].abs() == 448).all() and scale[4, 0] == clean[1][4, 0]
    each = scale[5, 1].double()
    assert ((value[5, 128:256].double() * each - x[5, 128:256].double()).abs() <=
            (2.0 ** -4 + 2.0 ** -10) * x[5, 128:256].double().abs() + 2.0 ** -10 * each + 448 * 2.0 ** -150).all()
    assert torch.isnan(scale).sum() == 2
    tiny = torch.full((1, 128), 2.0 ** -149, device="cuda")  # its scale is 0 in FP32
    q, scale = experts.quantize_blocks(handle, tiny)
    assert scale.item() == 0 and not q.float().any()


def _gate(torch, name, g):
    """(activation, bound of its own error) in 64 bits."""
    f = torch.nn.functional
    v = {"silu": lambda: g * torch.sigmoid(g), "gelu": lambda: g * torch.erfc(-g / 2 ** 0.5) / 2, "relu": lambda: g.clamp(min=0),
         "gelu_tanh": lambda: g * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3))}[name]()
    a = g.abs()
    return v, (8 + 6 * a + 2 * a ** 2 + a ** 3) * 2.0 ** -23 * v.abs() + a * 2.0 ** -126


def _holds(torch, q, scale, h, off, name):
    """8-bit rows that stand for h, which is known to `off`."""
    rows, k = h.shape
    each = _spread(scale, rows, k, False)
    far = (q.double() * each - h).abs()
    limit = off + (UNIT[name] + 2.0 ** -22) * (h.abs() + off) + TINY[name] * each
    assert (far <= limit).all(), float((far / limit.clamp(min=1e-300)).max())
    kb = (k + 127) // 128
    pad = lambda t: torch.nn.functional.pad(t, (0, kb * 128 - k)).view(rows, kb, 128)  # noqa: E731
    top, most = pad(h.abs()).amax(2), pad(off).amax(2)
    assert ((scale.double() * MOST[name] - top).abs() <= most + 2.0 ** -23 * top).all()


@pytest.mark.parametrize("name", ["float8_e4m3fn", "float8_e5m2"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "relu"])
def test_gated_rows(handle, name, dtype, activation):
    torch, api, experts = _setup()
    for rows, hidden in ((1, 1), (5, 130), (70, 1024), (3, 257)):
        x = (torch.randn(rows, 2 * hidden, device="cuda") * 2).to(getattr(torch, dtype))
        q, scale = experts.quantize_blocks(handle, x, activation=activation, dtype=getattr(torch, name))
        act, off = _gate(torch, activation, x[:, :hidden].double())
        up = x[:, hidden:].double()
        _holds(torch, q, scale, act * up, off * up.abs() + 2.0 ** -23 * (act * up).abs(), name)


@pytest.mark.parametrize("name", ["float8_e4m3fn", "float8_e5m2"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("experts_,n,k", [(1, 1, 1), (2, 129, 130), (3, 128, 256), (1, 300, 1000), (2, 40, 2047)])
def test_weights_exactly(handle, name, dtype, experts_, n, k):
    torch, api, experts = _setup()
    w = torch.randn(experts_, n, k, device="cuda").to(getattr(torch, dtype))
    nb, kb = (n + 127) // 128, (k + 127) // 128
    t = torch.nn.functional.pad(w.float(), (0, kb * 128 - k, 0, nb * 128 - n)).view(experts_, nb, 128, kb, 128)
    top = t.abs().amax((2, 4), keepdim=True)
    most = torch.full_like(top, MOST[name])
    want = (t * most / top).reshape(experts_, nb * 128, kb * 128)[:, :n, :k].to(getattr(torch, name))
    for source in (w, torch.nn.functional.pad(w, (3, 2))[..., 3:-2]):
        q, scale = experts.quantize_weight_blocks(handle, source, dtype=getattr(torch, name))
        assert torch.equal(scale, (top / most).view(experts_, nb, kb)) and _same_values(torch, q, want)
    if experts_ == 1:
        q, scale = experts.quantize_weight_blocks(handle, w[0], dtype=getattr(torch, name))
        assert q.shape == (n, k) and scale.shape == (nb, kb) and _same_values(torch, q, want[0])


def _operands(torch, experts, handle, rows, n, k, groups, seed, x_name="float8_e4m3fn", w_name="float8_e4m3fn"):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(rows, k, generator=g, device="cuda")
    x *= torch.rand(1, k, generator=g, device="cuda") * 3
    w = torch.randn(groups, n, k, generator=g, device="cuda") * k ** -0.5
    w[:, : n // 2] *= 4
    q, s = experts.quantize_blocks(handle, x, dtype=getattr(torch, x_name))
    wq, ws = experts.quantize_weight_blocks(handle, w, dtype=getattr(torch, w_name))
    return q, s, wq, ws


def _product(torch, q, s, wq, ws, counts, rows):
    """(y, bound) in 64 bits, without the rounding of the result."""
    groups, n, k = wq.shape
    y, off = (torch.zeros(rows, n, dtype=torch.float64, device="cuda") for _ in range(2))
    x = q.double() * _spread(s, rows, k, False)
    for e, (a, b) in enumerate(_spans(counts)):
        w = wq[e].double() * _spread(ws[e], n, k, True)
        y[a:b] = x[a:b] @ w.t()
        off[a:b] = (6 + (k + 127) // 128 / 4) * 2.0 ** -22 * (x[a:b].abs() @ w.abs().t())
    return y, off


def _close(torch, got, want, off):
    unit = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[got.dtype]
    limit = off + unit * (want.abs() + off) + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    far = (got.double() - want).abs()
    assert (far <= limit).all(), float((far / limit.clamp(min=1e-300)).max())


SHAPES = [  # n, k, rows of each expert, rows behind the last
    (64, 128, [1], 0), (256, 512, [5, 0, 300, 1], 7), (1, 1, [3, 2], 0), (129, 100, [64, 65], 1), (260, 1040, [257], 0),
    (72, 8192, [2, 0, 0, 9], 3), (1000, 200, [0, 700, 33], 0), (130, 127, [40, 1], 0), (64, 64, [0, 0], 5), (513, 640, [128, 256, 512], 0),
    (2048, 4096, [1], 0), (300, 65536, [3], 0), (4096, 256, [600], 0)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("n,k,counts,spare", SHAPES)
def test_products(handle, dtype, n, k, counts, spare):
    torch, api, experts = _setup()
    rows = sum(counts) + spare
    q, s, wq, ws = _operands(torch, experts, handle, rows, n, k, len(counts), n + k)
    s[sum(counts):] = float("nan")  # rows of no group count for nothing
    want, off = _product(torch, q, s, wq, ws, counts, rows)
    ends = _ends(torch, counts)
    y = experts.f8_matmul(handle, q, s, wq, ws, ends, out_dtype=getattr(torch, dtype))
    _close(torch, y, want, off)
    bias = torch.randn(len(counts), n, device="cuda")
    for e, (a, b) in enumerate(_spans(counts)):
        want[a:b] += bias[e].double()
        off[a:b] += 2.0 ** -24 * (want[a:b].abs() + off[a:b])
    _close(torch, experts.f8_matmul(handle, q, s, wq, ws, ends, bias=bias, out_dtype=getattr(torch, dtype)), want, off)
    if len(counts) == 1 and spare == 0:
        plain = experts.f8_matmul(handle, q, s, wq[0], ws[0], out_dtype=getattr(torch, dtype))
        assert torch.equal(plain, y)


@pytest.mark.parametrize("x_name", ["float8_e4m3fn", "float8_e5m2"])
@pytest.mark.parametrize("w_name", ["float8_e4m3fn", "float8_e5m2"])
def test_types_mixed(handle, x_name, w_name):
    torch, api, experts = _setup()
    counts = [100, 0, 77]
    q, s, wq, ws = _operands(torch, experts, handle, 177, 200, 300, 3, 1, x_name, w_name)
    want, off = _product(torch, q, s, wq, ws, counts, 177)
    _close(torch, experts.f8_matmul(handle, q, s, wq, ws, _ends(torch, counts), out_dtype=torch.float32), want, off)


def test_strides_and_alignment(handle):
    """Operands in rows that lie anywhere, scales in either order, results in a wider matrix."""
    torch, api, experts = _setup()
    counts, rows, n, k = [150, 0, 71], 221, 136, 272
    q, s, wq, ws = _operands(torch, experts, handle, rows, n, k, 3, 2)
    want, off = _product(torch, q, s, wq, ws, counts, rows)
    ends = _ends(torch, counts)
    first = experts.f8_matmul(handle, q, s, wq, ws, ends)
    _close(torch, first, want, off)

    def placed(t, pad, offset):
        *batch, r, c = t.shape
        count = r * (c + pad)
        for b in batch:
            count *= b
        buf = torch.full((offset + count,), 0x7f, dtype=torch.uint8, device="cuda").view(t.dtype)  # NaN of e4m3
        view = buf[offset:].view(*batch, r, c + pad)[..., :c]
        view.copy_(t)
        return view

    for pad, offset in ((16, 0), (1, 0), (0, 5), (7, 3)):
        assert torch.equal(experts.f8_matmul(handle, placed(q, pad, offset), s, placed(wq, pad, offset), ws, ends), first)
    assert torch.equal(experts.f8_matmul(handle, q, s.contiguous(), wq, ws, ends), first)
    wide = torch.randn(rows, 9, device="cuda")
    wide[:, 3:6] = s
    assert torch.equal(experts.f8_matmul(handle, q, wide[:, 3:6], wq, ws, ends), first)
    one = torch.full((1, 1), 0.5, device="cuda").expand(rows, 3)  # one scale for everything
    want, off = _product(torch, q, one, wq, ws, counts, rows)
    _close(torch, experts.f8_matmul(handle, q, one, wq, ws, ends), want, off)
    for dtype in (torch.bfloat16, torch.float32):
        for pad, offset in ((8, 8), (3, 1)):
            buf = torch.full((offset + rows * (n + pad),), 7.0, dtype=dtype, device="cuda")
            out = buf[offset:].view(rows, n + pad)[:, :n]
            assert experts.f8_matmul(handle, q, s, wq, ws, ends, out=out) is out
            assert torch.equal(out, experts.f8_matmul(handle, q, s, wq, ws, ends, out_dtype=dtype))
            assert (buf[:offset] == 7).all() and (buf[offset:].view(rows, -1)[:, n:] == 7).all()


@pytest.mark.parametrize("name", ["float8_e4m3fn", "float8_e5m2"])
@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("hidden,k,counts,spare", [(128, 128, [1], 0), (256, 300, [5, 0, 300, 1], 7), (384, 64, [64, 65], 0),
                                                   (128, 4096, [2, 0, 9], 3), (1024, 512, [700, 33], 0), (100, 256, [30, 4], 2),
                                                   (129, 130, [0, 200], 0)])
def test_gated_products(handle, name, activation, hidden, k, counts, spare):
    torch, api, experts = _setup()
    rows = sum(counts) + spare
    q, s, wq, ws = _operands(torch, experts, handle, rows, 2 * hidden, k, len(counts), hidden + k)
    s[sum(counts):] = float("nan")
    pre, off = _product(torch, q, s, wq, ws, counts, rows)
    if hidden % 128:  # by way of FP32
        off = off + 2.0 ** -24 * pre.abs()
    gate, up, eg, eu = pre[:, :hidden], pre[:, hidden:], off[:, :hidden], off[:, hidden:]
    act, own = _gate(torch, activation, gate)
    h = act * up
    far = (1.13 * eg + own) * (up.abs() + eu) + act.abs() * eu + 2.0 ** -22 * h.abs()
    got, scale = experts.f8_gated_matmul(handle, q, s, wq, ws, _ends(torch, counts), activation=activation,
                                         dtype=getattr(torch, name))
    assert got.shape == (rows, hidden) and got.dtype == getattr(torch, name)
    _holds(torch, got, scale, h, far, name)
    assert not got[sum(counts):].float().any() and not scale[sum(counts):].any()
    if len(counts) == 1:
        again = experts.f8_gated_matmul(handle, q, s, wq[0], ws[0], activation=activation, dtype=getattr(torch, name))
        assert _same_values(torch, again[0], got) and torch.equal(again[1], scale)


def test_a_block_from_end_to_end(handle):
    """Quantise and gather, gated product, product: as a layer of experts is served; against the same in 64 bits from each
    step's operands, and near the layer that is not quantised."""
    torch, api, experts = _setup()
    tokens, topk, width, hidden, num = 90, 2, 256, 384, 4
    x = torch.randn(tokens, width, device="cuda", dtype=torch.bfloat16)
    gate_up = (torch.randn(num, 2 * hidden, width, device="cuda") * width ** -0.5).bfloat16()
    down = (torch.randn(num, width, hidden, device="cuda") * hidden ** -0.5).bfloat16()
    counts = [70, 0, 100, 10]
    index = (torch.randperm(tokens * topk, device="cuda") // topk).to(torch.int32)
    ends = _ends(torch, counts)
    guq, gus = experts.quantize_weight_blocks(handle, gate_up)
    dq, ds = experts.quantize_weight_blocks(handle, down)
    q, s = experts.quantize_blocks(handle, x, index)
    hq, hs = experts.f8_gated_matmul(handle, q, s, guq, gus, ends)
    y = experts.f8_matmul(handle, hq, hs, dq, ds, ends)
    want, off = _product(torch, hq, hs, dq, ds, counts, tokens * topk)
    _close(torch, y, want, off)
    full = experts.gated_feed_forward(handle, x[index.long()], gate_up, down, ends).double()
    # each of the five operands of 8 bits is off by at most 2^-4 of an element, some 2^-4 / 2 in the mean, and the
    # errors of a sum's terms are independent: 5^(1/2) 2^-5 of the norm at most
    assert float((y.double() - full).norm() / full.norm()) < 5 ** 0.5 * 2.0 ** -5


def test_nan_and_infinity_stay_where_they_are(handle):
    torch, api, experts = _setup()
    counts, rows, n, k = [20, 30], 50, 300, 400
    x = torch.randn(rows, k, device="cuda")
    w = torch.randn(2, n, k, device="cuda")
    ends = _ends(torch, counts)
    wq, ws = experts.quantize_weight_blocks(handle, w)
    clean = experts.f8_matmul(handle, *experts.quantize_blocks(handle, x), wq, ws, ends)
    x[3, 200] = float("inf")
    x[40, 399] = float("nan")
    w[1, 130, 7] = float("nan")
    y = experts.f8_matmul(handle, *experts.quantize_blocks(handle, x), *experts.quantize_weight_blocks(handle, w), ends)
    want = torch.isnan(torch.zeros_like(clean))
    want[3] = want[40] = True
    want[20:, 128:256] = True
    assert torch.equal(torch.isnan(y), want) and torch.equal(y[~want], clean[~want])


def test_slices_of_k_with_and_without_room(handle):
    """Few tiles are cut along K where there is memory for their sums; without it they stay whole."""
    torch, api, experts = _setup()
    for rows, n, k in ((1, 512, 8192), (300, 256, 16384)):
        q, s, wq, ws = _operands(torch, experts, handle, rows, 2 * n, k, 1, 5)
        want, off = _product(torch, q, s, wq, ws, [rows], rows)
        cut = experts.f8_matmul(handle, q, s, wq, ws, out_dtype=torch.float32)
        again = experts.f8_matmul(handle, q, s, wq, ws, out_dtype=torch.float32)
        gated = experts.f8_gated_matmul(handle, q, s, wq, ws)
        assert torch.equal(cut, again)
        handle.set_workspace_limit(1 << 20)
        whole = experts.f8_matmul(handle, q, s, wq, ws, out_dtype=torch.float32)
        gated_whole = experts.f8_gated_matmul(handle, q, s, wq, ws)
        handle.set_workspace_limit(0)
        _close(torch, cut, want, off)
        _close(torch, whole, want, off)
        act, own = _gate(torch, "silu", want[:, :n])
        far = (1.13 * off[:, :n] + own) * (want[:, n:].abs() + off[:, n:]) + act.abs() * off[:, n:] + 2.0 ** -22 * (act * want[:, n:]).abs()
        for g in (gated, gated_whole):
            _holds(torch, *g, act * want[:, n:], far, "float8_e4m3fn")


@pytest.mark.parametrize("counts", [[1000], [400, 0, 580]])
def test_the_larger_kernel_cut_along_k(handle, counts):
    """Too many rows for the kernel for few of them, and few enough tiles to be cut; without room they stay whole."""
    torch, api, experts = _setup()
    rows, hidden, k = sum(counts), 1024, 6000
    q, s, wq, ws = _operands(torch, experts, handle, rows, 2 * hidden, k, len(counts), 8)
    want, off = _product(torch, q, s, wq, ws, counts, rows)
    ends = _ends(torch, counts)
    act, own = _gate(torch, "silu", want[:, :hidden])
    far = (1.13 * off[:, :hidden] + own) * (want[:, hidden:].abs() + off[:, hidden:]) + act.abs() * off[:, hidden:]
    far += 2.0 ** -22 * (act * want[:, hidden:]).abs()
    for limit in (0, 1 << 20):
        handle.set_workspace_limit(limit)
        y = experts.f8_matmul(handle, q, s, wq, ws, ends, out_dtype=torch.float32)
        assert torch.equal(y, experts.f8_matmul(handle, q, s, wq, ws, ends, out_dtype=torch.float32))
        _close(torch, y, want, off)
        _holds(torch, *experts.f8_gated_matmul(handle, q, s, wq, ws, ends), act * want[:, hidden:], far, "float8_e4m3fn")
    handle.set_workspace_limit(0)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("n", [1152, 1160, 1153])
@pytest.mark.parametrize("pad,offset", [(8, 8), (0, 0), (3, 1)])
def test_results_of_the_larger_kernel(handle, dtype, n, pad, offset):
    """Groups that end inside 32 rows, columns that end inside a tile, results in a wider matrix: nothing else is written."""
    torch, api, experts = _setup()
    counts, spare, k, dtype = [300, 77, 0, 513, 310], 37, 200, getattr(torch, dtype)
    rows = sum(counts) + spare
    q, s, wq, ws = _operands(torch, experts, handle, rows, n, k, len(counts), n + pad)
    want, off = _product(torch, q, s, wq, ws, counts, rows)
    bias = torch.randn(len(counts), n, device="cuda")
    for e, (a, b) in enumerate(_spans(counts)):
        want[a:b] += bias[e].double()
        off[a:b] += 2.0 ** -24 * (want[a:b].abs() + off[a:b])
    buf = torch.full((offset + rows * (n + pad),), 7.0, dtype=dtype, device="cuda")
    out = buf[offset:].view(rows, n + pad)[:, :n]
    for _ in range(3):  # one behind the other
        experts.f8_matmul(handle, q, s, wq, ws, _ends(torch, counts), bias=bias, out=out)
    _close(torch, out, want, off)
    assert (buf[:offset] == 7).all() and (buf[offset:].view(rows, -1)[:, n:] == 7).all()


@pytest.mark.parametrize("pad,offset", [(16, 16), (0, 0), (3, 1)])
def test_gated_results_of_the_larger_kernel(handle, pad, offset):
    torch, api, experts = _setup()
    counts, spare, k, hidden, E4M3 = [300, 77, 0, 513, 310], 37, 200, 1152, api.CUDA_R_8F_E4M3
    rows = sum(counts) + spare
    q, s, wq, ws = _operands(torch, experts, handle, rows, 2 * hidden, k, len(counts), 9)
    ends = _ends(torch, counts)
    first, first_scale = experts.f8_gated_matmul(handle, q, s, wq, ws, ends)
    want, off = _product(torch, q, s, wq, ws, counts, rows)
    act, own = _gate(torch, "silu", want[:, :hidden])
    far = (1.13 * off[:, :hidden] + own) * (want[:, hidden:].abs() + off[:, hidden:]) + act.abs() * off[:, hidden:]
    far += 2.0 ** -22 * (act * want[:, hidden:]).abs()
    _holds(torch, first, first_scale, act * want[:, hidden:], far, "float8_e4m3fn")
    buf = torch.full((offset + rows * (hidden + pad),), 7, dtype=torch.uint8, device="cuda")
    out = buf[offset:].view(rows, hidden + pad)[:, :hidden]
    scale = torch.full((rows, hidden // 128 + 1), 7.0, device="cuda")
    handle.f8_grouped_gemm_gated(rows, hidden, k, len(counts), ends, q.data_ptr(), q.stride(0), E4M3, s.data_ptr(), *s.stride(),
                                 wq.data_ptr(), wq.stride(1), wq.stride(0), E4M3, ws.data_ptr(), 0, out.data_ptr(), hidden + pad,
                                 E4M3, scale.data_ptr(), hidden // 128 + 1, 1)
    assert torch.equal(out, first.view(torch.uint8)) and torch.equal(scale[:, :-1], first_scale)
    assert (buf[:offset] == 7).all() and (buf[offset:].view(rows, -1)[:, hidden:] == 7).all() and (scale[:, -1] == 7).all()


@pytest.mark.parametrize("counts", [[200, 3, 0, 0, 0, 0, 37, 0], [0, 0, 256, 0, 0, 0, 0, 0], [31, 32, 33, 64, 65, 7, 0, 24]])
def test_few_rows_unevenly_spread(handle, counts):
    """At most 32 rows a group on average, some of them with more; the same numbers as one group after another, and for
    the gated product with and without room for the FP32 products in between."""
    torch, api, experts = _setup()
    rows, hidden, k = sum(counts), 640, 700
    q, s, wq, ws = _operands(torch, experts, handle, rows, 2 * hidden, k, 8, 6)
    want, off = _product(torch, q, s, wq, ws, counts, rows)
    ends = _ends(torch, counts)
    y = experts.f8_matmul(handle, q, s, wq, ws, ends, out_dtype=torch.float32)
    _close(torch, y, want, off)
    act, own = _gate(torch, "gelu", want[:, :hidden])
    far = (1.13 * off[:, :hidden] + own) * (want[:, hidden:].abs() + off[:, hidden:]) + act.abs() * off[:, hidden:]
    far += 2.0 ** -22 * (act * want[:, hidden:]).abs()
    for limit in (0, 4096):
        handle.set_workspace_limit(limit)
        _holds(torch, *experts.f8_gated_matmul(handle, q, s, wq, ws, ends, activation="gelu"), act * want[:, hidden:], far,
               "float8_e4m3fn")
    handle.set_workspace_limit(0)


def test_totals_that_are_wrong(handle):
    torch, api, experts = _setup()
    q, s, wq, ws = _operands(torch, experts, handle, 90, 256, 128, 4, 3)
    bad = torch.tensor([30, -5, 2000000000, 7], dtype=torch.int32).cuda()
    good = _ends(torch, [30, 0, 60, 0])
    assert torch.equal(experts.f8_matmul(handle, q, s, wq, ws, bad), experts.f8_matmul(handle, q, s, wq, ws, good))
    a, b = (experts.f8_gated_matmul(handle, q, s, wq, ws, e) for e in (bad, good))
    assert _same_values(torch, a[0], b[0]) and torch.equal(a[1], b[1])


def test_many_groups(handle):
    torch, api, experts = _setup()
    counts = [(7 * i) % 5 for i in range(1024)]
    rows = sum(counts)
    q, s, wq, ws = _operands(torch, experts, handle, rows, 40, 136, 1024, 4)
    want, off = _product(torch, q, s, wq, ws, counts, rows)
    _close(torch, experts.f8_matmul(handle, q, s, wq, ws, _ends(torch, counts)), want, off)


def test_replayed_from_a_graph_and_on_two_streams(handle):
    torch, api, experts = _setup()
    counts = [40, 0, 25]
    x, ends = torch.randn(65, 256, device="cuda", dtype=torch.bfloat16), _ends(torch, counts)
    gate_up, down = torch.randn(3, 512, 256, device="cuda"), torch.randn(3, 256, 256, device="cuda")
    weights = (*experts.quantize_weight_blocks(handle, gate_up), *experts.quantize_weight_blocks(handle, down))

    def serve(h, x, ends):
        q, s = experts.f8_gated_matmul(h, *experts.quantize_blocks(h, x), *weights[:2], ends)
        return experts.f8_matmul(h, q, s, *weights[2:], ends)

    serve(handle, x, ends)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        handle.use_current_torch_stream()
        out = serve(handle, x, ends)
    handle.use_current_torch_stream()
    for seed, counts in ((1, [40, 0, 25]), (2, [0, 65, 0])):
        torch.manual_seed(seed)
        fresh, now = torch.randn_like(x), _ends(torch, counts)
        x.copy_(fresh)
        ends.copy_(now)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.clone(), serve(handle, fresh, now))
    # a handle of its own for each stream, both at work at once
    want = serve(handle, x, ends)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    handles, got = [], []
    for st in streams:
        with torch.cuda.stream(st):
            h = api.Handle()
            h.use_current_torch_stream()
            handles.append(h)
    for _ in range(20):
        for h, st in zip(handles, streams):
            with torch.cuda.stream(st):
                got.append(serve(h, x, ends))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    for h in handles:
        assert h.kernel_status() == 0
        h.destroy()


def test_refusals(handle):
    torch, api, experts = _setup()
    q, s, wq, ws = _operands(torch, experts, handle, 8, 256, 200, 2, 1)
    ends = _ends(torch, [4, 4])
    x = torch.randn(8, 200, device="cuda")
    for bad in (lambda: experts.f8_matmul(handle, q, s[:, :1], wq, ws, ends),
                lambda: experts.f8_matmul(handle, q, s.double(), wq, ws, ends),
                lambda: experts.f8_matmul(handle, q, s, wq, ws[:, :1], ends),
                lambda: experts.f8_matmul(handle, q, s, wq, ws.transpose(1, 2), ends),
                lambda: experts.f8_matmul(handle, q.view(torch.int8), s, wq, ws, ends),
                lambda: experts.f8_matmul(handle, q, s, wq.float(), ws, ends),
                lambda: experts.f8_matmul(handle, q, s, wq, ws),
                lambda: experts.f8_matmul(handle, q[:, :199], s, wq, ws, ends),
                lambda: experts.f8_matmul(handle, q, s, wq, ws, ends, bias=torch.zeros(2, 255, device="cuda")),
                lambda: experts.f8_matmul(handle, q, s, wq, ws, ends, out_dtype=torch.float8_e4m3fn),
                lambda: experts.f8_matmul(handle, q, s, wq, ws, ends.long()),
                lambda: experts.f8_matmul(handle, q, s, wq, ws, ends, out=torch.empty(8, 255, device="cuda")),
                lambda: experts.f8_gated_matmul(handle, q, s, wq[:, :255], ws, ends),
                lambda: experts.f8_gated_matmul(handle, q, s, wq, ws, ends, activation="none"),
                lambda: experts.f8_gated_matmul(handle, q, s, wq, ws, ends, dtype=torch.float16),
                lambda: experts.quantize_blocks(handle, x, dtype=torch.int8),
                lambda: experts.quantize_blocks(handle, x.double()),
                lambda: experts.quantize_blocks(handle, x[:, :199], activation="silu"),
                lambda: experts.quantize_blocks(handle, x, torch.zeros(3, device="cuda")),
                lambda: experts.quantize_weight_blocks(handle, x, dtype=torch.float32),
                lambda: experts.quantize_weight_blocks(handle, x.t())):
        with pytest.raises(ValueError):
            bad()
    invalid = api.CUBLAS_STATUS_INVALID_VALUE
    place = (ends, q, 208, 28, s, 1, 8, wq, 208, 256 * 208, 28, ws)
    y = torch.empty(8, 256, device="cuda")
    assert handle.f8_grouped_gemm(8, 256, 200, 2, *place, None, y, 255, api.CUDA_R_32F, check=False) == invalid
    assert handle.f8_grouped_gemm(8, 256, 200, 2, *place, None, y, 256, api.CUDA_R_8F_E4M3, check=False) == invalid
    assert handle.f8_grouped_gemm_gated(8, 100, 200, 2, *place, 0, y, 256, 28, y, 1, 8, check=False) == invalid
    assert handle.f8_grouped_gemm_gated(8, 128, 200, 2, *place, -1, y, 256, 28, y, 1, 8, check=False) == invalid
    assert handle.f8_grouped_gemm_gated(8, 128, 200, 2, *place, 0, y, 256, 0, y, 1, 8, check=False) == invalid
    assert handle.quantize_rows_f8(8, 200, x, 200, 0, None, 7, -1, y, 200, 28, y, 1, 8, check=False) == invalid
    assert handle.quantize_rows_f8(8, 200, x, 200, 0, None, 8, 0, y, 200, 28, y, 1, 8, check=False) == invalid
    assert handle.quantize_blocks_f8(2, 8, 100, x, 100, 700, 0, y, 100, 800, 28, y, check=False) == invalid
    empty = experts.f8_matmul(handle, q[:0], s[:0], wq, ws, _ends(torch, [0, 0]))
    assert empty.shape == (0, 256)
    assert experts.quantize_blocks(handle, x[:0])[0].shape == (0, 200)


def test_offsets_past_32_bits(handle):
    """Rows behind 2^32 bytes of operands and results; 128 values of k, so that the sums are the same in any call."""
    torch, api, experts = _setup()
    rows, k, n, last = 140000, 128, 32768, 300
    q, s, wq, ws = _operands(torch, experts, handle, rows, n, k, 1, 4)
    y = experts.f8_matmul(handle, q, s, wq, ws)
    few = (q[-last:], s[-last:].t().contiguous().t())
    assert torch.equal(y[-last:], experts.f8_matmul(handle, *few, wq, ws))
    part = experts.quantize_blocks(handle, y[-last:])
    whole = experts.quantize_blocks(handle, y)
    assert torch.equal(whole[0][-last:].view(torch.uint8), part[0].view(torch.uint8)) and torch.equal(whole[1][-last:], part[1])
    w, index = torch.randn(1, 128, n, device="cuda"), torch.tensor([rows - 1, 0, rows], dtype=torch.int32, device="cuda")
    wq, ws = experts.quantize_weight_blocks(handle, w)
    tail = experts.f8_matmul(handle, *whole, wq, ws, out_dtype=torch.float32)[-last:]
    want, off = _product(torch, *part, wq, ws, [last], last)
    _close(torch, tail, want, off)
    gathered = experts.quantize_blocks(handle, y, row_index=index)[0].view(torch.uint8)
    assert torch.equal(gathered[0], part[0][-1].view(torch.uint8)) and not gathered[2].any()
    q, s = experts.f8_gated_matmul(handle, *few, *experts.quantize_weight_blocks(handle, torch.randn(1, 2 * n, k, device="cuda")))
    assert q.shape == (last, n) and torch.isfinite(s).all()
