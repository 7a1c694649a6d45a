"""Gated feed-forward blocks against their definition in 64 bits.

Every tolerance is a bound that is carried along with the value, element by element (``_Value``: a value in 64 bits
and how far the computed one may be from it):
* a product x w of K terms: what x and w are off by, and the FP32 sums.  With S = sum |x| |w|, 16-bit operands are
  added 16 at a time by the tensor core, which truncates: (K / 16 + 1) 2^-22 S.  FP32 operands: (13 + K / 512) 2^-22 S
  for the split and the sums, and 2^-36 of the sum of |x| and |w| where lo halves are subnormal (FP16TCEC).
* a rounding to 16 bits: 2^-8 (bfloat16) or 2^-11 (float16) of the value, and half the smallest subnormal of float16.
* an activation: exp to (2 + 1.173 |v|) 2^-23 of itself, a quotient to 2^-22, erfc to 4 units in the last place, their
  arguments' roundings: together (8 + 6 |g| + 2 g^2 + |g|^3) 2^-23 of the value, as much times 1 + |g| for a slope.
  The slope of each is at most 1.13, its slope at most 0.8; relu's jumps at 0.
"""
import itertools

import pytest

pytestmark = pytest.mark.gpu

ACTIVATIONS = ["silu", "gelu", "gelu_tanh", "relu"]


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


def _placed(torch, values, ld, offset):
    """The values in rows `ld` apart, `offset` elements into their allocation, NaN in between."""
    *batch, rows, cols = values.shape
    count = rows * ld
    for b in batch:
        count *= b
    buf = torch.full((offset + count,), float("nan"), dtype=values.dtype, device="cuda")
    view = buf[offset:].view(*batch, rows, ld)[..., :cols]
    view.copy_(values)
    return view


class _Value:
    def __init__(self, v, off=None):
        self.v = v.double()
        self.off = self.v.new_zeros(self.v.shape) if off is None else off

    def rounded(self, torch, dtype):
        if dtype == torch.float32:
            return _Value(self.v, self.off + 2.0 ** -24 * (self.v.abs() + self.off))
        unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
        return _Value(self.v, self.off + unit * (self.v.abs() + self.off) + (2.0 ** -25 if dtype == torch.float16 else 0.0))

    def t(self):
        return _Value(self.v.t(), self.off.t())

    def __getitem__(self, at):
        return _Value(self.v[at], self.off[at])


def _product(torch, dtype, x, w):
    """x w of matrices with bounds."""
    k = x.v.shape[1]
    ax, aw = x.v.abs(), w.v.abs()
    size = (ax + x.off) @ (aw + w.off)
    if dtype == torch.float32:
        off = (13 + k / 512) * 2.0 ** -22 * size + 2.0 ** -36 * (ax.sum(1, keepdim=True) + aw.sum(0, keepdim=True))
    else:
        off = (k / 16 + 1) * 2.0 ** -22 * size
    return _Value(x.v @ w.v, off + x.off @ (aw + w.off) + ax @ w.off)


def _act(torch, name, v):
    import math

    if name == "relu":
        return v.clamp(min=0), (v > 0).double()
    if name == "silu":
        p = 1 / (1 + torch.exp(-v))
        return v * p, p * (1 + v * (1 - p))
    if name == "gelu":
        p = 0.5 * torch.erfc(-v / math.sqrt(2))
        return v * p, p + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    r = math.sqrt(2 / math.pi)  # (1 + tanh z) / 2 = 1 / (1 + exp(-2 z)), which cancels nothing
    z = r * (v + 0.044715 * v ** 3)
    p, q = torch.sigmoid(2 * z), torch.sigmoid(-2 * z)
    return v * p, p + 2 * v * p * q * r * (1 + 3 * 0.044715 * v * v)


def _activated(torch, name, g):
    """(activation, slope) of g, each with its bound."""
    value, slope = _act(torch, name, g.v)
    a = g.v.abs() + g.off
    own = (8 + 6 * a + 2 * a ** 2 + a ** 3) * 2.0 ** -23
    jump = (g.v.abs() <= g.off).double() if name == "relu" else 0.8 * g.off
    # Where exp(-v) passes 2^126 the fast quotient p = 1 / (1 + exp(-v)) is 0 for at most 2^-126: g p loses |g| 2^-126,
    # and the slope p + 2 g p (1 - p) z', with z' at most 1 + g^2, (1 + 2 |g| (1 + g^2)) 2^-126.
    lost = 2.0 ** -126
    return (_Value(value, 1.13 * g.off + own * (value.abs() + 1.13 * g.off) + a * lost),
            _Value(slope, jump + own * (1 + a) + (1 + 2 * a * (1 + a * a)) * lost))


def _times(*values):
    """Their product in FP32."""
    v, off = values[0].v, values[0].off
    for x in values[1:]:
        off = off * (x.v.abs() + x.off) + v.abs() * x.off
        v = v * x.v
        off = off + 2.0 ** -24 * (v.abs() + off)
    return _Value(v, off)


def _block(torch, dtype, name, x, gate_up, down, dy, counts, rows):
    """{name: _Value} of everything a block computes, rows of no group being 0; gradients where dy is given."""
    h, w = gate_up.shape[1] // 2, x.shape[1]
    zero = lambda *s: _Value(torch.zeros(*s, dtype=torch.float64, device="cuda"))  # noqa: E731
    out = {"h": zero(rows, h), "pre": zero(rows, 2 * h), "y": zero(rows, w), "dpre": zero(rows, 2 * h), "dx": zero(rows, w),
           "dgate_up": zero(*gate_up.shape), "ddown": zero(gate_up.shape[0], w, h)}

    def put(key, at, value):
        out[key].v[at], out[key].off[at] = value.v, value.off

    for e, (a, b) in enumerate(_spans(counts)):
        here = slice(a, b)
        xe, gu = _Value(x[here]), _Value(gate_up[e])
        raw = _product(torch, dtype, xe, gu.t())
        pre = raw.rounded(torch, dtype) if dtype != torch.float32 else raw
        put("pre", here, pre)
        act, _ = _activated(torch, name, raw[:, :h])
        hid = _times(act, raw[:, h:]).rounded(torch, dtype)
        put("h", here, hid)
        if down is None:
            continue
        dn = _Value(down[e])
        put("y", here, _product(torch, dtype, hid, dn.t()).rounded(torch, dtype))
        if dy is None:
            continue
        dye = _Value(dy[here])
        dh = _product(torch, dtype, dye, dn)
        if dtype == torch.float32:
            dh = dh.rounded(torch, dtype)
        act, slope = _activated(torch, name, pre[:, :h])
        parts = _times(dh, pre[:, h:], slope), _times(dh, act)
        dpre = _Value(torch.cat([p.v for p in parts], 1), torch.cat([p.off for p in parts], 1)).rounded(torch, dtype)
        put("dpre", here, dpre)
        put("dx", here, _product(torch, dtype, dpre, gu).rounded(torch, dtype))
        put("dgate_up", e, _product(torch, dtype, dpre.t(), xe).rounded(torch, dtype))
        put("ddown", e, _product(torch, dtype, dye.t(), hid).rounded(torch, dtype))
    return out


def _close(got, want, what):
    off = (got.double() - want.v).abs()
    bad = ~(off <= want.off)
    assert not bad.any(), (what, int(bad.sum()), float((off / want.off.clamp(min=1e-300)).max()))


def _operands(torch, dtype, rows, hidden, width, experts, seed, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    new = lambda *s, by=1.0: torch.randn(*s, generator=g, device="cuda").mul_(by).to(dtype)  # noqa: E731
    return (new(rows, width), new(experts, 2 * hidden, width, by=width ** -0.5),
            new(experts, width, hidden, by=hidden ** -0.5), new(rows, width, by=scale))


SHAPES = [  # hidden, width, rows of each expert, rows behind the last
    (16, 64, [1], 0), (128, 128, [5, 0, 300, 1], 7), (1, 8, [3, 2], 0), (129, 100, [64, 65], 1),
    (264, 520, [257], 0), (72, 4096, [2, 0, 0, 9], 3), (1000, 200, [0, 700, 33], 0), (33, 1, [40, 1], 0),
    (64, 64, [0, 0], 5), (520, 1032, [128, 256, 512], 0)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("hidden,width,counts,spare", SHAPES)
def test_block_and_its_gradients(handle, dtype, hidden, width, counts, spare):
    torch, api, experts = _setup()
    dtype = getattr(torch, dtype)
    rows = sum(counts) + spare
    name = ACTIVATIONS[(hidden + width) % 4]
    x, gate_up, down, dy = _operands(torch, dtype, rows, hidden, width, len(counts), hidden + rows)
    x[sum(counts):] = float("nan")  # rows of no group count for nothing
    dy[sum(counts):] = float("nan")
    want = _block(torch, dtype, name, x, gate_up, down, dy, counts, rows)
    leaves = [t.detach().requires_grad_() for t in (x, gate_up, down)]
    y = experts.gated_feed_forward(handle, *leaves, _ends(torch, counts), activation=name)
    grads = torch.autograd.grad(y, leaves, dy)
    for key, got in zip(("y", "dx", "dgate_up", "ddown"), (y, *grads)):
        _close(got, want[key], key)
    with torch.no_grad():
        assert torch.equal(experts.gated_feed_forward(handle, x, gate_up, down, _ends(torch, counts), activation=name), y)
        h = experts.gated_matmul(handle, x, gate_up, _ends(torch, counts), activation=name)
    _close(h, want["h"], "h")


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("name", ACTIVATIONS)
def test_gated_matmul_and_its_gradients(handle, dtype, name):
    torch, api, experts = _setup()
    dtype, counts, hidden, width = getattr(torch, dtype), [70, 0, 31], 200, 96
    rows = sum(counts)
    x, gate_up, _, _ = _operands(torch, dtype, rows, hidden, width, 3, 11)
    x *= 3  # gates of about -10 to 10
    dh = torch.randn(rows, hidden, device="cuda").to(dtype)
    want = _block(torch, dtype, name, x, gate_up, None, None, counts, rows)
    xs, ws = x.detach().requires_grad_(), gate_up.detach().requires_grad_()
    h = experts.gated_matmul(handle, xs, ws, _ends(torch, counts), activation=name)
    _close(h, want["h"], "h")
    dx, dw = torch.autograd.grad(h, (xs, ws), dh)
    for e, (a, b) in enumerate(_spans(counts)):
        pre = want["pre"][slice(a, b)]
        act, slope = _activated(torch, name, pre[:, :hidden])
        parts = _times(_Value(dh[a:b]), pre[:, hidden:], slope), _times(_Value(dh[a:b]), act)
        dpre = _Value(torch.cat([p.v for p in parts], 1), torch.cat([p.off for p in parts], 1)).rounded(torch, dtype)
        _close(dx[a:b], _product(torch, dtype, dpre, _Value(gate_up[e])).rounded(torch, dtype), "dx")
        _close(dw[e], _product(torch, dtype, dpre.t(), _Value(x[a:b])).rounded(torch, dtype), "dgate_up")


FEW = [  # hidden, width, rows of each expert, rows behind the last: eight rows or fewer
    (1, 8, [1], 0), (5, 64, [2], 1), (8, 1000, [3, 0, 2], 2), (129, 4096, [8], 0), (72, 200, [1] * 4 + [0] * 60, 0),
    (520, 72, [0, 0], 4), (33, 2056, [0] * 300 + [1, 0, 5], 1), (64, 1024, [7], 1), (16, 520, [0, 4, 0, 4], 0)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("pad", [0, 8])
@pytest.mark.parametrize("hidden,width,counts,spare", FEW)
def test_few_rows(handle, dtype, pad, hidden, width, counts, spare):
    """A handful of rows, for one expert or for many; nothing outside h and pre is touched."""
    torch, api, experts = _setup()
    dtype, rows, n = getattr(torch, dtype), sum(counts) + spare, len(counts)
    name = ACTIVATIONS[(hidden + width // 8) % 4]
    x, gate_up, _, _ = _operands(torch, dtype, rows, hidden, width, n, hidden + width)
    x[sum(counts):] = float("nan")  # rows of no group count for nothing, nor do weights without rows
    for e in range(n):
        if counts[e] == 0:
            gate_up[e] = float("nan")
    want = _block(torch, dtype, name, x, gate_up, None, None, counts, rows)
    xs, ws = _placed(torch, x, width + pad, 0), _placed(torch, gate_up, width + pad, 0)
    hid = _placed(torch, torch.zeros(rows, hidden, dtype=dtype, device="cuda"), hidden + 3, 1)
    pre = _placed(torch, torch.zeros(rows, 2 * hidden, dtype=dtype, device="cuda"), 2 * hidden + 1, 1)
    # (totals that fall back or are too large are the one in front and the number of rows)
    ends = _ends(torch, counts)
    handle.grouped_gemm_gated(rows, hidden, width, n, ends, xs.data_ptr(), width + pad, ws.data_ptr(), width + pad,
                              2 * hidden * (width + pad), experts._activation(name), hid.data_ptr(), hidden + 3,
                              pre.data_ptr(), 2 * hidden + 1, experts._data_type(dtype))
    _close(hid, want["h"], "h")
    _close(pre, want["pre"], "pre")
    for t, cols, ld in ((hid, hidden, hidden + 3), (pre, 2 * hidden, 2 * hidden + 1)):
        base = t._base.view(-1)
        assert torch.isnan(base[:1]).all() and torch.isnan(base[1:].view(rows, ld)[:, cols:]).all()
    assert torch.equal(experts.gated_matmul(handle, xs, ws, ends, activation=name), hid)
    if spare == 0 and n > 1:
        wrong = ends.clone()
        wrong[-1] = rows + 100
        wrong[1:-1] -= torch.arange(n - 2, device="cuda", dtype=torch.int32) % 2 * (wrong[1:-1] == wrong[:-2]).int()
        assert torch.equal(experts.gated_matmul(handle, xs, ws, wrong, activation=name), hid)
    assert handle.kernel_status() == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 8), (3, 1), (5, 0)])
@pytest.mark.parametrize("hidden", [40, 37])
def test_any_leading_dimension_and_alignment(handle, dtype, pad, offset, hidden):
    """Operands, h, pre and the gradient of pre in rows that lie anywhere; nothing outside them is touched."""
    torch, api, experts = _setup()
    dtype, counts, width, name = getattr(torch, dtype), [130, 0, 61], 72, "gelu"
    rows, h = sum(counts), hidden
    x, gate_up, down, dy = _operands(torch, dtype, rows, hidden, width, 3, 5)
    want = _block(torch, dtype, name, x, gate_up, down, dy, counts, rows)
    place = lambda t: _placed(torch, t, t.shape[-1] + pad, offset)  # noqa: E731
    xs, ws, ds, dys = (place(t) for t in (x, gate_up, down, dy))
    hid = place(torch.zeros(rows, h, dtype=dtype, device="cuda"))
    pre, dpre = (place(torch.zeros(rows, 2 * h, dtype=dtype, device="cuda")) for _ in range(2))
    ends, act, kind = _ends(torch, counts), experts._activation(name), experts._data_type(dtype)
    handle.grouped_gemm_gated(rows, h, width, 3, ends, xs.data_ptr(), width + pad, ws.data_ptr(), width + pad,
                              2 * h * (width + pad), act, hid.data_ptr(), h + pad, pre.data_ptr(), 2 * h + pad, kind)
    _close(hid, want["h"], "h")
    _close(pre, want["pre"], "pre")
    handle.grouped_gemm_gated_grad(api.CUBLAS_OP_N, rows, h, width, 3, ends, dys.data_ptr(), width + pad, ds.data_ptr(),
                                   h + pad, width * (h + pad), act, pre.data_ptr(), 2 * h + pad, dpre.data_ptr(),
                                   2 * h + pad, kind, api.ComputeMode.FP16TCEC)
    _close(dpre, want["dpre"], "dpre")
    # the weights the other way round
    turned = place(down.transpose(1, 2).contiguous())
    again = place(torch.zeros(rows, 2 * h, dtype=dtype, device="cuda"))
    handle.grouped_gemm_gated_grad(api.CUBLAS_OP_T, rows, h, width, 3, ends, dys.data_ptr(), width + pad,
                                   turned.data_ptr(), width + pad, h * (width + pad), act, pre.data_ptr(), 2 * h + pad,
                                   again.data_ptr(), 2 * h + pad, kind, api.ComputeMode.FP16TCEC)
    _close(again, want["dpre"], "dpre")
    for t in (hid, pre, dpre, again):
        base = t._base.view(-1)
        assert torch.isnan(base[:offset]).all()
        if pad:
            assert torch.isnan(base[offset:].view(rows, -1)[:, t.shape[1]:]).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("name", ACTIVATIONS)
def test_elementwise_passes(handle, dtype, name):
    """act(gate) * up and its gradient by themselves, over all magnitudes, in rows of odd sizes."""
    torch, api, experts = _setup()
    dtype = getattr(torch, dtype)
    act, kind = experts._activation(name), experts._data_type(dtype)
    for rows, hidden, pad in ((1, 1, 0), (3, 517, 1), (40, 1024, 8), (9, 130, 0)):
        gate = torch.linspace(-30, 30, rows * hidden, device="cuda").view(rows, hidden)
        up, dh = torch.randn(rows, hidden, device="cuda"), torch.randn(rows, hidden, device="cuda").to(dtype)
        pre = _placed(torch, torch.cat([gate, up], 1).to(dtype), 2 * hidden + pad, pad)
        h, dpre = torch.empty(rows, hidden, dtype=dtype, device="cuda"), torch.empty(rows, 2 * hidden, dtype=dtype, device="cuda")
        handle.gated_rows(rows, hidden, pre, 2 * hidden + pad, None, 0, act, h, hidden, kind)
        handle.gated_rows(rows, hidden, pre, 2 * hidden + pad, dh, hidden, act, dpre, 2 * hidden, kind)
        a, s = _activated(torch, name, _Value(pre[:, :hidden]))
        u, d = _Value(pre[:, hidden:]), _Value(dh)
        for got, want in ((h, _times(a, u)), (dpre[:, :hidden], _times(d, u, s)), (dpre[:, hidden:], _times(d, a))):
            _close(got, want.rounded(torch, dtype), name)


def test_special_values(handle):
    """Infinities and NaN as the formulas have them; a NaN in one row or expert stays there."""
    torch, api, experts = _setup()
    inf, nan = float("inf"), float("nan")
    gate = torch.tensor([[inf, -inf, nan, 0.0, -0.0, 1.0, 1.0, 100.0]], device="cuda")
    up = torch.tensor([[2.0, 2.0, 2.0, inf, 3.0, nan, -inf, 1.0]], device="cuda")
    pre = torch.cat([gate, up], 1)
    for name in ACTIVATIONS:
        h = torch.empty(1, 8, device="cuda")
        handle.gated_rows(1, 8, pre, 16, None, 0, experts._activation(name), h, 8, api.CUDA_R_32F)
        low = 0.0 if name == "relu" else nan  # -inf * 0
        want = torch.tensor([[inf, low, nan, nan, -0.0, nan, -inf, 100.0]], device="cuda")
        assert torch.equal(torch.isnan(h), torch.isnan(want)), name
        assert torch.equal(h[~torch.isnan(want)], want[~torch.isnan(want)]), name
    x, gate_up, down, dy = _operands(torch, torch.bfloat16, 40, 48, 64, 2, 1)
    ends = _ends(torch, [20, 20])
    clean = experts.gated_feed_forward(handle, x, gate_up, down, ends)
    x[3] = nan
    gate_up[1, 5] = inf  # a row of the gate of the second expert
    y = experts.gated_feed_forward(handle, x, gate_up, down, ends)
    others = [r for r in range(20) if r != 3]
    assert torch.isnan(y[3]).all() and torch.equal(y[others], clean[others])


def test_gradient_against_differences(handle):
    """FP32: the slope along a direction from two forward passes."""
    torch, api, experts = _setup()
    counts, hidden, width, eps = [17, 0, 30], 40, 56, 2.0 ** -5
    rows, mode = sum(counts), api.ComputeMode.FP16TCEC_SCALING
    for name in ("silu", "gelu", "gelu_tanh"):
        x, gate_up, down, dy = _operands(torch, torch.float32, rows, hidden, width, 3, 3)
        ends = _ends(torch, counts)
        ways = [torch.randn_like(t) * t.std() for t in (x, gate_up, down)]
        leaves = [t.detach().requires_grad_() for t in (x, gate_up, down)]
        y = experts.gated_feed_forward(handle, *leaves, ends, activation=name, mode=mode)
        grads = torch.autograd.grad(y, leaves, dy)
        slope = sum((g.double() * v.double()).sum() for g, v in zip(grads, ways))
        bounds = _block(torch, torch.float32, name, x, gate_up, down, dy, counts, rows)
        exact = sum((bounds[k].v * v.double()).sum() for k, v in zip(("dx", "dgate_up", "ddown"), ways))
        off = sum((bounds[k].off * v.double().abs()).sum() for k, v in zip(("dx", "dgate_up", "ddown"), ways))
        assert abs(slope - exact) <= off
        found, true, far = 0.0, 0.0, 0.0
        for sign in (1, -1):
            at = [(t.double() + sign * eps * v.double()).float() for t, v in zip((x, gate_up, down), ways)]
            got = experts.gated_feed_forward(handle, *at, ends, activation=name, mode=mode)
            here = _block(torch, torch.float32, name, *at, None, counts, rows)["y"]
            found += sign * (got.double() * dy.double()).sum() / (2 * eps)
            true += sign * (here.v * dy.double()).sum() / (2 * eps)
            far += (here.off * dy.double().abs()).sum() / (2 * eps)
        # the difference of the exact function says how far a difference is from the slope
        assert abs(found - slope) <= far + off + abs(true - exact)


def test_gradients_of_gradients(handle):
    torch, api, experts = _setup()
    counts, name = [9, 14], "silu"
    x, gate_up, down, dy = _operands(torch, torch.float32, 23, 24, 32, 2, 9)
    ends, mode = _ends(torch, counts), api.ComputeMode.FP16TCEC_SCALING
    ways = [torch.randn_like(t) for t in (x, gate_up, down)]

    def second(function, leaves, ways, dy):
        leaves = [t.detach().requires_grad_() for t in leaves]
        first = torch.autograd.grad(function(*leaves), leaves, dy, create_graph=True)
        return torch.autograd.grad(sum((g * v).sum() for g, v in zip(first, ways)), leaves)

    def exact(x, gate_up, down):
        out = []
        for e, (a, b) in enumerate(_spans(counts)):
            g, u = gate_up[e].split(24)
            out.append(torch.nn.functional.silu(x[a:b] @ g.t()) * (x[a:b] @ u.t()) @ down[e].t())
        return torch.cat(out)

    got = second(lambda *t: experts.gated_feed_forward(handle, *t, ends, activation=name, mode=mode), (x, gate_up, down), ways, dy)
    want = second(exact, [t.double() for t in (x, gate_up, down)], [v.double() for v in ways], dy.double())
    for g, w in zip(got, want):
        # six FP32 products one behind the other, each to some 20 * 2^-22 of its terms' magnitudes, which exceed the
        # result's some tenfold
        assert float((g.double() - w).norm() / w.norm()) < 6 * 20 * 2.0 ** -22 * 10
    h = second(lambda a, b: experts.gated_matmul(handle, a, b, ends, mode=mode), (x, gate_up), ways[:2], torch.randn(23, 24, device="cuda"))
    assert all(torch.isfinite(t).all() for t in h)


def test_gradients_asked_for_one_by_one(handle):
    torch, api, experts = _setup()
    x, gate_up, down, dy = _operands(torch, torch.bfloat16, 50, 64, 72, 2, 2)
    ends = _ends(torch, [20, 30])
    all_of = [t.detach().requires_grad_() for t in (x, gate_up, down)]
    grads = torch.autograd.grad(experts.gated_feed_forward(handle, *all_of, ends), all_of, dy)
    for which in itertools.chain.from_iterable(itertools.combinations(range(3), n) for n in (1, 2)):
        some = [t.detach().requires_grad_(i in which) for i, t in enumerate((x, gate_up, down))]
        got = torch.autograd.grad(experts.gated_feed_forward(handle, *some, ends), [some[i] for i in which], dy)
        assert all(torch.equal(a, grads[i]) for a, i in zip(got, which))
    # a gradient that is one value for all elements, and operands in another order
    turned = gate_up.transpose(1, 2).contiguous().transpose(1, 2).requires_grad_()
    xs = x.detach().requires_grad_()
    experts.gated_feed_forward(handle, xs, turned, down, ends).sum().backward()
    again = [t.detach().requires_grad_() for t in (x, gate_up)]
    ones = torch.ones(50, 72, dtype=torch.bfloat16, device="cuda")
    dx, dw = torch.autograd.grad(experts.gated_feed_forward(handle, *again, down, ends), again, ones)
    assert torch.equal(xs.grad, dx) and torch.equal(turned.grad, dw)


def test_saved_tensors_that_were_moved(handle):
    torch, api, experts = _setup()
    x, gate_up, down, dy = _operands(torch, torch.bfloat16, 50, 64, 72, 2, 5)
    ends = _ends(torch, [20, 30])
    dense = [t.detach().requires_grad_() for t in (x, gate_up, down)]
    want = torch.autograd.grad(experts.gated_feed_forward(handle, *dense, ends), dense, dy)
    # rows 96 apart when they are saved, 72 or 64 when they come back
    apart = [_placed(torch, t, 96, 0).requires_grad_() for t in (x, gate_up, down)]
    with torch.autograd.graph.save_on_cpu():
        y = experts.gated_feed_forward(handle, *apart, ends)
    got = torch.autograd.grad(y, apart, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_rows(handle):
    torch, api, experts = _setup()
    for dtype in (torch.bfloat16, torch.float32):
        x, gate_up, down, dy = _operands(torch, dtype, 0, 24, 32, 2, 9)
        leaves = [t.detach().requires_grad_() for t in (x, gate_up, down)]
        y = experts.gated_feed_forward(handle, *leaves, _ends(torch, [0, 0]))
        grads = torch.autograd.grad(y, leaves, dy)
        assert y.shape == (0, 32) and grads[0].shape == (0, 32)
        assert not grads[1].any() and not grads[2].any()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_totals_that_are_wrong(handle, dtype):
    """A total that falls back or is too large is taken as the one in front, or as the number of rows."""
    torch, api, experts = _setup()
    dtype = getattr(torch, dtype)
    x, gate_up, down, dy = _operands(torch, dtype, 90, 40, 64, 4, 4)
    bad, good = torch.tensor([30, -5, 2000000000, 7], dtype=torch.int32).cuda(), _ends(torch, [30, 0, 60, 0])
    for ends in (bad,):
        a = [t.detach().requires_grad_() for t in (x, gate_up, down)]
        b = [t.detach().requires_grad_() for t in (x, gate_up, down)]
        ya, yb = experts.gated_feed_forward(handle, *a, ends), experts.gated_feed_forward(handle, *b, good)
        assert torch.equal(ya, yb)
        for p, q in zip(torch.autograd.grad(ya, a, dy), torch.autograd.grad(yb, b, dy)):
            assert torch.equal(p, q)


def test_replayed_from_a_graph(handle):
    """A training step captured and replayed on other inputs gives what the eager step gives."""
    torch, api, experts = _setup()
    counts = [40, 0, 25]
    x, gate_up, down, dy = _operands(torch, torch.bfloat16, 65, 96, 128, 3, 6)
    ends = _ends(torch, counts)

    def step(x, gate_up, down, dy, ends):
        leaves = [t.detach().requires_grad_() for t in (x, gate_up, down)]
        y = experts.gated_feed_forward(handle, *leaves, ends)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    held = [t.clone() for t in (x, gate_up, down, dy, ends)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        handle.use_current_torch_stream()
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        handle.use_current_torch_stream()
        out = step(*held)
    handle.use_current_torch_stream()
    for seed, counts in ((20, [40, 0, 25]), (21, [0, 60, 1])):
        fresh = [*_operands(torch, torch.bfloat16, 65, 96, 128, 3, seed), _ends(torch, counts)]
        for t, v in zip(held, (fresh[0], fresh[1], fresh[2], fresh[3], fresh[4])):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step(*fresh)):
            assert torch.equal(a, b)


def test_refusals(handle):
    torch, api, experts = _setup()
    x, gate_up, down, _ = _operands(torch, torch.bfloat16, 8, 16, 32, 2, 1)
    ends = _ends(torch, [4, 4])
    for bad in (lambda: experts.gated_matmul(handle, x, gate_up[:, :31], ends),
                lambda: experts.gated_matmul(handle, x, gate_up.half(), ends),
                lambda: experts.gated_matmul(handle, x, gate_up, ends, activation="tanh"),
                lambda: experts.gated_matmul(handle, x, gate_up),
                lambda: experts.gated_matmul(handle, x, gate_up, ends[:1]),
                lambda: experts.gated_matmul(handle, x[:, :16], gate_up, ends),
                lambda: experts.gated_matmul(handle, x.double(), gate_up.double(), ends),
                lambda: experts.gated_matmul(handle, x, gate_up, ends, out=torch.empty(8, 17, device="cuda")),
                lambda: experts.gated_feed_forward(handle, x, gate_up, down[:, :, :15], ends),
                lambda: experts.gated_feed_forward(handle, x, gate_up, down[:1], ends),
                lambda: experts.gated_feed_forward(handle, x, gate_up, down.half(), ends),
                lambda: experts.gated_matmul(handle, x.requires_grad_(), gate_up, ends, out=torch.empty(8, 16, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    x = x.detach()
    with torch.cuda.stream(torch.cuda.Stream()):
        with pytest.raises(ValueError, match="stream"):
            experts.gated_matmul(handle, x, gate_up, ends)
    with pytest.raises(api.CuMpSGEMMError):
        experts.gated_matmul(handle, x.float(), gate_up.float(), ends, mode=api.ComputeMode.TF32TCEC)
    args = (x.data_ptr(), 32, gate_up.data_ptr(), 32, 1024, 0, x.data_ptr(), 16, None, 0)
    assert handle.grouped_gemm_gated(8, 16, 32, 2, ends, *args, api.CUDA_R_32F, check=False) == api.CUBLAS_STATUS_INVALID_VALUE
    assert handle.grouped_gemm_gated(8, 16, 32, 2, ends, x.data_ptr(), 32, gate_up.data_ptr(), 32, 1024, 4, x.data_ptr(),
                                     16, None, 0, api.CUDA_R_16BF, check=False) == api.CUBLAS_STATUS_INVALID_VALUE
    out = torch.empty(8, 16, dtype=torch.bfloat16, device="cuda")
    assert experts.gated_matmul(handle, x, gate_up, ends, out=out) is out
    assert torch.equal(out, experts.gated_matmul(handle, x, gate_up, ends))


def test_offsets_past_32_bits(handle):
    """Rows behind 2^32 bytes, and 2^31 elements, of what stands in front of the activation."""
    torch, api, experts = _setup()
    rows, hidden, width, last = 70000, 16384, 64, 300
    x, gate_up, down, dy = _operands(torch, torch.bfloat16, rows, hidden, width, 1, 1)

    def run(x, dy):
        n = x.shape[0]
        h, pre = experts._gated(handle, x, gate_up, None, api.Activation.SILU, api.ComputeMode.FP16TCEC, keep=True)
        dpre = torch.empty_like(pre)
        handle.grouped_gemm_gated_grad(api.CUBLAS_OP_N, n, hidden, width, 1, None, dy.data_ptr(), width, down.data_ptr(),
                                       hidden, hidden * width, api.Activation.SILU, pre.data_ptr(), 2 * hidden,
                                       dpre.data_ptr(), 2 * hidden, api.CUDA_R_16BF)
        again = torch.empty_like(pre)
        handle.gated_rows(n, hidden, pre.data_ptr(), 2 * hidden, h.data_ptr(), hidden, api.Activation.SILU, again.data_ptr(),
                          2 * hidden, api.CUDA_R_16BF)
        return [t[-last:].clone() for t in (h, pre, dpre, again)]

    assert all(torch.equal(a, b) for a, b in zip(run(x, dy), run(x[-last:], dy[-last:])))


def test_two_streams_and_a_graph_at_once(handle):
    """A handful of rows replayed from a graph while another handle multiplies many on a stream of its own."""
    torch, api, experts = _setup()
    x, gate_up, _, _ = _operands(torch, torch.bfloat16, 700, 264, 512, 4, 3)
    few, ends, few_ends = x[:6].clone(), _ends(torch, [300, 0, 7, 393]), _ends(torch, [1, 0, 3, 2])
    want_few, want = experts.gated_matmul(handle, few, gate_up, few_ends), experts.gated_matmul(handle, x, gate_up, ends)
    side, graph, out = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.zeros_like(want_few)
    with torch.cuda.graph(graph):
        handle.use_current_torch_stream()
        experts.gated_matmul(handle, few, gate_up, few_ends, out=out)
    handle.use_current_torch_stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = api.Handle()
        other.use_current_torch_stream()
        results = [experts.gated_matmul(other, x, gate_up, ends) for _ in range(20)]
    for _ in range(20):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want_few)
    few.copy_(x[100:106])  # read at each replay
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, experts.gated_matmul(handle, few, gate_up, few_ends))
    assert all(torch.equal(y, want) for y in results)
    assert handle.kernel_status() == 0 and other.kernel_status() == 0
    other.destroy()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("hidden", [5, 37, 100, 129])
@pytest.mark.parametrize("counts,spare", [([130, 0, 61], 9), ([3, 0, 5], 0)])
def test_results_in_padded_rows(handle, dtype, hidden, counts, spare):
    """Rows of h that begin at multiples of 16 bytes and end inside the last 16: all of them is written, and nothing else."""
    torch, api, experts = _setup()
    dtype, rows, name = getattr(torch, dtype), sum(counts) + spare, "silu"
    for width, pad in ((72, 0), (72, 16), (70, 0)):  # (of 70 values the kernel for a handful of rows takes none)
        x, gate_up, _, _ = _operands(torch, dtype, rows, hidden, width, 3, hidden + width)
        want = _block(torch, dtype, name, x, gate_up, None, None, counts, rows)
        ld = (hidden + 7) // 8 * 8 + pad
        out = _placed(torch, torch.full((rows, hidden), float("nan"), dtype=dtype, device="cuda"), ld, 0)
        ends = _ends(torch, counts)
        assert experts.gated_matmul(handle, x, gate_up, ends, activation=name, out=out) is out
        _close(out, want["h"], "h")
        # the same with what is in front of the activation, in rows of the same kind
        hid, ldp = torch.full_like(out._base.view(rows, ld), float("nan")), (2 * hidden + 7) // 8 * 8 + pad
        pre = _placed(torch, torch.full((rows, 2 * hidden), float("nan"), dtype=dtype, device="cuda"), ldp, 0)
        handle.grouped_gemm_gated(rows, hidden, width, 3, ends, x.data_ptr(), width, gate_up.data_ptr(), width,
                                  2 * hidden * width, experts._activation(name), hid.data_ptr(), ld, pre.data_ptr(), ldp,
                                  experts._data_type(dtype))
        _close(pre, want["pre"], "pre")
        assert torch.equal(hid[:, :hidden], out)
        for t, cols in ((out._base.view(rows, ld), hidden), (hid, hidden), (pre._base.view(rows, ldp), 2 * hidden)):
            assert torch.isnan(t[:, cols:]).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("order", ["rows apart", "columns first", "columns apart"])
def test_saved_tensors_in_another_order(handle, dtype, order):
    """Hooks that give back every tensor that the forward pass kept with other strides: the gradients are the same."""
    torch, api, experts = _setup()
    x, gate_up, down, dy = _operands(torch, getattr(torch, dtype), 50, 64, 72, 2, 5)
    ends, dh = _ends(torch, [20, 30]), torch.randn(50, 64, device="cuda").to(x.dtype)

    def other(t):
        if t.dim() == 1:
            return t
        if order == "columns first":
            return t.transpose(-1, -2).contiguous().transpose(-1, -2)
        wide = torch.full((*t.shape[:-1], 2 * t.shape[-1] + 8), float("nan"), dtype=t.dtype, device=t.device)
        part = wide[..., 8 : t.shape[-1] + 8] if order == "rows apart" else wide[..., 8::2]
        return part.copy_(t)

    for call, operands, grad in ((experts.gated_feed_forward, (x, gate_up, down), dy), (experts.gated_matmul, (x, gate_up), dh)):
        leaves = [t.detach().requires_grad_() for t in operands]
        want = torch.autograd.grad(call(handle, *leaves, ends), leaves, grad)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other):
            y = call(handle, *leaves, ends)
        got = torch.autograd.grad(y, leaves, grad, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        again = torch.autograd.grad(y, leaves, grad, create_graph=True)
        plain = torch.autograd.grad(call(handle, *leaves, ends), leaves, grad, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(again, plain))


def test_saved_tensors_that_do_not_fit(handle):
    """Hooks that leave a saved tensor in host memory, or give it back with another type: refused before anything runs."""
    torch, api, experts = _setup()
    x, gate_up, down, dy = _operands(torch, torch.bfloat16, 50, 64, 72, 2, 5)
    ends, dh = _ends(torch, [20, 30]), torch.randn(50, 64, device="cuda").bfloat16()
    pre, h, leaves = (50, 128), (50, 64), [t.detach().requires_grad_() for t in (x, gate_up, down)]
    kept = [tuple(t.shape) for t in (x, gate_up, ends)] + [pre]
    for call, count, grad, shapes in ((experts.gated_feed_forward, 3, dy, kept + [tuple(down.shape), h]),
                                      (experts.gated_matmul, 2, dh, kept)):
        for changed in shapes:
            for change in (lambda t: t.cpu(), lambda t: t.to(torch.float16)):
                with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if tuple(t.shape) == changed else t):
                    y = call(handle, *leaves[:count], ends)
                with pytest.raises(ValueError):
                    torch.autograd.grad(y, leaves[:count], grad)


@pytest.mark.parametrize("name", ACTIVATIONS)
def test_gradients_behind_what_passes_float16(handle, name):
    """Sums past 65504 are infinities in what the forward pass keeps.  Times nothing they are nothing: where the gradient is 0,
    where the activation has no slope, or the gate is far below 0; elsewhere the gradient is infinite too."""
    torch, api, experts = _setup()
    act, kind, inf = experts._activation(name), api.CUDA_R_16F, float("inf")
    for hidden, rows in ((64, 70), (37, 70), (64, 5)):
        pre, dy = torch.randn(rows, 2 * hidden, device="cuda").half(), torch.randn(rows, 48, device="cuda").half()
        down = torch.randn(1, 48, hidden, device="cuda").half()
        gate, up = pre[:, :hidden], pre[:, hidden:]
        dy[::3] = 0  # rows without a gradient, whatever their values
        gate[:, 3], up[:, 5], gate[:, 7], up[:, 7] = inf, -inf, -inf, inf
        gate[:, 9], up[:, 9], gate[:, 11] = -300.0, -inf, -inf
        dh = torch.randn(rows, hidden, device="cuda").half()
        dh[::3] = 0
        one, two = (torch.full((rows, 2 * hidden), float("nan"), device="cuda", dtype=torch.float16) for _ in range(2))
        handle.grouped_gemm_gated_grad(api.CUBLAS_OP_N, rows, hidden, 48, 1, None, dy, 48, down, hidden, 48 * hidden, act,
                                       pre, 2 * hidden, one, 2 * hidden, kind)
        handle.gated_rows(rows, hidden, pre, 2 * hidden, dh, hidden, act, two, 2 * hidden, kind)
        back = _product(torch, torch.float16, _Value(dy), _Value(down[0]))
        for got, d in ((one, back), (two, _Value(dh))):
            dgate, dup = got[:, :hidden], got[:, hidden:]
            assert not got[::3].any()
            assert not dgate[:, [7, 9, 11]].any() and not dup[:, [7, 9, 11]].any()
            real = torch.arange(rows, device="cuda") % 3 != 0
            assert torch.equal(dup[real, 3], (d.v[real, 3].sign() * inf).half())
            if name != "relu":
                assert torch.isinf(dgate[real, 5]).all()
            plain = [i for i in range(hidden) if i not in (3, 5, 7, 9, 11)]
            a, s = _activated(torch, name, _Value(gate[:, plain]))
            u, d = _Value(up[:, plain]), d[:, plain]
            _close(dgate[:, plain], _times(d, u, s).rounded(torch, torch.float16), name)
            _close(dup[:, plain], _times(d, a).rounded(torch, torch.float16), name)


def test_a_block_whose_sums_pass_float16(handle):
    """From end to end: gates below -65504, and rows that no gradient comes back to."""
    torch, api, experts = _setup()
    x, gate_up, down, dy = _operands(torch, torch.float16, 60, 64, 72, 1, 7, scale=2.0 ** -6)
    gate_up[0, :64:5] = -1000.0 * x.sign()[7]  # times x[7], some -60000 and less
    x[7] *= 4
    gate_up[0, 3, :], x[8] = 2000.0, x[8].abs() * 8  # above 65504 in row 8, which no gradient comes back to
    dy[8] = 0
    leaves = [t.detach().requires_grad_() for t in (x, gate_up, down)]
    ends = _ends(torch, [60])
    raw = x.double() @ gate_up[0].double().t()
    assert (raw[7, :64:5] < -65520).all() and raw[8, 3] > 65520
    y = experts.gated_feed_forward(handle, *leaves, ends)
    dx, dgate_up, _ = torch.autograd.grad(y, leaves, dy)
    want = _block(torch, torch.float16, "silu", x, gate_up, down, dy, [60], 60)  # (its sums pass nothing)
    assert want["dx"].v.abs().max() < 60000 and want["dgate_up"].v.abs().max() < 60000
    assert torch.isfinite(dgate_up).all() and torch.isfinite(dx).all() and not dx[8].any()
    _close(dx, want["dx"], "dx")
    _close(dgate_up, want["dgate_up"], "dgate_up")
