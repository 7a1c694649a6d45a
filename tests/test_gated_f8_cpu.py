"""Gated blocks and products in 8-bit floating point without a GPU: what is refused before anything runs."""
import pytest


def test_null_handle_is_refused(clib):
    assert clib.cuMpSGEMM_grouped_gemm_gated(None, 1, 1, 1, 1, None, None, 1, None, 1, 0, 0, None, 1, None, 2, 2, 1) == 1
    assert clib.cuMpSGEMM_grouped_gemm_gated_grad(None, 0, 1, 1, 1, 1, None, None, 1, None, 1, 0, 0, None, 2, None, 2, 2,
                                                  1) == 1
    assert clib.cuMpSGEMM_gated_rows(None, 1, 1, None, 2, None, 0, 0, None, 1, 0) == 1
    assert clib.cuMpSGEMM_quantize_rows_f8(None, 1, 1, None, 1, 0, None, 1, -1, None, 1, 28, None, 1, 1) == 1
    assert clib.cuMpSGEMM_quantize_blocks_f8(None, 1, 1, 1, None, 1, 1, 0, None, 1, 1, 28, None) == 1
    assert clib.cuMpSGEMM_f8_grouped_gemm(None, 1, 1, 1, 1, None, None, 1, 28, None, 1, 1, None, 1, 0, 28, None, None, None,
                                          1, 0) == 1
    assert clib.cuMpSGEMM_f8_grouped_gemm_gated(None, 1, 128, 1, 1, None, None, 1, 28, None, 1, 1, None, 1, 0, 28, None, 0,
                                                None, 128, 28, None, 1, 1) == 1


def test_operands_in_host_memory_are_refused():
    import torch

    from cumpsgemm_b200 import experts

    x, w, d = torch.zeros(4, 8), torch.zeros(2, 12, 8), torch.zeros(2, 8, 6)
    ends = torch.tensor([1, 4], dtype=torch.int32)
    q, s = torch.zeros(4, 8, dtype=torch.float8_e4m3fn), torch.zeros(4, 1)
    wq, ws = torch.zeros(2, 256, 8, dtype=torch.float8_e4m3fn), torch.zeros(2, 2, 1)
    for call in (lambda: experts.gated_matmul(None, x, w, ends),
                 lambda: experts.gated_feed_forward(None, x, w, d, ends),
                 lambda: experts.gated_feed_forward(None, x.requires_grad_(), w, d, ends),
                 lambda: experts.quantize_blocks(None, x),
                 lambda: experts.quantize_blocks(None, x, activation="silu"),
                 lambda: experts.quantize_weight_blocks(None, w),
                 lambda: experts.f8_matmul(None, q, s, wq, ws, ends),
                 lambda: experts.f8_gated_matmul(None, q, s, wq, ws, ends)):
        with pytest.raises(ValueError, match="device memory"):
            call()


def test_shapes_and_names_are_checked():
    import torch

    from cumpsgemm_b200 import experts

    x, w, d = torch.zeros(4, 8), torch.zeros(2, 12, 8), torch.zeros(2, 8, 6)
    q = torch.zeros(4, 8, dtype=torch.float8_e4m3fn)
    for call in (lambda: experts.gated_matmul(None, x, w, activation="swish"),
                 lambda: experts.gated_matmul(None, x, w[:, :11]),
                 lambda: experts.gated_matmul(None, x, w[0]),
                 lambda: experts.gated_matmul(None, x[0], w),
                 lambda: experts.gated_matmul(None, x[:, :7], w),
                 lambda: experts.gated_feed_forward(None, x, w, d[:1]),
                 lambda: experts.gated_feed_forward(None, x, w, d[:, :, :5]),
                 lambda: experts.gated_feed_forward(None, x, w, d[0]),
                 lambda: experts.gated_feed_forward(None, x, w, d.half()),
                 lambda: experts.quantize_blocks(None, x[:, :7], activation="gelu"),
                 lambda: experts.quantize_blocks(None, x, activation="none"),
                 lambda: experts.quantize_weight_blocks(None, x[0]),
                 lambda: experts.f8_gated_matmul(None, q, torch.zeros(4, 1), q[:3], torch.zeros(1, 1)),
                 lambda: experts.f8_matmul(None, q, torch.zeros(4, 1), q[:, :7], torch.zeros(1, 1))):
        with pytest.raises(ValueError):
            call()


class _Recorder:
    """Stands for a handle: what the calls would read of the tensors that a backward pass had saved."""

    def __init__(self):
        self.seen = {}

    def _put(self, what, at, rows, cols, ld):
        import ctypes

        import torch

        values = (ctypes.c_float * ((rows - 1) * ld + cols)).from_address(at)
        self.seen[what] = torch.tensor(list(values)).as_strided((rows, cols), (ld, 1)).clone()

    def grouped_gemm_gated_grad(self, op, rows, hidden, k, groups, ends, dy, lddy, w, ldw, stridew, act, pre, ldpre, dpre,
                                lddpre, kind, mode):
        self._put("dy", dy, rows, k, lddy)
        self._put("pre", pre, rows, 2 * hidden, ldpre)
        self._put("down", w, k, hidden, ldw)

    def grouped_gemm(self, op, rows, n, k, groups, ends, alpha, x, ldx, w, ldw, stridew, beta, y, ldy, kind, mode):
        self._put("gate_up", w, k, n, ldw)

    def grouped_gemm_wgrad(self, op, rows, n, k, groups, ends, alpha, x, ldx, dy, lddy, beta, dw, lddw, stridedw, kind, mode):
        self._put("x" if "x" not in self.seen else "h", x, rows, k, ldx)

    def gated_rows(self, rows, hidden, pre, ldpre, dh, lddh, act, out, ldo, kind):
        self._put("pre", pre, rows, 2 * hidden, ldpre)


def _orders(torch, t):
    """The same values with rows further apart, column after column, and with columns apart."""
    rows, cols = t.shape[-2:]
    wide = torch.full((*t.shape[:-1], 2 * cols + 6), float("nan"), dtype=t.dtype, device=t.device)
    wide[..., 3 : cols + 3] = t
    yield wide[..., 3 : cols + 3]
    yield t.transpose(-1, -2).contiguous().transpose(-1, -2)
    wide[..., 1 : 2 * cols : 2] = t
    yield wide[..., 1 : 2 * cols : 2]


def _saved(torch):
    g = torch.Generator().manual_seed(3)
    new = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    ends = torch.tensor([5], dtype=torch.int32)
    return {"x": new(5, 4), "gate_up": new(1, 6, 4), "down": new(1, 4, 3), "ends": ends, "pre": new(5, 6), "h": new(5, 3)}


def test_backward_passes_read_what_was_saved_in_any_order(monkeypatch):
    from types import SimpleNamespace

    import torch

    from cumpsgemm_b200 import experts

    monkeypatch.setattr(experts, "_check_place", lambda handle, device: None)
    dy = torch.randn(5, 4)
    for name in ("x", "gate_up", "down", "pre", "h"):
        for other in _orders(torch, _saved(torch)[name]):
            saved, handle = _saved(torch), _Recorder()
            saved[name] = other
            ctx = SimpleNamespace(saved_tensors=tuple(saved.values()), how=(handle, 0, 1), needs_input_grad=(True,) * 3)
            with torch.no_grad():
                experts._GatedFeedForward.backward(ctx, dy)
            assert torch.equal(handle.seen["dy"], dy)
            for key, t in handle.seen.items():
                assert key == "dy" or torch.equal(t, _saved(torch)[key].view(t.shape)), (name, key)
            if name not in ("x", "gate_up", "pre"):
                continue
            handle = _Recorder()
            ctx = SimpleNamespace(saved_tensors=(saved["x"], saved["gate_up"], saved["ends"], saved["pre"]),
                                  how=(handle, 0, 1), needs_input_grad=(True, True))
            with torch.no_grad():
                experts._GatedMatmul.backward(ctx, torch.randn(5, 3))
            for key in ("pre", "gate_up", "x"):
                assert torch.equal(handle.seen[key], _saved(torch)[key].view(handle.seen[key].shape)), (name, key)


@pytest.mark.parametrize("name", ["x", "gate_up", "down", "pre", "h", "ends"])
def test_saved_tensors_that_do_not_fit_are_refused(monkeypatch, name):
    """On another device (of no memory here), of another type, or of another size."""
    from types import SimpleNamespace

    import torch

    from cumpsgemm_b200 import experts

    monkeypatch.setattr(experts, "_check_place", lambda handle, device: None)

    class Elsewhere(torch.Tensor):
        def get_device(self):
            return 1

    whole = _saved(torch)
    for changed in (whole[name].as_subclass(Elsewhere), whole[name].double(), whole[name][:0],
                    torch.cat([whole[name], whole[name]], -1)):
        saved = dict(whole, **{name: changed})
        for block in (True, False):
            if not block and name in ("down", "h"):
                continue
            handle = _Recorder()
            for call in ("grouped_gemm", "grouped_gemm_wgrad", "grouped_gemm_gated_grad", "gated_rows"):
                monkeypatch.setattr(handle, call, lambda *a: None, raising=False)
            ctx = SimpleNamespace(how=(handle, 0, 1), needs_input_grad=(True,) * 3 if block else (True, True),
                                  saved_tensors=tuple(saved.values()) if block else
                                  (saved["x"], saved["gate_up"], saved["ends"], saved["pre"]))
            backward = experts._GatedFeedForward.backward if block else experts._GatedMatmul.backward
            with torch.no_grad(), pytest.raises(ValueError):
                backward(ctx, torch.randn(5, 4 if block else 3))
