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
