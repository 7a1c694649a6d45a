"""The products of rows grouped by expert without a GPU: what is refused before anything runs."""
import pytest


def test_null_handle_is_refused(clib):
    one = 1
    assert clib.cuMpSGEMM_get_device(None) == -1
    assert clib.cuMpSGEMM_grouped_gemm(None, 0, 1, 1, 1, one, None, None, None, 1, None, 1, 0, None, None, 1,
                                       0, 1) == 1
    assert clib.cuMpSGEMM_grouped_gemm_wgrad(None, 0, 1, 1, 1, one, None, None, None, 1, None, 1, None, None,
                                             1, 0, 0, 1) == 1
    assert clib.cuMpSGEMM_i8_grouped_gemm(None, 1, 1, 1, one, None, None, 1, None, None, 1, 0, None, None,
                                          None, 1, 0) == 1
    assert clib.cuMpSGEMM_quantize_rows_i8(None, 1, 1, None, 1, 0, None, 1, None, 1, None) == 1


def test_operands_in_host_memory_are_refused():
    import torch

    from cumpsgemm_b200 import experts

    x, w = torch.zeros(4, 8), torch.zeros(2, 8, 6)
    ends = torch.tensor([1, 4], dtype=torch.int32)
    q, s = torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)
    for call in (lambda: experts.grouped_matmul(None, x, w, ends),
                 lambda: experts.grouped_matmul_wgrad(None, x, torch.zeros(4, 6), ends),
                 lambda: experts.grouped_linear(None, x, w, ends),
                 lambda: experts.quantize_rows(None, x),
                 lambda: experts.i8_matmul(None, q, s, q, s)):
        with pytest.raises(ValueError, match="device memory"):
            call()


def test_shapes_are_checked():
    import torch

    from cumpsgemm_b200 import experts

    for x, w in ((torch.zeros(4, 8), torch.zeros(2, 6, 8)), (torch.zeros(4, 8), torch.zeros(8, 6)),
                 (torch.zeros(8), torch.zeros(2, 8, 6)), (torch.zeros(8, 4).t(), torch.zeros(2, 8, 6)),
                 (torch.zeros(1, 8).expand(4, 8), torch.zeros(2, 8, 6)),
                 (torch.zeros(4, 8), torch.zeros(1, 8, 6).expand(2, 8, 6))):
        with pytest.raises(ValueError):
            experts.grouped_matmul(None, x, w)
