"""The largest and smallest numbers of rows of the 8-bit linears."""
import pytest
import torch

DEV = "cuda:0"


def test_rows_beyond_the_limits_are_refused():
    """Before anything is launched (the addresses are read by nothing)."""
    from slim_amd import _lib
    P = 1 << 20
    for rows, K in ((1 << 24, 100), ((1 << 22) - 1, 16385)):
        lib = _lib.load()
        assert lib.slim_quantize_rows8(P, 1, rows, K, K, P, -(-K // 128) * 128, P, None) == _lib.ERR_INVALID
        assert b"too many rows" in lib.slim_last_error()


@pytest.mark.gpu
def test_more_than_four_million_long_rows():
    """2^22 + 3 rows of 8193: a workgroup of 256 threads for each fits a launch (one of 1024 would not)."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from slim_amd import ops
    R, K = (1 << 22) + 3, 8193
    x = torch.zeros(R, K, dtype=torch.bfloat16, device=DEV)
    x[-3:] = torch.randn(3, K, device=DEV)
    codes, scale = ops.quantize_rows8(x)
    few, few_scale = ops.quantize_rows8(x[-3:].clone())
    assert torch.equal(codes[-3:], few) and torch.equal(scale[-3:], few_scale) and bool(few.any())
    assert not bool(scale[:-3].any()) and not bool(codes[:5].any()) and not bool(codes[-8:-3].any())


@pytest.mark.gpu
def test_no_rows_at_all():
    """An empty batch through the parts, as through the whole: quantised, multiplied and sent back."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from slim_amd import ops
    codes, scale = ops.quantize_rows8(torch.randn(10, 100, device=DEV))
    a, sa = ops.quantize_rows8(torch.zeros(0, 100, device=DEV))
    out = ops.gemm8_nt(a, sa, codes, scale, torch.zeros(10, device=DEV), torch.float32, K=100)
    assert out.shape == (0, 10) and out.dtype == torch.float32
    assert ops.linear8_forward(torch.zeros(0, 100, device=DEV), codes, scale).shape == (0, 10)
    assert ops.linear8_backward(torch.zeros(0, 10, device=DEV), ops.transpose8(codes, 100), scale).shape == (0, 100)
    with pytest.raises(ValueError, match="b must be"):
        ops.gemm8_nt(codes, scale, a, sa)
