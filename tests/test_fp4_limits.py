"""Limits of the 4-bit linears' C entries that need no GPU."""
import torch

from q8_kernels_b200 import _lib

BUF = (torch.zeros(8192, dtype=torch.uint8).data_ptr() + 255) // 256 * 256


def test_refusals_of_the_gradient_operand():
    def quant(grad=BUF, dtype=_lib.DT_BF16, q=BUF, scales=BUF, rows=4, n=32):
        return _lib.lib.q8k_fp4_backward_quant(grad, dtype, q, scales, rows, n, None)

    assert quant(dtype=_lib.DT_F32) == -2 and quant(dtype=_lib.DT_E4M3) == -2 and quant(n=24) == -1 and quant(n=0) == -1 and quant(n=32784) == -2
    assert quant(grad=None) == -1 and quant(q=None) == -1 and quant(scales=None) == -1 and quant(grad=BUF + 8) == -1 and quant(q=BUF + 8) == -1
    assert quant(rows=-1) == -1 and quant(rows=0) == 0


def test_more_columns_than_a_store_can_name_are_refused():
    """The products' stores name a column by its byte, 2 n, in 32 bits: 2^30 columns are too many, whatever the number of rows."""
    for m in (1, 4, 300, 5000):
        for n in (1 << 30, (1 << 30) + 16, 0x7fffff00):
            assert _lib.lib.q8k_fp4_mm(2, BUF, BUF, BUF, BUF, BUF, BUF, None, None, _lib.DT_BF16, m, n, 64, 0, None, None) == _lib.lib.q8k_fp4_linear(
                2, BUF, _lib.DT_BF16, BUF, BUF, BUF, None, None, _lib.DT_BF16, m, n, 64, 0, BUF, 1 << 40, None, None) == -5
        # the largest number goes past that check, to the missing output
        assert _lib.lib.q8k_fp4_mm(2, BUF, BUF, BUF, BUF, BUF, BUF, None, None, _lib.DT_BF16, m, (1 << 30) - 16, 64, 0, None, None) == -1


def test_more_columns_than_a_store_of_the_8_bit_products_can_name_are_refused():
    """16-bit columns from 2^30 on, of rows enough for the kernel on CTA pairs (few rows have a kernel with plain stores)."""
    for mm in (_lib.lib.q8k_q8_mm, _lib.lib.q8k_fp8_mm):
        for m in (300, 5000):
            assert mm(BUF, BUF, None, BUF, BUF, BUF, _lib.DT_BF16, 1, 1, m, 1 << 30, 64, 0, None, None) == -5
            assert mm(BUF, BUF, None, BUF, BUF, BUF, _lib.DT_BF16, 1, 1, m, 0x7fffff00, 64, 1, None, None) == -5


def test_the_message_of_a_refused_output_type():
    """What is accepted depends on operands and epilogue: the message says on what."""
    def message(mm, dtype, gelu):
        assert mm(BUF, BUF, None, BUF, BUF, BUF, dtype, 1, 1, 8, 16, 64, gelu, None, None) == -2
        return _lib.lib.q8k_last_error_detail().decode()

    for mm in (_lib.lib.q8k_q8_mm, _lib.lib.q8k_fp8_mm):
        for gelu in (0, 1):
            assert "is not bf16 or e4m3" in message(mm, _lib.DT_F32, gelu)
    for mm, gelu in ((_lib.lib.q8k_q8_mm, 0), (_lib.lib.q8k_q8_mm, 1), (_lib.lib.q8k_fp8_mm, 1)):
        assert "fp16 is for e4m3 operands without GELU and residual" in message(mm, _lib.DT_F16, gelu)
