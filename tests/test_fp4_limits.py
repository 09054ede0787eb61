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
