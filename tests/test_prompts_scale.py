"""The scales that prompt attention takes (made-up addresses, never read)."""
import ctypes
import math

import pytest
import torch

from layer_quant_amd import _abi


@pytest.mark.parametrize("scale,rc", [(math.nan, -1), (math.inf, -1), (-math.inf, -1), (3e38, -1), (-2.4e38, -1),
                                      (2.3e38, 0), (-2.3e38, 0), (1e-45, 0), (0.0, 0)])
def test_scales(scale, rc):
    """Finite ones whose product with log2(e) is finite. (No rows: an accepted call launches nothing.)"""
    t = _abi.LQTensor()
    t.data, t.dtype, t.ndim = 0x1000, _abi.DTYPE_CODES[torch.float32], 4
    for i, n in enumerate((1, 0, 2, 8)):
        t.shape[i], t.stride[i] = n, 1
    p = ctypes.pointer(t)
    assert _abi.lib().lq_prompt_attention(p, p, p, None, p, scale, None) == rc, _abi.last_error()
