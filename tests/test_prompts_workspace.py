"""Workspace sizes: a call that is refused for its sizes has none, so that no scratch is allocated for it, and
every size that a call takes stays within what its launches use."""
import pytest
import torch

from layer_quant_amd import _abi

F32, F16, BF = (_abi.DTYPE_CODES[t] for t in (torch.float32, torch.float16, torch.bfloat16))


@pytest.mark.parametrize("sizes", [
    (1, 16384, 1, 128, 64, 257), (1, 16384, 1, 128, 64, 1 << 40), (70000, 1 << 20, 1, 8, 16, 16),
    (1, 1 << 31, 1, 8, 16, 16), (1 << 16, 1 << 16, 0, 8, 16, 16), (1, 16384, 1, 8, 1 << 17, 16),
    (1, 16384, 1, 1 << 20, 64, 128), (1, 16384, 1, 1 << 62, 64, 128), (1 << 62, 1 << 62, 0, 1 << 62, 1 << 62, 1)])
@pytest.mark.parametrize("dtype", [F32, F16, BF])
def test_scan_sizes_that_are_refused(dtype, sizes):
    assert _abi.lib().lq_prompt_scan_workspace(dtype, *sizes) == 0


def test_scan_sizes_that_are_taken():
    lib = _abi.lib()
    assert lib.lq_prompt_scan_workspace(F32, 1, 16384, 1, 128, 64, 256) > 0
    assert lib.lq_prompt_scan_workspace(BF, 65535, 1000, 1, 2, 64, 128) == 1000 * 2 * 16  # no segments


def test_scores_sizes():
    lib = _abi.lib()
    assert lib.lq_token_logprobs_workspace(64, 131072, 32) > 0
    for sizes in ((64, 131072, 33), (64, 131072, 1 << 30), (64, 1 << 40, 0), (64, 131072, -1)):
        assert lib.lq_token_logprobs_workspace(*sizes) == 0
