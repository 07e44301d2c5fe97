"""Attention over block-scaled pools whose scales differ widely from block to block, against float64
(``Case`` and its tolerance: ``test_gpu_block_attention``)."""

import pytest
import torch

from tests.test_gpu_block_attention import CODES, Case, _near, _say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kernel(pkg):
    return pkg.MI355XPagedAttention()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype,dim,bs", [(torch.bfloat16, 128, 16), (torch.float16, 64, 32), (torch.bfloat16, 96, 64),
                                          (torch.float16, 128, 48), (torch.bfloat16, 128, 8)])
def test_prompts_whose_key_scales_differ_by_tile(kernel, dev, codes, dtype, dim, bs):
    """Key scales a hundredfold apart, so that a tile's weights by another tile's scales would show; every
    repetition has the same bits, whatever its waves wait for."""
    _say("key scales", codes, dtype, dim, bs)
    c = Case(codes, dtype, [(1100, 1100), (900, 200), (130, 129), (65, 65), (64, 64)], 4, 2, dim, bs, seed=21,
             spread=0.01)
    for window in (0, 300):
        got = c.packed(kernel, dev, window)
        _near(got, *c.expect(window), c.q)
        for _ in range(8):
            assert torch.equal(c.packed(kernel, dev, window), got)
