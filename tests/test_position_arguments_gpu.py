"""Arguments of relative_attention at the edges of what its documentation allows."""
import math

import pytest
import torch

from pytorch_distributed_training_amd.ops import relative_attention
from pytorch_distributed_training_amd.ops.attention import mask_bits


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int8, torch.int16, torch.uint8, torch.int32, torch.int64, torch.bool])
@pytest.mark.parametrize("S", [50, 300])
def test_masks_of_every_whole_number_type(dtype, S):
    gen = torch.Generator(device="cuda").manual_seed(S)
    q, k, v = (torch.randn(2, S, 2, 64, generator=gen, device="cuda").half() for _ in range(3))
    valid = torch.rand(2, S, generator=gen, device="cuda") < 0.7
    value = {torch.int8: -128, torch.int16: 256, torch.int32: 1 << 30, torch.int64: 1 << 40, torch.uint8: 128}.get(dtype, 1)
    mask = valid.to(dtype) * value if dtype != torch.bool else valid
    assert torch.equal(relative_attention(q, k, v, key_mask=mask), relative_attention(q, k, v, key_mask=valid))
    assert torch.equal(mask_bits(mask), mask_bits(valid))


def test_complex_masks_are_refused():
    q = torch.zeros(1, 4, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="truth values"):
        relative_attention(q, q, q, key_mask=torch.ones(1, 4, dtype=torch.complex64))
