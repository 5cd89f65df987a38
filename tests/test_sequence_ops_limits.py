"""The sequence operators at the ends of their sizes: what does not fit the kernels' 32-bit sizes is refused, what does works."""
import pytest
import torch

from immunostruct_amd import functional as HF

BIG = 2 ** 32 + 1      # (1 in 32 bits)
FREQ = torch.ones(1, dtype=torch.float64)


def _wide(*shape, dtype=torch.bfloat16):
    return torch.zeros(1, dtype=dtype).expand(*shape)


@pytest.mark.parametrize("shape", [(BIG, 1, 1, 2), (1, BIG, 1, 2), (1, 1, BIG, 2), (1, 1, 1, BIG), (2 ** 31, 1, 1, 2)])
def test_rotary_refuses_sizes_beyond_32_bits(shape):
    with pytest.raises(ValueError, match="2\\^31"):
        HF.rotary(_wide(*shape), None, FREQ)
    with pytest.raises(ValueError, match="2\\^31"):
        HF.rotary(_wide(*shape[:2], 1, shape[3]), _wide(*shape), FREQ)


@pytest.mark.parametrize("q,k,v", [((BIG, 1, 2, 8), (BIG, 1, 2, 8), (BIG, 1, 1, 8)), ((1, BIG, 2, 8), (1, 1, 2, 8), (1, 1, 1, 8)),
                                   ((1, 1, 2, 8), (1, BIG, 2, 8), (1, BIG, 1, 8)), ((1, 1, 2 ** 32 + 2, 8), (1, 1, 2, 8), (1, 1, 1, 8))])
def test_attention_refuses_sizes_beyond_32_bits(q, k, v):
    with pytest.raises(ValueError, match="2\\^31"):
        HF.differential_attention(_wide(*q), _wide(*k), _wide(*v), _wide(q[2] // 2))


@pytest.mark.parametrize("shape", [(BIG, 1, 8), (1, BIG, 8), (1, 1, BIG), (BIG, 8), (1, 2 ** 16, 2 ** 16 + 1, 8)])
def test_group_norm_refuses_sizes_beyond_32_bits(shape):
    with pytest.raises(ValueError, match="2\\^31"):
        HF.group_norm(_wide(*shape), 1)
