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


@pytest.mark.gpu
@pytest.mark.parametrize("n,channels,groups", [(2, 6, 2), (34, 2, 1)])
def test_group_norm_beyond_a_launch(cuda_device, n, channels, groups):
    """more samples than one launch has threads for: every sample as in a small call"""
    small, b = 2 ** 10, 2 ** 24 + 2 ** 10
    gen = torch.Generator().manual_seed(3)
    x, dy = (torch.randn(small, n, channels, generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    w, o = (torch.randn(channels, generator=gen).cuda().requires_grad_(True) for _ in range(2))
    lens = torch.arange(small, dtype=torch.int32, device="cuda") % (n + 1)

    def run(times):
        leaf = x.repeat(times, 1, 1).requires_grad_(True)
        y = HF.group_norm(leaf, groups, w, o, activation="silu", lengths=lens.repeat(times))
        return (y.detach(),) + torch.autograd.grad(y, (leaf, w, o), dy.repeat(times, 1, 1))

    one, many = run(1), run(b // small)
    for a, c in zip(one[:2], many[:2]):
        # (the plan of a launch goes by its batch: another order of the same 32-bit sums ahead of the rounding to bf16, a step of which is 2^-7)
        c = c.view(-1, small, n, channels)
        assert torch.equal(c[:1].expand_as(c), c)
        assert bool(((c[0].float() - a.float()).abs() <= 2.0 ** -7 * a.float().abs() + 1e-5).all())
    for a, c in zip(one[2:], many[2:]):      # b / small times the same sums: 32 bits over a chain of up to b / 64 of them
        assert bool(((c / (b // small) - a).abs() <= (b / 64 + 64) * 2.0 ** -24 * (a.abs().max() + 1)).all())


@pytest.mark.gpu
def test_group_norm_joins_beyond_a_launch(cuda_device):
    """more samples and groups in the long form than one launch joins"""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB of device memory")
    small, times = 2 ** 10, 2 ** 11 + 1
    x = torch.randn(small, 129, 32, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).cuda()
    one, many = HF.group_norm(x, 32), HF.group_norm(x.repeat(times, 1, 1), 32).view(times, small, 129, 32)
    for i in range(0, times, 128):
        part = many[i:i + 128]
        assert torch.equal(many[:1].expand_as(part), part)
    assert bool(((many[0].float() - one.float()).abs() <= 2.0 ** -7 * one.float().abs() + 1e-5).all())


@pytest.mark.gpu
def test_attention_beyond_a_launch(cuda_device):
    """more rows than one launch of the backward's row sums has threads for"""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    small, times = 2 ** 12, 2 ** 16 + 1
    gen = torch.Generator().manual_seed(4)
    q, do = torch.randn(1, small, 2, 1, generator=gen).to(torch.bfloat16).cuda(), torch.randn(1, small, 1, 1, generator=gen).to(torch.bfloat16).cuda()
    k, v, lam = torch.randn(1, 5, 2, 1, generator=gen).to(torch.bfloat16).cuda(), torch.randn(1, 5, 1, 1, generator=gen).to(torch.bfloat16).cuda(), torch.tensor([0.5], device="cuda")

    def run(times):
        leaf = q.repeat(1, times, 1, 1).requires_grad_(True)
        out = HF.differential_attention(leaf, k, v, lam)
        return out.detach(), torch.autograd.grad(out, leaf, do.repeat(1, times, 1, 1))[0]

    for a, c in zip(run(1), run(times)):
        c = c.view(times, small, -1)
        assert torch.equal(c[:1].expand_as(c), c) and torch.equal(c[0], a.view(small, -1))
