"""Views that torch allows and kernels rarely meet: the strides of dimensions with one element, which mean nothing."""
import pytest
import torch

from immunostruct_amd import functional as HF

pytestmark = pytest.mark.gpu
FREQ = torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64)


def _odd(t):
    """the same elements, with strides nobody can use for every dimension of one element"""
    strides = [s if n > 1 else 5 + (1 << 26) for n, s in zip(t.shape, t.stride())]
    return t.detach().as_strided(t.shape, strides).requires_grad_(t.requires_grad)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("b,nq,nk,h", [(1, 7, 9, 2), (1, 1, 9, 1), (2, 1, 1, 1), (1, 1, 1, 1)])
def test_attention_and_rotary(cuda_device, dtype, b, nq, nk, h):
    gen = torch.Generator().manual_seed(1)
    make = lambda *s: torch.randn(*s, generator=gen).to(dtype).cuda().requires_grad_(True)
    q, k, v, lam, do = make(b, nq, 2 * h, 8), make(b, nk, 2 * h, 8), make(b, nk, h, 16), make(h), make(b, nq, h, 16).detach()
    run = lambda *t: (lambda out: (out,) + torch.autograd.grad(out, t, do))(HF.differential_attention(*t))
    assert all(torch.equal(x, y) for x, y in zip(run(q, k, v, lam), run(_odd(q), _odd(k), _odd(v), _odd(lam))))
    assert torch.equal(HF.rotary(q, None, FREQ)[0], HF.rotary(_odd(q), None, FREQ)[0])


@pytest.mark.parametrize("b,n,c", [(1, 30, 64), (5, 1, 64), (1, 1, 64), (1, 3000, 64), (5, 1, 1040)])
def test_group_norm(cuda_device, b, n, c):
    x = torch.randn(b, n, c, generator=torch.Generator().manual_seed(2)).bfloat16().cuda().requires_grad_(True)
    dy = torch.ones_like(x)
    run = lambda t: (lambda y: (y,) + torch.autograd.grad(y, t, dy))(HF.group_norm(t, 2, activation="silu"))
    assert all(torch.equal(p, r) for p, r in zip(run(x), run(_odd(x))))


def test_frequencies_changed_before_the_backward(cuda_device):
    freq, q = FREQ.clone(), torch.randn(1, 5, 2, 8, device="cuda", requires_grad=True)
    out = HF.rotary(q, None, freq)[0]
    freq.mul_(2.0)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


def test_views_of_conjugates(cuda_device):
    """a float view whose memory holds the opposite sign (torch keeps that as a mark on the tensor)"""
    def conjugate(t):
        return torch.complex(torch.zeros_like(t), -t.detach()).conj().imag.requires_grad_(True)

    gen = torch.Generator().manual_seed(5)
    make = lambda *s: torch.randn(*s, generator=gen).cuda().requires_grad_(True)
    q, k, v, lam, x, w, o = make(1, 7, 2, 8), make(1, 9, 2, 8), make(1, 9, 1, 16), make(1), make(3, 5, 8), make(8), make(8)
    assert conjugate(q).is_neg() and torch.equal(conjugate(q), q)
    for call, inputs in ((HF.differential_attention, (q, k, v, lam)), (lambda a, b: torch.cat(HF.rotary(a, b, FREQ), dim=1), (q, make(1, 7, 2, 8))),
                         (lambda a, b, c: HF.group_norm(a, 2, b, c, activation="silu"), (x, w, o))):
        want, marked = call(*inputs), [conjugate(t) for t in inputs]
        dy = torch.randn(want.shape, generator=gen).cuda()
        with torch.no_grad():
            assert torch.equal(call(*marked), want)
        full = torch.autograd.grad(want, inputs, dy)
        assert all(torch.equal(a, b) for a, b in zip(full, torch.autograd.grad(call(*marked), marked, conjugate(dy).detach())))
