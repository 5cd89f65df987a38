"""Differential attention in the 16-bit types rounds its results and nothing else: values and gradients against 64 bits within bounds that hold no
rounding of weights, score gradients or saved products to the type, and no farther from 64 bits than the rounding of the results alone."""
import pytest
import torch

from immunostruct_amd import functional as HF
from oracle import sequence_ref as SR

pytestmark = pytest.mark.gpu


def _randn(*shape, dtype, seed, mean=0.0, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * std + mean).to(dtype).cuda()


def _inputs(dtype, b, nq, nk, h, hk, d, dv):
    return (_randn(b, nq, 2 * h, d, dtype=dtype, seed=1), _randn(b, nk, 2 * hk, d, dtype=dtype, seed=2), _randn(b, nk, hk, dv, dtype=dtype, seed=3),
            _randn(h, dtype=dtype, seed=4, mean=0.5, std=0.2), _randn(b, nq, h, dv, dtype=dtype, seed=5))


# every build of the kernels: widths 32, 64, 128 and element by element; one pair of waves (<= 32 rows) and more; split keys, split rows
SHAPES = [(2, 150, 150, 2, 1, 32, 64, [150, 97], None), (1, 200, 200, 4, 2, 64, 128, None, "start"), (2, 70, 260, 2, 2, 128, 256, [260, 131], "end"),
          (1, 90, 1100, 1, 1, 20, 36, None, None), (3, 1, 600, 8, 2, 64, 128, [600, 0, 333], "end"), (1, 64, 2048, 1, 1, 32, 64, None, None),
          (1, 700, 90, 2, 1, 64, 128, None, "start")]
CASES = [(t, s) for s in SHAPES for t in (torch.bfloat16, torch.float16) if t == torch.bfloat16 or s[2] < 2048]


@pytest.mark.parametrize("dtype,shape", CASES, ids=lambda x: str(x)[6:] if isinstance(x, torch.dtype) else "-".join(str(i) for i in x[:7]) + f"-{x[8]}")
def test_only_the_results_are_rounded(cuda_device, dtype, shape):
    b, nq, nk, h, hk, d, dv, lengths, causal = shape
    *leaves, do = _inputs(dtype, b, nq, nk, h, hk, d, dv)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = SR.differential_attention(*leaves, lengths, causal, d ** -0.5, do, full=True)
    with torch.no_grad():
        got = {"o (no gradient)": HF.differential_attention(*leaves, lens, causal)}
    leaves = [t.requires_grad_(True) for t in leaves]
    got["o"] = HF.differential_attention(*leaves, lens, causal)
    got.update(zip(("dq", "dk", "dv", "dlam"), torch.autograd.grad(got["o"], leaves, do)))
    for name, t in got.items():
        value, bound = want[name.split()[0]]
        off = (t.detach().cpu().double() - value).abs()
        assert bool((off <= bound).all()), f"{name}: {float((off / bound.clamp(min=1e-300)).max()):.2f} x its bound"
        if t.numel() >= 1000:
            # the norm of the error against that of rounding the 64-bit value.  A 32-bit score of d = 128 products is off by 1.2e-4 / sqrt(d) =
            # 1.1e-5 (f of the oracle, with random signs), a result by the like of it, dS by three such (P, dP, D); rounding to fp16 alone is
            # 2.1e-4 of the norm: sqrt(1 + 3 (1.1e-5 / 2.1e-4)^2) = 1.004
            alone = (value.to(dtype).double() - value).norm()
            assert off.norm() <= 1.01 * alone, f"{name}: {float(off.norm() / alone):.3f} x the error of rounding alone"
