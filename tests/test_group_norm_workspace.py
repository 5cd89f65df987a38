"""The group norm's scratch: what the parameters' gradients pass through is bounded by the workgroups of a launch, not by the samples."""
import ctypes

import pytest
import torch

from immunostruct_amd import _lib, functional as HF
from oracle import sequence_ref as SR


def _floats(batch, n, channels, groups, type, offset=0, backward=1):
    p = 4096 + offset      # (alignment alone is looked at)
    args = _lib.GroupNorm(x=p, weight=4096, bias=4096, stats=4096, batch=batch, n=n, channels=channels, groups=groups, x_b=n * channels, x_n=channels,
                          type=type, weight_type=type, eps=1e-5)
    return _lib.load().is_group_norm_work_floats(ctypes.byref(args), backward)


@pytest.mark.parametrize("n,channels,groups,offset", [
    (1, 768, 16, 0), (1, 768, 32, 0), (1, 60, 12, 0), (1, 512, 8, 2), (1, 6, 2, 0), (3, 64, 8, 0), (16, 96, 3, 0), (1, 8200 * 2, 2, 0), (2, 4112, 2, 0),
    (9, 1031, 1, 0), (190, 64, 8, 0)])
def test_records_do_not_grow_with_the_batch(n, channels, groups, offset):
    """groups of 48, 24 and 5 channels, unaligned rows, a few rows a sample, groups wider than a workgroup: records of 2 fp32 rows of channels for 2048
    workgroups; 64 MB of them where a sample has several rows; an eighth of x in 16 bits where it has 32 or more (and per sample and group a few
    floats where a sample is spread over several workgroups)"""
    for type in (0, 1, 2):
        for batch in (3, 4096, 1 << 19):
            need = _floats(batch, n, channels, groups, type, offset)
            spread = _floats(batch, n, channels, groups, type, offset, backward=0)
            most = 2 * channels * min(batch, 2048)
            if n > 1:
                most = max(most, min(2 * channels * batch, 1 << 24))
            if n >= 32:
                most = max(most, batch * n * channels * 2 // 8 // 4)
            assert need - spread <= most, (type, batch)
            assert spread <= 2 * batch * groups * (1 + (channels // groups + 255) // 256)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("b,n,c,groups", [(5000, 1, 48, 2), (4100, 1, 15, 3), (2500, 2, 24, 1), (2100, 1, 8208, 1), (1100, 2, 2 * 2056, 2), (2060, 17, 512, 2)])
def test_many_samples(cuda_device, dtype, b, n, c, groups):
    """more samples than workgroups: values and gradients within the counted bounds, an empty sample and short ones among them"""
    gen = torch.Generator().manual_seed(7)
    x, dy = ((torch.randn(b, n, c, generator=gen) + 0.3).to(dtype).cuda() for _ in range(2))
    w, o = ((torch.randn(c, generator=gen) * 0.3 + 1).to(dtype).cuda().requires_grad_(True) for _ in range(2))
    lengths = [max(0, n - i % 3) for i in range(b)]
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    x.requires_grad_(True)
    y = HF.group_norm(x, groups, w, o, activation="silu", lengths=lens)
    got = dict(zip(("y", "dx", "dweight", "dbias"), (y,) + torch.autograd.grad(y, (x, w, o), dy)))
    want = SR.group_norm(x, groups, w, o, 1e-5, "silu", lengths, dy)
    for name, t in got.items():
        value, bound = want[name]
        off = (t.detach().cpu().double() - value).abs()
        assert bool((off <= bound).all()), f"{name}: {float((off / bound.clamp(min=1e-300)).max()):.2f} x its bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("cg", [1, 2, 3, 5, 7, 24, 33, 40, 63, 64, 65, 80, 96, 160, 264, 504, 520])
@pytest.mark.parametrize("groups", [1, 5, 70])
def test_single_rows_of_any_group_width(cuda_device, dtype, cg, groups):
    """groups that are no power of two of chunks, single elements (also by a row start off 16 bytes), more groups than a workgroup holds, empty rows"""
    gen = torch.Generator().manual_seed(8)
    b, c = 300, cg * groups
    wide = (torch.randn(b, 1, c + 1, generator=gen) + 0.3).to(dtype).cuda()
    dy = torch.randn(b, 1, c, generator=gen).to(dtype).cuda()
    w, o = ((torch.randn(c, generator=gen) * 0.3 + 1).to(dtype).cuda().requires_grad_(True) for _ in range(2))
    lengths = [int(i % 7 != 3) for i in range(b)]
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for x in (wide[..., :c].contiguous(), wide[..., 1:]):
        x = x.detach().requires_grad_(True)
        y = HF.group_norm(x, groups, w, o, activation="gelu", lengths=lens)
        got = dict(zip(("y", "dx", "dweight", "dbias"), (y,) + torch.autograd.grad(y, (x, w, o), dy)))
        want = _rows_reference(x, groups, w, o, lengths, dy)
        for name, t in got.items():
            value, bound = want[name]
            off = (t.detach().double() - value).abs()
            assert bool((off <= bound).all()), f"{name}: {float((off / bound.clamp(min=1e-300)).max()):.2f} x its bound"


def _rows_reference(x, groups, w, o, lengths, dy):
    """oracle.sequence_ref.group_norm's values and bounds for samples that are whole or empty (lengths 1 or 0), GELU and eps 1e-5, all samples and groups
    at once, in float64 on x's device"""
    b, n, c = x.shape
    cg = c // groups
    u, tiny, E32 = SR.half_step(x.dtype), SR.tiny_step(x.dtype), SR.E32
    X, DY, W, O = (t.detach().double() for t in (x, dy, w, o))
    live = torch.tensor(lengths, device=x.device).double()[:, None, None]
    part, d0 = (t.view(b, n, groups, cg).transpose(1, 2).reshape(b, groups, n * cg) for t in (X, DY))
    W3, O3 = (t.view(groups, 1, cg).expand(groups, n, cg).reshape(groups, n * cg) for t in (W, O))
    k = (n * cg / 64 + 32) * E32
    r = 1 / torch.sqrt(part.var(-1, correction=0, keepdim=True) + 1e-5)
    hat = (part - part.mean(-1, keepdim=True)) * r
    big = part.abs().amax(-1, keepdim=True) * r
    dhat = k * (big + hat.abs() * (1 + big * big * k))
    z = hat * W3 + O3
    y, slope = SR._activation(z, "gelu")
    dz_bound = dhat * W3.abs() + 4 * E32 * (z.abs() + O3.abs())
    out = {"y": (y, 1.2 * dz_bound + 32 * E32 * (y.abs() + z.abs()) + u * y.abs() + tiny)}
    d = d0 * slope
    dd = d0.abs() * (dz_bound + 32 * E32) + 4 * E32 * d.abs()
    t, dt = d * W3, dd * W3.abs() + 2 * E32 * (d * W3).abs()
    m1, m2 = t.mean(-1, keepdim=True), (t * hat).mean(-1, keepdim=True)
    dm1 = dt.mean(-1, keepdim=True) + k * t.abs().mean(-1, keepdim=True)
    dm2 = (dt * hat.abs() + t.abs() * dhat).mean(-1, keepdim=True) + k * (t * hat).abs().mean(-1, keepdim=True)
    dx = r * (t - m1 - hat * m2)
    out["dx"] = (dx, r * (dt + dm1 + hat.abs() * dm2 + dhat * m2.abs()) + (k + 8 * E32) * r * (t.abs() + m1.abs() + (hat * m2).abs()) + u * dx.abs() + tiny)
    out = {name: tuple((f * live).view(b, groups, n, cg).transpose(1, 2).reshape(b, n, c) for f in pair) for name, pair in out.items()}
    more, wt = (b / 4 + 8) * E32, SR.tiny_step(w.dtype)
    for name, v, e in (("dweight", d * hat, dd * hat.abs() + d.abs() * dhat + k * (d * hat).abs()), ("dbias", d, dd + k * d.abs())):
        v, e = ((f * live).sum(0).view(groups, n, cg).sum(1).flatten() for f in (v, e))
        out[name] = (v, e * (1 + more) + more * v.abs() * 4 + SR.half_step(w.dtype) * v.abs() + E32 * e + wt)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("b,n,groups,cg", [(1050, 2, 32, 256), (1050, 5, 32, 256), (1000, 2, 67, 128), (1000, 2, 67, 127)])
def test_records_beyond_64_megabytes(cuda_device, dtype, b, n, groups, cg):
    """workgroups that walk several samples with one, four and sixteen chunks a thread, and single elements"""
    gen = torch.Generator(device="cuda").manual_seed(9)
    assert b > (1 << 23) // (groups * cg)
    x, dy = ((torch.randn(b, n, groups * cg, generator=gen, device="cuda") + 0.3).to(dtype) for _ in range(2))
    w, o = ((torch.randn(groups * cg, generator=gen, device="cuda") * 0.3 + 1).to(dtype).requires_grad_(True) for _ in range(2))
    live = [int(i % 5 != 3) for i in range(b)]
    x.requires_grad_(True)
    y = HF.group_norm(x, groups, w, o, activation="gelu", lengths=torch.tensor(live, dtype=torch.int32, device="cuda") * n)
    got = dict(zip(("y", "dx", "dweight", "dbias"), (y,) + torch.autograd.grad(y, (x, w, o), dy)))
    want = _rows_reference(x, groups, w, o, live, dy)
    for name, t in got.items():
        value, bound = want[name]
        off = (t.detach().double() - value).abs()
        assert bool((off <= bound).all()), f"{name}: {float((off / bound.clamp(min=1e-300)).max()):.2f} x its bound"
