"""Rotary positions, differential attention and group norm against their plain 64-bit forms (oracle.sequence_ref), place by place within the
bounds that count the kernels' roundings; and as they are used: strided inputs, masks that leave nothing, other streams, captured graphs."""
import itertools

import pytest
import torch

from immunostruct_amd import functional as HF
from immunostruct_amd import nn as HN
from oracle import sequence_ref as SR

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = {torch.float32: "fp32", torch.bfloat16: "bf16", torch.float16: "fp16"}
each_type = pytest.mark.parametrize("dtype", TYPES, ids=[NAMES[t] for t in TYPES])


def _randn(*shape, dtype, seed, mean=0.0, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * std + mean).to(dtype).cuda()


def _within(got, want, what):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - value).abs()
    worst = (off / bound.clamp(min=1e-300)).masked_fill(off == 0, 0.0)
    assert bool((off <= bound).all()), f"{what}: {float(worst.max()):.2f} x the bound at {tuple(int(i) for i in (worst == worst.max()).nonzero()[0])}"


# ---- rotary ---------------------------------------------------------------------------------------------------------------
@each_type
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("b,n,heads,kv,width,dims,start", [
    (1, 1, 1, 1, 2, 2, 0), (2, 5, 3, 1, 16, 16, 0), (3, 17, 4, 2, 24, 10, 7), (2, 33, 2, 2, 64, 32, 1_000_003), (1, 3, 5, 1, 80, 80, 2 ** 33),
    (4, 190, 2, 2, 32, 32, 0), (2, 9, 40, 8, 128, 64, 131072)])
def test_rotary(cuda_device, dtype, layout, b, n, heads, kv, width, dims, start):
    q, k = _randn(b, n, heads, width, dtype=dtype, seed=1).requires_grad_(True), _randn(b, n, kv, width, dtype=dtype, seed=2).requires_grad_(True)
    pos = (start + torch.arange(n) * 3 + torch.arange(b)[:, None]).cuda()
    rope = HN.RotaryEmbedding(dims, layout=layout, scaling=dict(kind="yarn", factor=4.0, original_length=4096) if dims > 8 else None)
    gq, gk = _randn(b, n, heads, width, dtype=dtype, seed=3), _randn(b, n, kv, width, dtype=dtype, seed=4)
    out = rope(q, k, pos)
    grads = torch.autograd.grad(out, (q, k), (gq, gk))
    for x, o, g, d, name in ((q, out[0], gq, grads[0], "q"), (k, out[1], gk, grads[1], "k")):
        _within(o, SR.rotary(x, rope.freq, pos, layout, rope.amplitude), name)
        _within(d, SR.rotary(g, rope.freq, pos, layout, rope.amplitude, inverse=True), "d" + name)


def test_rotary_positions_and_strides(cuda_device):
    """int32 and one-dimensional positions, none at all, a broadcast one; q and k as views of one projection; only one of them needing grad"""
    b, n, d = 3, 7, 32
    rope = HN.RotaryEmbedding(d)
    qkv = _randn(b, n, 6, d, dtype=torch.bfloat16, seed=5)
    q, k = qkv[:, :, :4], qkv[:, :, 4:]
    base = rope(q.contiguous(), k.contiguous())
    for pos in (None, torch.arange(n, device="cuda", dtype=torch.int32), torch.arange(n, device="cuda").expand(b, n),
                torch.arange(2 * n, device="cuda")[::2] // 2):
        got = rope(q, k, pos)
        assert all(torch.equal(x, y) for x, y in zip(got, base))
    turned = rope(q.transpose(1, 2).contiguous().transpose(1, 2), k.expand(b, n, 2, d))      # head-major memory
    assert all(torch.equal(x, y) for x, y in zip(turned, base))
    alone, none = rope(q)
    assert none is None and torch.equal(alone, base[0])
    odd = torch.zeros(b, n, 4, d + 1, dtype=torch.bfloat16, device="cuda")[..., 1:]      # rows that are not 16-byte aligned
    odd.copy_(q)
    assert torch.equal(rope(odd)[0], base[0])
    shared = _randn(1, n, 1, d, dtype=torch.float32, seed=6).expand(b, n, 4, d)      # a broadcast input: its gradient is a sum
    leaf = shared[:1, :, :1].clone().requires_grad_(True)
    out, _ = rope(leaf.expand(b, n, 4, d))
    out.sum().backward()
    one = leaf.detach().clone().requires_grad_(True)
    rope(one)[0].sum().backward()
    assert torch.allclose(leaf.grad, 12 * one.grad, rtol=1e-6, atol=1e-6)
    kk = k.clone().requires_grad_(True)
    (rope(q, kk)[1].float().sum()).backward()
    assert kk.grad is not None
    assert [t.shape for t in rope(q[:0], k[:0])] == [(0, n, 4, d), (0, n, 2, d)]


# ---- differential attention ---------------------------------------------------------------------------------------------------
def _attention_inputs(dtype, b, nq, nk, h, hk, d, dv, lam_dtype=None):
    lam = _randn(h, dtype=lam_dtype or dtype, seed=14, mean=0.5, std=0.2)
    return (_randn(b, nq, 2 * h, d, dtype=dtype, seed=11), _randn(b, nk, 2 * hk, d, dtype=dtype, seed=12), _randn(b, nk, hk, dv, dtype=dtype, seed=13), lam)


SHAPES = [      # b, nq, nk, heads, kv_heads, d, dv, lengths, causal
    (1, 1, 1, 1, 1, 1, 1, None, None), (2, 3, 5, 2, 1, 4, 8, [5, 0], None), (1, 33, 31, 1, 1, 8, 16, None, "start"),
    (3, 70, 70, 4, 2, 16, 32, [70, 33, 1], "start"), (2, 45, 130, 2, 2, 32, 64, [130, 64], "end"), (2, 129, 65, 3, 1, 24, 48, [65, 20], "end"),
    (2, 190, 190, 1, 1, 32, 64, [190, 171], None), (1, 257, 300, 4, 1, 64, 128, None, "end"), (4, 1, 700, 8, 2, 64, 128, [700, 1, 0, 333], "end"),
    (1, 40, 513, 2, 1, 40, 72, [512], None), (2, 5, 40, 1, 1, 20, 7, [40, 3], "end")]
WIDE = [(2, 37, 70, 4, 2, 128, 256, [70, 9], None), (1, 130, 130, 1, 1, 96, 192, None, "start"), (3, 1, 300, 4, 4, 128, 256, [300, 0, 17], "end")]


@each_type
@pytest.mark.parametrize("shape", SHAPES + WIDE, ids=lambda s: "-".join(str(x) for x in s[:7]) + f"-{s[8]}")
def test_differential_attention(cuda_device, dtype, shape):
    b, nq, nk, h, hk, d, dv, lengths, causal = shape
    if dtype == torch.float32 and d > 64:
        with pytest.raises(NotImplementedError):
            HF.differential_attention(*_attention_inputs(dtype, b, nq, nk, h, hk, d, dv))
        return
    q, k, v, lam = (t.requires_grad_(True) for t in _attention_inputs(dtype, b, nq, nk, h, hk, d, dv))
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    do = _randn(b, nq, h, dv, dtype=dtype, seed=15)
    want = SR.differential_attention(q, k, v, lam, lengths, causal, d ** -0.5, do)
    with torch.no_grad():
        _within(HF.differential_attention(q, k, v, lam, lens, causal), want["o"], "o (no gradient)")
    out = HF.differential_attention(q, k, v, lam, lens, causal)
    _within(out, want["o"], "o")
    grads = torch.autograd.grad(out, (q, k, v, lam), do)
    for g, name in zip(grads, ("dq", "dk", "dv", "dlam")):
        _within(g, want[name], name)
    again = torch.autograd.grad(HF.differential_attention(q, k, v, lam, lens, causal), (q, k, v, lam), do)
    assert all(torch.equal(x, y) for x, y in zip(grads, again)), "not reproducible"


def test_attention_garbage_behind_the_lengths(cuda_device):
    """whatever stands at or behind a sample's length (NaN, infinities) has no effect, and those keys get zero gradients"""
    for dtype, causal in itertools.product(TYPES, (None, "start", "end")):
        q, k, v, lam = _attention_inputs(dtype, 3, 50, 90, 2, 1, 32, 64)
        lens = torch.tensor([90, 41, 0], dtype=torch.int32, device="cuda")
        do = _randn(3, 50, 2, 64, dtype=dtype, seed=16)

        def run(fill):
            kk, vv = k.clone(), v.clone()
            for i, n in enumerate(lens.tolist()):
                kk[i, n:], vv[i, n:] = fill, fill
            leaves = [t.clone().requires_grad_(True) for t in (q, kk, vv, lam)]
            out = HF.differential_attention(*leaves, lens, causal)
            return (out,) + torch.autograd.grad(out, leaves, do)

        clean = run(0.0)
        for fill in (float("nan"), float("inf"), torch.finfo(dtype).min):
            assert all(torch.equal(x, y) for x, y in zip(clean, run(fill)))
        assert not clean[2][1, 41:].any() and not clean[3][1, 41:].any() and not clean[2][2].any() and not clean[0][2].any()


@each_type
@pytest.mark.parametrize("nq,nk", [(5, 64), (40, 200), (130, 131)])
def test_attention_garbage_that_no_query_sees(cuda_device, dtype, nq, nk):
    """queries from the start over a buffer that is longer than they are: what stands behind the last query's position does not matter"""
    q, k, v, lam = _attention_inputs(dtype, 2, nq, nk, 2, 1, 32, 64)
    k[:, nq:], v[:, nq:] = float("nan"), float("inf")
    do = _randn(2, nq, 2, 64, dtype=dtype, seed=16)
    want = SR.differential_attention(q, k[:, :nq], v[:, :nq], lam, None, "start", 32 ** -0.5, do)
    leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]
    out = HF.differential_attention(*leaves, causal="start")
    _within(out, want["o"], "o")
    grads = torch.autograd.grad(out, leaves, do)
    assert not grads[1][:, nq:].any() and not grads[2][:, nq:].any()
    for g, name in zip(grads, ("dq", "dk", "dv", "dlam")):
        _within(g[:, :nq] if name in ("dk", "dv") else g, want[name], name)


def test_attention_strides_scale_and_types(cuda_device):
    dtype = torch.bfloat16
    q, k, v, lam = _attention_inputs(dtype, 2, 70, 70, 4, 2, 32, 64)
    base = HF.differential_attention(q, k, v, lam)
    pack = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], dim=2)      # one projection's output
    qs, ks, vs = pack.split([8 * 32, 4 * 32, 2 * 64], dim=2)
    assert torch.equal(HF.differential_attention(qs.view(2, 70, 8, 32), ks.view(2, 70, 4, 32), vs.view(2, 70, 2, 64), lam), base)
    head_major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(HF.differential_attention(*head_major, lam), base)
    odd = []      # rows that are not 16-byte aligned
    for t in (q, k, v):
        o = torch.zeros(*t.shape[:3], t.shape[3] + 1, dtype=dtype, device="cuda")[..., 1:]
        odd.append(o.copy_(t))
    # (those run element by element in tiles of another width, another order of the same sums: within the bound, not bit for bit)
    _within(HF.differential_attention(*odd, lam), SR.differential_attention(q, k, v, lam, None, None, 32 ** -0.5)["o"], "unaligned")
    column = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)]      # an innermost stride that is not 1: copied
    assert torch.equal(HF.differential_attention(*column, lam), base)
    want = SR.differential_attention(q, k, v, lam.float(), None, None, 0.3, base)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, lam.float())]
    out = HF.differential_attention(*leaves, scale=0.3)
    _within(out, want["o"], "o")
    for g, name in zip(torch.autograd.grad(out, leaves, base), ("dq", "dk", "dv", "dlam")):
        _within(g, want[name], name)
    # a broadcast batch: the gradient is the sum over what it was broadcast to
    leaf = k[:1].clone().requires_grad_(True)
    HF.differential_attention(q, leaf.expand(2, -1, -1, -1), v, lam).float().sum().backward()
    assert leaf.grad.shape == (1, 70, 4, 32)
    assert HF.differential_attention(q[:, :0], k, v, lam).shape == (2, 0, 4, 64)
    empty = HF.differential_attention(q, k[:, :0].detach().requires_grad_(True), v[:, :0], lam)
    assert not empty.any() and empty.requires_grad


@each_type
def test_attention_lam_of_any_sign(cuda_device, dtype):
    """negative, zero and mixed weights of the second map, in groups that do and do not divide a tile of 32 rows"""
    for heads, lam in ((2, (-0.7, -0.2)), (2, (0.0, 0.4)), (3, (0.5, -1.5, 0.0)), (5, (0.1, 2.0, -0.3, 1.0, 0.6))):
        q, k, v, _ = _attention_inputs(dtype, 2, 50, 77, heads, 1, 32, 64)
        leaves = [t.requires_grad_(True) for t in (q, k, v, torch.tensor(lam, dtype=dtype, device="cuda"))]
        do = _randn(2, 50, heads, 64, dtype=dtype, seed=17)
        lens = torch.tensor([77, 60], dtype=torch.int32, device="cuda")
        want = SR.differential_attention(*leaves, lens.tolist(), "end", 32 ** -0.5, do)
        out = HF.differential_attention(*leaves, lens, "end")
        _within(out, want["o"], f"o {lam}")
        for g, name in zip(torch.autograd.grad(out, leaves, do), ("dq", "dk", "dv", "dlam")):
            _within(g, want[name], f"{name} {lam}")


@each_type
@pytest.mark.parametrize("nq,nk,heads,kv,lengths,causal", [
    (1, 700, 33, 1, [700, 31], "end"), (5, 300, 7, 1, [300, 3], "end"), (1, 2100, 4, 2, [5000, -3], "end"), (3, 40, 40, 1, [-1, 41], None),
    (33, 129, 64, 2, [129, 64], "end"), (2, 5000, 1, 1, [4999, 1], None)])
def test_attention_group_sizes_and_lengths_out_of_range(cuda_device, dtype, nq, nk, heads, kv, lengths, causal):
    """groups that do not divide a tile or are wider than one, lengths below zero and above nk (taken as 0 and nk), split keys and rows"""
    leaves = [t.requires_grad_(True) for t in _attention_inputs(dtype, 2, nq, nk, heads, kv, 16, 32)]
    do = _randn(2, nq, heads, 32, dtype=dtype, seed=19)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = SR.differential_attention(*leaves, [max(0, min(nk, n)) for n in lengths], causal, 0.25, do)
    with torch.no_grad():
        _within(HF.differential_attention(*leaves, lens, causal), want["o"], "o (no gradient)")
    out = HF.differential_attention(*leaves, lens, causal)
    _within(out, want["o"], "o")
    for g, name in zip(torch.autograd.grad(out, leaves, do), ("dq", "dk", "dv", "dlam")):
        _within(g, want[name], name)


def test_attention_infinite_scores_of_narrow_heads(cuda_device):
    """a key whose last element is -inf has weight 0 for the queries that are positive there (heads narrower than the kernels' width: the
    elements that are not there must not meet the infinity)"""
    for dtype, d in ((torch.float32, 8), (torch.bfloat16, 40), (torch.float16, 8)):
        q, k, v, lam = _attention_inputs(dtype, 1, 40, 70, 1, 1, d, 2 * d)
        q[..., -1] = q[..., -1].abs() + 0.5
        k[:, 13, :, -1] = float("-inf")
        keep = [i for i in range(70) if i != 13]
        want = SR.differential_attention(q, k[:, keep], v[:, keep], lam, None, None, d ** -0.5)
        _within(HF.differential_attention(q, k, v, lam), want["o"], "o")


def test_attention_unaligned_gradient_and_second_derivative(cuda_device):
    q, k, v, lam = (t.requires_grad_(True) for t in _attention_inputs(torch.bfloat16, 1, 33, 33, 1, 1, 16, 32))
    out = HF.differential_attention(q, k, v, lam)
    g = _randn(1 * 33 * 32 + 1, dtype=torch.bfloat16, seed=18)[1:].view(1, 33, 1, 32)
    got = torch.autograd.grad(out, (q, k, v, lam), g, retain_graph=True)
    want = torch.autograd.grad(out, (q, k, v, lam), g.clone(), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(out, q, g, create_graph=True)
    x = _randn(3, 8, dtype=torch.float32, seed=19).requires_grad_(True)
    y = HF.group_norm(x, 2)
    gy = _randn(25, dtype=torch.float32, seed=20)[1:].view(3, 8)
    assert torch.equal(*(torch.autograd.grad(y, x, t, retain_graph=True)[0] for t in (gy, gy.clone())))


def test_errors_are_the_packages(cuda_device):
    """what the library refuses behind the package's own checks arrives as HipExtensionError with the library's text"""
    from immunostruct_amd import _lib
    q, k, v, lam = _attention_inputs(torch.float32, 1, 3, 3, 1, 1, 8, 16)
    with pytest.raises(_lib.HipExtensionError, match="is_diff_attention_fwd: invalid argument"):
        HF.differential_attention(q, k, v, lam, scale=3e38)


def test_attention_large_scores_and_offsets(cuda_device):
    """scores far apart (the running maximum moves at the end), all equal, and of magnitude 1e4"""
    for dtype in TYPES:
        q, k, v, lam = _attention_inputs(dtype, 1, 40, 200, 1, 1, 32, 64)
        k = k * torch.linspace(0.01, 12.0, 200, device="cuda")[:, None, None].to(dtype)
        want = SR.differential_attention(q, k, v, lam, None, None, 32 ** -0.5)
        _within(HF.differential_attention(q, k, v, lam), want["o"], "rising scores")
        want = SR.differential_attention(q, k.flip(1), v, lam, None, None, 32 ** -0.5)
        _within(HF.differential_attention(q, k.flip(1), v, lam), want["o"], "falling scores")
        flat = torch.zeros_like(k)
        want = SR.differential_attention(q, flat, v, lam, None, None, 32 ** -0.5)
        _within(HF.differential_attention(q, flat, v, lam), want["o"], "equal scores")


def test_attention_cache_beyond_32_bit_offsets(cuda_device):
    """one key head of a cache whose samples lie more than 2^31 elements apart"""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    big = torch.zeros(2, (2 ** 31 + 4096) // 64, 64, dtype=torch.bfloat16, device="cuda")
    k, v = big[:, -96:, :32].unflatten(2, (2, 16)), big[:, -96:, 32:].unflatten(2, (1, 32))
    kk, vv = _randn(2, 96, 2, 16, dtype=torch.bfloat16, seed=21), _randn(2, 96, 1, 32, dtype=torch.bfloat16, seed=22)
    k.copy_(kk), v.copy_(vv)
    q, lam = _randn(2, 3, 2, 16, dtype=torch.bfloat16, seed=23), _randn(1, dtype=torch.bfloat16, seed=24)
    assert torch.equal(HF.differential_attention(q, k, v, lam), HF.differential_attention(q, kk, vv, lam))


# ---- group norm -------------------------------------------------------------------------------------------------------------
@each_type
@pytest.mark.parametrize("activation", [None, "silu", "gelu", "relu"])
@pytest.mark.parametrize("b,n,c,groups,lengths", [
    (1, 1, 1, 1, None), (3, 1, 64, 8, None), (300, 1, 128, 4, None), (5, 1, 60, 4, None), (2, 1, 4096, 2, None), (2, 11, 64, 4, [11, 5]), (3, 190, 64, 8, [190, 77, 0]),
    (2, 33, 6, 3, None), (2, 40, 100, 5, [40, 1]), (1, 2100, 96, 3, None), (2, 3000, 32, 32, [3000, 2999]), (2, 1300, 40, 1, [7, 1300]),
    (3, 2, 2560, 8, [2, 1, 0])])
def test_group_norm(cuda_device, dtype, activation, b, n, c, groups, lengths):
    x = _randn(b, n, c, dtype=dtype, seed=31, mean=0.7, std=1.5).requires_grad_(True)
    w, o = _randn(c, dtype=dtype, seed=32, mean=1.0, std=0.3).requires_grad_(True), _randn(c, dtype=dtype, seed=33, std=0.3).requires_grad_(True)
    dy = _randn(b, n, c, dtype=dtype, seed=34)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = SR.group_norm(x, groups, w, o, 1e-5, activation, lengths, dy)
    y = HF.group_norm(x, groups, w, o, activation=activation, lengths=lens)
    _within(y, want["y"], "y")
    grads = torch.autograd.grad(y, (x, w, o), dy)
    for g, name in zip(grads, ("dx", "dweight", "dbias")):
        _within(g, want[name], name)
    again = torch.autograd.grad(HF.group_norm(x, groups, w, o, activation=activation, lengths=lens), (x, w, o), dy)
    assert all(torch.equal(p, r) for p, r in zip(grads, again)), "not reproducible"


@each_type
@pytest.mark.parametrize("b,n,c,groups", [(3, 5, 4096, 1), (2, 1, 8200, 2), (1, 40, 2056, 1), (2, 9, 1031, 1), (4, 3, 514, 1), (2, 33, 3 * 2072, 3), (2100, 1, 1040, 1), (7, 1, 4 * 519, 4), (5, 1, 8192, 2),
                                        (3, 1, 516, 1)])
def test_group_norm_wide_groups(cuda_device, dtype, b, n, c, groups):
    """groups wider than a workgroup (a last part that is narrower; single elements and chunks), a sample that is short or empty"""
    x, dy = (_randn(b, n, c, dtype=dtype, seed=s, mean=0.2).requires_grad_(s == 21) for s in (21, 22))
    w, o = (_randn(c, dtype=dtype, seed=s).requires_grad_(True) for s in (23, 24))
    lengths = [max(n - 2 * i, 0) for i in range(b)] if n > 1 else [i % 3 != 1 for i in range(b)]
    want = SR.group_norm(x, groups, w, o, 1e-5, "gelu", lengths, dy)
    y = HF.group_norm(x, groups, w, o, activation="gelu", lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    _within(y, want["y"], "y")
    for g, name in zip(torch.autograd.grad(y, (x, w, o), dy), ("dx", "dweight", "dbias")):
        _within(g, want[name], name)


def test_group_norm_many_rows(cuda_device):
    """more rows than 2^20: every row as in a small call"""
    x = _randn(1 << 12, 64, dtype=torch.bfloat16, seed=25)
    w, o = _randn(64, dtype=torch.float32, seed=26), _randn(64, dtype=torch.float32, seed=27)
    y = HF.group_norm(x, 4, w, o, activation="silu")
    many = HF.group_norm(x.repeat(300, 1), 4, w, o, activation="silu")
    assert torch.equal(many, y.repeat(300, 1))
    wide = HF.group_norm(x.view(64, 4096).repeat(33000, 1)[:, :1040], 1)
    assert torch.equal(wide, HF.group_norm(x.view(64, 4096)[:, :1040], 1).repeat(33000, 1))


def test_group_norm_forms(cuda_device):
    """without parameters, fp32 parameters on 16-bit rows, strided rows, images, single rows, garbage behind the lengths, a large mean"""
    x = _randn(2, 30, 64, dtype=torch.bfloat16, seed=41)
    _within(HF.group_norm(x, 4), SR.group_norm(x, 4, None, None, 1e-5, None, None)["y"], "plain")
    w, o = _randn(64, dtype=torch.float32, seed=42).requires_grad_(True), _randn(64, dtype=torch.float32, seed=43).requires_grad_(True)
    leaf = x.clone().requires_grad_(True)
    y = HF.group_norm(leaf, 4, w, o, activation="silu")
    dy = _randn(2, 30, 64, dtype=torch.bfloat16, seed=44)
    want = SR.group_norm(x, 4, w, o, 1e-5, "silu", None, dy)
    _within(y, want["y"], "y")
    for g, name in zip(torch.autograd.grad(y, (leaf, w, o), dy), ("dx", "dweight", "dbias")):
        _within(g, want[name], name)
    wide = torch.zeros(2, 30, 100, dtype=torch.bfloat16, device="cuda")
    for at in (0, 8, 3):
        wide[..., at:at + 64] = x
        assert torch.equal(HF.group_norm(wide[..., at:at + 64], 4, w, o, activation="silu"), y)
    assert torch.equal(HF.group_norm(x.transpose(1, 2).contiguous().transpose(1, 2), 4, w, o, activation="silu"), y)
    assert torch.equal(HF.group_norm(x.view(2, 5, 6, 64), 4, w, o, activation="silu").view(2, 30, 64), y)
    rows = HF.group_norm(x.view(60, 64), 4, w, o)
    _within(rows.view(60, 1, 64), SR.group_norm(x.view(60, 1, 64), 4, w, o, 1e-5, None, None)["y"], "rows")
    lens = torch.tensor([30, 12], dtype=torch.int32, device="cuda")
    dirty = x.clone()
    dirty[1, 12:] = float("nan")
    clean = HF.group_norm(x, 4, w, o, lengths=lens)
    assert torch.equal(HF.group_norm(dirty, 4, w, o, lengths=lens), clean) and not clean[1, 12:].any()
    leaf = dirty.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(HF.group_norm(leaf, 4, w, o, lengths=lens), leaf, torch.where(dirty.isnan(), dirty, dy))
    assert torch.isfinite(dx).all() and not dx[1, 12:].any()
    far = _randn(2, 300, 32, dtype=torch.float32, seed=45, mean=1000.0)
    _within(HF.group_norm(far, 2), SR.group_norm(far, 2, None, None, 1e-5, None, None)["y"], "large mean")
    assert HF.group_norm(x[:0], 4, w, o).shape == (0, 30, 64) and HF.group_norm(x[:, :0], 4).shape == (2, 0, 64)


# ---- as a program uses them ---------------------------------------------------------------------------------------------------
def _block(q, k, v, lam, w, o, rope, lens):
    q, k = rope(q, k)
    y = HF.differential_attention(q, k, v, lam, lens, "start")
    return HF.group_norm(y.flatten(2), y.shape[2], w, o, activation="silu", lengths=lens)


def _block_inputs(dtype=torch.bfloat16):
    q, k, v, lam = _attention_inputs(dtype, 3, 83, 83, 4, 2, 32, 64)
    leaves = [q, k, v, lam, _randn(256, dtype=dtype, seed=51, mean=1.0, std=0.1), _randn(256, dtype=dtype, seed=52, std=0.1)]
    return [t.requires_grad_(True) for t in leaves], torch.tensor([83, 40, 0], dtype=torch.int32, device="cuda")


def test_block_gradients_against_differences(cuda_device):
    """the three operators in a row: the directional derivative of a weighted sum, in fp32, against central differences in 64 bits of the
    plain forms (a step of 1e-4: a truncation error of about 1e-8 of the third derivative, far below the 1e-3 asked)"""
    leaves, lens = _block_inputs(torch.float32)
    rope = HN.RotaryEmbedding(32)
    dy = _randn(3, 83, 256, dtype=torch.float32, seed=53)
    grads = torch.autograd.grad(_block(*leaves, rope, lens), leaves, dy)
    dirs = [torch.randn(t.shape, generator=torch.Generator().manual_seed(60 + i)).double() for i, t in enumerate(leaves)]

    def plain(step):
        q, k, v, lam, w, o = (t.detach().cpu().double() + step * d for t, d in zip(leaves, dirs))
        q = SR.rotary(q, rope.freq, None, "half", 1.0)[0]
        k = SR.rotary(k, rope.freq, None, "half", 1.0)[0]
        y = SR.differential_attention(q, k, v, lam, lens.tolist(), "start", 32 ** -0.5)["o"][0].flatten(2)
        return (SR.group_norm(y, 4, w, o, 1e-5, "silu", lens.tolist())["y"][0] * dy.cpu().double()).sum()

    want = float((plain(1e-4) - plain(-1e-4)) / 2e-4)
    got = float(sum((g.cpu().double() * d).sum() for g, d in zip(grads, dirs)))
    assert abs(got - want) <= 1e-3 * abs(want)


def test_block_on_another_stream(cuda_device):
    leaves, lens = _block_inputs()
    rope = HN.RotaryEmbedding(32)
    dy = _randn(3, 83, 256, dtype=torch.bfloat16, seed=53)
    base = _block(*leaves, rope, lens)
    base = (base,) + torch.autograd.grad(base, leaves, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = _block(*leaves, rope, lens)
        got = (out,) + torch.autograd.grad(out, leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(base, got))


def test_block_in_captured_graphs(cuda_device):
    """forward and backward captured twice (two graphs, their own workspaces), replayed in turn with new inputs and eager work between: every
    replay equals the eager result"""
    rope = HN.RotaryEmbedding(32)
    leaves, lens = _block_inputs()
    dy = _randn(3, 83, 256, dtype=torch.bfloat16, seed=53)
    cache_q, cache_k, cache_v, lam = _attention_inputs(torch.bfloat16, 2, 1, 600, 4, 2, 32, 64)      # split keys: a workspace
    cache_len = torch.tensor([600, 77], dtype=torch.int32, device="cuda")

    def step():
        out = _block(*leaves, rope, lens)
        grads = torch.autograd.grad(out, leaves, dy)
        with torch.no_grad():
            token = HF.differential_attention(cache_q, cache_k, cache_v, lam, cache_len, "end")
        return (out, *grads, token)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = step()
        graphs.append((g, held))
    for turn in range(3):
        with torch.no_grad():
            for t in leaves + [cache_q, cache_k]:
                t.mul_(0.9).add_(0.01 * (turn + 1))
            cache_len.fill_(100 * turn + 1)
            lens.copy_(torch.tensor([83 - turn, 40 + turn, turn], dtype=torch.int32))
        want = [t.clone() for t in step()]
        for g, held in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(want, held))


def test_capture_beside_a_living_eager_graph_is_refused(cuda_device):
    """an eager graph of the same leaves on another stream: the capture is refused with an error before anything is recorded, and works once the
    eager outputs are gone"""
    q, k, v, lam = (t.requires_grad_(True) for t in _attention_inputs(torch.bfloat16, 1, 40, 40, 2, 2, 16, 32))
    x, w, o = (_randn(*s, dtype=torch.float32, seed=i).requires_grad_(True) for i, s in enumerate([(3, 8), (8,), (8,)]))
    freq = HN.RotaryEmbedding(16).freq
    calls = [lambda: HF.differential_attention(q, k, v, lam), lambda: HF.group_norm(x, 2, w, o), lambda: HF.rotary(q, k, freq)[1]]
    eager = [f() for f in calls]
    torch.cuda.synchronize()
    for f in calls:
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                f()
    want = [e.detach().clone() for e in eager]
    del eager
    for f, value in zip(calls, want):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = f()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, value)


def test_token_equals_the_last_row_of_the_prompt(cuda_device):
    """serving: the new token over the cache against the same position of the whole causal pass (another kernel and summation order)"""
    for dtype in TYPES:
        q, k, v, lam = _attention_inputs(dtype, 2, 300, 300, 4, 2, 64, 128)
        whole = SR.differential_attention(q, k, v, lam, None, "start", 64 ** -0.5)["o"]
        token = HF.differential_attention(q[:, -1:], k, v, lam, None, "end")
        _within(token, (whole[0][:, -1:], whole[1][:, -1:]), "token")
        _within(HF.differential_attention(q, k, v, lam, None, "start"), whole, "prompt")


def _plain_block(m, x, positions, lengths, causal):
    """models.layers.DifferentialAttention in float64 on the CPU, from elementary operations"""
    p = {k: v.detach().cpu().double().requires_grad_(True) for k, v in m.named_parameters()}
    x = x.detach().cpu().double().requires_grad_(True)
    b, n, _ = x.shape
    h, hk, d = m.n_head, m.kv_heads, m.head_dim
    lin = lambda name, t: t @ p[name + ".weight"].t() + p[name + ".bias"]
    q, k, v = lin("w_q", x).view(b, n, 2 * h, d), lin("w_k", x).view(b, n, 2 * hk, d), lin("w_v", x).view(b, n, hk, 2 * d)
    if m.rotary is not None:
        t = positions.cpu().double().expand(b, n)[:, :, None, None] * m.rotary.freq
        half = m.rotary.freq.numel()
        turn = lambda z: torch.cat([z[..., :half] * t.cos() - z[..., half:2 * half] * t.sin(), z[..., :half] * t.sin() + z[..., half:2 * half] * t.cos(),
                                    z[..., 2 * half:]], dim=-1)
        q, k = turn(q), turn(k)
    lam = (p["lambda_q1"] * p["lambda_k1"]).sum(1).exp() - (p["lambda_q2"] * p["lambda_k2"]).sum(1).exp() + m.lambda_init
    at, length = torch.arange(n), torch.full((b,), n) if lengths is None else lengths.cpu().long()
    seen = (at < length[:, None, None]).expand(b, n, n)
    if causal is not None:
        seen = seen & (at[None, None, :] <= at[None, :, None] + ((length - n)[:, None, None] if causal == "end" else 0))
    maps = []
    for j in range(2):
        s = torch.einsum("bihd,bjhd->bhij", q[:, :, j::2], k[:, :, j::2].repeat_interleave(h // hk, dim=2)) / d ** 0.5
        s = s.masked_fill(~seen[:, None], -1e300)
        maps.append(torch.softmax(s, -1).masked_fill(~seen[:, None], 0.0))
    y = torch.einsum("bhij,bjhd->bihd", maps[0] - lam[:, None, None] * maps[1], v.repeat_interleave(h // hk, dim=2))
    y = (y - y.mean(-1, keepdim=True)) / torch.sqrt(y.var(-1, correction=0, keepdim=True) + m.norm.eps)
    y = lin("w_concat", y.reshape(b, n, -1) * p["norm.weight"] + p["norm.bias"])
    return y.masked_fill((at >= length[:, None])[:, :, None], 0.0), x, p


@pytest.mark.parametrize("heads,kv,dims,causal,ragged", [(1, 1, 0, None, True), (4, 2, 8, "start", False), (2, 1, 16, "end", True)])
def test_differential_attention_module(cuda_device, heads, kv, dims, causal, ragged):
    """the whole block in fp32, values and every gradient against float64: relative to each tensor's largest entry within 2e-4 (a chain of three
    products of up to 64 terms, a softmax and a norm whose rstd of up to ~10 multiplies all of their errors: 10 * 3 * (64 + 72) * 2^-24 = 2.4e-4
    if every rounding had its worst sign)"""
    from immunostruct_amd.models.layers import DifferentialAttention
    torch.manual_seed(5)
    rope = HN.RotaryEmbedding(dims) if dims else None
    m = DifferentialAttention(64, heads, kv_heads=kv, input_dim=20, rotary=rope).cuda()
    with torch.no_grad():
        m.norm.bias.normal_()
    x = _randn(3, 83, 20, dtype=torch.float32, seed=71).requires_grad_(True)
    pos = torch.arange(83, device="cuda") + 5
    lens = torch.tensor([83, 40, 11], dtype=torch.int32, device="cuda") if ragged else None
    want, xd, p = _plain_block(m, x, pos, lens, causal)
    got = m(x, pos, lens, causal)
    dy = torch.randn(want.shape, generator=torch.Generator().manual_seed(9))
    want.backward(dy.double())
    got.backward(dy.cuda())

    def close(a, b, what, top=None):
        top = float(b.detach().abs().max()) if top is None else top
        off = float((a.detach().cpu().double() - b.detach()).abs().max())
        assert off <= 2e-4 * top, f"{what}: {off / top:.2e}"

    close(got, want, "out")
    close(x.grad, xd.grad, "dx")
    for name, par in m.named_parameters():
        # a bias' gradient is a sum of the terms its layer's weight gradient multiplies with x (of order 1): that is what its rounding is relative
        # to (w_k.bias without positions: it adds the same to a row's scores, the terms cancel and the gradient is 0)
        weight = p[name.replace("bias", "weight")]
        close(par.grad, p[name].grad, name, float(max(weight.grad.abs().max(), p[name].grad.abs().max())))
    if causal is None:
        mean = m.pooled_mean(x, pos, lens)
        n = torch.tensor([83.0, 40.0, 11.0]) if ragged else torch.full((3,), 83.0)
        close(mean, want.sum(1) / n[:, None].double(), "mean")


def test_module_token_by_token(cuda_device):
    """serving: projecting one position at a time into a cache and attending over it gives the whole causal pass"""
    from immunostruct_amd.models.layers import DifferentialAttention
    torch.manual_seed(6)
    m = DifferentialAttention(64, 4, kv_heads=2, rotary=HN.RotaryEmbedding(8)).cuda().to(torch.bfloat16)
    x = _randn(2, 9, 64, dtype=torch.bfloat16, seed=72)
    with torch.no_grad():
        whole = m(x, torch.arange(9, device="cuda"), None, "start")
        k, v = torch.full((2, 16, 4, 8), float("nan"), dtype=torch.bfloat16, device="cuda"), torch.full((2, 16, 2, 16), float("nan"), dtype=torch.bfloat16, device="cuda")
        for t in range(9):
            q, kt, vt = m.project(x[:, t:t + 1], torch.tensor([t], device="cuda"))
            k[:, t:t + 1], v[:, t:t + 1] = kt, vt
            one = m.attend_cached(q, k, v, torch.full((2,), t + 1, dtype=torch.int32, device="cuda"), "end")
            # two summation orders ahead of roundings to bf16 (2^-8 each) of the block's steps: attention, norm (whose rstd of up to ~10
            # multiplies the attention's), projection
            assert float((one[:, 0] - whole[:, t]).abs().max()) <= 12 * 2.0 ** -8 * float(whole.abs().max())
