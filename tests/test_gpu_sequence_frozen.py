"""Inputs without gradients: what is asked for equals the full backward pass bit for bit, and nothing else is computed."""
import ctypes
import itertools

import pytest
import torch

from immunostruct_amd import _lib, functional as HF

pytestmark = pytest.mark.gpu


@pytest.fixture
def backward_calls(cuda_device):
    """the argument structures that reach the backward entry points, between the C++ functions and the library"""
    ops, lib, calls = _lib.torch_ops(), _lib.load(), []
    names = ["is_last_error_string"] + [n for n in _lib.SIGNATURES if n.startswith(("is_rotary", "is_diff_attention", "is_group_norm"))]
    real = {n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names}
    kinds = {"is_diff_attention_bwd": _lib.DiffAttention, "is_group_norm_bwd": _lib.GroupNorm}
    proto = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p)

    def listen(name):
        def call(args, stream):
            calls.append(kinds[name].from_buffer_copy(ctypes.string_at(args, ctypes.sizeof(kinds[name]))))
            return proto(real[name])(args, stream)
        return proto(call)

    heard = {n: listen(n) for n in kinds}
    ops.bind({**real, **{n: ctypes.cast(f, ctypes.c_void_p).value for n, f in heard.items()}}, _lib.HipExtensionError)
    yield calls
    ops.bind(real, _lib.HipExtensionError)


def _subsets(n):
    return [s for s in itertools.product((False, True), repeat=n) if any(s)]


def _check(call, inputs, asked, dy):
    leaves = [t.clone().requires_grad_(True) for t in inputs]
    full = torch.autograd.grad(call(*leaves), leaves, dy)
    some = [t.clone().requires_grad_(a) for t, a in zip(inputs, asked)]
    got = torch.autograd.grad(call(*some), [t for t in some if t.requires_grad], dy)
    assert all(torch.equal(x, y) for x, y in zip(got, [f for f, a in zip(full, asked) if a]))


@pytest.mark.parametrize("asked", _subsets(4), ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
def test_attention(backward_calls, asked, dtype):
    gen = torch.Generator().manual_seed(1)
    make = lambda *s: torch.randn(*s, generator=gen).to(dtype).cuda()
    for nq, nk in ((40, 70), (600, 130)):      # (one and several row splits)
        inputs = [make(2, nq, 4, 32), make(2, nk, 2, 32), make(2, nk, 1, 64), make(2)]
        _check(lambda q, k, v, lam: HF.differential_attention(q, k, v, lam, causal="end"), inputs, asked, make(2, nq, 2, 64))
        args = backward_calls[-1]
        assert bool(args.dk) == bool(args.dv_out) == (asked[1] or asked[2])
        assert bool(args.dq) == (asked[0] or asked[3]) and bool(args.dlam) == asked[3]


@pytest.mark.parametrize("asked", _subsets(3), ids=str)
@pytest.mark.parametrize("b,n,c,groups", [(50, 1, 64, 4), (50, 1, 60, 4), (9, 1, 1040, 1), (7, 30, 64, 4), (2, 3000, 64, 2), (3, 2, 4112, 1)])
def test_group_norm(backward_calls, asked, b, n, c, groups):
    gen = torch.Generator().manual_seed(2)
    make = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).cuda()
    lens = torch.full((b,), n, dtype=torch.int32, device="cuda")
    lens[-1] = n // 2
    _check(lambda x, w, o: HF.group_norm(x, groups, w, o, activation="silu", lengths=lens), [make(b, n, c), make(c), make(c)], asked, make(b, n, c))
    args = backward_calls[-1]
    assert bool(args.dx) == asked[0] and bool(args.dweight) == bool(args.dbias) == (asked[1] or asked[2])


def test_rotary(cuda_device):
    """the turned half of a frozen input is a constant: what follows it owes it no gradient"""
    freq = torch.tensor([1.0, 0.1], dtype=torch.float64)
    q, k = torch.randn(2, 5, 3, 4, device="cuda"), torch.randn(2, 5, 1, 4, device="cuda")
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    full = torch.autograd.grad(HF.rotary(q.requires_grad_(True), k.requires_grad_(True), freq), (q, k), (dq, dk))
    only_q, only_k = HF.rotary(q, k.detach(), freq), HF.rotary(q.detach(), k, freq)
    assert only_q[0].requires_grad and not only_q[1].requires_grad and only_k[1].requires_grad and not only_k[0].requires_grad
    assert torch.equal(torch.autograd.grad(only_q[0], q, dq)[0], full[0]) and torch.equal(torch.autograd.grad(only_k[1], k, dk)[0], full[1])
    both = HF.rotary(q, k, freq)
    assert torch.equal(torch.autograd.grad(both, k, (dq, dk))[0], full[1])      # (one of two asked for)
