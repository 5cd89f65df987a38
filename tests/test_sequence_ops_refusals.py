"""What the sequence operators refuse, and what their frequencies are (no GPU: the checks come before the device)."""
import ctypes
import math

import pytest
import torch

from immunostruct_amd import _lib, functional as HF
from immunostruct_amd.nn import GroupNorm, RotaryEmbedding

Z = torch.zeros


def _diff(q=(2, 3, 4, 8), k=(2, 5, 2, 8), v=(2, 5, 1, 16), lam=(2,), types=(torch.float32,) * 4, **kw):
    return HF.differential_attention(*(Z(*s, dtype=t) for s, t in zip((q, k, v, lam), types)), **kw)


@pytest.mark.parametrize("kw", [
    dict(q=(2, 3, 3, 8)), dict(q=(2, 3, 4, 7)), dict(k=(2, 4, 2, 8)), dict(k=(1, 5, 2, 8)), dict(v=(2, 5, 2, 16)), dict(lam=(3,)), dict(lam=(2, 1)),
    dict(q=(3, 4, 8)), dict(q=(2, 3, 0, 8), lam=(0,)), dict(types=(torch.float32, torch.bfloat16, torch.float32, torch.float32)),
    dict(types=(torch.float64,) * 4), dict(types=(torch.float32,) * 3 + (torch.bfloat16,)), dict(causal=True), dict(causal="middle"),
    dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(lengths=Z(3, dtype=torch.int32)),
    dict(lengths=Z(2, dtype=torch.int64)), dict(lengths=Z(2, 1, dtype=torch.int32))])
def test_attention_refuses(kw):
    with pytest.raises(ValueError):
        _diff(**kw)


def test_attention_limits_and_device():
    with pytest.raises(NotImplementedError):
        _diff(q=(2, 3, 4, 65), k=(2, 5, 2, 65))
    with pytest.raises(NotImplementedError):
        _diff(v=(2, 5, 1, 257), types=(torch.bfloat16,) * 4)
    with pytest.raises(_lib.HipExtensionError):
        _diff()


@pytest.mark.parametrize("kw", [
    dict(q=(2, 3, 8)), dict(k=(2, 4, 1, 8)), dict(k=(2, 3, 1, 6)), dict(freq=Z(5).double()), dict(freq=Z(4)), dict(freq=Z(0).double()),
    dict(freq=Z(2, 2).double()), dict(layout="quarter"), dict(positions=Z(3)), dict(positions=Z(4, dtype=torch.int64)),
    dict(positions=Z(3, 2, dtype=torch.int64)), dict(dtype=torch.float64), dict(q=(2, 3, 0, 8))])
def test_rotary_refuses(kw):
    kw = dict(dict(q=(2, 3, 4, 8), k=(2, 3, 1, 8), freq=Z(4).double(), layout="half", positions=None, dtype=torch.float32), **kw)
    with pytest.raises(ValueError):
        HF.rotary(Z(*kw["q"], dtype=kw["dtype"]), Z(*kw["k"], dtype=kw["dtype"]), kw["freq"], kw["positions"], kw["layout"])


def test_rotary_needs_the_device():
    with pytest.raises(_lib.HipExtensionError):
        HF.rotary(Z(2, 3, 4, 8), None, Z(4).double())


@pytest.mark.parametrize("kw", [
    dict(groups=3), dict(groups=0), dict(activation="tanh"), dict(bias=None), dict(weight=Z(4)), dict(weight=Z(8).double(), bias=Z(8).double()),
    dict(weight=Z(8).bfloat16()), dict(lengths=Z(3, dtype=torch.int32)), dict(lengths=Z(2, dtype=torch.int64)), dict(eps=-1.0), dict(eps=float("nan")),
    dict(x=Z(8)), dict(x=Z(2, 3, 4, 8), lengths=Z(2, dtype=torch.int32)), dict(x=Z(2, 3, 8).double()), dict(x=Z(2, 3, 0))])
def test_group_norm_refuses(kw):
    kw = dict(dict(x=Z(2, 3, 8), groups=2, weight=Z(8), bias=Z(8)), **kw)
    with pytest.raises(ValueError):
        HF.group_norm(**kw)


def test_group_norm_needs_the_device():
    with pytest.raises(_lib.HipExtensionError):
        GroupNorm(2, 8)(Z(2, 3, 8))


def test_entry_points_refuse_without_a_device():
    lib = _lib.load()
    assert lib.is_diff_attention_fwd(None, None) == -22 and lib.is_diff_attention_bwd(None, None) == -22
    assert lib.is_group_norm_fwd(None, None) == -22 and lib.is_group_norm_bwd(None, None) == -22
    p = 4096      # (never dereferenced: every call below is refused)
    good = dict(q=p, k=p, v=p, lam=p, o=p, batch=1, nq=1, nk=1, heads=2, kv_heads=1, d=8, dv=8, causal=0, type=0, lam_type=0, splits=1, row_splits=1, scale=1.0)
    for change, code in ((dict(q=None), -22), (dict(batch=0), -22), (dict(kv_heads=3), -22), (dict(type=3), -22), (dict(lam_type=1), -22),
                         (dict(causal=3), -22), (dict(scale=0.0), -22), (dict(splits=0), -22), (dict(splits=2), -22), (dict(lse=p), -22),
                         (dict(d=65), -38), (dict(dv=129), -38), (dict(type=1, lam_type=1, d=129), -38), (dict(nq=2 ** 31 - 1), -22),
                         (dict(batch=2 ** 31 - 1, kv_heads=2), -22),
                         (dict(k_n=2 ** 24), -22), (dict(q_n=-1), -22)):
        assert lib.is_diff_attention_fwd(ctypes.byref(_lib.DiffAttention(**dict(good, **change))), None) == code, change
    assert lib.is_diff_attention_bwd(ctypes.byref(_lib.DiffAttention(**good)), None) == -22      # nothing saved
    norm = dict(x=p, y=p, stats=p, batch=1, n=1, channels=8, groups=2, eps=1e-5)
    for change in (dict(x=None), dict(stats=None), dict(y=None), dict(groups=3), dict(batch=0), dict(activation=4), dict(weight=p), dict(weight=p, bias=p, weight_type=1),
                   dict(type=5), dict(eps=-1.0)):
        assert lib.is_group_norm_fwd(ctypes.byref(_lib.GroupNorm(**dict(norm, **change))), None) == -22, change
    assert lib.is_group_norm_bwd(ctypes.byref(_lib.GroupNorm(**norm)), None) == -22
    freq = (ctypes.c_double * 4)(1, 1, 1, 1)
    args = [p, 8, 8, 8, p, 1, None, 0, 0, 0, None, 0, None, 0, 0, 0, ctypes.addressof(freq), 1, 1, 8, 8, 0, 0, 1.0, 0, None]
    for at, value in ((0, None), (4, None), (5, 0), (11, 1), (16, None), (17, 0), (18, 0), (20, 7), (20, 10), (20, 0), (24, 3)):
        assert lib.is_rotary(*[value if i == at else a for i, a in enumerate(args)]) == -22, at


def test_splits_cover_the_chip():
    lib = _lib.load()
    assert lib.is_diff_attention_splits(16, 4, 4, 16384, 1) == 16      # single tokens: 64 workgroups alone
    assert lib.is_diff_attention_splits(128, 1, 190, 190, 0) == 1 and lib.is_diff_attention_splits(2, 4, 16384, 4096, 1) == 1
    assert lib.is_diff_attention_splits(1, 1, 1, 100, 2) == 1 and lib.is_diff_attention_splits(1, 1, 1, 2 ** 20, 0) == 64
    assert lib.is_diff_attention_splits(1, 1, 256, 2048, 1) == 4 and lib.is_diff_attention_splits(1, 1, 256, 2048, 0) == 16
    assert lib.is_diff_attention_work_floats(16, 4, 4, 128, 1) == 0
    assert lib.is_diff_attention_work_floats(16, 4, 4, 128, 16) == 2 * 16 * 4 * 16 * 4 * 130
    assert lib.is_diff_attention_row_splits(2, 4, 16384, 4096, 1) == 2 and lib.is_diff_attention_row_splits(2, 4, 16384, 4096, 0) == 1
    assert lib.is_diff_attention_row_splits(1, 1, 4096, 128, 0) == 16 and lib.is_diff_attention_row_splits(1, 1, 100, 128, 1) == 1
    assert lib.is_diff_attention_row_work_floats(2, 4, 100, 64, 128, 2) == 2 * 2 * 4 * 100 * 256


def test_rotary_frequencies():
    f = RotaryEmbedding(8).freq
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14, atol=0)
    assert torch.equal(RotaryEmbedding(8, scaling=dict(kind="linear", factor=4)).freq, f / 4)
    ntk = RotaryEmbedding(8, scaling=dict(kind="ntk", factor=4)).freq
    assert ntk[0] == 1.0 and math.isclose(float(ntk[3]), 0.001 / 4, rel_tol=1e-12)      # the slowest pair is stretched by the factor
    yarn = RotaryEmbedding(64, scaling=dict(kind="yarn", factor=4, original_length=4096))
    plain = RotaryEmbedding(64).freq
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(yarn.freq[turns > 64], plain[turns > 64]) and torch.allclose(yarn.freq[turns < 0.5], plain[turns < 0.5] / 4, rtol=1e-14, atol=0)
    assert math.isclose(yarn.amplitude, 0.1 * math.log(4) + 1)
    assert RotaryEmbedding(8).state_dict() == {}
    for kw in (dict(dims=7), dict(dims=0), dict(dims=514), dict(dims=8, layout="x"), dict(dims=8, base=1.0), dict(dims=8, scaling=dict(kind="x")),
               dict(dims=8, scaling=dict(factor=2)), dict(dims=8, scaling=dict(kind="linear", factor=0.5)), dict(dims=8, scaling=dict(kind="linear", factor=2, foo=1)),
               dict(dims=2, scaling=dict(kind="ntk", factor=2)), dict(dims=8, scaling=dict(kind="yarn", factor=2, original_length=0))):
        with pytest.raises(ValueError):
            RotaryEmbedding(**kw)


def test_group_norm_module_refuses():
    with pytest.raises(ValueError):
        GroupNorm(3, 8)
    assert [tuple(p.shape) for p in GroupNorm(2, 8).parameters()] == [(8,), (8,)] and not list(GroupNorm(2, 8, affine=False).parameters())


def test_autograd_functions_load_and_raise_the_package_error():
    """the C++ side loads against this torch and is bound to the library; host tensors never reach it through the package"""
    ops = _lib.torch_ops()
    assert ops is _lib.torch_ops() and all(callable(getattr(ops, n)) for n in ("rotary", "differential_attention", "group_norm"))
