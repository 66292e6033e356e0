"""Sizes, types and arguments at the limits of the operators behind the encoder stem: what cannot be
served is refused in front of any device work (no GPU needed)."""
import ctypes

import pytest
import torch

from mlx_audio_amd import _lib, frontends as f
from mlx_audio_amd.frontends import transformer

P = ctypes.c_void_p(256)  # never followed: every call here ends in the checks


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
def test_key_lengths_of_every_integer_type(dtype):
    """Also where the number of keys does not fit the type."""
    got = transformer._check_lengths(torch.tensor([3, 0, 120], dtype=dtype), 3, 70000)
    assert got.dtype == torch.int32 and got.tolist() == [3, 0, 120]


@pytest.mark.parametrize("dtype", [torch.bool, torch.float32, torch.complex64, torch.complex128, torch.uint16, torch.uint64])
def test_key_lengths_that_are_no_integers_are_refused(dtype):
    q = torch.empty(2, 3, 4, 16)
    with pytest.raises(ValueError, match="key_lengths"):
        f.attention(q, q, q, key_lengths=torch.zeros(2).to(dtype))


def attention_desc(**kw):
    d = dict(dtype=0, batch=1, queries=2, keys=3, heads=4, kv_heads=2, dim=16, causal=0, scale=0.25)
    d.update(kw)
    s = (ctypes.c_int64 * 3)(1, 1, 1)
    return ctypes.byref(_lib.AttentionDesc(**d, stride_q=s, stride_k=s, stride_v=s))


def test_attention_refuses_more_workgroups_than_one_launch_holds():
    """A launch counts its threads in 32 bits: 2^24 workgroups of 256."""
    lib = _lib.lib()
    s = (ctypes.c_int64 * 3)(1, 1, 1)
    many = attention_desc(batch=1 << 24, queries=1)
    assert lib.mia_attention(many, P, P, P, None, P, None, None, 0, None) == _lib.MIA_ERR_UNSUPPORTED
    assert lib.mia_attention_backward(many, P, s, P, P, P, P, s, P, None, P, P, P, P, 1 << 40, None) == _lib.MIA_ERR_UNSUPPORTED
    # dk / dv alone is too large: refused before dq is enqueued
    keys = attention_desc(batch=1 << 20, queries=1, keys=4096, heads=1, kv_heads=1)
    assert lib.mia_attention_backward(keys, P, s, P, P, P, P, s, P, None, P, P, P, P, 1 << 62, None) == _lib.MIA_ERR_UNSUPPORTED


def test_attention_refuses_a_scale_that_overflows():
    """Exponents are taken to base 2: scale / ln 2 has to be finite as well."""
    lib = _lib.lib()
    assert lib.mia_attention(attention_desc(scale=3e38), P, P, P, None, P, None, None, 0, None) == _lib.MIA_ERR_INVALID
    assert lib.mia_attention(attention_desc(scale=3e38, batch=0), P, P, P, None, P, None, None, 0, None) == _lib.MIA_ERR_INVALID


def test_linear_refuses_more_workgroups_than_one_launch_holds():
    lib = _lib.lib()

    def linear(rows, k, n):
        return lib.mia_linear(P, k, P, k, None, 0, None, 0, 0, rows, k, n, 0, P, None, P, 1 << 62, None)

    wide = (1 << 26) + 1
    for rows, k, n in ((1, 8, wide), (1, wide, 8), (100, 8, wide)):
        assert linear(rows, k, n) == _lib.MIA_ERR_UNSUPPORTED
    # rows of seven elements go through registers: no kernel there that walks tiles
    assert linear((1 << 30) - 4096, 7, 1000) == _lib.MIA_ERR_UNSUPPORTED
    assert lib.mia_linear_backward(P, wide, P, 8, P, 8, None, 0, 0, 1, 8, wide, 0, P, P, P, P, 1 << 62,
                                   None) == _lib.MIA_ERR_UNSUPPORTED


def test_layer_norm_refuses_more_workgroups_than_one_launch_holds():
    lib = _lib.lib()
    wide = (1 << 25) + 1

    def forward(rows, dim):
        return lib.mia_layer_norm(P, rows, dim, dim, 0, None, None, 0, 1e-5, P, None, None, None)

    def backward(rows, dim):
        return lib.mia_layer_norm_backward(P, dim, P, dim, P, P, rows, dim, 0, P, 0, P, P, P, P, 1 << 62, None)

    for rows, dim in ((1, wide), (1 << 24, 8193)):
        assert forward(rows, dim) == _lib.MIA_ERR_INVALID
        assert backward(rows, dim) == _lib.MIA_ERR_INVALID


def test_layer_norm_backward_refuses_a_workspace_that_is_not_aligned():
    lib = _lib.lib()
    odd = ctypes.c_void_p(257)
    assert lib.mia_layer_norm_backward(P, 8, P, 8, P, P, 2, 8, 0, P, 0, P, P, P, odd, 1 << 20, None) == _lib.MIA_ERR_INVALID


def test_linear_serves_a_long_result_that_goes_through_registers():
    """2^23 tiles of one launch: planned, and refused here only for what else is wrong (no weight)."""
    lib = _lib.lib()
    assert lib.mia_linear_workspace_bytes((1 << 30) - 4096, 7, 1, 0) == 0  # one part of k
