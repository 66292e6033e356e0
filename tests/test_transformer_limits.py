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
