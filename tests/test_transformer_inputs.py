"""Inputs that the operators behind the encoder stem must take as they mean, or refuse (no GPU needed)."""
import ctypes

import pytest

from mlx_audio_amd import _lib


@pytest.mark.parametrize("sizes", [(0, 5, 7), (1, 0, 7), (1, 5, 0), (0, 0, 0), (3, 1, 1), (2, 1500, 1500)])
def test_workspaces_of_attention_backward(sizes):
    """Sizes of zero too; float16 keeps its norms there beside what the other two-byte type keeps."""
    batch, queries, keys = sizes
    s = (ctypes.c_int64 * 3)(1, 1, 1)
    need = [_lib.lib().mia_attention_backward_workspace_bytes(ctypes.byref(
        _lib.AttentionDesc(t, batch, queries, keys, 4, 2, 16, 0, 0.25, s, s, s))) for t in (_lib.F16, _lib.BF16)]
    assert (need[0] > need[1]) == (batch > 0)
