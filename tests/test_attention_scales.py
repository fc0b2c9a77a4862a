"""Scales of an attention's scores whose logarithm's base, or one over them for the biases, float32 does not hold: refused on the host."""
import ctypes

import pytest
import torch

from crystalframer_amd import _lib
from test_sequence_attention_refusals import A, TABLE, _args


@pytest.mark.parametrize("change", [dict(scale=2.4e38), dict(scale=3.4e38), dict(TABLE, scale=2.0 ** 65), dict(TABLE, scale=1e38)])
def test_library(change):
    lib, a = _lib.load(), _args(**change)
    assert lib.cfh_attention_forward(ctypes.byref(a), A, None, None, A, 1 << 30, None) < 0 and b"scale" in lib.cfh_last_error()
    assert lib.cfh_attention_forward_workspace_bytes(ctypes.byref(a)) == 0
    assert lib.cfh_attention_backward_workspace_bytes(ctypes.byref(a)) == 0


@pytest.mark.gpu
def test_calls():
    from crystalframer_amd import cuda_funcs
    x = torch.randn(1, 5, 2, 16, device="cuda")
    for scale in (2.4e38, 3.4e38, 1e39):
        with pytest.raises(ValueError, match="scale"):
            cuda_funcs.cross_attention(x, x, x, scale=scale)
    of, table = cuda_funcs.position_buckets(8, 20, device="cuda"), torch.zeros(8, 2, device="cuda")
    for scale in (2.0 ** -65, 2.0 ** 65):
        with pytest.raises(ValueError, match="scale"):
            cuda_funcs.relative_attention(x, x, x, table, of, scale=scale)
    # powers of two change no other bit, up to the largest with a table
    table = torch.randn(8, 2, device="cuda")
    for scale in (2.0 ** -64, 2.0 ** 64):
        y = x * scale ** -0.5
        assert torch.equal(cuda_funcs.cross_attention(y, y, x, scale=scale), cuda_funcs.cross_attention(x, x, x, scale=1.0))
        assert torch.equal(cuda_funcs.relative_attention(y, y, x, table, of, scale=scale), cuda_funcs.relative_attention(x, x, x, table, of, scale=1.0))
