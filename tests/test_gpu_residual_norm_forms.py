"""``cuda_funcs.residual_norm`` in every width of a row's team and number of pieces per lane, whole and with a tail, for the forms that have
kernels of their own without a layer norm or a bias; tolerances as in test_gpu_residual_norm.

Widths: teams of 8, 16, 32 and 64 lanes (to 256 channels in float32, 512 in 16 bits), a workgroup per row with one piece per
lane (to 4096 and 8192), with two (to 8192, 16384) and with four (to 16384, float32)."""
import pytest
import torch

from test_gpu_residual_norm import BF16, F16, F32, _compare

pytestmark = pytest.mark.gpu
DIMS = [5, 32, 60, 64, 100, 128, 256, 300, 512, 1001, 1024, 4096, 5000, 8192, 8200, 12345, 16384]


def _shape(dim):
    return (6, 50, dim) if dim <= 512 else (3, 7, dim)         # several strips of rows, some of them across an end of a gate's rows


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim", DIMS)
def test_root_mean_squares_on_both_sides(dim, dtype):
    shape = _shape(dim)
    for k, gate in enumerate((None, (dim,), (shape[0], 1, dim), shape)):
        _compare(shape, dtype, F32 if k % 2 else dtype, "rms", "rms", gate, keep=k != 1, scales=(1.0, 1.0) if k < 2 else (0.9, 0.22), seed=k)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim", DIMS)
def test_a_root_mean_square_alone(dim, dtype):
    shape = _shape(dim)
    for k, gate in enumerate((None, (dim,), (shape[0], 1, dim), shape)):
        _compare(shape, dtype, dtype if k % 2 else F32, "rms", None, gate, keep=k != 2, scales=(1.0, 1.0) if k < 2 else (0.9, 0.22), seed=k)
    _compare(shape, dtype, norm="rms", block=False, keep=dim % 2 == 0)
    _compare(shape, dtype, norm=None, block_norm="rms")
