"""Tensors whose class makes torch's operations itself, at the residual norms and the encoder's layer norms: looked at on the CPU, with
tensors that say they are on a device and have no memory."""
import pytest
import torch

from crystalframer_amd import encoder, norms


class Wrapped(torch.Tensor):
    @staticmethod
    def __new__(cls, *shape):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=torch.float32, device="cuda")

    @classmethod
    def __torch_dispatch__(cls, f, types, args=(), kwargs=None):
        raise AssertionError(f)


class WrappedQuietly(Wrapped):
    __torch_function__ = torch._C._disabled_torch_function_impl


class Overriding(torch.Tensor):
    calls = []

    @classmethod
    def __torch_function__(cls, f, types, args=(), kwargs=None):
        cls.calls.append(f)
        return super().__torch_function__(f, types, args, kwargs or {})


@pytest.mark.parametrize("kind", [Wrapped, WrappedQuietly])
def test_residual_norm_refuses_what_has_no_memory(kind):
    x, v = kind(4, 32), kind(32)
    for name, call in (("x", lambda: norms.residual_norm(x)), ("weight", lambda: norms.residual_norm(torch.zeros(4, 32), weight=v)),
                       ("bias", lambda: norms.residual_norm(torch.zeros(4, 32), bias=v)),
                       ("gate", lambda: norms.residual_norm(torch.zeros(4, 32), torch.zeros(4, 32), gate=v))):
        with pytest.raises(TypeError, match="^" + name + " is a tensor of a class"):
            call()


@pytest.mark.parametrize("kind", [Wrapped, WrappedQuietly])
def test_the_encoder_leaves_them_to_the_module(kind):
    norm = torch.nn.LayerNorm(32, elementwise_affine=False)
    assert not encoder._norm_is_plain(norm, kind(4, 32))
    assert not encoder._leave_it_to_torch(torch.zeros(3), None, kind(3))
    assert encoder._leave_it_to_torch(torch.zeros(3), None, torch.nn.Parameter(torch.zeros(3)))


def test_a_class_that_overrides_torchs_functions():
    assert not encoder._leave_it_to_torch(torch.zeros(3), torch.zeros(3).as_subclass(Overriding))
