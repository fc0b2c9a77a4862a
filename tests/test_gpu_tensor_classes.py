"""The encoder's layer norms with tensors of other classes: torch's module runs."""
import pytest
import torch

from test_tensor_classes import Overriding

pytestmark = pytest.mark.gpu


def test_a_class_that_overrides_torchs_functions_sees_the_norm():
    from crystalframer_amd import encoder
    norm = torch.nn.LayerNorm(32).cuda()
    x, block = torch.randn(5, 32, device="cuda"), torch.randn(5, 32, device="cuda")
    for a, b in ((x.as_subclass(Overriding), block), (x, block.as_subclass(Overriding))):
        del Overriding.calls[:]
        y = encoder._normed_sum(norm, a, b)
        assert type(y) is Overriding and torch.nn.functional.layer_norm in Overriding.calls
        assert torch.allclose(y.as_subclass(torch.Tensor), norm(x + block))
    del Overriding.calls[:]
    assert type(encoder._normed(norm, x.as_subclass(Overriding))) is Overriding and torch.nn.functional.layer_norm in Overriding.calls


def test_a_compiled_function_has_the_module_in_its_graph():
    from crystalframer_amd import encoder
    norm = torch.nn.LayerNorm(32).cuda()
    x, block = torch.randn(5, 32, device="cuda", requires_grad=True), torch.randn(5, 32, device="cuda")
    graphs = []

    def backend(graph, example):
        graphs.append(str(graph.code))
        return graph.forward
    whole = torch.compile(lambda a, b: encoder._normed_sum(norm, encoder._normed(norm, a), b), backend=backend, fullgraph=True)
    y = whole(x, block)
    assert len(graphs) == 1 and graphs[0].count("layer_norm(") == 2
    assert torch.allclose(y, norm(norm(x) + block))
