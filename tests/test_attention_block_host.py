"""The attention block's host side without a GPU: what asks for a derivative, what the package needs to be imported, what an
export holds, sizes of workspaces."""
import pytest
import torch


@pytest.fixture(scope="module")
def DB():
    import ppl.pmx_b200.torch_function as F
    return F.dynamic_batching


def test_gradients_and_tangents_are_noticed(DB):
    import torch.autograd.forward_ad as fw
    from ppl.pmx_b200.torch_function.dynamic_batching._common import wants_grad
    x = torch.ones(3)
    assert not wants_grad(x, None) and wants_grad(None, x.clone().requires_grad_())
    with torch.no_grad():
        assert not wants_grad(x.clone().requires_grad_())
    with fw.dual_level():
        dual = fw.make_dual(x, x)
        assert wants_grad(x, dual) and not wants_grad(x)
        with torch.no_grad():
            assert wants_grad(dual)
    assert not wants_grad(dual)
