"""norm_rope, token_logprobs and dropout at the edges of what they take, as far as that shows without a GPU:
calls that do nothing, calls on fake tensors (shapes, types and devices only), refusals."""
import pytest
import torch
import torch.nn.functional as F
from torch._subclasses.fake_tensor import FakeTensorMode


@pytest.fixture(autouse=True)
def backend():
    import torch_webgpu  # noqa: F401
    yield


# -------------------------------------------------------------------------------- dropout

@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
def test_dropout_that_drops_nothing_returns_its_input(inplace, grad):
    """in evaluation and for p = 0, whatever the input's type, also where it requires grad"""
    state = torch.webgpu.get_rng_state()
    with FakeTensorMode():
        for dtype in (torch.float32, torch.bfloat16, torch.float64):
            leaf = torch.empty(3, 4, device="webgpu", dtype=dtype, requires_grad=grad)
            for x in (leaf, leaf.view(12)):
                assert F.dropout(x, 0.5, training=False, inplace=inplace) is x
                assert F.dropout(x, 0.0, inplace=inplace) is x
                assert torch.nn.Dropout(0.5, inplace=inplace).eval()(x) is x
    assert torch.equal(torch.webgpu.get_rng_state(), state)
