"""norm_rope, token_logprobs and dropout on the GPU: the calls at the edges of what they take, through the
functions on tensors of twg_capi and behind device="webgpu", against the float64 definitions of steps_ref.py."""
import math

import pytest
import torch

import steps_ref as ref
import twg_capi as capi

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def backend():
    import torch_webgpu  # noqa: F401
    capi.load()
    torch.webgpu.init()
    yield


def dev(t, grad=False):
    return None if t is None else t.to("webgpu").requires_grad_(grad)


def host(t):
    return t.detach().to("cpu")


def leave_nan_behind(dtype, n, device):
    """blocks of n elements that hold NaN when the allocator hands them out next"""
    blocks = [torch.full((n,), math.nan, dtype=dtype).to(device) for _ in range(8)]
    del blocks


# ---------------------------------------------------------------------- parts without heads

@pytest.mark.parametrize("device", ["webgpu", "cuda"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("q_heads, k_heads", [(0, 2), (3, 0), (0, 0)])
def test_a_weight_without_heads_has_a_gradient_of_zeros(device, dtype, q_heads, k_heads):
    g = torch.Generator().manual_seed(q_heads)
    q, k, dq, dk = (torch.randn(2, 5, h, 64, generator=g).to(dtype) for h in (q_heads, k_heads, q_heads, k_heads))
    w = (1 + 0.3 * torch.randn(2, 64, generator=g)).to(dtype)
    pos, inv_freq = torch.arange(5), torch.rand(32, generator=g)
    args = [t.to(device) for t in (dq, dk, q, k, pos, inv_freq, w[0], w[1])]
    leave_nan_behind(dtype, 64, device)
    grads = capi.norm_rope_backward(*args)
    for i, (x, dy) in enumerate(((q, dq), (k, dk))):
        assert grads[i].shape == x.shape
        _, _, dw, bound = ref.norm_rope_backward(dy, x, pos, inv_freq, w[i])
        ref.assert_within(host(grads[2 + i]), dw, bound, f"weight {i}")


@pytest.mark.parametrize("q_heads, k_heads", [(0, 2), (3, 0)])
def test_a_weight_without_heads_in_a_backward_pass(q_heads, k_heads):
    q, k = torch.randn(1, 4, q_heads, 32), torch.randn(1, 4, k_heads, 32)
    qd, kd, wq, wk = dev(q, True), dev(k, True), dev(torch.ones(32), True), dev(torch.ones(32), True)
    out = torch.ops.webgpu.norm_rope(qd, kd, dev(torch.arange(4)), dev(torch.rand(16)), wq, wk)
    leave_nan_behind(F32, 32, "webgpu")
    torch.autograd.backward(out, [dev(torch.ones(q.shape)), dev(torch.ones(k.shape))])
    for heads, w in ((q_heads, wq), (k_heads, wk)):
        grad = host(w.grad)
        assert bool(torch.isfinite(grad).all()) and bool((grad == 0).all()) == (heads == 0)
