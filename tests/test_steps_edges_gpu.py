"""norm_rope, token_logprobs and dropout on the GPU: the calls at the edges of what they take, through the
functions on tensors of twg_capi and behind device="webgpu", against the float64 definitions of steps_ref.py."""
import math

import pytest
import torch
import torch.nn.functional as F

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


# ------------------------------------------------------------------------- dropout in place

def kept(n, p, seed, offset=0):
    """what dropout multiplies n elements by"""
    threshold = math.floor(p * 65536 + 0.5)
    return ref.keep_mask(n, p, seed, offset).double() * (65536 / (65536 - threshold))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_dropout_in_place_trains(dtype):
    torch.manual_seed(41)
    x, dy = torch.randn(30, 21).to(dtype), torch.randn(30, 21).to(dtype)
    xd = dev(x, True)
    y = torch.ops.webgpu.dropout(xd, 0.0, 0)  # a tensor with a history
    version, address = y._version, y.data_ptr()
    z = torch.nn.Dropout(0.4, inplace=True)(y)
    assert z is y and y.data_ptr() == address and y._version > version and y.grad_fn is not None
    ref.assert_within(host(y), *ref.dropout(x, 0.4, 41, 0))
    y.backward(dev(dy))
    ref.assert_within(host(xd.grad), *ref.dropout(dy, 0.4, 41, 0))


def test_dropout_in_place_on_a_view_of_a_tensor_with_a_history():
    torch.manual_seed(42)
    x, dy = torch.randn(6, 10), torch.randn(6, 10)
    xd = dev(x, True)
    y = xd * 1.0
    F.dropout(y[:, 2:7], 0.5, inplace=True)
    y.backward(dev(dy))
    times = torch.ones(6, 10, dtype=torch.float64)
    times[:, 2:7] = kept(30, 0.5, 42).view(6, 5)
    # products of a float32 with 0, 1 or 2
    assert torch.equal(host(y).double(), x.double() * times)
    assert torch.equal(host(xd.grad).double(), dy.double() * times)


def test_dropout_in_place_twice_and_second_derivatives():
    torch.manual_seed(43)
    x = torch.randn(64)
    xd = dev(x, True)
    y = xd * xd
    F.dropout(F.dropout(y, 0.5, inplace=True), 0.5, inplace=True)
    times = kept(64, 0.5, 43, 0) * kept(64, 0.5, 43, 1)
    (g,) = torch.autograd.grad(y, xd, dev(torch.ones(64)), create_graph=True)
    (gg,) = torch.autograd.grad(g, xd, dev(torch.ones(64)))
    assert torch.equal(host(g).double(), 2 * x.double() * times)
    assert torch.equal(host(gg).double(), 2 * times)


def test_dropout_in_place_is_seen_by_what_saved_the_tensor():
    xd = dev(torch.randn(20), True)
    y = xd * 1.0
    z = y * y  # saves y
    F.dropout(y, 0.5, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward(dev(torch.ones(20)))


def test_dropout_in_place_refuses_leaves_before_it_draws():
    x = torch.randn(4, 6)
    xd = dev(x, True)
    state = torch.webgpu.get_rng_state()
    for leaf in (xd, xd[1:]):
        with pytest.raises(RuntimeError, match="leaf Variable"):
            F.dropout(leaf, 0.5, inplace=True)
    with pytest.raises(RuntimeError):
        F.dropout(dev(x[:1]).expand(4, 6), 0.5, inplace=True)  # several elements in one place
    with pytest.raises(RuntimeError):
        F.dropout(dev(x.double()), 0.5, inplace=True)
    assert torch.equal(host(xd), x) and torch.equal(torch.webgpu.get_rng_state(), state)
    torch.manual_seed(44)
    with torch.no_grad():  # outside of autograd it may
        F.dropout(xd, 0.5, inplace=True)
    ref.assert_within(host(xd), *ref.dropout(x, 0.5, 44, 0))
