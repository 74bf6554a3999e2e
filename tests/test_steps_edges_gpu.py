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


# ------------------------------------------------------------------------------- compiled

def step_inputs():
    g = torch.Generator().manual_seed(51)
    q, r = torch.randn(2, 5, 3, 32, generator=g), torch.randn(2, 5, 96, generator=g)
    t = torch.randint(0, 96, (2, 5), generator=g)
    return q, r, 1 + 0.3 * torch.randn(32, generator=g), torch.arange(5), torch.rand(16, generator=g), t


def step(q, r, w, pos, inv_freq, t):
    y = torch.ops.webgpu.norm_rope(q, None, pos, inv_freq, w)[0].view(2, 5, 96)
    h = torch.ops.webgpu.dropout(F.dropout(y, 0.25), 0.5, 9, 1, r)
    lp, ent, top, ids = torch.ops.webgpu.token_logprobs(h, t, 4)
    return lp, ent, top, ids, h


@pytest.mark.parametrize("backend_name, outputs", [("webgpu_backend", 5), ("aot_eager", 2)])
def test_a_compiled_step_gives_what_the_eager_one_gives(backend_name, outputs):
    """(for an output without a gradient the second backend asks for zeros, which the device does not make)"""
    q, r, w, pos, inv_freq, t = step_inputs()

    def some(*args):
        return step(*args)[:outputs]

    def run(f, seed):
        torch.manual_seed(seed)
        leaves = [dev(q, True), dev(r, True), dev(w, True)]
        out = f(*leaves, dev(pos), dev(inv_freq), dev(t))
        grads = torch.autograd.grad(out[:2], leaves, [dev(torch.ones(2, 5))] * 2)
        return [host(v) for v in (*out, *grads)]

    torch._dynamo.reset()
    compiled = torch.compile(some, backend=backend_name, fullgraph=True)
    results = []
    for seed in (1, 2):  # a compiled graph takes the seed of each run, not of its trace
        results.append(run(compiled, seed))
        for a, b in zip(results[-1], run(some, seed)):
            assert torch.equal(a, b)
    assert not torch.equal(results[0][0], results[1][0])
    torch._dynamo.reset()


@pytest.mark.parametrize("backend_name", ["webgpu_backend", "aot_eager"])
def test_a_compiled_dropout_in_place(backend_name):
    def f(x):
        y = x * 2.0
        F.dropout(y, 0.5, inplace=True)
        return y

    torch._dynamo.reset()
    compiled = torch.compile(f, backend=backend_name, fullgraph=True)
    x = torch.randn(64)
    for seed in (5, 6):
        torch.manual_seed(seed)
        xd = dev(x, True)
        y = compiled(xd)
        assert torch.equal(host(y).double(), 2 * x.double() * kept(64, 0.5, seed))
        y.backward(dev(torch.ones(64)))
        assert torch.equal(host(xd.grad).double(), 2 * kept(64, 0.5, seed))
    torch._dynamo.reset()


def test_a_dispatch_mode_sees_the_operators():
    from torch.utils._python_dispatch import TorchDispatchMode
    seen = []

    class Look(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func)
            return func(*args, **(kwargs or {}))

    args = [dev(t, t.is_floating_point()) for t in step_inputs()]
    with Look():
        lp = step(*args)[0]
        lp.backward(dev(torch.ones(2, 5)))
    ops = torch.ops.webgpu
    for op in (ops.norm_rope, ops._norm_rope_backward, ops.dropout, ops._draw_dropout, ops._redo_dropout, ops._token_logprobs,
               ops._token_logprobs_backward):
        assert op.default in seen, op


# -------------------------------------------------------------- the functions on tensors and autograd

@pytest.mark.parametrize("device", ["webgpu", "cuda"])
def test_the_functions_on_tensors_count_what_they_write(device):
    """with inputs that require grad, where gradients are not recorded"""
    g = torch.Generator().manual_seed(61)
    q = torch.randn(1, 4, 2, 32, generator=g).to(device).requires_grad_()
    w = torch.ones(32).to(device).requires_grad_()
    x = torch.randn(3, 40, generator=g).to(device).requires_grad_()
    t, gl = torch.arange(3).to(device), torch.ones(3).to(device)
    pos, f = torch.arange(4).to(device), torch.rand(16, generator=g).to(device)
    with torch.no_grad():
        apart = capi.norm_rope(q, None, pos, f, w)[0]
        versions = [v._version for v in (q, w, x, apart)]
        capi.norm_rope(q, None, pos, f, w, q_out=q)
        assert torch.equal(host(q), host(apart))
        got = capi.token_logprobs(x, t)
        assert [v._version for v in (q, w, x, apart)] == [versions[0] + 1, *versions[1:]]
        capi.dropout(x, 0.5, 1, out=x)
        capi.token_logprobs_backward(gl, None, x, t, got.row_max, got.row_sum, out=x)
        assert x._version == versions[2] + 2
    with torch.inference_mode():
        y = x * 1.0
        capi.dropout(y, 0.5, 1, out=y)  # (a tensor without a version)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return capi.dropout(x, 0.5, 7)

    @staticmethod
    def backward(ctx, g):
        return capi.dropout(g, 0.5, 7)


def test_the_functions_on_tensors_in_an_autograd_function():
    x = torch.randn(5, 8)
    xd = dev(x, True)
    y = _Dropout.apply(xd)
    y.backward(dev(torch.ones(5, 8)))
    times = kept(40, 0.5, 7).view(5, 8)
    assert torch.equal(host(y).double(), x.double() * times) and torch.equal(host(xd.grad).double(), times)


# ---------------------------------------------------------------------- rows that are not finite

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, vocab", [(4, 40000), (5, 500), (600, 9000)])
def test_the_maximum_of_a_row_that_is_not_finite(rows, vocab, dtype):
    """NaN where the row holds one, wherever it stands, +inf in a row of others; gradients by the formula"""
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(rows, vocab, generator=g) * 2).to(dtype)
    x[0, vocab - 1] = math.nan
    x[1] = -math.inf
    x[1, 3] = math.nan
    x[2, 5], x[2, 77] = math.inf, math.nan
    x[3, vocab // 2] = math.inf
    t = torch.arange(rows)
    xd, td = dev(x), dev(t)
    got = capi.token_logprobs(xd, td, top_k=3)
    m = host(got.row_max)
    assert bool(torch.isnan(m[:3]).all()) and float(m[3]) == math.inf
    assert torch.equal(m[4:], x[4:].float().amax(1))
    for v in (got.logprob, got.entropy, got.row_sum, got.top_logprobs):
        assert bool(torch.isnan(host(v)[:4]).all()) and not bool(torch.isnan(host(v)[4:]).any())
    grad = host(capi.token_logprobs_backward(dev(torch.ones(rows)), None, xd, td, got.row_max, got.row_sum))
    assert bool(torch.isnan(grad[:4]).all()) and not bool(torch.isnan(grad[4:]).any())


# ------------------------------------------------------------------- where nothing flows back

@pytest.mark.parametrize("how", ["F.dropout", "in place", "operator", "operator's residual", "twice"])
def test_dropout_before_a_result_that_nothing_uses(how):
    """the queries' heads come from a dropout, and only the keys' result is used"""
    q, k = torch.randn(1, 3, 2, 16), torch.randn(1, 3, 1, 16)
    qd, kd = dev(q, True), dev(k, True)
    ops = torch.ops.webgpu
    x = {"F.dropout": lambda: F.dropout(qd, 0.5), "in place": lambda: F.dropout(qd * 1.0, 0.5, inplace=True),
         "operator": lambda: ops.dropout(qd, 0.5, 1), "operator's residual": lambda: ops.dropout(dev(q), 0.5, 1, 0, qd),
         "twice": lambda: F.dropout(F.dropout(qd, 0.5), 0.5)}[how]()
    yk = ops.norm_rope(x, kd, dev(torch.arange(3)), dev(torch.rand(8)))[1]
    yk.backward(dev(torch.ones(1, 3, 1, 16)))
    assert qd.grad is None and kd.grad is not None


def test_dropout_in_place_on_tensors_of_inference_mode():
    x = torch.randn(10)
    torch.manual_seed(3)
    with torch.inference_mode():
        inside = dev(x)
        F.dropout(inside, 0.5, inplace=True)
        ref.assert_within(host(inside), *ref.dropout(x, 0.5, 3, 0))
    normal = dev(x)
    version = normal._version
    with torch.inference_mode():
        F.dropout(normal, 0.5, inplace=True)
    assert normal._version > version
    state = torch.webgpu.get_rng_state()
    before = host(inside)
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        F.dropout(inside, 0.5, inplace=True)
    assert torch.equal(host(inside), before) and torch.equal(torch.webgpu.get_rng_state(), state)
