"""norm_rope, token_logprobs and dropout at the edges of what they take, as far as that shows without a GPU:
calls that do nothing, calls on fake tensors (shapes, types and devices only), refusals."""
import os
import subprocess

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


# ------------------------------------------------------------------------- fake tensors, tracing

def fake(*shape, dtype=torch.float32, grad=False):
    return torch.empty(*shape, dtype=dtype, device="webgpu", requires_grad=grad)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad, torch.inference_mode])
def test_dropout_of_a_fake_tensor_draws_nothing(inplace, grad, mode):
    state = torch.webgpu.get_rng_state()
    with FakeTensorMode(), mode():
        leaf = fake(3, 4, 8, dtype=torch.bfloat16, grad=grad)
        x = leaf if inplace and not grad else leaf * 1
        version = 0 if mode is torch.inference_mode else x._version
        y = F.dropout(x.transpose(0, 1) if not inplace else x, 0.25, inplace=inplace)
        assert y.device.type == "webgpu" and y.dtype == torch.bfloat16
        assert y.shape == ((3, 4, 8) if inplace else (4, 3, 8))
        if inplace:
            assert y is x
            assert mode is torch.inference_mode or x._version > version
        else:
            assert y.transpose(0, 1).is_contiguous()
        assert y.requires_grad == (grad and mode is torch.enable_grad)
        if y.requires_grad:
            y.backward(torch.empty_like(y))
            assert leaf.grad.shape == leaf.shape and leaf.grad.device.type == "webgpu"
        if inplace and grad and mode is torch.enable_grad:
            with pytest.raises(RuntimeError, match="leaf Variable"):
                F.dropout(leaf, 0.25, inplace=True)
    assert torch.equal(torch.webgpu.get_rng_state(), state)


def test_dropout_that_is_refused_draws_nothing():
    state = torch.webgpu.get_rng_state()
    x = torch.empty(0, device="webgpu")
    for p in (-0.1, 1.5, float("nan")):
        for inplace in (False, True):
            with pytest.raises((RuntimeError, ValueError)):
                F.dropout(x, p, inplace=inplace)
    assert torch.equal(torch.webgpu.get_rng_state(), state)


@pytest.mark.parametrize("mode", [torch.enable_grad, torch.inference_mode])
def test_the_operators_on_fake_tensors(mode):
    ops = torch.ops.webgpu
    with FakeTensorMode(), mode():
        on = mode is torch.enable_grad
        q = fake(2, 4, 5, 64, dtype=torch.float16, grad=on).transpose(1, 2)  # heads first
        k = fake(2, 5, 2, 64, dtype=torch.float16, grad=on)
        w = fake(64, grad=on)
        pos, inv_freq = torch.arange(5, device="webgpu"), fake(32)
        yq, yk = ops.norm_rope(q, k, pos, inv_freq, w)
        assert yq.shape == (2, 5, 4, 64) and yk.shape == (2, 5, 2, 64) and yq.stride() == q.stride()
        assert yq.dtype == yk.dtype == torch.float16 and yq.device.type == "webgpu"
        assert ops.norm_rope(q, None, pos, inv_freq)[0].shape == yq.shape
        odd = fake(1, 3, 2, 64, 2)[..., 0]  # head_dim is not dense: the result's is
        assert ops.norm_rope(odd, None, pos[:3], inv_freq)[0].stride(3) == 1
        x = fake(3, 7, 100, dtype=torch.bfloat16, grad=on)
        t = torch.empty(3, 7, dtype=torch.int64, device="webgpu")
        lp, h, top, ids = ops.token_logprobs(x, t, top_k=6)
        assert lp.shape == h.shape == (3, 7) and top.shape == ids.shape == (3, 7, 6)
        assert lp.dtype == h.dtype == top.dtype == torch.float32 and ids.dtype == torch.int64
        d = ops.dropout(yk, 0.1, 1, 2, yk)
        assert d.shape == yk.shape and d.dtype == torch.float16
        for v in (yq, yk, lp, h, top, ids, d):
            assert v.device.type == "webgpu"
            assert v.requires_grad == (on and v is not top and v is not ids)
        if on:
            grads = torch.autograd.grad([yq, yk], [q, k, w], [torch.empty_like(yq), torch.empty_like(yk)])
            assert [g.shape for g in grads] == [q.shape, k.shape, w.shape] and grads[2].dtype == torch.float32
            assert torch.autograd.grad(lp, x, torch.empty_like(lp), retain_graph=True)[0].shape == x.shape
            assert torch.autograd.grad(h, x, torch.empty_like(h))[0].dtype == torch.bfloat16


def test_a_traced_dropout_is_one_that_draws():
    """the seed and the offset of the trace are not in the graph: each run of it draws anew"""
    from torch.fx.experimental.proxy_tensor import make_fx
    state = torch.webgpu.get_rng_state()
    with FakeTensorMode():
        x = fake(8, 8, grad=True)

        def step(x):
            y = F.dropout(F.dropout(x, 0.5), 0.5)
            return y, torch.autograd.grad(y, x, torch.ones_like(y))[0]

        graph = make_fx(step)(x)
        called = [n.target for n in graph.graph.nodes if n.op == "call_function"]
    ops = torch.ops.webgpu
    assert called.count(ops._draw_dropout.default) == 2 and called.count(ops._redo_dropout.default) == 2
    assert torch.equal(torch.webgpu.get_rng_state(), state)


# ------------------------------------------------------------------------- the current device

def test_launches_go_to_the_bound_device(tmp_path):
    """tests/native/current_device_check.cpp: entry points called while another device is current"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    libs = os.path.join(root, "torch-webgpu_amd", "torch_webgpu")
    exe = tmp_path / "check"
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(root, "include"), "-I", os.path.join(rocm, "include"),
                    os.path.join(root, "tests", "native", "current_device_check.cpp"), "-o", str(exe), "-L", libs, "-ltwg_hip",
                    "-Wl,-rpath," + libs, "-Wl,-rpath-link," + os.path.join(rocm, "lib")], check=True)
    done = subprocess.run([str(exe)], stdout=subprocess.PIPE, text=True, timeout=120)
    assert done.returncode == 0 and "every launch on device 0" in done.stdout, done.stdout


# -------------------------------------------------------------- the functions on tensors and autograd

def test_the_functions_on_tensors_refuse_what_they_would_not_differentiate():
    import twg_capi as capi
    with FakeTensorMode():
        q, k, w, f = fake(1, 2, 3, 8), fake(1, 2, 1, 8), fake(8), fake(4)
        pos, x, t, g = torch.arange(2, device="webgpu"), fake(2, 5), torch.zeros(2, dtype=torch.int64, device="webgpu"), fake(2)

        def on(t):
            return t.clone().requires_grad_()

        calls = [lambda: capi.norm_rope(on(q), k, pos, f, w, w), lambda: capi.norm_rope(q, on(k), pos, f, w, w),
                 lambda: capi.norm_rope(q, k, pos, f, on(w), w), lambda: capi.norm_rope(q, k, pos, f, w, on(w)),
                 lambda: capi.norm_rope(q, k, pos, on(f)), lambda: capi.norm_rope(q, k, pos, f, q_out=on(q)),
                 lambda: capi.norm_rope_backward(on(q), k, q, k, pos, f), lambda: capi.token_logprobs(on(x), t),
                 lambda: capi.token_logprobs_backward(on(g), None, x, t, g, g),
                 lambda: capi.token_logprobs_backward(g, None, x, t, g, g, out=on(x)), lambda: capi.dropout(on(x), 0.5, 1),
                 lambda: capi.dropout(x, 0.5, 1, residual=on(x)), lambda: capi.dropout(x, 0.5, 1, out=on(x))]
        for call in calls:
            with pytest.raises(ValueError, match="no gradient is recorded"):
                call()


# ------------------------------------------------------------------------- what large sizes do

def test_the_large_sizes_of_norm_rope_reach_the_loops():
    """of test_steps_large_gpu.py, from the number of workgroups that leave sums: a workgroup of 256 lanes has
    256 / (lanes per head) groups, and a piece of its work is 4 heads a group and 16 tokens at most"""
    import ctypes

    import test_steps_large_gpu as large
    import twg_capi as capi
    P, L, sums = 1 << 20, capi.load(), {}
    for name, (T, Hq, Hk, D, rot, axes, adjacent, dtype, longer) in large.ROPE.items():
        d = capi.NormRope()
        d.dtype, d.weight_dtype, d.position_dtype = capi.DTYPES[dtype], capi.DTYPES[torch.float32], capi.DTYPES[torch.int64]
        d.norm, d.eps, d.n_axes, d.adjacent, d.head_dim, d.rot_dim = 1, 1e-6, axes, adjacent, D, rot
        d.batch, d.tokens, d.positions, d.inv_freq = 1, T, P, P
        for part, H in zip(d.part, (Hq, Hk)):
            part.heads, part.x, part.dy, part.out, part.weight, part.dweight = H, P, P, P, P, P if H else None
            part.x_stride[:] = T * H * (D + longer), H * (D + longer), D + longer
            part.dy_stride[:] = part.out_stride[:] = T * H * D, H * D, D
        workgroups = L.twg_norm_rope_backward_scratch_bytes(ctypes.byref(d)) // (4 * D)
        size = 4 if dtype is torch.float32 else 2
        lanes = max(1, D * size // 32)  # 2 runs of 16 bytes a lane
        if longer:
            lanes = D // 2  # one element a run
        lanes = 1 << (lanes - 1).bit_length()
        if "pieces" in name:
            assert workgroups <= 4096
            assert max(T / 16, T * (Hq + Hk) / (256 // lanes * 4)) > workgroups, name  # more than one piece each
        else:
            assert T * (Hq + Hk) > workgroups * (256 // lanes), name  # more than one head for a group
        sums[name] = T * (Hq + Hk) * D * size * 2
    for name, moved in sums.items():  # the forward call moves the least
        assert ("hinted" in name) == (moved > 256 << 20 and large.ROPE[name][3:5] == (128, 128)), name


def test_norm_rope_backward_wants_a_gradient_for_each_input():
    import twg_capi as capi
    with FakeTensorMode():
        q, k, f, pos = fake(1, 2, 3, 8), fake(1, 2, 1, 8), fake(4), torch.arange(2, device="webgpu")
        for dq, dk, with_k in ((None, k, k), (q, None, k), (q, k, None), (q[:, :1], k, k), (q, k.to(torch.float16), k)):
            with pytest.raises(ValueError):
                capi.norm_rope_backward(dq, dk, q, with_k, pos, f)
