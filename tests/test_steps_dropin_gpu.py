"""The transformer-step operators behind device="webgpu": torch.ops.webgpu.norm_rope,
token_logprobs and dropout with their autograd formulas, F.dropout / nn.Dropout, and a run of all of
them together, against float64 definitions (steps_ref.py) and float64 autograd on the CPU."""
import math

import pytest
import torch
import torch.nn.functional as F

import steps_ref as ref

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def backend():
    import torch_webgpu  # noqa: F401
    torch.webgpu.init()
    yield


def dev(t, grad=False):
    return None if t is None else t.to("webgpu").requires_grad_(grad)


def host(t):
    return t.detach().to("cpu")


def ops():
    return torch.ops.webgpu


def rope_inputs(B=2, T=5, Hq=4, Hk=2, D=64, rot=48, axes=3, dtype=BF16, seed=0):
    g = torch.Generator().manual_seed(seed)
    packed = torch.randn(B, T, Hq + 2 * Hk, D, generator=g).to(dtype)
    pos = torch.randint(0, 5000, (axes, B, T), generator=g)
    inv_freq = (10000.0 ** (-torch.arange(rot // 2) / (rot // 2))).float()
    axis = [i % axes for i in range(rot // 2)]
    wq, wk = (1 + 0.3 * torch.randn(2, D, generator=g)).to(dtype)
    return packed, pos, inv_freq, axis, wq, wk


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("adjacent", [False, True])
def test_norm_rope_and_its_gradients(dtype, adjacent):
    Hq, Hk = 4, 2
    packed, pos, inv_freq, axis, wq, wk = rope_inputs(dtype=dtype)
    q, k = packed[:, :, :Hq], packed[:, :, Hq:Hq + Hk]
    qd, kd = dev(q.contiguous(), True), dev(k.contiguous(), True)
    wqd, wkd = dev(wq, True), dev(wk, True)
    yq, yk = ops().norm_rope(qd, kd, dev(pos), dev(inv_freq), wqd, wkd, pair_axis=axis, adjacent=adjacent)
    how = dict(pair_axis=axis, adjacent=adjacent)
    ref.assert_within(host(yq), *ref.norm_rope(q, pos, inv_freq, wq, **how))
    ref.assert_within(host(yk), *ref.norm_rope(k, pos, inv_freq, wk, **how))
    g = torch.Generator().manual_seed(1)
    dq, dk = torch.randn(q.shape, generator=g).to(dtype), torch.randn(k.shape, generator=g).to(dtype)
    torch.autograd.backward([yq, yk], [dev(dq), dev(dk)])
    for x, w, dy, xd, wd in ((q, wq, dq, qd, wqd), (k, wk, dk, kd, wkd)):
        dx, dxb, dw, dwb = ref.norm_rope_backward(dy, x, pos, inv_freq, w, **how)
        ref.assert_within(host(xd.grad), dx, dxb)
        assert wd.grad.dtype == dtype
        ref.assert_within(host(wd.grad), dw, dwb)


def test_norm_rope_takes_views_and_keeps_their_order():
    packed, pos, inv_freq, axis, wq, wk = rope_inputs()
    pd = dev(packed)
    q = pd[:, :, :4]  # a view of the packed projection
    y = ops().norm_rope(q, None, dev(pos), dev(inv_freq), dev(wq), None, pair_axis=axis)
    assert len(y) == 1
    ref.assert_within(host(y[0]), *ref.norm_rope(packed[:, :, :4], pos, inv_freq, wq, pair_axis=axis))
    first = packed[:, :, :4].transpose(1, 2).contiguous()  # heads first
    y = ops().norm_rope(dev(first).transpose(1, 2), None, dev(pos), dev(inv_freq), dev(wq), None, pair_axis=axis)[0]
    assert y.transpose(1, 2).is_contiguous()
    ref.assert_within(host(y), *ref.norm_rope(packed[:, :, :4], pos, inv_freq, wq, pair_axis=axis))
    odd = packed[..., ::2]  # head_dim stepped by 2: made dense first
    y = ops().norm_rope(pd[:, :, :4][..., ::2], None, dev(pos), dev(inv_freq)[:16].contiguous(), None, None, eps=None,
                        pair_axis=axis[:16])[0]
    ref.assert_within(host(y), *ref.norm_rope(odd[:, :, :4], pos, inv_freq[:16], None, None, axis[:16]))


def test_norm_rope_part_of_the_outputs_used_and_no_tokens():
    packed, pos, inv_freq, axis, wq, wk = rope_inputs(dtype=F32)
    qd, kd, wkd = dev(packed[:, :, :4].contiguous(), True), dev(packed[:, :, 4:6].contiguous(), True), dev(wk, True)
    yq, yk = ops().norm_rope(qd, kd, dev(pos), dev(inv_freq), dev(wq), wkd, pair_axis=axis)
    dk = torch.randn(yk.shape)
    yk.backward(dev(dk))
    assert qd.grad is None
    dx, dxb, dw, dwb = ref.norm_rope_backward(dk, packed[:, :, 4:6], pos, inv_freq, wk, pair_axis=axis)
    ref.assert_within(host(kd.grad), dx, dxb)
    ref.assert_within(host(wkd.grad), dw, dwb)
    none = dev(torch.zeros(2, 0, 4, 64), True)
    w = dev(torch.ones(64), True)
    y = ops().norm_rope(none, None, dev(torch.zeros(2, 0, dtype=torch.int64)), dev(inv_freq), w)[0]
    assert y.shape == (2, 0, 4, 64)
    y.backward(dev(torch.zeros(2, 0, 4, 64)))
    assert bool((host(w.grad) == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_token_logprobs_and_its_gradient(dtype):
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(2, 7, 1009, generator=g) * 3).to(dtype)
    t = torch.randint(0, 1009, (2, 7), generator=g)
    t[0, 3] = -100
    xd = dev(x, True)
    lp, h, top, ids = ops().token_logprobs(xd, dev(t), top_k=6, scale=0.9)
    want = ref.token_logprobs(x.view(14, -1), t.view(14), 6, 0.9)
    assert lp.shape == h.shape == (2, 7) and top.shape == ids.shape == (2, 7, 6) and ids.dtype == torch.int64
    assert lp.requires_grad and h.requires_grad and not top.requires_grad
    ref.assert_within(host(lp).view(14), *want["logprob"])
    ref.assert_within(host(h).view(14), *want["entropy"])
    ref.assert_within(host(top).view(14, 6), *want["top_logprobs"])
    assert torch.equal(host(ids).view(14, 6), want["top_ids"])
    gl, gh = torch.randn(2, 7, generator=g), torch.randn(2, 7, generator=g)
    torch.autograd.backward([lp, h], [dev(gl), dev(gh)])
    ref.assert_within(host(xd.grad).view(14, -1),
                      *ref.token_logprobs_backward(gl.view(14), gh.view(14), x.view(14, -1), t.view(14), 0.9))
    x2 = dev(x, True)  # only the log probability used
    ops().token_logprobs(x2, dev(t))[0].backward(dev(gl))
    ref.assert_within(host(x2.grad).view(14, -1), *ref.token_logprobs_backward(gl.view(14), None, x.view(14, -1), t.view(14)))


def test_token_logprobs_of_views_one_row_and_no_rows():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(6, 500, generator=g)
    t = torch.randint(0, 400, (6,), generator=g)
    xd = dev(x)
    for view, host_view in ((xd[:, :400], x[:, :400]), (xd[::2, 50:450], x[::2, 50:450]), (xd[1:4, ::2], x[1:4, ::2])):
        n = host_view.shape[0]
        tt = t[:n] % host_view.shape[1]
        ref.assert_within(host(ops().token_logprobs(view, dev(tt))[0]), *ref.token_logprobs(host_view, tt)["logprob"])
    one = ops().token_logprobs(xd[0], dev(t[0]))[0]
    assert one.shape == ()
    ref.assert_within(host(one).view(1), *ref.token_logprobs(x[:1], t[:1])["logprob"])
    none = dev(torch.zeros(0, 500), True)
    lp = ops().token_logprobs(none, dev(torch.zeros(0, dtype=torch.int64)), top_k=2)[0]
    lp.backward(dev(torch.zeros(0)))
    assert none.grad.shape == (0, 500)


def test_masks_of_the_framework_choose_the_rows_of_a_loss():
    """ne.Scalar on the targets, masked_select on the log probabilities"""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(50, 300, generator=g)
    t = torch.randint(0, 300, (50,), generator=g)
    t[::3] = -100
    td = dev(t)
    lp = ops().token_logprobs(dev(x), td)[0]
    chosen = torch.masked_select(lp, td.ne(-100))
    want, bound = ref.token_logprobs(x, t)["logprob"]
    ref.assert_within(host(chosen), want[t != -100], bound[t != -100])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_dropout_op_and_its_gradients(dtype):
    g = torch.Generator().manual_seed(6)
    x, r, dy = (torch.randn(3, 40, 24, generator=g).to(dtype) for _ in range(3))
    xd, rd = dev(x, True), dev(r, True)
    y = ops().dropout(xd, 0.3, 123, 7, rd)
    ref.assert_within(host(y), *ref.dropout(x, 0.3, 123, 7, r))
    y.backward(dev(dy))
    ref.assert_within(host(xd.grad), *ref.dropout(dy, 0.3, 123, 7))
    assert torch.equal(host(rd.grad), dy)
    # an incoming gradient stored in another order meets the same elements
    xd.grad = None
    y = ops().dropout(xd, 0.3, 123, 7)
    y.backward(dev(dy.permute(2, 0, 1).contiguous()).permute(1, 2, 0))
    ref.assert_within(host(xd.grad), *ref.dropout(dy, 0.3, 123, 7))
    # and a transposed input keeps its storage order in the result
    y = ops().dropout(dev(x).transpose(0, 2), 0.3, 123, 7)
    assert y.transpose(0, 2).is_contiguous()
    ref.assert_within(host(y), *ref.dropout(x.transpose(0, 2), 0.3, 123, 7))


def test_f_dropout_draws_from_the_seed_and_one_offset_per_call():
    x = torch.randn(1000)
    xd = dev(x)
    torch.manual_seed(99)
    a, b = F.dropout(xd, 0.25), F.dropout(xd, 0.25)
    ref.assert_within(host(a), *ref.dropout(x, 0.25, 99, 0))
    ref.assert_within(host(b), *ref.dropout(x, 0.25, 99, 1))
    state = torch.webgpu.get_rng_state()
    c = F.dropout(xd, 0.25)
    torch.webgpu.set_rng_state(state)
    assert torch.equal(host(F.dropout(xd, 0.25)), host(c))
    torch.manual_seed(99)
    assert torch.webgpu.initial_seed() == 99
    assert torch.equal(host(F.dropout(xd, 0.25)), host(a))
    # nothing drawn, and the input itself, where there is nothing to drop
    state = torch.webgpu.get_rng_state()
    assert F.dropout(xd, 0.0) is xd or torch.equal(host(F.dropout(xd, 0.0)), x)
    assert torch.equal(host(F.dropout(xd, 0.5, training=False)), x)
    assert torch.equal(torch.webgpu.get_rng_state(), state)
    assert bool((host(F.dropout(xd, 1.0)) == 0).all())


def test_nn_dropout_trains_and_works_in_place():
    torch.manual_seed(7)
    layer = torch.nn.Dropout(0.4)
    x, dy = torch.randn(64, 33), torch.randn(64, 33)
    xd = dev(x, True)
    y = layer(xd)
    y.backward(dev(dy))
    ref.assert_within(host(y), *ref.dropout(x, 0.4, 7, 0))
    ref.assert_within(host(xd.grad), *ref.dropout(dy, 0.4, 7, 0))
    assert torch.equal(host(layer.eval()(xd)), x)
    z = dev(x)
    version = z._version
    out = F.dropout(z, 0.4, inplace=True)
    assert out.data_ptr() == z.data_ptr() and z._version > version
    ref.assert_within(host(z), *ref.dropout(x, 0.4, 7, 1))
    with torch.inference_mode():
        ref.assert_within(host(F.dropout(dev(x), 0.4)), *ref.dropout(x, 0.4, 7, 2))
    with pytest.raises(RuntimeError):
        F.dropout(xd, 0.4, inplace=True)


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_recomputed_dropout_drops_the_same_elements(reentrant):
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(21)
    x, dy = torch.randn(500), torch.randn(500)
    xd = dev(x, True)
    y = checkpoint(lambda t: F.dropout(t, 0.5), xd, use_reentrant=reentrant)
    F.dropout(dev(x), 0.5)  # another draw in between
    y.backward(dev(dy))
    ref.assert_within(host(y), *ref.dropout(x, 0.5, 21, 0))
    ref.assert_within(host(xd.grad), *ref.dropout(dy, 0.5, 21, 0))


def test_cpu_gradients_in_the_same_process():
    x = torch.arange(6.0).requires_grad_()
    (x * x).sum().backward()
    assert torch.equal(x.grad, 2 * torch.arange(6.0))


def test_one_tensor_used_twice_gets_the_sum_of_its_gradients():
    x = torch.randn(4, 30)
    t = torch.tensor([1, 2, 3, 4])
    xd = dev(x, True)
    h = ops().dropout(xd, 0.25, 1, 1, xd)  # x is the residual, too
    lp = ops().token_logprobs(h, dev(t))[0]
    ent = ops().token_logprobs(xd, dev(t))[1]
    torch.autograd.backward([lp, ent], [dev(torch.ones(4)), dev(torch.ones(4))])
    x6 = x.double().requires_grad_()
    keep = ref.keep_mask(120, 0.25, 1, 1).view(4, 30)
    logp = torch.log_softmax(x6 + keep * x6 / 0.75, -1)
    plain = torch.log_softmax(x6, -1)
    (logp.gather(1, t[:, None]).sum() - (plain.exp() * plain).sum()).backward()
    # three float32 gradients of order 1 added: 100 U each
    assert float((host(xd.grad).double() - x6.grad).abs().max()) <= 300 * ref.U * 4


def test_a_training_step_of_all_of_them_together():
    """q and k heads -> norm and rotation -> residual with dropout -> log probability, entropy -> gradients of the
    inputs and the norm weights; against float64 autograd of the same chain on the CPU."""
    B, T, H, D = 2, 6, 3, 32
    g = torch.Generator().manual_seed(11)
    q, r = torch.randn(B, T, H, D, generator=g), torch.randn(B, T, H * D, generator=g)
    w = 1 + 0.3 * torch.randn(D, generator=g)
    pos = torch.randint(0, 1000, (2, B, T), generator=g)
    inv_freq = (100.0 ** (-torch.arange(D // 2) / (D // 2))).float()
    axis = [i % 2 for i in range(D // 2)]
    t = torch.randint(0, H * D, (B, T), generator=g)
    t[1, 2] = -100
    qd, rd, wd = dev(q, True), dev(r, True), dev(w, True)
    rot = ops().norm_rope(qd, None, dev(pos), dev(inv_freq), wd, pair_axis=axis)[0]
    hidden = ops().dropout(rot.view(B, T, H * D), 0.2, 5, 1, rd)
    lp, ent, _, _ = ops().token_logprobs(hidden, dev(t))
    gl, gh = torch.randn(B, T, generator=g), torch.randn(B, T, generator=g)
    torch.autograd.backward([lp, ent], [dev(gl), dev(gh)])

    q6, r6, w6 = (v.double().requires_grad_() for v in (q, r, w))
    z = q6 / torch.sqrt(q6.square().mean(-1, keepdim=True) + 1e-6) * w6
    angle = torch.stack([pos[a].double() * f for a, f in zip(axis, inv_freq.double())], -1)[:, :, None]
    lo, hi = z[..., :D // 2], z[..., D // 2:]
    y = torch.cat((lo * angle.cos() - hi * angle.sin(), hi * angle.cos() + lo * angle.sin()), -1)
    keep = ref.keep_mask(B * T * H * D, 0.2, 5, 1).view(B, T, H * D)
    scale = 65536 / (65536 - math.floor(0.2 * 65536 + 0.5))
    h6 = r6 + keep * y.reshape(B, T, H * D) * scale
    logp = torch.log_softmax(h6, -1)
    lp6 = torch.where(t == -100, 0.0, logp.gather(-1, t.clamp(min=0)[..., None])[..., 0])
    ent6 = -(logp.exp() * logp).sum(-1)
    torch.autograd.backward([lp6, ent6], [gl.double(), gh.double()])
    # values of order 1 to 10 through four binary32 steps: 200 U of the largest magnitude a result is summed from
    for got, want in ((lp, lp6), (ent, ent6), (hidden, h6), (qd.grad, q6.grad), (rd.grad, r6.grad), (wd.grad, w6.grad)):
        room = 200 * ref.U * max(10.0, float(want.detach().abs().max()) * (B * T * H if want.dim() == 1 else 1))
        assert float((host(got).double() - want.detach()).abs().max()) <= room


def test_refusals():
    packed, pos, inv_freq, axis, wq, wk = rope_inputs()
    q, pd, fd = dev(packed[:, :, :4].contiguous()), dev(pos), dev(inv_freq)
    nr = ops().norm_rope
    bad = [lambda: nr(q[0], None, pd, fd, pair_axis=axis), lambda: nr(q, None, pd, fd), lambda: nr(q, None, pd, fd, pair_axis=axis[1:]),
           lambda: nr(q, None, pd, fd, pair_axis=[5] * 24), lambda: nr(q, None, pd[:, :1], fd, pair_axis=axis),
           lambda: nr(q, None, pd.to(torch.int16), fd, pair_axis=axis), lambda: nr(q, None, pd, fd.to(F16), pair_axis=axis),
           lambda: nr(q, q.to(F32), pd, fd, pair_axis=axis), lambda: nr(q, None, pd, fd, dev(wq), eps=None, pair_axis=axis),
           lambda: nr(q, None, pd, fd, dev(wq)[:5], pair_axis=axis), lambda: nr(q, None, pd, fd, dev(wq.to(F16)), pair_axis=axis),
           lambda: nr(q, None, pos, fd, pair_axis=axis), lambda: nr(q, None, pd, fd, eps=-1.0, pair_axis=axis),
           lambda: nr(q.to(torch.int32), None, pd, fd, pair_axis=axis), lambda: nr(q[..., :47], None, pd, fd, pair_axis=axis)]
    x, t = dev(torch.randn(4, 10)), dev(torch.zeros(4, dtype=torch.int64))
    tl = ops().token_logprobs
    bad += [lambda: tl(x, t[:3]), lambda: tl(x, t.to(F32)), lambda: tl(x, t, 11), lambda: tl(x, t, -1), lambda: tl(x, t, 0, 0.0),
            lambda: tl(x, t, 0, math.inf), lambda: tl(x, t, 0, 1e-60), lambda: tl(x.to(torch.int32), t), lambda: tl(x, t.to("cpu")),
            lambda: tl(x[:, :0], t)]
    do = ops().dropout
    bad += [lambda: do(x, 1.5, 1), lambda: do(x, -0.1, 1), lambda: do(x, math.nan, 1), lambda: do(x.to(torch.float64), 0.5, 1),
            lambda: do(x, 0.5, 1, 0, x[:2]), lambda: do(x, 0.5, 1, 0, x.to(F16)), lambda: F.dropout(x, 1.5)]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            call()
            pytest.fail(f"call {i} was not refused")


def test_no_second_derivative():
    x = dev(torch.randn(3, 8), True)
    lp = ops().token_logprobs(x, dev(torch.zeros(3, dtype=torch.int64)))[0]
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(lp, x, dev(torch.ones(3)), create_graph=True)
