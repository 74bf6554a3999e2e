"""norm_rope, token_logprobs and dropout on the GPU against their definitions in float64
(steps_ref.py), through the functions on tensors of twg_capi: "webgpu" tensors on the library's
stream, PyTorch-ROCm tensors on torch's current stream, and captured graphs."""
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
    capi.init()
    yield


def dev(t):
    """t on the device with its own strides"""
    if t is None:
        return None
    base = torch.empty(0, dtype=t.dtype).set_(t.untyped_storage())
    return base.to("webgpu").as_strided(t.size(), t.stride(), t.storage_offset())


def host(t):
    return t.to("cpu")


# ----------------------------------------------------------------------------- norm_rope

def heads(g, B, T, H, D, dtype, layout):
    """[B, T, H, D] stored in some way, with other data around it"""
    if layout == "packed":  # a slice of a projection with more heads
        return (torch.randn(B, T, H + 3, D, generator=g) * 1.5).to(dtype)[:, :, 1:H + 1]
    if layout == "heads_first":
        return (torch.randn(B, H, T, D, generator=g) * 1.5).to(dtype).transpose(1, 2)
    if layout == "ragged":  # rows of D + 1 elements, starting at the third
        return (torch.randn(B * T * H * (D + 1) + 3, generator=g) * 1.5).to(dtype)[3:].view(B, T, H, D + 1)[..., :D]
    if layout == "broadcast":  # one head for all
        return (torch.randn(B, T, 1, D, generator=g) * 1.5).to(dtype).expand(B, T, H, D)
    return (torch.randn(B, T, H, D, generator=g) * 1.5).to(dtype)


def rope_inputs(B, T, Hq, Hk, D, rot, axes, dtype, layout, positions, weights=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = heads(g, B, T, Hq, D, dtype, layout)
    k = heads(g, B, T, Hk, D, dtype, layout) if Hk else None
    pos = torch.randint(0, 1 << 20, (axes, B, T), generator=g)
    pos = (pos / 7).float() if positions is F32 else pos.to(positions)
    inv_freq = (10000.0 ** (-torch.arange(rot // 2).double() / max(1, rot // 2))).float()
    pair_axis = [int(v) for v in torch.randint(0, axes, (rot // 2,), generator=g)] if axes > 1 else None
    wq = (1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if weights else None
    wk = (1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if weights and Hk else None
    dq = torch.randn(B, T, Hq, D, generator=g).to(dtype)
    dk = torch.randn(B, T, Hk, D, generator=g).to(dtype) if Hk else None
    return q, k, pos, inv_freq, pair_axis, wq, wk, dq, dk


I64, I32 = torch.int64, torch.int32
ROPE = [
    # B, T, Hq, Hk, D, rot, axes, norm, adjacent, dtype, layout, position type
    (1, 1, 1, 0, 2, 2, 1, True, False, F32, "dense", I64),
    (1, 1, 32, 8, 128, 128, 1, True, False, BF16, "packed", I64),
    (3, 1, 5, 1, 64, 64, 1, True, True, F16, "dense", I32),
    (2, 17, 4, 2, 80, 80, 3, True, True, BF16, "heads_first", I64),
    (2, 33, 3, 3, 72, 40, 2, True, False, F16, "packed", F32),
    (1, 5, 2, 1, 34, 34, 1, True, False, BF16, "ragged", I64),
    (1, 7, 3, 2, 34, 18, 2, True, True, F32, "ragged", I64),
    (2, 9, 6, 2, 96, 0, 1, True, False, BF16, "dense", I64),
    (2, 3, 2, 2, 256, 64, 1, True, False, F32, "dense", I64),
    (1, 4, 2, 1, 512, 512, 8, True, True, BF16, "dense", I64),
    (1, 3, 2, 1, 512, 512, 1, True, False, F32, "ragged", I64),
    (1, 6, 3, 1, 510, 254, 2, True, False, F16, "packed", I64),
    (2, 40, 16, 4, 64, 64, 1, False, False, BF16, "packed", I32),
    (2, 21, 4, 4, 80, 80, 3, False, True, F16, "heads_first", F32),
    (1, 13, 2, 1, 6, 6, 1, False, True, F32, "ragged", I64),
    (3, 50, 7, 0, 128, 128, 1, True, False, BF16, "dense", I64),
    (1, 1500, 3, 1, 64, 64, 1, True, False, BF16, "packed", I64),
    (2, 4, 4, 4, 64, 64, 1, True, False, F16, "broadcast", I64),
    (1, 2, 200, 40, 32, 32, 1, True, True, BF16, "dense", I64),
]


@pytest.mark.parametrize("case", ROPE, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_norm_rope(case):
    B, T, Hq, Hk, D, rot, axes, norm, adjacent, dtype, layout, ptype = case
    q, k, pos, inv_freq, pair_axis, wq, wk, dq, dk = rope_inputs(B, T, Hq, Hk, D, rot, axes, dtype, layout, ptype, norm)
    how = dict(eps=1e-6 if norm else None, pair_axis=pair_axis, adjacent=adjacent)
    qd, kd, posd, fd, wqd, wkd = (dev(t) for t in (q, k, pos, inv_freq, wq, wk))
    got = capi.norm_rope(qd, kd, posd, fd, wqd, wkd, **how)
    for x, w, y, name in ((q, wq, got[0], "q"), (k, wk, got[1], "k")):
        if x is None:
            assert y is None
            continue
        want, bound = ref.norm_rope(x, pos, inv_freq, w, **how)
        ref.assert_within(host(y), want, bound, name)
    grads = capi.norm_rope_backward(dev(dq), dev(dk), qd, kd, posd, fd, wqd, wkd, **how)
    for i, (x, w, dy, name) in enumerate(((q, wq, dq, "q"), (k, wk, dk, "k"))):
        if x is None:
            assert grads[i] is None and grads[2 + i] is None
            continue
        dx, dxb, dw, dwb = ref.norm_rope_backward(dy, x, pos, inv_freq, w, **how)
        ref.assert_within(host(grads[i]), dx, dxb, "d" + name)
        if w is None:
            assert grads[2 + i] is None
        else:
            ref.assert_within(host(grads[2 + i]), dw, dwb, "dw" + name)
    again = capi.norm_rope_backward(dev(dq), dev(dk), qd, kd, posd, fd, wqd, wkd, **how)
    for a, b in zip(grads, again):  # sums in a fixed order
        assert (a is None and b is None) or torch.equal(host(a), host(b))


def test_norm_rope_float32_weights_beside_16_bit_heads():
    q, k, pos, inv_freq, _, wq, wk, dq, dk = rope_inputs(2, 6, 4, 2, 64, 64, 1, BF16, "packed", I64)
    wq, wk = wq.float() * 1.001, None
    args = [dev(t) for t in (q, k, pos, inv_freq, wq, wk)]
    got = capi.norm_rope(*args)
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        ref.assert_within(host(y), *ref.norm_rope(x, pos, inv_freq, w))
    grads = capi.norm_rope_backward(dev(dq), dev(dk), *args)
    dx, dxb, dw, dwb = ref.norm_rope_backward(dq, q, pos, inv_freq, wq)
    ref.assert_within(host(grads[0]), dx, dxb)
    assert grads[2].dtype == F32 and grads[3] is None
    ref.assert_within(host(grads[2]), dw, dwb)


def test_norm_rope_positions_shared_by_the_batch_and_far_out():
    q, k, _, inv_freq, _, wq, wk, _, _ = rope_inputs(3, 5, 2, 1, 64, 64, 1, F32, "dense", I64)
    for pos in (torch.tensor([0, 1, 2_000_000, 400_000_000, 2 ** 31 - 1]), torch.tensor([-5, -4, 0, 3, -(2 ** 31)])):
        got = capi.norm_rope(*(dev(t) for t in (q, k, pos, inv_freq, wq, wk)))
        want, bound = ref.norm_rope(q, pos.expand(3, 5), inv_freq, wq)
        # 2^31 turns in binary64: the reference's own angle is off by 2^31 * 2^-53 rad, the
        # kernel's by 3 roundings of the turns, 2 pi 3 * 2^-53 * 2^31 / (2 pi) rad
        ref.assert_within(host(got[0]), want, bound + 4 * 2.0 ** -22 * want.abs().amax(-1, keepdim=True))


def test_norm_rope_in_place_and_into_a_wider_buffer():
    q, k, pos, inv_freq, _, wq, wk, _, _ = rope_inputs(2, 12, 4, 2, 64, 48, 1, BF16, "packed", I64)
    args = [dev(t) for t in (q, k, pos, inv_freq, wq, wk)]
    apart = capi.norm_rope(*args)
    cache = torch.full((2, 2, 30, 64), 7.0, dtype=BF16)  # keys go into rows 10..21 of a longer buffer, heads first
    cached = dev(cache)
    capi.norm_rope(*args, k_out=cached[:, :, 10:22].transpose(1, 2))
    back = host(cached)
    assert torch.equal(back[:, :, 10:22].transpose(1, 2), host(apart[1]))
    assert bool((back[:, :, :10] == 7).all()) and bool((back[:, :, 22:] == 7).all())
    capi.norm_rope(*args, q_out=args[0], k_out=args[1])
    assert torch.equal(host(args[0]), host(apart[0])) and torch.equal(host(args[1]), host(apart[1]))


def test_norm_rope_weights_off_their_alignment():
    q, k, pos, inv_freq, _, wq, wk, dq, dk = rope_inputs(2, 6, 4, 2, 64, 64, 1, BF16, "dense", I64)
    wide = dev(torch.cat((torch.zeros(1, dtype=BF16), wq, wk)))
    args = [dev(t) for t in (q, k, pos, inv_freq)] + [wide[1:65], wide[65:]]
    got = capi.norm_rope(*args)
    ref.assert_within(host(got[0]), *ref.norm_rope(q, pos, inv_freq, wq))
    grads = capi.norm_rope_backward(dev(dq), dev(dk), *args)
    for i, (x, w, dy) in enumerate(((q, wq, dq), (k, wk, dk))):
        dx, dxb, dw, dwb = ref.norm_rope_backward(dy, x, pos, inv_freq, w)
        ref.assert_within(host(grads[i]), dx, dxb)
        ref.assert_within(host(grads[2 + i]), dw, dwb)


def test_two_streams_at_once():
    """calls on two of torch's streams share nothing"""
    g = torch.Generator().manual_seed(31)
    q, k, pos, inv_freq, _, wq, wk, dq, dk = (t.cuda() if torch.is_tensor(t) else t for t in
                                              rope_inputs(2, 300, 4, 2, 64, 64, 1, BF16, "packed", I64))
    x, t = torch.randn(5, 60000, generator=g).cuda(), torch.randint(0, 60000, (5,), generator=g).cuda()

    def work():
        return [*capi.norm_rope_backward(dq, dk, q, k, pos, inv_freq, wq, wk), *capi.token_logprobs(x, t, top_k=10)]

    alone = work()
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(work())
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, alone))


def test_norm_rope_zero_heads_and_special_values():
    q, k, pos, inv_freq, _, wq, wk, dq, dk = rope_inputs(1, 4, 3, 1, 64, 64, 1, F32, "dense", I64)
    q[0, 1, 2] = 0.0         # the norm of nothing: 0 * eps^(-1/2)
    q[0, 2, 0, 5] = math.nan  # stays in its head
    q[0, 3, 1, 7] = 1e-25     # squares underflow to 0 beside eps
    got = host(capi.norm_rope(*(dev(t) for t in (q, k, pos, inv_freq, wq, wk)))[0])
    assert bool((got[0, 1, 2] == 0).all())
    assert bool(torch.isnan(got[0, 2, 0]).all()) and int(torch.isnan(got).sum()) == 64
    want, bound = ref.norm_rope(q, pos, inv_freq, wq)
    ref.assert_within(got[0, 3], want[0, 3], bound[0, 3])


def test_norm_rope_gradients_against_differences():
    """dx and dw as directional derivatives of the float64 definition: the kernel's float32 gradient times a
    direction against a central difference of step h, whose own error is h^2 times a third derivative."""
    q, _, pos, inv_freq, pair_axis, wq, _, dq, _ = rope_inputs(1, 6, 2, 0, 32, 20, 2, F32, "dense", I64)
    how = dict(pair_axis=pair_axis, adjacent=True)
    gq, _, gw, _ = capi.norm_rope_backward(dev(dq), None, dev(q), None, dev(pos), dev(inv_freq), dev(wq), None, **how)
    g = torch.Generator().manual_seed(5)
    vx, vw, h = torch.randn(q.shape, generator=g).double(), torch.randn(wq.shape, generator=g).double(), 1e-5

    def loss(x, w):
        return float((ref.norm_rope(x, pos, inv_freq, w, **how)[0] * dq.double()).sum())

    for grad, v, f in ((gq, vx, lambda s: loss(q.double() + s * vx, wq)), (gw, vw, lambda s: loss(q, wq.double() + s * vw))):
        slope = (f(h) - f(-h)) / (2 * h)
        along = float((host(grad).double() * v).sum())
        # float64 differences: 2^-52 of a loss of order |dq||y| over h; gradient: 100 U per term
        room = 2.0 ** -52 * float(dq.abs().sum()) * 8 / h + 100 * ref.U * float((host(grad).double() * v).abs().sum()) + 1e-7
        assert abs(slope - along) <= room, (slope, along, room)


# ------------------------------------------------------------------------ token_logprobs

def check_logprobs(x, t, top_k, scale=1.0, on=dev):
    got = capi.token_logprobs(on(x), on(t), top_k=top_k, scale=scale)
    want = ref.token_logprobs(x, t, top_k, scale)
    for name in ("logprob", "entropy", "row_max", "row_sum", "top_logprobs"):
        ref.assert_within(host(getattr(got, name)), *want[name], what=name)
    assert torch.equal(host(got.top_ids), want["top_ids"]), "top_ids"
    return got


LOGITS = [
    # rows, vocab, dtype, top_k, scale, pitch beyond vocab, first element
    (1, 1, F32, 1, 1.0, 0, 0), (3, 2, BF16, 2, 1.0, 0, 0), (2, 63, F16, 20, 0.5, 0, 0), (5, 64, BF16, 64, 1.0, 3, 1),
    (4, 65, F32, 5, 2.0, 0, 3), (1, 1000, BF16, 20, 1.0, 0, 0), (7, 1023, F16, 33, 0.7, 1, 5), (2, 4096, BF16, 0, 1.0, 0, 0),
    (3, 4099, F32, 20, 1.0, 0, 1), (1, 32768, F32, 20, 1.25, 0, 0), (2, 50257, BF16, 5, 1.0, 0, 0), (1, 131071, BF16, 64, 1.0, 0, 7),
    (300, 257, BF16, 3, 1.0, 7, 2), (700, 1024, F16, 5, 1.0, 0, 0), (33, 20011, F32, 20, 1.0, 2, 1),
]


@pytest.mark.parametrize("rows, vocab, dtype, top_k, scale, extra, first", LOGITS)
def test_token_logprobs(rows, vocab, dtype, top_k, scale, extra, first):
    g = torch.Generator().manual_seed(rows * 1000 + vocab)
    flat = (torch.randn(rows * (vocab + extra) + first, generator=g) * 3).to(dtype)
    x = flat[first:].view(rows, vocab + extra)[:, :vocab]
    t = torch.randint(0, vocab, (rows,), generator=g)
    t[rows // 2] = -100 if rows > 1 else t[0]
    if rows % 2:
        t = t.int()
    got = check_logprobs(x, t, top_k, scale)
    # backward
    for gl, gh in ((torch.randn(rows, generator=g), None), (torch.randn(rows, generator=g), torch.randn(rows, generator=g)),
                   (None, torch.randn(rows, generator=g))):
        grad = capi.token_logprobs_backward(dev(gl), dev(gh), dev(x), dev(t), got.row_max, got.row_sum, got.entropy, scale=scale)
        ref.assert_within(host(grad), *ref.token_logprobs_backward(gl, gh, x, t, scale), what="grad")


@pytest.mark.parametrize("rows, vocab", [(1, 70001), (6, 3001), (900, 130)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_token_logprobs_masks(rows, vocab, dtype):
    """-inf entries, rows with one entry or none left, rows of the type's lowest value"""
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    x[torch.rand(rows, vocab, generator=g) < 0.6] = -math.inf
    t = torch.randint(0, vocab, (rows,), generator=g)
    variants = [lambda r: r.fill_(-math.inf), lambda r: r.fill_(-math.inf)[vocab // 2:vocab // 2 + 1].fill_(1.5),
                lambda r: r.fill_(torch.finfo(dtype).min), lambda r: r[:vocab // 2].fill_(torch.finfo(dtype).min),
                lambda r: r.fill_(torch.finfo(dtype).max), lambda r: r[::2].fill_(-math.inf)]
    for i, change in enumerate(variants[:max(rows, 1)] if rows > 1 else variants):
        y = x.clone() if rows == 1 else x
        change(y[0 if rows == 1 else i])
        if rows == 1:
            check_logprobs(y, t, 20)
    if rows > 1:
        got = check_logprobs(x, t, 20)
        gl, gh = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
        grad = capi.token_logprobs_backward(dev(gl), dev(gh), dev(x), dev(t), got.row_max, got.row_sum, got.entropy)
        ref.assert_within(host(grad), *ref.token_logprobs_backward(gl, gh, x, t), what="grad")
        assert bool((host(grad)[0] == 0).all())  # nothing left in row 0


@pytest.mark.parametrize("rows, vocab", [(1, 40000), (3, 500), (600, 300)])
def test_token_logprobs_not_a_number(rows, vocab):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(rows, vocab, generator=g)
    x[0, 7], x[0, vocab - 3] = math.nan, math.nan
    if rows > 1:
        x[1, 11] = math.inf
    t = torch.randint(0, vocab, (rows,), generator=g)
    got = capi.token_logprobs(dev(x), dev(t), top_k=4)
    bad = [0, 1] if rows > 1 else [0]
    for name in ("logprob", "entropy", "row_sum", "top_logprobs"):
        v = host(getattr(got, name))
        assert bool(torch.isnan(v[bad]).all()), name
        assert not bool(torch.isnan(v[len(bad):]).any()), name
    ids = host(got.top_ids)
    assert ids[0, :2].tolist() == [7, vocab - 3]  # NaN above everything, the lower id first
    if rows > 1:
        assert int(ids[1, 0]) == 11


def test_token_logprobs_ties_take_the_lowest_ids():
    x = torch.zeros(2, 5000, dtype=BF16)
    x[0, 4000:] = 1.0
    x[1, 1::2] = -0.0  # equal to 0
    got = capi.token_logprobs(dev(x), dev(torch.zeros(2, dtype=torch.int64)), top_k=6)
    assert host(got.top_ids).tolist() == [[4000, 4001, 4002, 4003, 4004, 4005], [0, 1, 2, 3, 4, 5]]


def test_token_logprobs_targets_out_of_range():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, 1000, generator=g)
    t = torch.tensor([1000, -1, -100, 999])
    got = capi.token_logprobs(dev(x), dev(t))
    lp = host(got.logprob)
    assert bool(torch.isnan(lp[:2]).all()) and float(lp[2]) == 0.0 and math.isfinite(float(lp[3]))
    gl = torch.ones(4)
    grad = host(capi.token_logprobs_backward(dev(gl), None, dev(x), dev(t), got.row_max, got.row_sum))
    assert bool(torch.isnan(grad[:2]).all()) and bool((grad[2] == 0).all()) and bool(torch.isfinite(grad[3]).all())
    # another ignore_index; with no gradient asked for, nothing of the row is read
    got = capi.token_logprobs(dev(x), dev(t), ignore_index=1000)
    assert float(host(got.logprob)[0]) == 0.0 and bool(torch.isnan(host(got.logprob)[2]))
    x[0, 3] = math.nan
    gl = torch.tensor([0.0, 0.0, 0.0, 1.0])
    grad = host(capi.token_logprobs_backward(dev(gl), None, dev(x), dev(t), got.row_max, got.row_sum))
    assert bool((grad[:3] == 0).all())


@pytest.mark.parametrize("order", ["rising", "falling", "last lanes", "one wave"])
@pytest.mark.parametrize("rows, vocab", [(1, 70000), (3, 9000), (300, 9000), (1100, 5000), (2, 1500)])
def test_token_logprobs_alternatives_in_unkind_orders(rows, vocab, order):
    """every element a new best, the best at the very end, all of the best in one lane's or one wavefront's elements,
    and values that tie at the place of the last alternative"""
    x = torch.linspace(-5, 5, vocab).repeat(rows, 1)
    if order == "falling":
        x = x.flip(1).contiguous()
    elif order == "last lanes":
        x = torch.zeros(rows, vocab)
        x[:, 504:512] = torch.arange(8.0) + 1
        x[:, -12:] = 9.0
    elif order == "one wave":
        x = torch.full((rows, vocab), -1.0)
        x[:, 512:1024] = 2.0
    t = torch.zeros(rows, dtype=torch.int64)
    for dtype in (F32, BF16):
        xd = x.to(dtype)
        got = capi.token_logprobs(dev(xd), dev(t), top_k=40)
        assert torch.equal(host(got.top_ids), torch.sort(xd.float(), dim=1, descending=True, stable=True).indices[:, :40])


def test_token_logprobs_more_rows_than_one_launch_takes():
    rows = (1 << 22) + 3
    x = torch.zeros(rows, 2, dtype=F16)
    x[:, 1] = (torch.arange(rows) % 7).to(F16)
    t = (torch.arange(rows) % 2).int()
    xd, td = dev(x), dev(t)
    got = capi.token_logprobs(xd, td, top_k=1)
    lp = torch.log_softmax(x.double(), 1).gather(1, t.long()[:, None])[:, 0]
    assert float((host(got.logprob).double() - lp).abs().max()) <= 64 * ref.U * 7
    assert torch.equal(host(got.top_ids)[:, 0], (x[:, 1] > 0).long())
    grad = host(capi.token_logprobs_backward(dev(torch.ones(rows)), None, xd, td, got.row_max, got.row_sum))
    p = torch.softmax(x.double(), 1)
    want = torch.nn.functional.one_hot(t.long(), 2) - p
    assert float((grad.double() - want).abs().max()) <= 2.0 ** -11 + 2.0 ** -20


def test_offsets_beyond_32_bits():
    """rows and tokens 2^31 and more elements apart"""
    far = (1 << 31) + 64
    buf = torch.empty(far + 4096, dtype=F16, device="webgpu")
    g = torch.Generator().manual_seed(12)
    x = torch.randn(2, 3000, generator=g).to(F16)
    rows = buf.as_strided((2, 3000), (far, 1))
    rows.copy_(dev(x))
    t = torch.randint(0, 3000, (2,), generator=g)
    got = capi.token_logprobs(rows, dev(t), top_k=3)
    want = ref.token_logprobs(x, t, 3)
    ref.assert_within(host(got.logprob), *want["logprob"])
    assert torch.equal(host(got.top_ids), want["top_ids"])
    gl = torch.ones(2)
    capi.token_logprobs_backward(dev(gl), None, rows, dev(t), got.row_max, got.row_sum, out=rows)
    ref.assert_within(host(rows.contiguous()), *ref.token_logprobs_backward(gl, None, x, t))
    q, _, pos, inv_freq, _, wq, _, _, _ = rope_inputs(1, 2, 2, 0, 64, 64, 1, F16, "dense", I64)
    cache = buf.as_strided((1, 2, 2, 64), (4 * far, far, 128, 1))
    capi.norm_rope(dev(q), None, dev(pos), dev(inv_freq), dev(wq), q_out=cache)
    ref.assert_within(host(cache.contiguous()), *ref.norm_rope(q, pos, inv_freq, wq))
    y = capi.dropout(rows, 0.5, 3, out=rows)
    keep = ref.keep_mask(6000, 0.5, 3, 0).view(2, 3000)
    assert bool((host(y.contiguous())[~keep] == 0).all())
    del buf, rows, cache, y
    torch.webgpu.empty_cache()


def test_token_logprobs_gradient_in_place_and_into_padded_rows():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(5, 1003, generator=g).to(BF16)
    t = torch.randint(0, 1003, (5,), generator=g)
    gl = torch.randn(5, generator=g)
    xd, td = dev(x), dev(t)
    got = capi.token_logprobs(xd, td)
    apart = host(capi.token_logprobs_backward(dev(gl), None, xd, td, got.row_max, got.row_sum))
    wide = dev(torch.full((5, 1100), 3.0, dtype=BF16))
    capi.token_logprobs_backward(dev(gl), None, xd, td, got.row_max, got.row_sum, out=wide[:, 1:1004])
    back = host(wide)
    assert torch.equal(back[:, 1:1004], apart) and bool((back[:, 0] == 3).all()) and bool((back[:, 1004:] == 3).all())
    capi.token_logprobs_backward(dev(gl), None, xd, td, got.row_max, got.row_sum, out=xd)
    assert torch.equal(host(xd), apart)


def test_token_logprobs_gradient_against_differences():
    g = torch.Generator().manual_seed(6)
    x, v = torch.randn(2, 50, generator=g), torch.randn(2, 50, generator=g).double()
    t, gl, gh, h = torch.tensor([3, 49]), torch.tensor([1.0, -0.5]), torch.tensor([0.3, 0.8]), 1e-5
    got = capi.token_logprobs(dev(x), dev(t), scale=0.8)
    grad = host(capi.token_logprobs_backward(dev(gl), dev(gh), dev(x), dev(t), got.row_max, got.row_sum, got.entropy, scale=0.8))

    def loss(s):
        f = ref.token_logprobs(x.double() + s * v, t, 0, 0.8)
        return float((f["logprob"][0] * gl.double() + f["entropy"][0] * gh.double()).sum())

    along = float((grad.double() * v).sum())
    room = 2.0 ** -52 * 40 / h + 100 * ref.U * float((grad.double() * v).abs().sum()) + 1e-7
    assert abs((loss(h) - loss(-h)) / (2 * h) - along) <= room


# -------------------------------------------------------------------------------- dropout

@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 1000), (5, 7, 33), (2, 64, 128)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(shape, dtype, p):
    g = torch.Generator().manual_seed(len(shape))
    x, r = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)
    seed, offset = 0x123456789ABCDEF1, (1 << 33) + 5
    for res in (None, r):
        got = host(capi.dropout(dev(x), p, seed, offset, residual=dev(res)))
        want, bound = ref.dropout(x, p, seed, offset, res)
        ref.assert_within(got, want, bound)
        if res is None:
            assert torch.equal(got == 0, want == 0)


def test_dropout_mask_goes_by_logical_index():
    """the mask of a tensor does not depend on how x, the residual or the result are stored"""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(6, 40, 24, generator=g)
    want, bound = ref.dropout(x, 0.3, 11, 2, x)
    for how in (lambda t: t, lambda t: t.transpose(0, 2).contiguous().transpose(0, 2),
                lambda t: torch.nn.functional.pad(t, (1, 2))[..., 1:-2], lambda t: t.flip(0).contiguous().flip(0)):
        for out in (None, torch.empty(24, 6, 40).permute(1, 2, 0), torch.empty(6, 40, 26)[..., 1:25]):
            got = capi.dropout(dev(how(x)), 0.3, 11, 2, residual=dev(x), out=dev(out))
            ref.assert_within(host(got), want, bound)
    flat = dev(torch.cat((torch.zeros(1), x.flatten())))[1:]  # dense, off its alignment
    want_flat, bound_flat = ref.dropout(x.flatten(), 0.3, 11, 2)
    ref.assert_within(host(capi.dropout(flat, 0.3, 11, 2)), want_flat, bound_flat)
    ref.assert_within(host(capi.dropout(flat, 0.3, 11, 2, out=flat)), want_flat, bound_flat)
    wide = dev(torch.full((6, 40, 26), 5.0))
    capi.dropout(dev(x), 0.3, 11, 2, residual=dev(x), out=wide[..., 1:25])
    back = host(wide)
    ref.assert_within(back[..., 1:25], want, bound)
    assert bool((back[..., 0] == 5).all()) and bool((back[..., 25] == 5).all())


def test_dropout_of_special_values_and_broadcast_residual():
    x = torch.tensor([math.inf, math.nan, -math.inf, 1.0] * 64)
    keep = ref.keep_mask(256, 0.5, 77, 0)
    got = host(capi.dropout(dev(x), 0.5, 77))
    assert bool((got[~keep] == 0).all())  # dropped, whatever was there
    assert torch.equal(torch.isnan(got), torch.isnan(x) & keep) and torch.equal(torch.isinf(got), torch.isinf(x) & keep)
    x, r = torch.randn(9, 50), torch.randn(1, 50).expand(9, 50)
    want, bound = ref.dropout(x, 0.2, 5, 0, r)
    ref.assert_within(host(capi.dropout(dev(x), 0.2, 5, residual=dev(r[:1]).expand(9, 50))), want, bound)


def test_dropout_backward_finds_the_same_elements_and_the_rate_is_p():
    n = 1 << 20
    ones = dev(torch.ones(n))
    y = host(capi.dropout(ones, 0.1, 42, 7))
    g = host(capi.dropout(ones, 0.1, 42, 7))
    assert torch.equal(y, g)
    kept = float((y != 0).double().mean())
    # binomial: 6 standard deviations of sqrt(p (1 - p) / n), and p's rounding
    assert abs(kept - 0.9) < 6 * math.sqrt(0.09 / n) + 2.0 ** -17
    other = host(capi.dropout(ones, 0.1, 42, 8))
    both = float(((y != 0) & (other != 0)).double().mean())
    assert abs(both - 0.81) < 6 * math.sqrt(0.81 * 0.19 / n) + 2.0 ** -15


# -------------------------------------------------------- streams, other devices, graphs

def test_on_torchs_streams_between_its_own_kernels():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(64, 4000, generator=g)
    t = torch.randint(0, 4000, (64,), generator=g)
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            a = torch.zeros(64, 4000, device="cuda")
            for _ in range(40):
                a = a + 0.025 * x.cuda()
            got = capi.token_logprobs(a, t.cuda(), top_k=5)
            twice = got.logprob * 2
        stream.synchronize()
        want = ref.token_logprobs(a.cpu(), t, 5)
        ref.assert_within(got.logprob.cpu(), *want["logprob"])
        assert torch.equal(got.top_ids.cpu(), want["top_ids"]) and torch.equal(twice.cpu(), got.logprob.cpu() * 2)


def test_captured_and_replayed_with_new_inputs():
    g = torch.Generator().manual_seed(8)
    q, k, pos, inv_freq, _, wq, wk, dq, dk = (None if t is None else t.cuda() if torch.is_tensor(t) else t for t in
                                              rope_inputs(2, 9, 4, 2, 64, 64, 1, BF16, "packed", I64))
    x = torch.randn(3, 50000, generator=g).cuda()
    t = torch.randint(0, 50000, (3,), generator=g).cuda()
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    gl, gh = torch.ones(3, device="cuda"), torch.full((3,), 0.1, device="cuda")

    def all_of_it():
        rot = capi.norm_rope(q, k, pos, inv_freq, wq, wk)
        back = capi.norm_rope_backward(dq, dk, q, k, pos, inv_freq, wq, wk)
        lp = capi.token_logprobs(x, t, top_k=20)
        grad = capi.token_logprobs_backward(gl, gh, x, t, lp.row_max, lp.row_sum, lp.entropy)
        drop = capi.dropout(x, 0.2, 99, residual=x, d_offset=step)
        return [*rot, *back, *lp, grad, drop]

    all_of_it()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = all_of_it()
    for replay in range(4):
        with torch.no_grad():
            for v in (q, k, dq, dk, x):
                v.copy_(torch.randn(v.shape, generator=g).to(v.dtype))
            pos.add_(17)
            t.copy_(torch.randint(0, 50000, (3,), generator=g))
            step.fill_(replay)
        graph.replay()
        torch.cuda.synchronize()
        eager = all_of_it()
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b)
