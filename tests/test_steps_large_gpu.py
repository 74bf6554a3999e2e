"""norm_rope, token_logprobs and dropout at sizes where a group of lanes takes one head after another, a
workgroup one piece of work after another, and loads and stores carry the nontemporal hint; on PyTorch-ROCm
tensors, against the float64 definitions of steps_ref.py computed on the GPU, a stretch of tokens at a time.
test_steps_edges.py shows that the sizes do what they are here for."""
import math

import pytest
import torch

import steps_ref as ref
import twg_capi as capi

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def backend():
    capi.load()
    capi.init()
    yield
    torch.cuda.empty_cache()


# ----------------------------------------------------------------------------- norm_rope

# tokens, q heads, k heads, head_dim, rot_dim, axes, adjacent, dtype, elements a head is longer in memory
ROPE = {
    "several heads per group": (8192, 32, 8, 128, 128, 1, False, BF16, 0),
    "several heads, three axes, adjacent": (6001, 16, 16, 80, 80, 3, True, F16, 0),
    "several heads, float32, part rotated": (9001, 12, 3, 64, 48, 2, False, F32, 0),
    "several heads, narrow runs": (3000, 12, 5, 34, 18, 2, False, BF16, 1),
    "several heads, shares of a token": (700, 300, 0, 32, 32, 1, False, F16, 0),
    "several pieces": (100003, 1, 0, 8, 8, 1, False, F32, 0),
    "several pieces, two parts": (40000, 32, 16, 32, 32, 1, True, BF16, 0),
    "several pieces, hinted": (32768, 32, 8, 128, 128, 1, False, BF16, 0),
    "hinted, float32": (16400, 20, 4, 128, 128, 1, False, F32, 0),
}


def heads(g, T, H, D, dtype, longer):
    return torch.randn(1, T, H, D + longer, device="cuda", generator=g).to(dtype)[..., :D] if H else None


@pytest.mark.parametrize("name", ROPE)
def test_norm_rope(name):
    T, Hq, Hk, D, rot, axes, adjacent, dtype, longer = ROPE[name]
    g = torch.Generator(device="cuda").manual_seed(T)
    q, k = heads(g, T, Hq, D, dtype, longer), heads(g, T, Hk, D, dtype, longer)
    pos = torch.randint(0, 1 << 18, (axes, 1, T), device="cuda", generator=g)
    f = (10000.0 ** (-torch.arange(rot // 2, device="cuda").double() / (rot // 2))).float()
    how = dict(pair_axis=[i % axes for i in range(rot // 2)] if axes > 1 else None, adjacent=adjacent)
    wq, wk = (1 + 0.2 * torch.randn(2, D, device="cuda", generator=g))
    got = capi.norm_rope(q, k, pos, f, wq, wk if Hk else None, **how)
    # the result as incoming gradient: what the weights' gradients sum is then positive nearly everywhere,
    # and a head left out or taken twice shows beside the rounding of the sums
    grads = capi.norm_rope_backward(got[0], got[1], q, k, pos, f, wq, wk if Hk else None, **how)
    again = capi.norm_rope_backward(got[0], got[1], q, k, pos, f, wq, wk if Hk else None, **how)
    for a, b in zip(grads, again):  # sums in a fixed order
        assert (a is None and b is None) or torch.equal(a, b)
    for i, (x, w) in enumerate(((q, wq), (k, wk))):
        if x is None:
            continue
        dw, room = torch.zeros(2, D, dtype=torch.float64, device="cuda")
        step = max(1, (1 << 24) // (x.shape[2] * D))
        for t in range(0, T, step):
            part = slice(t, t + step)
            xp, dy, p = x[:, part], got[i][:, part], pos[:, :, part]
            ref.assert_within(dy, *ref.norm_rope(xp, p, f, w, **how), name)
            dx, bound, dwp, _ = ref.norm_rope_backward(dy, xp, p, f, w, **how)
            ref.assert_within(grads[i][:, part], dx, bound, name)
            dw += dwp
            angle = -ref._angles(p, f, how["pair_axis"], 1, xp.shape[1])
            _, mag = ref._turn(dy.double(), angle, rot, adjacent)
            xd = xp.double()
            room += (mag * (xd / torch.sqrt(xd.square().mean(-1, keepdim=True) + 1e-6)).abs()).sum((0, 1, 2))
        # 64 U on each product, and the additions that a product goes through: a lane's heads (at most 16
        # here), 6 joins of lanes, 4 of wavefronts, at most 16 rows of sums in a chain and their tree
        ref.assert_within(grads[2 + i], dw, 128 * ref.U * room + ref.rounding(F32, dw), name)
        del dw, room
    outs = capi.norm_rope(q, k, pos, f, wq, wk if Hk else None, q_out=q, k_out=k, **how)  # in place
    for a, b in zip(outs, got):
        assert (a is None and b is None) or torch.equal(a, b)


# ------------------------------------------------------------------------- token_logprobs

@pytest.mark.parametrize("rows, vocab, dtype", [(700, 40009, BF16), (300, 65536, F32), (2000, 20011, F16)])
def test_gradient_of_logits_beyond_the_caches_share(rows, vocab, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.randn(rows, vocab, device="cuda", generator=g) * 2.5).to(dtype)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    gl, gh = torch.randn(2, rows, device="cuda", generator=g)
    t[::7], gl[::5], gh[::5] = -100, 0.0, 0.0
    got = capi.token_logprobs(x, t, top_k=2)
    grad = torch.full_like(x, math.nan)
    capi.token_logprobs_backward(gl, gh, x, t, got.row_max, got.row_sum, got.entropy, out=grad)
    for r in range(0, rows, 100):
        part = slice(r, r + 100)
        xc, tc = x[part].cpu(), t[part].cpu()
        ref.assert_within(grad[part].cpu(), *ref.token_logprobs_backward(gl[part].cpu(), gh[part].cpu(), xc, tc))
        ref.assert_within(got.logprob[part].cpu(), *ref.token_logprobs(xc, tc)["logprob"])


def test_gradient_of_more_logits_than_one_workgroup_a_stretch():
    """beyond 2^31 threads' worth of logits a workgroup takes several stretches of its row: 2^21 rows of
    16390, all with the same logits (a broadcast input), 69 GB of gradient"""
    rows, vocab = 1 << 21, 16390
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("needs 90 GiB of GPU memory")
    g = torch.Generator(device="cuda").manual_seed(3)
    one = torch.randn(1, vocab, device="cuda", generator=g).to(F16)
    x = one.expand(rows, vocab)
    t = torch.arange(rows, device="cuda") % vocab
    got = capi.token_logprobs(one, t[:1])
    stats = [v.expand(rows).contiguous() for v in (got.row_max, got.row_sum)]
    gl = torch.ones(rows, device="cuda")
    grad = torch.full((rows, vocab), math.nan, dtype=F16, device="cuda")
    capi.token_logprobs_backward(gl, None, x, t, *stats, out=grad)
    p = -torch.softmax(one.double(), 1)[0]
    room = ref.rounding(F16, p) + 4096 * ref.U * p.abs()  # (a chain of vocab / 64 additions, and an exponential's 48 U)
    step = 1 << 15
    for r in range(0, rows, step):
        part = grad[r:r + step].double()
        at = t[r:r + step, None]
        hit = part.gather(1, at)
        part.scatter_(1, at, p[at])
        assert bool(((part - p).abs() <= room).all()), r
        # 1 - p: a step of float16 below 1 is 2^-11, so half of it, and the room of p
        assert bool(((hit - 1 - p[at]).abs() <= 2.0 ** -12 + room[at]).all()), r
    del grad, part
    torch.cuda.empty_cache()


# -------------------------------------------------------------------------------- dropout

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("pitch", [0, 24])
def test_dropout_beyond_the_caches_share(dtype, residual, pitch):
    """pitch: elements between two rows of x (the kernel for rows of whole packs instead of one dense run)"""
    rows, cols, p, seed, offset = 5003, 8200 if pitch else 8203, 0.3, (1 << 61) + 5, 1 << 39
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, cols + pitch, device="cuda", generator=g).to(dtype)[:, :cols]
    r = torch.randn(rows, cols, device="cuda", generator=g).to(dtype) if residual else None
    out = torch.full((rows, cols), math.nan, dtype=dtype, device="cuda")
    capi.dropout(x, p, seed, offset, residual=r, out=out)
    assert not bool(torch.isnan(out).any())
    n = rows * cols
    threshold = math.floor(p * 65536 + 0.5)
    for first in (0, 12345 * 8 + 3, n // 2 + 1, n - 4000):
        keep = ref.keep_mask(4000, p, seed, offset, first).double().cuda()
        at = torch.arange(first, first + 4000, device="cuda")
        want = keep * x[at // cols, at % cols].double() * (65536 / (65536 - threshold))
        mag = want.abs()
        if residual:
            res = r.view(-1)[at].double()
            want, mag = want + res, mag + res.abs()
        ref.assert_within(out.view(-1)[at], want, 4 * ref.U * mag + ref.rounding(dtype, want))
    if not residual:  # binomial: 6 standard deviations, and p's rounding; an element of 0 counts as dropped
        kept = float((out != 0).double().mean()) + float((x == 0).double().mean())
        assert abs(kept - (1 - p)) < 6 * math.sqrt(p * (1 - p) / n) + 2.0 ** -15


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_dropout_of_more_than_2_to_the_32_elements(dtype):
    n, p, seed = (1 << 32) + 4101, 0.5, 17
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GiB of GPU memory")
    x = torch.ones(n, dtype=dtype, device="cuda")
    capi.dropout(x, p, seed, out=x)
    for first in (0, (1 << 31) - 100, (1 << 32) - 2000, n - 4000):
        keep = ref.keep_mask(4000, p, seed, 0, first)
        assert torch.equal(x[first:first + 4000].cpu() != 0, keep)
    del x
    torch.cuda.empty_cache()
