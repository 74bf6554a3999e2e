"""The transformer-step operators in float64 on the CPU, from their definitions, and the bounds
their binary32 kernels are held to.

U = 2^-24 is half a step of binary32; a result of type t is off by another eps(t) / 2 of itself for
its one rounding.  Every bound counts roundings and multiplies them by the magnitudes they act on."""
import math

import torch

U = 2.0 ** -24


def rounding(dtype, y):
    """What one rounding to dtype is off by at most: half a step, eps / 2 relative for normal
    numbers.  Below the smallest normal number the step stays what it is there, so half of it,
    tiny * eps / 2 (2^-14 * 2^-11 = 2^-25 for float16), bounds the rounding of every smaller y."""
    f = torch.finfo(dtype)
    return f.eps / 2 * y.abs() + f.tiny * f.eps / 2


# -------------------------------------------------------------------------- norm_rope

def _angles(positions, inv_freq, pair_axis, B, T):
    pos = positions.double()
    pos = pos.expand(1, B, T) if pos.dim() < 3 else pos.expand(pos.shape[0], B, T)
    axis = list(pair_axis) if pair_axis is not None else [0] * len(inv_freq)
    if not axis:
        return torch.zeros(B, T, 1, 0, dtype=torch.float64)
    return torch.stack([pos[a] * f for a, f in zip(axis, inv_freq.double())], -1)[:, :, None]


def _turn(z, angle, rot, adjacent):
    """The rotated heads and, for each element, the sum of the magnitudes of its pair."""
    out, mag = z.clone(), z.abs()
    lo = slice(0, rot, 2) if adjacent else slice(0, rot // 2)
    hi = slice(1, rot, 2) if adjacent else slice(rot // 2, rot)
    c, s = angle.cos(), angle.sin()
    out[..., lo] = z[..., lo] * c - z[..., hi] * s
    out[..., hi] = z[..., hi] * c + z[..., lo] * s
    mag[..., lo] = mag[..., hi] = z[..., lo].abs() + z[..., hi].abs()
    return out, mag


def norm_rope(x, positions, inv_freq, weight=None, eps=1e-6, pair_axis=None, adjacent=False):
    """(result, bound) for one of the two tensors.

    Roundings that meet an element of z: the sum of squares (a chain of at most 16 products a
    lane and 6 joins; its relative error is halved by the square root), root and quotient, two
    products: 16.  The rotation: sine and cosine within 4 U (the angle's rounding, pi/2 U, and the
    function's own), a product and a sum: 7 more.  32 U of |lo| + |hi| covers them."""
    B, T, _, D = x.shape
    z = x.double()
    if eps is not None:
        z = z / torch.sqrt(z.square().mean(-1, keepdim=True) + eps)
        if weight is not None:
            z = z * weight.double()
    y, mag = _turn(z, _angles(positions, inv_freq, pair_axis, B, T), 2 * len(inv_freq), adjacent)
    return y, 32 * U * mag + rounding(x.dtype, y)


def norm_rope_backward(dy, x, positions, inv_freq, weight=None, eps=1e-6, pair_axis=None, adjacent=False):
    """(dx, bound, dweight, bound).  dx = r (g - u mean(g u)): 32 U on g as above, twice that on the
    mean's products and its sum; dw: the same 64 U on each product, and a chain of at most
    as many additions as there are heads."""
    B, T, H, D = x.shape
    dz, mag = _turn(dy.double(), -_angles(positions, inv_freq, pair_axis, B, T), 2 * len(inv_freq), adjacent)
    if eps is None:
        return dz, 32 * U * mag + rounding(x.dtype, dz), None, None
    xd = x.double()
    r = 1 / torch.sqrt(xd.square().mean(-1, keepdim=True) + eps)
    u = xd * r
    w = torch.ones(D, dtype=torch.float64) if weight is None else weight.double()
    g, gm = dz * w, mag * w.abs()
    dx = r * (g - u * (g * u).mean(-1, keepdim=True))
    bound = 96 * U * r * (gm + u.abs() * (gm * u.abs()).mean(-1, keepdim=True)) + rounding(x.dtype, dx)
    dw = (dz * u).sum((0, 1, 2))
    dwb = (64 + B * T * H) * U * (mag * u.abs()).sum((0, 1, 2))
    if weight is not None:
        dwb = dwb + rounding(weight.dtype, dw)
    return dx, bound, dw, dwb


# --------------------------------------------------------------------- token_logprobs

def token_logprobs(logits, targets, top_k=0, scale=1.0, ignore_index=-100):
    """{name: (value, bound)}; ids exact.

    An exponent c (x - m) carries 4 U of itself, an exponential and its addition 4 U, a
    chain of at most vocab / 64 + 32 additions U each; log s and the final difference 4 U."""
    x = logits.double()
    R, V = x.shape
    m = x.amax(1)
    y = torch.where(torch.isneginf(x), torch.full_like(x, -math.inf), scale * (x - m[:, None]))
    e = torch.exp(y)
    s = e.sum(1)
    log_s = torch.log(s)
    ey = torch.where(e > 0, e * y, torch.zeros_like(e))
    mean = -ey.sum(1) / s
    empty = s == 0
    chain = V / 64 + 32
    s_rel = U * (chain + 4 + 4 * mean)
    entropy = torch.where(empty, torch.zeros_like(s), log_s + mean)
    ey2 = torch.where(e > 0, e * y * y, torch.zeros_like(e)).sum(1) / s
    entropy_bound = 2 * s_rel * (1 + mean) + U * (4 * ey2 + 8 * (log_s.abs() + mean + 1))

    def lp_of(yt):
        lp = torch.where(empty.view(-1, *[1] * (yt.dim() - 1)), torch.full_like(yt, -math.inf),
                         yt - log_s.view(-1, *[1] * (yt.dim() - 1)))
        return lp, (s_rel + 8 * U * (1 + log_s.abs())).view(-1, *[1] * (yt.dim() - 1)) + 8 * U * yt.abs()

    t = targets.long()
    inside = (t >= 0) & (t < V)
    lp, lp_bound = lp_of(y.gather(1, t.clamp(0, V - 1)[:, None])[:, 0])
    lp = torch.where(inside, lp, torch.full_like(lp, math.nan))
    lp = torch.where(t == ignore_index, torch.zeros_like(lp), lp)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top_k]
    top, top_bound = lp_of(y.gather(1, ids))

    def single(v, bound):  # beyond binary32's range: its infinities; an empty row's values are exact
        return torch.where(torch.isinf(v.float()), v.float().double(), v), torch.nan_to_num(bound, nan=0.0)

    return {"logprob": single(lp, lp_bound), "entropy": single(entropy, entropy_bound), "row_max": (m, 0 * s),
            "row_sum": single(s, s * s_rel), "top_logprobs": single(top, top_bound), "top_ids": ids}


def token_logprobs_backward(g_logprob, g_entropy, logits, targets, scale=1.0, ignore_index=-100):
    """(grad, bound) by the formula; s_rel as above on p and the entropy."""
    x = logits.double()
    R, V = x.shape
    f = token_logprobs(logits, targets, 0, scale, ignore_index)
    m, s, H = f["row_max"][0], f["row_sum"][0], f["entropy"][0]
    gl = torch.zeros(R, dtype=torch.float64) if g_logprob is None else g_logprob.double()
    gh = torch.zeros(R, dtype=torch.float64) if g_entropy is None else g_entropy.double()
    t = targets.long()
    gl = torch.where(t == ignore_index, torch.zeros_like(gl), gl)
    y = torch.where(torch.isneginf(x), torch.full_like(x, -math.inf), scale * (x - m[:, None]))
    p = torch.where(s[:, None] > 0, torch.exp(y) / s[:, None], torch.zeros_like(y))
    logp = torch.where(p > 0, y - torch.log(s)[:, None], torch.zeros_like(y))
    hit = torch.arange(V)[None] == t[:, None]
    grad = gl[:, None] * (hit.double() - p) - gh[:, None] * p * (logp + H[:, None])
    live = (s > 0) & ((gl != 0) | (gh != 0))
    grad = torch.where(live[:, None], scale * grad, torch.zeros_like(grad))
    y0 = torch.where(p > 0, y.abs(), torch.zeros_like(y))
    rel = U * (V / 64 + 48 + 8 * y0 + 4 * torch.log(s)[:, None].abs())
    mag = gl.abs()[:, None] + gh.abs()[:, None] * (logp.abs() + H[:, None] + 1 + torch.log(s)[:, None].abs())
    bound = scale * (4 * rel * p * mag + 4 * U * gl.abs()[:, None] * hit)
    return grad, torch.nan_to_num(bound) + rounding(logits.dtype, grad)


# ---------------------------------------------------------------------------- dropout

def philox(counter, key):
    """Philox4x32-10 (Salmon et al., SC 2011) on Python integers: four words."""
    c, k = list(counter), list(key)
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def keep_mask(numel, p, seed, offset, first=0):
    """keep or not for elements first .. first + numel - 1, element by element"""
    low = 0xFFFFFFFF
    threshold = math.floor(p * 65536 + 0.5)
    keep, words, block = [], None, None
    for e in range(first, first + numel):
        if e // 8 != block:
            block = e // 8
            words = philox((block & low, block >> 32, offset & low, (offset >> 32) & low), (seed & low, (seed >> 32) & low))
        bits = (words[(e // 2) % 4] >> (16 * (e % 2))) & 0xFFFF
        keep.append(bits >= threshold)
    return torch.tensor(keep, dtype=torch.bool)


def dropout(x, p, seed, offset, residual=None):
    """(result, bound): a product and a sum in binary32, and the rounding."""
    threshold = math.floor(p * 65536 + 0.5)
    scale = 65536 / (65536 - threshold) if threshold < 65536 else 0.0
    keep = keep_mask(x.numel(), p, seed, offset).view(x.shape)
    y = torch.where(keep, x.double() * scale, torch.zeros(x.shape, dtype=torch.float64))
    mag = y.abs()
    if residual is not None:
        y, mag = y + residual.double(), mag + residual.double().abs()
    return y, 4 * U * mag + rounding(x.dtype, y)


# ------------------------------------------------------------------------- comparison

def assert_within(got, want, bound, what=""):
    """|got - want| <= bound, infinities and NaN in the same places"""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN elsewhere"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: infinities differ"
    off = (got - want).abs()[fine] - bound.expand_as(want)[fine]
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 0, f"{what}: {int((off > 0).sum())} of {off.numel()} outside their bound, worst by {worst:.3g}"
