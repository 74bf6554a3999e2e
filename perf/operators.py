"""Cases of the transformer-step operators, their plain forms and their definition in 64 bits.

norm_rope         RMS norm of each query and key head and the rotation by position, one or several
                  position axes, forward and backward
token_logprobs    log probability of a given token per row of logits, entropy, top alternatives,
                  and the gradient with respect to the logits
dropout           counter-based dropout, with or without the residual that it is added to
"""
import math
import sys

import torch

own = False

BF16, F16, F32 = "bfloat16", "float16", "float32"
IGNORE = -100
_PHILOX_M = (0xD2511F53, 0xCD9E8D57)
_PHILOX_W = (0x9E3779B9, 0xBB67AE85)
_MASK32 = 0xFFFFFFFF


# ------------------------------------------------------------------------------- cases

def _rope(name, **kw):
    case = {"name": name, "op": "norm_rope", "dir": "forward", "batch": 1, "tokens": 1, "q_heads": 32,
            "k_heads": 8, "head_dim": 128, "rot_dim": 128, "axes": 1, "norm": True, "adjacent": False,
            "layout": "packed", "dtype": BF16, "far": 0}
    case.update(kw)
    return case


def _logprobs(name, **kw):
    case = {"name": name, "op": "token_logprobs", "dir": "forward", "rows": 1, "vocab": 32768, "top_k": 0,
            "scale": 1.0, "masked": 0.0, "ignored": 0.0, "dtype": BF16}
    case.update(kw)
    return case


def _dropout(name, **kw):
    case = {"name": name, "op": "dropout", "rows": 1, "cols": 1024, "p": 0.1, "residual": False,
            "dtype": BF16, "offset": 3}
    case.update(kw)
    return case


def listed():
    return [
        # one new token of 64 sequences, deep into their contexts: latency
        _rope("rope_step_64_sequences", batch=64, far=1000000),
        # a prompt, queries and keys as views of the packed projection
        _rope("rope_prompt_4096", tokens=4096),
        # video patches: three axes, no norm, neighbouring pairs, ragged patch count, heads first
        _rope("rope_video_3_axes", batch=2, tokens=7921, q_heads=16, k_heads=16, head_dim=80, rot_dim=80,
              axes=3, norm=False, adjacent=True, layout="heads_first", dtype=F16),
        # the training step's backward pass of the prompt shape, with the norms' weight gradients
        _rope("rope_train_backward", dir="backward", batch=4, tokens=4096),
        # image patches in float32, two axes, part of the head rotated
        _rope("rope_image_backward_f32", dir="backward", batch=3, tokens=1025, q_heads=12, k_heads=12,
              head_dim=64, rot_dim=48, axes=2, layout="heads_first", dtype=F32),
        # one sampling step: one row, temperature, 20 alternatives
        _logprobs("logprobs_next_token", rows=1, vocab=131072, top_k=20, scale=1.25, dtype=F32),
        # scoring prompts with 5 alternatives per token
        _logprobs("logprobs_score_4096", rows=4096, vocab=131072, top_k=5),
        # an odd vocabulary under a grammar's mask: a third of the columns -inf, one row empty
        _logprobs("logprobs_masked_odd", rows=517, vocab=50257, top_k=20, masked=0.3, dtype=F16),
        # the loss's backward pass, prompt tokens ignored
        _logprobs("logprobs_backward", dir="backward", rows=2048, vocab=151643, ignored=0.25),
        # a few tokens' hidden states
        _dropout("dropout_small", rows=7, cols=1000, dtype=F32),
        # the residual path of a training step
        _dropout("dropout_residual_bf16", rows=32768, cols=4096, residual=True),
        # one large float32 activation
        _dropout("dropout_f32", rows=16384, cols=16384, p=0.25, dtype=F32),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "norm_rope", "token_logprobs", "token_logprobs", "dropout"])
    dtype = rng.choice([BF16, BF16, F16, F32])
    if op == "norm_rope":
        head_dim = rng.choice([32, 34, 48, 64, 64, 72, 80, 96, 128, 128, 128, 160, 192, 256])
        rot_dim = head_dim if rng.random() < 0.7 else 2 * rng.randint(1, head_dim // 2)
        k_heads = rng.choice([1, 2, 4, 8, 12])
        q_heads = k_heads * rng.choice([1, 2, 4, 5])
        per_token = (q_heads + k_heads) * head_dim
        tokens_all = _log_int(rng, 1, max(1, 80000000 // per_token))
        batch = rng.randint(1, min(tokens_all, 8)) if rng.random() < 0.7 else tokens_all
        batch = min(batch, 256)
        axes = rng.choice([1, 1, 2, 3])
        case = _rope("", dir=rng.choice(["forward", "backward"]), batch=batch, tokens=max(1, tokens_all // batch),
                     q_heads=q_heads, k_heads=k_heads, head_dim=head_dim, rot_dim=rot_dim,
                     axes=min(axes, rot_dim // 2), norm=rng.random() < 0.6, adjacent=rng.random() < 0.4,
                     layout=rng.choice(["packed", "heads_first"]), dtype=dtype,
                     far=rng.choice([0, 0, 1000, 1000000]))
    elif op == "token_logprobs":
        vocab = _log_int(rng, 50, 152000)
        rows = _log_int(rng, 1, max(1, min(8192, 300000000 // vocab)))
        case = _logprobs("", dir=rng.choice(["forward", "forward", "backward"]), rows=rows, vocab=vocab,
                         top_k=rng.choice([0, 1, 5, 20, 33]), scale=rng.choice([1.0, 1.0, 0.7, 1.25]),
                         masked=rng.choice([0.0, 0.0, 0.3]), ignored=rng.choice([0.0, 0.25]), dtype=dtype)
    else:
        cols = _log_int(rng, 64, 16384)
        rows = _log_int(rng, 1, max(1, 130000000 // cols))
        case = _dropout("", rows=rows, cols=cols, p=rng.choice([0.0, 0.05, 0.1, 0.25, 0.5]),
                        residual=rng.random() < 0.5, dtype=dtype, offset=rng.randint(0, 1 << 40))
    del case["name"]
    return case


# ------------------------------------------------------------------------------ inputs

def _sections(pairs, axes):
    """pairs of a head dealt to the axes in consecutive runs, the first axis the shortest"""
    first = pairs if axes == 1 else max(1, pairs // (axes + 1))
    rest = [0] * first
    for i in range(pairs - first):
        rest.append(1 + i * (axes - 1) // (pairs - first))
    return rest


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, case["dtype"])

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    s = {"case": dict(case)}
    if case["op"] == "norm_rope":
        B, T, D = case["batch"], case["tokens"], case["head_dim"]
        Hq, Hk, pairs, axes = case["q_heads"], case["k_heads"], case["rot_dim"] // 2, case["axes"]

        def heads():
            if case["layout"] == "packed":
                x = randn(B, T, Hq + 2 * Hk, D).to(dt)
                return x[:, :, :Hq], x[:, :, Hq:Hq + Hk]
            return (randn(B, Hq, T, D).to(dt).transpose(1, 2), randn(B, Hk, T, D).to(dt).transpose(1, 2))

        s["q"], s["k"] = heads()
        if case["dir"] == "backward":
            s["dq"] = randn(B, T, Hq, D).to(dt)
            s["dk"] = randn(B, T, Hk, D).to(dt)
        s["wq"] = (1 + 0.2 * randn(D)).to(dt) if case["norm"] else None
        s["wk"] = (1 + 0.2 * randn(D)).to(dt) if case["norm"] else None
        s["eps"] = 1e-6 if case["norm"] else None
        # positions: running from a start of its own for each sequence; further axes walk a grid
        start = torch.randint(0, case["far"] + 1, (B, 1), device="cuda", generator=g)
        t = torch.arange(T, device="cuda")
        side = max(1, int(math.isqrt(T)))
        walk = [t, t // side, t % side][:axes] if axes > 1 else [t]
        s["positions"] = torch.stack([w + start for w in walk]).contiguous()  # [axes, B, T], int64
        s["inv_freq"] = (10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)).float()
        s["pair_axis"] = bytes(_sections(pairs, axes)) if axes > 1 else None
        s["pair_axis_dev"] = torch.tensor(_sections(pairs, axes), device="cuda")
    elif case["op"] == "token_logprobs":
        R, V = case["rows"], case["vocab"]
        x = randn(R, V).mul_(2.5).to(dt)
        if case["masked"]:
            x.masked_fill_(torch.rand(R, V, device="cuda", generator=g) < case["masked"], -math.inf)
            x[R // 2] = -math.inf
        s["logits"] = x
        t = torch.randint(0, V, (R,), device="cuda", generator=g)
        if case["ignored"]:
            t = torch.where(torch.rand(R, device="cuda", generator=g) < case["ignored"], IGNORE, t)
        s["targets"] = t
        if case["dir"] == "backward":
            # what the forward pass handed over: the row's maximum, sum and entropy
            c = case["scale"]
            m = x.float().amax(1)
            y = torch.where(torch.isneginf(x), -math.inf, c * (x.float() - m[:, None]))
            e = torch.exp(y)
            s["row_max"], s["row_sum"] = m, e.sum(1)
            ey = torch.where(e > 0, e * y, 0.0).sum(1)
            s["entropy"] = torch.where(s["row_sum"] > 0, torch.log(s["row_sum"]) - ey / s["row_sum"], 0.0)
            s["g_logprob"] = torch.where(t == IGNORE, 0.0, -(0.5 + torch.rand(R, device="cuda", generator=g)))
            s["g_entropy"] = torch.where(t == IGNORE, 0.0, torch.full((R,), 0.01, device="cuda"))
    else:
        s["x"] = randn(case["rows"], case["cols"]).to(dt)
        s["residual"] = randn(case["rows"], case["cols"]).to(dt) if case["residual"] else None
        s["seed"] = int(torch.randint(0, 1 << 62, (1,), generator=torch.Generator().manual_seed(seed)))
    return s


def work(case):
    size = 4 if case["dtype"] == F32 else 2
    if case["op"] == "norm_rope":
        n = case["batch"] * case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["head_dim"]
        small = 8 * case["axes"] * case["batch"] * case["tokens"]
        back = case["dir"] == "backward"
        return {"bytes": n * size * (3 if back else 2) + small, "flops": n * (14 if back else 7)}
    if case["op"] == "token_logprobs":
        n = case["rows"] * case["vocab"]
        if case["dir"] == "backward":  # rows whose incoming gradients are 0 need not be read
            return {"bytes": int(n * size * (2 - case["ignored"])) + 32 * case["rows"], "flops": n * 5}
        return {"bytes": n * size + case["rows"] * (24 + 12 * min(case["top_k"], case["vocab"])), "flops": n * 5}
    n = case["rows"] * case["cols"]
    return {"bytes": n * size * (3 if case["residual"] else 2), "flops": n * 2}


# --------------------------------------------------------------------------- plain forms

def _tables(s):
    """cos and sin of each token's angles, [B, T, 1, pairs]"""
    pos = s["positions"][s["pair_axis_dev"]].permute(1, 2, 0).double()
    angle = pos * s["inv_freq"].double()
    return angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]


def _rotate(x, cos, sin, rot, adjacent):
    """x rotated pair by pair, float32 [B, T, H, D]"""
    r, rest = x[..., :rot], x[..., rot:]
    if adjacent:
        lo, hi = r[..., 0::2], r[..., 1::2]
        turned = torch.stack((lo * cos - hi * sin, hi * cos + lo * sin), -1).flatten(-2)
    else:
        lo, hi = r[..., :rot // 2], r[..., rot // 2:]
        turned = torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1)
    return torch.cat((turned, rest), -1)


def _plain_rope(s, x, w, cos, sin):
    z = x.float()
    if s["eps"] is not None:
        z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + s["eps"]) * w.float()
    return _rotate(z, cos, sin, s["case"]["rot_dim"], s["case"]["adjacent"]).to(x.dtype)


def _plain_rope_backward(s, dy, x, w, cos, sin):
    dz = _rotate(dy.float(), cos, -sin, s["case"]["rot_dim"], s["case"]["adjacent"])
    if s["eps"] is None:
        return dz.to(x.dtype), None
    z = x.float()
    r = torch.rsqrt((z * z).mean(-1, keepdim=True) + s["eps"])
    u = z * r
    gw = dz * w.float()
    dx = r * (gw - u * (gw * u).mean(-1, keepdim=True))
    return dx.to(x.dtype), (dz * u).sum((0, 1, 2)).to(w.dtype)


def _plain_logprobs(s):
    c, k = s["case"]["scale"], min(s["case"]["top_k"], s["case"]["vocab"])
    x = s["logits"].float()
    m = x.amax(1)
    d = torch.where(torch.isneginf(x), -math.inf, c * (x - m[:, None]))
    e = torch.exp(d)
    total = e.sum(1)
    log_s = torch.log(total)
    entropy = torch.where(total > 0, log_s - torch.where(e > 0, e * d, 0.0).sum(1) / total, 0.0)
    t = s["targets"]
    lp = torch.gather(d, 1, t.clamp(min=0)[:, None])[:, 0] - log_s
    lp = torch.where(t == IGNORE, 0.0, torch.where(total > 0, lp, -math.inf))
    # ids by value, the lowest first among equals: one whole-number key for both
    bits = x.view(torch.int32).long()
    V = x.shape[1]
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) + (V - 1 - torch.arange(V, device=x.device))
    ids = V - 1 - (torch.topk(key, k, 1).values & ((1 << 20) - 1))
    top = torch.where(total[:, None] > 0, torch.gather(d, 1, ids) - log_s[:, None], -math.inf)
    return lp, entropy, m, total, top, ids


def _plain_logprobs_backward(s):
    c = s["case"]["scale"]
    x, t = s["logits"].float(), s["targets"]
    d = torch.where(torch.isneginf(x), -math.inf, c * (x - s["row_max"][:, None]))
    p = torch.where(s["row_sum"][:, None] > 0, torch.exp(d) / s["row_sum"][:, None], 0.0)
    g_lp = torch.where(t == IGNORE, 0.0, s["g_logprob"])
    shift = (s["entropy"] - torch.log(s["row_sum"]))[:, None]
    grad = -g_lp[:, None] * p - s["g_entropy"][:, None] * torch.where(p > 0, p * (d + shift), 0.0)
    alive = (s["row_sum"] > 0) & (t != IGNORE)
    grad.scatter_add_(1, t.clamp(min=0)[:, None], torch.where(alive, g_lp, 0.0)[:, None])
    return (grad * c).to(s["logits"].dtype)


def _words(blocks, offset, seed):
    """Philox4x32-10 of the counters (block, offset): four 32-bit words for each block, [blocks, 4]"""
    b = torch.arange(blocks, device="cuda")
    c0, c1 = b & _MASK32, b >> 32
    c2, c3 = torch.full_like(b, offset & _MASK32), torch.full_like(b, offset >> 32)
    k0, k1 = seed & _MASK32, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * _PHILOX_M[0], c2 * _PHILOX_M[1]
        c0, c1, c2, c3 = (((p1 >> 32) & _MASK32) ^ c1 ^ k0, p1 & _MASK32,
                          ((p0 >> 32) & _MASK32) ^ c3 ^ k1, p0 & _MASK32)
        k0, k1 = (k0 + _PHILOX_W[0]) & _MASK32, (k1 + _PHILOX_W[1]) & _MASK32
    return torch.stack((c0, c1, c2, c3), 1)


def _plain_dropout(s):
    x = s["x"]
    n = x.numel()
    threshold = int(s["case"]["p"] * 65536 + 0.5)
    w = _words((n + 7) // 8, s["case"]["offset"], s["seed"])
    draws = torch.stack((w & 0xFFFF, w >> 16), -1).flatten()[:n].view_as(x)
    y = torch.where(draws >= threshold, x.float() * (65536.0 / (65536 - threshold)), 0.0)
    if s["residual"] is not None:
        y = s["residual"].float() + y
    return y.to(x.dtype)


# ---------------------------------------------------------------------------------- run

def _run_own(s):
    if "torch-webgpu_amd" not in sys.path:
        sys.path.insert(0, "torch-webgpu_amd")
    import twg_capi as capi

    case = s["case"]
    if case["op"] == "norm_rope":
        how = dict(q_weight=s["wq"], k_weight=s["wk"], eps=s["eps"], pair_axis=s["pair_axis"],
                   adjacent=case["adjacent"])
        if case["dir"] == "forward":
            return list(capi.norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], **how))
        grads = capi.norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["positions"], s["inv_freq"], **how)
        return [g for g in grads if g is not None]
    if case["op"] == "token_logprobs":
        if case["dir"] == "forward":
            return list(capi.token_logprobs(s["logits"], s["targets"], top_k=min(case["top_k"], case["vocab"]),
                                            scale=case["scale"], ignore_index=IGNORE))
        return capi.token_logprobs_backward(s["g_logprob"], s["g_entropy"], s["logits"], s["targets"], s["row_max"],
                                            s["row_sum"], s["entropy"], scale=case["scale"], ignore_index=IGNORE)
    return capi.dropout(s["x"], case["p"], seed=s["seed"], offset=case["offset"], residual=s["residual"])


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    if case["op"] == "norm_rope":
        cos, sin = _tables(s)
        if case["dir"] == "forward":
            return [_plain_rope(s, s["q"], s["wq"], cos, sin), _plain_rope(s, s["k"], s["wk"], cos, sin)]
        gq, gwq = _plain_rope_backward(s, s["dq"], s["q"], s["wq"], cos, sin)
        gk, gwk = _plain_rope_backward(s, s["dk"], s["k"], s["wk"], cos, sin)
        return [g for g in (gq, gk, gwq, gwk) if g is not None]
    if case["op"] == "token_logprobs":
        return list(_plain_logprobs(s)) if case["dir"] == "forward" else _plain_logprobs_backward(s)
    return _plain_dropout(s)


# -------------------------------------------------------------------------------- exact

def _exact_rope(s, which):
    """Each pair as a complex number turned by e^(i a), the norm as a quotient by the root mean square."""
    case, rot = s["case"], s["case"]["rot_dim"]
    x = s[which].double()
    w = None if s["w" + which] is None else s["w" + which].double()
    axis = [0] * (rot // 2) if s["pair_axis"] is None else list(s["pair_axis"])
    angle = torch.stack([s["positions"][a].double() * float(f) for a, f in zip(axis, s["inv_freq"].tolist())], -1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, :, None]

    def spin(z, by):
        out = z.clone()
        lo = slice(0, rot, 2) if case["adjacent"] else slice(0, rot // 2)
        hi = slice(1, rot, 2) if case["adjacent"] else slice(rot // 2, rot)
        v = torch.complex(z[..., lo].contiguous(), z[..., hi].contiguous()) * by
        out[..., lo], out[..., hi] = v.real, v.imag
        return out

    rms = None if s["eps"] is None else (x.square().sum(-1, keepdim=True) / x.shape[-1] + s["eps"]).sqrt()
    if case["dir"] == "forward":
        return spin(x if rms is None else x / rms * w, turn), None
    dz = spin(s["d" + which].double(), turn.conj())
    if rms is None:
        return dz, None
    # dx from z_j = w_j x_j / rms: dz_j w_j / rms - x_j (sum_i dz_i w_i x_i) / (D rms^3)
    gw = dz * w
    dx = gw / rms - x * (gw * x).sum(-1, keepdim=True) / (x.shape[-1] * rms ** 3)
    return dx, (dz * x / rms).sum((0, 1, 2))


def _exact_logprobs(s):
    case, c = s["case"], s["case"]["scale"]
    k, V = min(case["top_k"], case["vocab"]), case["vocab"]
    rows = []
    for x, t in zip(s["logits"].split(256), s["targets"].split(256)):
        x = x.double()
        z = x * c
        lse = torch.logsumexp(z, 1)
        empty = torch.isneginf(lse)
        lp = z - lse[:, None]
        h = -torch.special.xlogy(lp.exp(), lp.exp()).sum(1)
        # values in descending order, equal ones in the order of their ids
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
        at = lp[torch.arange(len(t), device=x.device), t.clamp(min=0)]
        at = torch.where(empty, -math.inf, at).masked_fill(t == IGNORE, 0.0)
        top = lp.gather(1, order).masked_fill(empty[:, None], -math.inf)
        m = x.max(1).values
        total = torch.where(empty, 0.0, torch.exp(lse - c * m))
        rows.append((at, h.masked_fill(empty, 0.0), m, total, top, order))
    return [torch.cat(v) for v in zip(*rows)]


def _exact_logprobs_backward(s):
    c = s["case"]["scale"]
    m, total, h = s["row_max"].double(), s["row_sum"].double(), s["entropy"].double()
    out = []
    for r in range(0, len(m), 256):
        x, t = s["logits"][r:r + 256].double(), s["targets"][r:r + 256]
        part = slice(r, r + 256)
        lse = c * m[part] + total[part].log()
        lp = x * c - lse[:, None]
        p = lp.exp()
        hit = torch.arange(x.shape[1], device=x.device) == t[:, None]
        g = torch.where(t == IGNORE, 0.0, s["g_logprob"][part].double())[:, None]
        grad = g * (hit.double() - p) - s["g_entropy"][part].double()[:, None] * (
            torch.special.xlogy(p, p) + p * h[part][:, None])
        out.append(torch.where(total[part][:, None] > 0, grad * c, 0.0))
    return torch.cat(out)


def _exact_dropout(s):
    """The generator on 16-bit limbs, so that no product leaves 63 bits; a block of elements at a time."""
    x, case = s["x"].flatten(), s["case"]
    low = 0xFFFF

    def product(a, m):
        m0, m1 = m & low, m >> 16
        a0, a1 = a & low, a >> 16
        mid = a1 * m0 + ((a0 * m0) >> 16)
        mid2 = a0 * m1 + (mid & low)
        return a1 * m1 + (mid >> 16) + (mid2 >> 16), ((mid2 & low) << 16) | ((a0 * m0) & low)

    drop = math.floor(case["p"] * 65536 + 0.5)
    scale = 65536 / (65536 - drop)
    out = torch.empty(x.numel(), dtype=torch.float64, device=x.device)
    step = 1 << 25
    for first in range(0, x.numel(), step):
        n = min(step, x.numel() - first)
        b = torch.arange(first // 8, (first + n + 7) // 8, device=x.device)
        ctr = [b % 2**32, b // 2**32, torch.full_like(b, case["offset"] % 2**32), torch.full_like(b, case["offset"] // 2**32)]
        for r in range(10):
            key = [(s["seed"] // 2**(32 * i) % 2**32 + r * _PHILOX_W[i]) % 2**32 for i in range(2)]
            h0, l0 = product(ctr[0], _PHILOX_M[0])
            h1, l1 = product(ctr[2], _PHILOX_M[1])
            ctr = [h1 ^ ctr[1] ^ key[0], l1, h0 ^ ctr[3] ^ key[1], l0]
        bits = torch.stack([v for word in ctr for v in (word % 65536, word // 65536)], 1).reshape(-1)[:n]
        part = x[first:first + n].double() * scale
        part[bits < drop] = 0.0
        if s["residual"] is not None:
            part += s["residual"].flatten()[first:first + n].double()
        out[first:first + n] = part
    return out.view_as(s["x"])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm_rope":
        (a, wa), (b, wb) = _exact_rope(s, "q"), _exact_rope(s, "k")
        return [v for v in (a, b, wa, wb) if v is not None]
    if case["op"] == "token_logprobs":
        return _exact_logprobs(s) if case["dir"] == "forward" else _exact_logprobs_backward(s)
    return _exact_dropout(s)
