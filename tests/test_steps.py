"""The transformer-step entry points without a GPU: what they refuse, before any device is
touched, the layout of their argument structures, and the oracle's random generator."""
import ctypes
import os
import subprocess

import pytest
import torch

import steps_ref as ref
import twg_capi as capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD, UNSUPPORTED, SMALL, LARGE = -1, -2, -3, -5
P = 1 << 20  # an aligned address that no refused call may touch


def test_argument_structures_match_the_header(tmp_path):
    fields = {capi.RopePart: ("twg_rope_part_t", ["heads", "x", "weight", "x_stride", "out_stride"]),
              capi.NormRope: ("twg_norm_rope_t", ["eps", "batch", "positions", "pos_stride", "inv_freq", "pair_axis", "part"]),
              capi.TokenLogprobsArgs: ("twg_token_logprobs_t", ["rows", "ignore_index", "scale", "top_k", "logprob", "top_ids",
                                                                "g_entropy", "grad", "grad_stride"])}
    lines, want = [], []
    for cls, (name, members) in fields.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for m in members:
            lines.append(f'printf("%zu\\n", offsetof({name}, {m}));')
            want.append(getattr(cls, m).offset)
    c = tmp_path / "layout.c"
    c.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "twg.h"\nint main(){' + "\n".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], check=True, stdout=subprocess.PIPE, text=True).stdout.split()
    assert [int(v) for v in got] == want


# ----------------------------------------------------------------------- norm_rope

def rope(**kw):
    """A call that the library takes, changed by kw."""
    d = capi.NormRope()
    d.dtype, d.weight_dtype, d.position_dtype = capi.DTYPES[torch.bfloat16], capi.DTYPES[torch.float32], capi.DTYPES[torch.int64]
    d.norm, d.eps, d.n_axes, d.head_dim, d.rot_dim = 1, 1e-6, 1, 64, 64
    d.batch, d.tokens, d.positions, d.inv_freq = 2, 5, P, P
    d.pos_stride[:] = 10, 5, 1
    for p in d.part:
        p.heads, p.x, p.dy, p.out = 3, P, P, P
        for st in (p.x_stride, p.dy_stride, p.out_stride):
            st[:] = 5 * 3 * 64, 3 * 64, 64
    for name, v in kw.items():
        at = d
        *path, last = name.split("__")
        for step in path:
            at = at[int(step)] if step.isdigit() else getattr(at, step)
        if last.isdigit():
            at[int(last)] = v
        else:
            setattr(at, last, v)
    return d


@pytest.mark.parametrize("change, code", [
    (dict(dtype=7), BAD), (dict(dtype=-1), BAD), (dict(weight_dtype=3), BAD), (dict(weight_dtype=4), UNSUPPORTED),
    (dict(position_dtype=5), BAD), (dict(head_dim=63), BAD), (dict(head_dim=0), BAD), (dict(head_dim=514), BAD),
    (dict(rot_dim=66), BAD), (dict(rot_dim=-2), BAD), (dict(rot_dim=31), BAD), (dict(n_axes=0), BAD), (dict(n_axes=9), BAD),
    (dict(pair_axis__31=1), BAD), (dict(eps=-1.0), BAD), (dict(eps=float("nan")), BAD), (dict(eps=float("inf")), BAD),
    (dict(batch=-1), BAD), (dict(tokens=-1), BAD), (dict(batch=1 << 40, tokens=1 << 40), BAD),
    (dict(batch=1 << 16, tokens=1 << 16), LARGE), (dict(part__0__heads=-1), BAD), (dict(part__1__heads=1 << 40), BAD),
    (dict(part__0__x=None), BAD), (dict(part__1__out=None), BAD), (dict(part__0__x=P + 1), BAD), (dict(part__0__out=P + 1), BAD),
    (dict(part__0__weight=P + 2), BAD), (dict(positions=None), BAD), (dict(positions=P + 4), BAD), (dict(inv_freq=None), BAD),
    (dict(inv_freq=P + 2), BAD), (dict(part__0__out_stride__0=0), BAD), (dict(part__0__out_stride__1=0), BAD),
    (dict(part__1__out_stride__2=0), BAD),
])
def test_norm_rope_refuses(change, code):
    d, L = rope(**change), capi.load()
    assert L.twg_norm_rope(ctypes.byref(d), None) == code
    assert L.twg_norm_rope_backward(ctypes.byref(d), P, 1 << 30, None) == code
    assert L.twg_norm_rope_backward_scratch_bytes(ctypes.byref(d)) == 0


def test_norm_rope_backward_refuses():
    L = capi.load()
    assert L.twg_norm_rope(None, None) == BAD
    d = rope(part__0__dy=None)
    assert L.twg_norm_rope_backward(ctypes.byref(d), None, 0, None) == BAD
    d = rope(part__0__dweight=P)
    need = L.twg_norm_rope_backward_scratch_bytes(ctypes.byref(d))
    assert need >= 64 * 4
    assert L.twg_norm_rope_backward(ctypes.byref(d), None, 0, None) == SMALL
    assert L.twg_norm_rope_backward(ctypes.byref(d), P, need - 1, None) == SMALL
    assert L.twg_norm_rope_backward(ctypes.byref(d), P + 1, need, None) == BAD
    d = rope(part__0__dweight=P + 1)
    assert L.twg_norm_rope_backward(ctypes.byref(d), P, 1 << 30, None) == BAD


def test_nothing_to_do_needs_no_gpu():
    L = capi.load()
    for change in (dict(batch=0), dict(tokens=0), dict(part__0__heads=0, part__1__heads=0)):
        d = rope(**change)
        assert L.twg_norm_rope(ctypes.byref(d), None) == 0
        assert L.twg_norm_rope_backward(ctypes.byref(d), None, 0, None) == 0
    d = logprobs(rows=0, logits=None, targets=None)
    assert L.twg_token_logprobs(ctypes.byref(d), None, 0, None) == 0
    assert L.twg_token_logprobs_backward(ctypes.byref(d), None) == 0
    it = capi.dense_iter(0)
    assert L.twg_dropout(None, None, None, capi.DTYPES[torch.float32], 0.5, 1, 0, None, ctypes.byref(it), None) == 0


# ------------------------------------------------------------------- token_logprobs

def logprobs(**kw):
    d = capi.TokenLogprobsArgs()
    d.dtype, d.target_dtype = capi.DTYPES[torch.float32], capi.DTYPES[torch.int64]
    d.rows, d.vocab, d.row_stride, d.logits, d.targets = 4, 100, 100, P, P
    d.ignore_index, d.scale, d.top_k = -100, 1.0, 5
    d.logprob = d.entropy = d.row_max = d.row_sum = d.top_logprobs = d.top_ids = P
    d.g_logprob = d.g_entropy = d.grad = P
    d.grad_stride = 100
    for name, v in kw.items():
        setattr(d, name, v)
    return d


@pytest.mark.parametrize("change, code", [
    (dict(dtype=7), BAD), (dict(target_dtype=6), BAD), (dict(rows=-1), BAD), (dict(rows=1 << 40), LARGE), (dict(vocab=0), BAD),
    (dict(vocab=(1 << 30) + 1), BAD), (dict(scale=0.0), BAD), (dict(scale=-1.0), BAD), (dict(scale=float("nan")), BAD),
    (dict(scale=float("inf")), BAD), (dict(logits=None), BAD), (dict(logits=P + 2), BAD), (dict(targets=None), BAD),
    (dict(targets=P + 4), BAD),
])
def test_token_logprobs_refuses(change, code):
    d, L = logprobs(**change), capi.load()
    assert L.twg_token_logprobs(ctypes.byref(d), P, 1 << 30, None) == code
    assert L.twg_token_logprobs_backward(ctypes.byref(d), None) == code


@pytest.mark.parametrize("change", [dict(top_k=-1), dict(top_k=65), dict(vocab=4, row_stride=4), dict(logprob=P + 2),
                                    dict(top_ids=P + 4)])
def test_token_logprobs_forward_refuses(change):
    d = logprobs(**change)
    assert capi.load().twg_token_logprobs(ctypes.byref(d), P, 1 << 30, None) == BAD


@pytest.mark.parametrize("change", [dict(grad=None), dict(grad=P + 1), dict(row_max=None), dict(row_sum=None), dict(entropy=None),
                                    dict(grad_stride=99), dict(grad_stride=0), dict(g_logprob=P + 2)])
def test_token_logprobs_backward_refuses(change):
    d = logprobs(**change)
    assert capi.load().twg_token_logprobs_backward(ctypes.byref(d), None) == BAD


def test_token_logprobs_scratch():
    L = capi.load()
    for rows, vocab, k in ((1, 131072, 20), (3, 50257, 64), (5000, 100, 5)):
        d = logprobs(rows=rows, vocab=vocab, row_stride=vocab, top_k=k)
        need = L.twg_token_logprobs_scratch_bytes(ctypes.byref(d))
        if need:
            assert L.twg_token_logprobs(ctypes.byref(d), P, need - 1, None) == SMALL
            assert L.twg_token_logprobs(ctypes.byref(d), None, 0, None) == SMALL
            assert L.twg_token_logprobs(ctypes.byref(d), P + 4, need, None) == BAD
    assert L.twg_token_logprobs_scratch_bytes(None) == 0


# -------------------------------------------------------------------------- dropout

def test_dropout_refuses():
    L, f32 = capi.load(), capi.DTYPES[torch.float32]
    it = capi.dense_iter(64)

    def call(out=P, x=P, res=None, dtype=f32, p=0.5, d_offset=None, it=it):
        return L.twg_dropout(out, x, res, dtype, p, 1, 0, d_offset, ctypes.byref(it) if it is not None else None, None)

    for bad in (dict(out=None), dict(x=None), dict(dtype=3), dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(out=P + 1),
                dict(x=P + 2), dict(res=P + 2), dict(d_offset=P + 4), dict(it=None)):
        assert call(**bad) == BAD, bad
    wrong = capi.dense_iter(64)
    wrong.numel = 63
    assert call(it=wrong) == BAD
    assert call(it=capi.make_iter((4, 16), (0, 1), (16, 1))) == BAD  # rows of the result in one place


def test_the_oracles_generator_gives_the_published_vectors():
    # the known answers published with the generator (counter and key all 0, all 1)
    assert ref.philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert ref.philox((ones,) * 4, (ones,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


# ----------------------------------------------- the functions on tensors, argument checks

def test_functions_on_tensors_want_gpu_memory():
    x = torch.zeros(1, 2, 3, 8)
    with pytest.raises(ValueError):
        capi.norm_rope(x, None, torch.arange(2), torch.ones(4))
    with pytest.raises(ValueError):
        capi.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        capi.dropout(torch.zeros(4), 0.5, 1)


def test_operators_are_registered_with_their_gradients():
    import torch_webgpu  # noqa: F401
    for op in ("webgpu::norm_rope", "webgpu::token_logprobs", "webgpu::dropout", "aten::dropout", "aten::dropout_"):
        lines = torch._C._dispatch_dump(op).splitlines()
        for key in ("PrivateUse1:", "AutogradPrivateUse1:"):
            line = [l for l in lines if l.startswith(key)]
            assert line and "fallthrough" not in line[0], (op, key)


def test_the_generators_state():
    import torch_webgpu  # noqa: F401
    before = torch.webgpu.get_rng_state()
    torch.manual_seed(1234)
    assert torch.webgpu.initial_seed() == 1234
    assert not torch.equal(torch.webgpu.get_rng_state(), before)
    torch.webgpu.set_rng_state(before)
    assert torch.equal(torch.webgpu.get_rng_state(), before)
    torch.webgpu.manual_seed(-1)
    assert torch.webgpu.initial_seed() == 2 ** 64 - 1
    with pytest.raises(ValueError):
        torch.webgpu.set_rng_state(torch.zeros(3, dtype=torch.uint8))
    torch.webgpu.set_rng_state(before)


def test_the_device_context_takes_the_one_device():
    import torch_webgpu  # noqa: F401
    for d in (None, 0, "webgpu", "webgpu:0", torch.device("webgpu", 0)):
        with torch.webgpu.device(d):
            assert torch.webgpu.current_device() == 0
    with pytest.raises(ValueError):
        torch.webgpu.device(1)
