"""What the operators of a transformer layer's steps give for fake tensors: shapes, types, strides and
devices, without memory.  Tracers (torch.compile among them) run these instead of the kernels."""
import torch
from torch.library import register_fake


def _heads_like(x):
    """in the order in which x's heads are stored, where that leaves head_dim dense"""
    if x.shape[3] > 1 and x.stride(3) != 1:
        x = x.contiguous()
    out = torch.empty_like(x)
    return out if x.shape[3] <= 1 or out.stride(3) == 1 else x.new_empty(x.shape)


@register_fake("webgpu::norm_rope")
def _(q, k, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6, pair_axis=None, adjacent=False):
    return [_heads_like(x) for x in (q, k) if x is not None]


@register_fake("webgpu::_norm_rope_backward")
def _(dq, dk, q, k, positions, inv_freq, q_weight, k_weight, eps, pair_axis, adjacent, q_weight_grad, k_weight_grad):
    return (None if dq is None else _heads_like(q), None if dk is None else _heads_like(k),
            q_weight.new_empty(q_weight.shape) if dq is not None and q_weight_grad else None,
            k_weight.new_empty(k_weight.shape) if dk is not None and k_weight_grad else None)


@register_fake("webgpu::token_logprobs")
def _(logits, targets, top_k=0, scale=1.0, ignore_index=-100):
    def result(shape, dtype):
        return logits.new_empty(shape, dtype=dtype)

    top = (*targets.shape, top_k)
    return (result(targets.shape, torch.float32), result(targets.shape, torch.float32), result(top, torch.float32),
            result(top, torch.int64))


@register_fake("webgpu::_token_logprobs")
def _(logits, targets, top_k, scale, ignore_index):
    def result(shape, dtype):
        return logits.new_empty(shape, dtype=dtype)

    top, rows = (*targets.shape, top_k), (targets.numel(),)
    return (result(targets.shape, torch.float32), result(targets.shape, torch.float32), result(top, torch.float32),
            result(top, torch.int64), result(rows, torch.float32), result(rows, torch.float32))


@register_fake("webgpu::_token_logprobs_backward")
def _(g_logprob, g_entropy, logits, targets, row_max, row_sum, entropy, scale, ignore_index):
    return logits.new_empty(logits.shape)


@register_fake("webgpu::dropout")
def _(x, p, seed, offset=0, residual=None):
    return torch.empty_like(x)


def _draw():
    return torch.empty(2, dtype=torch.int64, device="cpu")


@register_fake("webgpu::_draw_dropout")
def _(x, p):
    return torch.empty_like(x), _draw()


@register_fake("webgpu::_draw_dropout_")
def _(x, p):
    return _draw()


@register_fake("webgpu::_redo_dropout")
def _(x, p, draw):
    return torch.empty_like(x)
