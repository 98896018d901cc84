"""Differentiable forms of the operators that have a gradient.

:func:`cross_attention`, :func:`relative_position_bias` and :func:`relative_position_encoding` are those of
:mod:`boltz_lumi_b200.kernels` with autograd recorded: ``loss.backward()`` runs the library's backward kernels.  Without
grad mode or inputs that need a gradient they are the plain calls.

They have reverse-mode gradients of first order: an input that carries a forward-mode tangent is refused.

Under CUDA graph capture they refuse inputs that need a gradient.  A captured autograd pass would run the leaves' gradient
accumulation on whatever stream an earlier, still living eager graph of the same leaves recorded, which ends the process
inside torch; capture the explicit pair instead (``kernels.cross_attention(..., return_lse=True)`` and
``kernels.cross_attention_backward``, and likewise for the others), which records no graph.
"""

import torch

from . import kernels


def _recorded(name, *tensors):
    """Whether the call records autograd; refuses to do so under stream capture."""
    kernels._refuse_tangents(*tensors)
    if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)):
        return False
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{name} does not record gradients under CUDA graph capture: capture "
                           f"kernels.{name} and kernels.{name}_backward instead")
    return True


def _no_capture(name):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"the backward pass of {name} cannot be captured: capture kernels.{name}_backward instead")


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, gate, mask, inf, scale):
        out, lse = kernels.cross_attention(q, k, v, bias=bias, mask=mask, inf=inf, gate=gate, scale=scale, return_lse=True)
        ctx.save_for_backward(q, k, v, bias, gate, mask, out, *lse)
        ctx.inf, ctx.scale = inf, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _no_capture("cross_attention")
        q, k, v, bias, gate, mask, out, rows, low = ctx.saved_tensors
        dq, dk, dv, dbias, dgate = kernels.cross_attention_backward(
            grad, q, k, v, out, kernels.AttentionStats(rows, low), bias=bias, mask=mask, inf=ctx.inf, gate=gate, scale=ctx.scale,
            need_bias_grad=ctx.needs_input_grad[3])
        return dq, dk, dv, dbias, dgate, None, None, None


def cross_attention(q, k, v, bias=None, mask=None, inf=None, gate=None, scale=None):
    """:func:`boltz_lumi_b200.kernels.cross_attention`, differentiable in q, k, v, bias and gate."""
    if not _recorded("cross_attention", q, k, v, bias, gate):
        return kernels.cross_attention(q, k, v, bias=bias, mask=mask, inf=inf, gate=gate, scale=scale)
    return _CrossAttention.apply(q, k, v, bias, gate, mask, inf, scale)


class _RelativePositionBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, q_pos, k_pos, lut, q_group, k_group, out_dtype):
        ctx.save_for_backward(q_pos, k_pos, lut, q_group, k_group)
        ctx.buckets = table.shape[0]
        return kernels.relative_position_bias(table, q_pos, k_pos, lut, q_group, k_group, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _no_capture("relative_position_bias")
        dtable = kernels.relative_position_bias_backward(grad, *ctx.saved_tensors, num_buckets=ctx.buckets)
        return dtable, None, None, None, None, None, None


def relative_position_bias(table, q_pos, k_pos, lut, q_group=None, k_group=None, out_dtype=None):
    """:func:`boltz_lumi_b200.kernels.relative_position_bias`, differentiable in its table."""
    if not _recorded("relative_position_bias", table):
        return kernels.relative_position_bias(table, q_pos, k_pos, lut, q_group, k_group, out_dtype)
    return _RelativePositionBias.apply(table, q_pos, k_pos, lut, q_group, k_group, out_dtype)


class _RelativePositionEncoding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, r_max, s_max, fix_sym_check, out_dtype, *features):
        ctx.save_for_backward(*features)
        ctx.args = r_max, s_max, fix_sym_check
        return kernels.relative_position_encoding(weight, *features, r_max, s_max, fix_sym_check, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _no_capture("relative_position_encoding")
        dweight = kernels.relative_position_encoding_backward(grad, *ctx.saved_tensors, *ctx.args)
        return (dweight,) + (None,) * 9


def relative_position_encoding(weight, residue_index, asym_id, entity_id, token_index, sym_id, r_max=32, s_max=2,
                               fix_sym_check=False, out_dtype=None):
    """:func:`boltz_lumi_b200.kernels.relative_position_encoding`, differentiable in its weight."""
    features = residue_index, asym_id, entity_id, token_index, sym_id
    if not _recorded("relative_position_encoding", weight):
        return kernels.relative_position_encoding(weight, *features, r_max, s_max, fix_sym_check, out_dtype)
    return _RelativePositionEncoding.apply(weight, r_max, s_max, fix_sym_check, out_dtype, *features)


__all__ = ["cross_attention", "relative_position_bias", "relative_position_encoding"]
