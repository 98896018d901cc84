"""Torch-facing wrappers of the C-ABI kernels (one per reference native op).

Each function mirrors a native function of the reference (the pybind11
bindings of ``kernels/*_hip.cpp`` and the Triton ``ordered_softmax``): same
argument meaning, a freshly allocated output, inference only, and the current
CUDA stream of the input's device.  Errors raise ``RuntimeError``; there is
no fallback path.
"""

import functools
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import call, launch, ptr, size_of, stream_of


def _refuse_tangents(*tensors):
    if forward_ad._current_level >= 0:  # inside dual_level(): the kernels would drop a tangent
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("boltz_lumi_b200 operators have no forward-mode derivatives (an input carries a tangent)")


def _require_inference(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("boltz_lumi_b200 kernels are inference-only (grad mode with requires_grad inputs)")
    _refuse_tangents(*tensors)


def _require_cuda(*tensors):
    device = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("boltz_lumi_b200 kernels need CUDA tensors")
        if device is None:
            device = t.device
        elif t.device != device:
            raise RuntimeError("all tensors must be on the same device")
    return device


def norm(x, weight, bias, eps, channel_first=False, bf16_output=True):
    """LayerNorm over 128 channels (reference ``extension("multiplication").norm``,
    ``kernels/multiplication_hip.cu:149``).

    Row-major ``x`` is [M, C]; channel-first ``x`` is [128, M].  Returns [M, C]
    in bf16 (``bf16_output``) or fp32.
    """
    _require_inference(x)
    _require_cuda(x, weight, bias)
    if x.dim() != 2 or not x.is_contiguous():
        raise RuntimeError("norm expects a contiguous 2-D tensor")
    rows, cols = (x.shape[1], x.shape[0]) if channel_first else (x.shape[0], x.shape[1])
    for v in (weight, bias):
        if v is not None and (v.dtype != torch.float32 or v.numel() != cols or not v.is_contiguous()):
            raise RuntimeError("norm weight/bias must be contiguous fp32 with one value per channel")
    out = torch.empty(rows, cols, device=x.device, dtype=torch.bfloat16 if bf16_output else torch.float32)
    call("bl_layernorm", x.data_ptr(), _lib.dtype_code(x.dtype), rows, cols, int(channel_first), ptr(weight),
         ptr(bias), float(eps), out.data_ptr(), _lib.dtype_code(out.dtype), stream_of(x))
    return out


def layer_norm(x, weight, bias, eps, out_dtype=None):
    """LayerNorm over the last dimension of any-rank ``x`` (fp32 statistics)."""
    _require_inference(x)
    _require_cuda(x, weight, bias)
    x = x.contiguous()
    cols = x.shape[-1]
    out = torch.empty(x.shape, device=x.device, dtype=out_dtype or x.dtype)
    call("bl_layernorm", x.data_ptr(), _lib.dtype_code(x.dtype), x.numel() // max(cols, 1), cols, 0,
         ptr(weight), ptr(bias), float(eps), out.data_ptr(), _lib.dtype_code(out.dtype), stream_of(x))
    return out


def gate(p, g):
    """``bf16(p * bf16(sigmoid(g)))`` (reference ``multiplication_gate_hip.cu:81``)."""
    _require_inference(p, g)
    _require_cuda(p, g)
    if p.shape != g.shape or p.dtype != torch.bfloat16 or g.dtype != torch.bfloat16:
        raise RuntimeError("gate expects two bf16 tensors of the same shape")
    p, g = p.contiguous(), g.contiguous()
    out = torch.empty_like(p)
    call("bl_gate", p.data_ptr(), g.data_ptr(), out.data_ptr(), p.numel(), stream_of(p))
    return out


def _gate_operands(p, g, mask):
    _require_inference(p, g)
    _require_cuda(p, g, mask)
    if p.dtype != torch.bfloat16 or g.dtype != torch.bfloat16:
        raise RuntimeError("gate operands must be bf16")
    if p.dim() != 4 or p.shape[0] != 1 or p.shape[1] != p.shape[2] or p.shape[3] != 256:
        raise RuntimeError("expected projections of shape [1, N, N, 256]")
    stride = p.stride(2)
    if stride not in (256, 512) or p.stride(3) != 1 or p.stride(1) != p.shape[2] * stride or g.stride() != p.stride():
        raise RuntimeError("expected dense or joint-projection rows")
    if mask.dtype != torch.float32 or not mask.is_contiguous() or mask.numel() * 256 != p.shape[1] * p.shape[2] * 256:
        raise RuntimeError("mask must be contiguous fp32 [1, N, N]")
    return p.shape[1], stride


def pack(p, g, mask, outgoing):
    """Gate, mask and channel-first pack (reference ``multiplication_gate_hip.cu:140``)."""
    n, stride = _gate_operands(p, g, mask)
    left = torch.empty(128, n, n, device=p.device, dtype=torch.bfloat16)
    right = torch.empty_like(left)
    call("bl_gate_pack", p.data_ptr(), g.data_ptr(), stride, mask.data_ptr(), n, int(bool(outgoing)),
         left.data_ptr(), right.data_ptr(), stream_of(p))
    return left, right


def split(p, g, mask):
    """Gate and mask into channel-last halves (reference ``multiplication_gate_hip.cu:96``)."""
    n, stride = _gate_operands(p, g, mask)
    a = torch.empty(1, n, n, 128, device=p.device, dtype=torch.bfloat16)
    b = torch.empty_like(a)
    call("bl_gate_split", p.data_ptr(), g.data_ptr(), stride, mask.data_ptr(), n, a.data_ptr(), b.data_ptr(),
         stream_of(p))
    return a, b


def silu_mul(a, b):
    """``bf16(bf16(silu(a)) * b)`` (reference ``kernels/pair_hip.cu:42``)."""
    _require_inference(a, b)
    _require_cuda(a, b)
    if a.shape != b.shape or a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
        raise RuntimeError("silu_mul expects two bf16 tensors of the same shape")
    if not (a.is_contiguous() and b.is_contiguous()):
        raise RuntimeError("silu_mul expects contiguous inputs")
    out = torch.empty_like(a)
    call("bl_silu_mul", a.data_ptr(), b.data_ptr(), out.data_ptr(), a.numel(), stream_of(a))
    return out


MODULATION, GATE, GATED_SWIGLU = _lib.BL_EPI_MODULATION, _lib.BL_EPI_GATE, _lib.BL_EPI_GATED_SWIGLU
SWIGLU = _lib.BL_EPI_SWIGLU  # silu(a[:, :C]) * a[:, C:] (an fp32 Transition's fc1 | fc2 product)


def epilogue(a, b, c, kind):
    """fp32 diffusion epilogues (reference ``kernels/diffusion_hip.cu:80``)."""
    _require_inference(a, b, c)
    _require_cuda(a, b, c)
    if kind not in (MODULATION, GATE, GATED_SWIGLU, SWIGLU):
        raise RuntimeError(f"unknown epilogue kind {kind}")
    for t in (a, b, c):
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous()):
            raise RuntimeError("epilogue expects contiguous fp32 tensors")
    shape = list(a.shape)
    cols = shape[-1]
    if kind in (GATED_SWIGLU, SWIGLU):
        if cols % 2:
            raise RuntimeError("SwiGLU epilogues need an even last dimension")
        cols //= 2
        shape[-1] = cols
    out = torch.empty(shape, device=a.device, dtype=torch.float32)
    if (kind != SWIGLU and tuple(b.shape) != tuple(shape)) or \
            (kind == MODULATION and (c is None or tuple(c.shape) != tuple(shape))):
        raise RuntimeError("epilogue operand shapes disagree")
    rows = out.numel() // max(cols, 1)
    call("bl_diffusion_epilogue", a.data_ptr(), ptr(b), ptr(c), out.data_ptr(), rows, cols, kind, stream_of(a))
    return out


def adaln_modulate(a, scale, shift, eps):
    """``sigmoid(scale) * LayerNorm(a) + shift`` with a non-affine LayerNorm (fp32)."""
    _require_inference(a, scale, shift)
    _require_cuda(a, scale, shift)
    a, scale, shift = a.contiguous(), scale.contiguous(), shift.contiguous()
    if not (a.dtype == scale.dtype == shift.dtype == torch.float32) or not (a.shape == scale.shape == shift.shape):
        raise RuntimeError("adaln_modulate expects fp32 tensors of one shape")
    out = torch.empty_like(a)
    cols = a.shape[-1]
    call("bl_adaln_modulate", a.data_ptr(), scale.data_ptr(), shift.data_ptr(), out.data_ptr(),
         a.numel() // max(cols, 1), cols, float(eps), stream_of(a))
    return out


def ordered_softmax(scores, bias, mask):
    """``softmax(round(round(s + mask) + bias))`` over materialised triangle scores.

    Reference ``kernels/triangle_softmax.py:120`` / ``triangle_block_softmax_hip.cu:120``.
    ``scores`` [B, I, H, N, N]; ``bias`` broadcastable as [B, 1, H, N, N];
    ``mask`` fp32 broadcastable as [B, I, 1, 1, N].
    """
    _require_inference(scores, bias)
    _require_cuda(scores, bias, mask)
    if scores.dim() != 5 or scores.shape[-1] != scores.shape[-2]:
        raise RuntimeError("expected square score matrices [B, I, H, N, N]")
    if bias.dtype != scores.dtype or mask.dtype != torch.float32:
        raise RuntimeError("bias must share the score dtype; mask must be fp32")
    b, i, h, n, _ = scores.shape
    bias = bias.expand(b, 1, h, n, n)
    mask = mask.expand(b, i, 1, 1, n)
    out = torch.empty(scores.shape, device=scores.device, dtype=scores.dtype)
    ss = _lib.int64_array(scores.stride())
    bs = _lib.int64_array((bias.stride(0), bias.stride(2), bias.stride(3), bias.stride(4)))
    ms = _lib.int64_array((mask.stride(0), mask.stride(1), mask.stride(4)))
    call("bl_triangle_softmax", scores.data_ptr(), _lib.dtype_code(scores.dtype), b, i, h, n, ss, bias.data_ptr(), bs,
         mask.data_ptr(), ms, out.data_ptr(), stream_of(scores))
    return out


def _operand_layout(t, name):
    """Return (mn_major, ld, batch_stride) for a [batch, rows, k]-shaped view."""
    if t.stride(-1) == 1:
        return False, t.stride(-2), t.stride(0)
    if t.stride(-2) == 1:
        return True, t.stride(-1), t.stride(0)
    raise RuntimeError(f"{name} needs one unit stride among its last two dimensions")


def bmm(a, b_t, bias=None, out=None):
    """``out[b] = a[b] @ b_t[b]^T (+ bias)`` in bf16 on tcgen05 tensor cores.

    ``a`` [B, M, K] and ``b_t`` [B, N, K] may each be K-contiguous or
    M/N-contiguous (e.g. ``x.transpose(1, 2)`` of a dense tensor); nothing is copied.
    """
    _require_inference(a, b_t)
    _require_cuda(a, b_t, bias)
    if a.dtype != torch.bfloat16 or b_t.dtype != torch.bfloat16:
        raise RuntimeError("bmm operands must be bf16")
    if a.dim() != 3 or b_t.dim() != 3 or a.shape[0] != b_t.shape[0] or a.shape[2] != b_t.shape[2]:
        raise RuntimeError("bmm expects a [B, M, K] and b_t [B, N, K]")
    batch, m, k = a.shape
    n = b_t.shape[1]
    a_mn, a_ld, a_bs = _operand_layout(a, "a")
    b_mn, b_ld, b_bs = _operand_layout(b_t, "b_t")
    if out is None:
        out = torch.empty(batch, m, n, device=a.device, dtype=torch.bfloat16)
    if bias is not None and (bias.dtype != torch.float32 or bias.numel() != n):
        raise RuntimeError("bias must be fp32 with N elements")
    call("bl_batched_gemm", a.data_ptr(), int(a_mn), a_ld, a_bs, b_t.data_ptr(), int(b_mn), b_ld, b_bs,
         out.data_ptr(), out.stride(1), out.stride(0), batch, m, n, k, ptr(bias), stream_of(a))
    return out


@functools.lru_cache(maxsize=None)
def attention_scale(head_dim):
    """fp32(1 / fp32(sqrt(head_dim))): the factor torch's CUDA division by the
    Python scalar ``head_dim ** 0.5`` applies (pair_bias.py:31)."""
    return float(torch.tensor(1.0, dtype=torch.float32) / torch.tensor(head_dim ** 0.5, dtype=torch.float32))


def launch_token_attention(q_ptr, k_ptr, v_ptr, g_ptr, strides, bias, mask, inf, batch, heads, n, d, out, stream,
                           out3=None, n_q=0):
    """bl_token_attention on raw operand pointers sharing ``strides`` (batch,
    token, head) -- no validation; callers have checked shapes and dtypes.
    With ``out3`` (bf16 [3, batch * n_q, heads * d]) the result is written as the
    split planes instead of into ``out``.  ``n_q`` (0: n) queries from q_ptr / g_ptr
    and the bias rows attend over n keys."""
    mask_ptr, mask_sb = (None, 0) if mask is None else (mask.data_ptr(), mask.stride(0))
    bs = bias.stride()
    call("bl_token_attention", q_ptr, k_ptr, v_ptr, g_ptr, strides[0], strides[1], strides[2], bias.data_ptr(),
         bs[0], bs[1], bs[2], bs[3], batch // bias.shape[0], mask_ptr, mask_sb, attention_scale(d), float(inf),
         batch, heads, n, n_q, d, ptr(out), ptr(out3), stream)
    return out


def token_attention(q, k, v, bias, mask, inf, gate=None, scale=None):
    """Fused fp32 attention of the diffusion token transformer (and the
    Pairformer's single track): ``sigmoid(gate) * softmax(q k^T * scale + bias
    + inf * (mask - 1)) v`` per head, the core of pair_bias.py:28-36.

    ``q``, ``k``, ``v`` (and ``gate``): fp32 [B, N, H, d] views with a common
    stride layout and contiguous head dims (e.g. slices of one joint
    projection).  ``bias``: fp32 [Bb, H, N, N] with any strides, where ``Bb``
    divides ``B`` -- sample ``b`` reads bias ``b // (B // Bb)``, which is the
    reference's ``repeat_interleave(multiplicity, 0)`` without the copy.
    ``mask``: [B, N] key mask or None.  Returns fp32 [B, N, H, d].
    """
    _require_inference(q, k, v, gate, bias, mask)
    _require_cuda(q, k, v, gate, bias, mask)
    tensors = [q, k, v] + ([gate] if gate is not None else [])
    if any(t.dtype != torch.float32 for t in tensors + [bias]):
        raise RuntimeError("token attention operands must be fp32")
    if any(t.dim() != 4 or t.shape != q.shape or t.stride() != q.stride() for t in tensors):
        raise RuntimeError("q, k, v and gate must be [B, N, H, d] views with the same strides")
    batch, n, heads, d = q.shape
    if q.stride(3) != 1:
        raise RuntimeError("q/k/v head dims must be contiguous")
    if bias.dim() != 4 or tuple(bias.shape[1:]) != (heads, n, n) or bias.shape[0] < 1 or batch % bias.shape[0]:
        raise RuntimeError(f"bias must be [B', {heads}, {n}, {n}] with B' dividing {batch}, got {tuple(bias.shape)}")
    mask_sb = 0
    if mask is not None:
        if tuple(mask.shape) != (batch, n):
            raise RuntimeError("mask must be [B, N]")
        mask = mask.float()
        if mask.stride(1) != 1:
            mask = mask.contiguous()
        mask_sb = mask.stride(0)
    if scale is None:
        scale = attention_scale(d)
    out = torch.empty(batch, n, heads, d, device=q.device, dtype=torch.float32)
    if n == 0 or batch == 0:
        return out
    call("bl_token_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr(gate), q.stride(0), q.stride(1),
         q.stride(2), bias.data_ptr(), bias.stride(0), bias.stride(1), bias.stride(2), bias.stride(3),
         batch // bias.shape[0], ptr(mask), mask_sb, float(scale), float(inf), batch, heads, n, 0, d, out.data_ptr(),
         None, stream_of(q))
    return out


def split3(x):
    """fp32 ``x`` [..., K] -> bf16 planes [3, rows, K] with x = x1 + x2 + x3
    (bl_split3_bf16); the operand form of :func:`linear_f32`."""
    _require_cuda(x)
    if x.dtype != torch.float32:
        raise RuntimeError("split3 expects fp32")
    cols = x.shape[-1]
    x2 = x.reshape(-1, cols)
    if x2.stride(-1) != 1 or x2.data_ptr() % 16 or x2.stride(0) % 4:
        x2 = x2.contiguous()
    out = torch.empty(3, x2.shape[0], cols, device=x.device, dtype=torch.bfloat16)
    call("bl_split3_bf16", x2.data_ptr(), x2.shape[0], cols, x2.stride(0), out.data_ptr(), stream_of(x))
    return out


def split3_fast(x):
    """:func:`split3` for callers that have checked x (fp32, CUDA, K % 8 == 0)."""
    cols = x.shape[-1]
    if not x.is_contiguous():
        x = x.contiguous()
    rows = x.numel() // cols
    out = torch.empty(3, rows, cols, device=x.device, dtype=torch.bfloat16)
    call("bl_split3_bf16", x.data_ptr(), rows, cols, cols, out.data_ptr(), _lib.current_stream_handle())
    return out


def linear_split3_fast(x3, w3, bias, y, residual=None):
    """bl_linear_split3 into the contiguous fp32 ``y`` [..., N] for callers
    that have checked the operands (x3 = split3(x), w3 = split3(W)); with
    ``residual`` (contiguous fp32 [..., N]) the result is y = x W^T + bias + residual."""
    m, k = x3.shape[1], x3.shape[2]
    n = w3.shape[1]
    call("bl_linear_split3", x3.data_ptr(), m, k, w3.data_ptr(), n, ptr(bias), ptr(residual),
         0 if residual is None else n, y.data_ptr(), n, _lib.current_stream_handle())
    return y


def linear_f32(x, w3, bias=None, x3=None):
    """fp32 ``x @ W^T + bias`` on the tensor cores (error within 2^-17 of the largest output)
    (bl_linear_split3).  ``w3`` = ``split3(W)`` (bf16 [3, N, K]); ``x3`` may
    pass ``split3(x)`` when one input feeds several linears."""
    _require_inference(x)
    _require_cuda(x, w3, bias)
    k = x.shape[-1]
    n = w3.shape[1]
    if w3.shape != (3, n, k) or w3.dtype != torch.bfloat16:
        raise RuntimeError(f"w3 must be bf16 [3, N, {k}]")
    if bias is not None and (bias.dtype != torch.float32 or bias.numel() != n or not bias.is_contiguous()):
        raise RuntimeError("bias must be contiguous fp32 with N elements")
    if x3 is None:
        x3 = split3(x)
    m = x3.shape[1]
    y = torch.empty(*x.shape[:-1], n, device=x.device, dtype=torch.float32)
    return linear_split3_fast(x3, w3, bias, y)


def layer_norm_split3(x, weight, bias, eps):
    """LayerNorm of fp32 rows written as split planes [3, rows, C] (bl_layernorm_split3);
    C % 128 == 0 and <= 1024."""
    cols = x.shape[-1]
    x = x.contiguous()
    rows = x.numel() // cols
    out = torch.empty(3, rows, cols, device=x.device, dtype=torch.bfloat16)
    call("bl_layernorm_split3", x.data_ptr(), rows, cols, ptr(weight), ptr(bias), float(eps), out.data_ptr(),
         _lib.current_stream_handle())
    return out


def adaln_modulate_split3(a, scale, shift, eps):
    """:func:`adaln_modulate` written as split planes [3, rows, C]."""
    a, scale, shift = a.contiguous(), scale.contiguous(), shift.contiguous()
    cols = a.shape[-1]
    rows = a.numel() // cols
    out = torch.empty(3, rows, cols, device=a.device, dtype=torch.bfloat16)
    call("bl_adaln_modulate_split3", a.data_ptr(), scale.data_ptr(), shift.data_ptr(), out.data_ptr(), rows, cols,
         float(eps), _lib.current_stream_handle())
    return out


def epilogue_split3(a, b, c, kind):
    """:func:`epilogue` written as split planes [3, rows, C] (C = output width)."""
    cols = a.shape[-1] // 2 if kind in (GATED_SWIGLU, SWIGLU) else a.shape[-1]
    rows = a.numel() // a.shape[-1]
    out = torch.empty(3, rows, cols, device=a.device, dtype=torch.bfloat16)
    call("bl_diffusion_epilogue_split3", a.data_ptr(), ptr(b), ptr(c), out.data_ptr(), rows, cols, kind,
         _lib.current_stream_handle())
    return out


# ---------------------------------------------------------------------------
# Relative positions by buckets
# ---------------------------------------------------------------------------
def _workspace(nbytes, device):
    return torch.empty(max(int(nbytes), 16), device=device, dtype=torch.uint8)


def _index(name, t, device, shape):
    """An integer index tensor as contiguous int64 of ``shape`` on ``device`` (None stays None)."""
    if t is None or t.dtype is torch.int64 and t.shape == shape and t.device == device and t.is_contiguous():
        return t
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}, got {t.device}")
    if t.shape != shape:
        raise RuntimeError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype not in (torch.int64, torch.int32, torch.int16, torch.uint8):
        raise RuntimeError(f"{name} must hold integers, got {t.dtype}")
    return t.to(torch.int64).contiguous()


def _token_features(device, shape, residue_index, asym_id, entity_id, token_index, sym_id):
    return (_index("residue_index", residue_index, device, shape), _index("asym_id", asym_id, device, shape),
            _index("entity_id", entity_id, device, shape), _index("token_index", token_index, device, shape),
            _index("sym_id", sym_id, device, shape))


def _float_dtype(dtype, what):
    if dtype not in (torch.float32, torch.bfloat16):
        raise RuntimeError(f"{what} must be fp32 or bf16, got {dtype}")
    return dtype


def relative_position_columns(r_max=32, s_max=2):
    """Columns of the relative position encoding's weight: residue offsets, token offsets, entity, chain copies."""
    return 2 * (2 * r_max + 2) + 1 + 2 * s_max + 2


def relative_position_encoding(weight, residue_index, asym_id, entity_id, token_index, sym_id, r_max=32, s_max=2,
                               fix_sym_check=False, out_dtype=None, residual=None):
    """Relative position encoding of token pairs, [B, N, N, C] (AF3 supplementary Algorithm 3).

    ``weight`` is upstream ``RelativePositionEncoder.linear_layer.weight``, fp32
    [C, 4 r_max + 2 s_max + 7], C a multiple of 4; the token features are
    integers [B, N].  Pair (i, j) gets the sum of the weight columns of its
    clipped residue offset, token offset and chain-copy offset, and of the
    entity column if the entities agree (``fix_sym_check``: the chain-copy
    offset counts within an entity instead of between chains).  The sum is
    fp32, rounded once to ``out_dtype`` (default fp32).  With ``residual`` (a
    contiguous fp32 [B, N, N, C]) it is added into that tensor, which is
    returned.  For gradients see :func:`relative_position_encoding_backward`
    and :mod:`boltz_lumi_b200.autograd`.
    """
    _require_inference(weight, residual)
    _require_cuda(weight, residue_index, residual)
    if residue_index.dim() != 2:
        raise RuntimeError("token features must be [B, N]")
    b, n = residue_index.shape
    if weight.dtype != torch.float32 or weight.dim() != 2 or weight.shape[1] != relative_position_columns(r_max, s_max):
        raise RuntimeError(f"weight must be fp32 [C, {relative_position_columns(r_max, s_max)}] for r_max {r_max}, "
                           f"s_max {s_max}, got {weight.dtype} {list(weight.shape)}")
    c = weight.shape[0]
    features = _token_features(weight.device, (b, n), residue_index, asym_id, entity_id, token_index, sym_id)
    if residual is not None:
        if residual.dtype != torch.float32 or not residual.is_contiguous() or tuple(residual.shape) != (b, n, n, c):
            raise RuntimeError(f"residual must be a contiguous fp32 tensor [{b}, {n}, {n}, {c}]")
        if out_dtype not in (None, torch.float32):
            raise RuntimeError("an fp32 residual keeps its dtype")
        out = residual
    else:
        out = torch.empty(b, n, n, c, device=weight.device, dtype=_float_dtype(out_dtype or torch.float32, "out_dtype"))
    weight = weight.contiguous()
    launch(weight.device, "bl_relative_position_encoding", weight.data_ptr(), *[t.data_ptr() for t in features], b, n, c,
           r_max, s_max, int(fix_sym_check), out.data_ptr(), _lib.dtype_code(out.dtype), int(residual is not None))
    return out


def relative_position_encoding_backward(grad, residue_index, asym_id, entity_id, token_index, sym_id, r_max=32, s_max=2,
                                        fix_sym_check=False):
    """Gradient of :func:`relative_position_encoding` with respect to its weight: fp32 [C, columns] from the
    gradient of the output, fp32 or bf16 [B, N, N, C].  Sums are fp32 in a fixed order."""
    _require_inference(grad)
    _require_cuda(grad, residue_index)
    if grad.dim() != 4 or grad.shape[1] != grad.shape[2]:
        raise RuntimeError("grad must be [B, N, N, C]")
    _float_dtype(grad.dtype, "grad")
    b, n, _, c = grad.shape
    device = grad.device
    features = _token_features(device, (b, n), residue_index, asym_id, entity_id, token_index, sym_id)
    grad = grad.contiguous()
    if grad.data_ptr() % 16:
        grad = grad.clone()
    dweight = torch.empty(c, relative_position_columns(r_max, s_max), device=device, dtype=torch.float32)
    nbytes = size_of("bl_relative_position_encoding_workspace", b, n, c, r_max, s_max)
    work = _workspace(nbytes, device)
    launch(device, "bl_relative_position_encoding_backward", grad.data_ptr(), _lib.dtype_code(grad.dtype),
           *[t.data_ptr() for t in features], b, n, c, r_max, s_max, int(fix_sym_check), dweight.data_ptr(),
           work.data_ptr(), nbytes)
    return dweight


def clipped_buckets(max_distance, device="cuda"):
    """Bucket table of :func:`relative_position_bias` with one bucket per offset clipped to
    [-max_distance, max_distance] (int32, 2 max_distance + 1 buckets)."""
    return torch.arange(2 * max_distance + 1, dtype=torch.int32, device=device)


def log_spaced_buckets(num_buckets, max_distance, bidirectional=True, device="cuda"):
    """Bucket table of :func:`relative_position_bias` with log-spaced far offsets (int32, 2 max_distance + 1).

    Half of the buckets (of each sign, with ``bidirectional``) hold one offset each; the others grow
    geometrically up to ``max_distance``.  Offset = query position - key position; with
    ``bidirectional`` keys ahead of the query (negative offsets) take the upper half of the buckets,
    without it they share the bucket of offset 0.
    """
    side = num_buckets // 2 if bidirectional else num_buckets
    exact = side // 2
    if exact < 1 or max_distance <= exact:
        raise RuntimeError("log_spaced_buckets needs num_buckets >= 4 (2 one-sided) and a larger max_distance")
    lut = []
    for offset in range(-max_distance, max_distance + 1):
        m = abs(offset) if bidirectional else max(offset, 0)
        if m >= exact:
            m = min(side - 1, exact + int(math.log(m / exact) / math.log(max_distance / exact) * (side - exact)))
        lut.append(m + (side if bidirectional and offset < 0 else 0))
    return torch.tensor(lut, dtype=torch.int32, device=device)


def _bias_positions(device, q_pos, k_pos, lut, q_group, k_group):
    if q_pos.dim() != 2 or k_pos.dim() != 2 or q_pos.shape[0] != k_pos.shape[0]:
        raise RuntimeError("q_pos must be [B, Nq] and k_pos [B, Nk]")
    if (q_group is None) != (k_group is None):
        raise RuntimeError("give both q_group and k_group or neither")
    if lut.dim() != 1 or lut.dtype != torch.int32 or lut.numel() % 2 == 0 or lut.device != device:
        raise RuntimeError("lut must be an int32 vector of odd length on the device of the other tensors")
    return (_index("q_pos", q_pos, device, q_pos.shape), _index("k_pos", k_pos, device, k_pos.shape), lut.contiguous(),
            _index("q_group", q_group, device, q_pos.shape), _index("k_group", k_group, device, k_pos.shape))


def padded_planes(b, h, nq, nk, device, dtype):
    """An uninitialised [b, h, nq, nk] whose rows start on 16-byte boundaries (the layout the attention kernels
    read fastest): rows padded to a multiple of 8 elements."""
    ld = (nk + 7) // 8 * 8
    return torch.empty_strided((b, h, nq, nk), (h * nq * ld, nq * ld, ld, 1), device=device, dtype=dtype)


def relative_position_bias(table, q_pos, k_pos, lut, q_group=None, k_group=None, out_dtype=None):
    """Learned relative position bias of attention heads by buckets, [B, H, Nq, Nk].

    ``out[b, h, i, j] = table[u, h]`` with ``u = lut[clip(q_pos[b, i] - k_pos[b, j], -D, D) + D]``, or the last
    bucket where ``q_group[b, i] != k_group[b, j]`` (other chains, when groups are given).  ``table`` is fp32
    [buckets, H] (at most 256 buckets); ``lut`` int32 [2 D + 1], see :func:`clipped_buckets` and
    :func:`log_spaced_buckets` (entries outside the table count as its last bucket); positions and groups are integers
    [B, Nq] and [B, Nk].  The planes come in ``out_dtype`` (fp32 or bf16, default fp32) with rows on 16-byte boundaries,
    as :func:`cross_attention` takes them.  Gradient: :func:`relative_position_bias_backward`.
    """
    _require_inference(table)
    _require_cuda(table, q_pos, k_pos, lut)
    if table.dim() != 2 or table.dtype != torch.float32:
        raise RuntimeError("table must be fp32 [buckets, heads]")
    device = table.device
    qp, kp, lut, qg, kg = _bias_positions(device, q_pos, k_pos, lut, q_group, k_group)
    (b, nq), nk = qp.shape, kp.shape[1]
    buckets, h = table.shape
    out = padded_planes(b, h, nq, nk, device, _float_dtype(out_dtype or torch.float32, "out_dtype"))
    table = table.contiguous()
    launch(device, "bl_relative_position_bias", table.data_ptr(), qp.data_ptr(), kp.data_ptr(), lut.data_ptr(),
           lut.numel() // 2, ptr(qg), ptr(kg), b, h, nq, nk, buckets, out.data_ptr(), _lib.dtype_code(out.dtype),
           out.stride(0), out.stride(1), out.stride(2))
    return out


def relative_position_bias_backward(grad, q_pos, k_pos, lut, q_group=None, k_group=None, num_buckets=None):
    """Gradient of :func:`relative_position_bias` with respect to its table: fp32 [num_buckets, H] from the gradient of
    the planes, fp32 or bf16 [B, H, Nq, Nk] of any strides with contiguous rows.  Sums are fp32 in a fixed order."""
    _require_inference(grad)
    _require_cuda(grad, q_pos, k_pos, lut)
    if grad.dim() != 4 or num_buckets is None:
        raise RuntimeError("grad must be [B, H, Nq, Nk] and num_buckets be given")
    _float_dtype(grad.dtype, "grad")
    device = grad.device
    qp, kp, lut, qg, kg = _bias_positions(device, q_pos, k_pos, lut, q_group, k_group)
    b, h, nq, nk = grad.shape
    if tuple(qp.shape) != (b, nq) or tuple(kp.shape) != (b, nk):
        raise RuntimeError(f"positions must be [{b}, {nq}] and [{b}, {nk}]")
    if grad.stride(3) != 1:
        grad = grad.contiguous()
    dtable = torch.empty(num_buckets, h, device=device, dtype=torch.float32)
    nbytes = size_of("bl_relative_position_bias_workspace", b, h, nq, nk, num_buckets)
    work = _workspace(nbytes, device)
    launch(device, "bl_relative_position_bias_backward", grad.data_ptr(), _lib.dtype_code(grad.dtype), grad.stride(0),
           grad.stride(1), grad.stride(2), qp.data_ptr(), kp.data_ptr(), lut.data_ptr(), lut.numel() // 2, ptr(qg), ptr(kg),
           b, h, nq, nk, num_buckets, dtable.data_ptr(), work.data_ptr(), nbytes)
    return dtable


# ---------------------------------------------------------------------------
# Cross attention to states of another length
# ---------------------------------------------------------------------------
def _attention_rows(t, dtype, name, shape):
    """A [B, N, H, d] operand whose rows the kernels can read in place, copied only if they cannot."""
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise RuntimeError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    sb, si, sh, sd = t.stride()
    vec = 16 // t.element_size()
    if sd != 1 or sb % vec or si % vec or sh % vec or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


_NO_STRIDES = (0, 0, 0)


def _attention_args(q, k, v, bias, mask, inf, gate, scale):
    """(the filled argument structure, the tensors it points into)."""
    device = _require_cuda(q, k, v, bias, mask, gate)
    if q.dim() != 4 or k.dim() != 4:
        raise RuntimeError("q must be [B, Nq, H, d], k and v [B, Nk, Hk, d]")
    b, nq, h, d = q.shape
    nk, hk = k.shape[1], k.shape[2]
    dtype = _float_dtype(q.dtype, "q")
    if hk < 1 or h % hk:
        raise RuntimeError(f"{hk} key/value heads must divide the {h} query heads")
    if d % 8 or not 8 <= d <= 128:
        raise RuntimeError(f"head_dim must be a multiple of 8, at most 128, got {d}")
    q = _attention_rows(q, dtype, "q", (b, nq, h, d))
    k = _attention_rows(k, dtype, "k", (b, nk, hk, d))
    v = _attention_rows(v, dtype, "v", (b, nk, hk, d))
    gate_ptr = bias_ptr = mask_ptr = 0
    gate_stride = bias_stride = _NO_STRIDES
    share, mask_stride, mask_kind = 1, 0, 0
    if gate is not None:
        gate = _attention_rows(gate, dtype, "gate", (b, nq, h, d))
        gate_ptr, gate_stride = gate.data_ptr(), gate.stride()
    if bias is not None:
        if bias.dtype != dtype or bias.dim() != 4 or tuple(bias.shape[1:]) != (h, nq, nk) \
                or (b % bias.shape[0] if bias.shape[0] else b):
            raise RuntimeError(f"bias must be {dtype} [B', {h}, {nq}, {nk}] with B' dividing {b}, got {bias.dtype} "
                               f"{list(bias.shape)}")
        if bias.stride(3) != 1 and nk > 1:
            planes = padded_planes(*bias.shape, device, dtype)
            bias = planes.copy_(bias)
        bias_ptr, bias_stride, share = bias.data_ptr(), bias.stride(), b // bias.shape[0] if b else 1
    if mask is not None:
        if tuple(mask.shape) != (b, nk):
            raise RuntimeError(f"mask must be [{b}, {nk}], got {list(mask.shape)}")
        if inf is None:
            if mask.dtype != torch.bool:
                raise RuntimeError("a mask without inf must be bool (True: the key is kept)")
            mask_kind = 1
        else:
            mask = mask.float()
            mask_kind = 2
        if mask.stride(1) != 1 and nk > 1:
            mask = mask.contiguous()
        mask_ptr, mask_stride = mask.data_ptr(), mask.stride(0)
    x = _lib.CrossAttentionArgs()
    x.PACKING.pack_into(x, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), gate_ptr, bias_ptr, mask_ptr, *q.stride()[:3],
                        *k.stride()[:3], *v.stride()[:3], *gate_stride[:3], *bias_stride[:3], mask_stride, share,
                        b, h, hk, nq, nk, d, 0, 0, 0, d ** -0.5 if scale is None else scale,
                        inf if mask_kind == 2 else 0.0, _lib.dtype_code(dtype), mask_kind)
    return x, (q, k, v, bias, mask, gate)


class AttentionStats(NamedTuple):
    """What :func:`cross_attention_backward` takes from the forward call besides its output."""

    rows: torch.Tensor  # fp32 [2, B, H, Nq]: reference of a row's scores (-inf: no keys), log of the sum relative to it
    low: Optional[torch.Tensor]  # bf16 [B, Nq, H, d]: what rounding took from the output; None for fp32


def cross_attention(q, k, v, bias=None, mask=None, inf=None, gate=None, scale=None, return_lse=False):
    """Attention of Nq queries to Nk states: ``sigmoid(gate) * softmax(q k^T * scale + bias + mask term) v``.

    ``q`` (and the gate logits ``gate``) are [B, Nq, H, d], ``k`` and ``v`` [B, Nk, Hk, d] with Hk dividing H (head
    ``h`` reads key/value head ``h // (H / Hk)``); d a multiple of 8, at most 128; all fp32 or all bf16, any strides
    (copied only if the rows do not start on 16-byte boundaries), so overlapping windows of one tensor are a view.
    ``bias``: [B', H, Nq, Nk] of the same dtype, B' dividing B (sample ``b`` reads bias ``b // (B / B')``), fastest with
    rows on 16-byte boundaries (:func:`padded_planes`, :func:`relative_position_bias`).  ``mask`` [B, Nk]: bool, False
    keys are left out whatever they hold; or, with ``inf``, any real mask added as ``inf * (mask - 1)`` (upstream
    AttentionPairBias).  ``scale`` defaults to d ** -0.5.  A query whose keys are all left out gets zeros.

    Scores, softmax statistics and sums are fp32; bf16 probabilities are rounded to bf16 for the product with ``v``.
    ``q`` and the keys and values that a bool mask does not leave out are finite: fp32 products split them into two
    terms, so an infinity (or a magnitude of 2^127 and more) may give NaN where the formula has an infinity.  ``bias``
    may hold -inf.
    Returns [B, Nq, H, d], with ``return_lse`` also the :class:`AttentionStats` that :func:`cross_attention_backward`
    takes (``rows.sum(0)`` is the log-sum-exp of the scores).
    """
    _require_inference(q, k, v, bias, gate)
    x, kept = _attention_args(q, k, v, bias, mask, inf, gate, scale)
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    x.out = out.data_ptr()
    lse = None
    if return_lse:
        rows = torch.empty(2, x.batch, x.heads, x.nq, device=q.device, dtype=torch.float32)
        low = torch.empty_like(out) if out.dtype == torch.bfloat16 else None
        lse = AttentionStats(rows, low)
        x.lse, x.low = rows.data_ptr(), ptr(low)
    launch(q.device, "bl_cross_attention", x)
    del kept
    return (out, lse) if return_lse else out


def cross_attention_backward(grad, q, k, v, out, lse, bias=None, mask=None, inf=None, gate=None, scale=None,
                             need_bias_grad=True):
    """Gradients of :func:`cross_attention`: (dq, dk, dv, dbias, dgate), None where there is no such input.

    ``grad`` is the gradient of ``out``; the other arguments are the forward call's, ``out`` and ``lse`` (an
    :class:`AttentionStats`) its results.
    In bf16 p and ds are rounded to bf16 for their products.  ``dk`` and ``dv`` are summed over the query heads that share a key/value head and ``dbias`` ([B', H, Nq, Nk], rows on
    16-byte boundaries) over the samples that share a bias, in fp32 and in a fixed order: the same inputs give the same
    bits.  The mask is a constant.  ``need_bias_grad=False`` skips dbias.
    """
    _require_inference(grad, q, k, v, bias, gate)
    x, kept = _attention_args(q, k, v, bias, mask, inf, gate, scale)
    b, nq, h, d = q.shape
    device, dtype = q.device, q.dtype
    for name, t in (("grad", grad), ("out", out)):
        if tuple(t.shape) != (b, nq, h, d) or t.dtype != dtype or t.device != device:
            raise RuntimeError(f"{name} must be {dtype} {[b, nq, h, d]} on {device}")
    rows, low = lse
    if rows.dtype != torch.float32 or tuple(rows.shape) != (2, b, h, nq) or not rows.is_contiguous() \
            or rows.device != device:
        raise RuntimeError("lse must be the forward call's statistics (contiguous fp32 rows [2, B, H, Nq])")
    if low is not None and (low.shape != out.shape or low.dtype != torch.bfloat16 or dtype != torch.bfloat16
                            or not low.is_contiguous() or low.data_ptr() % 16 or low.device != device):
        raise RuntimeError("lse.low must be the forward call's contiguous bf16 [B, Nq, H, d]")
    grad, out = (t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
                 for t in (grad, out))
    x.out, x.lse, x.low = out.data_ptr(), rows.data_ptr(), ptr(low)
    dq = torch.empty(b, nq, h, d, device=device, dtype=dtype)
    dk = torch.empty(k.shape, device=device, dtype=dtype)
    dv = torch.empty(k.shape, device=device, dtype=dtype)
    dgate = None if gate is None else torch.empty(b, nq, h, d, device=device, dtype=dtype)
    dbias, ld = None, 0
    if bias is not None and need_bias_grad:
        dbias = padded_planes(*bias.shape, device, dtype)
        if b == 0:
            dbias.zero_()  # a bias that no sample reads
        ld = (x.nk + 7) // 8 * 8
    nbytes = size_of("bl_cross_attention_workspace", x)
    work = _workspace(nbytes, device)
    launch(device, "bl_cross_attention_backward", x, grad.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
           ptr(dbias), ld, ptr(dgate), work.data_ptr(), nbytes)
    del kept
    return dq, dk, dv, dbias, dgate
