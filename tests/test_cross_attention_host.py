"""Refusals of the cross attention, on the CPU: nothing is launched."""

import pytest
import torch

from boltz_lumi_b200 import _lib, kernels


def args(**given):
    x = _lib.CrossAttentionArgs()
    for n in ("q", "k", "v", "out"):
        setattr(x, n, 16)
    x.batch, x.heads, x.kv_heads, x.nq, x.nk, x.head_dim, x.bias_share = 2, 4, 2, 3, 5, 32, 1
    for n in ("q_stride", "k_stride", "v_stride"):
        getattr(x, n)[:] = (1024, 128, 32)
    x.scale = 1.0
    for n, value in given.items():
        if n.endswith("stride") and n != "mask_stride":
            getattr(x, n)[:] = value
        else:
            setattr(x, n, value)
    return x


@pytest.mark.parametrize("given,words", [
    (dict(dtype=3), "dtype"), (dict(heads=0), "bad shape"), (dict(nk=-1), "bad shape"), (dict(kv_heads=3), "divide"),
    (dict(head_dim=20), "head_dim"), (dict(head_dim=136), "head_dim"), (dict(head_dim=0), "head_dim"),
    (dict(mask_kind=4), "mask kind"), (dict(mask_kind=1), "mask is missing"), (dict(q=None), "null"), (dict(v=None), "null"),
    (dict(q=8), "16-byte"), (dict(k_stride=(1024, 126, 32)), "16-byte"), (dict(gate=16, gate_stride=(1, 4, 4)), "16-byte"),
    (dict(bias=16, bias_share=3), "samples per bias"), (dict(bias=16, bias_share=0), "samples per bias"),
    (dict(nq=1 << 40), "too large"),
])
def test_entry_refuses(given, words):
    with pytest.raises(RuntimeError, match=words):
        _lib.call("bl_cross_attention", args(**given), None)


def test_backward_entry_refuses():
    call = lambda x, dbias=None, ld=8, dgate=None, work=16, size=1 << 30: _lib.call(  # noqa: E731
        "bl_cross_attention_backward", x, 16, 16, 16, 16, dbias, ld, dgate, work, size, None)
    with pytest.raises(RuntimeError, match="null arguments"):
        _lib.call("bl_cross_attention_backward", None, 16, 16, 16, 16, None, 8, None, 16, 1 << 30, None)
    need = _lib.size_of("bl_cross_attention_workspace", args())
    assert need == 2 * 4 * 3 * 4
    with pytest.raises(RuntimeError, match=f"workspace of {need} bytes"):
        call(args(lse=16), size=need - 1)
    with pytest.raises(RuntimeError, match="null pointer"):
        call(args())  # no lse
    with pytest.raises(RuntimeError, match="null pointer"):
        call(args(lse=16), dbias=16)  # no bias
    with pytest.raises(RuntimeError, match="null pointer"):
        call(args(lse=16, gate=16, gate_stride=(1024, 128, 32)))  # no dgate
    with pytest.raises(RuntimeError, match="multiple of 8"):
        call(args(lse=16, bias=16), dbias=16, ld=5)
    assert _lib.size_of("bl_cross_attention_workspace", args(gate=16)) == need + 2 * 3 * 4 * 32 * 4
    assert _lib.size_of("bl_cross_attention_workspace", args(nq=0)) == 0


def test_wrappers_refuse():
    q, k = torch.zeros(2, 3, 4, 32), torch.zeros(2, 5, 2, 32)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.cross_attention(q, k, k)
    with pytest.raises(RuntimeError, match="grad"):
        kernels.cross_attention(q.requires_grad_(), k, k)
    with pytest.raises(RuntimeError, match="grad"):
        kernels.cross_attention_backward(q, q, k, k, q, q)


def shaped(**given):
    """_attention_args on CPU stand-ins (the device check passes them)."""
    q, k = torch.zeros(2, 3, 4, 32), torch.zeros(2, 5, 2, 32)
    call = dict(q=q, k=k, v=k, bias=None, mask=None, inf=None, gate=None, scale=None)
    call.update(given)
    return kernels._attention_args(**call)


@pytest.mark.parametrize("given,words", [
    (dict(q=torch.zeros(2, 3, 32)), "must be"), (dict(v=torch.zeros(2, 6, 2, 32)), "v must be"),
    (dict(k=torch.zeros(2, 5, 3, 32)), "divide"), (dict(k=torch.zeros(2, 5, 2, 32).bfloat16()), "k must be"),
    (dict(q=torch.zeros(2, 3, 4, 20), k=torch.zeros(2, 5, 2, 20), v=torch.zeros(2, 5, 2, 20)), "head_dim"),
    (dict(q=torch.zeros(2, 3, 4, 32).half()), "fp32 or bf16"), (dict(gate=torch.zeros(2, 3, 2, 32)), "gate"),
    (dict(bias=torch.zeros(3, 4, 3, 5)), "bias"), (dict(bias=torch.zeros(2, 4, 5, 3)), "bias"),
    (dict(bias=torch.zeros(2, 4, 3, 5).bfloat16()), "bias"), (dict(mask=torch.zeros(2, 5)), "bool"),
    (dict(mask=torch.zeros(2, 6, dtype=torch.bool)), "mask must be"),
])
def test_argument_checks(monkeypatch, given, words):
    monkeypatch.setattr(kernels, "_require_cuda", lambda *ts: ts[0].device)
    with pytest.raises(RuntimeError, match=words):
        shaped(**given)


def test_arguments_filled(monkeypatch):
    monkeypatch.setattr(kernels, "_require_cuda", lambda *ts: ts[0].device)
    bias = torch.zeros(1, 4, 3, 5)
    x, (q, k, v, b, mask, gate) = shaped(bias=bias, mask=torch.ones(2, 5), inf=7.0)
    assert (x.batch, x.heads, x.kv_heads, x.nq, x.nk, x.head_dim, x.bias_share) == (2, 4, 2, 3, 5, 32, 2)
    assert x.mask_kind == 2 and x.inf == 7.0 and x.mask_stride == 5 and x.dtype == _lib.BL_F32 and not x.gate
    assert abs(x.scale - 32 ** -0.5) < 1e-8 and list(x.q_stride) == [384, 128, 32] and x.bias == bias.data_ptr()
    odd = torch.zeros(2 * 3 * 4 * 32 + 1)[1:].view(2, 3, 4, 32)  # rows off the 16-byte grid are copied
    x, (q, *_) = shaped(q=odd)
    assert q.data_ptr() != odd.data_ptr() and q.data_ptr() % 16 == 0
    turned = torch.zeros(1, 4, 5, 3).transpose(2, 3)  # a bias without contiguous rows is laid out in padded rows
    x, (_, _, _, b, _, _) = shaped(bias=turned)
    assert list(x.bias_stride) == [4 * 3 * 8, 3 * 8, 8]


def test_install_rebinds_atom_attention_on_request():
    from torch import nn

    from boltz_lumi_b200 import adapters, layers

    model = nn.Module()
    model.structure_module = nn.Module()
    score = model.structure_module.score_model = nn.Module()
    for name in ("atom_attention_encoder", "atom_attention_decoder", "token_transformer"):
        part = nn.Module()
        part.attention = layers.AttentionPairBias(64, num_heads=4, compute_pair_bias=False)
        setattr(score, name, part)
    assert adapters.install(model, require_device=False) == 1
    adapters.uninstall(model)
    assert adapters.install(model, require_device=False, atom_attention=True) == 3
    assert "forward" in score.atom_attention_decoder.attention.__dict__
    adapters.uninstall(model)
    assert "forward" not in score.atom_attention_decoder.attention.__dict__


def test_cross_lengths_refused_on_cpu():
    from boltz_lumi_b200 import forwards, layers

    m = layers.AttentionPairBias(64, num_heads=4, compute_pair_bias=False).eval()
    with torch.inference_mode(), pytest.raises(RuntimeError, match="cross attention covers"):
        forwards.attend_with_bias(m, torch.zeros(1, 3, 64), torch.zeros(1, 4, 3, 5), torch.ones(1, 5), torch.zeros(1, 5, 64))


def test_relative_position_encoder_refuses_cyclic():
    from boltz_lumi_b200 import layers

    with pytest.raises(NotImplementedError, match="cyclic"):
        layers.RelativePositionEncoder(128, cyclic_pos_enc=True)
