"""Modules on the cross attention and the relative position encoding: AttentionPairBias with keys of another length,
the installed atom transformer attention, RelativePositionEncoder."""

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu


def attention(c, heads, seed=0):
    from boltz_lumi_b200 import layers

    torch.manual_seed(seed)
    module = layers.AttentionPairBias(c, num_heads=heads, inf=1e6, compute_pair_bias=False)
    with torch.no_grad():
        for p in module.parameters():
            p.copy_(torch.randn(p.shape) * p.shape[-1] ** -0.5)
    return module.cuda().eval()


def eager(m, s, z, mask, k_in):
    """Upstream attentionv2's math in fp64 (pair_bias.py:22-36)."""
    b, nq, nk = s.shape[0], s.shape[1], k_in.shape[1]
    w = {n: p.double() for n, p in m.named_parameters()}
    s, k_in, z = s.double(), k_in.double(), z.double()
    split = lambda t, n: t.view(b, n, m.num_heads, -1)  # noqa: E731
    q = split(s @ w["proj_q.weight"].t() + w["proj_q.bias"], nq)
    k, v = (split(k_in @ w[f"proj_{x}.weight"].t(), nk) for x in "kv")
    g = torch.sigmoid(s @ w["proj_g.weight"].t())
    x = torch.einsum("bihd,bjhd->bhij", q, k) / m.head_dim ** 0.5
    x = x + z.permute(0, 3, 1, 2).repeat_interleave(b // z.shape[0], 0) + (m.inf * (mask.double() - 1))[:, None, None]
    o = torch.einsum("bhij,bjhd->bihd", x.softmax(-1), v).reshape(b, nq, -1)
    return (g * o) @ w["proj_o.weight"].t()


@pytest.mark.parametrize("b,bb,nq,nk,c,heads", [(6, 6, 32, 128, 128, 4), (4, 2, 32, 128, 128, 4), (2, 1, 5, 77, 64, 2),
                                                (1, 1, 130, 40, 384, 16)])
def test_attention_pair_bias_other_length(b, bb, nq, nk, c, heads):
    m = attention(c, heads)
    g = torch.Generator().manual_seed(3)
    s, k_in = torch.randn(b, nq, c, generator=g).cuda(), torch.randn(b, nk, c, generator=g).cuda()
    z = torch.randn(bb, nq, nk, heads, generator=g).cuda()
    mask = (torch.rand(b, nk, generator=g) < 0.8).float().cuda()
    with torch.inference_mode():
        y = m(s, z, mask, k_in, multiplicity=b // bb)
        r = m.attend(s, z.permute(0, 3, 1, 2), mask, k_in, residual=s)
    want = eager(m, s, z, mask, k_in)
    # fp32 throughout: the package's bound for its fp32 attention modules.
    assert (y.double() - want).abs().max() <= 1e-4
    assert (r.double() - want - s.double()).abs().max() <= 1e-4


def test_installed_atom_attention():
    """install(atom_attention=True) runs the windows of the atom encoder on the kernel; without it upstream's forward."""
    from boltz_lumi_b200 import adapters, layers

    class AttentionPairBias(layers.AttentionPairBias):
        def forward(self, s, z, mask, k_in, multiplicity=1):
            return eager(self, s, z, mask, k_in).float()

    model = nn.Module()
    model.structure_module = nn.Module()
    model.structure_module.score_model = nn.Module()
    model.structure_module.score_model.atom_attention_encoder = nn.Module()
    made = attention(128, 4)
    atom = AttentionPairBias(128, num_heads=4, compute_pair_bias=False)
    atom.load_state_dict(made.state_dict())
    model.structure_module.score_model.atom_attention_encoder.attention = atom
    model = model.cuda().eval()
    assert adapters.install(model) == 0
    model._b200_optimized = False
    assert adapters.install(model, atom_attention=True) == 1
    g = torch.Generator().manual_seed(4)
    s, k_in = torch.randn(8, 32, 128, generator=g).cuda(), torch.randn(8, 128, 128, generator=g).cuda()
    z, mask = torch.randn(8, 32, 128, 4, generator=g).cuda(), torch.ones(8, 128).cuda()
    with torch.inference_mode():
        y = atom(s, z, mask, k_in)
        assert (y - AttentionPairBias.forward(atom, s, z, mask, k_in)).abs().max() <= 1e-4
    adapters.uninstall(model)
    assert "forward" not in atom.__dict__


def test_relative_position_encoder_module():
    from boltz_lumi_b200 import layers

    n = 50
    feats = {k: torch.randint(0, 4, (2, n)).cuda() for k in ("asym_id", "entity_id", "sym_id")}
    feats["residue_index"] = torch.arange(n).expand(2, n).cuda() // 2
    feats["token_index"] = torch.arange(n).expand(2, n).cuda()
    module = layers.RelativePositionEncoder(64).cuda()
    assert tuple(module.linear_layer.weight.shape) == (64, 139)  # upstream's 4 (r + 1) + 2 (s + 1) + 1 columns
    y = module(feats)
    y.sum().backward()
    counts = module.linear_layer.weight.grad[0]
    assert int(counts[:66].sum()) == 2 * n * n and int(counts[66:132].sum()) == 2 * n * n  # every pair picks one of each
    assert int(counts[133:].sum()) == 2 * n * n
    module.eval()
    with torch.inference_mode():
        z = torch.randn(2, n, n, 64, device="cuda")
        before = z.clone()
        assert module.add_to(z, feats) is z and torch.allclose(z, before + y, atol=1e-5)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert torch.equal(module(feats), y.detach().bfloat16())
