"""Cross attention of empty batches and sizes beside a bias, a mask and a gate, forward, gradients and modules."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,biases,nq,nk", [(0, 0, 40, 70), (0, 1, 40, 70), (0, 3, 130, 200), (0, 2, 0, 5), (0, 2, 5, 0),
                                            (2, 1, 0, 5), (2, 2, 5, 0)])
def test_empty_with_bias(b, biases, nq, nk, dtype):
    from boltz_lumi_b200 import autograd

    ones = lambda *s: torch.ones(*s, device="cuda", dtype=dtype).requires_grad_()  # noqa: E731
    leaves = dict(q=ones(b, nq, 4, 32), k=ones(b, nk, 2, 32), v=ones(b, nk, 2, 32), bias=ones(biases, 4, nq, nk),
                  gate=ones(b, nq, 4, 32))
    for extra in (dict(), dict(mask=torch.ones(b, nk, device="cuda", dtype=torch.bool)),
                  dict(mask=torch.ones(b, nk, device="cuda"), inf=1e6)):
        out = autograd.cross_attention(**leaves, **extra)
        assert out.shape == (b, nq, 4, 32) and not out.any()
        grads = torch.autograd.grad(out, list(leaves.values()), torch.ones_like(out))
        for (n, t), g in zip(leaves.items(), grads):
            assert g.shape == t.shape and not g.any(), n


@pytest.mark.parametrize("biases", [0, 1])
def test_module_of_an_empty_batch(biases):
    from boltz_lumi_b200 import layers

    m = layers.AttentionPairBias(128, num_heads=4, compute_pair_bias=False).cuda().eval()
    s, k_in = torch.zeros(0, 32, 128, device="cuda"), torch.zeros(0, 128, 128, device="cuda")
    with torch.inference_mode():
        y = m(s, torch.zeros(biases, 32, 128, 4, device="cuda"), torch.ones(0, 128, device="cuda"), k_in)
        r = m.attend(s, torch.zeros(biases, 4, 32, 128, device="cuda"), None, k_in, residual=s)
    assert y.shape == r.shape == (0, 32, 128)


def test_installed_module_of_an_empty_batch():
    """The rebound atom attention answers an empty batch as upstream's forward does."""
    from torch import nn

    from boltz_lumi_b200 import adapters, layers

    model = nn.Module()
    model.structure_module = nn.Module()
    model.structure_module.score_model = nn.Module()
    model.structure_module.score_model.atom_attention_encoder = nn.Module()
    atom = layers.AttentionPairBias(128, num_heads=4, compute_pair_bias=False)
    model.structure_module.score_model.atom_attention_encoder.attention = atom
    model = model.cuda().eval()
    assert adapters.install(model, atom_attention=True) == 1
    with torch.inference_mode():
        for n in (0, 1):
            y = atom(torch.zeros(0, 32, 128, device="cuda"), torch.zeros(n, 32, 128, 4, device="cuda"),
                     torch.ones(0, 128, device="cuda"), torch.zeros(0, 128, 128, device="cuda"))
            assert y.shape == (0, 32, 128)
    adapters.uninstall(model)
