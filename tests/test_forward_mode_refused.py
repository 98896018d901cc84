"""Inputs that carry a forward-mode tangent are refused instead of losing it, on the CPU: nothing is launched."""

import pytest
import torch
from torch.autograd import forward_ad

from boltz_lumi_b200 import autograd, kernels

Q, K, GATE = torch.ones(1, 3, 2, 8), torch.ones(1, 5, 2, 8), torch.ones(1, 3, 2, 8)
BIAS = torch.ones(1, 2, 3, 5)
FEATURES = [torch.zeros(1, 4, dtype=torch.int64)] * 5
LUT = torch.zeros(3, dtype=torch.int32)


@pytest.mark.parametrize("place", [kernels, autograd])
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", ["q", "k", "v", "bias", "gate"])
def test_cross_attention(place, grad, name):
    given = dict(q=Q, k=K, v=K, bias=BIAS, gate=GATE)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        given[name] = forward_ad.make_dual(given[name], torch.ones_like(given[name]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            place.cross_attention(**given)
        with pytest.raises(RuntimeError, match="CUDA"):  # inside the level, without a tangent
            place.cross_attention(Q, K, K, bias=BIAS, gate=GATE)


@pytest.mark.parametrize("place", [kernels, autograd])
def test_relative_positions(place):
    weight, table, pos = torch.ones(8, kernels.relative_position_columns()), torch.ones(2, 4), torch.zeros(1, 3, dtype=torch.int64)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        with pytest.raises(RuntimeError, match="forward-mode"):
            place.relative_position_encoding(dual(weight), *FEATURES)
        with pytest.raises(RuntimeError, match="forward-mode"):
            place.relative_position_bias(dual(table), pos, pos, LUT)


def test_gradients():
    with torch.no_grad(), forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        stats = kernels.AttentionStats(torch.zeros(2, 1, 2, 3), None)
        with pytest.raises(RuntimeError, match="forward-mode"):
            kernels.cross_attention_backward(dual(Q), Q, K, K, Q, stats)
        with pytest.raises(RuntimeError, match="forward-mode"):
            kernels.relative_position_encoding_backward(dual(torch.ones(1, 4, 4, 8)), *FEATURES)
        with pytest.raises(RuntimeError, match="forward-mode"):
            kernels.relative_position_bias_backward(dual(BIAS), torch.zeros(1, 3, dtype=torch.int64),
                                                    torch.zeros(1, 5, dtype=torch.int64), LUT, num_buckets=2)


def test_a_leaf_with_a_tangent():
    """With a gradient to record as well."""
    with forward_ad.dual_level():
        q = forward_ad.make_dual(Q.clone().requires_grad_(), torch.ones_like(Q))
        with pytest.raises(RuntimeError, match="forward-mode"):
            autograd.cross_attention(q, K, K)
