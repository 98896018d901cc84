"""Arguments of the cross attention that reach its entry points, on the CPU: nothing is launched."""

import pytest
import torch

from boltz_lumi_b200 import kernels


@pytest.mark.parametrize("biases", [0, 1, 3])
def test_empty_batch_with_a_bias(monkeypatch, biases):
    """No samples share any number of biases; one bias per sample is what the entry point hears."""
    monkeypatch.setattr(kernels, "_require_cuda", lambda *ts: ts[0].device)
    q, k = torch.zeros(0, 3, 4, 32), torch.zeros(0, 5, 2, 32)
    x, _ = kernels._attention_args(q, k, k, torch.zeros(biases, 4, 3, 5), None, None, None, None)
    assert (x.batch, x.bias_share) == (0, 1)
    with pytest.raises(RuntimeError, match="bias"):  # samples without any bias
        kernels._attention_args(torch.zeros(2, 3, 4, 32), *[torch.zeros(2, 5, 2, 32)] * 2, torch.zeros(0, 4, 3, 5), None, None,
                                None, None)
