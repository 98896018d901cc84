"""Refusals of the relative position operators, on the CPU: nothing is launched."""

import pytest
import torch

from boltz_lumi_b200 import _lib, kernels


def test_wrappers_refuse_cpu_tensors():
    f = [torch.zeros(1, 4, dtype=torch.int64)] * 5
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.relative_position_encoding(torch.zeros(128, 139), *f)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.relative_position_encoding_backward(torch.zeros(1, 4, 4, 128), *f)
    lut = kernels.clipped_buckets(2, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.relative_position_bias(torch.zeros(5, 2), f[0], f[0], lut)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.relative_position_bias_backward(torch.zeros(1, 2, 4, 4), f[0], f[0], lut, num_buckets=5)


def test_wrappers_refuse_gradients():
    w = torch.zeros(128, 139, requires_grad=True)
    with pytest.raises(RuntimeError, match="grad"):
        kernels.relative_position_encoding(w, *[torch.zeros(1, 4, dtype=torch.int64)] * 5)


def encoding(batch=1, n=4, channels=128, r=32, s=2, dtype=0, add=0, weight=None):
    return _lib.call("bl_relative_position_encoding", weight, 16, 16, 16, 16, 16, batch, n, channels, r, s, 0, None,
                     dtype, add, None)


@pytest.mark.parametrize("given,words", [
    (dict(channels=6), "multiple of 4"), (dict(channels=0), "multiple of 4"), (dict(r=97), "r_max"),
    (dict(r=-1), "r_max"), (dict(s=17), "s_max"), (dict(n=-1), "bad shape"), (dict(n=1 << 16), "bad shape"),
    (dict(r=1 << 33), "r_max"), (dict(dtype=5), "dtype"), (dict(add=1, dtype=1), "adding"), (dict(), "null"),
])
def test_encoding_entry_refuses(given, words):
    with pytest.raises(RuntimeError, match=words):
        encoding(**given)


def test_gradient_entries_refuse_small_workspaces():
    need = _lib.size_of("bl_relative_position_encoding_workspace", 1, 40, 128, 32, 2)
    assert need > 0 and need % (139 * 128 * 4) == 0
    with pytest.raises(RuntimeError, match=f"workspace of {need} bytes"):
        _lib.call("bl_relative_position_encoding_backward", 16, 0, 16, 16, 16, 16, 16, 1, 40, 128, 32, 2, 0, 16, 16,
                  need - 1, None)
    need = _lib.size_of("bl_relative_position_bias_workspace", 2, 8, 40, 70, 33)
    with pytest.raises(RuntimeError, match=f"workspace of {need} bytes"):
        _lib.call("bl_relative_position_bias_backward", 16, 0, 8, 8, 8, 16, 16, 16, 4, None, None, 2, 8, 40, 70, 33, 16,
                  16, need - 1, None)
    assert _lib.size_of("bl_relative_position_encoding_workspace", 0, 40, 128, 32, 2) == 0
    assert _lib.size_of("bl_relative_position_bias_workspace", 1, 8, 0, 70, 33) == 0


@pytest.mark.parametrize("heads,buckets,distance,groups,words", [
    (0, 5, 2, (None, None), "heads"), (4, 257, 2, (None, None), "buckets"), (1024, 256, 2, (None, None), "heads"),
    (4, 5, 9000, (None, None), "distance"), (4, 5, 2, (16, None), "groups"),
])
def test_bias_entry_refuses(heads, buckets, distance, groups, words):
    with pytest.raises(RuntimeError, match=words):
        _lib.call("bl_relative_position_bias", 16, 16, 16, 16, distance, *groups, 1, heads, 4, 4, buckets, 16, 0, 64, 16,
                  4, None)


def test_log_spaced_buckets_refuses_degenerate_tables():
    with pytest.raises(RuntimeError, match="max_distance"):
        kernels.log_spaced_buckets(32, 8, device="cpu")
    with pytest.raises(RuntimeError, match="num_buckets"):
        kernels.log_spaced_buckets(2, 64, device="cpu")
