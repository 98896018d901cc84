"""Views, graphs, streams and long offsets at sizes that reach the bf16 tensor-core kernels (more than 64 queries, 64 keys
or more), forward and gradients."""

import pytest
import torch

from attention_reference import check, reference
from test_cross_attention_gpu import inputs, run, to_cuda

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
NQ, NK = 130, 200


def same(got, want):
    for n in want:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("share", [1, 2])
@pytest.mark.parametrize("d", [32, 72])
def test_views_of_operands(d, share, dtype):
    """Column blocks of one projection, head-first storage, every second row, operands off the 16-byte grid: the bits of
    the contiguous call."""
    b, h = 2, 4
    x = to_cuda(inputs(b, NQ, NK, h, h, d, dtype, share, True, "keep"))
    want = run(x)
    joint = torch.zeros(b, NK, 3, h, d, device="cuda", dtype=dtype)
    joint[:, :NQ, 0], joint[:, :, 1], joint[:, :, 2] = x["q"], x["k"], x["v"]
    same(run(dict(x, q=joint[:, :NQ, 0], k=joint[:, :, 1], v=joint[:, :, 2])), want)
    first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    same(run(dict(x, **{n: first(x[n]) for n in ("q", "k", "v", "gate", "dy")})), want)
    second = lambda t: torch.stack([t, t + 1], 2).flatten(1, 2)[:, ::2]  # noqa: E731
    same(run(dict(x, **{n: second(x[n]) for n in ("q", "k", "v", "gate")})), want)
    odd = lambda t: torch.empty(t.numel() + 1, device="cuda", dtype=dtype)[1:].view(t.shape).copy_(t)  # noqa: E731
    same(run(dict(x, **{n: odd(x[n]) for n in ("q", "k", "v", "gate", "dy")})), want)
    turned = x["bias"].transpose(2, 3).contiguous().transpose(2, 3)
    same(run(dict(x, bias=turned)), want)
    heads_last = x["bias"].permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
    same(run(dict(x, bias=heads_last)), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_planes_of_a_larger_bias(dtype):
    """A layer's slice of planes for several layers, rows on 16-byte boundaries."""
    from boltz_lumi_b200 import kernels

    x = to_cuda(inputs(2, NQ, NK, 2, 2, 48, dtype, 2, True, "tail"))
    want = run(x)
    planes = kernels.padded_planes(1, 6, NQ, NK, "cuda", dtype)
    planes.fill_(float("nan"))
    planes[:, 2:4] = x["bias"]
    same(run(dict(x, bias=planes[:, 2:4])), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_broadcast_operands(dtype):
    """Strides of 0 (one bias plane or row for all, keys of one sample for all heads): kernels without tensor maps take
    over where there are none."""
    b, h, d = 2, 4, 32
    x = inputs(b, NQ, NK, h, h, d, dtype, 1, False, "keep")
    for given in (dict(bias=x["bias"][:1, :1].expand(b, h, NQ, NK)), dict(bias=x["bias"][:, :, :1].expand(b, h, NQ, NK)),
                  dict(k=x["k"][:1].expand(b, NK, h, d), v=x["v"][:1].expand(b, NK, h, d)),
                  dict(q=x["q"][:, :, :1].expand(b, NQ, h, d))):
        on_device = {n: t.as_strided([m if s else 1 for m, s in zip(t.shape, t.stride())], t.stride()).cuda()
                     for n, t in given.items()}
        cuda = dict(to_cuda(x), **{n: t.expand(given[n].shape) for n, t in on_device.items()})
        check(run(cuda), *reference(**dict(x, **given)))


@pytest.mark.parametrize("dtype", TYPES)
def test_overlapping_windows(dtype):
    """Windows of 128 queries over 256 keys each, 128 apart, as views of one tensor."""
    h, d, n = 2, 64, 5
    g = torch.Generator().manual_seed(1)
    states = torch.randn(1, 128 * (n + 1), h, d, generator=g).to(dtype).cuda()
    keys = states.as_strided((n, 256, h, d), (128 * h * d, h * d, d, 1))
    x = dict(q=torch.randn(n, 128, h, d, generator=g).to(dtype).cuda(), k=keys, v=keys,
             dy=torch.randn(n, 128, h, d, generator=g).to(dtype).cuda())
    same(run(x), run(dict(x, k=keys.contiguous(), v=keys.contiguous())))


@pytest.mark.parametrize("share", [1, 2])
def test_graphs_and_streams(share):
    """Forward and backward captured twice, replayed on new inputs from two streams and next to an eager call."""
    sizes = (2, NQ, NK, 4, 2, 32, torch.bfloat16, share, True, "keep")
    x1, x2 = (to_cuda(inputs(*sizes, seed=s)) for s in (1, 2))
    want = [run(x1), run(x2)]
    buffers = [{n: t.clone() for n, t in x1.items()} for _ in range(2)]
    graphs, outs = [], []
    for buf in buffers:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(buf))
        graphs.append(graph)
    for buf, x in zip(buffers, (x2, x1)):
        for n, t in x.items():
            buf[n].copy_(t)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = run(x1)
    torch.cuda.synchronize()
    same(outs[0], want[1])
    same(outs[1], want[0])
    same(eager, want[0])


@pytest.mark.parametrize("nq", [70, 130])
def test_long_offsets(nq):
    """Key offsets past 2^31 elements through the tensor maps: the last keys are read where they are."""
    nk, h, d = 520, 1, 64
    stride = (2 ** 31 // (nk - 1) // 64 + 1) * 64  # elements between tokens: the last token starts past 2^31
    assert (nk - 1) * stride > 2 ** 31
    cache = torch.empty((nk - 1) * stride + d, device="cuda", dtype=torch.bfloat16)
    keys = cache.as_strided((1, nk, h, d), (nk * stride, stride, d, 1))
    x = to_cuda(inputs(1, nq, nk, h, h, d, torch.bfloat16, 1, True, "keep"))
    keys.copy_(x["k"])
    x["v"] = x["k"]
    same(run(dict(x, k=keys, v=keys)), run(x))
