"""Cross attention and its gradients against a 64-bit reference with derived error bounds (attention_reference)."""

import math

import pytest
import torch

from attention_reference import check, reference

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]


def inputs(b, nq, nk, h, hk, d, dtype, share=0, gate=True, mask="none", seed=0):
    """Seeded operands (CPU); ``share``: samples per bias, 0 for none."""
    g = torch.Generator().manual_seed(seed + 7 * nq + nk)
    randn = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    x = dict(q=randn(b, nq, h, d), k=randn(b, nk, hk, d), v=randn(b, nk, hk, d))
    if share:
        x["bias"] = randn(b // share, h, nq, nk)
    if gate:
        x["gate"] = randn(b, nq, h, d)
    if mask == "keep":
        x["mask"] = torch.rand(b, nk, generator=g) < 0.7
    elif mask == "tail":  # padded batch
        x["mask"] = torch.arange(nk)[None] < torch.randint(0, nk + 1, (b, 1), generator=g)
    elif mask == "add":
        x["mask"], x["inf"] = (torch.rand(b, nk, generator=g) < 0.7).float(), 1e6
    elif mask == "fraction":
        x["mask"], x["inf"] = torch.rand(b, nk, generator=g), 3.0
    x["dy"] = randn(b, nq, h, d)
    return x


def to_cuda(x):
    return {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in x.items()}


def run(x, backward=True):
    from boltz_lumi_b200 import kernels

    x = dict(x)
    dy = x.pop("dy", None)
    q, k, v = (x.pop(n) for n in "qkv")
    if not backward:
        return dict(out=kernels.cross_attention(q, k, v, **x))
    out, lse = kernels.cross_attention(q, k, v, **x, return_lse=True)
    grads = kernels.cross_attention_backward(dy, q, k, v, out, lse, **x)
    names = ("dq", "dk", "dv", "dbias", "dgate")
    return dict(out=out, lse=lse.rows, **{n: t for n, t in zip(names, grads) if t is not None})


CASES = [
    # b, nq, nk, h, hk, d, share, gate, mask
    (1, 1, 1, 1, 1, 8, 0, False, "none"),
    (1, 1, 200, 4, 4, 32, 1, True, "none"),
    (2, 3, 130, 8, 2, 64, 0, False, "tail"),
    (2, 16, 65, 2, 1, 128, 2, True, "keep"),
    (3, 17, 64, 2, 2, 24, 1, True, "add"),
    (6, 32, 128, 4, 4, 32, 3, True, "add"),
    (2, 37, 97, 3, 3, 48, 1, False, "keep"),
    (1, 64, 63, 2, 2, 16, 1, True, "fraction"),
    (1, 100, 257, 4, 1, 80, 1, False, "tail"),
    (4, 130, 70, 4, 2, 64, 4, True, "tail"),
    (1, 200, 301, 2, 2, 128, 0, False, "keep"),
    (2, 129, 515, 2, 2, 48, 2, True, "keep"),
    (1, 300, 1030, 1, 1, 56, 1, True, "tail"),
    (2, 5, 2100, 6, 3, 128, 1, True, "keep"),
    (1, 1, 5000, 16, 4, 64, 0, True, "tail"),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", TYPES)
def test_values_and_gradients(case, dtype):
    b, nq, nk, h, hk, d, share, gate, mask = case
    x = inputs(b, nq, nk, h, hk, d, dtype, share, gate, mask)
    value, bound = reference(**x)
    actual = run(to_cuda(x))
    check(actual, value, bound)
    again = run(to_cuda(x))
    assert all(torch.equal(actual[n], again[n]) for n in actual)  # fixed order of every sum
    x.pop("dy")
    check(run(to_cuda(x), backward=False), *reference(**x))


WINDOWS = [
    # b, nq, nk, h, hk, d, share, gate, mask: enough (bias, head) pairs to fill the GPU with windows
    (192, 32, 128, 4, 4, 32, 2, True, "add"),
    (90, 17, 33, 3, 3, 24, 1, False, "keep"),
    (128, 31, 127, 2, 2, 64, 0, True, "tail"),
    (160, 20, 96, 4, 4, 40, 2, True, "fraction"),
    (80, 32, 65, 4, 4, 8, 1, True, "none"),
    (60, 16, 128, 4, 2, 32, 1, True, "keep"),
]


@pytest.mark.parametrize("case", WINDOWS)
def test_windows(case):
    test_values_and_gradients(case, torch.float32)


def test_windows_left_out_keys_hold_anything():
    """NaN and infinities of left-out keys reach nothing, rows without keys and of lowest values follow the definition."""
    x = inputs(160, 24, 100, 4, 4, 32, torch.float32, 2, True, "keep")
    x["mask"][1] = False
    x["mask"][2, :64] = False
    x["mask"][2, 64] = True
    x["bias"][3, :, 0] = -math.inf
    x["bias"][4, :, 1] = torch.finfo(torch.float32).min
    clean = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in x.items()}
    bad = ~x["mask"]
    x["k"][bad], x["v"][bad] = math.nan, math.inf
    both = ~(x["mask"][0::2] | x["mask"][1::2])
    x["bias"] = torch.where(both[:, None, None], math.nan, x["bias"])
    actual, want = run(to_cuda(x)), run(to_cuda(clean))
    for n in actual:
        assert torch.equal(actual[n], want[n]), n
    assert not actual["dq"][1].any() and not actual["dk"][bad.cuda()].any() and not actual["dv"][bad.cuda()].any()
    check(actual, *reference(**clean))


LONG = [
    # few query tiles over many keys: the keys are divided
    (1, 70, 1500, 2, 1, 128, 0, True, "keep"),
    (2, 100, 2000, 2, 2, 32, 2, True, "add"),
    (1, 257, 4099, 1, 1, 64, 1, False, "tail"),
    (1, 128, 256, 3, 3, 96, 1, True, "fraction"),
    (3, 90, 777, 1, 1, 40, 3, True, "none"),
]


@pytest.mark.parametrize("case", LONG)
@pytest.mark.parametrize("dtype", TYPES)
def test_long_keys(case, dtype):
    test_values_and_gradients(case, dtype)


FEW = [
    (1, 20, 1100, 4, 2, 64, 1, True, "tail"),
    (2, 33, 700, 2, 2, 48, 2, False, "keep"),
    (1, 17, 4000, 8, 8, 128, 0, True, "add"),
    (20, 40, 300, 8, 8, 32, 5, True, "keep"),
]


@pytest.mark.parametrize("case", FEW)
@pytest.mark.parametrize("dtype", TYPES)
def test_few_queries_many_keys(case, dtype):
    test_values_and_gradients(case, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [48, 128])
def test_long_keys_left_out(dtype, d):
    """Whole parts of the keys left out, a sample with one key, one without, rows of -inf and of lowest values."""
    x = inputs(4, 100, 2050, 2, 2, d, dtype, 2, True, "keep")
    x["mask"][0, :1300] = False
    x["mask"][1, 600:] = False
    x["mask"][2] = False
    x["mask"][2, 2049] = True
    x["mask"][3] = False
    x["bias"][0, :, 0] = -math.inf
    x["bias"][0, :, 1] = torch.finfo(dtype).min
    x["bias"][0, :, 2, :1900] = -math.inf
    actual = run(to_cuda(x))
    assert not actual["out"][3].any() and (actual["lse"][0, 3] == -math.inf).all()
    check(actual, *reference(**x))


@pytest.mark.parametrize("d", [48, 128])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("share", [0, 1, 2])
def test_many_tiles(d, gate, share):
    """Every variant of the tensor-core kernels over rings that turn several times, in both directions."""
    test_values_and_gradients((2, 650, 710, 4, 2, d, share, gate, "keep"), torch.bfloat16)


@pytest.mark.parametrize("d", range(8, 129, 8))
def test_head_dims(d):
    test_values_and_gradients((2, 70, 80, 2, 1, d, 2, d % 16 == 0, "keep"), torch.bfloat16)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq,nk", [(3, 50), (24, 100), (130, 200)])
def test_scales(dtype, nq, nk):
    """A negative scale is that of the negated queries; scale 0 leaves the bias alone."""
    x = inputs(2, nq, nk, 2, 2, 32, dtype, 2, True, "keep")
    value, bound = reference(**{**x, "q": -x["q"]}, scale=0.3)
    value["dq"] = -value["dq"]
    check(run(to_cuda(dict(x, scale=-0.3))), value, bound)
    actual = run(to_cuda(dict(x, scale=0.0)))
    assert not actual["dq"].any() and not actual["dk"].any()
    check(actual, *reference(**x, scale=0.0))


@pytest.mark.parametrize("mask", ["none", "keep", "add"])
def test_more_keys_than_mask_bits(mask):
    test_values_and_gradients((2, 70, 65601, 1, 1, 16, 2, True, mask), torch.bfloat16)


@pytest.mark.parametrize("dtype", TYPES)
def test_unaligned_bias_of_long_rows(dtype):
    x = inputs(2, 140, 333, 2, 1, 48, dtype, 1, True, "fraction")
    value, bound = reference(**x)
    wide = torch.zeros(2, 2, 140, 335, dtype=dtype)
    wide[..., 1:334] = x["bias"]
    given = to_cuda(x)
    given["bias"] = wide.cuda()[..., 1:334]
    check(run(given), value, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq", [2, 90, 260])
def test_left_out_keys_hold_anything(dtype, nq):
    """NaN and infinities in the k, v and bias of left-out keys reach nothing; a sample without keys gives zeros."""
    x = inputs(4, nq, 150, 2, 2, 32, dtype, 2, True, "keep")
    x["mask"][1] = False
    x["mask"][2, :64] = False  # a whole tile
    x["mask"][2, 64] = True
    clean = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in x.items()}
    bad = ~x["mask"]
    x["k"][bad], x["v"][bad] = math.nan, math.inf
    both = ~(x["mask"][0::2] | x["mask"][1::2])  # a bias column that no sample of the pair reads
    x["bias"] = torch.where(both[:, None, None], math.nan, x["bias"].float()).to(dtype)
    actual, want = run(to_cuda(x)), run(to_cuda(clean))
    for n in actual:
        if n != "lse":
            assert torch.equal(actual[n], want[n]), n
            assert torch.isfinite(actual[n]).all(), n
    assert not actual["out"][1].any() and not actual["dq"][1].any() and not actual["dgate"][1].any()
    assert not actual["dk"][bad.cuda()].any() and not actual["dv"][bad.cuda()].any()
    assert (actual["lse"][0, 1] == -math.inf).all()
    check(actual, *reference(**clean))


@pytest.mark.parametrize("dtype", TYPES)
def test_bias_of_lowest_values_and_infinities(dtype):
    """Rows of -inf have no keys; rows of the type's lowest value are uniform; mixtures follow the definition."""
    x = inputs(1, 70, 90, 2, 2, 32, dtype, 1, False)
    low = torch.finfo(dtype).min
    x["bias"][0, :, 0] = -math.inf
    x["bias"][0, :, 1] = low
    x["bias"][0, :, 2, ::2] = low
    x["bias"][0, :, 3, 1::3] = -math.inf
    x["bias"][0, :, 4], x["bias"][0, :, 4, 7] = -math.inf, low
    x["q"][0, 1], x["q"][0, 4] = 0, 0  # logits of exactly the lowest value
    actual = run(to_cuda(x))
    value, bound = reference(**x)
    uniform = x["v"].double().mean(1)[0]
    assert ((value["out"][0, 1] - uniform).abs() < 1e-12).all()
    for n in ("out", "dq", "dk", "dv", "dbias"):
        assert torch.isfinite(actual[n]).all(), n
    # A logit that adds to the lowest value is lost to it in any format: bounds of those rows come from p = 1 / n.
    lost = 2.0 ** -19
    for n in ("out", "dq", "dbias"):
        rows = bound[n][:, [1, 4]] if n != "dbias" else bound[n][:, :, [1, 4]]
        assert rows.isfinite().all()
    size = {n: value[n].abs().amax() for n in value}
    u = torch.finfo(dtype).eps / 2
    for n in value:
        tol = torch.minimum(bound[n], (8 * u + 64 * lost) * size[n])
        over = (actual[n].double().cpu() - value[n]).abs() - tol
        assert not (over > 0).any(), (n, float(over.max()))
    assert not actual["out"][0, 0].any() and not actual["dq"][0, 0].any()
    one = x["v"][0, 7].double()  # a single key: v itself, to the 22 bits of a split fp32 operand
    assert ((actual["out"][0, 4].cpu().double() - one).abs() <= 2.0 ** -20 * one.abs()).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    """Slices of one projection, head-first storage, overlapping windows, odd offsets, broadcast and unaligned biases."""
    from boltz_lumi_b200 import kernels

    b, nq, nk, h, d = 2, 40, 70, 4, 32
    g = torch.Generator().manual_seed(3)
    joint = torch.randn(b, nk, 3 * h * d, generator=g).to(dtype).cuda()
    q_all, k, v = (t.unflatten(-1, (h, d)) for t in joint.split(h * d, -1))
    q = q_all[:, :nq]
    heads_first = torch.randn(b, h, nq, d, generator=g).to(dtype).cuda().transpose(1, 2)
    bias = torch.randn(1, h, 1, nk, generator=g).to(dtype).cuda().expand(1, h, nq, nk)
    dy = torch.randn(b, nq, h, d, generator=g).to(dtype).cuda()
    want = run(dict(q=q.contiguous(), k=k.contiguous(), v=v.contiguous(), gate=heads_first.contiguous(),
                    bias=bias.contiguous(), dy=dy))
    for given in (dict(q=q, k=k, v=v, gate=heads_first, bias=bias, dy=dy),
                  dict(q=q, k=k, v=v, gate=heads_first, bias=bias.transpose(2, 3).contiguous().transpose(2, 3), dy=dy)):
        got = run(given)
        assert all(torch.equal(got[n], want[n]) for n in want)
    odd = torch.empty(q.numel() + 1, device="cuda", dtype=dtype)[1:].view(q.shape).copy_(q)  # not on 16 bytes
    planes = torch.randn(1, h, nq, nk + 3, generator=g).to(dtype).cuda()[..., 1:nk + 1]
    got = run(dict(q=odd, k=k, v=v, bias=planes, dy=dy.transpose(1, 2).contiguous().transpose(1, 2)))
    want = run(dict(q=q, k=k, v=v, bias=planes.contiguous(), dy=dy))
    assert all(torch.equal(got[n], want[n]) for n in want)
    # Windows of 32 queries over 64 keys each, 32 apart: a view of one key tensor.
    keys = torch.randn(1, 32 * 6, h, d, generator=g).to(dtype).cuda()
    windows = keys.as_strided((5, 64, h, d), (32 * h * d, h * d, d, 1))
    queries = torch.randn(5, 32, h, d, generator=g).to(dtype).cuda()
    assert torch.equal(kernels.cross_attention(queries, windows, windows),
                       kernels.cross_attention(queries, windows.contiguous(), windows.contiguous()))


def test_empty():
    from boltz_lumi_b200 import kernels

    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    out, lse = kernels.cross_attention(torch.ones(2, 3, 4, 32, device="cuda"), z(2, 0, 4, 32), z(2, 0, 4, 32),
                                       return_lse=True)
    assert not out.any() and (lse.rows[0] == -math.inf).all()
    got = kernels.cross_attention_backward(out, torch.ones(2, 3, 4, 32, device="cuda"), z(2, 0, 4, 32), z(2, 0, 4, 32), out,
                                           lse)
    assert not got[0].any() and got[1].shape == (2, 0, 4, 32)
    k = torch.ones(2, 5, 4, 32, device="cuda")
    out, lse = kernels.cross_attention(z(2, 0, 4, 32), k, k, return_lse=True)
    got = kernels.cross_attention_backward(out, z(2, 0, 4, 32), k, k, out, lse)
    assert out.shape == (2, 0, 4, 32) and not got[1].any() and not got[2].any()
    assert kernels.cross_attention(z(0, 3, 4, 32), z(0, 5, 4, 32), z(0, 5, 4, 32)).shape == (0, 3, 4, 32)


def test_differences():
    """Directional derivatives of the fp32 forward by central differences.

    Along a unit-scale direction the loss sum(out w) has third derivatives of the order of its first; step h leaves a
    relative error of h^2, plus the forward's rounding (1e-6 of sum |out w|) over 2 h.
    """
    from boltz_lumi_b200 import kernels

    x = to_cuda(inputs(2, 20, 45, 2, 1, 16, torch.float32, 2, True, "keep"))
    dy = x.pop("dy")
    x = {n: t * 0.5 if t.is_floating_point() else t for n, t in x.items()}
    loss = lambda y: float((kernels.cross_attention(**y).double() * dy).sum())  # noqa: E731
    grads = run(dict(x, dy=dy))
    h = 2.0 ** -6
    scale = float((kernels.cross_attention(**x).double() * dy).abs().sum())
    for n in ("q", "k", "v", "bias", "gate"):
        g = torch.Generator().manual_seed(11)
        step = torch.randn(x[n].shape, generator=g).cuda()
        step = step / step.norm()
        slope = (loss(dict(x, **{n: x[n] + h * step})) - loss(dict(x, **{n: x[n] - h * step}))) / (2 * h)
        want = float((grads["d" + n].double() * step).sum())
        size = float(grads["d" + n].double().norm())
        assert abs(slope - want) <= h * h * size * 4 + 1e-6 * scale / h, (n, slope, want)


def test_bias_table_to_gradient_together():
    """Bucketed bias -> attention -> gradients of q, k, v and the bias table, through autograd, in one program."""
    from boltz_lumi_b200 import autograd, kernels

    b, nq, nk, h, d, buckets = 4, 50, 131, 4, 32, 33
    x = inputs(b, nq, nk, h, h, d, torch.float32, 0, True, "keep")
    g = torch.Generator().manual_seed(5)
    table = torch.randn(buckets, h, generator=g)
    q_pos, k_pos = torch.arange(nq).expand(2, nq), torch.arange(nk).expand(2, nk) * nq // nk
    q_group, k_group = (q_pos >= 30).long(), (k_pos >= 30).long()
    lut = kernels.log_spaced_buckets(buckets - 1, 40, device="cpu")

    leaves = {n: x[n].double().requires_grad_() for n in ("q", "k", "v", "gate")}
    wide = table.double().requires_grad_()
    index = lut.long()[(q_pos[:, :, None] - k_pos[:, None]).clamp(-40, 40) + 40]
    index = index.masked_fill(q_group[:, :, None] != k_group[:, None], buckets - 1)
    bias = wide[index].permute(0, 3, 1, 2).repeat_interleave(2, 0)
    z = torch.einsum("bihd,bjhd->bhij", leaves["q"], leaves["k"]) * d ** -0.5 + bias
    p = torch.softmax(z.masked_fill(~x["mask"][:, None, None], -math.inf), -1)
    y = torch.einsum("bhij,bjhd->bihd", p, leaves["v"]) * torch.sigmoid(leaves["gate"])
    (y * x["dy"].double()).sum().backward()

    mine = {n: x[n].cuda().requires_grad_() for n in ("q", "k", "v", "gate")}
    tab = table.cuda().requires_grad_()
    planes = autograd.relative_position_bias(tab, q_pos.cuda(), k_pos.cuda(), lut.cuda(), q_group.cuda(), k_group.cuda())
    out = autograd.cross_attention(mine["q"], mine["k"], mine["v"], bias=planes, mask=x["mask"].cuda(), gate=mine["gate"])
    out.backward(x["dy"].cuda())
    # The bounds of the pieces in fp32 are below 1e-4 of the largest element here (attention_reference's sums).
    for got, want in [(out, y), (tab.grad, wide.grad)] + [(mine[n].grad, leaves[n].grad) for n in mine]:
        assert (got.detach().double().cpu() - want.detach()).abs().max() <= 1e-4 * want.abs().max()


def test_autograd_matches_explicit_and_refuses_capture():
    from boltz_lumi_b200 import autograd, kernels

    x = to_cuda(inputs(2, 20, 45, 2, 1, 16, torch.bfloat16, 1, True, "keep"))
    dy = x.pop("dy")
    want = run(dict(x, dy=dy))
    leaves = {n: x[n].clone().requires_grad_() for n in ("q", "k", "v", "bias", "gate")}
    out = autograd.cross_attention(**leaves, mask=x["mask"])
    out.backward(dy)
    assert torch.equal(out, want["out"])
    assert all(torch.equal(leaves[n].grad, want["d" + n]) for n in leaves)
    with torch.no_grad():
        assert torch.equal(autograd.cross_attention(**leaves, mask=x["mask"]), want["out"])
    w = torch.randn(128, 139, device="cuda", requires_grad=True)
    f = [torch.arange(12, device="cuda")[None]] + [torch.zeros(1, 12, dtype=torch.int64, device="cuda")] * 4
    pair = autograd.relative_position_encoding(w, *f)
    pair.backward(torch.ones_like(pair))
    assert torch.equal(w.grad, kernels.relative_position_encoding_backward(torch.ones_like(pair), *f))
    # An eager graph of the same leaves is alive here (out, pair): recording under capture is refused before any launch.
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            autograd.cross_attention(**leaves, mask=x["mask"])
        with pytest.raises(RuntimeError, match="capture"):
            autograd.relative_position_encoding(w, *f)
        kept = kernels.relative_position_encoding(w.detach(), *f)
    graph.replay()
    assert torch.equal(kept, pair.detach())


def test_two_graphs_streams_and_replays():
    """Forward and backward captured twice, replayed on new inputs from two streams: no shared state."""
    x1 = to_cuda(inputs(2, 40, 130, 4, 2, 32, torch.bfloat16, 2, True, "keep", seed=1))
    x2 = to_cuda(inputs(2, 40, 130, 4, 2, 32, torch.bfloat16, 2, True, "keep", seed=2))
    want = [run(x1), run(x2)]
    buffers = [{n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in x1.items()} for _ in range(2)]
    graphs, outs = [], []
    for buf in buffers:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(buf))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for buf, x in zip(buffers, (x2, x1)):
        for n, t in x.items():
            if isinstance(t, torch.Tensor):
                buf[n].copy_(t)
    torch.cuda.synchronize()
    for graph, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for got, w in zip(outs, (want[1], want[0])):
        assert all(torch.equal(got[n], w[n]) for n in w)


def test_long_offsets():
    """Key offsets past 2^31 elements (a strided cache): the last keys are read where they are."""
    from boltz_lumi_b200 import kernels

    nk, h, d = 520, 1, 64
    stride = (2 ** 31 // (nk - 1) // 64 + 1) * 64  # elements between tokens: the last token starts past 2^31
    assert (nk - 1) * stride > 2 ** 31
    cache = torch.empty((nk - 1) * stride + d, device="cuda", dtype=torch.bfloat16)
    keys = cache.as_strided((1, nk, h, d), (nk * stride, stride, d, 1))
    x = inputs(1, 3, nk, h, h, d, torch.bfloat16, 0, False)
    keys.copy_(x["k"].cuda())
    assert torch.equal(kernels.cross_attention(x["q"].cuda(), keys, keys),
                       kernels.cross_attention(x["q"].cuda(), x["k"].cuda(), x["k"].cuda()))
