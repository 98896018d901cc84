"""Relative position encoding and bias by buckets, and their gradients, against plain 64-bit forms.

Tolerances: a forward value is a sum of at most four fp32 weights (three roundings, each at most
2^-24 of the partial sum) rounded once to the output type (half a step, eps / 2 relative).  A
gradient element sums m fp32 values in chains of at most ``_chain`` additions: its error is at most
``_chain * 2^-24 * sum |x|`` (first order).
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FEATURES = ("residue_index", "asym_id", "entity_id", "token_index", "sym_id")


def features(b, n, seed, spread=3):
    """Chains of random length (some share an entity), ligand-like tokens of one residue; any integers are legal."""
    g = torch.Generator().manual_seed(seed)
    out = {k: torch.zeros(b, n, dtype=torch.int64) for k in FEATURES}
    for i in range(b):
        chains = int(torch.randint(1, spread + 1, (1,), generator=g))
        cuts = sorted(torch.randint(0, n + 1, (chains - 1,), generator=g).tolist())
        for c, (lo, hi) in enumerate(zip([0] + cuts, cuts + [n])):
            out["asym_id"][i, lo:hi], out["entity_id"][i, lo:hi], out["sym_id"][i, lo:hi] = c, c // 2, 2 * c
            out["residue_index"][i, lo:hi] = torch.arange(hi - lo) // (1 + c)  # c + 1 tokens of a residue
        out["token_index"][i] = torch.arange(n)
    return out


def one_hot(index, count):
    return (index[..., None] == torch.arange(count)).double()


def encode_features(f, r, s, fix_sym):
    """Algorithm 3's concatenated features [B, N, N, 4 r + 2 s + 7] in fp64."""
    d = {k: f[k][:, :, None] - f[k][:, None, :] for k in FEATURES}
    chain, residue, entity = d["asym_id"] == 0, d["residue_index"] == 0, d["entity_id"] == 0
    p = (d["residue_index"] + r).clamp(0, 2 * r).masked_fill(~chain, 2 * r + 1)
    t = (d["token_index"] + r).clamp(0, 2 * r).masked_fill(~(chain & residue), 2 * r + 1)
    c = (d["sym_id"] + s).clamp(0, 2 * s).masked_fill(~entity if fix_sym else chain, 2 * s + 1)
    return torch.cat([one_hot(p, 2 * r + 2), one_hot(t, 2 * r + 2), entity.double()[..., None],
                      one_hot(c, 2 * s + 2)], -1)


def cuda(f):
    return {k: v.cuda() for k, v in f.items()}


ENCODING_CASES = [
    # b, n, c, r, s, fix_sym
    (1, 1, 128, 32, 2, False),
    (2, 7, 128, 32, 2, False),
    (1, 33, 64, 32, 2, True),
    (1, 117, 128, 32, 2, False),
    (1, 200, 128, 32, 2, True),
    (3, 65, 132, 4, 1, False),
    (1, 40, 4, 0, 0, False),
    (1, 50, 260, 96, 16, True),
]


@pytest.mark.parametrize("b,n,c,r,s,fix", ENCODING_CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_encoding(b, n, c, r, s, fix, dtype):
    from boltz_lumi_b200 import kernels

    f = features(b, n, seed=n)
    w = torch.randn(c, 4 * r + 2 * s + 7, generator=torch.Generator().manual_seed(1))
    x = encode_features(f, r, s, fix)
    expected, size = x @ w.double().t(), x @ w.double().abs().t()
    out = kernels.relative_position_encoding(w.cuda(), *cuda(f).values(), r_max=r, s_max=s, fix_sym_check=fix,
                                             out_dtype=dtype)
    assert out.dtype == dtype and out.shape == (b, n, n, c)
    bound = 3 * 2.0 ** -24 * size + torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -20) * expected.abs() + 1e-30
    assert ((out.cpu().double() - expected).abs() <= bound).all()


def test_encoding_large_and_residual():
    """The 128-channel form (many pairs), adding into z; z is changed by the encoding alone."""
    from boltz_lumi_b200 import kernels

    b, n, c = 1, 300, 128
    f = features(b, n, seed=5)
    w = torch.randn(c, 139, generator=torch.Generator().manual_seed(2))
    x = encode_features(f, 32, 2, False)
    enc, size = x @ w.double().t(), x @ w.double().abs().t()
    z = torch.randn(b, n, n, c, generator=torch.Generator().manual_seed(3))
    zc = z.cuda()
    out = kernels.relative_position_encoding(w.cuda(), *cuda(f).values(), residual=zc)
    assert out.data_ptr() == zc.data_ptr()
    bound = 4 * 2.0 ** -24 * (size + z.double().abs())
    assert ((zc.cpu().double() - (enc + z.double())).abs() <= bound).all()
    plain = kernels.relative_position_encoding(w.cuda(), *cuda(f).values())
    assert ((plain.cpu().double() - enc).abs() <= 3 * 2.0 ** -24 * size).all()
    short = kernels.relative_position_encoding(w.cuda(), *cuda(f).values(), out_dtype=torch.bfloat16)
    assert torch.equal(short, plain.bfloat16())  # one rounding of the same fp32 sum


@pytest.mark.parametrize("b,n,c,r,s,fix", ENCODING_CASES + [(1, 300, 128, 32, 2, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_encoding_gradient(b, n, c, r, s, fix, dtype):
    from boltz_lumi_b200 import kernels

    f = features(b, n, seed=n + 1)
    dy = torch.randn(b, n, n, c, generator=torch.Generator().manual_seed(4)).to(dtype)
    x = encode_features(f, r, s, fix)
    expected = torch.einsum("bijc,bijf->cf", dy.double(), x)
    size = torch.einsum("bijc,bijf->cf", dy.double().abs(), x)
    fc = cuda(f)
    out = kernels.relative_position_encoding_backward(dy.cuda(), *fc.values(), r_max=r, s_max=s, fix_sym_check=fix)
    chain = min(b * n * n, 40 * n + 600)  # units of one group x 32 steps + partial tables
    assert ((out.cpu().double() - expected).abs() <= chain * 2.0 ** -24 * size).all()
    again = kernels.relative_position_encoding_backward(dy.cuda(), *fc.values(), r_max=r, s_max=s, fix_sym_check=fix)
    assert torch.equal(out, again)


def test_encoding_extreme_features():
    """Offsets past 32 bits clip like any other; features may be views and narrower integers."""
    from boltz_lumi_b200 import kernels

    n = 9
    f = features(1, n, seed=3, spread=1)
    f["residue_index"] = torch.tensor([[0, 1, 2 ** 40, -2 ** 40, 5, 5, 2 ** 31, -2 ** 31, 7]])
    w = torch.randn(128, 139, generator=torch.Generator().manual_seed(1))
    expected = encode_features(f, 32, 2, False) @ w.double().t()
    fc = cuda(f)
    fc["asym_id"] = fc["asym_id"].int()
    fc["sym_id"] = torch.stack([fc["sym_id"], fc["sym_id"]], -1)[..., 0]
    out = kernels.relative_position_encoding(w.cuda(), *fc.values())
    assert (out.cpu().double() - expected).abs().max() <= 3 * 2.0 ** -24 * 4 * w.abs().max()


def bias_reference(table, q_pos, k_pos, lut, q_group, k_group):
    d = lut.numel() // 2
    u = lut.long()[(q_pos[:, :, None] - k_pos[:, None, :]).clamp(-d, d) + d]
    last = table.shape[0] - 1
    u = torch.where((u < 0) | (u > last), last, u)
    if q_group is not None:
        u = u.masked_fill(q_group[:, :, None] != k_group[:, None, :], last)
    return u


BIAS_CASES = [
    # b, h, nq, nk, buckets, distance, groups
    (1, 16, 1, 1, 33, 128, True),
    (2, 4, 5, 130, 33, 128, False),
    (1, 3, 70, 517, 9, 4, True),
    (3, 16, 33, 7, 65, 32, True),
    (1, 5, 129, 1030, 200, 90, False),
    (2, 8, 200, 64, 1, 0, False),
]


def bias_inputs(b, h, nq, nk, buckets, distance, groups):
    from boltz_lumi_b200 import kernels

    g = torch.Generator().manual_seed(nq + nk)
    table = torch.randn(buckets, h, generator=g)
    lut = (kernels.log_spaced_buckets(buckets - 1, distance, device="cpu") if buckets == 33 else
           torch.randint(0, buckets, (2 * distance + 1,), generator=g, dtype=torch.int32))
    q_pos = torch.arange(nq).expand(b, nq) + torch.randint(-50, 50, (b, 1), generator=g)
    k_pos = torch.randint(-20, nq + 20, (b, nk), generator=g).sort(1).values
    qg = torch.randint(0, 2, (b, nq), generator=g) if groups else None
    kg = torch.randint(0, 2, (b, nk), generator=g) if groups else None
    return table, q_pos, k_pos, lut, qg, kg


def to_cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


@pytest.mark.parametrize("case", BIAS_CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_bias(case, dtype):
    from boltz_lumi_b200 import kernels

    args = bias_inputs(*case)
    u = bias_reference(*args)
    out = kernels.relative_position_bias(*to_cuda(*args), out_dtype=dtype)
    assert out.shape == (case[0], case[1], case[2], case[3]) and out.stride(2) % 8 == 0
    assert torch.equal(out.cpu(), args[0][u].permute(0, 3, 1, 2).to(dtype))


@pytest.mark.parametrize("case", BIAS_CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("padded", [False, True])
def test_bias_gradient(case, dtype, padded):
    from boltz_lumi_b200 import kernels

    args = bias_inputs(*case)
    b, h, nq, nk, buckets = case[:5]
    u = bias_reference(*args)
    dy = torch.randn(b, h, nq, nk, generator=torch.Generator().manual_seed(9)).to(dtype)
    x = one_hot(u, buckets)
    expected = torch.einsum("bhij,biju->uh", dy.double(), x)
    size = torch.einsum("bhij,biju->uh", dy.double().abs(), x)
    dyc = dy.cuda()
    if padded:
        wide = kernels.padded_planes(b, h, nq, nk, "cuda", dtype)
        wide.copy_(dyc)
        dyc = wide
    where = to_cuda(*args[1:])
    out = kernels.relative_position_bias_backward(dyc, *where, num_buckets=buckets)
    chain = 64 * 4 + b * nq * nk // 128 + 400  # a thread's rows and columns + its other units + partial sums
    assert ((out.cpu().double() - expected).abs() <= chain * 2.0 ** -24 * size).all()
    assert torch.equal(out, kernels.relative_position_bias_backward(dyc, *where, num_buckets=buckets))


@pytest.mark.parametrize("nk", [68, 70])
def test_wide_positions_and_groups(nk):
    """Positions and groups past 32 bits, in some samples and columns: offsets clip and groups differ in 64 bits."""
    from boltz_lumi_b200 import kernels

    g = torch.Generator().manual_seed(nk)
    b, h, nq, buckets, distance = 3, 5, 37, 9, 6
    table = torch.randn(buckets, h, generator=g)
    lut = torch.randint(0, buckets, (2 * distance + 1,), generator=g, dtype=torch.int32)
    q_pos, k_pos = torch.randint(-9, 9, (b, nq), generator=g), torch.randint(-9, 9, (b, nk), generator=g)
    q_pos[1] += 2 ** 40
    k_pos[1] += 2 ** 40  # far from zero, near one another
    k_pos[2, ::7] += 2 ** 33
    q_pos[2, ::5] += 2 ** 33
    q_pos[0, 3], k_pos[0, 5] = 2 ** 62, -2 ** 61
    q_group, k_group = torch.randint(0, 2, (b, nq), generator=g), torch.randint(0, 2, (b, nk), generator=g)
    q_group[0, ::3] += 2 ** 32  # equal to another group in the low word
    k_group[2, ::4] += 2 ** 32
    k_group[0, 10] = 2 ** 32
    for groups in ((None, None), (q_group, k_group)):
        args = (table, q_pos, k_pos, lut, *groups)
        u = bias_reference(*args)
        assert torch.equal(kernels.relative_position_bias(*to_cuda(*args)).cpu(), table[u].permute(0, 3, 1, 2))
        dy = torch.randint(-8, 9, (b, h, nq, nk), generator=g).float()  # exact sums
        expected = torch.einsum("bhij,biju->uh", dy.double(), one_hot(u, buckets))
        out = kernels.relative_position_bias_backward(dy.cuda(), *to_cuda(*args[1:]), num_buckets=buckets)
        assert torch.equal(out.cpu().double(), expected)


def test_bad_bucket_entries_count_as_last():
    """Entries of the bucket table outside the table never index past it."""
    from boltz_lumi_b200 import kernels

    table = torch.randn(5, 2)
    lut = torch.tensor([-1, 7, 2 ** 31 - 1, 4, -2 ** 31], dtype=torch.int32)
    pos = torch.arange(6)[None]
    args = (table, pos, pos, lut, None, None)
    out = kernels.relative_position_bias(*to_cuda(*args))
    assert torch.equal(out.cpu(), table[bias_reference(*args)].permute(0, 3, 1, 2))
    grad = kernels.relative_position_bias_backward(torch.ones(1, 2, 6, 6, device="cuda"), *to_cuda(*args[1:]),
                                                   num_buckets=5)
    assert grad[4].tolist() == [36.0, 36.0] and not grad[:4].any()


def test_log_spaced_buckets():
    from boltz_lumi_b200 import kernels

    lut = kernels.log_spaced_buckets(32, 128, device="cpu").tolist()
    at = lambda offset: lut[max(-128, min(128, offset)) + 128]  # noqa: E731
    assert [at(o) for o in range(8)] == list(range(8)) and [at(-o) for o in range(1, 8)] == list(range(17, 24))
    assert at(128) == at(1000) == 15 and at(-1000) == 31
    assert all(at(o) <= at(o + 1) for o in range(0, 128))
    for o in (9, 20, 63, 100):
        assert at(o) == 8 + int(math.log(o / 8) / math.log(16) * 8)
    one = kernels.log_spaced_buckets(16, 64, bidirectional=False, device="cpu").tolist()
    assert one[:65] == [0] * 65 and one[-1] == 15


def test_empty():
    from boltz_lumi_b200 import kernels

    w = torch.randn(128, 139, device="cuda")
    none = torch.zeros(1, 0, dtype=torch.int64, device="cuda")
    assert kernels.relative_position_encoding(w, *[none] * 5).shape == (1, 0, 0, 128)
    assert not kernels.relative_position_encoding_backward(torch.zeros(1, 0, 0, 128, device="cuda"), *[none] * 5).any()
    lut = kernels.clipped_buckets(4)
    q = torch.zeros(1, 3, dtype=torch.int64, device="cuda")
    assert kernels.relative_position_bias(torch.randn(9, 2, device="cuda"), q, none, lut).shape == (1, 2, 3, 0)
    assert not kernels.relative_position_bias_backward(torch.zeros(1, 2, 3, 0, device="cuda"), q, none, lut,
                                                       num_buckets=9).any()


def test_graph_capture_and_side_stream():
    """Captured and replayed on new values, and run on another stream, the gradients stay right."""
    from boltz_lumi_b200 import kernels

    args = bias_inputs(2, 8, 60, 200, 33, 128, True)
    table, *where = to_cuda(*args)
    u = bias_reference(*args)
    dy = torch.zeros(2, 8, 60, 200, device="cuda")
    kernels.relative_position_bias_backward(dy, *where, num_buckets=33)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        planes = kernels.relative_position_bias(table, *where)
        out = kernels.relative_position_bias_backward(dy, *where, num_buckets=33)
    for seed in (1, 2):
        new = torch.randn(2, 8, 60, 200, generator=torch.Generator().manual_seed(seed))
        dy.copy_(new)
        graph.replay()
        expected = torch.einsum("bhij,biju->uh", new.double(), one_hot(u, 33))
        assert (out.cpu().double() - expected).abs().max() < 1e-3
        assert torch.equal(planes.cpu(), args[0][u].permute(0, 3, 1, 2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = kernels.relative_position_bias_backward(dy, *where, num_buckets=33)
    side.synchronize()
    assert torch.equal(other, out)
