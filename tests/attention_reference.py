"""Cross attention in 64 bits with, beside every output, a bound of the kernels' rounding errors.

Unit roundoffs: u = eps / 2 of the tensors' type for every tensor that is written or handed to a product; fp32
accumulation in a product of n terms makes at most one error of 2^-23 of the running sum per mma step (16 terms in bf16;
8 terms, three steps each, in fp32, whose operands are split in tf32 pairs with at most 3 2^-21 lost per product).
A logit error e moves every probability of its row by at most a factor exp(2 e).
"""

import math

import torch


def _steps(dtype, n):
    if dtype == torch.bfloat16:
        return math.ceil(n / 16) * 2.0 ** -23
    return 3 * 2.0 ** -21 + 3 * math.ceil(n / 8) * 2.0 ** -23


def reference(q, k, v, dy=None, bias=None, mask=None, inf=None, gate=None, scale=None):
    """({name: value}, {name: bound}) in fp64 on the CPU; gradients where ``dy`` is given."""
    dtype, u = q.dtype, torch.finfo(q.dtype).eps / 2
    rounded = u if dtype == torch.bfloat16 else 0.0  # p, ds and do are rounded to the type for their products
    q, k, v, dy, bias, gate = (None if t is None else t.detach().double().cpu() for t in (q, k, v, dy, bias, gate))
    (b, nq, h, d), (nk, hk) = q.shape, k.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    keep = torch.ones(b, nk, dtype=torch.bool)
    add = torch.zeros(b, nk, dtype=torch.float64)
    if mask is not None and inf is None:
        keep = mask.cpu()
    elif mask is not None:
        add = inf * (mask.cpu().double() - 1)
    q = q.transpose(1, 2)  # [b, h, i, d]
    clean = lambda t: torch.where(keep[:, :, None, None], t, 0.0)  # noqa: E731  (left-out keys hold anything)
    k, v = (clean(t).transpose(1, 2).repeat_interleave(h // hk, 1) for t in (k, v))
    x = scale * q @ k.mT + add[:, None, None]
    size = scale * q.abs() @ k.abs().mT
    if bias is not None:
        wide = torch.where(keep.view(bias.shape[0], -1, nk).any(1)[:, None, None], bias, 0.0)
        x = x + wide.repeat_interleave(b // bias.shape[0], 0)
    x = x.masked_fill(~keep[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True) if nk else x.new_full((b, h, nq, 1), -math.inf)
    empty = top == -math.inf
    p = torch.exp(x - torch.where(empty, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(empty, 1.0, total)
    rel = 2.0 ** -19
    if nk:  # e of a row: rounding of the dot products and of the terms added to them
        magnitude = torch.where(p > 0, x.abs(), 0.0)
        rel = 2 * ((_steps(dtype, d) * size).amax(-1, keepdim=True) + 3 * 2.0 ** -24 * magnitude.amax(-1, keepdim=True)) \
            + 2.0 ** -19
    pv = p @ v.abs()
    o = p @ v
    sig = torch.ones_like(o) if gate is None else torch.sigmoid(gate.transpose(1, 2))
    y = o * sig
    row = lambda t: t.transpose(1, 2)  # noqa: E731  back to [b, i, h, d]
    e_y = (rel + rounded + _steps(dtype, nk)) * pv * sig + 1.01 * u * y.abs() + 2.0 ** -21 * y.abs()
    value, bound = dict(out=row(y)), dict(out=row(e_y))
    if dy is None:
        return value, bound
    dy = dy.transpose(1, 2)
    do = dy * sig
    u_do = 2.0 ** -21 + (u if gate is not None else 0.0)
    if gate is not None:
        value["dgate"] = row(dy * o * sig * (1 - sig))
        bound["dgate"] = row(dy.abs() * (1 - sig) * e_y + (u + 2.0 ** -20) * (dy * o * sig * (1 - sig)).abs())
    delta = (dy * y).sum(-1, keepdim=True)
    e_delta = (dy.abs() * e_y).sum(-1, keepdim=True) + 2.0 ** -20 * (dy * y).abs().sum(-1, keepdim=True)
    dp = do @ v.mT
    e_dp = (2.0 ** -16 + 2 * _steps(dtype, d)) * (do.abs() @ v.abs().mT)  # do as two terms of the type
    ds = p * (dp - delta)
    e_ds = rel * ds.abs() + p * (e_dp + e_delta) + 2.0 ** -22 * p * (dp.abs() + delta.abs())
    if bias is not None:
        group = lambda t: t.unflatten(0, (bias.shape[0], -1)).sum(1)  # noqa: E731
        value["dbias"] = group(ds)
        bound["dbias"] = group(e_ds) + 2.0 ** -21 * group(ds.abs()) + u * value["dbias"].abs()
    shared = lambda t: row(t.unflatten(1, (hk, -1)).sum(2))  # noqa: E731
    rows = nq * (h // hk)
    value["dv"] = shared(p.mT @ do)
    bound["dv"] = shared(((rel + 0 * p) * p).mT @ do.abs()) \
        + (rounded + u_do + _steps(dtype, rows)) * shared(p.mT @ do.abs()) + u * value["dv"].abs()
    e_ds = e_ds + rounded * ds.abs()
    value["dq"] = row(scale * ds @ k)
    bound["dq"] = row(scale * (e_ds + _steps(dtype, nk) * ds.abs()) @ k.abs()) + 2 * u * value["dq"].abs()
    value["dk"] = shared(scale * ds.mT @ q)
    bound["dk"] = shared(scale * (e_ds + _steps(dtype, rows) * ds.abs()).mT @ q.abs()) + 2 * u * value["dk"].abs()
    return value, bound


def check(actual, value, bound):
    """Every output within its bound (finite everywhere)."""
    for name, want in value.items():
        got = actual[name].detach().double().cpu()
        assert got.shape == want.shape, (name, got.shape, want.shape)
        assert torch.isfinite(got).all(), name
        over = (got - want).abs() - bound[name] * 1.001 - 1e-30
        assert not (over > 0).any(), (name, int((over > 0).sum()), float((got - want).abs().max()),
                                      float(((got - want).abs() / (bound[name] + 1e-30)).max()))
