"""Timed cases of the relative-position and cross-attention operators, with their plain forms.

Three operators, each with its gradient:

* ``encoding``: the relative position encoding of a pair tensor (AlphaFold 3 supplementary
  Algorithm 3, upstream Boltz's ``RelativePositionEncoder``): every token pair picks one learned
  row by clipped residue offset, one by clipped token offset, one by clipped chain-copy offset and
  one if the entities agree; their sum is the pair's row of C channels.
* ``bias``: a learned relative position bias of attention heads by buckets of the clipped (or
  log-spaced) offset, head-major, queries and keys of different lengths.
* ``attention``: gated cross attention of queries to states of another length, with an additive
  bias that the samples of one input share and a key mask.

``run`` computes the plain form (elementary torch operations in fp32) or, with ``own``, calls the
package's kernels.
"""

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_R_MAX, _S_MAX = 32, 2
_BUCKETS, _DISTANCE = 32, 128


def _encoding(name, dtype, b, n, grad):
    return dict(name=name, op="encoding", dtype=dtype, grad=grad, b=b, n=n, c=128)


def _bias(name, dtype, b, h, nq, nk, grad):
    return dict(name=name, op="bias", dtype=dtype, grad=grad, b=b, h=h, nq=nq, nk=nk)


def _attention(name, dtype, b, bb, nq, nk, h, hk, d, mask, gate, grad):
    """``bb``: biases of the batch (0: no bias; each serves b / bb samples); ``hk``: key/value
    heads; ``mask``: "none", "keep" (left-out keys) or "inf" (additive inf * (mask - 1))."""
    return dict(name=name, op="attention", dtype=dtype, grad=grad, b=b, bb=bb, nq=nq, nk=nk, h=h, hk=hk, d=d,
                mask=mask, gate=gate)


def listed():
    return [
        # The pair tensor of one Pairformer input at the benchmarked 512 tokens, fp32 as z is stored.
        _encoding("encoding_f32_512", "f32", 1, 512, False),
        # A small protein (117 tokens) under bf16 autocast: latency counts.
        _encoding("encoding_bf16_117", "bf16", 1, 117, False),
        # Weight gradient at 384 residues + a 40-atom ligand, fp32 pair gradients.
        _encoding("encoding_grad_f32_424", "f32", 1, 424, True),
        # Bias of the token transformer's 16 heads for a small protein.
        _bias("bias_f32_117", "f32", 1, 16, 117, 117, False),
        # Tokens of a large complex against its atoms (4 per token, ragged), bf16 planes.
        _bias("bias_bf16_2048_8190", "bf16", 1, 16, 2048, 8190, False),
        # Table gradient from fp32 bias gradients, two inputs of a training batch.
        _bias("bias_grad_f32_768_1134", "f32", 2, 16, 768, 1134, True),
        # One query token per sample reading long encoder states: the step of serving.
        _attention("attention_step_bf16", "bf16", 5, 0, 1, 16384, 16, 4, 64, "keep", True, False),
        # The atom transformer's windows (32 queries to 128 keys), 128 windows x 5 diffusion samples.
        _attention("attention_windows_f32", "f32", 640, 128, 32, 128, 4, 4, 32, "inf", True, False),
        # The same windows in training: 96 windows, 4 noise levels each, gradients of all inputs.
        _attention("attention_windows_f32_train", "f32", 384, 96, 32, 128, 4, 4, 32, "inf", True, True),
        # Tokens attending to the atoms of a large complex, one bias for two samples.
        _attention("attention_tokens_bf16", "bf16", 2, 1, 2048, 8190, 16, 16, 48, "keep", True, False),
        # The same in training at a crop of 384 tokens + its atoms.
        _attention("attention_tokens_bf16_train", "bf16", 2, 1, 384, 1734, 16, 16, 48, "keep", True, True),
        # Shared key/value heads, wide heads, no bias: encoder states of a text or sequence model.
        _attention("attention_shared_bf16_train", "bf16", 4, 0, 777, 2048, 16, 4, 128, "keep", False, True),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["encoding", "bias", "attention", "attention"])
    dtype, grad = rng.choice(["f32", "bf16"]), rng.random() < 0.5
    if op == "encoding":
        case = _encoding("", dtype, rng.choice([1, 1, 2]), _log(rng, 16, 512), grad)
    elif op == "bias":
        b, h = rng.choice([1, 1, 2, 4]), rng.choice([4, 8, 16])
        nq, nk = _log(rng, 1, 2048), _log(rng, 16, 8192)
        while b * h * nq * nk > 16 * 2048 * 4096:
            nq = (nq + 1) // 2
        case = _bias("", dtype, b, h, nq, nk, grad)
    else:
        h = rng.choice([4, 8, 16])
        hk = rng.choice([h, h, h // 4])
        d = rng.choice([24, 32, 48, 64, 128])
        nq, nk = _log(rng, 1, 2048), _log(rng, 32, 8192)
        bb, share = _log(rng, 1, 256), rng.choice([1, 1, 2, 5])
        budget = 4_000_000_000 if grad or dtype == "f32" else 16_000_000_000
        while (bb * share * h * nq * nk * d > budget or bb * share * h * (nk + nq) * d > 60_000_000
               or bb * h * nq * nk > 64_000_000):
            if bb > 1:
                bb = (bb + 1) // 2
            elif nq > 256:
                nq = (nq + 1) // 2
            else:
                nk = (nk + 1) // 2
        biased = rng.random() < 0.7
        case = _attention("", dtype, bb * share, bb if biased else 0, nq, nk, h, hk, d,
                          rng.choice(["none", "keep", "keep", "inf"]), rng.random() < 0.6, grad)
    del case["name"]
    return case


def _tokens(b, n, g):
    """Token features of ``b`` inputs of ``n`` tokens: chains of random length (copies of an entity
    among them) and, from 32 tokens on, a ligand at the end whose atoms share one residue index."""
    asym, residue, entity, token, sym = (torch.zeros(b, n, dtype=torch.int64) for _ in range(5))
    for i in range(b):
        ligand = min(40, n // 8) if n >= 32 else 0
        chains = int(torch.randint(1, 4, (1,), generator=g))
        cuts = torch.sort(torch.randint(0, n - ligand + 1, (chains - 1,), generator=g)).values.tolist()
        begin = 0
        for c, end in enumerate(cuts + [n - ligand]):
            asym[i, begin:end], entity[i, begin:end], sym[i, begin:end] = c, c // 2, c % 2
            residue[i, begin:end] = torch.arange(end - begin)
            begin = end
        asym[i, n - ligand:], entity[i, n - ligand:] = chains, chains
        token[i] = torch.arange(n)
    return [t.cuda() for t in (residue, asym, entity, token, sym)]


def _log_spaced():
    """Bucket of each offset clipped to [-_DISTANCE, _DISTANCE]: _BUCKETS / 2 per sign; half of those one
    offset each, the others log-spaced."""
    half, exact = _BUCKETS // 2, _BUCKETS // 4
    lut = []
    for offset in range(-_DISTANCE, _DISTANCE + 1):
        m = abs(offset)
        if m >= exact:
            m = min(half - 1, exact + int(math.log(m / exact) / math.log(_DISTANCE / exact) * (half - exact)))
        lut.append(m + (half if offset < 0 else 0))
    return torch.tensor(lut, dtype=torch.int32)


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def randn(*shape, t=dtype):
        return torch.randn(*shape, generator=g, device="cuda").to(t)

    s = dict(case=case)
    if case["op"] == "encoding":
        b, n, c = case["b"], case["n"], case["c"]
        s["tokens"] = _tokens(b, n, host)
        s["weight"] = randn(c, 4 * (_R_MAX + 1) + 2 * (_S_MAX + 1) + 1, t=torch.float32) * 0.1
        if case["grad"]:
            s["grad"] = randn(b, n, n, c)
    elif case["op"] == "bias":
        b, h, nq, nk = case["b"], case["h"], case["nq"], case["nk"]
        s["table"] = randn(_BUCKETS + 1, h, t=torch.float32)
        s["lut"] = _log_spaced().cuda()
        # Tokens, and atoms in runs of one residue each; two chains.
        s["q_pos"] = torch.arange(nq, device="cuda").expand(b, nq).contiguous()
        s["k_pos"] = (torch.arange(nk, device="cuda") * nq // nk).expand(b, nk).contiguous()
        cut = torch.randint(0, nq + 1, (b, 1), generator=host).cuda()
        s["q_group"], s["k_group"] = (s["q_pos"] >= cut).long(), (s["k_pos"] >= cut).long()
        if case["grad"]:
            s["grad"] = randn(b, h, nq, nk)
    else:
        b, nq, nk, h, hk, d = (case[x] for x in ("b", "nq", "nk", "h", "hk", "d"))
        s["q"], s["k"], s["v"] = randn(b, nq, h, d), randn(b, nk, hk, d), randn(b, nk, hk, d)
        s["gate"] = randn(b, nq, h, d) if case["gate"] else None
        s["bias"] = None
        if case["bb"]:  # planes with rows of whole 16-byte groups, as the package's bias producers lay them out
            planes = torch.zeros(case["bb"], h, nq, (nk + 7) // 8 * 8, device="cuda", dtype=dtype)
            for i in range(case["bb"]):
                planes[i, ..., :nk] = randn(h, nq, nk)
            s["bias"] = planes[..., :nk]
        s["mask"] = None
        if case["mask"] != "none":  # padded batch: each sample has its own number of real keys
            real = torch.randint(nk - nk // 8, nk + 1, (b, 1), generator=host).cuda()
            s["mask"] = torch.arange(nk, device="cuda") < real
        s["inf"] = None
        if case["mask"] == "inf":
            s["mask"], s["inf"] = s["mask"].float(), 1e6
        if case["grad"]:
            s["grad"] = randn(b, nq, h, d)
    return s


def _pick(tokens):
    """The four picks of every pair: rows of weight^T (residue, token, chain copy) and whether the entities agree."""
    residue, asym, entity, token, sym = tokens
    chain = asym[:, :, None] == asym[:, None, :]
    same = residue[:, :, None] == residue[:, None, :]
    agree = entity[:, :, None] == entity[:, None, :]
    offset = lambda t, m: torch.clamp(t[:, :, None] - t[:, None, :] + m, 0, 2 * m)  # noqa: E731
    apart = 2 * _R_MAX + 1
    p = torch.where(chain, offset(residue, _R_MAX), apart)
    t = torch.where(chain & same, offset(token, _R_MAX), apart) + apart + 1
    c = torch.where(chain, 2 * _S_MAX + 1, offset(sym, _S_MAX)) + 2 * (apart + 1) + 1
    return p, t, agree, c


def _encoding_plain(s):
    rows = s["weight"].t().contiguous()
    p, t, agree, c = _pick(s["tokens"])
    e = 4 * (_R_MAX + 1)
    y = rows[p] + rows[t] + agree[..., None] * rows[e] + rows[c]
    return y.to(_DTYPES[s["case"]["dtype"]])


def _encoding_grad_plain(s):
    p, t, agree, c = _pick(s["tokens"])
    dy = s["grad"].double().flatten(0, 2)
    out = dy.new_zeros(s["weight"].shape[1], s["weight"].shape[0])
    for pick in (p, t, c):
        out.index_add_(0, pick.flatten(), dy)
    out[4 * (_R_MAX + 1)] += (dy * agree.flatten()[:, None]).sum(0)
    return out.t().float()


def _buckets(s):
    d = torch.clamp(s["q_pos"][:, :, None] - s["k_pos"][:, None, :], -_DISTANCE, _DISTANCE) + _DISTANCE
    same = s["q_group"][:, :, None] == s["k_group"][:, None, :]
    return torch.where(same, s["lut"][d].long(), _BUCKETS)


def _bias_plain(s):
    return s["table"][_buckets(s)].permute(0, 3, 1, 2).contiguous().to(_DTYPES[s["case"]["dtype"]])


def _bias_grad_plain(s):
    dy = s["grad"].double().transpose(0, 1).flatten(1)
    out = dy.new_zeros(_BUCKETS + 1, dy.shape[0])
    out.index_add_(0, _buckets(s).flatten(), dy.t())
    return out.float()


def _logits(s, q, k):
    """[B, H, Nq, Nk] logits and the plain probabilities' operands, in the dtype of q and k."""
    case = s["case"]
    x = torch.matmul(q, k.transpose(-1, -2)) * case["d"] ** -0.5
    if s["bias"] is not None:
        x = (x.unflatten(0, (case["bb"], -1)) + s["bias"].to(x.dtype).unsqueeze(1)).flatten(0, 1)
    if s["mask"] is not None:
        if s["inf"] is None:
            x = torch.where(s["mask"][:, None, None, :], x, -math.inf)
        else:
            x = x + s["inf"] * (s["mask"].to(x.dtype)[:, None, None, :] - 1)
    return x


def _attention_plain(s):
    case, dtype = s["case"], s["q"].dtype
    share = case["h"] // case["hk"]
    q, k, v = (s[x].float().transpose(1, 2) for x in ("q", "k", "v"))
    if share > 1:
        k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    x = _logits(s, q, k)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = torch.matmul(p, v)
    sig = None
    y = o
    if s["gate"] is not None:
        sig = 1 / (1 + torch.exp(-s["gate"].float().transpose(1, 2)))
        y = o * sig
    out = dict(out=y.transpose(1, 2).to(dtype))
    if not case["grad"]:
        return out
    dy = s["grad"].float().transpose(1, 2)
    do = dy if sig is None else dy * sig
    if sig is not None:
        out["dgate"] = (dy * o * sig * (1 - sig)).transpose(1, 2).to(dtype)
    dv = torch.matmul(p.transpose(-1, -2), do)
    dp = torch.matmul(do, v.transpose(-1, -2))
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    if s["bias"] is not None:
        out["dbias"] = ds.unflatten(0, (case["bb"], -1)).sum(1).to(dtype)
    scale = case["d"] ** -0.5
    dq, dk = torch.matmul(ds, k) * scale, torch.matmul(ds.transpose(-1, -2), q) * scale
    if share > 1:
        dk, dv = (t.unflatten(1, (-1, share)).sum(2) for t in (dk, dv))
    out["dq"], out["dk"], out["dv"] = (t.transpose(1, 2).to(dtype) for t in (dq, dk, dv))
    return out


def _run_own(s):
    from boltz_lumi_b200 import kernels

    case = s["case"]
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "encoding":
        if case["grad"]:
            return kernels.relative_position_encoding_backward(s["grad"], *s["tokens"], r_max=_R_MAX, s_max=_S_MAX)
        return kernels.relative_position_encoding(s["weight"], *s["tokens"], r_max=_R_MAX, s_max=_S_MAX,
                                                  out_dtype=dtype)
    if case["op"] == "bias":
        where = (s["q_pos"], s["k_pos"], s["lut"], s["q_group"], s["k_group"])
        if case["grad"]:
            return kernels.relative_position_bias_backward(s["grad"], *where, num_buckets=_BUCKETS + 1)
        return kernels.relative_position_bias(s["table"], *where, out_dtype=dtype)
    args = (s["q"], s["k"], s["v"])
    given = dict(bias=s["bias"], mask=s["mask"], inf=s["inf"], gate=s["gate"])
    if not case["grad"]:
        return dict(out=kernels.cross_attention(*args, **given))
    out, lse = kernels.cross_attention(*args, **given, return_lse=True)
    grads = kernels.cross_attention_backward(s["grad"], *args, out, lse, **given)
    names = ("dq", "dk", "dv", "dbias", "dgate")
    return dict(out=out, **{n: t for n, t in zip(names, grads) if t is not None})


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] == "encoding":
        return _encoding_grad_plain(state) if case["grad"] else _encoding_plain(state)
    if case["op"] == "bias":
        return _bias_grad_plain(state) if case["grad"] else _bias_plain(state)
    return _attention_plain(state)


def work(case):
    size = {"f32": 4, "bf16": 2}[case["dtype"]]
    if case["op"] == "encoding":
        pairs, rows = case["b"] * case["n"] ** 2, 4 * (_R_MAX + 1) + 2 * (_S_MAX + 1) + 1
        return dict(bytes=pairs * case["c"] * size + rows * case["c"] * 4 + 5 * 8 * case["b"] * case["n"],
                    flops=3 * pairs * case["c"])
    if case["op"] == "bias":
        planes = case["b"] * case["h"] * case["nq"] * case["nk"]
        return dict(bytes=planes * size + (_BUCKETS + 1) * case["h"] * 4 + 16 * case["b"] * (case["nq"] + case["nk"]),
                    flops=planes if case["grad"] else 0)
    b, bb, nq, nk, h, hk, d = (case[x] for x in ("b", "bb", "nq", "nk", "h", "hk", "d"))
    rows, keys, scores = b * nq * h * d, b * nk * hk * d, b * h * nq * nk
    once = 2 + bool(case["gate"])  # q, out and the gate logits
    elements = once * rows + 2 * keys + bb * h * nq * nk
    if case["grad"]:  # the upstream gradient and the gradient of every input
        elements += rows + (1 + bool(case["gate"])) * rows + 2 * keys + bb * h * nq * nk
    masks = {"none": 0, "keep": b * nk, "inf": 4 * b * nk}[case["mask"]]
    return dict(bytes=elements * size + masks, flops=(14 if case["grad"] else 4) * scores * d)


# ---------------------------------------------------------------------------
# The operators from their definitions, in 64 bits
# ---------------------------------------------------------------------------
def _hot(index, count):
    return (index[..., None] == torch.arange(count, device=index.device)).double()


def _exact_features(tokens, i):
    """One-hot features [N, N, 139] of input ``i``: Algorithm 3's concatenation."""
    residue, asym, entity, token, sym = (t[i] for t in tokens)
    diff = lambda t: t.unsqueeze(1) - t.unsqueeze(0)  # noqa: E731
    chain, same = diff(asym) == 0, diff(residue) == 0
    r, sm = _R_MAX, _S_MAX
    d_residue = diff(residue).clip(-r, r) + r
    d_residue[~chain] = 2 * r + 1
    d_token = diff(token).clip(-r, r) + r
    d_token[~(chain & same)] = 2 * r + 1
    d_chain = diff(sym).clip(-sm, sm) + sm
    d_chain[chain] = 2 * sm + 1
    agree = (diff(entity) == 0).double()[..., None]
    return torch.cat([_hot(d_residue, 2 * r + 2), _hot(d_token, 2 * r + 2), agree, _hot(d_chain, 2 * sm + 2)], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "encoding":
        if case["grad"]:
            return sum(torch.tensordot(s["grad"][i].double(), _exact_features(s["tokens"], i), ([0, 1], [0, 1]))
                       for i in range(case["b"]))
        return torch.stack([_exact_features(s["tokens"], i) @ s["weight"].double().t() for i in range(case["b"])])
    if case["op"] == "bias":
        offset = (s["q_pos"].unsqueeze(2) - s["k_pos"].unsqueeze(1)).clip(-_DISTANCE, _DISTANCE)
        index = s["lut"].long()[offset + _DISTANCE]
        index[s["q_group"].unsqueeze(2) != s["k_group"].unsqueeze(1)] = _BUCKETS
        table = s["table"].double()
        if case["grad"]:
            return torch.stack([(s["grad"].double() * (index == u).unsqueeze(1)).sum((0, 2, 3))
                                for u in range(_BUCKETS + 1)])
        return torch.stack([table[:, h][index] for h in range(case["h"])], 1)
    share = case["b"] // case["bb"] if case["bb"] else 1
    names = [x for x in ("q", "k", "v", "bias", "gate") if s[x] is not None]
    leaves = {x: s[x].double().requires_grad_(case["grad"]) for x in names}
    rows = []
    for i in range(case["b"]):
        q = leaves["q"][i].transpose(0, 1).unflatten(0, (case["hk"], -1))
        k, v = (leaves[x][i].transpose(0, 1).unsqueeze(1) for x in ("k", "v"))
        z = q @ k.mT / math.sqrt(case["d"])
        if "bias" in leaves:
            z = z + leaves["bias"][i // share].unflatten(0, (case["hk"], -1))
        if s["mask"] is not None:
            keep = s["mask"][i]
            z = z.masked_fill(~keep, -math.inf) if s["inf"] is None else z - s["inf"] * (1 - keep.double())
        empty = (z == -math.inf).all(-1, keepdim=True)
        p = torch.softmax(z.masked_fill(empty, 0.0), -1).masked_fill(empty, 0.0)
        o = (p @ v).flatten(0, 1).transpose(0, 1)
        rows.append(o if "gate" not in leaves else o * torch.sigmoid(leaves["gate"][i]))
        if not case["grad"]:
            continue
        rows[-1].backward(s["grad"][i].double())
        rows[-1] = rows[-1].detach()
    out = dict(out=torch.stack(rows))
    if case["grad"]:
        out.update({"d" + x: leaves[x].grad for x in names})
    return out
