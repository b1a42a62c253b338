"""The operators of an attention block over ragged graphs, as a user's program calls them: layer norm, the gated
linear layer and attention inside graphs, each forward and as a training step.

`own` false: their plain form, elementary torch operations in 32 bits, rounded once at the end.  `own` true: the calls
of `tsdiff_amd.block_ops`.  A case names its operator, its sizes, its type and whether gradients are asked for."""
import math
import random

import torch

own = False

DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
NORM_MOST = 262144 * 256         # elements of the largest layer norm
GATED_MOST = 65536 * 256 * 1024  # rows * in * out of the largest gated layer
SCORES_MOST = 10000000 * 8 * 64  # query-key pairs * heads * dim of the largest attention


def listed():
    return [
        # node rows of one reaction's graph between two blocks of a sampling step: latency counts
        norm("norm one graph", 17, 256, "f32", False),
        # node rows of a training batch of 200 graphs
        norm("norm batch", 3600, 256, "f32", True),
        # pair rows of a dense batch
        norm("norm pairs", 262144, 256, "bf16", True),
        # a width that fills no vector and no wave
        norm("norm odd width", 4099, 1030, "f16", True),
        # the feed-forward half of a block on one graph: latency counts
        gated("gated one graph", 17, 256, 512, "f32", False),
        # the same in a training batch of 200 graphs
        gated("gated batch", 3600, 256, 1024, "f32", True),
        # 1024 graphs of 64 atoms in mixed precision: the largest
        gated("gated dense", 65536, 256, 1024, "bf16", True),
        # rows and widths that end inside every tile
        gated("gated odd", 5003, 204, 530, "f16", True),
        # 100 small molecules, sampling: many short graphs
        attention("attention molecules", 100, 6, 30, 0, 8, 8, 32, "f32", False, False),
        # 1024 graphs of 64 atoms, training
        attention("attention dense", 1024, 64, 64, 0, 8, 8, 32, "f32", True, False),
        # a few long graphs, key heads shared by four query heads, some atoms masked
        attention("attention long", 3, 1200, 2600, 0, 8, 2, 64, "bf16", True, True),
        # a readout: one query a graph over all its atoms
        attention("attention readout", 8, 2000, 8192, 1, 8, 8, 64, "f16", False, True),
    ]


def norm(name, rows, dim, dtype, train):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "dtype": dtype, "train": train}


def gated(name, rows, inner, outer, dtype, train):
    return {"name": name, "op": "gated", "rows": rows, "in": inner, "out": outer, "dtype": dtype, "train": train}


def attention(name, graphs, low, high, queries, heads, kv_heads, dim, dtype, train, masked):
    """`queries` 0: a graph's nodes attend to each other; otherwise so many queries of their own a graph"""
    return {"name": name, "op": "attention", "graphs": graphs, "low": low, "high": high, "queries": queries,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "train": train, "masked": masked}


def between(rng, low, high):
    """a whole number, spread over the logarithm"""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("norm", "gated", "attention"))
    dtype, train = rng.choice(("f32", "f32", "bf16", "f16")), rng.random() < 0.6
    if op == "norm":
        dim = between(rng, 16, 2048)
        c = norm("", min(between(rng, 1, 262144), NORM_MOST // dim), dim, dtype, train)
    elif op == "gated":
        inner, outer = between(rng, 16, 1024), between(rng, 16, 2048)
        c = gated("", min(between(rng, 1, 65536), GATED_MOST // (inner * outer)), inner, outer, dtype, train)
    else:
        kv_heads, group, dim = rng.choice((1, 2, 4, 8)), rng.choice((1, 1, 2, 4)), rng.choice((16, 24, 32, 64, 128))
        cost = kv_heads * group * dim
        queries = rng.choice((0, 0, 1, between(rng, 2, 64)))
        high = between(rng, 1, 8192 if queries else 4096)
        if not queries:
            high = min(high, math.isqrt(SCORES_MOST // cost))
        low = between(rng, 1, high)
        graphs = max(1, min(between(rng, 1, 1024), SCORES_MOST // (high * (queries or high) * cost)))
        c = attention("", graphs, low, high, queries, kv_heads * group, kv_heads, dim, dtype, train, rng.random() < 0.5)
    del c["name"]
    return c


def lengths(case):
    """nodes of each graph: the same for every seed, so that the work is known"""
    rng = random.Random(case["graphs"] * 8191 + case["high"])
    return [rng.randint(case["low"], case["high"]) for _ in range(case["graphs"])]


def work(case):
    size, t = BYTES[case["dtype"]], case["train"]
    if case["op"] == "norm":
        n, d = case["rows"] * case["dim"], case["dim"]
        return {"bytes": size * ((4 if t else 2) * n + (4 if t else 2) * d), "flops": (20 if t else 8) * n}
    if case["op"] == "gated":
        m, k, f = case["rows"], case["in"], case["out"]
        return {"bytes": size * (2 if t else 1) * (m * k + 2 * k * f + m * f), "flops": (12 if t else 4) * m * k * f}
    ks = lengths(case)
    qs = [case["queries"] or n for n in ks]
    pairs = sum(a * b for a, b in zip(qs, ks))
    values = 2 * sum(qs) * case["heads"] + 2 * sum(ks) * case["kv_heads"]
    return {"bytes": size * (2 if t else 1) * values * case["dim"],
            "flops": (12 if t else 4) * pairs * case["heads"] * case["dim"]}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype, train = DTYPE[case["dtype"]], case["train"]

    def normal(*shape, scale=1.0, shift=0.0, leaf=True):
        t = (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)
        return t.requires_grad_(train and leaf)

    s = {"op": case["op"], "train": train}
    if case["op"] == "norm":
        s["x"] = normal(case["rows"], case["dim"], scale=2.0, shift=0.5)
        s["weight"], s["bias"] = normal(case["dim"], scale=0.1, shift=1.0), normal(case["dim"], scale=0.1)
        s["dy"] = normal(case["rows"], case["dim"], leaf=False)
    elif case["op"] == "gated":
        m, k, f = case["rows"], case["in"], case["out"]
        s["x"], s["dy"] = normal(m, k), normal(m, f, leaf=False)
        s["w_gate"], s["w_up"] = normal(f, k, scale=k ** -0.5), normal(f, k, scale=k ** -0.5)
        s["b_gate"], s["b_up"] = normal(f, scale=0.1), normal(f, scale=0.1)
    else:
        ks = lengths(case)
        qs = [case["queries"] or n for n in ks]
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        s["q"], s["k"], s["v"] = normal(sum(qs), h, d), normal(sum(ks), hk, d), normal(sum(ks), hk, d)
        s["dy"] = normal(sum(qs), h, d, leaf=False)

        def offsets(sizes):
            return torch.tensor([0] + sizes, device="cuda").cumsum(0).to(torch.int32)

        s["k_ptr"] = offsets(ks)
        s["q_ptr"] = offsets(qs) if case["queries"] else s["k_ptr"]
        s["q_max"], s["k_max"] = max(qs), max(ks)
        s["mask"] = None
        if case["masked"]:  # a fifth of the atoms, and the whole of the first graph
            s["mask"] = torch.rand(sum(ks), generator=g, device="cuda") > 0.2
            if case["graphs"] > 1:
                s["mask"][: ks[0]] = False
    return s


def run(s):
    if not s["train"]:
        with torch.no_grad():
            return kernels(s) if own else plain(s, False)
    if not own:
        with torch.no_grad():
            return plain(s, True)
    y = kernels(s)
    return (y,) + torch.autograd.grad(y, leaves(s), s["dy"])


def leaves(s):
    names = {"norm": ("x", "weight", "bias"), "gated": ("x", "w_gate", "w_up", "b_gate", "b_up"), "attention": ("q", "k", "v")}
    return tuple(s[n] for n in names[s["op"]])


def kernels(s):
    from tsdiff_amd import block_ops

    if s["op"] == "norm":
        return block_ops.layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5)
    if s["op"] == "gated":
        return block_ops.gated_linear(s["x"], s["w_gate"], s["w_up"], s["b_gate"], s["b_up"], act="swish")
    return block_ops.graph_attention(s["q"], s["k"], s["v"], s["q_ptr"], key_ptr=s["k_ptr"], key_mask=s["mask"])


def plain(s, train):
    return {"norm": plain_norm, "gated": plain_gated, "attention": plain_attention}[s["op"]](s, train)


def plain_norm(s, train):
    dtype = s["x"].dtype
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    centred = x - x.mean(-1, keepdim=True)
    r = (centred.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    xhat = centred * r
    y = (xhat * w + b).to(dtype)
    if not train:
        return y
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return y, dx.to(dtype), (dy * xhat).sum(0).to(dtype), dy.sum(0).to(dtype)


def plain_gated(s, train):
    dtype = s["x"].dtype
    x, wg, wu, bg, bu = (s[n].float() for n in ("x", "w_gate", "w_up", "b_gate", "b_up"))
    g, u = x @ wg.t() + bg, x @ wu.t() + bu
    sig = 1 / (1 + torch.exp(-g))
    y = (g * sig * u).to(dtype)
    if not train:
        return y
    dy = s["dy"].float()
    du = dy * (g * sig)
    dg = dy * u * (sig * (1 + g * (1 - sig)))
    dx = dg @ wg + du @ wu
    return (y,) + tuple(t.to(dtype) for t in (dx, dg.t() @ x, du.t() @ x, dg.sum(0), du.sum(0)))


def places(ptr, most):
    """[graph, slot] -> row and whether the graph has that slot"""
    start, end = ptr[:-1].long(), ptr[1:].long()
    row = start[:, None] + torch.arange(most, device=ptr.device)
    return torch.minimum(row, (end - 1).clamp(min=0)[:, None]), row < end[:, None]


def plain_attention(s, train):
    dtype, (h, d), hk = s["q"].dtype, s["q"].shape[1:], s["k"].shape[1]
    scale = d ** -0.5
    qi, qok = places(s["q_ptr"], s["q_max"])
    ki, kok = places(s["k_ptr"], s["k_max"])
    open_ = kok if s["mask"] is None else kok & s["mask"][ki]

    def padded(t, i):  # [graph, head, slot, dim]
        return t.float()[i].transpose(1, 2).contiguous()

    q = padded(s["q"], qi)
    k, v = (padded(s[n], ki).repeat_interleave(h // hk, 1) for n in "kv")
    score = (q @ k.transpose(-1, -2)) * scale
    score = score.masked_fill(~open_[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    y = (p @ v).transpose(1, 2)[qok].to(dtype)
    if not train:
        return y
    do = padded(s["dy"], qi) * qok[:, None, :, None]
    dv = p.transpose(-1, -2) @ do
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (dp * p).sum(-1, keepdim=True)) * scale
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q

    def shared(t):  # a key head's gradient is the sum over the query heads that read it
        return t.unflatten(1, (hk, h // hk)).sum(2).transpose(1, 2)[kok].to(dtype)

    return y, dq.transpose(1, 2)[qok].to(dtype), shared(dk), shared(dv)


def exact(case, seed):
    """The definitions in 64 bits, graph by graph, with gradients by automatic differentiation."""
    s = prepare(case, seed)
    x = [t.detach().double().requires_grad_(case["train"]) for t in leaves(s)]
    if case["op"] == "norm":
        mean, var = x[0].mean(1, keepdim=True), x[0].var(1, unbiased=False, keepdim=True)
        y = (x[0] - mean) / (var + 1e-5).sqrt() * x[1] + x[2]
    elif case["op"] == "gated":
        gate = torch.addmm(x[3], x[0], x[1].t())
        y = gate * torch.sigmoid(gate) * torch.addmm(x[4], x[0], x[2].t())
    else:
        group = case["heads"] // case["kv_heads"]
        ends = zip(s["q_ptr"].tolist(), s["q_ptr"].tolist()[1:], s["k_ptr"].tolist(), s["k_ptr"].tolist()[1:])
        got, grads = [], [torch.zeros_like(t) for t in x]
        for a, b, c, e in ends:  # one graph at a time: the scores of all of them need not fit
            part = [x[0][a:b].detach(), x[1][c:e].detach(), x[2][c:e].detach()]
            part = [t.requires_grad_(case["train"]) for t in part]
            y = exact_graph(*part, group, None if s["mask"] is None else s["mask"][c:e])
            if case["train"] and y.requires_grad:
                for t, f, (i, j) in zip(torch.autograd.grad(y, part, s["dy"][a:b].double()), grads, ((a, b), (c, e), (c, e))):
                    f[i:j] = t
            got.append(y.detach())
        y = torch.cat(got)
        return (y, *grads) if case["train"] else y
    if not case["train"]:
        return y
    return (y.detach(),) + torch.autograd.grad(y, x, s["dy"].double())


def exact_graph(q, k, v, group, mask):
    if mask is not None:
        k, v = k[mask], v[mask]
    if not k.shape[0]:
        return torch.zeros_like(q, requires_grad=False)
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    p = torch.softmax(torch.bmm(q.permute(1, 0, 2), k.permute(1, 2, 0)) / math.sqrt(q.shape[2]), -1)
    return torch.bmm(p, v.permute(1, 0, 2)).permute(1, 0, 2)
