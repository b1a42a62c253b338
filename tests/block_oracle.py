"""The operators of tsdiff_amd.block_ops in 64 bits on the CPU, each value with the error that a kernel may make on it.

Every function returns {name: (value, tolerance)}, tolerances element by element and from arithmetic alone:
  * u = half a step of the tensors' type (torch.finfo(t).eps / 2): one rounding of an output, |value| u; where the kernel
    rounds an intermediate to feed a matrix product (the weights P and dS, D = [dg | du]), its magnitude times u beside it;
  * e = 2^-24: a sum of n products in fp32 is off by at most (n + PAD) e times the sum of the products' magnitudes; PAD
    covers the three-plane operands of fp32 products (each product off by < 4 e) and the handful of operations around a sum;
  * exp2 and the reciprocal of the hardware are good to one unit of the last place (2 e), of an argument off by its own e; a
    result of exp2 below the smallest normal number of fp32 is 0, which TINY = 2^-126 beside a weight covers.
Second-order terms are covered by the factor SAFE."""
import math

import torch

E = 2.0 ** -24
TINY = 2.0 ** -126
PAD = 16
SAFE = 1.05


def rounded(x, dtype):
    """the error of one rounding to the type: half a step, of the subnormal numbers below the normal ones"""
    f = torch.finfo(dtype)
    return f.eps / 2 * x.abs() + f.smallest_normal * f.eps / 2


def norm(x, w, b, eps, dy=None, dtype=torch.float32):
    x, n = x.double(), x.shape[-1]
    w = torch.ones(n, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(n, dtype=torch.float64) if b is None else b.double()
    m = x.mean(-1, keepdim=True)
    c = x - m
    r = (c.square().mean(-1, keepdim=True) + eps).rsqrt()
    h = c * r
    # a row's sums go over at most 32 values a lane and 8 levels of lanes
    em = (32 + PAD) * E * x.abs().mean(-1, keepdim=True)   # of the mean
    ec = em + E * c.abs()                                  # of a centred value
    # of r, relative: half the relative error of var + eps: 2 mean |c| ec + (32 + PAD) E var
    er = 0.5 * r.square() * (2 * (c.abs() * ec).mean(-1, keepdim=True) + (32 + PAD) * E * c.square().mean(-1, keepdim=True)) + 4 * E
    eh = r * ec + h.abs() * (er + 2 * E)
    y = h * w + b
    got = {"y": (y, SAFE * (w.abs() * eh + 2 * E * ((h * w).abs() + b.abs())) + rounded(y, dtype))}
    if dy is not None:
        dy = dy.double()
        g = dy * w
        s0, s1 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
        e0 = (32 + PAD) * E * g.abs().mean(-1, keepdim=True)
        e1 = (g.abs() * eh).mean(-1, keepdim=True) + (32 + PAD) * E * (g * h).abs().mean(-1, keepdim=True)
        dx = r * (g - s0 - h * s1)
        ei = 2 * E * g.abs() + e0 + h.abs() * e1 + eh * s1.abs() + 4 * E * (g.abs() + s0.abs() + (h * s1).abs())
        got["dx"] = (dx, SAFE * (r * ei + dx.abs() * (er + 2 * E)) + rounded(dx, dtype))
        rows = x.shape[0]
        dw, db = (dy * h).sum(0), dy.sum(0)
        got["dw"] = (dw, SAFE * ((dy.abs() * eh).sum(0) + (rows + PAD) * E * (dy * h).abs().sum(0)) + rounded(dw, dtype))
        got["db"] = (db, SAFE * (rows + PAD) * E * dy.abs().sum(0) + rounded(db, dtype))
    return got


def act(kind, g):
    """a(g), a'(g) and bounds of |a'| and |a''|"""
    s = torch.sigmoid(g)
    if kind == "swish":
        return g * s, s * (1 + g * (1 - s)), 1.1, 0.5
    if kind == "ReLU":
        return g.clamp(min=0), (g > 0).double(), 1.0, 0.0
    sp = torch.nn.functional.softplus(g, threshold=1000.0)
    return sp - (math.log(2) if kind == "ssp" else 0.0), s, 1.0, 0.25


def gated(x, wg, wu, bg, bu, kind, dh=None, dtype=torch.float32):
    x, wg, wu = x.double(), wg.double(), wu.double()
    bg = torch.zeros(wg.shape[0], dtype=torch.float64) if bg is None else bg.double()
    bu = torch.zeros(wg.shape[0], dtype=torch.float64) if bu is None else bu.double()
    n = x.shape[1]
    g, v = x @ wg.t() + bg, x @ wu.t() + bu
    eg = (n + PAD) * E * (x.abs() @ wg.abs().t() + bg.abs())
    ev = (n + PAD) * E * (x.abs() @ wu.abs().t() + bu.abs())
    a, da, c1, c2 = act(kind, g)
    # the function itself: exp2 of an argument off by |g| e, a reciprocal or logarithm, and the operations around them
    own = (8 + 2 * g.abs()) * E * (g.abs() + 1)
    ea, eda = c1 * eg + own, c2 * eg + own
    if kind == "ReLU":  # its slope jumps where g is nothing but its error
        eda = eda + (g.abs() <= eg).double()
    h = a * v
    got = {"h": (h, SAFE * (ea * v.abs() + a.abs() * ev + 2 * E * h.abs()) + rounded(h, dtype))}
    if dh is None:
        return got
    dh = dh.double()
    dg, dv = dh * v * da, dh * a
    edg = SAFE * (dh.abs() * (ev * da.abs() + v.abs() * eda) + 4 * E * dg.abs())
    edv = SAFE * (dh.abs() * ea + 4 * E * dv.abs())
    for k, d, ed in (("dbg", dg, edg), ("dbu", dv, edv)):
        s = d.sum(0)
        got[k] = (s, SAFE * (ed.sum(0) + (d.shape[0] + PAD) * E * d.abs().sum(0)) + rounded(s, dtype))
    rg, rv = edg + rounded(dg, dtype), edv + rounded(dv, dtype)  # as rounded for the products (fp32: u is the split's own error)
    dx = dg @ wg + dv @ wu
    k = (2 * wg.shape[0] + PAD) * E
    got["dx"] = (dx, SAFE * (rg @ wg.abs() + rv @ wu.abs() + k * (dg.abs() @ wg.abs() + dv.abs() @ wu.abs())) + rounded(dx, dtype))
    k = (x.shape[0] + PAD) * E
    for name, d, rd in (("dwg", dg, rg), ("dwu", dv, rv)):
        s = d.t() @ x
        got[name] = (s, SAFE * (rd.t() @ x.abs() + k * d.abs().t() @ x.abs()) + rounded(s, dtype))
    return got


def attention(q, k, v, q_ptr, k_ptr, mask, scale, dout=None, dtype=torch.float32):
    """Values at masked keys are never read.  Rows and keys outside of every graph: zeros."""
    q, k, v = q.double(), k.double(), v.double()
    H, Hk, D = q.shape[1], k.shape[1], q.shape[2]
    names = ["out"] + (["dq", "dk", "dv"] if dout is not None else [])
    got = {n: (torch.zeros_like(t), torch.zeros_like(t)) for n, t in zip(names, (q, q, k, v))}
    for gi in range(len(q_ptr) - 1):
        a, b, c, d = q_ptr[gi], q_ptr[gi + 1], k_ptr[gi], k_ptr[gi + 1]
        idx = torch.arange(c, d)
        if mask is not None:
            idx = idx[mask[c:d].bool()]
        if a == b or len(idx) == 0:
            continue
        L = len(idx)
        for h in range(H):
            Q, K, V = q[a:b, h], k[idx, h * Hk // H], v[idx, h * Hk // H]
            S = scale * (Q @ K.t())
            eS = (D + PAD) * E * abs(scale) * (Q.abs() @ K.abs().t()) + 4 * E * S.abs()
            P = torch.softmax(S, -1)
            # relative error of a weight: its score's and the maximum's and sum's own, the sum over keys, exp2
            eP = eS + (P * eS).sum(-1, keepdim=True) + 2 * eS.amax(-1, keepdim=True) + (L + PAD) * E
            wP = P * eP + TINY + rounded(P, dtype)  # as the matrix operand of P V, P^T dO
            O = P @ V
            eO = SAFE * (wP @ V.abs() + (L + PAD) * E * (P @ V.abs()))
            got["out"][0][a:b, h], got["out"][1][a:b, h] = O, eO + rounded(O, dtype)
            if dout is None:
                continue
            G = dout[a:b, h].double()
            dP = G @ V.t()
            delta = (G * O).sum(-1, keepdim=True)
            e1 = (D + PAD) * E * (G.abs() @ V.abs().t())
            e2 = (G.abs() * (eO + rounded(O, dtype))).sum(-1, keepdim=True) + (D + PAD) * E * (G * O).abs().sum(-1, keepdim=True)
            dS = P * (dP - delta)
            edS = SAFE * (P * (e1 + e2) + ((eP + 4 * E) * P + TINY) * (dP.abs() + delta.abs())) + rounded(dS, dtype)
            dQ = scale * (dS @ K)
            eQ = SAFE * abs(scale) * (edS @ K.abs() + (L + PAD) * E * (dS.abs() @ K.abs())) + rounded(dQ, dtype)
            got["dq"][0][a:b, h], got["dq"][1][a:b, h] = dQ, eQ
            # a key head's gradient goes over the rows of all its heads
            n = ((b - a) * (H // Hk) + PAD) * E
            for name, x, t in (("dk", scale * (dS.t() @ Q), abs(scale) * (edS.t() @ Q.abs() + n * (dS.abs().t() @ Q.abs()))),
                               ("dv", P.t() @ G, wP.t() @ G.abs() + n * (P.t() @ G.abs()))):
                got[name][0][idx, h * Hk // H] += x
                got[name][1][idx, h * Hk // H] += SAFE * t
    for name in names[2:]:  # rounded once, behind the sum over the heads
        got[name][1].add_(rounded(got[name][0], dtype))
    return got


def check(got, want, what=""):
    """got within the tolerance of want, everywhere; an exact zero where the tolerance is zero"""
    value, tol = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, f"{what}: shape {tuple(got.shape)}, {tuple(value.shape)} expected"
    bad = ~((got - value).abs() <= tol)
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at {i}: {got[i]:.9g}, "
                             f"{value[i]:.9g} +- {tol[i]:.3g} expected")
