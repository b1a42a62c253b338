"""MI355X: the operators of an attention block at the ends of their types' ranges: gradients far from 1 in float16, whose
intermediates lie among its subnormal numbers or beyond its largest one, weights of many far keys, and float32 values that no bfloat16 holds.

Tolerances are those of tests/block_oracle.py with one change: an intermediate that is rounded to feed a matrix product
(D = [dg | du], P, dS) may be off by half a step of its own size and by what its place in the type's range costs AFTER a
power of two has moved it there -- no longer by half a step of the type's subnormal numbers."""
import math
from unittest import mock

import pytest
import torch

from tests import block_oracle as O
from tests.test_gpu_block_ops import DEV, attention_case, dev, normal

pytestmark = pytest.mark.gpu
HALF = torch.float16
STEP = 2.0 ** -25  # half a step of float16's subnormal numbers


def oracle(f, floor, *args):
    """f(*args) with roundings of half a relative step and floor(x) beside it; outputs have the type's subnormal numbers"""
    with mock.patch.object(O, "rounded", lambda x, dtype: torch.finfo(dtype).eps / 2 * x.abs() + floor(x)):
        return {n: (v, t + STEP) for n, (v, t) in f(*args).items()}


def check(got, want, what):
    """O.check, where the value lies inside of the type's range; beyond it the type has infinity alone"""
    value, tol = want
    inside = value.abs() + tol < torch.finfo(got.dtype).max
    zero = torch.zeros(())
    assert inside.any()
    O.check(torch.where(inside, got.detach().double().cpu(), zero.double()),
            (torch.where(inside, value, zero.double()), torch.where(inside, tol, zero.double())), what)


# ---- gated linear layer ---------------------------------------------------------------------------------------
def gated_want(x, wg, wu, bg, bu, dh, act="swish"):
    # D is scaled by a power of two that takes the bound B of its values into 2^14 .. 2^15; half a step of the subnormal
    # numbers there is B 2^-39 at most in D's own units
    most = [float(t.double().norm(dim=1).max()) for t in (x, torch.cat((wg, wu)))] + [float(t.abs().max()) for t in (torch.cat((bg, bu)), dh)]
    bound = most[3] * 1.25 * (most[0] * most[1] * 1.02 + most[2] + 1)  # (norms are bf16 rounded up)
    return oracle(O.gated, lambda v: bound * 2.0 ** -39, x, wg, wu, bg, bu, act, dh, HALF)


def gated_run(x, wg, wu, bg, bu, dh, act="swish"):
    from tsdiff_amd.block_ops import gated_linear
    t = dev(x, wg, wu, bg, bu)
    h = gated_linear(*t, act=act)
    return dict(zip(("h", "dx", "dwg", "dwu", "dbg", "dbu"), (h,) + torch.autograd.grad(h, t, dh.to(DEV))))


@pytest.mark.parametrize("rows,fin,out,act", [(40, 64, 48, a) for a in ("swish", "ssp", "ReLU", "Softplus")] +
                         [(300, 72, 104, "ssp"), (2100, 121, 77, "swish"), (4096, 256, 512, "swish")])
@pytest.mark.parametrize("size", [1e-3, 1e-5])
def test_gated_linear_of_small_half_precision_gradients(size, rows, fin, out, act):
    """tiles whose D keeps what its rounding left, others, copied rows, large tiles"""
    x, wg, wu = (normal(1, rows, fin, dtype=HALF), normal(2, out, fin, dtype=HALF, scale=fin ** -0.5),
                 normal(3, out, fin, dtype=HALF, scale=fin ** -0.5))
    bg, bu, dh = normal(4, out, dtype=HALF), normal(5, out, dtype=HALF), normal(6, rows, out, dtype=HALF, scale=size)
    want, got = gated_want(x, wg, wu, bg, bu, dh, act), gated_run(x, wg, wu, bg, bu, dh, act)
    for n in want:
        check(got[n], want[n], n)


@pytest.mark.parametrize("rows,fin,out", [(3, 16, 8), (40, 64, 48), (300, 72, 104), (2100, 121, 77), (4096, 256, 512)])
def test_gated_linear_of_large_half_precision_gradients(rows, fin, out):
    """dg and du beyond 65504 whose products are not"""
    x, wg, wu = (normal(s, *shape, dtype=HALF, scale=2.0 ** -9) for s, shape in ((1, (rows, fin)), (2, (out, fin)), (3, (out, fin))))
    bg, bu, dh = normal(4, out, dtype=HALF, scale=3.0), normal(5, out, dtype=HALF, scale=3.0), normal(6, rows, out, dtype=HALF, scale=8192.0)
    dh = dh.clamp(-60000, 60000)
    want, got = gated_want(x, wg, wu, bg, bu, dh), gated_run(x, wg, wu, bg, bu, dh)
    if rows > 3:
        u = x.double() @ wu.double().t() + bu
        g = x.double() @ wg.double().t() + bg
        assert float((dh * u * O.act("swish", g)[1]).abs().max()) > 65504
    for n in ("h", "dx", "dwg", "dwu"):
        assert got[n].isfinite().all(), n
        check(got[n], want[n], n)


@pytest.mark.parametrize("rows,fin,out", [(40, 64, 48), (300, 1000, 104), (2100, 121, 77)])
def test_gated_linear_with_single_large_values(rows, fin, out):
    """one large value in x and in the weights: the other rows' gradients stay what they are"""
    x, wg, wu = (normal(1, rows, fin, dtype=HALF), normal(2, out, fin, dtype=HALF, scale=fin ** -0.5),
                 normal(3, out, fin, dtype=HALF, scale=fin ** -0.5))
    bg, bu, dh = normal(4, out, dtype=HALF), normal(5, out, dtype=HALF), normal(6, rows, out, dtype=HALF)
    x[3, 5] = 30000.0
    wu[2, 7] = 50.0
    dh[3] = 0
    want, got = gated_want(x, wg, wu, bg, bu, dh), gated_run(x, wg, wu, bg, bu, dh)
    for n in ("dx", "dwg", "dwu", "dbg", "dbu"):
        check(got[n], want[n], n)


@pytest.mark.parametrize("rows", [1040])
def test_gated_linear_of_half_precision_rows_far_apart(rows):
    """rows of x and of dh 2^21 values apart: the last ones lie past 2^31 values"""
    from tsdiff_amd.block_ops import gated_linear
    gap = 1 << 21
    far = torch.empty(rows * gap, dtype=HALF, device=DEV).view(rows, gap)
    x, wg, wu, dh = (normal(s, *shape, dtype=HALF).to(DEV) for s, shape in ((1, (rows, 64)), (2, (24, 64)), (3, (24, 64)), (4, (rows, 24))))
    far[:, :64], far[:, 64:88] = x, dh * 1e-5
    got = []
    for a, d in ((x, far[:, 64:88].contiguous()), (far[:, :64], far[:, 64:88])):
        a = a.detach().requires_grad_()
        got.append(torch.autograd.grad(gated_linear(a, wg, wu), a, d)[0])
    assert torch.equal(*got)


def test_gated_linear_scale_ignores_what_is_not_finite():
    """an infinite gradient of one row leaves the other rows' gradients what they are; no gradient at all gives zeros"""
    x, wg, wu = (normal(s, *shape, dtype=HALF, scale=0.2) for s, shape in ((1, (40, 64)), (2, (48, 64)), (3, (48, 64))))
    bg, bu, dh = normal(4, 48, dtype=HALF), normal(5, 48, dtype=HALF), normal(6, 40, 48, dtype=HALF, scale=1e-5)
    plain = gated_run(x, wg, wu, bg, bu, dh)
    d2, x2 = dh.clone(), x.clone()
    d2[7, 3] = float("inf")
    x2[9, 5] = float("nan")
    d2[9] = 0
    got = gated_run(x2, wg, wu, bg, bu, d2)
    rest = [i for i in range(40) if i not in (7, 9)]
    want = gated_want(x, wg, wu, bg, bu, dh)
    check(got["dx"][rest], tuple(t[rest] for t in want["dx"]), "dx")
    assert not got["dx"][7].isfinite().all() and plain["dx"].isfinite().all()
    for n, t in gated_run(x, wg, wu, bg, bu, torch.zeros_like(dh)).items():
        assert n == "h" or not t.any(), n


# ---- attention ------------------------------------------------------------------------------------------------
def attention_want(q, k, v, do, qp, kp, mask, scale):
    # weights of the forward are off by 2^-34 of the largest, those of dV by 2^-40; dS by 2^-39 of the largest of its row or key
    return oracle(O.attention, lambda x: 2.0 ** -40 + 2.0 ** -34 * x.abs().amax(), q, k, v, qp, kp, mask, scale, do, HALF)


def attention_run(q, k, v, do, qp, kp, mask, scale):
    from tsdiff_amd.block_ops import graph_attention
    t = dev(q, k, v)
    out = graph_attention(*t, torch.tensor(qp, dtype=torch.int32, device=DEV), torch.tensor(kp, dtype=torch.int32, device=DEV),
                          None if mask is None else mask.to(DEV), scale)
    return dict(zip(("out", "dq", "dk", "dv"), (out,) + torch.autograd.grad(out, t, do.to(DEV))))


SHAPES = [([20, 31, 9], None, 4, 2, 32), ([20, 31, 9], None, 2, 2, 33), ([300, 129], None, 4, 2, 64), ([2000], None, 2, 1, 64),
          ([1, 1], [3000, 700], 2, 2, 32), ([1500], [3], 2, 2, 40), ([90, 70], None, 2, 2, 100)]


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("qs,ks,heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("size", [1e-3, 1e-5])
def test_attention_of_small_half_precision_gradients(size, qs, ks, heads, kv_heads, dim, masked):
    q, k, v, do, qp, kp, mask, _ = attention_case(qs, ks, heads, kv_heads, dim, HALF, masked and len(qs) > 1, seed=3)
    do = (do.float() * size).half()
    want = attention_want(q, k, v, do, qp, kp, mask, dim ** -0.5)
    got = attention_run(q, k, v, do, qp, kp, mask, dim ** -0.5)
    for n in want:
        check(got[n], want[n], n)


@pytest.mark.parametrize("qs,ks,heads,kv_heads,dim", SHAPES)
def test_attention_of_large_half_precision_gradients(qs, ks, heads, kv_heads, dim):
    """dS beyond 65504 whose products are not; rows whose gradients differ by a factor of 2^20"""
    q, k, v, do, qp, kp, mask, _ = attention_case(qs, ks, heads, kv_heads, dim, HALF, False, seed=3)
    q, k, v = q * 2.0 ** -4, k * 2.0 ** -4, v * 8
    rows = torch.arange(do.shape[0])
    do = (do.float() * torch.where(rows % 3 == 0, 2.0 ** 13, torch.where(rows % 3 == 1, 1.0, 2.0 ** -7))[:, None, None]).clamp(-60000, 60000).half()
    want = attention_want(q, k, v, do, qp, kp, mask, dim ** -0.5)
    got = attention_run(q, k, v, do, qp, kp, mask, dim ** -0.5)
    for n in want:
        assert not got[n].isnan().any(), n
        check(got[n], want[n], n)


@pytest.mark.parametrize("dim", [32, 33, 128])
def test_attention_keeps_the_weights_of_many_far_keys(dim):
    """one key's weight is 1 and its value 0, each of 60000 others' is 2^-25.2: alone the others answer"""
    n = 60001
    q, k, v = torch.zeros(1, 1, dim), torch.zeros(n, 1, dim), torch.ones(n, 1, dim)
    q[..., 0] = 1
    k[1:, 0, 0] = -25.2 * math.log(2)
    v[0] = 0
    q, k, v = q.half(), k.half(), v.half()
    do = normal(1, 1, 1, dim, dtype=HALF)
    want = attention_want(q, k, v, do, [0, 1], [0, n], None, 1.0)
    got = attention_run(q, k, v, do, [0, 1], [0, n], None, 1.0)
    assert 1.4e-3 < float(want["out"][0].min()) < 1.7e-3
    for name in ("out", "dq", "dv"):
        check(got[name], want[name], name)


# ---- float32 values that no bfloat16 holds ---------------------------------------------------------------------
LARGEST = torch.finfo(torch.float32).max


@pytest.mark.parametrize("rows,fin,out", [(3, 8, 8), (5, 7, 9), (130, 64, 72), (9000, 64, 64)])
def test_gated_linear_of_the_largest_floats(rows, fin, out):
    """finite operands whose first bfloat16 plane would round to infinity: 0 times them is 0, 1 / 2^120 of them is 2^8"""
    x, wg, wu, dh = normal(1, rows, fin), normal(2, out, fin), normal(3, out, fin), normal(4, rows, out)
    x[:, 1], x[0, 1] = LARGEST, -LARGEST
    wg[:, 1] = wu[:, 1] = 0
    wu[2, 1] = 2.0 ** -120
    bg, bu = normal(5, out), normal(6, out)
    want = O.gated(x, wg, wu, bg, bu, "swish")
    from tsdiff_amd.block_ops import gated_linear
    got = gated_linear(*dev(x, wg, wu, bg, bu, grad=False))
    assert got.isfinite().all()
    # the zeros' products cost nothing, the last places of 2^8 do (their tolerance is in the oracle's sums of magnitudes)
    O.check(got, want["h"], "h")
    t = dev(x, wg, wu, bg, bu)
    dx = torch.autograd.grad(gated_linear(*t), t[0], dh.to(DEV))[0]
    assert dx.isfinite().all()


@pytest.mark.parametrize("n,dim", [(1, 32), (40, 32), (200, 64), (3, 33), (500, 128)])
def test_attention_passes_the_largest_floats_on(n, dim):
    """values of a graph whose rows each have one open key: out = v, whatever v's size"""
    from tsdiff_amd.block_ops import graph_attention
    q, k, v = torch.zeros(n, 2, dim), normal(2, n, 2, dim), normal(3, n, 2, dim)  # (scores of 0: a weight of exactly 1)
    v[n // 2] = torch.where(torch.arange(dim) % 2 == 0, LARGEST, -LARGEST)
    mask = torch.zeros(n, dtype=torch.bool)
    mask[n // 2] = True
    out = graph_attention(*dev(q, k, v, grad=False), torch.tensor([0, n], dtype=torch.int32, device=DEV), key_mask=mask.to(DEV))
    assert torch.equal(out.cpu(), v[n // 2].expand(n, 2, dim))
