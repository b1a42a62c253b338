"""MI355X: the operators of an attention block at the ends of their types' ranges: gradients far from 1 in float16, whose
intermediates lie among its subnormal numbers or beyond its largest one.

Tolerances are those of tests/block_oracle.py with one change: an intermediate that is rounded to feed a matrix product
(D = [dg | du]) may be off by half a step of its own size and by what its place in the type's range costs AFTER a
power of two has moved it there -- no longer by half a step of the type's subnormal numbers."""
from unittest import mock

import pytest
import torch

from tests import block_oracle as O
from tests.test_gpu_block_ops import DEV, dev, normal

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
    n, most = x.shape[1], [float(t.abs().max()) for t in (x, torch.cat((wg, wu)), torch.cat((bg, bu)), dh)]
    bound = most[3] * 1.25 * (n * most[0] * most[1] + most[2] + 1)
    return oracle(O.gated, lambda v: bound * 2.0 ** -39, x, wg, wu, bg, bu, act, dh, HALF)


def gated_run(x, wg, wu, bg, bu, dh, act="swish"):
    from tsdiff_amd.block_ops import gated_linear
    t = dev(x, wg, wu, bg, bu)
    h = gated_linear(*t, act=act)
    return dict(zip(("h", "dx", "dwg", "dwu", "dbg", "dbu"), (h,) + torch.autograd.grad(h, t, dh.to(DEV))))


@pytest.mark.parametrize("act", ["swish", "ssp", "ReLU", "Softplus"])
@pytest.mark.parametrize("rows,fin,out", [(40, 64, 48), (300, 72, 104), (2100, 121, 77), (4096, 256, 512)])
@pytest.mark.parametrize("size", [1e-3, 1e-5])
def test_gated_linear_of_small_half_precision_gradients(size, rows, fin, out, act):
    """tiles whose D keeps what its rounding left, others, copied rows, large tiles"""
    if act != "swish" and rows > 300:
        pytest.skip("one activation is enough for the sizes")
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
