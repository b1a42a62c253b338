"""MI355X: the gated linear layer at sizes that take every tile of its four products, each ending inside of one; the oracle of
tests/block_oracle.py on the GPU, in 64 bits."""
import pytest
import torch

from tests import block_oracle as O
from tests.test_gpu_block_ops import DEV, normal

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype,rows,fin,out", [
    (BF, 8229, 1016, 1016), (HF, 8229, 1016, 1016),  # dW 256 x 256
    (BF, 105003, 120, 24), (HF, 105003, 120, 24),    # dx 256 x 128
    (BF, 1500, 200, 520), (HF, 1500, 200, 520), (F, 1500, 200, 520),  # the first launch, dW and dx 64 x 64, dx in shares
    (F, 3601, 256, 1020),                            # all 128 x 128, dx in shares
    (F, 33001, 200, 64),                             # many shares of dW
])
def test_gated_linear_tiles(dtype, rows, fin, out):
    from tsdiff_amd.block_ops import gated_linear
    x, wg, wu, bg, bu, dh = (normal(s, *shape, dtype=dtype, scale=scale).to(DEV) for s, shape, scale in (
        (1, (rows, fin), 1.0), (2, (out, fin), fin ** -0.5), (3, (out, fin), fin ** -0.5), (4, (out,), 1.0), (5, (out,), 1.0),
        (6, (rows, out), 1.0)))
    want = {n: (v.cpu(), t.cpu()) for n, (v, t) in O.gated(x, wg, wu, bg, bu, "swish", dh, dtype).items()}
    t = [v.clone().requires_grad_() for v in (x, wg, wu, bg, bu)]
    h = gated_linear(*t)
    for n, g in zip(("h", "dx", "dwg", "dwu", "dbg", "dbu"), (h,) + torch.autograd.grad(h, t, dh)):
        O.check(g, want[n], n)
