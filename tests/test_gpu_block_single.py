"""MI355X: graphs of which one key is open.  Its weight is 1 whatever the scores are, so the gradients of q and k are zeros, not
what the difference of two equal sums leaves in 24 bits."""
import pytest
import torch

from tests import block_oracle as O
from tests.test_gpu_block_ops import DEV, TYPES, dev, normal, offsets

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [24, 33, 64, 128])
@pytest.mark.parametrize("qs,ks,where", [
    ([1, 1, 3, 20], [1, 1, 1, 1], None),                       # graphs of one node, readouts over one
    ([4, 9, 0, 2], [7, 30, 5, 1], [6, 0, 2, 0]),               # one open key of several, one wave a tile
    ([100, 3, 70], [200, 65, 129], [64, 64, 0]),               # four waves, in the first tile of keys and behind it
    ([2, 1], [3000, 700], [2999, 300]),                        # keys in shares
    ([1500], [70], [69]),                                      # rows in shares
])
def test_one_open_key_passes_no_gradient_to_q_and_k(qs, ks, where, dim, dtype):
    from tsdiff_amd.block_ops import graph_attention
    qp, kp = offsets(qs), offsets(ks)
    q, k, v, do = (normal(s, n, h, dim, dtype=dtype) for s, n, h in ((1, qp[-1], 4), (2, kp[-1], 2), (3, kp[-1], 2), (4, qp[-1], 4)))
    mask = None
    if where is not None:
        mask = torch.zeros(kp[-1], dtype=torch.bool)
        mask[[a + w for a, w in zip(kp, where)]] = True
    want = O.attention(q, k, v, qp, kp, mask, dim ** -0.5, do, dtype)
    t = dev(q, k, v)
    out = graph_attention(*t, torch.tensor(qp, dtype=torch.int32, device=DEV), torch.tensor(kp, dtype=torch.int32, device=DEV),
                          None if mask is None else mask.to(DEV))
    dq, dk, dv = torch.autograd.grad(out, t, do.to(DEV))
    O.check(out, want["out"], "out")
    O.check(dv, want["dv"], "dv")
    assert not dq.any() and not dk.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_other_graphs_of_the_batch_keep_their_gradients(dtype):
    from tsdiff_amd.block_ops import graph_attention
    sizes = [1, 40, 1, 200, 30, 90, 2]
    p = offsets(sizes)
    q, k, v, do = (normal(s, p[-1], h, 32, dtype=dtype) for s, h in ((1, 4), (2, 2), (3, 2), (4, 4)))
    mask = torch.rand(p[-1], generator=torch.Generator().manual_seed(5)) > 0.3
    mask[p[3]:p[4]] = False
    mask[p[3] + 150] = True        # one of 200
    mask[p[5]:p[6]] = False
    mask[[p[5] + 3, p[5] + 80]] = True  # two, far apart
    want = O.attention(q, k, v, p, p, mask, 32 ** -0.5, do, dtype)
    t = dev(q, k, v)
    out = graph_attention(*t, torch.tensor(p, dtype=torch.int32, device=DEV), key_mask=mask.to(DEV))
    for n, g in zip(("out", "dq", "dk", "dv"), (out,) + torch.autograd.grad(out, t, do.to(DEV))):
        O.check(g, want[n], n)
        if n in ("dq", "dk"):
            assert not g[p[3]:p[4]].any() and g[p[5]:p[6]].any()


def test_what_is_not_finite_stays_so():
    from tsdiff_amd.block_ops import graph_attention
    q, k, v, do = (normal(s, 1, 1, 32) for s in (1, 2, 3, 4))
    do[0, 0, 3] = float("nan")
    t = dev(q, k, v)
    out = graph_attention(*t, torch.tensor([0, 1], dtype=torch.int32, device=DEV))
    assert all(g.isnan().any() for g in torch.autograd.grad(out, t, do.to(DEV)))
