"""MI355X: the global encoder on batches without nodes, as its operators accept them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("graphs", [0, 3])
@pytest.mark.parametrize("masked", [False, True])
def test_encoder_without_nodes(graphs, masked):
    from tsdiff_amd.encoder import GraphTransformerEncoder
    enc = GraphTransformerEncoder(64, num_blocks=2, num_heads=4, num_kv_heads=2, ff_dim=96).to(DEV)
    h = torch.empty(0, 64, device=DEV, requires_grad=True)
    ptr = torch.zeros(graphs + 1, dtype=torch.int32, device=DEV)
    mask = torch.empty(0, dtype=torch.bool, device=DEV) if masked else None
    with torch.no_grad():
        assert enc(h, ptr, mask).shape == (0, 64)
    out = enc(h, ptr, mask)
    assert out.shape == (0, 64)
    grads = torch.autograd.grad(out.sum(), [h] + list(enc.parameters()))
    torch.cuda.synchronize()
    assert grads[0].shape == (0, 64)
    for g, p in zip(grads[1:], enc.parameters()):
        assert g.shape == p.shape and not g.any()
