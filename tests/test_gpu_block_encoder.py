"""MI355X: the global encoder on batches without nodes, which its operators accept, and in calls side by side."""
import copy

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


def encoders(n):
    from tsdiff_amd.encoder import GraphTransformerEncoder
    torch.manual_seed(n)
    return [GraphTransformerEncoder(128, num_blocks=2, num_heads=4, ff_dim=256).to(DEV) for _ in range(n)]


def step(enc, h, ptr, d):
    out = enc(h, ptr)
    return (out,) + torch.autograd.grad(out, [h] + list(enc.parameters()), d)


def test_encoders_on_several_streams_at_once():
    """calls side by side share no scratch"""
    encs = encoders(3)
    ptr = torch.tensor([0, 30, 700], dtype=torch.int32, device=DEV)
    h = [torch.randn(700, 128, device=DEV).requires_grad_() for _ in encs]
    d = torch.randn(700, 128, device=DEV)
    want = [step(e, x, ptr, d) for e, x in zip(encs, h)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in encs]
    got = []
    for _ in range(6):
        for s, e, x in zip(streams, encs, h):
            with torch.cuda.stream(s):
                got.append(step(e, x, ptr, d))
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[k % len(encs)]))


def test_a_captured_encoder_keeps_its_scratch():
    """layers that need more scratch than the captured ones, and tensors where it may have been, between the replays"""
    from tsdiff_amd.train_ops import linear
    enc, = encoders(1)
    eager = copy.deepcopy(enc)  # leaves of its own beside the captured ones
    ptr = torch.tensor([0, 30, 300], dtype=torch.int32, device=DEV)
    h, d = torch.randn(300, 128, device=DEV).requires_grad_(), torch.randn(300, 128, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(enc, h, ptr, d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [t.detach() for t in step(enc, h, ptr, d)]
    kept = []
    for k in range(4):
        size = 256 * (k + 1)
        w = torch.randn(size, size, device=DEV).requires_grad_()
        y = linear(torch.randn(64, size, device=DEV), w)
        torch.autograd.grad(y.sum(), w)
        kept.append([torch.full((n,), 7.0, device=DEV) for n in (1 << 14, 1 << 16, 1 << 18, 1 << 20)])
        with torch.no_grad():
            h.copy_(torch.randn(300, 128, device=DEV))
        graph.replay()
        x = h.detach().clone().requires_grad_()
        want = step(eager, x, ptr, d)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(bool((t == 7).all()) for many in kept for t in many)


def test_encoders_of_several_threads_on_one_stream():
    import threading
    encs = encoders(3)
    ptr = torch.tensor([0, 30, 200], dtype=torch.int32, device=DEV)
    h = [torch.randn(200, 128, device=DEV) for _ in encs]
    with torch.no_grad():
        want = [e(x, ptr) for e, x in zip(encs, h)]
    torch.cuda.synchronize()
    wrong = []

    def go(k):
        with torch.no_grad():
            for _ in range(50):
                if not torch.equal(encs[k](h[k], ptr), want[k]):
                    wrong.append(k)

    threads = [threading.Thread(target=go, args=(k,)) for k in range(len(encs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_the_encoder_works_on_its_tensors_device(monkeypatch):
    """whichever device is current (the dense layers ask for the current one)"""
    enc, = encoders(1)
    entered, device = [], torch.cuda.device

    class Recorded(device):
        def __enter__(self):
            entered.append(self.idx)
            return super().__enter__()

    monkeypatch.setattr(torch.cuda, "device", Recorded)
    enc(torch.zeros(3, 128, device=DEV), torch.tensor([0, 3], dtype=torch.int32, device=DEV))
    assert entered == [0]
