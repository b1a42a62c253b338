"""MI355X: derivatives that the operators of an attention block do not have raise, where autograd would take a missing tangent
for zero."""
import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def calls():
    from tsdiff_amd import block_ops as B
    ptr = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    return [(B.layer_norm, [torch.randn(s, device=DEV) for s in ((3, 8), (8,), (8,))]),
            (B.gated_linear, [torch.randn(s, device=DEV) for s in ((3, 8), (4, 8), (4, 8), (4,), (4,))]),
            (lambda q, k, v: B.graph_attention(q, k, v, ptr), [torch.randn(3, 2, 8, device=DEV) for _ in range(3)])]


@pytest.mark.parametrize("recorded", [True, False])
@pytest.mark.parametrize("leaves", [True, False])
def test_forward_mode_raises(leaves, recorded):
    for f, tensors in calls():
        for k in range(len(tensors)):
            with fw.dual_level(), torch.set_grad_enabled(recorded):
                t = [x.clone().requires_grad_(leaves) for x in tensors]
                t[k] = fw.make_dual(t[k], torch.ones_like(t[k]))
                with pytest.raises(NotImplementedError):
                    f(*t)
            f(*tensors)  # outside of the level the same tensors are ordinary ones


def test_forward_over_reverse_raises():
    for f, tensors in calls():
        t = [x.clone().requires_grad_() for x in tensors]
        y = f(*t)
        d = torch.randn_like(y)
        with fw.dual_level():
            with pytest.raises((NotImplementedError, RuntimeError), match="forward"):
                torch.autograd.grad(y, t, fw.make_dual(d, torch.ones_like(d)))


def test_function_transforms_raise():
    for f, tensors in calls():
        for call in (lambda: torch.func.jvp(lambda x: f(x, *tensors[1:]), (tensors[0],), (torch.ones_like(tensors[0]),)),
                     lambda: torch.func.vmap(lambda x: f(x, *tensors[1:]))(torch.stack([tensors[0]] * 2)),
                     lambda: torch.func.grad(lambda x: f(x, *tensors[1:]).sum())(tensors[0])):
            with pytest.raises((NotImplementedError, RuntimeError)):
                call()
