"""CPU: forward-mode derivatives, which the operators of an attention block do not have, are refused before anything else is
looked at (no GPU call is made)."""
import pytest
import torch
import torch.autograd.forward_ad as fw


def calls():
    """(name, function of its tensors, the tensors)"""
    from tsdiff_amd import block_ops as B
    ptr = torch.tensor([0, 3], dtype=torch.int32)
    return [("layer_norm", lambda *t: B.layer_norm(*t), [torch.randn(s) for s in ((3, 8), (8,), (8,))]),
            ("gated_linear", lambda *t: B.gated_linear(*t), [torch.randn(s) for s in ((3, 8), (4, 8), (4, 8), (4,), (4,))]),
            ("graph_attention", lambda *t: B.graph_attention(*t, ptr), [torch.randn(3, 2, 8) for _ in range(3)])]


@pytest.mark.parametrize("recorded", [True, False])
def test_a_tangent_is_refused_in_every_place(recorded):
    with torch.set_grad_enabled(recorded):
        for name, f, tensors in calls():
            for k in range(len(tensors)):
                with fw.dual_level():
                    dual = list(tensors)
                    dual[k] = fw.make_dual(tensors[k], torch.ones_like(tensors[k]))
                    with pytest.raises(NotImplementedError, match=f"{name}.*forward"):
                        f(*dual)


def test_a_tangent_of_another_mode_is_refused_too():
    for name, f, tensors in calls():
        with pytest.raises(NotImplementedError, match=f"{name}.*forward"):
            torch.func.jvp(lambda x: f(x, *tensors[1:]), (tensors[0],), (torch.ones_like(tensors[0]),))
