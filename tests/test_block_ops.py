"""CPU: what the operators of an attention block refuse, in Python and at the C boundary, and their oracle against
differences of the formulas (no GPU call is made)."""
import ctypes as C

import pytest
import torch

from tests import block_oracle as O


def f32(*shape):
    return torch.zeros(*shape)


def test_shapes_are_refused():
    from tsdiff_amd import block_ops as B
    for call in (lambda: B.layer_norm(f32(3, 8), f32(7)), lambda: B.layer_norm(f32(3, 8), f32(8), f32(1, 8)),
                 lambda: B.layer_norm(torch.zeros(())), lambda: B.layer_norm(f32(3, 0)),
                 lambda: B.gated_linear(f32(3, 8), f32(4, 8), f32(5, 8)), lambda: B.gated_linear(f32(3, 8), f32(4, 7), f32(4, 7)),
                 lambda: B.gated_linear(f32(3, 8), f32(4, 8), f32(4, 8), f32(5)),
                 lambda: B.gated_linear(f32(3, 8), f32(0, 8), f32(0, 8)),
                 lambda: B.graph_attention(f32(3, 8), f32(3, 8), f32(3, 8), f32(2)),
                 lambda: B.graph_attention(f32(3, 3, 8), f32(3, 2, 8), f32(3, 2, 8), f32(2)),
                 lambda: B.graph_attention(f32(3, 2, 8), f32(3, 2, 4), f32(3, 2, 4), f32(2)),
                 lambda: B.graph_attention(f32(3, 2, 8), f32(3, 2, 8), f32(4, 2, 8), f32(2))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        B.gated_linear(f32(3, 8), f32(4, 8), f32(4, 8), act="tanh")


def test_cpu_tensors_are_refused():
    from tsdiff_amd import _lib, block_ops as B
    from tsdiff_amd.encoder import GraphTransformerEncoder
    ptr = torch.tensor([0, 3], dtype=torch.int32)
    for call in (lambda: B.layer_norm(f32(3, 8)), lambda: B.gated_linear(f32(3, 8), f32(4, 8), f32(4, 8)),
                 lambda: B.graph_attention(f32(3, 2, 8), f32(3, 2, 8), f32(3, 2, 8), ptr),
                 lambda: GraphTransformerEncoder(16, 1, 2)(f32(3, 16), ptr)):
        with pytest.raises(_lib.TsdError):
            call()
    with pytest.raises(ValueError):
        GraphTransformerEncoder(16, 1, 3)


def test_c_entries_refuse_before_any_launch():
    from tsdiff_amd import _lib
    lib = _lib.load()
    bad, no = _lib.TSD_ERR_INVALID, _lib.TSD_ERR_UNSUPPORTED
    p = 4096  # a pointer that nothing reads
    fwd = lib.tsd_layer_norm_fwd
    assert fwd(3, 4, 8, p, 8, p, p, 1e-5, p, None, None, None) == bad       # type
    assert fwd(0, 4, 0, p, 8, p, p, 1e-5, p, None, None, None) == bad       # dim
    assert fwd(0, -1, 8, p, 8, p, p, 1e-5, p, None, None, None) == bad      # rows
    assert fwd(0, 4, 8, p, 7, p, p, 1e-5, p, None, None, None) == bad       # row stride
    assert fwd(0, 4, 8, None, 8, p, p, 1e-5, p, None, None, None) == bad    # null
    assert fwd(0, 4, 8, p, 8, p, p, 1e-5, p, p, None, None) == bad          # mean without rstd
    assert fwd(0, 4, 8193, p, 8193, p, p, 1e-5, p, None, None, None) == no
    assert b"8192" in lib.tsd_last_error()
    assert fwd(0, 0, 8, None, 8, None, None, 1e-5, None, None, None, None) == 0
    bwd = lib.tsd_layer_norm_bwd
    assert bwd(0, 4, 8, p, 8, p, None, 8, p, p, p, p, p, p, 1 << 20, None) == bad
    assert bwd(0, 4, 8, p, 8, p, p, 8, p, p, p, p, p, p, 1, None) == bad    # scratch
    assert bwd(0, 4, 8, p, 8, p, p, 8, p, p, p, p, p, None, 0, None) == bad
    g = lib.tsd_gated_linear_fwd
    assert g(5, 0, 4, 8, 8, p, 8, p, p, None, None, p, None, 0, None) == bad
    assert g(0, 4, 4, 8, 8, p, 8, p, p, None, None, p, None, 0, None) == bad         # activation
    assert g(0, 0, 4, 0, 8, p, 8, p, p, None, None, p, None, 0, None) == bad
    assert g(0, 0, 4, 8, 8, p, 7, p, p, None, None, p, None, 0, None) == bad
    assert g(0, 0, 4, 8, 8, p, 8, p, None, None, None, p, None, 0, None) == bad
    assert g(0, 0, 4, 8, 8, p, 8, p, p, None, None, None, None, 0, None) == bad
    assert g(0, 0, 4, 1 << 21, 8, p, 1 << 21, p, p, None, None, p, None, 0, None) == no
    n = lib.tsd_gated_linear_scratch_floats(1, 4096, 33, 64, p, 33, p, p, 0)  # rows that no 16-byte load fits: copies
    assert n > 0 and g(1, 0, 4096, 33, 64, p, 33, p, p, None, None, p, p, n - 1, None) == bad
    assert lib.tsd_gated_linear_scratch_floats(1, 4096, 32, 64, p, 32, p, p, 0) == 0
    gb = lib.tsd_gated_linear_bwd
    n = lib.tsd_gated_linear_scratch_floats(0, 4, 8, 8, p, 8, p, p, 1)
    assert n > 0
    assert gb(0, 0, 4, 8, 8, p, 8, p, p, None, None, p, 8, p, p, p, None, None, p, n - 1, None) == bad
    assert gb(0, 0, 4, 8, 8, p, 8, p, p, None, None, p, 8, p, p, p, None, None, p + 4, n, None) == bad  # alignment
    assert gb(0, 0, 4, 8, 8, p, 8, p, p, None, None, p, 7, p, p, p, None, None, p, n, None) == bad

    def att(**kw):
        a = dict(dtype=0, num_graphs=2, num_queries=4, num_keys=4, heads=4, kv_heads=2, dim=8, scale=1.0, q=p, k=p, v=p,
                 q_row=32, q_head=8, k_row=16, k_head=8, v_row=16, v_head=8, q_ptr=p, k_ptr=p)
        a.update(kw)
        return C.byref(_lib.Attention(**a))

    af, ab = lib.tsd_graph_attention_fwd, lib.tsd_graph_attention_bwd
    for kw in (dict(dtype=7), dict(kv_heads=3), dict(kv_heads=0), dict(dim=0), dict(num_graphs=-1), dict(q=None), dict(v=None),
               dict(q_ptr=None), dict(k_ptr=None), dict(num_keys=-1)):
        assert af(att(**kw), p, None, None, None, 0, None) == bad, kw
    assert af(att(dim=129), p, None, None, None, 0, None) == no
    assert af(att(num_queries=1 << 30), p, None, None, None, 0, None) == no
    assert af(att(), None, None, None, None, 0, None) == bad
    assert ab(att(), p, None, p, p, 32, 8, p, p, p, None, 0, None) == bad          # scratch
    assert ab(att(), p, None, p, p, 32, 8, None, p, p, p, 1 << 20, None) == bad
    long = dict(num_graphs=1, num_queries=1, num_keys=1 << 16)               # few rows, many keys: parts to be joined
    n = lib.tsd_graph_attention_scratch_floats(att(**long), 0)
    assert n > 0 and af(att(**long), p, None, None, p, n - 1, None) == bad


def test_c_attention_refuses_what_its_launches_and_offsets_do_not_reach():
    from tsdiff_amd import _lib
    lib = _lib.load()
    p = 4096
    for sizes in (dict(num_queries=1 << 29), dict(num_keys=1 << 29), dict(num_graphs=1 << 23), dict(heads=1 << 17, kv_heads=1 << 17)):
        a = dict(dtype=1, num_graphs=2, num_queries=4, num_keys=4, heads=4, kv_heads=1, dim=8, scale=1.0, q=p, k=p, v=p, q_ptr=p,
                 k_ptr=p)
        a.update(sizes)
        a = C.byref(_lib.Attention(**a))
        assert lib.tsd_graph_attention_scratch_floats(a, 1) == 0
        assert lib.tsd_graph_attention_fwd(a, p, None, None, None, 0, None) == _lib.TSD_ERR_UNSUPPORTED
        assert lib.tsd_graph_attention_bwd(a, p, None, p, p, 32, 8, p, p, p, p, 1 << 40, None) == _lib.TSD_ERR_UNSUPPORTED


def close(got, want, tol=1e-6):
    assert float((got - want).abs().max()) <= tol * max(1.0, float(want.abs().max()))


@pytest.mark.parametrize("kind", ["swish", "ssp", "ReLU", "Softplus"])
def test_the_oracle_of_the_gated_layer_is_differentiable_as_it_says(kind):
    g = torch.Generator().manual_seed(1)
    x, wg, wu, bg, bu = (torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()
                         for s in ((5, 6), (7, 6), (7, 6), (7,), (7,)))
    dh = torch.randn(5, 7, generator=g, dtype=torch.float64)
    got = O.gated(x.detach(), wg.detach(), wu.detach(), bg.detach(), bu.detach(), kind, dh)
    a, v = x @ wg.t() + bg, x @ wu.t() + bu
    f = {"swish": torch.nn.functional.silu, "ReLU": torch.relu, "Softplus": torch.nn.functional.softplus,
         "ssp": lambda t: torch.nn.functional.softplus(t) - torch.log(torch.tensor(2.0, dtype=torch.float64))}[kind]
    h = f(a) * v
    close(got["h"][0], h.detach())
    for n, t in zip(("dx", "dwg", "dwu", "dbg", "dbu"), torch.autograd.grad(h, (x, wg, wu, bg, bu), dh)):
        close(got[n][0], t)


def test_the_oracle_of_layer_norm_is_differentiable_as_it_says():
    g = torch.Generator().manual_seed(2)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_() for s in ((5, 6), (6,), (6,)))
    dy = torch.randn(5, 6, generator=g, dtype=torch.float64)
    got = O.norm(x.detach(), w.detach(), b.detach(), 1e-5, dy)
    y = torch.nn.functional.layer_norm(x, (6,), w, b, 1e-5)
    close(got["y"][0], y.detach())
    for n, t in zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), dy)):
        close(got[n][0], t)


def test_the_oracle_of_attention_agrees_with_differences():
    g = torch.Generator().manual_seed(3)
    q, k, v, do = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((6, 4, 3), (7, 2, 3), (7, 2, 3), (6, 4, 3)))
    qp, kp, mask = [0, 2, 2, 5], [0, 3, 4, 6], torch.tensor([1, 0, 1, 1, 1, 1, 1], dtype=torch.bool)
    got = O.attention(q, k, v, qp, kp, mask, 0.7, do)
    assert float(got["out"][0][5].abs().max()) == 0 and float(got["dk"][0][[1, 3, 6]].abs().max()) == 0
    step = 1e-5
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        for i in range(0, t.numel(), 5):
            f = []
            for sign in (1, -1):
                u = t.clone()
                u.view(-1)[i] += sign * step
                args = {"dq": (u, k, v), "dk": (q, u, v), "dv": (q, k, u)}[name]
                f.append(float((O.attention(*args, qp, kp, mask, 0.7)["out"][0] * do).sum()))
            assert abs((f[0] - f[1]) / (2 * step) - float(got[name][0].reshape(-1)[i])) < 1e-7
