"""MI355X: the operators of an attention block (tsdiff_amd.block_ops) against their definitions in 64 bits, with the
tolerances that tests/block_oracle.py derives; gradients through autograd and the C ABI."""
import pytest
import torch

from tests import block_oracle as O

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
DEV = "cuda:0"


def normal(seed, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    """on the CPU, already of the type's values"""
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def dev(*tensors, grad=True):
    return [None if t is None else t.to(DEV).requires_grad_(grad) for t in tensors]


# ---- layer norm -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (17, 64), (5, 100), (130, 128), (17, 256), (33, 257), (9, 512), (7, 1000),
                                      (4, 1030), (3, 2047), (5, 2048), (3, 4096), (2, 4098), (2, 8191), (3, 8192)])
def test_layer_norm(rows, dim, dtype):
    from tsdiff_amd.block_ops import layer_norm
    x, w, b, dy = (normal(1, rows, dim, dtype=dtype, scale=2.0, shift=0.5), normal(2, dim, dtype=dtype, shift=1.0, scale=0.3),
                   normal(3, dim, dtype=dtype), normal(4, rows, dim, dtype=dtype))
    want = O.norm(x, w, b, 1e-5, dy, dtype)
    xd, wd, bd = dev(x, w, b)
    y = layer_norm(xd, wd, bd)
    assert y.dtype == dtype
    O.check(y, want["y"], "y")
    with torch.no_grad():
        assert torch.equal(layer_norm(xd, wd, bd), y)
    for n, t in zip(("dx", "dw", "db"), torch.autograd.grad(y, (xd, wd, bd), dy.to(DEV))):
        O.check(t, want[n], n)


@pytest.mark.parametrize("rows", [4099, 40000])
def test_layer_norm_of_many_rows(rows):
    from tsdiff_amd.block_ops import layer_norm
    x, w, b, dy = normal(1, rows, 64), normal(2, 64), normal(3, 64), normal(4, rows, 64)
    want = O.norm(x, w, b, 1e-5, dy)
    xd, wd, bd = dev(x, w, b)
    y = layer_norm(xd, wd, bd)
    O.check(y, want["y"], "y")
    for n, t in zip(("dx", "dw", "db"), torch.autograd.grad(y, (xd, wd, bd), dy.to(DEV))):
        O.check(t, want[n], n)


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_strides_shapes_and_missing_parameters(dtype):
    from tsdiff_amd.block_ops import layer_norm
    big, dyb = normal(1, 6, 5, 80, dtype=dtype), normal(2, 6, 5, 48, dtype=dtype)
    for cut, dcut in ((slice(0, 48), slice(0, 48)), (slice(3, 36), slice(0, 33)), (slice(0, 80, 2), slice(0, 40))):
        x, dy = big[..., cut], dyb[..., dcut]
        want = O.norm(x.reshape(30, -1), None, None, 1e-3, dy.reshape(30, -1), dtype)
        xd = big.to(DEV).requires_grad_()
        y = layer_norm(xd[..., cut], eps=1e-3)
        assert y.shape == x.shape
        O.check(y.reshape(30, -1), want["y"], "y")
        g, = torch.autograd.grad(y, xd, dyb.to(DEV)[..., dcut])
        O.check(g[..., cut].reshape(30, -1), want["dx"], "dx")
    # one row for all, one gradient for all: what broadcasting hands over
    x, w = normal(3, 1, 40, dtype=dtype), normal(4, 40, dtype=dtype)
    xd, wd = dev(x, w)
    y = layer_norm(xd.expand(9, 40), wd)
    want = O.norm(x.expand(9, 40), w, None, 1e-5, torch.ones(9, 40), dtype)
    O.check(y, want["y"], "y")
    gx, gw = torch.autograd.grad(y.sum(), (xd, wd))
    O.check(gw, want["dw"], "dw")
    dx, tol = want["dx"]
    O.check(gx, (dx.sum(0, keepdim=True), tol.sum(0, keepdim=True) + O.rounded(dx.sum(0, keepdim=True), dtype) +
                 9 * O.rounded(dx.abs().sum(0, keepdim=True), dtype)), "dx")


def test_layer_norm_of_far_means_infinities_and_no_rows():
    from tsdiff_amd.block_ops import layer_norm
    x = normal(1, 8, 256, shift=3000.0)  # the centred values are computed, not a difference of squares
    O.check(layer_norm(x.to(DEV)), O.norm(x, None, None, 1e-5)["y"], "y")
    y = torch.zeros(3, 64)
    y[1, 5] = float("inf")
    got = layer_norm(y.to(DEV)).cpu()
    assert torch.equal(got[[0, 2]], torch.zeros(2, 64)) and got[1].isnan().any()
    xd, wd = dev(torch.empty(0, 16), normal(2, 16))
    y = layer_norm(xd, wd)
    gx, gw = torch.autograd.grad(y.sum(), (xd, wd))
    assert y.shape == (0, 16) and gx.shape == (0, 16) and torch.equal(gw, torch.zeros(16, device=DEV))


# ---- gated linear layer ---------------------------------------------------------------------------------------
def gated_case(rows, fin, out, dtype, act, bias, seed=1):
    x, wg, wu, dh = (normal(seed, rows, fin, dtype=dtype), normal(seed + 1, out, fin, dtype=dtype, scale=fin ** -0.5),
                     normal(seed + 2, out, fin, dtype=dtype, scale=fin ** -0.5), normal(seed + 3, rows, out, dtype=dtype))
    bg, bu = (normal(seed + 4, out, dtype=dtype), normal(seed + 5, out, dtype=dtype)) if bias else (None, None)
    return x, wg, wu, bg, bu, dh, O.gated(x, wg, wu, bg, bu, act, dh, dtype)


def gated_check(got, grads, want):
    O.check(got, want["h"], "h")
    for n, t in grads.items():
        O.check(t, want[n], n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,fin,out", [(1, 1, 1), (1, 16, 8), (17, 256, 512), (5, 24, 40), (130, 33, 70), (64, 64, 64),
                                          (257, 100, 129), (300, 204, 530), (520, 965, 129), (1000, 8, 16), (40, 1000, 12)])
def test_gated_linear(rows, fin, out, dtype):
    from tsdiff_amd.block_ops import gated_linear
    x, wg, wu, bg, bu, dh, want = gated_case(rows, fin, out, dtype, "swish", True)
    t = dev(x, wg, wu, bg, bu)
    h = gated_linear(*t)
    assert h.dtype == dtype
    gated_check(h, dict(zip(("dx", "dwg", "dwu", "dbg", "dbu"), torch.autograd.grad(h, t, dh.to(DEV)))), want)


@pytest.mark.parametrize("dtype,rows,fin,out", [(torch.bfloat16, 16300, 1020, 136), (torch.float16, 56000, 240, 124),
                                                (torch.bfloat16, 8100, 40, 1016), (torch.float32, 9001, 72, 264)])
def test_gated_linear_of_many_rows(dtype, rows, fin, out):
    """the largest tiles, each ending inside of one"""
    from tsdiff_amd.block_ops import gated_linear
    x, wg, wu, bg, bu, dh, want = gated_case(rows, fin, out, dtype, "swish", True)
    t = dev(x, wg, wu, bg, bu)
    h = gated_linear(*t)
    gated_check(h, dict(zip(("dx", "dwg", "dwu", "dbg", "dbu"), torch.autograd.grad(h, t, dh.to(DEV)))), want)


@pytest.mark.parametrize("act", ["swish", "ssp", "ReLU", "Softplus"])
def test_gated_linear_activations_without_biases(act):
    from tsdiff_amd.block_ops import gated_linear
    x, wg, wu, _, _, dh, want = gated_case(70, 48, 72, torch.float32, act, False)
    t = dev(x, wg, wu)
    h = gated_linear(*t, act=act)
    gated_check(h, dict(zip(("dx", "dwg", "dwu"), torch.autograd.grad(h, t, dh.to(DEV)))), want)
    far = dev(torch.tensor([[400.0], [-400.0], [0.0]]), torch.ones(1, 1), torch.ones(1, 1))  # no overflow on the way
    h = gated_linear(*far, act=act)
    assert h.isfinite().all() and all(g.isfinite().all() for g in torch.autograd.grad(h.sum(), far))


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_linear_strides_and_single_gradients(dtype):
    from tsdiff_amd.block_ops import gated_linear
    x, wg, wu, bg, bu, dh, want = gated_case(66, 40, 48, dtype, "swish", True, seed=9)
    wide, dwide = torch.full((66, 51), 7.0, dtype=dtype), torch.full((66, 64), 9.0, dtype=dtype)
    for at in (0, 3, 8):
        wide[:, at:at + 40], dwide[:, at:at + 48] = x, dh
        xd = wide.to(DEV)[:, at:at + 40].requires_grad_()
        rest = dev(wg, wu, bg, bu)
        h = gated_linear(xd, *rest)
        grads = torch.autograd.grad(h, [xd] + rest, dwide.to(DEV)[:, at:at + 48])
        gated_check(h, dict(zip(("dx", "dwg", "dwu", "dbg", "dbu"), grads)), want)
    for k, n in enumerate(("dx", "dwg", "dwu", "dbg", "dbu")):
        t = dev(x, wg, wu, bg, bu, grad=False)
        t[k].requires_grad_()
        g, = torch.autograd.grad(gated_linear(*t), t[k], dh.to(DEV))
        O.check(g, want[n], n)


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_linear_copies_odd_rows_of_strided_inputs(dtype):
    """rows that no 16-byte load fits, long products: a slice of wider rows, weights between two borders"""
    from tsdiff_amd.block_ops import gated_linear
    x, wg, wu, bg, bu, dh, want = gated_case(600, 121, 77, dtype, "swish", True, seed=5)
    xd = torch.full((600, 130), float("nan"), dtype=dtype)
    xd[:, 3:124] = x
    xd = xd.to(DEV)[:, 3:124].requires_grad_()
    w = torch.cat((torch.zeros(1, dtype=dtype), wg.flatten(), wu.flatten())).to(DEV)
    rest = [w[1:1 + wg.numel()].view(77, 121).requires_grad_(), w[1 + wg.numel():].view(77, 121).requires_grad_()] + dev(bg, bu)
    h = gated_linear(xd, *rest)
    grads = torch.autograd.grad(h, [xd] + rest, dh.to(DEV))
    gated_check(h, dict(zip(("dx", "dwg", "dwu", "dbg", "dbu"), grads)), want)


def test_gated_linear_without_rows_and_in_three_dimensions():
    from tsdiff_amd.block_ops import gated_linear
    x, wg, wu, bg, bu, dh, want = gated_case(6, 16, 24, torch.float32, "swish", True)
    t = dev(torch.empty(0, 16), wg, wu)
    h = gated_linear(*t)
    grads = torch.autograd.grad(h.sum(), t)
    assert h.shape == (0, 24) and grads[0].shape == (0, 16) and not grads[1].any() and not grads[2].any()
    h = gated_linear(x.to(DEV).view(2, 3, 16), *dev(wg, wu, bg, bu))
    assert h.shape == (2, 3, 24)
    O.check(h.reshape(6, 24), want["h"], "h")


# ---- attention ------------------------------------------------------------------------------------------------
def offsets(sizes, first=0):
    p = [first]
    for s in sizes:
        p.append(p[-1] + s)
    return p


def attention_case(qs, ks, heads, kv_heads, dim, dtype, masked, seed=1, extra=0):
    """self attention where ks is None; `extra` rows and keys in front of the first graph and behind the last"""
    qp = offsets(qs, extra)
    kp = qp if ks is None else offsets(ks, extra)
    nq, nk = qp[-1] + extra, kp[-1] + extra
    q, k, v, do = (normal(seed, nq, heads, dim, dtype=dtype), normal(seed + 1, nk, kv_heads, dim, dtype=dtype),
                   normal(seed + 2, nk, kv_heads, dim, dtype=dtype), normal(seed + 3, nq, heads, dim, dtype=dtype))
    mask = None
    if masked:
        mask = torch.rand(nk, generator=torch.Generator().manual_seed(seed + 4)) > 0.3
        mask[kp[0]:kp[1]] = False  # the first graph has no open key
    return q, k, v, do, qp, kp, mask, O.attention(q, k, v, qp, kp, mask, dim ** -0.5, do, dtype)


def attention_run(q, k, v, do, qp, kp, mask, want, same=False):
    from tsdiff_amd.block_ops import graph_attention
    t = dev(q, k, v)
    ptr = torch.tensor(qp, dtype=torch.int32, device=DEV)
    kptr = None if same else torch.tensor(kp, device=DEV)
    m = None if mask is None else mask.to(DEV)
    out = graph_attention(*t, ptr, key_ptr=kptr, key_mask=m)
    assert out.dtype == q.dtype
    O.check(out, want["out"], "out")
    with torch.no_grad():
        assert torch.equal(graph_attention(*t, ptr, key_ptr=kptr, key_mask=m), out)
    grads = torch.autograd.grad(out, t, do.to(DEV))
    for n, g in zip(("dq", "dk", "dv"), grads):
        O.check(g, want[n], n)
    return (out,) + grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 8, 16, 24, 32, 33, 64, 72, 128])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (4, 1)])
def test_attention_of_small_graphs(heads, kv_heads, dim, dtype):
    c = attention_case([1, 17, 0, 16, 31, 2, 33], None, heads, kv_heads, dim, dtype, False)
    attention_run(*c, same=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [16, 64, 100])
def test_attention_of_middling_graphs_with_masks(dim, dtype):
    c = attention_case([70, 64, 129, 200, 1], None, 4, 2, dim, dtype, True, extra=3)
    attention_run(*c)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("qs,ks,heads,kv_heads,dim", [
    ([1, 1, 1], [300, 2000, 5], 4, 4, 32),       # a readout: the keys are split
    ([2, 0, 3], [1500, 40, 0], 6, 2, 64),
    ([1], [3000], 3, 1, 128),
    ([700, 900], [1, 3], 2, 2, 40),              # few keys, many rows: the rows are split
    ([2500], [2], 4, 1, 32),
    ([40, 5, 100], [9, 70, 64], 3, 3, 16),
])
def test_attention_with_queries_of_their_own(qs, ks, heads, kv_heads, dim, dtype):
    attention_run(*attention_case(qs, ks, heads, kv_heads, dim, dtype, len(qs) > 1))


@pytest.mark.parametrize("dtype,dim,masked", [(torch.float32, 8, False), (torch.float16, 72, False), (torch.float16, 72, True)])
def test_attention_over_more_keys_than_one_list_of_tiles_holds(dtype, dim, masked):
    attention_run(*attention_case([4, 512], [30, 4200], 64, 64, dim, dtype, masked))


@pytest.mark.parametrize("graphs", [1, 62, 63, 64, 65, 200, 4100])
def test_attention_finds_the_graph_of_every_tile(graphs):
    sizes = [(7 * i) % 5 for i in range(graphs)]
    attention_run(*attention_case(sizes, None, 1, 1, 8, torch.float32, False, extra=2), same=True)


def test_attention_without_graphs_rows_or_keys():
    for qs, ks, extra in (([], [], 0), ([], [], 5), ([0, 0], [0, 0], 0), ([3], [0], 0), ([0], [3], 0), ([0, 2], [70, 0], 1)):
        attention_run(*attention_case(qs, ks, 2, 2, 8, torch.float32, False, extra=extra))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_never_reads_masked_keys(dtype):
    """NaN and infinities behind the mask, outside of the graphs and in rows that no key answers change nothing"""
    q, k, v, do, qp, kp, mask, want = attention_case([20, 70, 9], None, 2, 1, 32, dtype, True, extra=4)
    plain = attention_run(q, k, v, do, qp, kp, mask, want)
    closed = ~mask
    closed[:4] = closed[-4:] = True
    for bad in (float("nan"), float("inf"), torch.finfo(dtype).min):
        q2, k2, v2, do2 = q.clone(), k.clone(), v.clone(), do.clone()
        k2[closed] = v2[closed] = bad
        for t in (q2, do2):  # the first graph has no open key
            t[:24] = t[-4:] = bad
        for a, b in zip(plain, attention_run(q2, k2, v2, do2, qp, kp, mask, want)):
            assert torch.equal(a, b)
    assert not plain[0][:24].any() and not plain[1][:24].any()
    assert not plain[2][closed.to(DEV)].any() and not plain[3][closed.to(DEV)].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_reads_slices_of_one_projection(dtype):
    from tsdiff_amd.block_ops import graph_attention
    q, k, v, do, qp, kp, mask, want = attention_case([30, 50], None, 4, 2, 24, dtype, False)
    ptr = torch.tensor(qp, dtype=torch.int32, device=DEV)
    for pad in (0, 1, 8):  # an odd row stride has no aligned rows
        row = torch.zeros(80, 8 * 24 + pad, dtype=dtype)
        row[:, :8 * 24] = torch.cat((q, k, v), 1).reshape(80, -1)
        rd = row.to(DEV).requires_grad_()
        qkv = rd[:, :8 * 24].view(80, 8, 24) if pad == 0 else rd[:, :8 * 24].unflatten(1, (8, 24))
        out = graph_attention(*qkv.split((4, 2, 2), 1), ptr)
        O.check(out, want["out"], "out")
        dod = do.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)  # heads first in memory
        g = torch.autograd.grad(out, rd, dod)[0][:, :8 * 24].view(80, 8, 24)
        for n, t in zip(("dq", "dk", "dv"), g.split((4, 2, 2), 1)):
            O.check(t, want[n], n)
    # one key head handed over as an expanded view, no contiguous last dimension
    qd, kd, vd = q.to(DEV), k.to(DEV)[:, :1].expand(80, 4, 24), v.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    want = O.attention(q, k[:, :1].expand(80, 4, 24), v.repeat_interleave(2, 1), qp, kp, None, 24 ** -0.5, None, dtype)
    O.check(graph_attention(qd, kd, vd.repeat_interleave(2, 1), ptr), want["out"], "out")


def test_attention_offsets_are_clamped_into_the_tensors():
    from tsdiff_amd.block_ops import graph_attention
    q = normal(1, 20, 2, 8).to(DEV)
    out = graph_attention(q, q, q, torch.tensor([-5, 7, 50], dtype=torch.int32, device=DEV))
    want = graph_attention(q, q, q, torch.tensor([0, 7, 20], dtype=torch.int32, device=DEV))
    assert torch.equal(out, want)


def test_large_scores_do_not_overflow():
    from tsdiff_amd.block_ops import graph_attention
    q, k, v = (normal(s, 40, 1, 32) for s in (1, 2, 3))
    ptr = torch.tensor([0, 40], dtype=torch.int32, device=DEV)
    for scale in (100.0, -100.0, 0.0):
        want = O.attention(q, k, v, [0, 40], [0, 40], None, scale)
        O.check(graph_attention(*dev(q, k, v), ptr, scale=scale), want["out"], f"scale {scale}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.4, 60.0, -60.0])
def test_attention_of_any_scale_with_masks(scale, dtype):
    """whatever the scale makes of the largest score, a masked key's is no candidate"""
    from tsdiff_amd.block_ops import graph_attention
    q, k, v, do, qp, kp, mask, _ = attention_case([20, 70, 9], None, 2, 1, 24, dtype, True, extra=4)
    want = O.attention(q, k, v, qp, kp, mask, scale, do, dtype)
    k, v = k.clone(), v.clone()
    k[~mask] = v[~mask] = float("nan")
    t = dev(q, k, v)
    out = graph_attention(*t, torch.tensor(qp, device=DEV), key_mask=mask.to(DEV).to(torch.uint8) * 254, scale=scale)
    O.check(out, want["out"], "out")
    for n, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, t, do.to(DEV))):
        O.check(g, want[n], n)


@pytest.mark.parametrize("n", [20, 200])
def test_rows_whose_scores_are_all_minus_infinity_count_as_rows_without_keys(n):
    from tsdiff_amd.block_ops import graph_attention
    q, k, v, do = (normal(s, 2 * n, 1, 32, dtype=torch.bfloat16) for s in (1, 2, 3, 4))
    q[:n] = q[:n].abs() + 1
    k[:n] = float("-inf")  # every key of the first graph
    t = dev(q, k, v)
    out = graph_attention(*t, torch.tensor([0, n, 2 * n], device=DEV))
    grads = torch.autograd.grad(out, t, do.to(DEV))
    want = O.attention(q[n:], k[n:], v[n:], [0, n], [0, n], None, 32 ** -0.5, do[n:], torch.bfloat16)
    for name, g in zip(("out", "dq", "dk", "dv"), (out,) + grads):
        assert not g[:n].any(), name
        O.check(g[n:], want[name], name)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_with_key_heads_that_no_power_of_two_divides(dtype):
    """5 key heads of 3 heads each, and so many graphs that a workgroup goes over several key heads"""
    attention_run(*attention_case([(7 * i) % 4 for i in range(700)], None, 15, 5, 8, dtype, False), same=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_c_attention_without_what_the_rounding_left(dtype):
    """the C entries, into the middle of buffers that nothing else of may change; out_rest and the forward's lse left out"""
    import ctypes as C

    from tsdiff_amd import _lib
    lib = _lib.load()
    q, k, v, do, qp, kp, mask, want = attention_case([20, 33], None, 2, 2, 32, dtype, False)
    t = dev(q, k, v, do, grad=False)
    ptr = torch.tensor(qp, dtype=torch.int32, device=DEV)
    a = _lib.Attention(dtype=1 if dtype == torch.bfloat16 else 2, num_graphs=2, num_queries=53, num_keys=53, heads=2, kv_heads=2,
                       dim=32, scale=32 ** -0.5, q=t[0].data_ptr(), k=t[1].data_ptr(), v=t[2].data_ptr(), q_row=64, q_head=32,
                       k_row=64, k_head=32, v_row=64, v_head=32, q_ptr=ptr.data_ptr(), k_ptr=ptr.data_ptr(), key_mask=None)
    n = 53 * 64
    whole = [torch.full((n + 128,), 5.0, dtype=dtype, device=DEV) for _ in range(5)]
    at = [w[64:].data_ptr() for w in whole]
    lse = torch.empty(53, 2, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.tsd_graph_attention_fwd(C.byref(a), at[4], None, None, None, 0, stream) == 0
    assert lib.tsd_graph_attention_fwd(C.byref(a), at[0], None, lse.data_ptr(), None, 0, stream) == 0
    floats = lib.tsd_graph_attention_scratch_floats(C.byref(a), 1)
    scratch = torch.empty(floats, device=DEV)
    assert lib.tsd_graph_attention_bwd(C.byref(a), at[0], None, lse.data_ptr(), t[3].data_ptr(), 64, 32, at[1], at[2], at[3],
                                       scratch.data_ptr(), floats, stream) == 0
    assert torch.equal(whole[0], whole[4])
    for name, w in zip(("out", "dq", "dk", "dv"), whole):
        assert (w[:64] == 5).all() and (w[64 + n:] == 5).all()
        O.check(w[64:64 + n].view(53, 2, 32), want[name], name)


# ---- all of them ----------------------------------------------------------------------------------------------
def three(seed, n=70, dtype=torch.float32, h=64):
    """a call of each operator: function of leaves, the leaves, a gradient"""
    from tsdiff_amd import block_ops as B
    ptr = torch.tensor([0, 20, n], dtype=torch.int32, device=DEV)
    x = dev(normal(seed, n, h, dtype=dtype), normal(seed + 1, h, dtype=dtype), normal(seed + 2, h, dtype=dtype))
    w = dev(normal(seed + 3, n, h, dtype=dtype), normal(seed + 4, 96, h, dtype=dtype), normal(seed + 5, 96, h, dtype=dtype),
            normal(seed + 6, 96, dtype=dtype), normal(seed + 7, 96, dtype=dtype))
    q = dev(*(normal(seed + 8 + i, n, 2, 32, dtype=dtype) for i in range(3)))
    return [(B.layer_norm, x, normal(seed + 11, n, h, dtype=dtype).to(DEV)),
            (B.gated_linear, w, normal(seed + 12, n, 96, dtype=dtype).to(DEV)),
            (lambda a, b, c: B.graph_attention(a, b, c, ptr), q, normal(seed + 13, n, 2, 32, dtype=dtype).to(DEV))]


@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_bits_every_time_and_on_other_streams(dtype):
    for f, leaves, d in three(20, dtype=dtype):
        def go():
            y = f(*leaves)
            return (y,) + torch.autograd.grad(y, leaves, d)
        first = go()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(3)]
        got = []
        for s in streams * 3:  # side by side: no call keeps anything for the next
            with torch.cuda.stream(s):
                got.append(go())
        torch.cuda.synchronize()
        for g in got:
            assert all(torch.equal(a, b) for a, b in zip(first, g))


def test_calls_of_several_threads_at_once():
    import threading
    want = [[f(*leaves) for f, leaves, _ in three(40 + k, n=60 + 10 * k)] for k in range(4)]
    torch.cuda.synchronize()
    wrong = []

    def go(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                for (f, leaves, d), w in zip(three(40 + k, n=60 + 10 * k), want[k]):
                    y = f(*leaves)
                    torch.autograd.grad(y, leaves, d)
                    if not torch.equal(y, w):
                        wrong.append(k)

    threads = [threading.Thread(target=go, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong


@pytest.mark.parametrize("dtype", TYPES)
def test_captured_forward_and_backward_replay(dtype):
    for f, leaves, d in three(40, dtype=dtype):
        static = [t.detach().clone().requires_grad_() for t in leaves]  # leaves of the graph's own
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y = f(*static)
            torch.autograd.grad(y, static, d)
        torch.cuda.current_stream().wait_stream(side)
        del y
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = f(*static)
            grads = torch.autograd.grad(y, static, d)
        for k in range(4):
            fresh = [(t.detach() * (1 + 0.1 * k)).requires_grad_() for t in leaves]
            with torch.no_grad():
                for a, b in zip(static, fresh):
                    a.copy_(b)
            graph.replay()
            eager = f(*fresh)
            want = torch.autograd.grad(eager, fresh, d)
            torch.cuda.synchronize()
            assert torch.equal(y, eager) and all(torch.equal(a, b) for a, b in zip(grads, want))


def test_second_derivatives_and_wrong_types_are_refused():
    from tsdiff_amd import block_ops as B
    for f, leaves, d in three(60):
        g = torch.autograd.grad(f(*leaves), leaves[0], d, create_graph=True)[0]
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), leaves[0])
    x = torch.zeros(4, 8, device=DEV)
    ptr = torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    q = x.view(4, 1, 8)
    for call in (lambda: B.layer_norm(x.double()), lambda: B.layer_norm(x, x[0].half()), lambda: B.layer_norm(x, x[0].cpu()),
                 lambda: B.gated_linear(x, x.half(), x.half()), lambda: B.graph_attention(q, q.half(), q.half(), ptr),
                 lambda: B.graph_attention(q, q, q, ptr.float()), lambda: B.graph_attention(q, q, q, ptr.cpu()),
                 lambda: B.graph_attention(q, q, q, ptr, key_ptr=ptr[:1]), lambda: B.graph_attention(q, q[:3], q[:3], ptr),
                 lambda: B.graph_attention(q, q, q, ptr, key_mask=torch.ones(4, device=DEV)),
                 lambda: B.graph_attention(q, q, q, ptr, key_mask=torch.ones(3, dtype=torch.bool, device=DEV)),
                 lambda: B.graph_attention(q, q, q, ptr, key_mask=torch.ones(4, dtype=torch.bool))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        B.layer_norm(torch.zeros(2, 8200, device=DEV))
    with pytest.raises(NotImplementedError):
        B.graph_attention(*(torch.zeros(4, 1, 136, device=DEV),) * 3, ptr)


def test_offsets_past_32_bits():
    """rows 2^21 values apart: the last ones lie past 2^31 values"""
    from tsdiff_amd import block_ops as B
    n, gap = 1040, 1 << 21
    far = torch.empty(n * gap, dtype=torch.bfloat16, device=DEV)
    x = normal(1, n, 64, dtype=torch.bfloat16).to(DEV)
    xf = far.view(n, gap)[:, :64]
    xf.copy_(x)
    w, wu = normal(2, 24, 64, dtype=torch.bfloat16).to(DEV), normal(3, 24, 64, dtype=torch.bfloat16).to(DEV)
    ptr = torch.tensor([0, 3, n], dtype=torch.int32, device=DEV)

    def all_of(t):
        t = t.detach().requires_grad_()
        h = t.view(n, 2, 32) if t.is_contiguous() else t.unflatten(1, (2, 32))
        outs = [B.layer_norm(t), B.gated_linear(t, w, wu), B.graph_attention(h, h, h, ptr)]
        return outs + [torch.autograd.grad(o, t, o.detach())[0] for o in outs]

    for a, b in zip(all_of(x), all_of(xf)):
        assert torch.equal(a, b)


def test_encoder_block_against_float64():
    """the operators together, as an encoder runs them: outputs and every parameter's gradient against the same block in 64
    bits on the CPU (errors of chained fp32 operators: 1e-5 of a tensor's scale, the bound of the package's parity tests)"""
    from tsdiff_amd.encoder import GraphTransformerEncoder
    torch.manual_seed(5)
    enc = GraphTransformerEncoder(64, num_blocks=2, num_heads=4, num_kv_heads=2, ff_dim=96)
    sizes = [9, 1, 23, 40]
    ptr = offsets(sizes)
    h, dy = normal(1, ptr[-1], 64), normal(2, ptr[-1], 64)
    mask = torch.rand(ptr[-1], generator=torch.Generator().manual_seed(3)) > 0.2
    mask[:9] = False
    ref = GraphTransformerEncoder(64, num_blocks=2, num_heads=4, num_kv_heads=2, ff_dim=96).double()
    ref.load_state_dict({k: v.double() for k, v in enc.state_dict().items()})
    hr = h.double().requires_grad_()
    x = hr
    for b in ref.blocks:
        y = b.qkv(b.norm1(x)).view(-1, 8, 16)
        q, k, v = y[:, :4], y[:, 4:6].repeat_interleave(2, 1), y[:, 6:].repeat_interleave(2, 1)
        outs = []
        for a, e in zip(ptr, ptr[1:]):
            s = torch.einsum("qhd,khd->hqk", q[a:e], k[a:e]) / 4.0
            s = s.masked_fill(~mask[a:e], float("-inf"))
            p = torch.softmax(s, -1) if mask[a:e].any() else torch.zeros_like(s)
            outs.append(torch.einsum("hqk,khd->qhd", p, v[a:e]).reshape(-1, 64))
        x = x + b.proj(torch.cat(outs))
        y = b.norm2(x)
        x = x + b.down(torch.nn.functional.silu(b.gate(y)) * b.up(y))
    want = torch.autograd.grad(x, [hr] + list(ref.parameters()), dy.double())
    enc = enc.to(DEV)
    hd = h.to(DEV).requires_grad_()
    got = enc(hd, torch.tensor(ptr, dtype=torch.int32, device=DEV), mask.to(DEV))
    grads = torch.autograd.grad(got, [hd] + list(enc.parameters()), dy.to(DEV))
    for a, b in zip((got,) + grads, (x,) + want):
        scale = max(float(b.abs().max()), 1e-3 * float(max(w.abs().max() for w in want)))
        assert float((a.detach().double().cpu() - b.detach()).abs().max()) <= 1e-5 * scale
