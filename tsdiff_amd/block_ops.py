"""Differentiable operators of an attention block over ragged graphs: layer norm, the gated linear layer and attention
inside graphs, as torch.autograd.Function nodes over the C ABI (tsd_layer_norm_*, tsd_gated_linear_*,
tsd_graph_attention_*), beside the dense and graph-shaped operators of train_ops.

float32, bfloat16 and float16 CUDA tensors; one call's tensors share their type and device.  Sums and statistics are
fp32 and an output is rounded once.  Work is queued on the current stream of the tensors' device; nothing waits for the
GPU, no state is kept between calls, and the results of a call are the same bits every time.  Calls may be captured into
a graph; to capture a backward pass, give the captured forward leaves of its own (x.detach().requires_grad_()), since
autograd ties a leaf's accumulation to the stream that used it first.  First derivatives only.
"""
import contextlib
import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACT = {"swish": 0, "ssp": 1, "ReLU": 2, "Softplus": 3}  # tsd_act_fwd's kinds


def _same(name, first, *others):
    """type and device of a call's tensors"""
    if first.device.type != "cuda":
        raise _lib.TsdError("tsdiff_amd runs on the GPU only (no CPU fallback)")
    if first.dtype not in _DTYPE:
        raise ValueError(f"{name}: float32, bfloat16 or float16 expected, got {first.dtype}")
    for t in others:
        if t is not None and (t.dtype != first.dtype or t.device != first.device):
            raise ValueError(f"{name}: {t.dtype} on {t.device} beside {first.dtype} on {first.device}")


def _on(t):
    """the tensors' device as the current one"""
    return contextlib.nullcontext() if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _p(t):
    return None if t is None else t.data_ptr()


def _rows(t):
    """t as [rows, features] with contiguous features, copied only where its strides ask for it"""
    t = t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t
    if t.shape[0] > 1 and t.stride(0) < t.shape[1] or t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _dense(t):
    return None if t is None else t.contiguous()


def _grad_on(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- layer norm -----------------------------------------------------------------------------------------------
def _norm_fwd(x, weight, bias, eps, keep):
    rows, dim = x.shape
    y = torch.empty(rows, dim, dtype=x.dtype, device=x.device)
    stats = torch.empty(2, rows, dtype=torch.float32, device=x.device) if keep else None
    mean = _p(stats)
    check(_lib.load().tsd_layer_norm_fwd(_DTYPE[x.dtype], rows, dim, _p(x), _ld(x), _p(weight), _p(bias), eps, _p(y),
                                         mean, mean + 4 * rows if keep else None, _stream()))
    return y, stats


class LayerNorm(torch.autograd.Function):
    """y = (x - mean) (var + eps)^-1/2 weight + bias over the rows of x [rows, dim]"""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        with _on(x):
            y, stats = _norm_fwd(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        dy = _rows(dy)
        rows, dim = x.shape
        lib = _lib.load()
        need = ctx.needs_input_grad
        with _on(x):
            dx = torch.empty(rows, dim, dtype=x.dtype, device=x.device) if need[0] else None
            dw = torch.empty(dim, dtype=x.dtype, device=x.device) if need[1] else None
            db = torch.empty(dim, dtype=x.dtype, device=x.device) if need[2] else None
            n = lib.tsd_layer_norm_scratch_floats(rows, dim) if need[1] or need[2] else 0
            scratch = torch.empty(n, dtype=torch.float32, device=x.device)
            mean = stats.data_ptr()
            check(lib.tsd_layer_norm_bwd(_DTYPE[x.dtype], rows, dim, _p(x), _ld(x), _p(weight), _p(dy), _ld(dy), mean,
                                         mean + 4 * rows, _p(dx), _p(dw), _p(db), _p(scratch), n, _stream()))
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last dimension (at most 8192) of x [..., dim]; weight and bias [dim] or None."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: x has shape {tuple(x.shape)}")
    for n, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"layer_norm: {n} has shape {tuple(t.shape)}, [{x.shape[-1]}] expected")
    _same("layer_norm", x, weight, bias)
    rows, weight, bias = _rows(x), _dense(weight), _dense(bias)
    if _grad_on(x, weight, bias):
        y = LayerNorm.apply(rows, weight, bias, float(eps))
    else:
        with _on(x):
            y, _ = _norm_fwd(rows, weight, bias, float(eps), False)
    return y if x.dim() == 2 else y.view(x.shape)


# ---- gated linear layer ---------------------------------------------------------------------------------------
def _gated_fwd(x, wg, wu, bg, bu, act):
    rows, fin = x.shape
    h = torch.empty(rows, wg.shape[0], dtype=x.dtype, device=x.device)
    check(_lib.load().tsd_gated_linear_fwd(_DTYPE[x.dtype], act, rows, fin, wg.shape[0], _p(x), _ld(x), _p(wg), _p(wu),
                                           _p(bg), _p(bu), _p(h), _stream()))
    return h


class GatedLinear(torch.autograd.Function):
    """h = act(x Wg^T + bg) * (x Wu^T + bu); the backward computes both projections again"""

    @staticmethod
    def forward(ctx, x, wg, wu, bg, bu, act):
        with _on(x):
            h = _gated_fwd(x, wg, wu, bg, bu, act)
        ctx.save_for_backward(x, wg, wu, bg, bu)
        ctx.act = act
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, wg, wu, bg, bu = ctx.saved_tensors
        dh = _rows(dh)
        (rows, fin), out = x.shape, wg.shape[0]
        lib = _lib.load()
        with _on(x):
            def grad(k, *shape):
                return torch.empty(*shape, dtype=x.dtype, device=x.device) if ctx.needs_input_grad[k] else None

            dx, dwg, dwu, dbg, dbu = grad(0, rows, fin), grad(1, out, fin), grad(2, out, fin), grad(3, out), grad(4, out)
            n = lib.tsd_gated_linear_scratch_floats(_DTYPE[x.dtype], rows, fin, out)
            scratch = torch.empty(n, dtype=torch.float32, device=x.device)
            check(lib.tsd_gated_linear_bwd(_DTYPE[x.dtype], ctx.act, rows, fin, out, _p(x), _ld(x), _p(wg), _p(wu), _p(bg),
                                           _p(bu), _p(dh), _ld(dh), _p(dx), _p(dwg), _p(dwu), _p(dbg), _p(dbu), _p(scratch),
                                           n, _stream()))
        return dx, dwg, dwu, dbg, dbu, None


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, act="swish"):
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up): the gated half of a feed-forward block (torch.nn.Linear's weights,
    [out, in]; biases [out] or None).  act: "swish", "ssp" (shifted softplus), "ReLU" or "Softplus"."""
    if act not in _ACT:
        raise NotImplementedError(f"gated_linear: activation {act!r}")
    if w_gate.dim() != 2 or w_gate.shape != w_up.shape or 0 in w_gate.shape or x.dim() < 1 or x.shape[-1] != w_gate.shape[1]:
        raise ValueError(f"gated_linear: x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)}")
    for n, t in (("b_gate", b_gate), ("b_up", b_up)):
        if t is not None and tuple(t.shape) != (w_gate.shape[0],):
            raise ValueError(f"gated_linear: {n} has shape {tuple(t.shape)}, [{w_gate.shape[0]}] expected")
    _same("gated_linear", x, w_gate, w_up, b_gate, b_up)
    rows, wg, wu, bg, bu = _rows(x), _dense(w_gate), _dense(w_up), _dense(b_gate), _dense(b_up)
    if _grad_on(x, wg, wu, bg, bu):
        h = GatedLinear.apply(rows, wg, wu, bg, bu, _ACT[act])
    else:
        with _on(x):
            h = _gated_fwd(rows, wg, wu, bg, bu, _ACT[act])
    return h if x.dim() == 2 else h.view(*x.shape[:-1], w_gate.shape[0])


# ---- attention ------------------------------------------------------------------------------------------------
def _heads(t):
    return t if t.shape[2] == 1 or t.stride(2) == 1 else t.contiguous()


def _attention_args(q, k, v, q_ptr, k_ptr, mask, scale):
    return _lib.Attention(_DTYPE[q.dtype], q_ptr.shape[0] - 1, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2],
                          scale, _p(q), _p(k), _p(v), q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0),
                          v.stride(1), _p(q_ptr), _p(k_ptr), _p(mask))


def _attention_fwd(q, k, v, q_ptr, k_ptr, mask, scale, keep):
    lib = _lib.load()
    a = _attention_args(q, k, v, q_ptr, k_ptr, mask, scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if keep else None
    n = lib.tsd_graph_attention_scratch_floats(C.byref(a), 0)
    scratch = torch.empty(n, dtype=torch.float32, device=q.device) if n else None
    check(lib.tsd_graph_attention_fwd(C.byref(a), _p(out), _p(lse), _p(scratch), n, _stream()))
    return out, lse


class GraphAttention(torch.autograd.Function):
    """softmax(scale q k^T) v inside each graph; the backward computes the probabilities again"""

    @staticmethod
    def forward(ctx, q, k, v, q_ptr, k_ptr, mask, scale):
        with _on(q):
            out, lse = _attention_fwd(q, k, v, q_ptr, k_ptr, mask, scale, True)
        ctx.save_for_backward(q, k, v, q_ptr, k_ptr, mask, out, lse)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, q_ptr, k_ptr, mask, out, lse = ctx.saved_tensors
        dout = _heads(dout)
        lib = _lib.load()
        with _on(q):
            dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
            a = _attention_args(q, k, v, q_ptr, k_ptr, mask, ctx.scale)
            n = lib.tsd_graph_attention_scratch_floats(C.byref(a), 1)
            scratch = torch.empty(n, dtype=torch.float32, device=q.device)
            check(lib.tsd_graph_attention_bwd(C.byref(a), _p(out), _p(lse), _p(dout), dout.stride(0), dout.stride(1), _p(dq),
                                              _p(dk), _p(dv), _p(scratch), n, _stream()))
        return dq, dk, dv, None, None, None, None


def graph_attention(q, k, v, graph_ptr, key_ptr=None, key_mask=None, scale=None):
    """Attention inside the graphs of a ragged batch: q [Nq, heads, dim], k and v [Nk, key heads, dim] -> [Nq, heads, dim].

    Queries graph_ptr[g] .. graph_ptr[g+1] attend to keys key_ptr[g] .. key_ptr[g+1] (key_ptr None: the same nodes); both
    offset lists are non-decreasing device tensors [graphs + 1] whose values are not checked.  Every heads / key heads
    query heads share a key head.  key_mask [Nk] (bool or uint8): the keys that may be attended to.  A query without such a
    key gives zeros.  Any strides with a contiguous last dimension are read as they are; dim <= 128; scale defaults to
    dim ** -0.5.  A readout is one query a graph; long key lists with few queries are split over the chip."""
    for n, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 3:
            raise ValueError(f"graph_attention: {n} has shape {tuple(t.shape)}, [nodes, heads, dim] expected")
    if k.shape != v.shape or q.shape[2] != k.shape[2] or 0 in q.shape[1:] or 0 in k.shape[1:] or q.shape[1] % k.shape[1]:
        raise ValueError(f"graph_attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    _same("graph_attention", q, k, v)
    if key_ptr is None:
        if k.shape[0] != q.shape[0]:
            raise ValueError(f"graph_attention: {q.shape[0]} queries and {k.shape[0]} keys need a key_ptr")
        key_ptr = graph_ptr
    for n, t in (("graph_ptr", graph_ptr), ("key_ptr", key_ptr)):
        if t.dim() != 1 or t.shape[0] < 1 or t.dtype not in (torch.int32, torch.int64) or t.device != q.device:
            raise ValueError(f"graph_attention: {n} is {t.dtype} {tuple(t.shape)} on {t.device}, integer offsets [graphs + 1] "
                             f"on {q.device} expected")
    if graph_ptr.shape != key_ptr.shape:
        raise ValueError(f"graph_attention: {graph_ptr.shape[0] - 1} graphs of queries, {key_ptr.shape[0] - 1} of keys")
    if key_mask is not None:
        if tuple(key_mask.shape) != (k.shape[0],) or key_mask.dtype not in (torch.bool, torch.uint8) or \
                key_mask.device != q.device:
            raise ValueError(f"graph_attention: key_mask is {key_mask.dtype} {tuple(key_mask.shape)} on {key_mask.device}, "
                             f"bool [{k.shape[0]}] on {q.device} expected")
        key_mask = key_mask.contiguous()
    with _on(q):
        q_ptr, k_ptr = (t.to(torch.int32).contiguous() for t in (graph_ptr, key_ptr))
    scale = float(q.shape[2]) ** -0.5 if scale is None else float(scale)
    q, k, v = _heads(q), _heads(k), _heads(v)
    if _grad_on(q, k, v):
        return GraphAttention.apply(q, k, v, q_ptr, k_ptr, key_mask, scale)
    with _on(q):
        return _attention_fwd(q, k, v, q_ptr, k_ptr, key_mask, scale, False)[0]
