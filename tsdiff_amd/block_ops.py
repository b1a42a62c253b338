"""Differentiable operators of an attention block over ragged graphs: layer norm, the gated linear layer and attention
inside graphs, beside the dense and graph-shaped operators of train_ops.  Their autograd nodes (csrc/block_autograd.cpp)
call the C ABI: tsd_layer_norm_*, tsd_gated_linear_*, tsd_graph_attention_*.

float32, bfloat16 and float16 CUDA tensors; one call's tensors share their type and device.  Sums and statistics are
fp32 and an output is rounded once.  What a bfloat16 or float16 call computes on the way to a matrix product is rounded to that
type for it: the softmax weights, and in a backward pass their gradients and those of the two projections of the gated layer.
Such a product is then about 1.4 times as far from the exact one as its rounded output alone would be; small calls (a gated layer
of up to 2^18 such values, attention in graphs of 32 rows on average whose rows fit 16-byte loads) go without that error.  float16
takes these values times a power of two, so gradients may be as small or as large as float16 itself holds.  Work is queued on the current stream of the tensors' device; nothing waits for the
GPU, no state is kept between calls, and the results of a call are the same bits every time.  Calls may be captured into
a graph; to capture a backward pass, give the captured forward leaves of its own (x.detach().requires_grad_()), since
autograd ties a leaf's accumulation to the stream that used it first.  First derivatives in reverse mode only: a second
derivative and a forward-mode tangent (also under no_grad) raise.
"""
import os

from . import _lib

_EXT_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_block_ops.so")
_ext = None


def _load():
    global _ext
    if _ext is None:
        import torch  # noqa: F401  (the extension's own libraries)
        _lib.load()
        if not os.path.exists(_EXT_PATH):
            raise _lib.TsdError(f"{_EXT_PATH} not found: the extension is not built (run `python __graft_entry__.py` or "
                                "`make -C tsdiff_amd/csrc`).")
        from . import _block_ops
        _ext = _block_ops
    return _ext


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) (var + eps)^-1/2 weight + bias over the last dimension (at most 8192) of x [..., dim]; weight and bias
    [dim] or None."""
    return (_ext or _load()).layer_norm(x, weight, bias, eps)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, act="swish"):
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up): the gated half of a feed-forward block (torch.nn.Linear's weights,
    [out, in]; biases [out] or None).  act: "swish", "ssp" (shifted softplus), "ReLU" or "Softplus".  The backward computes
    both projections again."""
    return (_ext or _load()).gated_linear(x, w_gate, w_up, b_gate, b_up, act)


def graph_attention(q, k, v, graph_ptr, key_ptr=None, key_mask=None, scale=None):
    """Attention inside the graphs of a ragged batch: q [Nq, heads, dim], k and v [Nk, key heads, dim] -> [Nq, heads, dim].

    Queries graph_ptr[g] .. graph_ptr[g+1] attend to keys key_ptr[g] .. key_ptr[g+1] (key_ptr None: the same nodes); both
    offset lists are non-decreasing device tensors [graphs + 1] whose values are not checked.  Every heads / key heads
    query heads share a key head.  key_mask [Nk] (bool or uint8): the keys that may be attended to.  A query without such a
    key gives zeros.  Any strides with a contiguous last dimension are read as they are; dim <= 128; scale defaults to
    dim ** -0.5.  A readout is one query a graph; long key lists with few queries are split over the chip.  The backward
    computes the probabilities again."""
    return (_ext or _load()).graph_attention(q, k, v, graph_ptr, key_ptr, key_mask, scale)
