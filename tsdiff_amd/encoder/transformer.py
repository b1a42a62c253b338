"""A global encoder over the nodes of ragged graphs, beside the message-passing ones of this package: pre-norm blocks of
attention inside each graph and a gated feed-forward layer (block_ops), with the dense layers of train_ops.  Differentiable.
No counterpart in the reference."""
import torch
from torch import nn

from .. import _lib
from ..block_ops import gated_linear, graph_attention, layer_norm
from ..train_ops import linear


class GraphTransformerBlock(nn.Module):
    def __init__(self, hidden_dim, num_heads, num_kv_heads=None, ff_dim=None):
        super().__init__()
        num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        if hidden_dim % num_heads or num_heads % num_kv_heads:
            raise ValueError(f"hidden_dim {hidden_dim}, {num_heads} heads, {num_kv_heads} key heads")
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, hidden_dim // num_heads
        ff_dim = 2 * hidden_dim if ff_dim is None else ff_dim
        self.norm1, self.norm2 = nn.LayerNorm(hidden_dim), nn.LayerNorm(hidden_dim)
        self.qkv = nn.Linear(hidden_dim, (num_heads + 2 * num_kv_heads) * self.head_dim)
        self.proj = nn.Linear(hidden_dim, hidden_dim)
        self.gate, self.up = nn.Linear(hidden_dim, ff_dim), nn.Linear(hidden_dim, ff_dim)
        self.down = nn.Linear(ff_dim, hidden_dim)

    def forward(self, h, graph_ptr, key_mask=None):
        x = layer_norm(h, self.norm1.weight, self.norm1.bias, self.norm1.eps)
        qkv = linear(x, self.qkv.weight, self.qkv.bias)
        qkv = qkv.view(h.shape[0], self.num_heads + 2 * self.num_kv_heads, self.head_dim)
        q, k, v = qkv.split((self.num_heads, self.num_kv_heads, self.num_kv_heads), dim=1)
        x = graph_attention(q, k, v, graph_ptr, key_mask=key_mask)
        h = h + linear(x.reshape(h.shape), self.proj.weight, self.proj.bias)
        x = layer_norm(h, self.norm2.weight, self.norm2.bias, self.norm2.eps)
        x = gated_linear(x, self.gate.weight, self.up.weight, self.gate.bias, self.up.bias)
        return h + linear(x, self.down.weight, self.down.bias)


class GraphTransformerEncoder(nn.Module):
    """forward(h [N, hidden_dim] float32, graph_ptr [graphs + 1]) -> [N, hidden_dim]; key_mask [N]: the nodes that others
    may attend to"""

    def __init__(self, hidden_dim, num_blocks=3, num_heads=8, num_kv_heads=None, ff_dim=None):
        super().__init__()
        self.hidden_dim = hidden_dim
        self.blocks = nn.ModuleList(GraphTransformerBlock(hidden_dim, num_heads, num_kv_heads, ff_dim)
                                    for _ in range(num_blocks))

    def forward(self, h, graph_ptr, key_mask=None):
        if h.device.type != "cuda":
            raise _lib.TsdError("tsdiff_amd runs on the GPU only (no CPU fallback)")
        if h.dim() != 2 or h.shape[1] != self.hidden_dim or h.dtype != torch.float32:
            raise ValueError(f"h is {h.dtype} {tuple(h.shape)}, float32 [nodes, {self.hidden_dim}] expected")
        with torch.cuda.device(h.device):  # the dense layers go to the current device
            for block in self.blocks:
                h = block(h, graph_ptr, key_mask)
        return h
