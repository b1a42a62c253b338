"""Mirrors of the secondary (legacy dual-encoder) encoders of the reference `models/encoder/`, and a global encoder of this
package's own (transformer)."""
from .gin import GINEConv, GINEncoder  # noqa: F401
from .edge import GaussianSmearingEdgeEncoder  # noqa: F401
from .transformer import GraphTransformerBlock, GraphTransformerEncoder  # noqa: F401
