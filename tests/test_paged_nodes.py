"""Refusals of the engine's nodes over a KV cache in pages that need no GPU."""
import pytest

from node_check import pyvai


@pytest.mark.parametrize("kind", ["PagedAppendNode", "PagedAttentionNode"])
def test_pages_are_fp32_or_fp16(kind):
    """Any other dtype (2 is that of a tensor without one) would be taken for another element size than the pools have."""
    pv = pyvai()

    class Net(pv.NeuralNet):
        def __init__(self):
            super().__init__()
            self.node = getattr(pv.nodes, kind)(4, 64)

    node = Net().node
    for dtype in (pv.Dtype.Q4, pv.Dtype(2), pv.Dtype(7)):
        with pytest.raises(ValueError, match="F32 or F16"):
            node.set_pages(256, 256, 256, 256, 256, 1, 1, 16, 1, dtype)
    for dtype in (pv.Dtype.F32, pv.Dtype.F16):
        node.set_pages(256, 256, 256, 256, 256, 1, 1, 16, 1, dtype)
