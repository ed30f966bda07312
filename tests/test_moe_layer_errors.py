"""The example layer passes on what the library refuses (a stand-in for it, no GPU)."""
import os
import sys

import pytest

import mxfp4hip as M

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


class Library:
    """Every call succeeds but the one named."""

    def __init__(self, refused):
        self.refused = refused

    def __getattr__(self, name):
        def call(*args):
            if name == "mx_alloc":
                args[2]._obj.value = 4096
            if name == "mx_last_error":
                return b"refused"
            return M.MX_EINVAL if name == self.refused else M.MX_OK
        return call


@pytest.mark.parametrize("refused", ["mx_fmt_quantize", "mx_mxfp4_quantize"])
def test_refused_weights_end_the_layer(monkeypatch, refused):
    import moe_layer
    monkeypatch.setattr(M, "load", lambda: Library(refused))
    dev = M.Device(0)
    with pytest.raises(M.MxError, match="refused"):
        moe_layer.Layer(dev, 64, 32, 2, 1)
