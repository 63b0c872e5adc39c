"""The transformer operators' workspace on the GPU: several pieces, graphs, streams."""
import pytest

from tests import test_gpu_linear_ce as lce

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_last_piece_takes_more_slices_than_a_whole_one():
    """Two pieces of the rows (20,736 and 18,176) whose products for dw are cut into 6 and 7 slices, from an empty workspace; the bounds are
    those of every other shape."""
    from tenmo_b200 import TenmoCuda
    from tests import gpu_util as g

    shared, g._handle = g._handle, TenmoCuda(0).require()
    try:
        x, w, b, y = lce.make(38912, 576, 6300, 31, bias=True)
        lce.compare(x, w, b, y)
        x, w, b, y = lce.make(38912, 576, 6300, 32, tied=True)
        lce.compare(x, w, b, y)
        g._handle.close()
    finally:
        g._handle = shared
