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


@pytest.mark.parametrize("size", [(700, 100, 31), (70000, 256, 100)], ids=str)
def test_captured_bias_gradient_survives_growth(size):
    """A bias gradient summed over more than 512 rows (blocks of rows), captured; column sums of other calls grow what the library
    shares before the replay."""
    from tests import gpu_util as g

    x, w, b, y = lce.make(*size, 33, bias=True)
    lce.run(x, w, b, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        got = lce.run(x, w, b, y)
    x2, w2, b2, y2 = lce.make(*size, 34, bias=True)
    for t, new in ((x, x2), (w, w2), (b, b2), (y, y2)):
        t.copy_(new)
    for rows, cols in ((20000, 1 << 15), (600, 1 << 20)):
        wide = torch.ones(rows, cols, device="cuda")
        out = g.empty(cols)
        g.handle().colsum(wide.data_ptr(), rows, cols, cols, out.data_ptr())
        assert bool((out == rows).all())
    graph.replay()
    torch.cuda.synchronize()
    want = lce.reference(x, w, b, y)
    for n in ("loss", "dx", "dw", "db"):
        lce.check(n, got[n], want[n])
    g.handle().check_device_status()


@pytest.mark.parametrize("ls", [0.0, 0.1])
def test_several_pieces_for_the_rows_of_x(ls):
    """Few classes, so that the rows of x and not the logits end a piece (131,072 rows, then 8,928)."""
    x, w, b, y = lce.make(140000, 1000, 60, 35, bias=True)
    lce.compare(x, w, b, y, ls=ls)
    loss = lce.run(x, w, b, y, ls=ls, forward_only=True)["loss"]
    lce.check("loss", loss, lce.reference(x, w, b, y, ls=ls)["loss"])
