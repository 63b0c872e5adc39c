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


def test_replays_beside_eager_calls():
    """A training step of attention and the head, captured, replayed on one stream while the same operators run eagerly on another, with
    nothing that orders the two: both give what they give alone."""
    from tests import gpu_util as g
    from tests import test_gpu_fused_attention as att

    gen = torch.Generator(device="cuda").manual_seed(36)
    a = [att._make(gen, 8, 8, 512, 64) for _ in range(4)]
    b = [att._make(gen, 8, 8, 500, 64) for _ in range(4)]
    head_a, head_b = lce.make(2000, 256, 4000, 37, bias=True), lce.make(2100, 256, 3900, 38, bias=True)
    step = lambda qkv, head: (att.run(*qkv), lce.run(*head))
    want = step(a, head_a), step(b, head_b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()

    def forward_and_backward(qkv, out, stats):
        from tenmo_b200 import make_heads

        q, k, v, go = qkv
        view = lambda t: make_heads(t.data_ptr(), t.stride())
        shape = (*q.shape[:2], k.shape[1], q.shape[2], k.shape[2], q.shape[3])
        h = g.handle()
        h.attention_fwd(shape, view(q), view(k), view(v), view(out["o"]), stats.data_ptr(), 0.125)
        h.attention_bwd(shape, view(q), view(k), view(v), view(out["o"]), stats.data_ptr(), view(go), view(out["dq"]), view(out["dk"]),
                        view(out["dv"]), 0.125)
    fresh = lambda qkv: (dict(zip(("o", "dq", "dk", "dv"), (torch.full_like(t, float("nan")) for t in qkv))), g.empty(*qkv[0].shape[:3], 2))
    out_a, stats_a = fresh(a)
    with torch.cuda.graph(graph, stream=stream):
        forward_and_backward(a, out_a, stats_a)
        head_out = lce.run(*head_a)
    outs = [fresh(b) for _ in range(12)]
    torch.cuda.synchronize()
    eager_heads = []
    for out, stats in outs:
        with torch.cuda.stream(stream):
            graph.replay()
        with torch.cuda.stream(other):
            forward_and_backward(b, out, stats)
            eager_heads.append(lce.run(*head_b))
    torch.cuda.synchronize()
    for name, t in out_a.items():
        assert torch.equal(t, want[0][0][name]), name
    for name, t in head_out.items():
        assert torch.equal(t, want[0][1][name]), name
    for (out, _), head in zip(outs, eager_heads):
        for name, t in out.items():
            assert torch.equal(t, want[1][0][name]), name
        for name, t in head.items():
            assert torch.equal(t, want[1][1][name]), name
    g.handle().check_device_status()


def test_a_stream_destroyed_behind_its_calls():
    """The context is bound to a stream of the caller's, which is destroyed while a long call may still be running on it; the next call, on
    another stream, uses the workspace after it."""
    import ctypes

    from tenmo_b200 import TenmoCuda
    from tests import gpu_util as g
    from tests import test_gpu_layernorm as ln

    runtime = ctypes.CDLL("libcudart.so.12")
    shared, h = g._handle, TenmoCuda(0).require()
    try:
        long, short = ln._inputs(200000, 1024, 39), ln._inputs(100, 1024, 40)

        def call(x, gamma, bias, dy, out):
            M, C = x.shape
            h.layernorm_fwd(x.data_ptr(), C, gamma.data_ptr(), bias.data_ptr(), 1e-5, out["y"].data_ptr(), out["mean"].data_ptr(), out["rstd"].data_ptr(), M, C)
            h.layernorm_bwd(x.data_ptr(), C, dy.data_ptr(), gamma.data_ptr(), out["mean"].data_ptr(), out["rstd"].data_ptr(), out["dx"].data_ptr(),
                            out["dgamma"].data_ptr(), out["dbias"].data_ptr(), M, C)

        def room(x, *_):
            M, C = x.shape
            return dict(y=g.empty(M, C), dx=g.empty(M, C), dgamma=g.empty(C), dbias=g.empty(C), mean=g.empty(M), rstd=g.empty(M))
        want = []
        for inputs in (long, short):
            want.append(room(*inputs))
            h.set_stream(torch.cuda.current_stream().cuda_stream)
            call(*inputs, want[-1])
        torch.cuda.synchronize()
        for _ in range(3):
            got = [room(*inputs) for inputs in (long, short)]
            torch.cuda.synchronize()
            stream = ctypes.c_void_p()
            assert runtime.cudaStreamCreateWithFlags(ctypes.byref(stream), 1) == 0
            h.set_stream(stream.value)
            call(*long, got[0])
            assert runtime.cudaStreamDestroy(stream) == 0
            h.set_stream(None)
            call(*short, got[1])
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                for name in a:
                    assert torch.equal(a[name], b[name]), name
        h.close()
    finally:
        g._handle = shared
