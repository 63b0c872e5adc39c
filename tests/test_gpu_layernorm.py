"""Layer norm forward and backward against the formula in 64 bits.

Bounds, with u = 2^-24.  A sum of C terms is 8 additions per thread, at most 5 + 5 levels of a tree and a rounding per term, so it
is off by at most 24 u of the sum of absolute values (wide rows, walked by 1024 threads: C / 1024 additions instead of 8).
  mean   e_m = n u mean|x|
  xhat   the difference inherits e_m, rstd is off by (n + 4) u relative and by the shift e_m^2 of the variance:
         e_h = (n + 8) u (|xhat| + 1) + 2 rstd e_m
  y      e_h |gamma| + 2 u (|xhat gamma| + |bias|)
  dx     rstd (g - mean g - xhat mean(g xhat)): every sum as above, e_h into its terms
  dgamma sum over rows: M terms added at most sequentially (M u of the absolute sum) plus e_h |dy|
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
EPS = 1e-5


def _reference(x, gamma, bias, dy, eps=EPS):
    x, gamma, bias, dy = (t.double() for t in (x, gamma, bias, dy))
    M, C = x.shape
    n = max(24, C / 1024 + 16)
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    h = (x - mean) * rstd
    e_h = (n + 8) * U * (h.abs() + 1) + 2 * rstd * n * U * x.abs().mean(1, keepdim=True)
    y = h * gamma + bias
    e_y = e_h * gamma.abs() + 2 * U * ((h * gamma).abs() + bias.abs())
    g = dy * gamma
    a, b = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = rstd * (g - a - h * b)
    e_a = (n + 2) * U * g.abs().mean(1, keepdim=True)
    e_b = (n + 2) * U * (g * h).abs().mean(1, keepdim=True) + (g.abs() * e_h).mean(1, keepdim=True)
    e_dx = rstd * (e_a + e_h * b.abs() + h.abs() * e_b) + (n + 8) * U * rstd * (g.abs() + a.abs() + (h * b).abs())
    dgamma, e_dg = (dy * h).sum(0), (dy.abs() * e_h).sum(0) + (M + 8) * U * (dy * h).abs().sum(0)
    dbias, e_db = dy.sum(0), (M + 8) * U * dy.abs().sum(0)
    return dict(y=(y, e_y), dx=(dx, e_dx), dgamma=(dgamma, e_dg), dbias=(dbias, e_db), mean=(mean[:, 0], (n * U * x.abs().mean(1))))


def _check(name, got, want):
    ref, bound = want
    off = (got.double() - ref).abs()
    assert bool(torch.all(off <= bound + 1e-37)), f"{name}: off by up to {float((off / (bound + 1e-37)).max()):.2f} of its bound"


def _inputs(M, C, seed, pad=0, shift=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    x = rnd(M, C + pad) * 2 + shift
    return x[:, :C], 1 + 0.3 * rnd(C), 0.3 * rnd(C), rnd(M, C)


def _run(x, gamma, bias, dy, beta=0.0, dx0=None, dg0=None, db0=None):
    from tests import gpu_util as g

    h = g.handle()
    M, C = x.shape
    y, mean, rstd = torch.full((M, C), float("nan"), device="cuda"), g.empty(M), g.empty(M)
    h.layernorm_fwd(x.data_ptr(), x.stride(0) if M else C, gamma.data_ptr(), bias.data_ptr(), EPS, y.data_ptr(), mean.data_ptr(),
                    rstd.data_ptr(), M, C)
    dx = dx0 if dx0 is not None else torch.full((M, C), float("nan"), device="cuda")
    dg = dg0 if dg0 is not None else torch.full((C,), float("nan"), device="cuda")
    db = db0 if db0 is not None else torch.full((C,), float("nan"), device="cuda")
    h.layernorm_bwd(x.data_ptr(), x.stride(0) if M else C, dy.data_ptr(), gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                    dx.data_ptr(), dg.data_ptr(), db.data_ptr(), M, C, beta=beta)
    return dict(y=y, dx=dx, dgamma=dg, dbias=db, mean=mean)


# one column, below / at / above a warp's 256 columns, odd columns (scalar loads), the widest register row, walked rows
@pytest.mark.parametrize("mc", [(1, 1), (3, 2), (5, 31), (64, 128), (7, 255), (9, 256), (9, 257), (300, 768), (2000, 260), (33, 1023),
                                (17, 4096), (5, 8191), (4, 8192), (3, 8200), (2, 20001)], ids=str)
def test_forward_and_backward(mc):
    M, C = mc
    x, gamma, bias, dy = _inputs(M, C, M * 31 + C)
    got, ref = _run(x, gamma, bias, dy), _reference(x, gamma, bias, dy)
    for name in ref:
        _check(name, got[name], ref[name])


@pytest.mark.parametrize("pad", [1, 4, 12])
def test_rows_inside_a_wider_matrix(pad):
    x, gamma, bias, dy = _inputs(50, 320, 5, pad=pad)
    got, ref = _run(x, gamma, bias, dy), _reference(x, gamma, bias, dy)
    for name in ref:
        _check(name, got[name], ref[name])


def test_unaligned_pointers():
    x, gamma, bias, dy = _inputs(40, 512, 6)
    off = lambda t: torch.cat([torch.zeros(1, device="cuda"), t.reshape(-1)])[1:].reshape(t.shape)
    x, gamma, bias, dy = (off(t) for t in (x, gamma, bias, dy))
    assert x.data_ptr() % 16
    got, ref = _run(x, gamma, bias, dy), _reference(x, gamma, bias, dy)
    for name in ref:
        _check(name, got[name], ref[name])


@pytest.mark.parametrize("C", [40, 300, 9000])
def test_rows_far_apart(C):
    """Rows of x so far apart that their offsets pass 2^31."""
    x, gamma, bias, dy = _inputs(300, C, 9)
    stride = (1 << 31) // 299 + 77
    far = torch.as_strided(torch.empty(300 * stride, device="cuda"), (300, C), (stride, 1))
    far.copy_(x)
    a, b = _run(far, gamma, bias, dy), _reference(far, gamma, bias, dy)
    for name in a:
        _check(name, a[name], b[name])


def test_large_mean_does_not_cancel():
    """mean 1e4, deviation 2: E[x^2] - mean^2 would lose everything in 32 bits."""
    x, gamma, bias, dy = _inputs(64, 1000, 7, shift=1e4)
    got, ref = _run(x, gamma, bias, dy), _reference(x, gamma, bias, dy)
    for name in ref:
        _check(name, got[name], ref[name])


def test_constant_rows_and_nan_rows():
    x, gamma, bias, dy = _inputs(6, 300, 8)
    x = x.clone()
    x[2] = 7.5
    x[4, 17] = float("nan")
    got = _run(x, gamma, bias, dy)
    assert torch.equal(got["y"][2], bias)  # xhat is exactly zero
    assert bool(got["y"][4].isnan().all()) and bool(got["dx"][4].isnan().all())
    rest = [0, 1, 3, 5]
    ref = _reference(x[rest], gamma, bias, dy[rest])
    _check("y", got["y"][rest], ref["y"])
    _check("dx", got["dx"][rest], ref["dx"])


@pytest.mark.parametrize("mc", [(50, 100), (40, 768), (3, 9000)], ids=str)
def test_accumulates_and_repeats(mc):
    M, C = mc
    x, gamma, bias, dy = _inputs(M, C, 9)
    first = _run(x, gamma, bias, dy)
    again = _run(x, gamma, bias, dy)
    for name in first:
        assert torch.equal(first[name], again[name])
    added = _run(x, gamma, bias, dy, beta=1.0, dx0=first["dx"].clone(), dg0=first["dgamma"].clone(), db0=first["dbias"].clone())
    for name in ("dx", "dgamma", "dbias"):
        assert torch.equal(added[name], 2 * first[name])


def test_dx_may_be_dy_and_sums_are_optional():
    from tests import gpu_util as g

    x, gamma, bias, dy = _inputs(30, 640, 10)
    ref = _run(x, gamma, bias, dy)
    h = g.handle()
    mean, rstd, d = ref["mean"], g.empty(30), dy.clone()
    y = g.empty(30, 640)
    h.layernorm_fwd(x.data_ptr(), 640, gamma.data_ptr(), bias.data_ptr(), EPS, y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), 30, 640)
    h.layernorm_bwd(x.data_ptr(), 640, d.data_ptr(), gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(), d.data_ptr(), 0, 0, 30, 640)
    assert torch.equal(d, ref["dx"])
    h.layernorm_fwd(x.data_ptr(), 640, gamma.data_ptr(), bias.data_ptr(), EPS, y.data_ptr(), 0, 0, 30, 640)
    assert torch.equal(y, ref["y"])


def test_no_rows():
    got = _run(torch.empty(0, 64, device="cuda"), torch.ones(64, device="cuda"), torch.zeros(64, device="cuda"),
               torch.empty(0, 64, device="cuda"))
    assert float(got["dgamma"].abs().max()) == 0 and float(got["dbias"].abs().max()) == 0


def test_refusals():
    from tenmo_b200 import TenmoError
    from tests import gpu_util as g

    h = g.handle()
    t = g.empty(64)
    p = t.data_ptr()
    for args in ((p, 3, p, p, EPS, p, p, p, 4, 4), (p, 4, p, p, -1.0, p, p, p, 4, 4), (p, 4, p, p, float("nan"), p, p, p, 4, 4),
                 (p, 0, p, p, EPS, p, p, p, 4, 0), (p, 4, p, p, EPS, p, p, p, -1, 4), (None, 4, p, p, EPS, p, p, p, 4, 4)):
        with pytest.raises(TenmoError):
            h.layernorm_fwd(*args)
    with pytest.raises(TenmoError):
        h.layernorm_bwd(p, 4, p, p, p, p, p, p, p, 4, 4, beta=0.5)
    with pytest.raises(TenmoError):
        h.layernorm_bwd(p, 4, None, p, p, p, p, p, p, 4, 4)


def test_captured_graph_replays_with_new_inputs():
    from tests import gpu_util as g

    x, gamma, bias, dy = _inputs(100, 384, 11)
    out = _run(x, gamma, bias, dy)  # sizes the workspace
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        out = _run(x, gamma, bias, dy)
    x.copy_(_inputs(100, 384, 12)[0])
    dy.copy_(_inputs(100, 384, 12)[3])
    graph.replay()
    ref = _reference(x, gamma, bias, dy)
    for name in ref:
        _check(name, out[name], ref[name])
    g.handle()


def test_layer_in_the_autograd_graph():
    import tenmo_b200.tensor as T
    from tenmo_b200.net import LayerNorm

    x, gamma, bias, dy = _inputs(24, 96, 13)
    X = T.Tensor.from_numpy(x.cpu().numpy().reshape(4, 6, 96), requires_grad=True)
    ln = LayerNorm(96, eps=EPS)
    ln.weight, ln.bias = (T.Tensor.from_numpy(t.cpu().numpy(), requires_grad=True) for t in (gamma, bias))
    out = ln(X)
    out.backward(T.Tensor.from_numpy(dy.cpu().numpy().reshape(4, 6, 96)))
    ref = _reference(x, gamma, bias, dy)
    back = lambda t: torch.from_numpy(t.numpy()).cuda()
    _check("y", back(out).reshape(24, 96), ref["y"])
    _check("dx", back(X.grad()).reshape(24, 96), ref["dx"])
    _check("dgamma", back(ln.weight.grad()), ref["dgamma"])
    _check("dbias", back(ln.bias.grad()), ref["dbias"])
    with pytest.raises(RuntimeError):
        ln(T.Tensor.zeros(3, 95))
