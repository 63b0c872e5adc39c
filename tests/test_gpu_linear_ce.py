"""Cross-entropy of a linear layer's logits, loss and gradients, against 64 bits.

Bounds (u = 2^-24).  A logit is a sum of D products, off by e_z = (D + 64) u (|x| |w| + |b|) and, for operands far below the
largest of their tile, 2^-37 D max|x| max|w| of it.  A probability is off by a factor 1 + r, r = 2 max_v e_z + c u with
c = 128 + V / 256 (the length of a thread's sum).  Then
  loss   max_v e_z + e_z,y + c u (|lse - z_y| + 1) per row, u of the sum once
  dz     |u_n| (r p + 4 u (p + 1[y] + ls / V)), and 2^-36 of the largest |dz| of the call where tiles are scaled
  dx     sum_v e_dz |w| + (64 + V / 32) u sum_v |dz w|;  dw, db alike over the rows
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
IGN = -100


def reference(x, w, b, y, ls=0.0, reduction=0, upstream=None, ignore=IGN):
    N, D = x.shape
    V = w.shape[1]
    keep = y.long() != ignore
    x = torch.where(keep[:, None], x.double(), 0.0)
    w = w.double()
    z = x @ w + (b.double() if b is not None else 0)
    e_z = (D + 64) * U * (x.abs() @ w.abs() + (b.double().abs() if b is not None else 0)) + 2.0 ** -37 * D * x.abs().max() * w.abs().max()
    c = 128 + V / 256
    lse = torch.logsumexp(z, 1, keepdim=True)
    p = (z - lse).exp()
    idx = torch.where(keep, y.long(), 0)[:, None]
    zy = z.gather(1, idx)
    row = ((1 - ls) * (lse - zy) + ls * (lse - z.mean(1, keepdim=True)))[:, 0]
    e_row = 2 * e_z.amax(1) + c * U * ((lse - zy).abs()[:, 0] + (lse - z.mean(1, keepdim=True)).abs()[:, 0] + 1)
    row, e_row = torch.where(keep, row, 0.0), torch.where(keep, e_row, 0.0)
    count = max(1, int(keep.sum()))
    if reduction == 2:
        loss, e_loss = row, e_row
    else:
        div = count if reduction == 0 else 1
        loss, e_loss = row.sum() / div, e_row.sum() / div + 4 * U * row.sum().abs() / div
    un = torch.ones(N, dtype=torch.float64, device=x.device) if upstream is None else upstream.double().reshape(-1).expand(N)
    un = torch.where(keep, un / (count if reduction == 0 else 1), 0.0)[:, None]
    hot = torch.zeros_like(z).scatter_(1, idx, 1.0)
    dz = un * (p - (1 - ls) * hot - ls / V)
    r = 2 * e_z.amax(1, keepdim=True) + c * U
    e_dz = un.abs() * (r * p + 4 * U * (p + hot + ls / V)) + 2.0 ** -36 * dz.abs().max() * keep[:, None]
    cn = 64 + N / 32
    out = dict(loss=(loss, e_loss), dx=(dz @ w.T, e_dz @ w.abs().T + (64 + V / 32) * U * (dz.abs() @ w.abs().T)),
               dw=(x.T @ dz, x.abs().T @ e_dz + cn * U * (x.abs().T @ dz.abs()) + 2.0 ** -37 * x.abs().max() * dz.abs().sum(0, keepdim=True)))
    if b is not None:
        out["db"] = (dz.sum(0), e_dz.sum(0) + cn * U * dz.abs().sum(0))
    return out


def check(name, got, want):
    ref, bound = want
    off = (got.double() - ref).abs()
    bad = ~(off <= bound + 1e-36)
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} beyond their bounds, worst "
                                 f"{float((off / (bound + 1e-36)).nan_to_num(nan=1e30).max()):.3g} times")


def make(N, D, V, seed, tied=False, bias=False, dtype=torch.int64, ignored=0.2, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    x = scale * rnd(N, D)
    w = rnd(V, D).t() if tied else rnd(D, V)
    w = w / D ** 0.5
    y = torch.randint(0, V, (N,), device="cuda", generator=gen)
    y[torch.rand(N, device="cuda", generator=gen) < ignored] = IGN
    return x, w, 0.5 * rnd(V) if bias else None, y.to(dtype)


def run(x, w, b, y, ls=0.0, reduction=0, upstream=None, ignore=IGN, forward_only=False):
    from tenmo_b200 import make_mat
    from tests import gpu_util as g

    h = g.handle()
    (N, D), V = x.shape, w.shape[1]
    loss = torch.full((N,) if reduction == 2 else (1,), float("nan"), device="cuda")
    valid = torch.full((1,), -7, dtype=torch.int32, device="cuda")
    args = (make_mat(x.data_ptr(), (N, D), x.stride()), make_mat(w.data_ptr(), (D, V), w.stride()), b.data_ptr() if b is not None else 0,
            y.data_ptr(), y.dtype == torch.int64, N, D, V, ignore, ls, reduction, loss.data_ptr(), valid.data_ptr())
    out = dict(loss=loss if reduction == 2 else loss[0], valid=valid)
    if forward_only:
        h.linear_ce_fwd(*args)
        return out
    nan = float("nan")
    dx = torch.full((N, D), nan, device="cuda")
    dw = torch.full((V, D), nan, device="cuda").t() if w.stride(0) == 1 and w.stride(1) != 1 else torch.full((D, V), nan, device="cuda")
    db = torch.full((V,), nan, device="cuda") if b is not None else None
    h.linear_ce_fwd_bwd(*args, upstream.data_ptr() if upstream is not None else 0, dx.data_ptr(), dw.data_ptr(),
                        db.data_ptr() if b is not None else 0)
    out.update(dx=dx, dw=dw)
    if b is not None:
        out["db"] = db
    return out


def compare(x, w, b, y, **kw):
    from tests import gpu_util as g

    got = run(x, w, b, y, **kw)
    g.handle().check_device_status()
    kw.pop("forward_only", None)
    want = reference(x, w, b, y, **kw)
    for name in got:
        if name != "valid":
            check(name, got[name], want[name])
    assert int(got["valid"]) == int((y.long() != kw.get("ignore", IGN)).sum())
    return got


# up to 16 rows (256 in small products): the few-row kernels; from 1e8 flop a product on (2e8 up to 256 rows): tensor cores; else the strict-fp32 GEMM
SHAPES = [(1, 1, 1), (1, 16, 10), (3, 5, 2), (7, 33, 1003), (13, 260, 4100), (32, 64, 130), (33, 128, 640), (64, 128, 1000), (64, 512, 4000), (130, 70, 129), (257, 64, 515), (300, 200, 4099), (515, 768, 2001),
          (16, 700, 20001), (17, 702, 20001), (16, 90, 90001), (256, 33, 700), (594, 40, 2465), (300, 40, 129), (700, 100, 31)]


@pytest.mark.parametrize("tied", [False, True], ids=["linear", "tied"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_64_bits(shape, tied):
    N, D, V = shape
    x, w, b, y = make(N, D, V, N + D + V, tied=tied, bias=not tied, ignored=0.0 if N < 4 else 0.2)
    compare(x, w, b, y)
    loss = run(x, w, b, y, forward_only=True)["loss"]
    check("loss", loss, reference(x, w, b, y)["loss"])


@pytest.mark.parametrize("size", [(30, 40, 201), (60, 40, 200), (100, 40, 200), (300, 40, 200), (300, 256, 3000)], ids=str)
@pytest.mark.parametrize("reduction", [0, 1, 2])
def test_reductions_smoothing_upstream_and_label_types(size, reduction):
    N, D, V = size
    for tied, ls, dtype in ((False, 0.0, torch.int32), (True, 0.1, torch.int64)):
        x, w, b, y = make(N, D, V, 3 + reduction, tied=tied, bias=True, dtype=dtype)
        up = torch.randn(N if reduction == 2 else 1, device="cuda")
        compare(x, w, b, y, ls=ls, reduction=reduction, upstream=up)


@pytest.mark.parametrize("size", [(30, 40, 201), (60, 40, 200), (100, 40, 200), (300, 40, 200), (300, 256, 3000)], ids=str)
def test_ignored_rows_may_hold_anything(size):
    x, w, b, y = make(*size, 4, bias=True, ignored=0.4)
    x[y == IGN] = float("nan")
    x[(y == IGN).nonzero()[0]] = float("inf")
    got = compare(x, w, b, y)
    assert float(got["dx"][y == IGN].abs().max()) == 0


@pytest.mark.parametrize("size", [(30, 20, 50), (100, 20, 50), (300, 20, 50), (200, 256, 2000)], ids=str)
def test_every_row_ignored(size):
    x, w, b, y = make(*size, 5, bias=True, ignored=2.0)
    got = run(x, w, b, y)
    assert float(got["loss"]) == 0 and int(got["valid"]) == 0
    for n in ("dx", "dw", "db"):
        assert float(got[n].abs().max()) == 0


@pytest.mark.parametrize("size", [(40, 32, 100), (100, 32, 100), (300, 32, 100), (256, 256, 2048)], ids=str)
def test_large_logits(size):
    x, w, b, y = make(*size, 6, scale=40.0)
    compare(x, w, b, y)


@pytest.mark.parametrize("size", [(40, 32, 100), (100, 32, 100), (300, 32, 100), (256, 256, 2048)], ids=str)
def test_rows_and_classes_of_very_different_size(size):
    N, D, V = size
    x, w, b, y = make(N, D, V, 7, tied=True)
    x = x * torch.exp2(-torch.arange(N, device="cuda") % 24)[:, None].float()
    w = w * torch.exp2(-torch.arange(V, device="cuda") % 24)[None, :].float()
    w = w.t().contiguous().t()
    compare(x, w, b, y)


def test_strided_x():
    x, w, b, y = make(50, 60, 300, 8)
    wide = torch.full((50, 2, 70), float("nan"), device="cuda")
    wide[:, 1, 5:65] = x
    compare(wide[:, 1, 5:65], w, b, y)
    compare(x.t().contiguous().t(), w, b, y)


@pytest.mark.parametrize("size", [(40, 32, 100), (100, 32, 100), (300, 32, 100), (256, 256, 2048)], ids=str)
def test_bad_label_sets_the_status_and_contributes_nothing(size):
    from tenmo_b200 import TenmoError
    from tests import gpu_util as g

    N, D, V = size
    x, w, b, y = make(N, D, V, 9, ignored=0.0)
    y[3], y[5] = V, -1
    got = run(x, w, b, y)
    with pytest.raises(TenmoError):
        g.handle().check_device_status()
    assert float(got["dx"][[3, 5]].abs().max()) == 0 and int(got["valid"]) == N


def test_several_pieces_give_what_one_gives():
    """Enough classes that the rows are taken in more than one piece."""
    x, w, b, y = make(3000, 24, 60000, 10, tied=True, bias=True)
    got = compare(x, w, b, y)
    again = run(x, w, b, y)
    for n in ("loss", "dx", "dw", "db"):
        assert torch.equal(got[n], again[n])


@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -math.inf], ids=["lowest", "-inf"])
@pytest.mark.parametrize("tied", [False, True], ids=["linear", "tied"])
@pytest.mark.parametrize("size", [(30, 20, 500), (100, 20, 500), (300, 20, 500), (200, 256, 2000)], ids=str)
def test_classes_masked_through_the_bias(size, tied, low):
    """Classes whose bias is the type's lowest value or -inf: the same loss and gradients as without them, and none of their own."""
    N, D, V = size
    x, w, b, y = make(N, D, V, 21, tied=tied, bias=True)
    keep = torch.rand(V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(22)) < 0.5
    keep[64:192] = False  # whole groups of columns too
    keep[:5] = True
    at = keep.nonzero()[:, 0]
    y = torch.where(y == IGN, y, at[y.clamp(min=0) % len(at)])
    got = run(x, w, torch.where(keep, b, low), y)
    place = torch.full((V,), -1, device="cuda", dtype=torch.int64)
    place[at] = torch.arange(len(at), device="cuda")
    y_kept = torch.where(y == IGN, y, place[y.clamp(min=0)])
    want = reference(x, w[:, at], b[at], y_kept)
    check("loss", got["loss"], want["loss"])
    check("dx", got["dx"], want["dx"])
    check("dw", got["dw"][:, at], want["dw"])
    check("db", got["db"][at], want["db"])
    assert float(got["dw"][:, ~keep].abs().max()) == 0 and float(got["db"][~keep].abs().max()) == 0


@pytest.mark.parametrize("tied", [False, True], ids=["linear", "tied"])
@pytest.mark.parametrize("size", [(7, 36, 200), (100, 36, 200), (300, 36, 200), (257, 256, 2000)], ids=str)
def test_pointers_that_are_not_aligned(size, tied):
    """Every buffer begins 4 bytes behind a 16-byte boundary, and nothing is written outside."""
    from tenmo_b200 import make_mat
    from tests import gpu_util as g

    N, D, V = size
    x, w, b, y = make(N, D, V, 23, tied=tied, bias=True)
    ref = run(x, w, b, y)

    def odd(t):
        buf = torch.full((t.numel() + 8,), float("nan"), device="cuda")
        return buf, torch.as_strided(buf, t.shape, t.stride(), 1)
    put = lambda t: odd(t)[1].copy_(t)
    xo, wo, bo = put(x), put(w), put(b)
    bufs = {n: odd(ref[n]) for n in ("dx", "dw", "db")}
    loss, valid = torch.empty(1, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    h = g.handle()
    h.linear_ce_fwd_bwd(make_mat(xo.data_ptr(), (N, D), xo.stride()), make_mat(wo.data_ptr(), (D, V), wo.stride()), bo.data_ptr(), y.data_ptr(), True,
                        N, D, V, IGN, 0.0, 0, loss.data_ptr(), valid.data_ptr(), 0, *(bufs[n][1].data_ptr() for n in ("dx", "dw", "db")))
    h.check_device_status()
    want = reference(x, w, b, y)
    check("loss", loss[0], want["loss"])
    for n, (buf, t) in bufs.items():
        check(n, t, want[n])
        assert bool(buf[0].isnan()) and bool(buf[1 + t.numel():].isnan().all()), n


@pytest.mark.parametrize("size", [(20, 32, 100), (300, 32, 100), (300, 256, 2000)], ids=str)
def test_rows_far_apart(size):
    """Rows of x so far apart that their offsets pass 2^31."""
    N, D, V = size
    x, w, b, y = make(N, D, V, 24)
    stride = (1 << 31) // (N - 1) + 77
    far = torch.as_strided(torch.empty(N * stride, device="cuda"), (N, D), (stride, 1))
    far.copy_(x)
    compare(far, w, b, y)


@pytest.mark.parametrize("N", [8, 40])
def test_more_than_2_31_weights(N):
    """A tied weight whose entries are counted beyond 2^31, on both sides of the choice of kernels."""
    D, V = 2048, 1049000
    gen = torch.Generator(device="cuda").manual_seed(25)
    x = torch.randn(N, D, device="cuda", generator=gen)
    w = torch.randn(V, D, device="cuda", generator=gen) / D ** 0.5
    y = torch.randint(V - 50, V, (N,), device="cuda", generator=gen)
    y[0] = 3
    got = run(x, w.t(), None, y)
    z = torch.cat([x.double() @ w[v0:v0 + (1 << 16)].double().t() for v0 in range(0, V, 1 << 16)], 1)
    lse = z.logsumexp(1)
    loss = (lse - z[torch.arange(N, device="cuda"), y]).mean()
    # a logit is off by at most (D + 64) u sum |x w|, some 2^-15; the rest follows as in reference()
    assert abs(float(got["loss"]) - float(loss)) <= 2.0 ** -15
    dz = (z - lse[:, None]).exp()
    dz[torch.arange(N, device="cuda"), y] -= 1
    dz /= N
    near = torch.cat([torch.arange(100, device="cuda"), torch.arange(V - 100, V, device="cuda")])
    dw = dz[:, near].t() @ x.double()
    off = (got["dw"].t()[near].double() - dw).abs()
    assert bool((off <= 2.0 ** -14 * (dz[:, near].abs().t() @ x.abs().double()) + 2.0 ** -36).all())
    dx = sum(dz[:, v0:v0 + (1 << 16)] @ w[v0:v0 + (1 << 16)].double() for v0 in range(0, V, 1 << 16))
    size = sum(dz[:, v0:v0 + (1 << 16)].abs() @ w[v0:v0 + (1 << 16)].abs().double() for v0 in range(0, V, 1 << 16))
    assert bool(((got["dx"].double() - dx).abs() <= 2.0 ** -14 * size).all())


def test_no_rows():
    x, w, b, y = make(0, 8, 20, 11, bias=True)
    got = run(x, w, b, y)
    assert float(got["loss"]) == 0 and float(got["dw"].abs().max()) == 0 and float(got["db"].abs().max()) == 0


def test_refusals():
    from tenmo_b200 import TenmoError, make_mat
    from tests import gpu_util as g

    h = g.handle()
    t = g.empty(4096)
    p = t.data_ptr()
    x, w = make_mat(p, (4, 8), (8, 1)), make_mat(p, (8, 16), (16, 1))
    y = torch.zeros(4, dtype=torch.int64, device="cuda").data_ptr()

    def refused(status, x=x, w=w, y=y, N=4, D=8, V=16, ls=0.0, red=0, loss=p):
        with pytest.raises(TenmoError) as e:
            h.linear_ce_fwd(x, w, 0, y, True, N, D, V, IGN, ls, red, loss, p)
        assert e.value.status == status
    refused(-1, N=-1)
    refused(-1, D=0)
    refused(-1, V=0)
    refused(-1, ls=1.5)
    refused(-1, ls=float("nan"))
    refused(-1, red=3)
    refused(-1, loss=None)
    refused(-1, y=None)
    refused(-1, x=make_mat(0, (4, 8), (8, 1)))
    refused(-1, x=make_mat(p, (4, 8), (-8, 1)))
    refused(-1, x=make_mat(p, (2, 4, 8), (32, 8, 1)))
    refused(-3, w=make_mat(p, (8, 16), (32, 2)))
    refused(-1, w=make_mat(p, (8, 16), (-16, 1)))
    refused(-1, w=make_mat(p, (8, 16), (1, -8)))
    with pytest.raises(TenmoError):
        h.linear_ce_fwd_bwd(x, w, 0, y, True, 4, 8, 16, IGN, 0.0, 0, p, p, 0, p, None)
    with pytest.raises(TenmoError):  # a bias gradient without a bias
        h.linear_ce_fwd_bwd(x, w, 0, y, True, 4, 8, 16, IGN, 0.0, 0, p, p, 0, p, p, p)


@pytest.mark.parametrize("size", [(40, 32, 100), (100, 32, 100), (300, 32, 100), (300, 256, 2100)], ids=str)
def test_captured_graph_replays_with_new_inputs(size):
    x, w, b, y = make(*size, 12, tied=True)
    run(x, w, b, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        got = run(x, w, b, y)
    x2, w2, _, y2 = make(*size, 13, tied=True)
    x.copy_(x2), w.copy_(w2), y.copy_(y2)
    graph.replay()
    torch.cuda.synchronize()
    want = reference(x, w, b, y)
    for n in ("loss", "dx", "dw"):
        check(n, got[n], want[n])


@pytest.mark.parametrize("tied", [False, True], ids=["linear", "tied"])
def test_loss_in_the_autograd_graph(tied):
    import tenmo_b200.tensor as T
    from tenmo_b200.crossentropy import LinearCrossEntropyLoss

    x, w, b, y = make(40, 24, 90, 14, bias=True)
    X, B = (T.Tensor.from_numpy(t.cpu().numpy(), requires_grad=True) for t in (x, b))
    W = T.Tensor.from_numpy((w.t() if tied else w).contiguous().cpu().numpy(), requires_grad=True)
    loss = LinearCrossEntropyLoss()(X, W.transpose() if tied else W, T.Tensor.labels(y.cpu().numpy()), B)
    loss.backward(2.0)
    want = reference(x, w, b, y, upstream=torch.full((1,), 2.0, device="cuda"))
    back = lambda t: torch.from_numpy(np.ascontiguousarray(t.numpy())).cuda()
    check("loss", back(loss).reshape(()), want["loss"])
    check("dx", back(X.grad()), want["dx"])
    check("dw", back(W.grad()).t() if tied else back(W.grad()), want["dw"])
    check("db", back(B.grad()), want["db"])
    with pytest.raises(RuntimeError):
        LinearCrossEntropyLoss()(X, T.Tensor.zeros(23, 90), T.Tensor.labels(y.cpu().numpy()))
