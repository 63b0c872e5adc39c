"""The widest rows that layer norm takes, 2^30 - 1 columns: column counts and their doubles at the end of 32 bits."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

C = 2 ** 30 - 1


def test_backward_of_the_widest_row():
    """One row, so dbias is dy and dgamma is dy * xhat: xhat is off by two roundings and the product by one (3 u, u = 2^-24, and their
    products).  The sums of dx have 2^20 terms a thread; dy is zero but in one column in 2^20, which leaves at most a term of dy * gamma for
    each addition that rounds: 1,024 of them, 2^10 u of sums below 2^10."""
    from tenmo_b200 import TenmoCuda, TenmoError

    torch.cuda.empty_cache()
    h = TenmoCuda(0).require()
    h.set_stream(torch.cuda.current_stream().cuda_stream)
    gen = torch.Generator(device="cuda").manual_seed(41)
    x = torch.rand(C, device="cuda", generator=gen)
    dy = torch.zeros(C, device="cuda")
    dy[5::1 << 20] = 0.5
    dy[-1] = 0.25
    gamma = torch.ones(C, device="cuda")
    mean, rstd = torch.full((1,), 0.5, device="cuda"), torch.full((1,), 3.0, device="cuda")
    dx, dgamma, dbias = (torch.full((C + 64,), float("nan"), device="cuda") for _ in range(3))
    args = lambda cols: (x.data_ptr(), cols, dy.data_ptr(), gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), dgamma.data_ptr(),
                         dbias.data_ptr(), 1, cols)
    h.layernorm_bwd(*args(C))
    h.synchronize()
    for t in (dx, dgamma, dbias):
        assert bool(t[C:].isnan().all())
    assert torch.equal(dbias[:C], dy)
    at = dy.nonzero()[:, 0]
    xh = (x[at].double() - 0.5) * 3
    want = dy[at].double() * xh
    assert bool(((dgamma[at].double() - want).abs() <= 3.01 * 2.0 ** -24 * want.abs()).all())
    dgamma[at] = 0
    assert float(dgamma[:C].abs().max()) == 0
    a, b = dy[at].double().sum() / C, want.sum() / C
    for c0 in range(0, C, 1 << 28):
        part = slice(c0, min(C, c0 + (1 << 28)))
        d = 3 * (dy[part].double() - a - (x[part].double() - 0.5) * 3 * b)
        assert float((dx[part].double() - d).abs().max()) <= 3 * (2.0 ** 10 * 2.0 ** -24 * 2.0 ** 10 * 2 / C + 8 * 2.0 ** -24)
    with pytest.raises(TenmoError):
        h.layernorm_bwd(*args(C + 1))
    h.close()
