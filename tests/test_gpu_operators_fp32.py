"""The strict-fp32 switch on attention and linear cross-entropy, at sizes that otherwise run on tensor cores."""
import numpy as np
import pytest

from tests import attention_reference as ar
from tests import test_gpu_fused_attention as att
from tests import test_gpu_linear_ce as lce

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture()
def strict():
    from tenmo_b200 import ALGO_AUTO, ALGO_SIMT_FP32
    from tests import gpu_util as g

    g.handle().operators_set_algo(ALGO_SIMT_FP32)
    yield
    g.handle().operators_set_algo(ALGO_AUTO)


@pytest.mark.parametrize("D", [40, 64, 128])
def test_attention(strict, D):
    """A key and a value of 2^30 in their tile, which the row does not see: 24 bits of the others are kept, where a scale per tile of 64 or 128
    would leave none."""
    gen = torch.Generator(device="cuda").manual_seed(D)
    q, go = (att._make(gen, 2, 4, 300, D) for _ in range(2))
    k, v = (att._make(gen, 2, 2, 310, D) for _ in range(2))
    att.compare(q, k, v, go, causal=True, k_lengths=att.ints([310, 129]))
    want = ar.reference(q, k, v, scale=D ** -0.5, causal=True)["o"]
    for t in (k, v):
        t[:, :, -1] = 2.0 ** 30
    got = att.run(q, k, v, causal=True)["o"]
    ar.check("o", got[:, :, :-1], (want[0][:, :, :-1], want[1][:, :, :-1]))


@pytest.mark.parametrize("tied", [False, True], ids=["linear", "tied"])
def test_linear_cross_entropy(strict, tied):
    x, w, b, y = lce.make(700, 300, 2000, 42, tied=tied, bias=True)
    lce.compare(x, w, b, y, ls=0.1)


def test_the_switch_of_the_host_mirror():
    """set_gemm_algo('simt') holds for Attention and LinearCrossEntropyLoss."""
    import tenmo_b200.tensor as T
    from tenmo_b200.attention import Attention
    from tenmo_b200.crossentropy import LinearCrossEntropyLoss
    from tenmo_b200 import ALGO_AUTO, ALGO_SIMT_FP32

    rng = np.random.default_rng(43)
    q, k, v = (T.Tensor.from_numpy(rng.standard_normal((2, 4, 300, 64)).astype(np.float32)) for _ in range(3))
    x, w, b, y = lce.make(700, 300, 2000, 44)
    X, W, Y = T.Tensor.from_numpy(x.cpu().numpy()), T.Tensor.from_numpy(w.cpu().numpy()), T.Tensor.labels(y.cpu().numpy())
    both = lambda: (Attention()(q, k, v).numpy(), LinearCrossEntropyLoss()(X, W, Y).numpy())
    before, h = T._gemm_algo, T.handle()
    try:
        results = []
        for name, operators in (("auto", ALGO_AUTO), ("simt", ALGO_SIMT_FP32), ("3xtf32", ALGO_AUTO)):
            T.set_gemm_algo(name)
            results.append(both())
            assert T.handle() is h and h._operators_algo == operators
    finally:
        T._gemm_algo = before
    fast, strict, again = results
    assert all(np.array_equal(a, b) for a, b in zip(fast, again))
    assert not np.array_equal(fast[0], strict[0])
    dev = lambda t: torch.from_numpy(np.ascontiguousarray(t.numpy())).cuda()
    ar.check("o", torch.from_numpy(strict[0]).cuda(), ar.reference(dev(q), dev(k), dev(v), scale=0.125)["o"])
    lce.check("loss", torch.from_numpy(strict[1]).cuda().reshape(()), lce.reference(x, w, None, y)["loss"])


@pytest.mark.parametrize("shape", [(385494, 1, 88), (400000, 10, 10), (100000, 16, 30), (3001, 40, 300), (300, 1, 160000), (400, 2, 60000), (300, 50000, 3),
                                   (300, 3, 2049), (300, 2049, 66), (2049, 100, 99), (300, 2048, 70)], ids=str)
@pytest.mark.parametrize("tied", [False, True], ids=["linear", "tied"])
def test_long_contractions_are_not_one_chain(shape, tied):
    """Products below the tensor cores' sizes with a long contraction.  A slice is a chain of at most L = max(512, K / 511) (or K up to 2048) terms, and
    at most 512 of them are added: (L + 512) u of the sum of the terms' sizes, in place of the (64 + K / 32) u that reference() allows."""
    N, D, V = shape
    x, w, b, y = lce.make(*shape, 45, tied=tied, bias=True)
    x = x + 3
    got = lce.run(x, w, b, y)
    want = lce.reference(x, w, b, y)
    chain = lambda K: K if K <= 2048 else max(512, K // 511 + 1) + 512
    xs = torch.where((y != lce.IGN)[:, None], x.double(), 0.0)
    z = xs @ w.double() + b.double()
    dz = torch.softmax(z, 1)
    dz = (dz - torch.zeros_like(z).scatter_(1, y.clamp(min=0)[:, None], 1.0)).abs() * (y != lce.IGN)[:, None] / int((y != lce.IGN).sum())
    for name, K, size, allowed in (("dx", V, dz @ w.double().abs().t(), 64 + V / 32), ("dw", N, xs.abs().t() @ dz, 64 + N / 32)):
        value, bound = want[name]
        lce.check(name, got[name], (value, bound + (chain(K) - allowed) * lce.U * size))
    for name in ("loss", "db"):
        lce.check(name, got[name], want[name])
