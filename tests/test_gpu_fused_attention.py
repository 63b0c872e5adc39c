"""Attention forward and backward against 64 bits: head layouts, masks, empty rows, odd sizes, strides."""
import math

import numpy as np
import pytest

from tests import attention_reference as ar

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

NAN = float("nan")


def _make(gen, B, H, S, D, layout="bhsd"):
    if layout == "bshd":
        return torch.randn(B, S, H, D, device="cuda", generator=gen).transpose(1, 2)
    return torch.randn(B, H, S, D, device="cuda", generator=gen)


def run(q, k, v, go=None, scale=None, causal=False, q_lengths=None, k_lengths=None, beta=0.0, into=None):
    from tenmo_b200 import make_heads
    from tests import gpu_util as g

    h = g.handle()
    B, H, Sq, D = q.shape
    shape = (B, H, k.shape[1], Sq, k.shape[2], D)
    scale = 1 / math.sqrt(D) if scale is None else scale
    view = lambda t: make_heads(t.data_ptr(), t.stride())
    new = lambda t: torch.full_like(t, NAN)
    o, stats = new(q), torch.full((B, H, Sq, 2), NAN, device="cuda")
    mask = dict(causal=causal, q_lengths=q_lengths.data_ptr() if q_lengths is not None else 0,
                k_lengths=k_lengths.data_ptr() if k_lengths is not None else 0)
    h.attention_fwd(shape, view(q), view(k), view(v), view(o), stats.data_ptr(), scale, **mask)
    out = dict(o=o)
    if go is not None:
        dq, dk, dv = into if into is not None else (new(q), new(k), new(v))
        h.attention_bwd(shape, view(q), view(k), view(v), view(o), stats.data_ptr(), view(go), view(dq), view(dk), view(dv), scale,
                        beta=beta, **mask)
        out.update(dq=dq, dk=dk, dv=dv)
    h.check_device_status()
    return out


def compare(q, k, v, go=None, **kw):
    got = run(q, k, v, go, **kw)
    kw.setdefault("scale", 1 / math.sqrt(q.shape[-1]))
    want = ar.reference(q, k, v, go, **kw)
    for name in want:
        ar.check(name, got[name], want[name])
    return got


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# batch, heads, kv_heads, q_len, k_len, dim: single rows and keys, lengths around 32 / 64 / 128, shared heads, odd dims
# (the tensor-core kernels take over from some 2500 rows x 128 keys on in the forward pass, from 64 rows or keys on in the backward pass)
SHAPES = [(1, 1, 1, 1, 1, 1), (2, 3, 3, 1, 7, 16), (6, 1, 1, 40, 40, 16), (2, 4, 2, 33, 65, 20), (1, 2, 1, 127, 129, 64),
          (1, 2, 2, 128, 128, 64), (2, 2, 1, 130, 300, 64), (1, 8, 2, 257, 255, 128), (2, 3, 1, 64, 64, 37), (1, 2, 2, 300, 70, 97),
          (1, 4, 4, 640, 640, 32), (3, 6, 3, 200, 1, 8), (1, 2, 1, 2, 900, 127),
          (4, 8, 8, 129, 127, 64), (4, 8, 2, 100, 257, 50), (3, 8, 4, 131, 260, 100), (2, 40, 10, 17, 129, 64), (40, 8, 4, 16, 5, 24),
          (20, 16, 8, 33, 31, 66)]


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_64_bits(shape, causal):
    B, H, Hkv, Sq, Sk, D = shape
    gen = torch.Generator(device="cuda").manual_seed(sum(shape) + causal)
    layout = "bshd" if D % 2 else "bhsd"
    q, go = (_make(gen, B, H, Sq, D, layout) for _ in range(2))
    k, v = (_make(gen, B, Hkv, Sk, D, layout) for _ in range(2))
    compare(q, k, v, go, causal=causal)


@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
def test_padded_batch_ignores_what_padding_holds(causal, layout):
    """Lengths 0, 1, inside a tile, on a tile's border and full; NaN and infinities behind them."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    B, H, Hkv, Sq, Sk, D = 6, 4, 2, 200, 300, 64
    q, go = (_make(gen, B, H, Sq, D, layout) for _ in range(2))
    k, v = (_make(gen, B, Hkv, Sk, D, layout) for _ in range(2))
    ql, kl = [200, 0, 1, 130, 128, 64], [300, 300, 77, 0, 128, 1]
    for b in range(B):
        q[b, :, ql[b]:] = NAN
        go[b, :, ql[b]:] = math.inf
        k[b, :, kl[b]:] = NAN
        v[b, :, kl[b]:] = -math.inf
    got = compare(q, k, v, go, causal=causal, q_lengths=ints(ql), k_lengths=ints(kl))
    for b in range(B):
        assert float(got["o"][b, :, ql[b]:].abs().sum()) == 0 and float(got["dq"][b, :, ql[b]:].abs().sum()) == 0
        assert float(got["dk"][b, :, kl[b]:].abs().sum()) == 0 and float(got["dv"][b, :, kl[b]:].abs().sum()) == 0


def test_lengths_outside_the_range_count_as_the_nearest_bound():
    gen = torch.Generator(device="cuda").manual_seed(4)
    q, k, v, go = (_make(gen, 3, 2, 50, 32) for _ in range(4))
    a = run(q, k, v, go, k_lengths=ints([-5, 1000, 50]), q_lengths=ints([50, 2 ** 31 - 1, -1]))
    b = run(q, k, v, go, k_lengths=ints([0, 50, 50]), q_lengths=ints([50, 50, 0]))
    for name in a:
        assert torch.equal(a[name], b[name])


def test_causal_with_more_rows_than_keys_leaves_rows_empty():
    gen = torch.Generator(device="cuda").manual_seed(5)
    for D, H in ((24, 2), (64, 16), (100, 16)):
        q, go = (_make(gen, 1, H, 300, D) for _ in range(2))
        k, v = (_make(gen, 1, H, 100, D) for _ in range(2))
        got = compare(q, k, v, go, causal=True)
        assert float(got["o"][:, :, :200].abs().max()) == 0 and float(got["dq"][:, :, :200].abs().max()) == 0


@pytest.mark.parametrize("q_len,k_len", [(5, 0), (0, 5), (300, 0), (0, 300)])
def test_no_keys_or_no_rows(q_len, k_len):
    gen = torch.Generator(device="cuda").manual_seed(6)
    q, go = (_make(gen, 2, 2, q_len, 16) for _ in range(2))
    k, v = (_make(gen, 2, 2, k_len, 16) for _ in range(2))
    got = run(q, k, v, go)
    for t in got.values():
        assert float(t.abs().sum()) == 0  # also: written, not left as NaN


@pytest.mark.parametrize("length", [7, 300])
def test_an_empty_batch(length):
    gen = torch.Generator(device="cuda").manual_seed(28)
    got = run(*(_make(gen, 0, 2, length, 16) for _ in range(4)))
    assert got["dk"].shape == (0, 2, length, 16)


@pytest.mark.parametrize("size", [40, 300])
def test_large_and_small_scores(size):
    """Scores of several hundred (a softmax that picks one key) and of almost zero (uniform), and the scale's sign."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    q, k, v, go = (_make(gen, 1, 2 if size < 100 else 4, size, 64) for _ in range(4))
    compare(30 * q, 30 * k, v, go)
    compare(1e-4 * q, 1e-4 * k, 1e3 * v, 1e-3 * go)
    compare(q, k, v, go, scale=-0.3)
    compare(q, k, v, go, scale=0.0)


@pytest.mark.parametrize("size", [40, 300])
def test_rows_of_very_different_size(size):
    """Keys, values, rows and upstream gradients whose sizes differ by 2^20 from row to row."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    q, k, v, go = (_make(gen, 1, 2 if size < 100 else 4, size, 64) for _ in range(4))
    spread = lambda t: t * torch.exp2(torch.randint(-20, 1, t.shape[:3], device="cuda", generator=gen).float())[..., None]
    compare(spread(q), spread(k), spread(v), spread(go))


@pytest.mark.parametrize("size", [20, 300])
def test_nan_and_infinity_stay_in_their_rows(size):
    gen = torch.Generator(device="cuda").manual_seed(9)
    q, k, v = (_make(gen, 1, 2 if size < 100 else 4, size, 64) for _ in range(3))
    q[0, 0, 3, 5] = NAN
    q[0, 1, 4, 5] = math.inf
    got = run(q, k, v)["o"]
    assert bool(got[0, 0, 3].isnan().all()) and bool(got[0, 1, 4].isnan().all())
    clean = torch.nan_to_num(q, nan=0.0, posinf=0.0)
    want = ar.reference(clean, k, v, scale=1 / 8)["o"]
    for h, bad in [(0, 3), (1, 4)] + [(h, None) for h in range(2, q.shape[1])]:
        rows = [i for i in range(size) if i != bad]
        ar.check("o", got[:, h, rows], (want[0][:, h, rows], want[1][:, h, rows]))


@pytest.mark.parametrize("Sq,Sk,H,D", [(50, 20, 2, 24), (60, 30, 2, 64), (300, 100, 16, 64), (300, 100, 16, 100), (320, 192, 16, 32)])
def test_rows_that_see_nothing_may_hold_anything(Sq, Sk, H, D):
    """Causal with more rows than keys: what the first Sq - Sk rows hold reaches nothing, and their own results are zeros."""
    gen = torch.Generator(device="cuda").manual_seed(19)
    q, go = (_make(gen, 2, H, Sq, D) for _ in range(2))
    k, v = (_make(gen, 2, H, Sk, D) for _ in range(2))
    q[:, :, :Sq - Sk] = NAN
    go[:, :, :Sq - Sk, ::2] = math.inf
    got = compare(q, k, v, go, causal=True)
    assert float(got["o"][:, :, :Sq - Sk].abs().max()) == 0 and float(got["dq"][:, :, :Sq - Sk].abs().max()) == 0


@pytest.mark.parametrize("size,H", [(50, 2), (200, 16)])
def test_keys_that_no_row_sees_may_hold_anything(size, H):
    """Causal with rows cut off by q_lengths: the keys behind the last row's are zeros in dk and dv and reach nothing."""
    gen = torch.Generator(device="cuda").manual_seed(20)
    q, k, v, go = (_make(gen, 2, H, size, 64) for _ in range(4))
    rows = [size - 21, 7]
    for b, n in enumerate(rows):
        k[b, :, n:] = NAN
        v[b, :, n:] = math.inf
        q[b, :, n:] = math.inf
        go[b, :, n:] = NAN
    got = compare(q, k, v, go, causal=True, q_lengths=ints(rows))
    for b, n in enumerate(rows):
        assert float(got["dk"][b, :, n:].abs().max()) == 0 and float(got["dv"][b, :, n:].abs().max()) == 0


@pytest.mark.parametrize("size", [40, 300])
@pytest.mark.parametrize("big", [300.0, 1e3, 2e3, 4e3, 1e4, 1e5])
def test_scores_beyond_the_whole_numbers(size, big):
    """Scores up to 1e11, whose 32-bit values are further apart than 1: a row whose best key leads by more than the scores' error takes that
    key's v, and everything stays finite."""
    gen = torch.Generator(device="cuda").manual_seed(21)
    q, k, v, go = (_make(gen, 1, 2 if size < 100 else 4, size, 64) for _ in range(4))
    q, k = big * q, big * k
    got = run(q, k, v, go)
    for t in got.values():
        assert bool(t.isfinite().all())
    s = q.double() @ k.double().transpose(-1, -2) / 8
    top = s.topk(2, dim=-1)
    # 2^-17 of the sum of |q k|: (dim + 64) u with room; exp(-60) of the others is below half a step of v's largest entry
    lead = top.values[..., 0] - top.values[..., 1] > 60 + 2.0 ** -16 * (q.abs().double() @ k.abs().double().transpose(-1, -2)).amax(-1) / 8
    assert int(lead.sum()) > size
    want = torch.take_along_dim(v, top.indices[..., :1], 2).double()
    # One term P v / P.  P = hi + lo misses 2^-22, v 2^-23 (or 2^-38 of its tile's largest), the dropped lo lo is at most 2^-10 2^-11; three partial
    # products are added with truncation, 2^-23 each, and the division and its product round, 2 * 2^-24:
    # 2^-22 + 2^-23 + 2^-21 + 3 * 2^-23 + 2^-23 = 1.375 * 2^-20 < 2^-19.
    off = (got["o"].double() - want).abs()
    assert bool((off <= 2.0 ** -19 * want.abs() + 2.0 ** -36 * v.abs().max())[lead].all())


def test_calls_on_two_streams_do_not_share_the_workspace_at_once():
    """A call on another stream right behind a long one: the workspace that both use is waited for."""
    gen = torch.Generator(device="cuda").manual_seed(22)
    a = [_make(gen, 8, 8, 1024, 64) for _ in range(4)]
    b = [_make(gen, 4, 8, 300, 40) for _ in range(4)]
    c = [_make(gen, 2, 4, 1, 40)] + [_make(gen, 2, 4, 3000, 40) for _ in range(2)]
    want = run(*a), run(*b), run(*c)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    from tenmo_b200 import make_heads
    from tests import gpu_util as g

    view = lambda t: make_heads(t.data_ptr(), t.stride())
    for _ in range(3):
        got = []
        for stream, (q, k, v, *go) in zip(streams, (a, b, c)):
            out = dict(o=torch.full_like(q, NAN))
            stats = g.empty(*q.shape[:3], 2)
            shape = (q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3])
            if go:
                out.update(dq=torch.full_like(q, NAN), dk=torch.full_like(k, NAN), dv=torch.full_like(v, NAN))
            got.append((stream, shape, q, k, v, go, out, stats))
        torch.cuda.synchronize()
        for stream, shape, q, k, v, go, out, stats in got:
            with torch.cuda.stream(stream):
                h = g.handle()
                scale = 1 / math.sqrt(q.shape[3])
                h.attention_fwd(shape, view(q), view(k), view(v), view(out["o"]), stats.data_ptr(), scale)
                if go:
                    h.attention_bwd(shape, view(q), view(k), view(v), view(out["o"]), stats.data_ptr(), view(go[0]), view(out["dq"]),
                                    view(out["dk"]), view(out["dv"]), scale)
        torch.cuda.synchronize()
        for (_, _, _, _, _, _, out, _), ref in zip(got, want):
            for name in out:
                assert torch.equal(out[name], ref[name]), name
    g.handle().check_device_status()


@pytest.mark.parametrize("q_len", [1, 20, 130])
def test_offsets_beyond_32_bits(q_len):
    """A cache whose rows lie 65536 numbers apart: offsets pass 2^31 (and, in bytes, 2^32)."""
    from tenmo_b200 import make_heads
    from tests import gpu_util as g

    gen = torch.Generator(device="cuda").manual_seed(23)
    n, stride, D = 36000, 65536, 40
    buf = torch.empty(n * stride, device="cuda")
    at = lambda c: torch.as_strided(buf, (1, 2, n, D), (0, D, stride, 1), c * 2 * D)
    k, v, dk, dv = (at(c) for c in range(4))
    for t in (k, v):
        t.copy_(torch.randn(t.shape, device="cuda", generator=gen))
    for t in (dk, dv):
        t.fill_(NAN)
    q, go = (_make(gen, 1, 4, q_len, D) for _ in range(2))
    o, dq, stats = torch.full_like(q, NAN), torch.full_like(q, NAN), g.empty(1, 4, q_len, 2)
    h = g.handle()
    view = lambda t: make_heads(t.data_ptr(), (n * stride, *t.stride()[1:]))
    shape = (1, 4, 2, q_len, n, D)
    h.attention_fwd(shape, view(q), view(k), view(v), view(o), stats.data_ptr(), 0.3)
    h.attention_bwd(shape, view(q), view(k), view(v), view(o), stats.data_ptr(), view(go), view(dq), view(dk), view(dv), 0.3)
    h.check_device_status()
    want = ar.reference(q, k.contiguous(), v.contiguous(), go, scale=0.3)
    for name, t in dict(o=o, dq=dq, dk=dk, dv=dv).items():
        ar.check(name, t, want[name])


@pytest.mark.parametrize("size", [30, 260])
def test_broadcast_inputs_and_wide_strides(size):
    """k and v shared by the whole batch (stride 0), q inside a wider row, o inside a wider row."""
    from tenmo_b200 import make_heads
    from tests import gpu_util as g

    gen = torch.Generator(device="cuda").manual_seed(10)
    B, H, D = 2, 2, 40
    qkv = torch.randn(B, size, 3 * H * D + 5, device="cuda", generator=gen)
    q = qkv[:, :, 7:7 + H * D].reshape(B, size, H, D)  # a copy when the slice cannot be viewed: take strides instead
    q = torch.as_strided(qkv, (B, H, size, D), (qkv.stride(0), D, qkv.stride(1), 1), 7)
    k, v = (torch.randn(1, H, size, D, device="cuda", generator=gen).expand(B, H, size, D) for _ in range(2))
    buf = torch.full((B, size, H, D + 3), NAN, device="cuda")
    o = torch.as_strided(buf, (B, H, size, D), (buf.stride(0), buf.stride(2), buf.stride(1), 1))
    h = g.handle()
    view = lambda t: make_heads(t.data_ptr(), t.stride())
    h.attention_fwd((B, H, H, size, size, D), view(q), view(k), view(v), view(o), 0, 0.2)
    ar.check("o", o, ar.reference(q, k, v, scale=0.2)["o"])
    assert bool(buf[..., D:].isnan().all())  # nothing written between the rows


@pytest.mark.parametrize("size", [40, 300])
def test_accumulates_and_repeats(size):
    gen = torch.Generator(device="cuda").manual_seed(11)
    q, go = (_make(gen, 2, 4, size, 64) for _ in range(2))
    k, v = (_make(gen, 2, 2, size, 64) for _ in range(2))
    first, again = run(q, k, v, go, causal=True), run(q, k, v, go, causal=True)
    for name in first:
        assert torch.equal(first[name], again[name])
    into = [first[n].clone() for n in ("dq", "dk", "dv")]
    added = run(q, k, v, go, causal=True, beta=1.0, into=into)
    for name in ("dq", "dk", "dv"):
        assert torch.equal(added[name], 2 * first[name])


@pytest.mark.parametrize("D,H,Hkv", [(64, 4, 1), (66, 6, 2), (128, 4, 4), (33, 4, 2)])
def test_accumulates_on_a_padded_batch(D, H, Hkv):
    """beta = 1 where whole tiles take no part (what is there stays), one head or several per key/value head, aligned rows and others."""
    gen = torch.Generator(device="cuda").manual_seed(26)
    q, go = (_make(gen, 4, H, 300, D) for _ in range(2))
    k, v = (_make(gen, 4, Hkv, 280, D) for _ in range(2))
    mask = dict(q_lengths=ints([300, 100, 0, 257]), k_lengths=ints([280, 3, 140, 0]))
    first = run(q, k, v, go, **mask)
    start = [_make(gen, *t.shape) for t in (q, k, v)]
    added = run(q, k, v, go, beta=1.0, into=[t.clone() for t in start], **mask)
    for name, t in zip(("dq", "dk", "dv"), start):
        assert torch.equal(added[name], t + first[name])


@pytest.mark.parametrize("causal", [False, True])
def test_heads_in_groups(causal):
    """So many heads that their tile images (105 MB) are worked on in two groups, of 161 and 160."""
    gen = torch.Generator(device="cuda").manual_seed(27)
    q, k, v, go = (_make(gen, 107, 3, 520, 40) for _ in range(4))
    compare(q, k, v, go, causal=causal)


@pytest.mark.parametrize("size", [24, 200])
def test_gradients_against_differences(size):
    """Central differences of sum(go * o) in 64 bits of the formula, along random directions, against the kernel's gradients."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    q, k, v, go = (_make(gen, 1, 2 if size < 100 else 8, size, 32) for _ in range(4))
    got = run(q, k, v, go, causal=True)
    f = lambda a, b, c: float((ar.reference(a, b, c, scale=1 / math.sqrt(32), causal=True)["o"][0] * go.double()).sum())
    for n, name in enumerate(("dq", "dk", "dv")):
        args = [t.double() for t in (q, k, v)]
        way = torch.randn(args[n].shape, device="cuda", generator=gen).double()
        eps = 1e-5
        hi, lo = list(args), list(args)
        hi[n], lo[n] = args[n] + eps * way, args[n] - eps * way
        slope = (f(*hi) - f(*lo)) / (2 * eps)
        along = float((got[name].double() * way).sum())
        # 32-bit gradient: 2^-18 of the terms' size; the difference quotient: eps^2 and rounding, far below
        assert abs(along - slope) <= 2.0 ** -18 * float((got[name].double() * way).abs().sum()) + 1e-6


def test_refusals():
    from tenmo_b200 import TenmoError, make_heads
    from tests import gpu_util as g

    h = g.handle()
    t = g.empty(4096)
    v = make_heads(t.data_ptr(), (1024, 256, 16))
    null = make_heads(0, (1024, 256, 16))
    ok = (1, 1, 1, 4, 4, 16)

    def refused(status, shape=ok, q=v, k=v, o=v, scale=1.0):
        with pytest.raises(TenmoError) as e:
            h.attention_fwd(shape, q, k, v, o, 0, scale)
        assert e.value.status == status
    for shape in ((1, 3, 2, 4, 4, 16), (1, 0, 1, 4, 4, 16), (1, 1, 1, -1, 4, 16), (1, 1, 1, 4, 4, 0), (-1, 1, 1, 4, 4, 16)):
        refused(-1, shape)
    refused(-3, (1, 1, 1, 4, 4, 129))
    refused(-3, (1 << 20, 1 << 12, 1, 4, 4, 16))
    refused(-1, q=null)
    refused(-1, k=null)
    refused(-1, o=null)
    refused(-1, scale=math.inf)
    refused(-1, scale=NAN)
    refused(-1, q=make_heads(t.data_ptr(), (1024, 256, -16)))
    refused(-1, o=make_heads(t.data_ptr(), (1024, 256, 8)))
    other = g.empty(65536)
    out = lambda *strides: make_heads(other.data_ptr(), strides)
    many = (2, 4, 2, 8, 8, 16)
    h.attention_fwd(many, v, v, v, out(512, 128, 16), 0, 1.0)
    h.attention_fwd(many, v, v, v, out(512, 16, 64), 0, 1.0)  # heads inside the row
    h.attention_fwd(many, v, v, v, out(16, 32, 128), 0, 1.0)
    for strides in ((512, 127, 16), (0, 128, 16), (511, 128, 16), (512, 0, 16), (512, 16, 63), (16, 16, 128), (512, 128, 2 ** 62)):
        refused(-1, many, o=out(*strides))
    refused(-1, many, o=v)  # o is an input
    refused(-1, scale=3e38)
    ok_out = [make_heads(other.data_ptr() + 4 * 4096 * e, (512, 128, 16)) for e in range(5)]
    stats = g.empty(1024)
    h.attention_bwd(many, v, v, v, ok_out[0], stats.data_ptr(), ok_out[1], *ok_out[2:], 1.0)
    for bad in ((v, ok_out[3], ok_out[4]), (ok_out[2], ok_out[0], ok_out[4]), (ok_out[2], ok_out[3], ok_out[1]), (ok_out[2], ok_out[2], ok_out[4]),
                (ok_out[2], ok_out[3], make_heads(other.data_ptr() + 16 * 4096 * 4, (512, 0, 16)))):
        with pytest.raises(TenmoError):
            h.attention_bwd(many, v, v, v, ok_out[0], stats.data_ptr(), ok_out[1], *bad, 1.0)
    with pytest.raises(TenmoError):
        h.attention_bwd(ok, v, v, v, v, None, v, v, v, v, 1.0)
    with pytest.raises(TenmoError):
        h.attention_bwd(ok, v, v, v, v, t.data_ptr(), v, v, v, v, 1.0, beta=2.0)
    with pytest.raises(ValueError):
        make_heads(0, (1, 2, 3, 4))
    with pytest.raises(ValueError):
        make_heads(0, (1, 2))


@pytest.mark.parametrize("size", [40, 384])
def test_captured_graph_replays_with_new_inputs_and_lengths(size):
    gen = torch.Generator(device="cuda").manual_seed(13)
    q, k, v, go = (_make(gen, 2, 2, size, 64) for _ in range(4))
    lengths = ints([size, size // 2])
    from tenmo_b200 import make_heads
    from tests import gpu_util as g

    view = lambda t: make_heads(t.data_ptr(), t.stride())
    outs = {n: torch.empty_like(q) for n in ("o", "dq", "dk", "dv")}
    stats = g.empty(2, 2, size, 2)
    shape = (2, 2, 2, size, size, 64)

    def step():
        h = g.handle()
        h.attention_fwd(shape, view(q), view(k), view(v), view(outs["o"]), stats.data_ptr(), 0.125, k_lengths=lengths.data_ptr())
        h.attention_bwd(shape, view(q), view(k), view(v), view(outs["o"]), stats.data_ptr(), view(go), view(outs["dq"]),
                        view(outs["dk"]), view(outs["dv"]), 0.125, k_lengths=lengths.data_ptr())
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        step()
    for t in (q, k, v, go):
        t.copy_(torch.randn(t.shape, device="cuda", generator=gen))
    lengths.copy_(ints([3, size - 1]))
    # another, larger call between capture and replay grows the workspace: the graph keeps its own
    big = [_make(gen, 1, 1, 5000, 64) for _ in range(4)]
    run(*big)
    graph.replay()
    torch.cuda.synchronize()
    want = ar.reference(q, k, v, go, scale=0.125, k_lengths=lengths)
    for name in want:
        ar.check(name, outs[name], want[name])
    g.handle().check_device_status()


def test_layer_in_the_autograd_graph():
    """The same numbers as the layer of three operators that the framework had before, and shared tensors as q = k = v."""
    import tenmo_b200.tensor as T
    from tenmo_b200.attention import Attention

    rng = np.random.default_rng(14)
    q, k, v = (rng.standard_normal((2, 3, 30, 16)).astype(np.float32) for _ in range(3))
    go = rng.standard_normal((2, 3, 30, 16)).astype(np.float32)
    Q, K, V = (T.Tensor.from_numpy(t, requires_grad=True) for t in (q, k, v))
    out = Attention()(Q, K, V)
    out.backward(T.Tensor.from_numpy(go))
    dev = lambda t: torch.from_numpy(np.ascontiguousarray(t)).cuda()
    want = ar.reference(dev(q), dev(k), dev(v), dev(go), scale=0.25)
    for name, t in (("o", out.numpy()), ("dq", Q.grad().numpy()), ("dk", K.grad().numpy()), ("dv", V.grad().numpy())):
        ar.check(name, dev(t), want[name])
    X = T.Tensor.from_numpy(q[:, 0], requires_grad=True)  # rank 3
    y = Attention(causal=True)(X, X, X)
    y.backward(T.Tensor.from_numpy(go[:, 0]))
    x4 = dev(q[:, :1])
    want = ar.reference(x4, x4, x4, dev(go[:, :1]), scale=0.25, causal=True)
    ar.check("o", dev(y.numpy())[:, None], want["o"])
    total = tuple(sum(want[n][e] for n in ("dq", "dk", "dv")) for e in (0, 1))
    ar.check("dx", dev(X.grad().numpy())[:, None], (total[0], total[1] + 4 * ar.U * sum(want[n][0].abs() for n in ("dq", "dk", "dv"))))
    with pytest.raises(RuntimeError):
        Attention()(Q, T.Tensor.zeros(2, 2, 30, 16), T.Tensor.zeros(2, 2, 30, 16))
    with pytest.raises(RuntimeError):
        Attention()(Q, K, V, k_lengths=T.Tensor.labels([1, 2], np.int64))
    heads_last = T.Tensor.from_numpy(np.ascontiguousarray(q.transpose(0, 2, 1, 3)), requires_grad=True)
    view = heads_last.transpose((1, 2))
    got = Attention()(view, K, V)
    got.backward(T.Tensor.from_numpy(go))
    ar.check("dq", dev(heads_last.grad().numpy().transpose(0, 2, 1, 3)), ar.reference(dev(q), dev(k), dev(v), dev(go), scale=0.25)["dq"])
