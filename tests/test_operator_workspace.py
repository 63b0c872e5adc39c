"""What the host code of the transformer operators does with its workspace: sizes, lifetimes and order, without a GPU."""
import random
import shutil

import pytest

from tests import fake_cuda

MB = 1 << 20


@pytest.fixture(scope="module")
def library(tmp_path_factory):
    return fake_cuda.build(tmp_path_factory.mktemp("fake"))


@pytest.fixture()
def fake(library, tmp_path):
    f = fake_cuda.Fake(shutil.copy(library, tmp_path))  # a copy: its state begins anew
    yield f
    f.handle.close()
    assert f.misuse() == []


def linear_ce(fake, N, D, V, tied=False, bias=False, forward_only=False, handle=None):
    """The operands' addresses are never read here."""
    from tenmo_b200 import make_mat

    x = make_mat(1 << 40, (N, D), (D, 1))
    w = make_mat(1 << 41, (D, V), (1, D) if tied else (V, 1))
    args = (x, w, (1 << 42) if bias else 0, 1 << 43, True, N, D, V, -100, 0.0, 0, 1 << 44, (1 << 44) + 64)
    h = handle or fake.handle
    if forward_only:
        h.linear_ce_fwd(*args)
    else:
        h.linear_ce_fwd_bwd(*args, 0, 1 << 45, 1 << 46, (1 << 47) if bias else 0)


# rows, dim and classes whose last piece of the rows splits its product for dw into more slices than a whole piece
MORE_SLICES_IN_THE_LAST_PIECE = [(38912, 576, 6300), (46080, 832, 5000), (151040, 1856, 1200), (50972, 1024, 4888)]


def check_slices(fake):
    """Every product cut into slices writes them inside the workspace: the fold reads (slices, M, ldp) floats from `partial`."""
    seen = 0
    for _, name, args in fake.launches():
        if "h3_fold_kernel" in name:
            partial, slices, M, N, ldp = args[:5]
            assert fake.lib.fake_room_behind(partial) >= slices * M * ldp * 4, (slices, M, N)
            seen += 1
    fake.lib.fake_forget_launches()
    return seen


@pytest.mark.parametrize("tied", [False, True], ids=["linear", "tied"])
@pytest.mark.parametrize("shape", MORE_SLICES_IN_THE_LAST_PIECE, ids=str)
def test_slices_of_every_piece_fit_the_workspace(fake, shape, tied):
    fake.watch("h3_fold_kernel", "PiqqqPqi")
    linear_ce(fake, *shape, tied=tied)
    assert check_slices(fake) > 0


def test_slices_fit_over_the_range(fake):
    """Sizes at random, most of them in several pieces, each from an empty workspace."""
    from tenmo_b200 import TenmoCuda, TenmoError

    rng = random.Random(1)
    fake.watch("h3_fold_kernel", "PiqqqPqi")
    seen = 0
    for _ in range(3000):
        D, V = 8 * int(2 ** rng.uniform(4, 8)), int(2 ** rng.uniform(9, 14))
        N = int((128 << 20) / V * 2 ** rng.uniform(-3, 2))
        handle = TenmoCuda(0, path=fake.path).require()
        try:
            linear_ce(fake, N, D, V, tied=rng.random() < 0.5, bias=rng.random() < 0.5, handle=handle)
        except TenmoError as e:
            assert e.status == -4  # more than the card holds
        seen += check_slices(fake)
        handle.close()
    assert seen > 1000


# row sums of db above 512 rows, in the strict-fp32 form (rows) and in the tensor-core form (blocks of 128 rows)
@pytest.mark.parametrize("shape", [(700, 100, 31), (100000, 256, 100)], ids=str)
def test_a_captured_bias_gradient_keeps_its_scratch(fake, shape):
    """Larger column sums after the capture grow the library's ordinary workspace and its tickets; what the graph uses stays allocated."""
    fake.watch("colsum_split_kernel", "PqqqPfPPi")
    linear_ce(fake, *shape, bias=True)
    stream = fake.lib.fake_stream_create(0)
    fake.handle.set_stream(stream)
    fake.lib.fake_capture(stream, 1)
    linear_ce(fake, *shape, bias=True)
    fake.lib.fake_capture(stream, 0)
    fake.handle.colsum(1 << 40, 100000, 1 << 19, 1 << 19, 1 << 41)
    fake.handle.colsum(1 << 40, 1000, 1 << 22, 1 << 22, 1 << 41)
    used = [args for i, name, args in fake.launches() if fake.captured(i) and "colsum_split_kernel" in name]
    assert len(used) == 1
    strips = -(-shape[2] // 32)
    rows = shape[0] if shape[0] == 700 else -(-shape[0] // 128)
    for x, M, N, _, _, _, partials, tickets, per_slab in used:
        assert (M, N) == (rows, shape[2])
        assert fake.lib.fake_room_behind(partials) >= -(-M // per_slab) * N * 4
        assert fake.lib.fake_room_behind(tickets) >= strips * 4
        assert fake.lib.fake_room_behind(x) >= M * N * 4


def test_column_sums_fit_over_the_range(fake):
    """Sizes at random whose bias gradient is summed over more than 512 rows, or over more than 512 blocks of rows."""
    from tenmo_b200 import TenmoCuda

    rng = random.Random(2)
    fake.watch("colsum_split_kernel", "PqqqPfPPi")
    seen = 0
    for e in range(600):
        if e % 2:
            N = int(2 ** rng.uniform(9.1, 14))
            V = int(2 ** rng.uniform(0, 20))
            D = max(1, int(4e7 / N / V))
        else:
            N, V, D = int(2 ** rng.uniform(16, 22)), int(2 ** rng.uniform(0, 9)), int(2 ** rng.uniform(6, 9))
        handle = TenmoCuda(0, path=fake.path).require()
        linear_ce(fake, N, D, V, tied=rng.random() < 0.5, bias=True, handle=handle)
        for _, name, args in fake.launches():
            if "colsum_split_kernel" in name:
                x, M, n, _, _, _, partials, tickets, per_slab = args
                assert fake.lib.fake_room_behind(partials) >= -(-M // per_slab) * n * 4, (N, D, V)
                assert partials - tickets >= -(-n // 32) * 4 and partials >= x + M * n * 4
                seen += 1
        fake.lib.fake_forget_launches()
        handle.close()
    assert seen > 300


def largest_operands(N, D, V):
    """Bytes beside a piece of the rows: the image of the weight, the row losses."""
    up = lambda n: -(-n // 128) * 128
    return 4 * up(D) * up(V) + 4 * N


@pytest.mark.parametrize("shape,forward_only", [((1000000, 4096, 1000), True), ((1000000, 2048, 1000), True), ((1000000, 4096, 100), False),
                                                ((3000000, 300, 10), False), ((1000000, 47, 1), False)], ids=str)
def test_a_piece_counts_the_rows_of_x(fake, shape, forward_only):
    """Few classes: many rows of logits fit the budget of a piece, but its copy of x has to fit one too.  (The slices of dx's and
    dw's products, at most 32 of a piece's or the weight's size, come on top.)"""
    N, D, V = shape
    linear_ce(fake, *shape, bias=True, forward_only=forward_only)
    assert fake.lib.fake_bytes_alive() < 3 * (512 * MB) + largest_operands(N, D, V)


# ---- graphs beside eager calls ----
def layer_norm_bwd(fake, C=512, M=4096):
    """A call that uses the workspace; returns where (its partial sums begin there)."""
    fake.handle.layernorm_bwd(1 << 40, C, 1 << 41, 1 << 42, 1 << 43, 1 << 43, 1 << 44, 1 << 45, 1 << 46, M, C)
    i, _, args = [l for l in fake.launches() if "ln_fold_kernel" in l[1]][-1]
    return args[0], args[1] * 2 * C * 4, i


def captured(fake, call, stream=None):
    stream = stream or fake.lib.fake_stream_create(0)
    fake.handle.set_stream(stream)
    fake.lib.fake_capture(stream, 1)
    try:
        return call()
    finally:
        fake.lib.fake_capture(stream, 0)
        fake.handle.set_stream(None)


def overlap(a, b):
    return a[0] < b[0] + b[1] and b[0] < a[0] + a[1]


def test_eager_calls_stay_off_a_captured_block(fake):
    """A replay and an eager call on another stream are not ordered by anything: they must not share a block."""
    fake.watch("ln_fold_kernel", "PiiPPi")
    layer_norm_bwd(fake)
    graph = captured(fake, lambda: layer_norm_bwd(fake))
    for C in (512, 64, 4096, 512):
        assert not overlap(graph, layer_norm_bwd(fake, C))
    assert fake.lib.fake_room_behind(graph[0]) >= graph[1]


def test_captures_and_eager_calls_in_turn(fake):
    """Two blocks serve them however often they alternate; a larger capture takes a larger block, and every graph keeps its own."""
    fake.watch("ln_fold_kernel", "PiiPPi")
    layer_norm_bwd(fake)
    captured(fake, lambda: layer_norm_bwd(fake))
    layer_norm_bwd(fake)
    before = fake.lib.fake_bytes_alive()
    for _ in range(40):
        captured(fake, lambda: layer_norm_bwd(fake))
        layer_norm_bwd(fake)
    assert fake.lib.fake_bytes_alive() == before
    graphs = []
    for n in range(40):
        eager = layer_norm_bwd(fake, 512 + 256 * n)
        graphs.append(captured(fake, lambda: layer_norm_bwd(fake, 512 + 256 * n)))
        assert fake.lib.fake_room_behind(eager[0]) >= eager[1]
        for g in graphs:
            assert fake.lib.fake_room_behind(g[0]) >= g[1] and not overlap(g, layer_norm_bwd(fake, 64))


def test_a_capture_larger_than_every_call_before_is_refused(fake):
    from tenmo_b200 import TenmoError

    fake.watch("ln_fold_kernel", "PiiPPi")
    layer_norm_bwd(fake, 64)
    with pytest.raises(TenmoError) as e:
        captured(fake, lambda: layer_norm_bwd(fake, 4096))
    assert e.value.status == -7
    layer_norm_bwd(fake, 4096)
    captured(fake, lambda: layer_norm_bwd(fake, 4096))


def test_an_eager_call_beside_a_capture_in_progress(fake):
    """The block went to the graph a moment ago; the eager call gets another although a stream is being captured."""
    fake.watch("ln_fold_kernel", "PiiPPi")
    layer_norm_bwd(fake)

    def call():
        graph = layer_norm_bwd(fake)
        fake.handle.set_stream(None)
        assert not overlap(graph, layer_norm_bwd(fake))
    captured(fake, call)


# ---- streams ----
def first_and_last(fake, call):
    """The launches of a call: its first and its last one."""
    n = fake.lib.fake_launches()
    call()
    assert fake.lib.fake_launches() > n
    return n, fake.lib.fake_launches() - 1


def test_calls_on_several_streams_wait_for_one_another(fake):
    streams = [0] + [fake.lib.fake_stream_create(0) for _ in range(3)]
    before = None
    fake.watch("ln_fold_kernel", "PiiPPi")
    for n in (0, 1, 1, 2, 0, 0, 3, 2, 1):
        fake.handle.set_stream(streams[n])
        at = first_and_last(fake, lambda: layer_norm_bwd(fake, 64 + 8 * n))
        assert before is None or fake.comes_before(before, at[0])
        before = at[1]


@pytest.mark.parametrize("used_before", [False, True], ids=["one stream so far", "several streams so far"])
def test_a_destroyed_stream_is_not_touched(fake, used_before):
    """A caller may destroy a stream as soon as its calls have returned: nothing may use the handle again, and what still runs there comes
    before the next call."""
    fake.watch("ln_fold_kernel", "PiiPPi")
    if used_before:
        layer_norm_bwd(fake, 64)
    stream = fake.lib.fake_stream_create(0)
    fake.handle.set_stream(stream)
    a = first_and_last(fake, lambda: layer_norm_bwd(fake, 512))
    fake.lib.fake_stream_destroy(stream)
    fake.handle.set_stream(None)
    b = first_and_last(fake, lambda: layer_norm_bwd(fake, 512))
    assert fake.comes_before(a[1], b[0])
    c = first_and_last(fake, lambda: layer_norm_bwd(fake, 8000))  # the workspace grows
    assert fake.comes_before(b[1], c[0])
    assert fake.misuse() == []


def test_a_handle_that_is_used_again_is_another_stream(fake):
    """A new stream can get the address of one that was destroyed while its work was still running."""
    fake.watch("ln_fold_kernel", "PiiPPi")
    stream = fake.lib.fake_stream_create(0)
    fake.handle.set_stream(stream)
    a = first_and_last(fake, lambda: layer_norm_bwd(fake))
    fake.lib.fake_stream_destroy(stream)
    assert fake.lib.fake_stream_create(stream) == stream
    fake.handle.set_stream(stream)
    b = first_and_last(fake, lambda: layer_norm_bwd(fake))
    assert fake.comes_before(a[1], b[0])


def test_every_operator_orders_its_workspace(fake):
    """Each entry point that uses the workspace, on one stream and then another."""
    from tenmo_b200 import make_heads

    streams = [fake.lib.fake_stream_create(0) for _ in range(2)]
    fake.watch("ln_fold_kernel", "PiiPPi")

    def attention(q_len, k_len, H, backward):
        B, D, Hkv = 2, 64, H // 2
        view = lambda at, heads, n: make_heads(at << 40, (heads * n * D, n * D, D))
        q, k, v, o = view(1, H, q_len), view(2, Hkv, k_len), view(3, Hkv, k_len), view(4, H, q_len)
        shape = (B, H, Hkv, q_len, k_len, D)
        if backward:
            fake.handle.attention_bwd(shape, q, k, v, o, 5 << 40, view(6, H, q_len), view(7, H, q_len), view(8, Hkv, k_len), view(9, Hkv, k_len), 0.125)
        else:
            fake.handle.attention_fwd(shape, q, k, v, o, 5 << 40, 0.125)
    calls = [lambda: attention(1, 4000, 4, False), lambda: attention(600, 600, 8, False), lambda: attention(20, 20, 4, True),
             lambda: attention(600, 600, 8, True), lambda: layer_norm_bwd(fake), lambda: linear_ce(fake, 20, 30, 40),
             lambda: linear_ce(fake, 300, 30, 400, bias=True), lambda: linear_ce(fake, 3000, 300, 4000, bias=True),
             lambda: linear_ce(fake, 3000, 300, 4000, forward_only=True)]
    before = None
    for call in calls + calls[::-1] + calls:
        fake.handle.set_stream(streams[0])
        streams.reverse()
        at = first_and_last(fake, call)
        assert before is None or fake.comes_before(before, at[0])
        before = at[1]


# ---- strict fp32 ----
def test_strict_fp32_reaches_no_tensor_core_kernel(fake):
    """Sizes that otherwise run on tensor cores, attention and linear cross-entropy."""
    from tenmo_b200 import ALGO_AUTO, ALGO_SIMT_FP32, ALGO_TC_3XTF32, TenmoError, make_heads

    view = lambda at, heads, n: make_heads(at << 40, (heads * n * 64, n * 64, 64))

    def kernels():
        B, H, n = 4, 8, 600
        shape, t = (B, H, H, n, n, 64), [view(at, H, n) for at in range(1, 10)]
        fake.lib.fake_forget_launches()
        fake.handle.attention_fwd(shape, *t[:4], 5 << 50, 0.125)
        fake.handle.attention_bwd(shape, *t[:4], 5 << 50, *t[4:8], 0.125)
        linear_ce(fake, 3000, 300, 4000, bias=True)
        linear_ce(fake, 100, 3000, 4000, bias=True, tied=True)
        linear_ce(fake, 3000, 300, 4000, forward_only=True)
        return [name for _, name, _ in fake.launches()]
    on_tensor_cores = ("attn_fwd_tc", "attn_bwd_tc", "attn_tiles", "h3_")
    some = kernels()
    for part in on_tensor_cores:
        assert any(part in name for name in some)
    fake.handle.operators_set_algo(ALGO_SIMT_FP32)
    assert not any(part in name for name in kernels() for part in on_tensor_cores)
    fake.handle.operators_set_algo(ALGO_AUTO)
    assert kernels() == some
    for bad in (ALGO_TC_3XTF32, 7, -2):
        with pytest.raises(TenmoError):
            fake.handle.operators_set_algo(bad)


def test_slices_of_long_contractions_fit_over_the_range(fake):
    """Strict fp32, sizes at random with long rows, classes and dims: the partial results that the sequential column sum adds lie in the
    workspace."""
    from tenmo_b200 import ALGO_SIMT_FP32, TenmoCuda, TenmoError

    rng = random.Random(3)
    fake.watch("colsum_seq_kernel", "PqqqPf")
    seen = 0
    for _ in range(600):
        size = [2 ** rng.uniform(0, 9), 2 ** rng.uniform(0, 12), 2 ** rng.uniform(8.1, 20)]
        rng.shuffle(size)
        N, D, V = max(257, int(size[0])), int(size[1]), int(size[2])
        handle = TenmoCuda(0, path=fake.path).require()
        handle.operators_set_algo(ALGO_SIMT_FP32)
        try:
            linear_ce(fake, N, D, V, tied=rng.random() < 0.5, bias=rng.random() < 0.5, handle=handle)
        except TenmoError as e:
            assert e.status == -4  # more than the card holds
        for _, name, args in fake.launches():
            if "colsum_seq_kernel" in name:
                x, M, n, ld, out, _ = args
                assert ld == n and M <= 512
                assert fake.lib.fake_room_behind(x) >= M * n * 4, (N, D, V)
                seen += fake.lib.fake_room_behind(out) == 0  # not the bias gradient's part of the workspace
        fake.lib.fake_forget_launches()
        handle.close()
    assert seen > 300
