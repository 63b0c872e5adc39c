"""Layer norm, attention and the language-model loss in a row, as a training step calls them: one block and a tied head, its
gradients against torch's own in 64 bits, and a step of SGD on them."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("size", [(2, 20, 4, 8, 50), (2, 160, 4, 64, 700)], ids=str)
def test_block_and_tied_head(size):
    import tenmo_b200.tensor as T
    from tenmo_b200.attention import Attention
    from tenmo_b200.crossentropy import LinearCrossEntropyLoss
    from tenmo_b200.net import LayerNorm, Linear
    from tenmo_b200.optim import SGD

    B, S, H, D, V = size
    E = H * D
    rng = np.random.default_rng(S)
    emb = (rng.standard_normal((V, E)) / math.sqrt(E)).astype(np.float32)
    hidden = rng.standard_normal((B, S, E)).astype(np.float32)
    target = rng.integers(0, V, B * S)
    lengths = np.array([S, S - S // 3], np.int32)
    for b in range(B):
        target.reshape(B, S)[b, lengths[b]:] = -100

    X = T.Tensor.from_numpy(hidden, requires_grad=True)
    W = T.Tensor.from_numpy(emb, requires_grad=True)
    norm, final = LayerNorm(E), LayerNorm(E)
    proj = [Linear(E, E, init_seed=n, init_method="xavier", bias=False) for n in range(3)]
    y = norm(X)

    def heads(t):  # (B, S, E) -> the (B, H, S, D) view of the same storage
        v = T.Tensor(t.buffer.view((B, H, S, D), (S * E, D, E, 1)), requires_grad=True)
        return v
    # the projections are leaves of the attention graph here: their outputs are viewed as heads, which the host mirror has no
    # tag for, so the gradient is carried over by hand
    q, k, v = (p(y) for p in proj)
    hq, hk, hv = heads(q), heads(k), heads(v)
    att = Attention(causal=True)(hq, hk, hv, k_lengths=T.Tensor.labels(lengths, np.int32))
    rows = T.Tensor(att.transpose((1, 2)).buffer.contiguous().reshape((B * S, E)), requires_grad=True)
    out = final(rows)
    loss = LinearCrossEntropyLoss()(out, W.transpose(), T.Tensor.labels(target))
    loss.backward()
    att.backward(T.Tensor(T.NDBuffer(rows.gradbox.storage, (B, S, H, D)).transpose((1, 2)).contiguous()))
    for t, h in ((q, hq), (k, hk), (v, hv)):
        t.backward(T.Tensor(h.gradbox.transpose((1, 2)).contiguous().reshape((B, S, E))))

    # the same in torch, 64 bits
    tx, tw = torch.tensor(hidden).double().requires_grad_(), torch.tensor(emb).double().requires_grad_()
    ws = [torch.tensor(p.weight.numpy()).double().requires_grad_() for p in proj]
    ty = torch.nn.functional.layer_norm(tx, (E,))
    a, b_, c = ((ty @ w_).reshape(B, S, H, D).transpose(1, 2) for w_ in ws)
    s = a @ b_.transpose(-1, -2) / math.sqrt(D)
    keep = torch.ones(S, S, dtype=torch.bool).tril() & (torch.arange(S) < torch.tensor(lengths)[:, None])[:, None, None, :]
    o = (torch.softmax(s.masked_fill(~keep, -math.inf), -1) @ c).transpose(1, 2).reshape(B * S, E)
    tl = torch.nn.functional.cross_entropy(torch.nn.functional.layer_norm(o, (E,)) @ tw.T, torch.tensor(target), ignore_index=-100)
    tl.backward()
    tl = tl.detach()

    # a chain of five operators in 32 bits: each is off by at most some 2^-18 of the terms it sums (see the operators' own
    # tests); 2^-13 of the gradient's largest entry leaves room for the five and for the cancellation in the layer norms
    def near(got, want, what):
        got = torch.tensor(got).double()
        assert float((got - want).abs().max()) <= 2.0 ** -13 * float(want.abs().max()), what
    assert abs(loss.item() - float(tl)) <= 2.0 ** -16 * abs(float(tl))
    near(W.grad().numpy(), tw.grad, "embedding")
    for p, w_ in zip(proj, ws):
        near(p.weight.grad().numpy(), w_.grad, "projection")
    near(X.grad().numpy(), tx.grad, "input")
    T.handle().check_device_status()

    before = W.numpy().copy()
    SGD([W] + [p.weight for p in proj] + norm.parameters() + final.parameters(), lr=0.1).step()
    near(W.numpy(), torch.tensor(before).double() - 0.1 * tw.grad, "updated embedding")
