"""The transformer operators of this framework as timed workloads: attention, layer normalisation and the language-model
head's loss, each forward alone (evaluation, one new token) and as a training pass that returns its gradients.

``run`` computes a case with elementary torch operations while ``own`` is false, and through the framework's public binding
(``tenmo_b200.TenmoCuda``) while it is true; both take what ``prepare`` made.  ``exact`` is the definition in 64 bits.

  attention    O = softmax(scale * Q K^T + mask) V per head; a key/value head may serve several query heads; the mask is
               causal (aligned to the last key), and / or the number of valid keys of each batch entry
  layer_norm   y = (x - mean) / sqrt(var + eps) * gamma + beta over the last axis
  linear_ce    softmax cross-entropy of the logits X W (+ b) against class indices, mean over the rows that are not ignored
"""
import math

import torch

own = False

EPS = 1e-5
IGNORE = -100


# ---- the cases -------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the reference's attention test shape with a few heads: what a unit-sized model calls, launch latency decides
        dict(name="attention train 6x40x16", op="attention", train=True, batch=6, heads=1, kv_heads=1, q_len=40, k_len=40,
             dim=16, causal=False, ragged=False, layout="bhsd"),
        # the attention configuration of the benchmark: 384 heads of 512 positions, 64 wide, evaluation
        dict(name="attention forward 384x512x64", op="attention", train=False, batch=32, heads=12, kv_heads=12, q_len=512,
             k_len=512, dim=64, causal=False, ragged=False, layout="bhsd"),
        # the same heads as a training pass, as they come out of a projection (heads inside the row), padded batch
        dict(name="attention train 384x512x64 ragged", op="attention", train=True, batch=32, heads=12, kv_heads=12, q_len=512,
             k_len=512, dim=64, causal=True, ragged=True, layout="bshd"),
        # long causal training with shared key/value heads and an odd length
        dict(name="attention train 16x4001x128 causal", op="attention", train=True, batch=1, heads=16, kv_heads=4, q_len=4001,
             k_len=4001, dim=128, causal=True, ragged=False, layout="bshd"),
        # one new token of each of 16 requests against the keys so far: evaluation token by token
        dict(name="attention forward one token", op="attention", train=False, batch=16, heads=16, kv_heads=4, q_len=1,
             k_len=4099, dim=64, causal=False, ragged=True, layout="bshd"),
        # layer norm after the first layer of the MNIST-shaped MLP: latency
        dict(name="layer_norm train 64x128", op="layer_norm", train=True, rows=64, cols=128),
        # the activations of the broadcast-matmul configuration, (32, 512, 768), as a training pass
        dict(name="layer_norm train 16384x768", op="layer_norm", train=True, rows=16384, cols=768),
        # the wide MLP's activations, evaluation
        dict(name="layer_norm forward 8192x4096", op="layer_norm", train=False, rows=8192, cols=4096),
        # a small head: the MNIST batch against a thousand classes
        dict(name="linear_ce train 64x128x1000", op="linear_ce", train=True, rows=64, dim=128, vocab=1000, tied=False, bias=True),
        # language-model head in training, weights shared with the embedding (vocab, dim), odd vocabulary
        dict(name="linear_ce train 4096x768x32011", op="linear_ce", train=True, rows=4096, dim=768, vocab=32011, tied=True,
             bias=False),
        # evaluation of a held-out text: the loss alone, weights as Linear keeps them (dim, vocab)
        dict(name="linear_ce forward 2000x1024x50000", op="linear_ce", train=False, rows=2000, dim=1024, vocab=50000, tied=False,
             bias=True),
        # the largest head
        dict(name="linear_ce train 8192x2048x65536", op="linear_ce", train=True, rows=8192, dim=2048, vocab=65536, tied=True,
             bias=False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "layer_norm", "linear_ce"])
    if op == "layer_norm":
        cols = _log_int(rng, 8, 8192)
        return dict(op=op, train=rng.random() < 0.7, rows=_log_int(rng, 1, min(32768, (1 << 25) // cols)), cols=cols)
    if op == "linear_ce":
        dim, vocab = _log_int(rng, 16, 2048), _log_int(rng, 10, 65536)
        rows = _log_int(rng, 1, max(1, min(8192, (1 << 38) // (dim * vocab))))
        return dict(op=op, train=rng.random() < 0.7, rows=rows, dim=dim, vocab=vocab, tied=rng.random() < 0.5,
                    bias=rng.random() < 0.5)
    train = rng.random() < 0.6
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4])
    dim = rng.choice([rng.randint(8, 128), 32, 64, 64, 80, 128])
    # with one key the gradients of the scores vanish and only rounding is left: training starts at eight keys
    k_len = _log_int(rng, 8 if train else 1, 4096)
    q_len = 1 if not train and rng.random() < 0.3 else k_len if rng.random() < 0.7 else _log_int(rng, 2, 4096)
    batch = _log_int(rng, 1, max(1, min(64, (1 << 27) // (kv_heads * group * q_len * k_len))))
    return dict(op=op, train=train, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, q_len=q_len, k_len=k_len, dim=dim,
                causal=rng.random() < 0.5, ragged=rng.random() < 0.4, layout=rng.choice(["bhsd", "bshd"]))


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _heads(gen, case, heads, length):
    """A (batch, heads, length, dim) tensor, contiguous ("bhsd") or as a projection leaves it ("bshd")."""
    b, d = case["batch"], case["dim"]
    if case["layout"] == "bshd":
        return torch.randn(b, length, heads, d, device="cuda", generator=gen).transpose(1, 2)
    return torch.randn(b, heads, length, d, device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    s = dict(case=case)
    if case["op"] == "attention":
        q = _heads(gen, case, case["heads"], case["q_len"])
        k, v = (_heads(gen, case, case["kv_heads"], case["k_len"]) for _ in range(2))
        s.update(q=q, k=k, v=v, o=torch.empty_like(q), scale=1.0 / math.sqrt(case["dim"]), lengths=None)
        s["stats"] = torch.empty(case["batch"], case["heads"], case["q_len"], 2, device="cuda")
        if case["ragged"]:
            low = (case["k_len"] + 1) // 2
            s["lengths"] = torch.randint(low, case["k_len"] + 1, (case["batch"],), device="cuda", generator=gen).to(torch.int32)
        if case["train"]:
            s.update(do=_heads(gen, case, case["heads"], case["q_len"]), dq=torch.empty_like(q), dk=torch.empty_like(k),
                     dv=torch.empty_like(v))
    elif case["op"] == "layer_norm":
        m, c = case["rows"], case["cols"]
        s["x"] = torch.randn(m, c, device="cuda", generator=gen) * 2 + torch.randn(m, 1, device="cuda", generator=gen)
        s["gamma"] = 1 + 0.2 * torch.randn(c, device="cuda", generator=gen)
        s["beta"] = 0.2 * torch.randn(c, device="cuda", generator=gen)
        s.update(y=torch.empty_like(s["x"]), mean=torch.empty(m, device="cuda"), rstd=torch.empty(m, device="cuda"))
        if case["train"]:
            s["dy"] = torch.randn(m, c, device="cuda", generator=gen)
            s.update(dx=torch.empty_like(s["x"]), dgamma=torch.empty_like(s["gamma"]), dbeta=torch.empty_like(s["beta"]))
    else:
        n, d, v = case["rows"], case["dim"], case["vocab"]
        s["x"] = torch.randn(n, d, device="cuda", generator=gen)
        w = torch.randn(*((v, d) if case["tied"] else (d, v)), device="cuda", generator=gen) * (1.5 / math.sqrt(d))
        s["w"] = w.t() if case["tied"] else w  # (dim, vocab), as Linear sees it
        s["bias"] = 0.1 * torch.randn(v, device="cuda", generator=gen) if case["bias"] else None
        s["labels"] = torch.randint(0, v, (n,), device="cuda", generator=gen)
        if n > 8:  # prompt positions and padding carry no loss
            s["labels"][torch.rand(n, device="cuda", generator=gen) < 0.1] = IGNORE
        s.update(loss=torch.empty((), device="cuda"), valid=torch.empty((), dtype=torch.int32, device="cuda"))
        if case["train"]:
            s.update(dx=torch.empty_like(s["x"]), dw=torch.empty_like(s["w"]),
                     db=torch.empty_like(s["bias"]) if case["bias"] else None)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    if own:
        return {"attention": _own_attention, "layer_norm": _own_layer_norm, "linear_ce": _own_linear_ce}[c["op"]](state, c)
    return {"attention": _attention, "layer_norm": _layer_norm, "linear_ce": _linear_ce}[c["op"]](state, c)


def _visible(c, lengths):
    """The (1 or batch, 1, 1, q_len, k_len) truth values of the mask, or None where every key is visible."""
    keep = None
    j = torch.arange(c["k_len"], device="cuda")
    if c["causal"]:
        i = torch.arange(c["q_len"], device="cuda")
        keep = (j[None, :] <= i[:, None] + (c["k_len"] - c["q_len"]))[None, None, None]
    if lengths is not None:
        valid = (j[None, :] < lengths[:, None])[:, None, None, None, :]
        keep = valid if keep is None else keep & valid
    return keep


def _attention(s, c):
    b, h, g = c["batch"], c["kv_heads"], c["heads"] // c["kv_heads"]
    q = s["q"].reshape(b, h, g, c["q_len"], c["dim"])
    k, v = s["k"].unsqueeze(2), s["v"].unsqueeze(2)
    p = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    keep = _visible(c, s["lengths"])
    if keep is not None:
        p = torch.where(keep, p, -math.inf)
    m = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = torch.matmul(p, v)
    out = dict(o=o.reshape(s["q"].shape))
    if c["train"]:
        do = s["do"].reshape(q.shape)
        ds = p * (torch.matmul(do, v.transpose(-1, -2)) - (do * o).sum(-1, keepdim=True)) * s["scale"]
        out["dq"] = torch.matmul(ds, k).reshape(s["q"].shape)
        out["dk"] = torch.matmul(ds.transpose(-1, -2), q).sum(2)
        out["dv"] = torch.matmul(p.transpose(-1, -2), do).sum(2)
    return out


def _own_attention(s, c):
    from tenmo_b200 import make_heads
    from tenmo_b200.tensor import handle

    h = handle()
    shape = (c["batch"], c["heads"], c["kv_heads"], c["q_len"], c["k_len"], c["dim"])
    view = {n: make_heads(s[n].data_ptr(), s[n].stride()) for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv") if n in s}
    lengths = s["lengths"].data_ptr() if s["lengths"] is not None else 0
    h.attention_fwd(shape, view["q"], view["k"], view["v"], view["o"], s["stats"].data_ptr(), s["scale"], causal=c["causal"],
                    k_lengths=lengths)
    out = dict(o=s["o"])
    if c["train"]:
        h.attention_bwd(shape, view["q"], view["k"], view["v"], view["o"], s["stats"].data_ptr(), view["do"], view["dq"],
                        view["dk"], view["dv"], s["scale"], causal=c["causal"], k_lengths=lengths)
        out.update(dq=s["dq"], dk=s["dk"], dv=s["dv"])
    return out


def _layer_norm(s, c):
    x = s["x"]
    centred = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    xhat = centred * rstd
    out = dict(y=xhat * s["gamma"] + s["beta"])
    if c["train"]:
        g = s["dy"] * s["gamma"]
        out["dx"] = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
        out["dgamma"] = (s["dy"] * xhat).sum(0)
        out["dbeta"] = s["dy"].sum(0)
    return out


def _own_layer_norm(s, c):
    from tenmo_b200.tensor import handle

    h, m, n = handle(), c["rows"], c["cols"]
    h.layernorm_fwd(s["x"].data_ptr(), n, s["gamma"].data_ptr(), s["beta"].data_ptr(), EPS, s["y"].data_ptr(),
                    s["mean"].data_ptr(), s["rstd"].data_ptr(), m, n)
    out = dict(y=s["y"])
    if c["train"]:
        h.layernorm_bwd(s["x"].data_ptr(), n, s["dy"].data_ptr(), s["gamma"].data_ptr(), s["mean"].data_ptr(),
                        s["rstd"].data_ptr(), s["dx"].data_ptr(), s["dgamma"].data_ptr(), s["dbeta"].data_ptr(), m, n)
        out.update(dx=s["dx"], dgamma=s["dgamma"], dbeta=s["dbeta"])
    return out


def _linear_ce(s, c):
    logits = torch.matmul(s["x"], s["w"])
    if s["bias"] is not None:
        logits = logits + s["bias"]
    used = s["labels"] != IGNORE
    label = torch.where(used, s["labels"], 0)[:, None]
    m = logits.amax(-1, keepdim=True)
    e = torch.exp(logits - m)
    total = e.sum(-1, keepdim=True)
    count = used.sum()
    row = (torch.log(total) + m - logits.gather(1, label))[:, 0]
    out = dict(loss=torch.where(used, row, 0.0).sum() / torch.clamp(count, min=1))
    if c["train"]:
        g = e / total
        g.scatter_add_(1, label, torch.full_like(g[:, :1], -1.0))
        g = g * (used / torch.clamp(count, min=1))[:, None]
        out["dx"] = torch.matmul(g, s["w"].t())
        out["dw"] = torch.matmul(g.t(), s["x"]).t() if c["tied"] else torch.matmul(s["x"].t(), g)
        if s["bias"] is not None:
            out["db"] = g.sum(0)
    return out


def _own_linear_ce(s, c):
    from tenmo_b200 import make_mat
    from tenmo_b200.tensor import handle

    h, n, d, v = handle(), c["rows"], c["dim"], c["vocab"]
    x, w = make_mat(s["x"].data_ptr(), (n, d), s["x"].stride()), make_mat(s["w"].data_ptr(), (d, v), s["w"].stride())
    bias = s["bias"].data_ptr() if s["bias"] is not None else 0
    if not c["train"]:
        h.linear_ce_fwd(x, w, bias, s["labels"].data_ptr(), True, n, d, v, IGNORE, 0.0, 0, s["loss"].data_ptr(),
                        s["valid"].data_ptr())
        return dict(loss=s["loss"])
    h.linear_ce_fwd_bwd(x, w, bias, s["labels"].data_ptr(), True, n, d, v, IGNORE, 0.0, 0, s["loss"].data_ptr(),
                        s["valid"].data_ptr(), 0, s["dx"].data_ptr(), s["dw"].data_ptr(),
                        s["db"].data_ptr() if s["bias"] is not None else 0)
    out = dict(loss=s["loss"], dx=s["dx"], dw=s["dw"])
    if s["bias"] is not None:
        out["db"] = s["db"]
    return out


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    if case["op"] == "layer_norm":
        m, c = case["rows"], case["cols"]
        return dict(bytes=4 * (m * c * (4 if case["train"] else 2) + 4 * c), flops=m * c * (19 if case["train"] else 8))
    if case["op"] == "linear_ce":
        n, d, v = case["rows"], case["dim"], case["vocab"]
        extra = v if case["bias"] else 0
        moved = n * d + d * v + extra
        return dict(bytes=4 * (2 * moved if case["train"] else moved) + 8 * n, flops=(6 if case["train"] else 2) * n * d * v)
    q_len, k_len, d = case["q_len"], case["k_len"], case["dim"]
    used = k_len * (0.75 if case["ragged"] else 1.0)  # the lengths are uniform over the upper half
    pairs = q_len * used
    if case["causal"]:  # rows i see min(used, i + k_len - q_len + 1) keys; the mean length stands for all of them
        pairs = sum(max(0, min(used, i + k_len - q_len + 1)) for i in range(q_len))
    rows, keys = case["batch"] * case["heads"], case["batch"] * case["kv_heads"]
    qo, kv = rows * q_len * d, keys * used * d
    if case["train"]:  # q, o, do, dq and k, v, dk, dv; six products: scores, output and four for the gradients
        return dict(bytes=4 * (4 * qo + 2 * kv + 2 * keys * k_len * d), flops=12 * rows * pairs * d)
    return dict(bytes=4 * (2 * qo + 2 * kv), flops=4 * rows * pairs * d)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "layer_norm": _exact_layer_norm, "linear_ce": _exact_linear_ce}[case["op"]](s, case)


def _exact_attention(s, c):
    group, names = c["heads"] // c["kv_heads"], ["o"] + (["dq", "dk", "dv"] if c["train"] else [])
    out = {n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in names}
    lengths = s["lengths"].tolist() if s["lengths"] is not None else [c["k_len"]] * c["batch"]
    for b in range(c["batch"]):
        n = lengths[b]
        for h in range(c["heads"]):
            q, k, v = s["q"][b, h].double(), s["k"][b, h // group, :n].double(), s["v"][b, h // group, :n].double()
            score = (q @ k.T) / math.sqrt(c["dim"])
            if c["causal"]:
                hidden = torch.ones(c["q_len"], c["k_len"], dtype=torch.bool, device="cuda").triu(c["k_len"] - c["q_len"] + 1)
                score.masked_fill_(hidden[:, :n], -math.inf)
            prob = torch.nan_to_num((score - torch.logsumexp(score, 1, keepdim=True)).exp(), nan=0.0)
            out["o"][b, h] = prob @ v
            if c["train"]:
                do = s["do"][b, h].double()
                dprob = do @ v.T
                dscore = (prob * (dprob - (prob * dprob).sum(1, keepdim=True))) / math.sqrt(c["dim"])
                out["dq"][b, h] = dscore @ k
                out["dk"][b, h // group, :n] += dscore.T @ q
                out["dv"][b, h // group, :n] += prob.T @ do
    return out


def _exact_layer_norm(s, c):
    x, n = s["x"].double(), c["cols"]
    var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    sigma = (var + EPS).sqrt()
    z = (x - mean) / sigma
    out = dict(y=z * s["gamma"].double() + s["beta"].double())
    if c["train"]:
        dy = s["dy"].double()
        dz = dy * s["gamma"].double()
        out["dx"] = (n * dz - dz.sum(1, keepdim=True) - z * (dz * z).sum(1, keepdim=True)) / (n * sigma)
        out["dgamma"] = torch.einsum("mc,mc->c", dy, z)
        out["dbeta"] = dy.sum(0)
    return out


def _exact_linear_ce(s, c):
    n, step = c["rows"], 1024
    w, bias = s["w"].double(), s["bias"].double() if s["bias"] is not None else None
    keep = s["labels"] != IGNORE
    count = max(1, int(keep.sum()))
    loss = torch.zeros((), dtype=torch.float64, device="cuda")
    out = {}
    if c["train"]:
        out.update(dx=torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda"), dw=torch.zeros_like(w))
        if bias is not None:
            out["db"] = torch.zeros_like(bias)
    for a in range(0, n, step):
        x, y, used = s["x"][a:a + step].double(), s["labels"][a:a + step].clamp(min=0), keep[a:a + step]
        log_p = torch.log_softmax(x @ w if bias is None else x @ w + bias, 1)
        rows = torch.arange(x.shape[0], device="cuda")
        loss -= (log_p[rows, y] * used).sum() / count
        if c["train"]:
            g = log_p.exp()
            g[rows, y] -= 1
            g *= used[:, None] / count
            out["dx"][a:a + step] = g @ w.T
            out["dw"] += x.T @ g
            if bias is not None:
                out["db"] += g.sum(0)
    out["loss"] = loss
    return out
