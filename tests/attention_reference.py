"""Attention in 64 bits with a bound for every element of a 32-bit result (u = 2^-24).

Any kernel here forms a score from products of operands that are represented to 2^-22 and sums of at most `dim` terms, so a score
is off by at most e_s = (dim + 64) u * scale * sum_d |q k| plus a floor for operands far below the largest of their tile
(2^-38 of the product of the largest entries, times dim).  A probability then is off by a factor 1 + 2 max_j e_s + c u, with c the
length of the sums and the exponential's own error, and the rest follows term by term:
  o   (r + c u) sum_j p |v|                    r = 2 max_j e_s,  c = 64 + sqrt-free count of tile joins (keys / 32)
  dv  sum_i p (r + c u) |go|
  ds  scale p [ (r + c u)(|dp| + |delta|) + (dim + 64) u (sum|go v| + sum|go o|) + |go| . e_o ]
  dq  sum_j e_ds |k| + c u sum_j |ds k|,  dk alike over the rows
"""
import torch

U = 2.0 ** -24


def visible(B, H, Sq, Sk, causal, q_lengths, k_lengths, device):
    keep = torch.ones(B, 1, Sq, Sk, dtype=torch.bool, device=device)
    i, j = torch.arange(Sq, device=device)[:, None], torch.arange(Sk, device=device)[None, :]
    if causal:
        keep = keep & (j <= i + Sk - Sq)
    if q_lengths is not None:
        keep = keep & (i < q_lengths.to(device).long()[:, None, None, None])
    if k_lengths is not None:
        keep = keep & (j < k_lengths.to(device).long()[:, None, None, None])
    return keep


def reference(q, k, v, go=None, scale=1.0, causal=False, q_lengths=None, k_lengths=None):
    """{name: (value, bound)} for o and, with `go`, dq, dk, dv.  Inputs (B, H | Hkv, S, D)."""
    B, H, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    G = H // Hkv
    keep = visible(B, H, Sq, Sk, causal, q_lengths, k_lengths, q.device)
    rows_in = keep.any(3, keepdim=True).expand(B, H, Sq, 1)
    keys_in = keep.any(2)[..., None].expand(B, Hkv, Sk, 1)
    q = torch.where(rows_in, q.double(), 0.0)  # what takes no part may hold anything
    k, v = (torch.where(keys_in, t.double(), 0.0) for t in (k, v))
    rep = lambda t: t.repeat_interleave(G, 1)
    K, V = rep(k), rep(v)
    c = 64 + Sk / 32
    s = scale * (q @ K.transpose(-1, -2))
    floor = 2.0 ** -38 * D * abs(scale) * q.abs().amax((-1, -2), keepdim=True) * K.abs().amax((-1, -2), keepdim=True) if Sk and Sq else 0.0
    e_s = (D + 64) * U * abs(scale) * (q.abs() @ K.abs().transpose(-1, -2)) + floor
    e_s = torch.where(keep, e_s, 0.0)
    s = torch.where(keep, s, -torch.inf)
    p = torch.where(rows_in, torch.softmax(s, -1), 0.0) if Sk else s
    r = 2 * e_s.amax(-1, keepdim=True) + c * U if Sk else 0.0
    vmax = V.abs().amax((-1, -2), keepdim=True) if Sk else 0.0
    o = p @ V
    e_o = r * (p @ V.abs()) + 2.0 ** -37 * vmax * rows_in
    out = dict(o=(o, e_o))
    if go is None:
        return out
    go = torch.where(rows_in, go.double(), 0.0)
    fold = lambda t: t.reshape(B, Hkv, G, *t.shape[2:]).sum(2)
    cq = 64 + G * Sq / 32
    T = lambda t: t.transpose(-1, -2)
    gmax = go.abs().amax((-1, -2), keepdim=True) if Sq else 0.0
    dv = fold(T(p) @ go)
    e_dv = fold(T(p * r) @ go.abs() + cq * U * (T(p) @ go.abs()) + 2.0 ** -37 * (gmax * T(rows_in.double()).sum(-1, keepdim=True)))
    dp, delta = go @ T(V), (go * o).sum(-1, keepdim=True)
    ds = scale * p * (dp - delta)
    e_dp = (D + 64) * U * (go.abs() @ T(V.abs()) + (go * o).abs().sum(-1, keepdim=True)) + (go.abs() * e_o).sum(-1, keepdim=True)
    size = go.norm(dim=-1, keepdim=True).amax(-2, keepdim=True) * V.norm(dim=-1).amax(-1)[..., None, None]
    e_ds = abs(scale) * (p * (r * (dp.abs() + delta.abs()) + e_dp) + 2.0 ** -36 * size * keep)
    dq = ds @ K
    out["dq"] = (dq, e_ds @ K.abs() + (c + 8) * U * (ds.abs() @ K.abs()))
    dk = fold(T(ds) @ q)
    out["dk"] = (dk, fold(T(e_ds) @ q.abs() + (cq + 8) * U * (T(ds).abs() @ q.abs())))
    out["dv"] = (dv, e_dv)
    return out


def check(name, got, want, tiny=1e-36):
    ref, bound = want
    off = (got.double() - ref).abs()
    bad = ~(off <= bound + tiny)
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} beyond their bounds, "
                                 f"worst {float((off / (bound + tiny)).nan_to_num(nan=1e30).max()):.3g} times, first at {bad.nonzero()[0].tolist()}")
