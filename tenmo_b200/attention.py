"""Attention over heads without a score matrix in memory: the chain Q.matmul(K^T) -> softmax -> matmul(V) of the reference's
attention tests (tests/test_attn_matmul.mojo:194-259) as one operator with its gradient."""
from __future__ import annotations

import math

import torch

from .lib import make_heads
from .tensor import BACKWARD_ATTENTION, Ancestry, NDBuffer, Tensor, handle, panic


class Attention:
    """``attention(q, k, v, q_lengths, k_lengths)`` with q (B, H, Sq, D), k and v (B, Hkv, Sk, D) and H a multiple of Hkv, or all
    of rank 3, (B, S, D), for one head each.  ``scale`` defaults to 1 / sqrt(D); ``causal`` hides key j from row i when
    j > i + Sk - Sq; the lengths are int32 labels-like tensors of shape (B,) (``Tensor.labels(values, np.int32)``): keys / rows
    from the length on take no part.  Transposed views (heads inside the row) are read in place when the last axis is
    contiguous."""

    def __init__(self, causal: bool = False, scale: float | None = None):
        self.causal, self.scale = bool(causal), scale
        self.training = True

    def __call__(self, q: Tensor, k: Tensor, v: Tensor, q_lengths: Tensor | None = None, k_lengths: Tensor | None = None) -> Tensor:
        rank = len(q.shape())
        if rank not in (3, 4) or len(k.shape()) != rank or k.shape() != v.shape():
            panic("Attention: q", q.shape(), "k", k.shape(), "v", v.shape(), "are not (B, H, S, D) or (B, S, D)")
        four = [_rank4(t.buffer) for t in (q, k, v)]
        (B, H, Sq, D), (Bk, Hkv, Sk, Dk) = four[0].shape, four[1].shape
        if Bk != B or Dk != D or Hkv < 1 or H % Hkv:
            panic("Attention: q", q.shape(), "and k", k.shape(), "do not fit")
        lengths = []
        for name, t in (("q_lengths", q_lengths), ("k_lengths", k_lengths)):
            if t is not None and (t.shape() != (B,) or t.buffer.storage.dtype != torch.int32):
                panic("Attention:", name, "must be int32 of shape", (B,), "got", t.shape())
            lengths.append(t.buffer.contiguous() if t is not None else None)
        out, stats = NDBuffer.empty((B, H, Sq, D)), NDBuffer.empty((B, H, Sq, 2))
        a = dict(q=four[0], k=four[1], v=four[2], o=out, stats=stats, shape=(B, H, Hkv, Sq, Sk, D),
                 scale=1.0 / math.sqrt(D) if self.scale is None else float(self.scale), causal=self.causal, lengths=lengths)
        handle().attention_fwd(a["shape"], *(_heads(a[n]) for n in "qkvo"), stats.data_ptr(), a["scale"], **_mask(a))
        t = Tensor(out.reshape(q.shape()))
        if self.training and (q.requires_grad or k.requires_grad or v.requires_grad):
            t.requires_grad = True
            t.ancestry = Ancestry(BACKWARD_ATTENTION, [q, k, v], arg=a)
        return t

    def parameters(self):
        return []


def _rank4(b: NDBuffer) -> NDBuffer:
    if b.rank() == 3:
        b = b.unsqueeze(1)
    return b if b.strides[3] == 1 or b.shape[3] == 1 else b.contiguous()


def _heads(b: NDBuffer):
    return make_heads(b.data_ptr(), b.strides[:3])


def _mask(a):
    return dict(causal=a["causal"], q_lengths=a["lengths"][0].data_ptr() if a["lengths"][0] is not None else 0,
                k_lengths=a["lengths"][1].data_ptr() if a["lengths"][1] is not None else 0)


def attention_backward(output: Tensor, retain_graph: bool):
    """dq, dk and dv from the upstream gradient and the two numbers per row that the forward pass kept."""
    a = output.ancestry.arg
    B, H, Hkv, Sq, Sk, D = a["shape"]
    go = output.gradbox.reshape((B, H, Sq, D))
    grads = [NDBuffer.empty((B, H, Sq, D)), NDBuffer.empty((B, Hkv, Sk, D)), NDBuffer.empty((B, Hkv, Sk, D))]
    handle().attention_bwd(a["shape"], *(_heads(a[n]) for n in "qkvo"), a["stats"].data_ptr(), _heads(go),
                           *(_heads(g) for g in grads), a["scale"], **_mask(a))
    touched = []
    for parent, g in zip(output.ancestry.parents, grads):
        if parent.requires_grad:
            parent.update_grad(g.reshape(parent.shape()))
            touched.append(parent)
    if not retain_graph:
        output.gradbox.fill(0.0)
    return touched
