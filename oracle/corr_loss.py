"""Losses over the all-pairs correlation (modules/corr.py:63-71's logits) in
float64: softmax cross entropy against sparse targets and distillation from a
teacher's top logits, with their gradients."""
import numpy as np


def targets(idx, logits, temperature):
    """Weights pi (E,P,K) of the targets and the rows that have any."""
    on = idx >= 0
    if logits is None:
        pi = on.astype(np.float64)
    else:
        t = np.where(on, logits.astype(np.float64) / temperature, -np.inf)
        on = on & (t > -np.inf)
        top = np.where(on.any(-1, keepdims=True), t.max(-1, keepdims=True), 0.0)
        e = np.where(on, np.exp(np.where(on, t, 0.0) - top), 0.0)
        pi = e / np.maximum(e.sum(-1, keepdims=True), 1e-300)
    return pi, on.any(-1)


def corr_loss(fmap1, fmap2, f1, f2, idx, logits=None, scale=1.0 / 16, temperature=1.0, g=None):
    """idx (E,P,K); logits (E,P,K) or None (K = 1, weight 1) -> loss (E,P); with
    the upstream gradient g (E,P) also df1, df2, and for error bounds the same
    sums over absolute values: per edge |ds|, p and the row's lse."""
    T = temperature
    pi, used = targets(idx, logits, T)
    E, P, K = idx.shape
    loss = np.zeros((E, P))
    d1, d2 = np.zeros(fmap1.shape), np.zeros(fmap2.shape)
    per_edge = []
    for e in range(E):
        a, b = fmap1[f1[e]].astype(np.float64), fmap2[f2[e]].astype(np.float64)
        s = (a @ b.T) * (scale / T)
        top = s.max(1, keepdims=True)
        lse = top[:, 0] + np.log(np.exp(s - top).sum(1))
        p = np.exp(s - lse[:, None])
        q = np.zeros_like(s)
        np.add.at(q, (np.arange(P)[:, None], np.maximum(idx[e], 0)), pi[e])
        with np.errstate(divide="ignore", invalid="ignore"):
            ent = np.where(pi[e] > 0, pi[e] * np.log(pi[e]), 0.0).sum(1)
        loss[e] = np.where(used[e], T * T * (ent + lse - (q * s).sum(1)), 0.0)
        if g is not None:
            ds = np.where(used[e][:, None], (p - q) * (g[e] * T * scale)[:, None], 0.0)
            d1[f1[e]] += ds @ b
            d2[f2[e]] += ds.T @ a
            per_edge.append((ds, p, q, lse))
    return (loss, d1, d2, per_edge) if g is not None else loss
