"""FP64 restatement of token scores (log probability, entropy, alternatives) and of their gradient."""
import numpy as np


def statistics(x):
    """lse [rows], entropy [rows] and log probabilities [rows, vocab] of f64 logits; -inf entries have none."""
    m = np.max(x, axis=1, keepdims=True)
    base = np.where(np.isneginf(m), 0.0, m)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.exp(x - base)
        s = e.sum(1, keepdims=True)
        lse = base + np.log(s)
        logp = np.where(np.isneginf(x), -np.inf, x - lse)
        p = np.exp(logp)
        entropy = -np.where(p > 0, p * logp, 0.0).sum(1)
    return lse[:, 0], entropy, logp


def scores(x, target, top):
    """(logp, entropy, lse, top_id, top_logp); a target of -1 has log probability 0."""
    x = np.asarray(x, dtype=np.float64)
    lse, entropy, logp = statistics(x)
    rows = np.arange(len(x))
    got = np.where(target >= 0, logp[rows, np.maximum(target, 0)], 0.0)
    order = np.argsort(-np.where(np.isnan(x), -np.inf, x), axis=1, kind="stable")[:, :top]
    return got, entropy, lse, order, np.take_along_axis(logp, order, 1)


def gradient(x, target, d_logp, d_entropy):
    """d logits of sum(d_logp * logp + d_entropy * entropy)."""
    x = np.asarray(x, dtype=np.float64)
    lse, entropy, logp = statistics(x)
    p = np.where(np.isneginf(x), 0.0, np.exp(logp))
    a = np.where(target >= 0, d_logp, 0.0)[:, None]
    g = -p * (a + d_entropy[:, None] * (np.where(p > 0, logp, 0.0) + entropy[:, None]))
    rows = np.arange(len(x))
    g[rows, np.maximum(target, 0)] += a[:, 0]
    return g
