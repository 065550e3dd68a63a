"""The sums over frames and utterances of the sequence operators on integers, in int64: with inputs whose products and partial sums stay
below 2^24, float32 computes every one of them exactly, whatever the order and the grouping -- so a kernel's sum either is the integer or
has lost, doubled or misplaced a term.  A bound on rounding cannot say that: one utterance of thousands is smaller than it.

Layer norm: mean 0 and inv_std 1 are given.  Convolution: linear.  Scan: A = 0 (a state keeps everything), the step sizes are integers
and no softplus.  ``biggest`` of every result is the largest sum of absolute values behind any of its elements, to be held against 2^24.
"""
import numpy as np

EXACT = 1 << 24


def _on(lens, B, T):
    return np.arange(T)[None, :] < (np.full(B, T) if lens is None else np.clip(lens, 0, T))[:, None]


def layer_norm_sums(x, dy, lens=None):
    """dict of dgamma, dbeta and biggest."""
    on = _on(lens, *x.shape[:2])[..., None]
    x, dy = np.where(on, x, 0), np.where(on, dy, 0)
    return {"dgamma": (dy * x).sum((0, 1)), "dbeta": dy.sum((0, 1)), "biggest": int(np.abs(dy * x).sum((0, 1)).max())}


def causal_conv_sums(x, taps, dy, lens=None):
    """dict of dweight, dbias and biggest."""
    B, T, D = x.shape
    on = _on(lens, B, T)[..., None]
    dy, xp = np.where(on, dy, 0), np.concatenate([np.zeros((B, taps - 1, D), np.int64), np.where(on, x, 0)], 1)
    terms = [dy * xp[:, k:k + T] for k in range(taps)]
    return {"dweight": np.stack([t.sum((0, 1)) for t in terms]), "dbias": dy.sum((0, 1)), "biggest": int(max(np.abs(t).sum((0, 1)).max() for t in terms))}


def scan(u, dt, Bm, Cm, D, state, dy, dlast, lens=None):
    """dict of every result of the scan and its backward pass with A = 0, and biggest; Bm, Cm (B, T, G, N)."""
    Bn, T, ch = u.shape
    G, N = Bm.shape[2:]
    on = _on(lens, Bn, T)
    o3 = on[..., None]
    u, dt, dy = (np.where(o3, v, 0) for v in (u, dt, dy))
    bm, cm = (np.where(on[..., None, None], np.repeat(m, ch // G, axis=2), 0) for m in (Bm, Cm))
    dtu = dt * u

    def passes(dtu, bm, cm, state, dy, dlast, f):
        after = state[:, None] + np.cumsum(dtu[..., None] * bm, 1)                               # f: sizes or values
        before = np.concatenate([state[:, None], after[:, :-1]], 1)
        later = dlast[:, None] + np.cumsum((cm * dy[..., None])[:, ::-1], 1)[:, ::-1]            # dh: the frame's own and all later ones'
        groups = lambda v: v.reshape(Bn, T, G, ch // G, N).sum(3)                               # noqa: E731
        ddtu = (later * bm).sum(-1)
        dx = f(u) * ddtu
        return {"y": (after * cm).sum(-1) + f(D) * f(u), "state": after[:, -1], "du": f(dt) * ddtu + dy * f(D), "ddelta": dx,
                "ddelta_bias": dx.sum((0, 1)), "dA": (f(dt)[..., None] * later * before).sum((0, 1)), "dD": (dy * f(u)).sum((0, 1)),
                "dB": groups(later * dtu[..., None]), "dC": groups(after * dy[..., None]), "dstate": later[:, 0]}
    out = passes(dtu, bm, cm, state, dy, dlast, lambda v: v)
    sizes = passes(*(np.abs(v) for v in (dtu, bm, cm, state, dy, dlast)), np.abs)
    out = {k: (np.where(o3, v, 0) if k in ("y", "du", "ddelta") else (np.where(on[..., None, None], v, 0) if k in ("dB", "dC") else v)) for k, v in out.items()}
    out["biggest"] = int(max(v.max() for v in sizes.values()))
    return out
