"""Layer norm, the short causal convolution and the selective scan restated in float64, with a running bound of the error that a float32
evaluation of the same formulas can make.

Every quantity is an ``R``: its value and a bound of the absolute error of its float32 counterpart, to first order.  An operation
passes its operands' errors on through its derivative and adds its own rounding, U = 2^-24 of the result's size per float32 operation
(fused or regrouped forms round less often); a sum over an axis adds ``DEPTH`` roundings of the sum of the sizes, more than any of
the kernels' summation trees is deep (a sum over all frames as many as it has terms); hardware exp2 / reciprocal and their like are taken as 4 U.  Tests compare |got - v| with
2 e (operations grouped otherwise) plus half a step of the result's type.
"""
import numpy as np

U = 2.0 ** -24
DEPTH = 64
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}
_TINY = 1e-38              # float32's smallest normal number: what is below may be flushed


class R(object):
    __array_ufunc__ = None

    def __init__(self, v, e=None):
        self.v = np.asarray(v, dtype=np.float64)
        self.e = np.zeros_like(self.v) if e is None else np.broadcast_to(e, self.v.shape)

    def _round(self, v, e, n=1):
        return R(v, e + n * U * np.abs(v) + np.where((v != 0) | (e > 0), _TINY, 0.0))        # (exact zeros stay exact)

    def __add__(self, o):
        o = o if isinstance(o, R) else R(o)
        return self._round(self.v + o.v, self.e + o.e)

    def __sub__(self, o):
        return self + (-(o if isinstance(o, R) else R(o)))

    def __rsub__(self, o):
        return R(o) - self

    def __neg__(self):
        return R(-self.v, self.e)

    def __mul__(self, o):
        o = o if isinstance(o, R) else R(o)
        return self._round(self.v * o.v, np.abs(self.v) * o.e + np.abs(o.v) * self.e)

    __radd__, __rmul__ = __add__, __mul__

    def __getitem__(self, k):
        return R(self.v[k], self.e[k])

    def sum(self, axis):
        return R(self.v.sum(axis), self.e.sum(axis) + DEPTH * U * np.abs(self.v).sum(axis))

    def sum_frames(self):
        """Over utterances and frames, which a lane may add one after the other."""
        n = max(DEPTH, self.v.shape[0] * self.v.shape[1])
        return R(self.v.sum((0, 1)), self.e.sum((0, 1)) + n * U * np.abs(self.v).sum((0, 1)))

    def exp(self):
        v = np.exp(self.v)               # far below float32's range both are zero
        return R(v, v * (self.e + 3 * U * np.abs(self.v) + 4 * U) + np.where(self.v > -200, _TINY, 0.0))

    def sigmoid(self):
        v = np.where(self.v >= 0, 1 / (1 + np.exp(-np.abs(self.v))), np.exp(-np.abs(self.v)) / (1 + np.exp(-np.abs(self.v))))
        return R(v, v * (1 - v) * (self.e + 3 * U * np.abs(self.v)) + 12 * U * v + _TINY)

    def softplus(self):
        v = np.maximum(self.v, 0) + np.log1p(np.exp(-np.abs(self.v)))
        s = self.sigmoid().v
        return R(v, s * (self.e + 3 * U * np.abs(self.v)) + 20 * U * v + _TINY)

    def rsqrt(self):
        v = self.v ** -0.5
        return R(v, 0.5 * v / self.v * self.e + 6 * U * v)


def stack(rs, axis):
    return R(np.stack([r.v for r in rs], axis), np.stack([r.e for r in rs], axis))


def where(on, r):
    """r where `on`, an exact zero elsewhere."""
    return R(np.where(on, r.v, 0.0), np.where(on, r.e, 0.0))


def valid(lens, B, T):
    lens = np.full(B, T) if lens is None else np.clip(np.asarray(lens), 0, T)
    return np.arange(T)[None, :] < lens[:, None]


def _clean(x, on):
    return R(np.where(on, np.asarray(x, np.float64), 0.0))


# ------------------------------------------------------------------------------------------------------------------ layer norm
def layer_norm(x, gamma, beta, eps, lens=None, dy=None):
    """dict of y, mean, inv_std and, with dy, dx, dgamma, dbeta."""
    x = np.asarray(x, np.float64)
    B, T, D = x.shape
    on = valid(lens, B, T)[..., None]
    gamma = np.ones(D) if gamma is None else gamma
    beta = np.zeros(D) if beta is None else beta
    x = _clean(x, on)
    mean = x.sum(-1)[..., None] * (1.0 / D)
    xc = x - mean
    inv = ((xc * xc).sum(-1)[..., None] * (1.0 / D) + eps).rsqrt()
    xhat = xc * inv
    out = {"y": where(on, xhat * gamma + beta), "mean": where(on, mean)[..., 0], "inv_std": where(on, inv)[..., 0]}
    if dy is not None:
        # mean and inv_std are read back as the forward pass rounded them, so their errors are in
        dy = _clean(dy, on)
        g = dy * gamma
        c0, c1 = g.sum(-1)[..., None] * (1.0 / D), (g * xhat).sum(-1)[..., None] * (1.0 / D)
        out["dx"] = where(on, inv * (g - c0 - xhat * c1))
        out["dgamma"] = where(on, dy * xhat).sum_frames()
        out["dbeta"] = dy.sum_frames()
    return out


# ------------------------------------------------------------------------------------------------------ short causal convolution
def causal_conv(x, weight, bias=None, state=None, lens=None, activation="silu", dy=None):
    """dict of y, state and, with dy, dx, dweight, dbias, dstate."""
    x = np.asarray(x, np.float64)
    B, T, D = x.shape
    K = len(weight)
    w = np.asarray(weight, np.float64)
    on = valid(lens, B, T)
    n = on.sum(1)
    past = np.zeros((B, K - 1, D)) if state is None else np.asarray(state, np.float64)
    xp = np.concatenate([past, np.where(on[..., None], x, 0.0)], 1)             # frame t at t + K - 1
    pre = stack([sum((R(xp[:, t + k]) * w[k] for k in range(K)), R(np.zeros((B, D)) if bias is None else np.broadcast_to(bias, (B, D))))
                 for t in range(T)], 1) if T else R(np.zeros((B, 0, D)))
    sg = pre.sigmoid()
    out = {"y": where(on[..., None], pre * sg if activation == "silu" else pre),
           "state": R(np.stack([xp[b, n[b]:n[b] + K - 1] for b in range(B)]) if B else np.zeros((0, K - 1, D)))}
    if dy is not None:
        d = _clean(dy, on[..., None])
        if activation == "silu":
            d = where(on[..., None], d * (sg * (1 + pre * (1 - sg))))
        dxp = []
        for s in range(T + K - 1):                                               # frame s - (K - 1)
            parts = [d[:, s - k] * w[k] for k in range(K) if 0 <= s - k < T]
            dxp.append(sum(parts[1:], parts[0]) if parts else R(np.zeros((B, D))))
        dxp = stack(dxp, 1) if dxp else R(np.zeros((B, 0, D)))
        out["dx"] = where(on[..., None], dxp[:, K - 1:])
        out["dstate"] = dxp[:, :K - 1]
        out["dweight"] = stack([(d * xp[:, k:k + T]).sum_frames() for k in range(K)], 0)
        out["dbias"] = d.sum_frames()
    return out


# ------------------------------------------------------------------------------------------------------------------ selective scan
def selective_scan(u, delta, A, Bm, Cm, D=None, z=None, delta_bias=None, state=None, lens=None, softplus=True, dy=None, dlast=None):
    """dict of y, state and, with dy, du, ddelta, dz, dB, dC, dA, dD, ddelta_bias, dstate.  Bm, Cm: (B, T, G, N)."""
    Bn, T, ch = np.shape(u)
    N = np.shape(A)[1]
    G = np.shape(Bm)[2]
    on = valid(lens, Bn, T)
    o3, o4 = on[..., None], on[..., None, None]
    A = np.asarray(A, np.float64)
    Dv = np.zeros(ch) if D is None else np.asarray(D, np.float64)
    u = _clean(u, o3)
    x = _clean(delta, o3) + (np.zeros(ch) if delta_bias is None else delta_bias)
    dt = where(o3, x.softplus() if softplus else x)
    bm, cm = (_clean(np.repeat(np.asarray(m, np.float64), ch // G, axis=2), o4) for m in (Bm, Cm))
    a = (dt[..., None] * A).exp()
    dtu = dt * u
    h = R(np.zeros((Bn, ch, N)) if state is None else state)
    hs, es = [], []
    for t in range(T):
        e = a[:, t] * h
        new = e + dtu[:, t][..., None] * bm[:, t]
        keep = on[:, t][:, None, None]
        h = R(np.where(keep, new.v, h.v), np.where(keep, new.e, h.e))
        hs.append(h)
        es.append(e)
    out = {"state": h}
    if T == 0:
        z3 = R(np.zeros((Bn, 0, ch)))
        hs, es = R(np.zeros((Bn, 0, ch, N))), R(np.zeros((Bn, 0, ch, N)))
    else:
        z3, hs, es = None, stack(hs, 1), stack(es, 1)
    ys = (hs * cm).sum(-1) + u * Dv
    if z is not None:
        zz = _clean(z, o3)
        sg = zz.sigmoid()
        out["y"] = where(o3, ys * (zz * sg))
    else:
        out["y"] = where(o3, ys)
    if dy is None:
        return out
    g = _clean(dy, o3)
    if z is not None:
        out["dz"] = where(o3, g * ys * sg * (1 + zz * (1 - sg)))
        g = g * (zz * sg)
    carry = R(np.zeros((Bn, ch, N)) if dlast is None else dlast)
    dhs = [None] * T
    for t in range(T - 1, -1, -1):
        dh = cm[:, t] * g[:, t][..., None] + carry
        keep = on[:, t][:, None, None]
        back = a[:, t] * dh
        dhs[t] = where(keep, dh)
        carry = R(np.where(keep, back.v, carry.v), np.where(keep, back.e, carry.e))
    dh = stack(dhs, 1) if T else R(np.zeros((Bn, 0, ch, N)))
    de = dh * es
    ddtu = (dh * bm).sum(-1)
    dx = (de * A).sum(-1) + u * ddtu
    if softplus:
        dx = dx * x.sigmoid()
    dx = where(o3, dx)
    split = lambda r: R(r.v.reshape(Bn, T, G, ch // G, N), r.e.reshape(Bn, T, G, ch // G, N)).sum(3)      # noqa: E731
    out.update(du=where(o3, dt * ddtu + g * Dv), ddelta=dx, ddelta_bias=dx.sum_frames(), dA=(de * dt[..., None]).sum_frames(),
               dD=(g * u).sum_frames(), dB=split(dh * dtu[..., None]), dC=split(where(o4, hs * g[..., None])), dstate=carry)
    return out
