"""oracle/sequence_oracle.py against its definitions: gradients by central differences, padding and carried states against plain loops,
and the running error bound against float32 evaluations of the same formulas."""
import numpy as np
import pytest

from oracle import sequence_oracle as S


def _rng(*key):
    return np.random.default_rng(list(key))


def _difference(f, x, i, step=1e-4):
    """Five-point central difference: its error is of order step^4 (a negative step size makes the scan grow fast, and the three-point
    form's step^2 error with it)."""
    def at(k):
        v = x.copy()
        v.flat[i] += k * step
        return f(v)
    return (8 * (at(1) - at(-1)) - (at(2) - at(-2))) / (12 * step)


def _check_gradients(run, leaves, names, dy, rng, extra=None):
    """run(leaves, dy) -> outputs; the loss is sum(y dy) (+ sum(state extra))."""
    base = run(leaves, dy)

    def loss(**over):
        o = run({**leaves, **over}, None)
        return (o["y"].v * dy).sum() + (0 if extra is None else (o["state"].v * extra).sum())
    for leaf, grad in names.items():
        x = leaves[leaf]
        for i in rng.choice(x.size, size=min(12, x.size), replace=False):
            want = _difference(lambda v: loss(**{leaf: v}), x, i)
            assert abs(base[grad].v.flat[i] - want) <= 1e-6 * max(1.0, abs(want)), (leaf, i)


@pytest.mark.parametrize("lens", [None, [5, 0, 3]])
def test_layer_norm_gradients(lens):
    rng = _rng(1, 0 if lens is None else 1)
    leaves = dict(x=rng.normal(size=(3, 5, 7)) + 0.5, gamma=1 + 0.2 * rng.normal(size=7), beta=rng.normal(size=7))
    _check_gradients(lambda v, dy: S.layer_norm(v["x"], v["gamma"], v["beta"], 1e-3, lens, dy), leaves,
                     {"x": "dx", "gamma": "dgamma", "beta": "dbeta"}, rng.normal(size=(3, 5, 7)), rng)


@pytest.mark.parametrize("taps", [1, 2, 4])
@pytest.mark.parametrize("activation", ["silu", "linear"])
@pytest.mark.parametrize("lens", [None, [6, 0, 2]])
def test_causal_conv_gradients(taps, activation, lens):
    rng = _rng(2, taps, len(activation), 0 if lens is None else 1)
    leaves = dict(x=rng.normal(size=(3, 6, 4)), weight=rng.normal(size=(taps, 4)), bias=rng.normal(size=4), state=rng.normal(size=(3, taps - 1, 4)))
    names = {"x": "dx", "weight": "dweight", "bias": "dbias"}
    if taps > 1:
        names["state"] = "dstate"
    _check_gradients(lambda v, dy: S.causal_conv(v["x"], v["weight"], v["bias"], v["state"], lens, activation, dy), leaves, names,
                     rng.normal(size=(3, 6, 4)), rng)


def test_causal_conv_in_pieces_is_the_whole():
    rng = _rng(3)
    x, w = rng.normal(size=(2, 9, 3)), rng.normal(size=(4, 3))
    whole = S.causal_conv(x, w)
    first = S.causal_conv(x[:, :2], w)
    rest = S.causal_conv(x[:, 2:], w, state=first["state"].v)
    np.testing.assert_allclose(np.concatenate([first["y"].v, rest["y"].v], 1), whole["y"].v, rtol=0, atol=1e-12)
    np.testing.assert_array_equal(rest["state"].v, x[:, -3:])


@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("softplus", [False, True])
@pytest.mark.parametrize("lens", [None, [5, 0, 2]])
def test_selective_scan_gradients(groups, gated, softplus, lens):
    rng = _rng(4, groups, gated, softplus, 0 if lens is None else 1)
    B, T, ch, N = 3, 5, 4, 3
    n = lambda *s: rng.normal(size=s)                                            # noqa: E731
    leaves = dict(u=n(B, T, ch), delta=0.5 * n(B, T, ch), A=-np.exp(n(ch, N)), Bm=n(B, T, groups, N), Cm=n(B, T, groups, N), D=n(ch),
                  delta_bias=n(ch) - 1, state=n(B, ch, N))
    if not softplus:         # step sizes themselves: positive (negative ones let the loss grow to 1e17, where differences say nothing)
        leaves.update(delta=np.abs(leaves["delta"]), delta_bias=np.abs(leaves["delta_bias"]) / 4)
    names = {"u": "du", "delta": "ddelta", "A": "dA", "Bm": "dB", "Cm": "dC", "D": "dD", "delta_bias": "ddelta_bias", "state": "dstate"}
    if gated:
        leaves["z"] = n(B, T, ch)
        names["z"] = "dz"
    extra = n(B, ch, N)
    _check_gradients(lambda v, dy: S.selective_scan(lens=lens, softplus=softplus, dy=dy, dlast=extra, **v), leaves, names, n(B, T, ch), rng, extra)


def test_selective_scan_is_its_recurrence():
    rng = _rng(5)
    B, T, ch, N = 2, 7, 3, 2
    u, delta, A = rng.normal(size=(B, T, ch)), rng.normal(size=(B, T, ch)), -np.exp(rng.normal(size=(ch, N)))
    Bm, Cm = rng.normal(size=(B, T, 1, N)), rng.normal(size=(B, T, 1, N))
    got = S.selective_scan(u, delta, A, Bm, Cm)
    for b in range(B):
        for c in range(ch):
            h = np.zeros(N)
            for t in range(T):
                dt = np.log1p(np.exp(delta[b, t, c]))
                h = np.exp(dt * A[c]) * h + dt * u[b, t, c] * Bm[b, t, 0]
                assert abs(got["y"].v[b, t, c] - h @ Cm[b, t, 0]) < 1e-12
            np.testing.assert_allclose(got["state"].v[b, c], h, rtol=0, atol=1e-12)


def test_the_error_bound_covers_a_float32_evaluation():
    f = np.float32
    rng = _rng(6)
    B, T, ch, N = 1, 40, 5, 4
    u, delta = (rng.normal(size=(B, T, ch)).astype(f) for _ in range(2))
    A = -np.exp(rng.normal(size=(ch, N))).astype(f)
    Bm, Cm = (rng.normal(size=(B, T, 1, N)).astype(f) for _ in range(2))
    want = S.selective_scan(u, delta, A, Bm, Cm)
    h = np.zeros((ch, N), f)
    worst = 0.0
    for t in range(T):
        dt = np.log1p(np.exp(delta[0, t])).astype(f)
        h = (np.exp((dt[:, None] * A).astype(f)) * h).astype(f) + (dt * u[0, t])[:, None] * Bm[0, t]
        y = (h * Cm[0, t]).sum(-1, dtype=f)
        worst = max(worst, (np.abs(y - want["y"].v[0, t]) / want["y"].e[0, t]).max())
    assert 0 < worst < 2                       # inside the bound, and the bound is no more than some tens of times too wide
    assert (want["y"].e < 1e-4 * np.abs(want["y"].v).max()).all()
