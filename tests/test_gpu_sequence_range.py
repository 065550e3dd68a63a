"""The sequence operators where values reach the ends of float32's range: scans that grow, decays of the type's lowest value, and
infinities or NaN beside frames that are padding."""
import numpy as np
import pytest

from oracle import sequence_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from ip_avsr_amd.custom import sequence
    return sequence


def _torch():
    import torch
    return torch


def _near(name, got, want, dtype="float32"):
    """Finite, and within twice the oracle's bound and half a step of the type (the oracle's header says why)."""
    g = got.double().cpu().numpy()
    assert g.shape == want.v.shape, (name, g.shape, want.v.shape)
    assert np.isfinite(g).all(), "%s: %d values are not finite, the first at %s" % (name, (~np.isfinite(g)).sum(), np.argwhere(~np.isfinite(g))[0])
    tol = 2 * want.e + O.HALF_STEP[dtype] * np.abs(want.v) * 1.01 + 1e-37
    off = np.abs(g - want.v)
    worst = (off / tol).max() if off.size else 0.0
    assert worst <= 1.0, "%s: %.2f times the bound at %s" % (name, worst, np.unravel_index((off / tol).argmax(), off.shape))


def _dev(x, dtype="float32"):
    """(float64 values exact in `dtype`, device tensor)"""
    torch = _torch()
    t = torch.tensor(np.asarray(x, np.float32), device="cuda").to(getattr(torch, dtype))
    return t.double().cpu().numpy(), t


def _both(pairs):
    return {k: p[0] for k, p in pairs.items()}, {k: p[1] for k, p in pairs.items()}


def _check_scan(S, v, t, dy, dl, lens, dtype, softplus):
    torch = _torch()
    want = O.selective_scan(dy=dy[0], dlast=dl[0], lens=lens, softplus=softplus, **v)
    for name in ("y", "state", "du", "ddelta", "dA", "dB", "dC", "dstate"):
        assert np.abs(want[name].v).max() < 1e38, name                # (the case itself stays inside the type)
    more = dict(lens=None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda"), softplus=softplus)
    y, state, saved = S.selective_scan_forward(save=True, **t, **more)
    _near("y", y, want["y"], dtype)
    _near("state", state, want["state"])
    g = S.selective_scan_backward(dy[1], saved=saved, dlast=dl[1], **t, **more)
    for name in ("du", "ddelta", "dB", "dC"):
        _near(name, g[name], want[name], dtype)
    for name in ("dA", "dD", "ddelta_bias", "dstate"):
        _near(name, g[name], want[name])
    return want


# states, channels, groups: 1, 2, 4 and 8 states per lane; 300 x 8: several workgroups along the channels
GROWTH = [(3, 70, 1), (8, 40, 2), (16, 24, 1), (8, 300, 1), (32, 12, 1)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("N,D,G", GROWTH)
def test_a_scan_that_grows_past_float32_within_a_piece_of_the_time_axis(S, dtype, softplus, N, D, G):
    """Two utterances, long enough for a time axis in pieces (of 32 or 64 frames).  The first starts from states of 1e-18 and grows by
    e^120 within 32 frames, the gradient of its last state, 1e-30, likewise on the way back: every h and dh is a float32 number, e^120 is
    none.  The second grows by e^3.75 a frame throughout, from zeros: its input comes in the last 20 frames, its gradient leaves in
    the first 10."""
    rng = np.random.default_rng([41, N, D, softplus])
    B, T, up = 2, 256, 3.75
    lens = [T, T - 3]
    assert S._lib.load().adn_op_selective_scan_workspace(B, T, D, N, G, 0) > 0      # pieces
    logs = np.full((B, T), 1e-3)                       # log of the growth of a frame
    logs[0, 64:96] = up
    logs[1] = up
    if softplus:       # dt = softplus(delta), A = 1 (to 0.1 %)
        delta, sign = np.log(np.expm1(logs)), 1.0
    else:              # dt < 0, A = -1
        delta, sign = -logs, -1.0
    u = rng.normal(size=(B, T, D))
    u[0, :192] = 0
    u[1, :T - 3 - 20] = 0
    dy = rng.normal(size=(B, T, D))
    dy[0, 48:] = 0                                      # (behind the growth: the gradient of the last state alone)
    dy[1, 10:] = 0
    state, dlast = 1e-18 * rng.normal(size=(B, D, N)), 1e-30 * rng.normal(size=(B, D, N))
    state[1] = dlast[1] = 0
    v, t = _both(dict(u=_dev(u, dtype), delta=_dev(np.broadcast_to(delta[..., None], (B, T, D)), dtype), A=_dev(sign * (1 + 1e-3 * rng.uniform(-1, 1, (D, N)))),
                      Bm=_dev(rng.normal(size=(B, T, G, N)), dtype), Cm=_dev(rng.normal(size=(B, T, G, N)), dtype), D=_dev(rng.normal(size=D)), state=_dev(state)))
    want = _check_scan(S, v, t, _dev(dy, dtype), _dev(dlast), lens, dtype, softplus)
    # it grew, and the bound still says something
    assert np.abs(want["state"].v).max() > 1e20 and np.abs(want["dstate"].v).max() > 1e15
    assert np.median(want["state"].e / np.abs(want["state"].v)) < 1e-2


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("T,N,D,lens", [(13, 5, 20, [13, 6]), (3, 3, 70, [1, 3]), (21, 16, 24, [9, 21]), (150, 8, 40, [150, 77]), (9, 32, 12, [5, 7])])
def test_a_scan_with_decays_of_the_lowest_float32(S, T, N, D, lens, softplus):
    """A = -3.4e38, a state that keeps nothing, also over frames that are padding and over steps of size 0; and single frames."""
    torch = _torch()
    rng = np.random.default_rng([42, T, N, D])
    a = -np.exp(rng.normal(size=(D, N)))
    a[rng.uniform(size=(D, N)) < 0.4] = np.finfo(np.float32).min
    delta = rng.normal(size=(2, T, D)) if softplus else rng.uniform(0.1, 1, size=(2, T, D))
    v, t = _both(dict(u=_dev(rng.normal(size=(2, T, D))), delta=_dev(delta), A=_dev(a), Bm=_dev(rng.normal(size=(2, T, 1, N))),
                      Cm=_dev(rng.normal(size=(2, T, 1, N))), D=_dev(rng.normal(size=D)), state=_dev(rng.normal(size=(2, D, N)))))
    want = _check_scan(S, v, t, _dev(rng.normal(size=(2, T, D))), _dev(rng.normal(size=(2, D, N))), lens, "float32", softplus)
    low = v["A"] < -1e38
    assert np.abs(want["dA"].v[low]).max() == 0 and np.abs(want["dA"].v[~low]).max() > 0
    # a frame of step size 0 (a softplus far below float32's range, or the size itself) leaves every state as it is
    h = t["state"].clone()
    nothing = torch.full((2, D), -200.0 if softplus else 0.0, device="cuda")
    S.selective_scan_step(t["u"][:, 0], nothing, t["A"], t["Bm"][:, 0], t["Cm"][:, 0], h, softplus=softplus)
    assert torch.equal(h, t["state"])
    one = {k: x[:, :1] for k, x in t.items() if k in ("u", "Bm", "Cm")}
    assert torch.equal(S.selective_scan_forward(delta=nothing[:, None], A=t["A"], state=t["state"], softplus=softplus, **one)[1], t["state"])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("D", [3, 8, 130])
def test_frames_before_padding_stay_out_of_the_weight_gradient_of_padding(S, dtype, D):
    """An infinity in the last frame of an utterance reaches the newest tap's gradient alone (the frames that the older taps would
    take it to are padding), and what the history of an utterance of length 0 holds reaches none."""
    torch = _torch()
    rng = np.random.default_rng([43, D])
    (_, x), (_, dy), (_, st) = (_dev(rng.normal(size=s), dtype) for s in ((4, 6, D), (4, 6, D), (4, 2, D)))
    (_, w), (_, b) = _dev(rng.normal(size=(3, D))), _dev(rng.normal(size=D))
    lens = torch.tensor([4, 6, 0, 5], dtype=torch.int32, device="cuda")
    for act in ("linear", "silu"):
        dx, dw, db, ds = S.causal_conv_backward(dy, x, w, b, state=st, lens=lens, activation=act)
        odd = st.clone()
        odd[2, 0], odd[2, 1] = float("nan"), float("inf")
        for got, want in zip(S.causal_conv_backward(dy, x, w, b, state=odd, lens=lens, activation=act), (dx, dw, db, ds)):
            assert torch.equal(got, want)
    far = x.clone()
    far[0, 3] = float("inf")
    dx, dw, db, _ = S.causal_conv_backward(dy, x, w, b, state=st, lens=lens, activation="linear")
    dx2, dw2, db2, _ = S.causal_conv_backward(dy, far, w, b, state=st, lens=lens, activation="linear")
    assert torch.equal(dw[:2], dw2[:2]) and torch.equal(dx, dx2) and torch.equal(db, db2)
    assert torch.equal(dw2[2], torch.sign(dy[0, 3].float()) * float("inf"))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("T,N,D,lens", [(13, 5, 20, [13, 6]), (5, 3, 70, [1, 3]), (21, 16, 24, [9, 20]), (150, 8, 40, [150, 77]), (9, 32, 12, [5, 7])])
def test_scan_gradients_of_padding_are_zeros_beside_infinities(S, dtype, value, T, N, D, lens):
    """The gradient of the last state, or the first state, is infinite or NaN: frames that are padding still come back as zeros, and the
    other utterance as if alone."""
    torch = _torch()
    rng = np.random.default_rng([44, T, N, D])
    (_, u), (_, delta), (_, z), (_, dy) = (_dev(rng.normal(size=(2, T, D)), dtype) for _ in range(4))
    (_, bm), (_, cm) = (_dev(rng.normal(size=(2, T, N)), dtype) for _ in range(2))
    (_, A), (_, Dv), (_, h), (_, dl) = _dev(-np.exp(rng.normal(size=(D, N)))), _dev(rng.normal(size=D)), _dev(rng.normal(size=(2, D, N))), _dev(rng.normal(size=(2, D, N)))
    more = dict(D=Dv, z=z, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))

    def passes(h, dl):
        y, state, saved = S.selective_scan_forward(u, delta, A, bm, cm, state=h, save=True, **more)
        g = S.selective_scan_backward(dy, u, delta, A, bm, cm, saved, state=h, dlast=dl, **more)
        return dict(y=y, **{k: g[k] for k in ("du", "ddelta", "dz", "dB", "dC")})
    plain = passes(h, dl)
    for bad_h, bad_dl in ((False, True), (True, False)):
        h2, dl2 = h.clone(), dl.clone()
        (h2 if bad_h else dl2)[1] = value
        for name, got in passes(h2, dl2).items():
            assert not got[1, lens[1]:].any(), name
            assert torch.equal(got[0], plain[name][0]), name


def test_refusals_of_bad_statistics_and_of_empty_tensors_with_a_dimension_of_2_31(S):
    torch = _torch()
    x = torch.randn(5, 8, device="cuda")
    _, m, i = S.layer_norm_forward(x)
    for mean, inv in ((None, i), (m, None), (1.0, i), (m[:4], i), (m, i.double()), (m, i.cpu())):
        with pytest.raises(ValueError, match="mean|inv_std"):
            S.layer_norm_backward(x, x, None, mean, inv)
    none = x[:0]
    assert not S.layer_norm_backward(none, none, None, m[:0], i[:0])[1].any()
    # the library's sizes are 32-bit: (2^32 + 1, 0, 1) is not (1, 0, 1)
    far = torch.empty((1 << 32) + 1, 0, 1, device="cuda")
    one = torch.ones(1, 1, device="cuda")
    for fn in (S.layer_norm_forward, lambda v: S.causal_conv_forward(v, one), lambda v: S.selective_scan_forward(v, v, -one, v, v)):
        with pytest.raises(ValueError, match=r"2\^31"):
            fn(far)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("N,D,G", GROWTH)
def test_an_input_that_cancels_a_growth_past_float32(S, dtype, N, D, G):
    """The first utterance's state of 1 is cancelled exactly by its input in frame 64, then the scan grows by e^120: a piece of the time
    axis alone ends in infinities, frame by frame there are zeros.  On the way back the gradient of the last state meets its opposite in
    frame 191, behind a growth by e^120.  The second utterance is an ordinary one."""
    torch = _torch()
    rng = np.random.default_rng([45, N, D])
    B, T, tiny = 2, 256, 2.0 ** -30
    assert S._lib.load().adn_op_selective_scan_workspace(B, T, D, N, G, 0) > 0      # pieces
    delta = np.full((B, T, D), tiny)
    delta[0, 65:97] = delta[0, 159:191] = 3.75
    delta[1] = rng.uniform(0.01, 0.02, (T, D))
    u, dy = rng.normal(size=(B, T, D)), rng.normal(size=(B, T, D))
    bm, cm = rng.normal(size=(B, T, G, N)), rng.normal(size=(B, T, G, N))
    u[0], dy[0], bm[0], cm[0] = 0, 0, 1, 1
    u[0, 64] = -1 / tiny
    dy[0, 191] = -1
    state, dlast = rng.normal(size=(B, D, N)), rng.normal(size=(B, D, N))
    state[0] = dlast[0] = 1
    (_, u), (_, delta), (_, bm), (_, cm), (_, dy) = (_dev(v, dtype) for v in (u, delta, bm, cm, dy))
    (_, A), (_, state), (_, dlast) = _dev(np.ones((D, N))), _dev(state), _dev(dlast)
    y, last, saved = S.selective_scan_forward(u, delta, A, bm, cm, state=state, softplus=False, save=True)
    h = state.clone()
    for t in range(T):
        yt = S.selective_scan_step(u[:, t], delta[:, t], A, bm[:, t], cm[:, t], h, softplus=False)
        assert torch.equal(y[0, t], yt[0]), t
    assert torch.isfinite(h).all() and not h[0].any() and torch.equal(last[0], h[0])
    assert torch.isfinite(y).all() and y[0, :64].any() and not y[0, 64:].any()
    g = S.selective_scan_backward(dy, u, delta, A, bm, cm, saved, state=state, softplus=False, dlast=dlast)
    assert not g["dstate"][0].any() and not g["du"][0, :192].any() and not g["ddelta"][0, :192].any()
    # dh = 1 (to the rounding of 64 factors of 1 + 2^-30) behind frame 191: du = dt sum_n dh B, ddelta = A sum_n dh h = 0
    assert ((g["du"][0, 192:].double() / (tiny * N) - 1).abs() <= (2.0 ** -8 if dtype == "bfloat16" else 64 * 2.0 ** -23)).all() and not g["ddelta"][0, 192:].any()
    assert all(torch.isfinite(v).all() for v in g.values() if v is not None)
    # the other utterance as if alone
    one = [v[1:].contiguous() for v in (u, delta, bm, cm, dy)]
    y1, last1, saved1 = S.selective_scan_forward(one[0], one[1], A, one[2], one[3], state=state[1:], softplus=False, save=True)
    g1 = S.selective_scan_backward(one[4], one[0], one[1], A, one[2], one[3], saved1, state=state[1:], softplus=False, dlast=dlast[1:])
    assert torch.equal(y[1:], y1) and torch.equal(last[1:], last1)
    for name in ("du", "ddelta", "dB", "dC", "dstate"):
        assert torch.equal(g[name][1:], g1[name]), name


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("N,D,G", GROWTH)
def test_a_scan_that_shrinks_below_float32_in_one_piece_and_grows_back_in_another(S, dtype, N, D, G):
    """States of 1e12 shrink by e^-100 within 32 frames, to 4e-32, and grow back later; the gradient of the last state the same on the way
    back (from 1e-10 to 3e33 to 1e-10).  Every h and dh is a float32 number, e^-100 (and e^100) is none."""
    rng = np.random.default_rng([46, N, D])
    B, T = 2, 256
    assert S._lib.load().adn_op_selective_scan_workspace(B, T, D, N, G, 0) > 0      # pieces
    delta = np.full((B, T, D), 2.0 ** -12)
    delta[0, 64:96], delta[0, 160:192] = 3.125, -3.125
    delta[1] = rng.uniform(0.01, 0.02, (T, D))
    u, dy = rng.normal(size=(B, T, D)), rng.normal(size=(B, T, D))
    u[0, :192] = 0
    dy[0] = 0
    state, dlast = rng.normal(size=(B, D, N)), rng.normal(size=(B, D, N))
    state[0], dlast[0] = 1e12 * np.abs(state[0]), 1e-10 * np.abs(dlast[0])
    v, t = _both(dict(u=_dev(u, dtype), delta=_dev(delta, dtype), A=_dev(np.full((D, N), -1.0)), Bm=_dev(rng.normal(size=(B, T, G, N)), dtype),
                      Cm=_dev(rng.normal(size=(B, T, G, N)), dtype), D=_dev(rng.normal(size=D)), state=_dev(state)))
    want = _check_scan(S, v, t, _dev(dy, dtype), _dev(dlast), [T, T - 3], dtype, False)
    for name in ("state", "dstate"):
        assert (np.abs(want[name].e[0] / want[name].v[0]) < 1e-2).mean() > 0.9, name
    assert (np.abs(want["state"].v[0] / v["state"][0] - 1) < 0.2).all()
