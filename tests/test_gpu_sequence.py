"""The sequence operators (ip_avsr_amd/custom/sequence.py) on the GPU against oracle/sequence_oracle.py: every result within the oracle's
running bound of what float32 arithmetic may lose (twice it: the kernels group operations otherwise) and half a step of its type."""
import numpy as np
import pytest

from oracle import sequence_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16"]


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


class Draw(object):
    """Inputs: float64 values that are exact in `dtype`, and their device tensors in a chosen layout."""

    def __init__(self, key, dtype, layout="plain"):
        import zlib
        self.rng = np.random.default_rng(zlib.crc32(repr(key).encode()))
        self.dtype, self.layout = dtype, layout

    def dev(self, x, dtype="float32"):
        torch = _torch()
        return torch.tensor(np.asarray(x, np.float32), device="cuda").to(getattr(torch, dtype))

    def param(self, *shape, scale=1.0, shift=0.0):
        t = self.dev(scale * self.rng.normal(size=shape) + shift)
        return t.double().cpu().numpy(), t

    def seq(self, *shape, scale=1.0, shift=0.0, lens=None):
        """(values, tensor): padding frames hold NaN, infinities and the lowest value in the tensor."""
        torch = _torch()
        t = self.dev(scale * self.rng.normal(size=shape) + shift, self.dtype)
        v = t.double().cpu().numpy()
        if lens is not None:
            bad = [float("nan"), float("inf"), float("-inf"), torch.finfo(t.dtype).min]
            for b, n in enumerate(lens):
                for k in range(max(0, min(int(n), shape[1])), shape[1]):
                    t[b, k] = bad[(b + k) % 4]
        return v, self.lay(t)

    def lay(self, t):
        torch = _torch()
        if t.dim() == 4:
            lead, tail = t.shape[:2], t.shape[2:]
            return self.lay(t.reshape(*lead, -1)).unflatten(-1, tail)
        if self.layout == "plain" or t.dim() < 3:
            return t
        if self.layout == "time-major":
            return t.transpose(0, 1).contiguous().transpose(0, 1)
        width = t.shape[2]                                     # columns of a wider array, off every alignment but the element's
        wide = torch.full((t.shape[0], t.shape[1] + 1, 2 * width + 3), float("nan"), dtype=t.dtype, device=t.device)
        wide[:, :-1, 3:3 + width] = t
        return wide[:, :-1, 3:3 + width]


def _near(name, got, want, dtype="float32"):
    g = got.double().cpu().numpy()
    assert g.shape == want.v.shape, (name, g.shape, want.v.shape)
    tol = 2 * want.e + O.HALF_STEP[dtype] * np.abs(want.v) * 1.01 + 1e-37
    off = np.abs(g - want.v)
    worst = (off / tol).max() if off.size else 0.0
    assert np.isfinite(g).all() and worst <= 1.0, "%s: %.2f times the bound at %s" % (name, worst, np.unravel_index((off / tol).argmax(), off.shape))


def _lens(lens):
    torch = _torch()
    return None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------------------------ layer norm
NORM = [((1, 1, 1), None), ((2, 3, 50), [3, 1]), ((1, 7, 255), None), ((3, 5, 256), [5, 0, 2]), ((2, 4, 1000), [0, 0]), ((1, 3, 1024), None),
        ((2, 2, 1032), [9, -3]), ((1, 5, 2000), None), ((1, 2, 4096), None), ((1, 2, 4100), [1]), ((1, 1, 16384), None), ((1, 2, 16381), None),
        ((70, 40, 33), None), ((9, 300, 64), None)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["plain", "time-major", "columns"])
@pytest.mark.parametrize("shape,lens", NORM, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else ("ragged" if v else "full"))
def test_layer_norm(S, dtype, layout, shape, lens):
    d = Draw(("norm", shape, lens), dtype, layout)
    (xv, x), (gv, g), (bv, b), (dyv, dy) = d.seq(*shape, scale=2, shift=0.5, lens=lens), d.param(shape[2], scale=0.3, shift=1), d.param(shape[2]), d.seq(*shape, lens=lens)
    want = O.layer_norm(xv, gv, bv, 1e-5, lens, dyv)
    y, mean, inv = S.layer_norm_forward(x, g, b, lens=_lens(lens))
    dx, dg, db = S.layer_norm_backward(dy, x, g, mean, inv, lens=_lens(lens))
    if shape[2] == 1:           # variance 0: y = beta; x - mean is exact
        want["dx"].e = want["dx"].e + 1e-6 * np.abs(dyv) * np.abs(gv) / np.sqrt(1e-5)
    for name, got, t in (("y", y, dtype), ("mean", mean, "float32"), ("inv_std", inv, "float32"), ("dx", dx, dtype), ("dgamma", dg, "float32"), ("dbeta", db, "float32")):
        _near(name, got, want[name], t)


def test_layer_norm_without_affine_and_of_rows(S):
    d = Draw("rows", "float32")
    (xv, x), (dyv, dy) = d.seq(1, 37, 130), d.seq(1, 37, 130)
    want = O.layer_norm(xv, None, None, 1e-3, None, dyv)
    y, mean, inv = S.layer_norm_forward(x[0], eps=1e-3)
    dx, dg, db = S.layer_norm_backward(dy[0], x[0], None, mean, inv)
    assert y.shape == (37, 130) and mean.shape == (37,)
    for name, got in (("y", y[None]), ("mean", mean[None]), ("inv_std", inv[None]), ("dx", dx[None]), ("dgamma", dg), ("dbeta", db)):
        _near(name, got, want[name])


def test_layer_norm_far_from_zero(S):
    """Rows whose mean is 1000 times their spread: the variance is taken of x - mean, nothing cancels."""
    d = Draw("far", "float32")
    xv, x = d.seq(2, 3, 777, shift=1000.0)
    want = O.layer_norm(xv, None, None, 1e-5)
    y, mean, inv = S.layer_norm_forward(x)
    _near("y", y, want["y"])
    _near("inv_std", inv, want["inv_std"])


# ------------------------------------------------------------------------------------------------------ short causal convolution
CONV = [((1, 1, 1), 1, None), ((2, 3, 5), 2, [3, 0]), ((2, 7, 64), 4, None), ((3, 8, 96), 4, [1, 8, 2]), ((2, 9, 130), 3, [2, 9]), ((1, 65, 513), 4, None),
        ((4, 130, 8), 8, [130, 7, 64, 6]), ((2, 40, 260), 5, [33, 12]), ((2, 2, 16), 8, [2, 1]), ((1, 33, 64), 6, None), ((2, 16, 40), 7, None),
        ((40, 70, 12), 4, None)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["plain", "time-major", "columns"])
@pytest.mark.parametrize("carried", [False, True])
@pytest.mark.parametrize("shape,taps,lens", CONV, ids=lambda v: str(v).replace(" ", "") if v else "full")
def test_causal_conv(S, dtype, layout, carried, shape, taps, lens):
    d = Draw(("conv", shape, taps, carried), dtype, layout)
    B, T, D = shape
    (xv, x), (wv, w), (bv, b), (dyv, dy) = d.seq(*shape, lens=lens), d.param(taps, D), d.param(D), d.seq(*shape, lens=lens)
    sv, st = Draw(("conv state", shape, taps), dtype).seq(B, taps - 1, D)
    if not carried:
        sv = st = None
    act = "silu" if taps != 3 else "linear"
    want = O.causal_conv(xv, wv, bv, sv, lens, act, dyv)
    y, out = S.causal_conv_forward(x, w, b, state=st, lens=_lens(lens), activation=act)
    dx, dw, db, ds = S.causal_conv_backward(dy, x, w, b, state=st, lens=_lens(lens), activation=act)
    _near("y", y, want["y"], dtype)
    np.testing.assert_array_equal(out.double().cpu().numpy(), want["state"].v)
    _near("dx", dx, want["dx"], dtype)
    _near("dweight", dw, want["dweight"])
    _near("dbias", db, want["dbias"])
    if carried:
        _near("dstate", ds, want["dstate"], dtype)
    else:
        assert ds is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,wide", [(9, 16), (65, 72), (1021, 1024), (1025, 1032)])
def test_causal_conv_of_odd_widths_gives_the_bits_of_the_wider_one(S, dtype, D, wide):
    torch = _torch()
    d = Draw(("conv width", D), dtype)
    (_, x), (_, dy), (_, w), (_, b), (_, st) = d.seq(3, 21, wide), d.seq(3, 21, wide), d.param(4, wide), d.param(wide), d.seq(3, 3, wide)
    lens = _lens([21, 2, 13])
    cut = [t[..., :D].contiguous() for t in (x, dy, w, b, st)]
    whole = S.causal_conv_forward(x, w, b, state=st, lens=lens) + S.causal_conv_backward(dy, x, w, b, state=st, lens=lens)
    part = S.causal_conv_forward(cut[0], cut[2], cut[3], state=cut[4], lens=lens) + S.causal_conv_backward(cut[1], cut[0], cut[2], cut[3], state=cut[4], lens=lens)
    for got, want in zip(part, whole):
        assert torch.equal(got, want[..., :D])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,taps", [(1, 1, 1), (3, 50, 4), (2, 2048, 4), (5, 33, 8), (70, 64, 2)])
def test_causal_conv_step_continues_the_sequence(S, dtype, B, D, taps):
    d = Draw(("conv step", B, D, taps), dtype)
    (xv, x), (wv, w), (bv, b) = d.seq(B, 6, D), d.param(taps, D), d.param(D)
    want = O.causal_conv(xv, wv, bv)
    y, state = S.causal_conv_forward(x[:, :3], w, b)
    for t in range(3, 6):
        got = S.causal_conv_step(x[:, t], state, w, b)
        _near("y", got, want["y"][:, t], dtype)
    np.testing.assert_array_equal(state.double().cpu().numpy(), want["state"].v)


# ------------------------------------------------------------------------------------------------------------------ selective scan
def _scan_inputs(d, shape, N, G, lens, gated, softplus=True, carried=False):
    B, T, D = shape
    v, t = {}, {}

    def put(k, pair):
        v[k], t[k] = pair
    put("u", d.seq(B, T, D, lens=lens))
    put("delta", d.seq(B, T, D, scale=0.7 if softplus else 0.02, shift=0.0 if softplus else 0.3, lens=lens))
    a = -np.exp(d.rng.normal(size=(D, N)))
    t["A"] = d.dev(a)
    v["A"] = t["A"].double().cpu().numpy()
    put("Bm", d.seq(B, T, G, N, lens=lens))
    put("Cm", d.seq(B, T, G, N, lens=lens))
    put("D", d.param(D))
    put("delta_bias", d.param(D, shift=-1.0 if softplus else 0.0, scale=1.0 if softplus else 0.01))
    put("z", d.seq(B, T, D, lens=lens) if gated else (None, None))
    put("state", d.param(B, D, N) if carried else (None, None))
    v.update(lens=lens, softplus=softplus)
    t.update(lens=_lens(lens), softplus=softplus)
    return v, t


SCAN = [((1, 1, 1), 1, 1, None), ((2, 3, 5), 3, 1, [3, 0]), ((2, 7, 64), 4, 1, None), ((3, 8, 96), 16, 1, [1, 8, 7]), ((2, 9, 130), 16, 2, [2, 9]),
        ((1, 65, 40), 16, 1, None), ((4, 50, 8), 8, 1, [50, 7, 25, 6]), ((2, 40, 252), 16, 3, [33, 12]), ((2, 16, 16), 32, 1, [16, 1]), ((1, 33, 70), 17, 1, None),
        ((2, 24, 36), 12, 2, None), ((3, 17, 30), 5, 1, [0, 0, 0]), ((5, 12, 600), 8, 1, [1, 2, 12, 11, 9]), ((1, 20, 100), 31, 4, [19]), ((9, 20, 20), 2, 1, None),
        # long enough, and few enough rows, for a time axis in pieces
        ((1, 200, 20), 16, 1, None), ((2, 261, 70), 5, 2, [261, 129]), ((3, 150, 16), 32, 1, [0, 150, 64]), ((2, 300, 40), 4, 1, [300, 1]),
        ((1, 129, 33), 1, 1, [128])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["plain", "time-major", "columns"])
@pytest.mark.parametrize("gated,carried,softplus", [(False, False, True), (True, True, True), (True, False, False)])
@pytest.mark.parametrize("shape,N,G,lens", SCAN, ids=lambda v: str(v).replace(" ", "") if v else "full")
def test_selective_scan(S, dtype, layout, gated, carried, softplus, shape, N, G, lens):
    d = Draw(("scan", shape, N, G, gated), dtype, layout)
    v, t = _scan_inputs(d, shape, N, G, lens, gated, softplus, carried)
    dyv, dy = d.seq(*shape, lens=lens)
    dlv, dl = d.param(shape[0], shape[2], N) if carried else (None, None)
    want = O.selective_scan(dy=dyv, dlast=dlv, **v)
    y, state, none = S.selective_scan_forward(**t)
    assert none is None
    y2, state2, saved = S.selective_scan_forward(save=True, **t)
    torch = _torch()
    assert torch.equal(y, y2) and torch.equal(state, state2)
    _near("y", y, want["y"], dtype)
    _near("state", state, want["state"])
    got = S.selective_scan_backward(dy, saved=saved, dlast=dl, **t)
    for name in ("du", "ddelta", "dB", "dC", "dz"):
        if name != "dz" or gated:
            _near(name, got[name], want[name], dtype)
    for name in ("dA", "dD", "ddelta_bias") + (("dstate",) if carried else ()):
        _near(name, got[name], want[name])
    assert (got["dz"] is None) == (not gated) and (got["dstate"] is None) == (not carried)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,N,G", [(1, 1, 1, 1), (3, 50, 16, 2), (2, 130, 5, 1), (1, 2048, 16, 1), (4, 33, 32, 3), (2, 64, 8, 1), (3, 30, 4, 1)])
def test_selective_scan_step_continues_the_sequence(S, dtype, B, D, N, G):
    d = Draw(("scan step", B, D, N, G), dtype)
    v, t = _scan_inputs(d, (B, 5, D), N, G, None, gated=N != 8)
    want = O.selective_scan(**v)
    frames = lambda a, b: {k: (t[k][:, a:b] if k in ("u", "delta", "Bm", "Cm", "z") and t[k] is not None else t[k]) for k in t}      # noqa: E731
    y, state, _ = S.selective_scan_forward(**frames(0, 2))
    for k in range(2, 5):
        one = {n: (x[:, 0] if n in ("u", "delta", "Bm", "Cm", "z") and x is not None else x) for n, x in frames(k, k + 1).items() if n not in ("lens", "state")}
        got = S.selective_scan_step(state=state, **one)
        _near("y", got, want["y"][:, k], dtype)
    _near("state", state, want["state"])


def test_scan_rows_without_groups(S):
    d = Draw("no groups", "float32")
    v, t = _scan_inputs(d, (2, 11, 48), 6, 1, None, False)
    y, state, saved = S.selective_scan_forward(save=True, **t)
    flat = dict(t, Bm=t["Bm"][:, :, 0], Cm=t["Cm"][:, :, 0])
    y2, state2, saved2 = S.selective_scan_forward(save=True, **flat)
    torch = _torch()
    assert torch.equal(y, y2) and torch.equal(state, state2)
    a, b = S.selective_scan_backward(y, saved=saved, **t), S.selective_scan_backward(y, saved=saved2, **flat)
    assert b["dB"].shape == flat["Bm"].shape and torch.equal(a["dB"][:, :, 0], b["dB"]) and torch.equal(a["dC"][:, :, 0], b["dC"])


def test_scan_of_extreme_step_sizes(S):
    """Step sizes from 1e-30 to 60: the softplus keeps its relative accuracy below, the decay reaches exact zeros above."""
    torch = _torch()
    d = Draw("extreme", "float32")
    v, t = _scan_inputs(d, (1, 24, 64), 4, 1, None, False)
    v["delta"] = np.broadcast_to(np.linspace(-68, 60, 24).astype(np.float32)[None, :, None], (1, 24, 64)).astype(np.float64)
    t["delta"] = d.dev(v["delta"])
    v["delta_bias"], t["delta_bias"] = None, None
    dyv, dy = d.seq(1, 24, 64)
    want = O.selective_scan(dy=dyv, **v)
    y, state, saved = S.selective_scan_forward(save=True, **t)
    _near("y", y, want["y"])
    _near("state", state, want["state"])
    got = S.selective_scan_backward(dy, saved=saved, **t)
    for name in ("du", "ddelta", "dB", "dC", "dA"):
        _near(name, got[name], want[name])
    assert torch.isfinite(got["ddelta"]).all()


# ------------------------------------------------------------------------------------------------------------- edges and use
def test_empty_batches_and_sequences(S):
    torch = _torch()
    for B, T in ((0, 4), (3, 0), (0, 0)):
        x = torch.randn(B, T, 8, device="cuda")
        y, m, i = S.layer_norm_forward(x)
        dx, dg, db = S.layer_norm_backward(x, x, None, m, i)
        assert y.shape == dx.shape == (B, T, 8) and not dg.any() and not db.any()
        w = torch.randn(4, 8, device="cuda")
        st = torch.randn(B, 3, 8, device="cuda")
        y, out = S.causal_conv_forward(x, w, state=st)
        assert torch.equal(out, st)
        dx, dw, db, ds = S.causal_conv_backward(x, x, w, state=st)
        assert not dw.any() and not db.any() and ds.shape == st.shape and not ds.any()
        A, bc, h = -torch.rand(8, 4, device="cuda"), torch.randn(B, T, 4, device="cuda"), torch.randn(B, 8, 4, device="cuda")
        y, out, saved = S.selective_scan_forward(x, x, A, bc, bc, state=h, save=True)
        assert torch.equal(out, h) and y.shape == (B, T, 8)
        dl = torch.randn(B, 8, 4, device="cuda")
        g = S.selective_scan_backward(x, x, x, A, bc, bc, saved, state=h, dlast=dl)
        assert torch.equal(g["dstate"], dl) and not g["dA"].any() and not g["dD"].any() and g["dB"].shape == bc.shape
    row = torch.randn(0, 8, device="cuda")
    assert S.causal_conv_step(row, row.new_empty(0, 3, 8), torch.randn(4, 8, device="cuda")).shape == (0, 8)
    assert S.selective_scan_step(row, row, A, row[:, :4].contiguous(), row[:, :4].contiguous(), row.new_empty(0, 8, 4)).shape == (0, 8)


def test_refusals_of_the_python_functions(S):
    torch = _torch()
    x = torch.randn(2, 3, 8, device="cuda")
    w = torch.randn(4, 8, device="cuda")
    A, bc = -torch.rand(8, 4, device="cuda"), torch.randn(2, 3, 4, device="cuda")

    def bad(match, fn, *a, **k):
        with pytest.raises(ValueError, match=match):
            fn(*a, **k)
    bad("float32 or bfloat16", S.layer_norm_forward, x.half())
    bad("gamma", S.layer_norm_forward, x, torch.ones(7, device="cuda"))
    bad("beta", S.layer_norm_forward, x, None, torch.ones(8, device="cuda").bfloat16())
    bad("lens", S.layer_norm_forward, x, lens=torch.tensor([1, 2], device="cuda"))              # int64
    bad("lens", S.layer_norm_forward, x, lens=torch.tensor([1], dtype=torch.int32, device="cuda"))
    bad("dense", S.layer_norm_forward, x.transpose(1, 2))
    bad("dimensions", S.layer_norm_forward, x[0, 0])
    y, m, i = S.layer_norm_forward(x)
    bad("dy", S.layer_norm_backward, x.bfloat16(), x, None, m, i)
    bad("dy", S.layer_norm_backward, x[:, :2], x, None, m, i)
    bad("mean", S.layer_norm_backward, x, x, None, None if False else m[:, :2], i)
    bad("taps", S.causal_conv_forward, x, torch.randn(9, 8, device="cuda"))
    bad("weight", S.causal_conv_forward, x, torch.randn(4, 7, device="cuda"))
    bad("activation", S.causal_conv_forward, x, w, activation="relu")
    bad("state", S.causal_conv_forward, x, w, state=torch.zeros(2, 3, 8, device="cuda").bfloat16())
    bad("state", S.causal_conv_step, x[:, 0], None, w)
    bad("state", S.causal_conv_step, x[:, 0], torch.zeros(2, 8, 3, device="cuda").transpose(1, 2), w)
    bad("delta", S.selective_scan_forward, x, x[:, :2], A, bc, bc)
    bad("states", S.selective_scan_forward, x, x, -torch.rand(8, 33, device="cuda"), bc, bc)
    bad("Bm", S.selective_scan_forward, x, x, A, bc.bfloat16(), bc)
    bad("groups", S.selective_scan_forward, x, x, A, torch.randn(2, 3, 3, 4, device="cuda"), bc)
    bad("groups", S.selective_scan_forward, x, x, A, torch.randn(2, 3, 2, 4, device="cuda"), bc)
    bad("z must", S.selective_scan_forward, x, x, A, bc, bc, z=x[:, :, :4])
    bad("saved", S.selective_scan_backward, x, x, x, A, bc, bc, torch.zeros(3, device="cuda"))
    bad("saves|saved", S.selective_scan_backward, x, x, x, A, bc, bc, None)
    bad("state", S.selective_scan_step, x[:, 0], x[:, 0], A, bc[:, 0], bc[:, 0], None)


def _block(S, t, w, lens):
    """norm -> projection -> convolution -> projections -> gated scan -> projection, and back; a dict of its results."""
    torch = _torch()
    x, dy = t
    D = w["conv"].shape[1]
    n, mean, inv = S.layer_norm_forward(x, w["gamma"], w["beta"], lens=lens)
    both = n @ w["w_in"]
    c, hist = S.causal_conv_forward(both[..., :D], w["conv"], w["cbias"], lens=lens)
    bc = c @ w["w_bc"]
    N = w["A"].shape[1]
    delta = c @ w["w_dt"]
    more = dict(D=w["D"], z=both[..., D:], delta_bias=w["dbias"], lens=lens)
    y, state, saved = S.selective_scan_forward(c, delta, w["A"], bc[..., :N], bc[..., N:], save=True, **more)
    out = y @ w["w_out"]
    dyy = dy @ w["w_out"].t().contiguous()
    g = S.selective_scan_backward(dyy, c, delta, w["A"], bc[..., :N], bc[..., N:], saved, **more)
    dbc = torch.cat([g["dB"], g["dC"]], -1)
    dc = g["du"] + dbc @ w["w_bc"].t().contiguous() + g["ddelta"] @ w["w_dt"].t().contiguous()
    dconv, dw, dcb, _ = S.causal_conv_backward(dc, both[..., :D], w["conv"], w["cbias"], lens=lens)
    dn = torch.cat([dconv, g["dz"]], -1) @ w["w_in"].t().contiguous()
    dx, dg, db = S.layer_norm_backward(dn, x, w["gamma"], mean, inv, lens=lens)
    return {"out": out, "hist": hist, "state": state, "dx": dx, "dgamma": dg, "dbeta": db, "dconv": dw, "dcbias": dcb, "dA": g["dA"], "dD": g["dD"],
            "ddbias": g["ddelta_bias"]}


def _block_inputs(B, T, E, D, N, seed=0):
    torch = _torch()
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, k=1.0: (k * torch.randn(*s, generator=g)).cuda()               # noqa: E731
    w = dict(gamma=1 + r(E, k=.1), beta=r(E, k=.1), w_in=r(E, 2 * D, k=E ** -.5), conv=r(4, D, k=.5), cbias=r(D, k=.1), w_bc=r(D, 2 * N, k=D ** -.5),
             w_dt=r(D, D, k=D ** -.5), A=-torch.exp(r(D, N, k=.5)), D=r(D), dbias=r(D) - 2, w_out=r(D, E, k=D ** -.5))
    return (r(B, T, E), r(B, T, E)), w


def _block_in_float64(x, dy, w, lens):
    """The same block on the CPU in float64, differentiated by torch."""
    torch = _torch()
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in w.items()}
    x = x.double().cpu().requires_grad_(True)
    on = (torch.arange(x.shape[1])[None] < lens[:, None])[..., None].double()
    D, N = p["A"].shape
    n = torch.nn.functional.layer_norm(x, (x.shape[2],), p["gamma"], p["beta"], 1e-5) * on
    both = n @ p["w_in"]
    xp = torch.nn.functional.pad(both[..., :D], (0, 0, 3, 0))
    c = torch.nn.functional.silu(sum(xp[:, k:k + x.shape[1]] * p["conv"][k] for k in range(4)) + p["cbias"]) * on
    bc, dt = c @ p["w_bc"], torch.nn.functional.softplus(c @ p["w_dt"] + p["dbias"]) * on
    h, ys = torch.zeros(x.shape[0], D, N, dtype=torch.float64), []
    for t in range(x.shape[1]):
        h = torch.exp(dt[:, t, :, None] * p["A"]) * h + (dt[:, t] * c[:, t])[..., None] * bc[:, t, None, :N]
        ys.append((h * bc[:, t, None, N:]).sum(-1) + p["D"] * c[:, t])
    out = (torch.stack(ys, 1) * torch.nn.functional.silu(both[..., D:]) * on) @ p["w_out"]
    out.backward(dy.double().cpu())
    return {"out": out.detach(), "state": h.detach(), "dx": x.grad, "dgamma": p["gamma"].grad, "dbeta": p["beta"].grad, "dconv": p["conv"].grad,
            "dcbias": p["cbias"].grad, "dA": p["A"].grad, "dD": p["D"].grad, "ddbias": p["dbias"].grad}


def test_a_block_forward_and_backward(S):
    """The operators one after the other as a model uses them, against a float64 evaluation: relative 2-norm 1e-5, float32's 6e-8 times
    the some hundred operations from the first norm to the last gradient."""
    torch = _torch()
    (x, dy), w = _block_inputs(3, 21, 24, 40, 16)
    lens = torch.tensor([21, 5, 14], dtype=torch.int32, device="cuda")
    on = (torch.arange(21, device="cuda")[None] < lens[:, None])[..., None]
    dy = dy * on
    got, want = _block(S, (x, dy), w, lens), _block_in_float64(x, dy, w, lens.cpu())
    for k, v in want.items():
        rel = float((got[k].double().cpu() - v).norm() / v.norm())
        assert rel < 1e-5, (k, rel)


def test_a_block_frame_by_frame(S):
    """A prompt, then single frames, against the whole sequence at once."""
    torch = _torch()
    (x, _), w = _block_inputs(2, 17, 24, 40, 16, seed=3)
    D, N = w["A"].shape
    whole = _block(S, (x, torch.zeros_like(x)), w, None)["out"]
    pre = 11
    n, _, _ = S.layer_norm_forward(x[:, :pre], w["gamma"], w["beta"])
    both = n @ w["w_in"]
    c, hist = S.causal_conv_forward(both[..., :D], w["conv"], w["cbias"])
    bc = c @ w["w_bc"]
    y, state, _ = S.selective_scan_forward(c, c @ w["w_dt"], w["A"], bc[..., :N], bc[..., N:], D=w["D"], z=both[..., D:], delta_bias=w["dbias"])
    outs = [y @ w["w_out"]]
    for t in range(pre, 17):
        n, _, _ = S.layer_norm_forward(x[:, t], w["gamma"], w["beta"])
        both = n @ w["w_in"]
        c = S.causal_conv_step(both[:, :D], hist, w["conv"], w["cbias"])
        bc = c @ w["w_bc"]
        y = S.selective_scan_step(c, c @ w["w_dt"], w["A"], bc[:, :N], bc[:, N:], state, D=w["D"], z=both[:, D:], delta_bias=w["dbias"])
        outs.append((y @ w["w_out"])[:, None])
    assert float((torch.cat(outs, 1) - whole).norm() / whole.norm()) < 1e-5


def test_two_runs_give_the_same_bits(S):
    torch = _torch()
    (x, dy), w = _block_inputs(37, 40, 24, 200, 16, seed=5)
    lens = torch.randint(0, 41, (37,), dtype=torch.int32, device="cuda")
    a, b = _block(S, (x, dy), w, lens), _block(S, (x, dy), w, lens)
    for k in a:
        assert torch.equal(a[k], b[k]), k


def test_on_another_stream(S):
    torch = _torch()
    (x, dy), w = _block_inputs(4, 30, 24, 72, 16, seed=6)
    want = _block(S, (x, dy), w, None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _block(S, (x, dy), w, None)
    side.synchronize()
    for k in want:
        assert torch.equal(got[k], want[k]), k


def test_captured_into_graphs(S):
    """Two graphs captured and replayed in turn, with eager work between: every replay equals the eager result.  (The operators alone:
    the projections between them are the library's.)"""
    torch = _torch()

    def passes(x, dy, w):
        D, N = w["A"].shape
        n, mean, inv = S.layer_norm_forward(x, w["gamma"], w["beta"])
        dx, dg, db = S.layer_norm_backward(dy, x, w["gamma"], mean, inv)
        c, hist = S.causal_conv_forward(n, w["c"], w["beta"])
        dc, dw, dcb, _ = S.causal_conv_backward(dy, n, w["c"], w["beta"])
        A = w["A"]
        y, st, saved = S.selective_scan_forward(c, n, A, w["Bm"], w["Cm"], D=w["gamma"], z=x, save=True)
        g = S.selective_scan_backward(dy, c, n, A, w["Bm"], w["Cm"], saved, D=w["gamma"], z=x)
        s1 = S.causal_conv_step(x[:, 0], hist, w["c"], w["beta"])
        s2 = S.selective_scan_step(x[:, 0], n[:, 0], A, w["Bm"][:, 0], w["Cm"][:, 0], st)
        return [n, mean, inv, dx, dg, db, c, dc, dw, dcb, y, s1, s2, hist, st] + [v for v in g.values() if v is not None]
    sets = []
    for seed, (B, T, D, N) in ((1, (3, 20, 64, 16)), (2, (2, 33, 96, 8))):
        (x, dy), w0 = _block_inputs(B, T, D, D, N, seed=seed)
        r = torch.Generator(device="cuda").manual_seed(seed)
        rn = lambda *s: torch.randn(*s, generator=r, device="cuda")               # noqa: E731
        sets.append((x, dy, dict(gamma=w0["gamma"], beta=w0["beta"], c=w0["conv"], A=w0["A"], Bm=rn(B, T, N), Cm=rn(B, T, N))))
    eager = [[v.clone() for v in passes(*s)] for s in sets]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for s in sets:
            passes(*s)
    side.synchronize()
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(passes(*s))
        graphs.append(g)
    for turn in range(4):
        for k in (0, 1, 0):
            for o in outs[k]:
                o.zero_()
            graphs[k].replay()
            if turn % 2:
                torch.cuda.synchronize()
                passes(*sets[1 - k])
            torch.cuda.synchronize()
            for got, want in zip(outs[k], eager[k]):
                assert torch.equal(got, want)


def test_frames_more_than_4_gib_apart(S):
    """Rows 8 MiB apart, 700 of them: the same bits as from a dense copy."""
    torch = _torch()
    T, D, wide = 700, 64, 1 << 22
    g = torch.Generator(device="cuda").manual_seed(11)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")                   # noqa: E731
    big = torch.empty(1, T, wide, dtype=torch.bfloat16, device="cuda")           # 5.5 GiB; only the columns below are written or read
    cols = [big[..., k * 128:k * 128 + D] for k in range(4)]
    dense = [rn(1, T, D).bfloat16() for _ in cols]
    for c, d in zip(cols, dense):
        c.copy_(d)
    gamma, beta, w = rn(D), rn(D), rn(4, D)
    A, bm = -torch.rand(D, 16, generator=g, device="cuda"), rn(1, T, 16).bfloat16()
    rows = big[..., 1 << 20:(1 << 20) + 16]
    rows.copy_(bm)

    def passes(x, u, z, dy, bm):
        y, m, i = S.layer_norm_forward(x, gamma, beta)
        out = [y, m, i] + list(S.layer_norm_backward(dy, x, gamma, m, i))
        y, st = S.causal_conv_forward(x, w, beta)
        out += [y, st] + list(S.causal_conv_backward(dy, x, w, beta)[:3])
        y, st, saved = S.selective_scan_forward(u, x, A, bm, bm, D=gamma, z=z, save=True)
        grads = S.selective_scan_backward(dy, u, x, A, bm, bm, saved, D=gamma, z=z)
        return out + [y, st] + [v for v in grads.values() if v is not None]
    for a, b in zip(passes(*cols, rows), passes(*dense, bm)):
        assert torch.equal(a, b)


def test_many_utterances(S):
    """More utterances than a grid dimension holds."""
    torch = _torch()
    B, D, N = 70001, 6, 3
    g = torch.Generator(device="cuda").manual_seed(12)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")                   # noqa: E731
    x, st, w = rn(B, D), rn(B, 2, D), rn(3, D)
    want = (torch.cat([st, x[:, None]], 1) * w).sum(1)
    after = torch.cat([st[:, 1:], x[:, None]], 1)
    y = S.causal_conv_step(x, st, w, activation="linear")
    # three products and their sum: 5 roundings of at most the sum of the sizes
    size = (torch.cat([st, x[:, None]], 1).abs().amax(1) * w.abs().sum(0)).max() + x.abs().max() * w.abs().sum(0).max()
    assert (y - want).abs().max() <= 5 * 2.0 ** -24 * 4 * size and torch.equal(st, after)
    A, bc, h = -torch.rand(D, N, generator=g, device="cuda"), rn(B, N), rn(B, D, N)
    dt = torch.rand(B, D, generator=g, device="cuda")
    want_h = torch.exp(dt.double()[..., None] * A.double()) * h.double() + (dt.double() * x.double())[..., None] * bc.double()[:, None]
    y = S.selective_scan_step(x, dt, A, bc, bc, h, softplus=False)
    # h: a and its product, dt u B: about 12 roundings of the sizes (all below 40)
    assert (h - want_h).abs().max() <= 12 * 2.0 ** -24 * 40
    assert (y - (want_h * bc.double()[:, None]).sum(-1)).abs().max() <= 20 * 2.0 ** -24 * 40 * 5 * N
    u = rn(B, 2, D)
    y, last, _ = S.selective_scan_forward(u, dt[:, None].expand(B, 2, D), A, bc[:, None].expand(B, 2, N), bc[:, None].expand(B, 2, N), softplus=False)
    h = torch.zeros(B, D, N, device="cuda")
    for t in range(2):
        yt = S.selective_scan_step(u[:, t], dt, A, bc, bc, h, softplus=False)
        assert (y[:, t] - yt).abs().max() <= 20 * 2.0 ** -24 * 40 * 5 * N
    assert (last - h).abs().max() <= 24 * 2.0 ** -24 * 40


def test_two_streams_at_once(S):
    torch = _torch()
    sets = [_block_inputs(4, 150, 24, 72, 16, seed=k) for k in (21, 22)]
    want = [_block(S, t, w, None) for t, w in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [None, None]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k] = _block(S, *sets[k], None)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for k in a:
            assert torch.equal(a[k], b[k]), k


def test_sizes_that_the_library_refuses(S):
    torch = _torch()
    from ip_avsr_amd._lib import AdenetError
    x = torch.zeros(1, 1, 16385, device="cuda")
    with pytest.raises(AdenetError, match="channels"):
        S.layer_norm_forward(x)
    with pytest.raises(ValueError, match="out of range"):
        S.layer_norm_backward(x, x, None, torch.zeros(1, 1, device="cuda"), torch.zeros(1, 1, device="cuda"))
    with pytest.raises(AdenetError, match="eps"):
        S.layer_norm_forward(x[..., :8].contiguous(), eps=-1.0)
    long = torch.zeros(1, 1, 1, device="cuda").expand(1, (1 << 31) + 8, 1)
    for fn in (S.layer_norm_forward, lambda v: S.causal_conv_forward(v, torch.ones(2, 1, device="cuda")),
               lambda v: S.selective_scan_forward(v, v, -torch.ones(1, 1, device="cuda"), v, v)):
        with pytest.raises(ValueError, match=r"2\^31"):
            fn(long)


def _random_lens(d, B, T):
    return [int(v) for v in d.rng.integers(0, T + 1, size=B)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(110, 60, 40), (30, 40, 1100), (26, 40, 2056), (3, 100, 4104), (3, 100, 8200), (2, 150, 4001), (2, 150, 9001)],
                         ids=lambda v: "x".join(map(str, v)))
def test_layer_norm_over_many_rows(S, dtype, shape):
    """More rows than workgroups, in every width of a row: the workgroups' own sums and their sum over workgroups."""
    d = Draw(("norm rows", shape), dtype)
    lens = _random_lens(d, shape[0], shape[1])
    (xv, x), (gv, g), (dyv, dy) = d.seq(*shape, lens=lens), d.param(shape[2], scale=0.3, shift=1), d.seq(*shape, lens=lens)
    want = O.layer_norm(xv, gv, None, 1e-5, lens, dyv)
    y, mean, inv = S.layer_norm_forward(x, g, lens=_lens(lens))
    dx, dg, db = S.layer_norm_backward(dy, x, g, mean, inv, lens=_lens(lens))
    for name, got, t in (("y", y, dtype), ("mean", mean, "float32"), ("inv_std", inv, "float32"), ("dx", dx, dtype), ("dgamma", dg, "float32"), ("dbeta", db, "float32")):
        _near(name, got, want[name], t)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_short_utterances(S, dtype):
    """More utterances than workgroups: several per workgroup, their sums in its registers."""
    d = Draw("short", dtype)
    lens = _random_lens(d, 5000, 3)
    (xv, x), (wv, w), (dyv, dy) = d.seq(5000, 3, 8, lens=lens), d.param(3, 8), d.seq(5000, 3, 8, lens=lens)
    want = O.causal_conv(xv, wv, None, None, lens, "silu", dyv)
    y, st = S.causal_conv_forward(x, w, lens=_lens(lens))
    dx, dw, db, _ = S.causal_conv_backward(dy, x, w, lens=_lens(lens))
    _near("y", y, want["y"], dtype)
    _near("dx", dx, want["dx"], dtype)
    _near("dweight", dw, want["dweight"])
    _near("dbias", db, want["dbias"])
    np.testing.assert_array_equal(st.double().cpu().numpy(), want["state"].v)
    B, T, D, N = 2500, 3, 20, 4
    lens = _random_lens(d, B, T)
    v, t = _scan_inputs(d, (B, T, D), N, 1, lens, True, True, True)
    dyv, dy = d.seq(B, T, D, lens=lens)
    want = O.selective_scan(dy=dyv, **v)
    y, state, saved = S.selective_scan_forward(save=True, **t)
    got = S.selective_scan_backward(dy, saved=saved, **t)
    _near("y", y, want["y"], dtype)
    _near("state", state, want["state"])
    for name in ("du", "ddelta", "dB", "dC", "dz"):
        _near(name, got[name], want[name], dtype)
    for name in ("dA", "dD", "ddelta_bias", "dstate"):
        _near(name, got[name], want[name])
