"""The sequence operators' sums over frames, utterances and workgroups: exactly, on integers (oracle/sequence_integers.py says why float32
computes them exactly), and time axes in pieces over several workgroups of channels against the float64 oracle."""
import numpy as np
import pytest

from oracle import sequence_integers as I
from oracle import sequence_oracle as O
from tests.test_gpu_sequence import Draw, _lens, _near, _scan_inputs

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16"]


@pytest.fixture(scope="module")
def S():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from ip_avsr_amd.custom import sequence
    return sequence


def _ints(rng, *shape, most=3):
    return rng.integers(-most, most + 1, size=shape)


def _dev(x, dtype="float32"):
    import torch
    return torch.tensor(x, dtype=torch.float32, device="cuda").to(getattr(torch, dtype))


def _equal(name, got, want):
    """The integers, rounded once where the result's type has fewer bits."""
    import torch
    want = torch.tensor(want, dtype=torch.float32).to(got.dtype)
    got = got.cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.equal(got, want), "%s: %d of %d are not the sum" % (name, (got != want).sum(), got.numel())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(110, 60, 40), (520, 40, 250), (30, 40, 1100), (26, 40, 2056), (3, 100, 4104), (3, 100, 8200), (2, 150, 4001), (2, 150, 9001),
                                   (700, 9, 33)], ids=lambda v: "x".join(map(str, v)))
def test_layer_norm_sums(S, dtype, shape):
    rng = np.random.default_rng([61, *shape])
    lens = rng.integers(0, shape[1] + 1, size=shape[0])
    x, dy = _ints(rng, *shape, most=8), _ints(rng, *shape, most=8)
    want = I.layer_norm_sums(x, dy, lens)
    assert want["biggest"] < I.EXACT
    mean, inv = _dev(np.zeros(shape[:2])), _dev(np.ones(shape[:2]))
    _, dg, db = S.layer_norm_backward(_dev(dy, dtype), _dev(x, dtype), _dev(rng.normal(size=shape[2])), mean, inv, lens=_lens([int(n) for n in lens]))
    _equal("dgamma", dg, want["dgamma"])
    _equal("dbeta", db, want["dbeta"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,taps", [((5000, 3, 8), 3), ((520, 40, 100), 4), ((520, 40, 1000), 4), ((3, 700, 300), 8), ((9000, 1, 3), 2), ((40, 97, 1030), 1),
                                        ((1, 5000, 65), 5)], ids=str)
def test_causal_conv_sums(S, dtype, shape, taps):
    rng = np.random.default_rng([62, *shape, taps])
    lens = rng.integers(0, shape[1] + 1, size=shape[0])
    lens[0] = shape[1]
    x, dy = _ints(rng, *shape, most=8), _ints(rng, *shape, most=8)
    want = I.causal_conv_sums(x, taps, dy, lens)
    assert want["biggest"] < I.EXACT
    _, dw, db, _ = S.causal_conv_backward(_dev(dy, dtype), _dev(x, dtype), _dev(rng.normal(size=(taps, shape[2]))), lens=_lens([int(n) for n in lens]), activation="linear")
    _equal("dweight", dw, want["dweight"])
    _equal("dbias", db, want["dbias"])


# the last five: long enough, and few enough rows, for pieces of the time axis, over several workgroups of channels in a group
SCAN = [((2500, 3, 20), 4, 1), ((1500, 2, 70), 16, 2), ((300, 9, 300), 8, 1), ((70, 30, 150), 16, 1), ((40, 17, 200), 31, 1), ((1200, 5, 18), 2, 3),
        ((2, 150, 150), 16, 1), ((1, 140, 300), 16, 2), ((2, 150, 130), 31, 1), ((2, 261, 300), 5, 1), ((1, 200, 600), 3, 2)]


def _scan_exactly(S, dtype, shape, N, G):
    rng = np.random.default_rng([63, *shape, N, G])
    B, T, D = shape
    lens = rng.integers(0, T + 1, size=B)
    lens[0] = T
    v = dict(u=_ints(rng, B, T, D, most=1), dt=rng.integers(0, 3, size=shape), Bm=_ints(rng, B, T, G, N, most=1), Cm=_ints(rng, B, T, G, N, most=1), D=_ints(rng, D),
             state=_ints(rng, B, D, N, most=2), dy=_ints(rng, B, T, D, most=1), dlast=_ints(rng, B, D, N, most=2))
    want = I.scan(lens=lens, **v)
    assert want["biggest"] < I.EXACT
    t = {k: _dev(x, dtype if k in ("u", "Bm", "Cm", "dy") else "float32") for k, x in v.items() if k != "dt"}
    dy, dlast = t.pop("dy"), t.pop("dlast")
    t.update(delta=_dev(v["dt"], dtype), A=_dev(np.zeros((D, N))), lens=_lens([int(n) for n in lens]), softplus=False)
    y, state, saved = S.selective_scan_forward(save=True, **t)
    g = S.selective_scan_backward(dy, saved=saved, dlast=dlast, **t)
    for name, got in dict(g, y=y, state=state).items():
        if name != "dz":
            _equal(name, got, want[name])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,N,G", SCAN, ids=str)
def test_selective_scan_exactly(S, dtype, shape, N, G):
    assert shape[1] < 128 or S._lib.load().adn_op_selective_scan_workspace(*shape, N, G, 0) > 0      # pieces
    _scan_exactly(S, dtype, shape, N, G)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,G,N", [(49, 130, 16, 4), (50, 140, 16, 17)])
def test_a_backward_pass_in_pieces_behind_a_forward_pass_in_one(S, dtype, B, T, G, N):
    """Rows enough for the forward pass to take the time axis whole (more than 768 waves, here one a group) and not for the backward pass."""
    need = S._lib.load().adn_op_selective_scan_workspace
    assert need(B, T, G, N, G, 0) == 0 and need(48, T, G, N, G, 0) > 0
    _scan_exactly(S, dtype, (B, T, G), N, G)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gated,carried,softplus", [(True, True, True), (False, False, True), (True, False, False)])
@pytest.mark.parametrize("shape,N,G,lens", [((2, 150, 150), 16, 1, [150, 70]), ((1, 140, 300), 16, 2, [133]), ((1, 150, 130), 24, 1, [149]), ((2, 130, 300), 7, 1, [129, 40]),
                                            ((1, 131, 520), 4, 2, None)], ids=str)
def test_pieces_of_the_time_axis_over_several_workgroups(S, dtype, gated, carried, softplus, shape, N, G, lens):
    B, T, D = shape
    lib = S._lib.load()
    assert lib.adn_op_selective_scan_workspace(B, T, D, N, G, 0) > 0
    d = Draw(("pieces", shape, N, G, gated), dtype, "columns")
    v, t = _scan_inputs(d, shape, N, G, lens, gated, softplus, carried)
    dyv, dy = d.seq(*shape, lens=lens)
    dlv, dl = d.param(B, D, N) if carried else (None, None)
    want = O.selective_scan(dy=dyv, dlast=dlv, **v)
    y, state, saved = S.selective_scan_forward(save=True, **t)
    g = S.selective_scan_backward(dy, saved=saved, dlast=dl, **t)
    _near("y", y, want["y"], dtype)
    _near("state", state, want["state"])
    for name in ("du", "ddelta", "dB", "dC") + (("dz",) if gated else ()):
        _near(name, g[name], want[name], dtype)
    for name in ("dA", "dD", "ddelta_bias") + (("dstate",) if carried else ()):
        _near(name, g[name], want[name])


def test_pieces_of_the_time_axis_captured_into_a_graph(S):
    """Forward and backward with a split time axis, captured, replayed on new inputs with eager work between; and two such graphs in turn."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(64)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")               # noqa: E731
    sets = []
    for B, T, D, N in ((2, 200, 130, 16), (1, 260, 70, 5)):
        assert S._lib.load().adn_op_selective_scan_workspace(B, T, D, N, 1, 0) > 0
        lens = torch.randint(1, T + 1, (B,), dtype=torch.int32, generator=g, device="cuda")
        sets.append(dict(u=rn(B, T, D), delta=rn(B, T, D), A=-torch.exp(rn(D, N)), Bm=rn(B, T, N), Cm=rn(B, T, N), D=rn(D), z=rn(B, T, D), state=rn(B, D, N), lens=lens))

    def passes(t):
        y, state, saved = S.selective_scan_forward(save=True, **t)
        out = S.selective_scan_backward(t["z"], saved=saved, dlast=t["state"], **t)
        return [y, state] + [out[k] for k in sorted(out)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for t in sets:
            passes(t)
    side.synchronize()
    graphs, outs = [], []
    for t in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(passes(t))
        graphs.append(graph)
    for turn in range(4):
        for k, t in enumerate(sets):
            for name in ("u", "delta", "Bm", "z"):
                t[name].copy_(rn(*t[name].shape))
            want = passes(t)
            for o in outs[k]:
                o.zero_()
            graphs[k].replay()
            if turn % 2:
                passes(sets[1 - k])
            torch.cuda.synchronize()
            for got, v in zip(outs[k], want):
                assert torch.equal(got, v)
