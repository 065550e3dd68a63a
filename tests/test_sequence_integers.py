"""oracle/sequence_integers.py against the float64 oracle, and that its results tell one utterance, or one frame, from none."""
import numpy as np
import pytest

from oracle import sequence_integers as I
from oracle import sequence_oracle as O


def _ints(rng, *shape, most=3):
    return rng.integers(-most, most + 1, size=shape)


@pytest.mark.parametrize("lens", [None, [6, 0, 2]])
def test_layer_norm_and_convolution_sums_are_the_oracles(lens):
    rng = np.random.default_rng([51, 0 if lens is None else 1])
    x, dy = _ints(rng, 3, 6, 4), _ints(rng, 3, 6, 4)
    for taps in (1, 3, 8):
        want = O.causal_conv(x, _ints(rng, taps, 4), None, None, lens, "linear", dy)
        got = I.causal_conv_sums(x, taps, dy, lens)
        np.testing.assert_array_equal(got["dweight"], want["dweight"].v)
        np.testing.assert_array_equal(got["dbias"], want["dbias"].v)
    # rows of mean 0 and variance 1 are twice their xhat at eps = 3
    x = np.broadcast_to(np.array([1, -1, -1, 1]), (3, 6, 4)) * rng.choice([-1, 1], size=(3, 6, 1))
    want, got = O.layer_norm(x, None, None, 3.0, lens, dy), I.layer_norm_sums(x, dy, lens)
    np.testing.assert_array_equal(got["dgamma"], 2 * want["dgamma"].v)
    np.testing.assert_array_equal(got["dbeta"], want["dbeta"].v)


@pytest.mark.parametrize("lens", [None, [7, 0, 2]])
@pytest.mark.parametrize("G", [1, 2])
def test_the_scan_is_the_oracles(lens, G):
    rng = np.random.default_rng([52, G, 0 if lens is None else 1])
    B, T, D, N = 3, 7, 6, 3
    v = dict(u=_ints(rng, B, T, D), Bm=_ints(rng, B, T, G, N), Cm=_ints(rng, B, T, G, N), D=_ints(rng, D), state=_ints(rng, B, D, N), dy=_ints(rng, B, T, D),
             dlast=_ints(rng, B, D, N))
    dt = rng.integers(0, 3, size=(B, T, D))
    got, want = I.scan(dt=dt, lens=lens, **v), O.selective_scan(delta=dt, A=np.zeros((D, N)), softplus=False, lens=lens, **v)
    for k in got:
        if k != "biggest":
            np.testing.assert_array_equal(got[k], want[k].v, err_msg=k)


def test_one_utterance_or_frame_less_is_seen():
    """The planted mistake: every sum over frames differs from the one that leaves out an utterance of thousands, or a frame of one."""
    rng = np.random.default_rng(53)
    B, T, D, N = 2500, 3, 8, 4
    lens = rng.integers(1, T + 1, size=B)
    x, dy = _ints(rng, B, T, D, most=8), _ints(rng, B, T, D, most=8)
    v = dict(dt=rng.integers(1, 3, size=(B, T, D)), Bm=_ints(rng, B, T, 1, N, most=1), Cm=_ints(rng, B, T, 1, N, most=1), D=_ints(rng, D), state=_ints(rng, B, D, N),
             dlast=_ints(rng, B, D, N))

    def sums(lens):
        s = I.scan(u=x, dy=dy, lens=lens, **v)
        return {**I.layer_norm_sums(x, dy, lens), **I.causal_conv_sums(x, 4, dy, lens), **{k: s[k] for k in ("dA", "dD", "ddelta_bias")}}
    whole = sums(lens)
    for b in rng.choice(B, size=6, replace=False):
        for n in {0, int(lens[b]) - 1}:
            less = lens.copy()
            less[b] = n
            for k, got in sums(less).items():
                assert k == "biggest" or (got != whole[k]).any(), (k, b, n)
