"""The sequence operators' refusals, on the CPU: the C entry points check their arguments before they touch the device, and the Python
functions check theirs before they call one."""
import ctypes as C

import pytest
import torch

from ip_avsr_amd import _lib


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        from ip_avsr_amd.build import build
        build(verbose=False)
    return _lib.load()


def _norm(**over):
    v = dict(dtype=0, batch=2, steps=3, channels=8, eps=1e-5, x=64, x_stride_b=24, x_stride_t=8, y=64, y_stride_b=24, y_stride_t=8, mean=64, inv_std=64)
    v.update(over)
    return _lib.NormArgs(**v)


def _conv(**over):
    v = dict(dtype=0, batch=2, steps=3, channels=8, taps=4, activation=1, x=64, x_stride_b=24, x_stride_t=8, y=64, y_stride_b=24, y_stride_t=8,
             weight=64, state_out=64)
    v.update(over)
    return _lib.ConvArgs(**v)


def _scan(**over):
    v = dict(dtype=0, batch=2, steps=3, channels=8, states=4, groups=1, softplus=1, A=64, state_out=64)
    for k in ("u", "delta", "b", "c", "y"):
        v.update({k: 64, k + "_stride_b": 24, k + "_stride_t": 8})
    v.update(over)
    return _lib.ScanArgs(**v)


def _refused(fn, args, word, lib):
    assert fn(C.byref(args), None) == _lib.ADN_ERR_INVALID
    assert word in lib.adn_last_error().decode()


def test_struct_sizes_match_the_library(lib):
    out = (C.c_int32 * 3)()
    lib.adn_op_abi_sizes(out)
    assert list(out) == [C.sizeof(_lib.NormArgs), C.sizeof(_lib.ConvArgs), C.sizeof(_lib.ScanArgs)]


def test_null_arguments(lib):
    for name in ("layer_norm_forward", "layer_norm_backward", "causal_conv_forward", "causal_conv_backward", "causal_conv_step",
                 "selective_scan_forward", "selective_scan_backward", "selective_scan_step"):
        assert getattr(lib, "adn_op_" + name)(None, None) == _lib.ADN_ERR_INVALID
        assert b"null arguments" in lib.adn_last_error()


@pytest.mark.parametrize("over,word", [
    (dict(dtype=2), "dtype"), (dict(channels=0), "channels"), (dict(channels=16385), "channels"), (dict(batch=-1), "batch"),
    (dict(batch=1 << 16, steps=1 << 15), "batch"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(mean=None), "statistics"),
    (dict(x=None), "tensor"), (dict(x=66), "misaligned"), (dict(y=None), "tensor")])
def test_layer_norm_refusals(lib, over, word):
    _refused(lib.adn_op_layer_norm_forward, _norm(**over), word, lib)


def test_layer_norm_backward_refusals(lib):
    full = dict(dy=64, dy_stride_b=24, dy_stride_t=8, dx=64, dx_stride_b=24, dx_stride_t=8, dgamma=64, dbeta=64, workspace=64)
    need = lib.adn_op_layer_norm_workspace(2, 3, 8)
    assert need > 0
    _refused(lib.adn_op_layer_norm_backward, _norm(**full, workspace_floats=need - 1), "workspace", lib)
    _refused(lib.adn_op_layer_norm_backward, _norm(**{**full, "workspace": None}, workspace_floats=need), "workspace", lib)
    _refused(lib.adn_op_layer_norm_backward, _norm(**{**full, "dgamma": None}, workspace_floats=need), "gradient", lib)
    _refused(lib.adn_op_layer_norm_backward, _norm(**{**full, "dx": None}, workspace_floats=need), "tensor", lib)
    assert lib.adn_op_layer_norm_workspace(2, 3, 0) < 0 and lib.adn_op_layer_norm_workspace(0, 3, 8) == 0


@pytest.mark.parametrize("over,word", [
    (dict(dtype=-1), "dtype"), (dict(taps=0), "taps"), (dict(taps=9), "taps"), (dict(activation=2), "activation"), (dict(weight=None), "weight"),
    (dict(steps=-1), "steps"), (dict(channels=0), "channels"), (dict(x=None), "tensor"), (dict(state_out=None), "state_out"), (dict(state=64), "state_out"), (dict(batch=1 << 28, steps=1), "batch too large")])
def test_causal_conv_refusals(lib, over, word):
    _refused(lib.adn_op_causal_conv_forward, _conv(**over), word, lib)


def test_causal_conv_backward_and_step_refusals(lib):
    full = dict(dy=64, dy_stride_b=24, dy_stride_t=8, dx=64, dx_stride_b=24, dx_stride_t=8, dweight=64, dbias=64, workspace=64)
    need = lib.adn_op_causal_conv_workspace(2, 3, 8, 4)
    _refused(lib.adn_op_causal_conv_backward, _conv(**full, workspace_floats=need - 1), "workspace", lib)
    _refused(lib.adn_op_causal_conv_backward, _conv(**{**full, "dbias": None}, workspace_floats=need), "gradient", lib)
    _refused(lib.adn_op_causal_conv_step, _conv(steps=2), "one frame", lib)
    _refused(lib.adn_op_causal_conv_step, _conv(steps=1, lens=64), "no lengths", lib)
    _refused(lib.adn_op_causal_conv_step, _conv(steps=1, state_out=None), "history", lib)


@pytest.mark.parametrize("over,word", [
    (dict(dtype=3), "dtype"), (dict(states=0), "states"), (dict(states=33), "states"), (dict(groups=3), "groups"), (dict(groups=0), "groups"),
    (dict(A=None), "A"), (dict(u=None), "tensor"), (dict(z=2), "gate"), (dict(y=None), "y"), (dict(state_out=None), "state_out"),
    (dict(state=64), "state_out"), (dict(u_stride_t=1 << 26), "frame stride"), (dict(c_stride_t=-8), "frame stride"), (dict(batch=1 << 20, steps=1, channels=1 << 12), "too large"), (dict(checkpoints=64, checkpoint_floats=1), "checkpoints")])
def test_selective_scan_refusals(lib, over, word):
    _refused(lib.adn_op_selective_scan_forward, _scan(**over), word, lib)


def test_selective_scan_backward_and_step_refusals(lib):
    full = dict(dB=64, dC=64, dA=64, dD=64, ddelta_bias=64, checkpoints=64, workspace=64)
    for k in ("dy", "du", "ddelta"):
        full.update({k: 64, k + "_stride_b": 24, k + "_stride_t": 8})
    n, m = lib.adn_op_selective_scan_checkpoints(2, 3, 8, 4, 1), lib.adn_op_selective_scan_workspace(2, 3, 8, 4, 1, 1)
    assert n > 0 and m > 0
    back = lib.adn_op_selective_scan_backward
    _refused(back, _scan(**full, checkpoint_floats=n - 1, workspace_floats=m), "checkpoints", lib)
    _refused(back, _scan(**full, checkpoint_floats=n, workspace_floats=m - 1), "workspace", lib)
    _refused(back, _scan(**{**full, "dB": None}, checkpoint_floats=n, workspace_floats=m), "gradient", lib)
    _refused(back, _scan(**{**full, "dy": None}, checkpoint_floats=n, workspace_floats=m), "gradient", lib)
    _refused(back, _scan(**full, z=64, checkpoint_floats=n, workspace_floats=m), "gradient", lib)         # a gate without dz
    _refused(lib.adn_op_selective_scan_step, _scan(steps=2), "one frame", lib)
    _refused(lib.adn_op_selective_scan_step, _scan(steps=1, state_out=None), "state", lib)
    _refused(lib.adn_op_selective_scan_step, _scan(steps=1, batch=1 << 21, channels=1 << 9), "too large", lib)
    _refused(lib.adn_op_selective_scan_forward, _scan(batch=1 << 24, steps=1), "too large", lib)
    assert lib.adn_op_selective_scan_checkpoints(2, 3, 8, 33, 1) < 0 and lib.adn_op_selective_scan_workspace(2, 3, 8, 4, 3, 1) < 0


def test_python_functions_refuse_host_tensors(lib):
    from ip_avsr_amd.custom import sequence as S
    x = torch.zeros(2, 3, 8)
    row = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        S.layer_norm_forward(x)
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        S.layer_norm_backward(x, x, None, None, None)
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        S.causal_conv_forward(x, torch.zeros(4, 8))
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        S.causal_conv_backward(x, x, torch.zeros(4, 8))
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        S.causal_conv_step(row, torch.zeros(2, 3, 8), torch.zeros(4, 8))
    A, bc = torch.zeros(8, 4), torch.zeros(2, 3, 4)
    with pytest.raises(ValueError, match="u must be a CUDA tensor"):
        S.selective_scan_forward(x, x, A, bc, bc)
    with pytest.raises(ValueError, match="u must be a CUDA tensor"):
        S.selective_scan_backward(x, x, x, A, bc, bc, None)
    with pytest.raises(ValueError, match="u must be a CUDA tensor"):
        S.selective_scan_step(row, row, A, bc[:, 0], bc[:, 0], torch.zeros(2, 8, 4))
