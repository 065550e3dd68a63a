"""Sequence operators on the GPU: layer norm, the short causal convolution and the selective state-space scan -- the blocks of the
sequence models that take the LSTM's place (norm -> projection -> convolution + SiLU -> projection -> gated scan -> projection).
No reference counterpart; the kernels are ``csrc/layernorm.hip``, ``csrc/causal_conv.hip`` and ``csrc/selective_scan.hip`` behind the
``adn_op_*`` entry points of the C ABI.

Every operator has a forward and a backward function (gradients by hand, as everywhere in this package: there is no autograd here)
and, where it carries a state, a ``*_step`` for one frame of every utterance, which moves the state on in place.

Tensors are CUDA torch tensors, nothing is copied or converted: activations (batch, time, channels) in float32 or bfloat16, all of one
call in the same type, with dense channels and any frame and utterance stride (column ranges of a wider projection, time-major
arrays; the scan takes frame strides below 2^26 elements); parameters, statistics and the scan's states in float32, dense.  Results are new dense tensors.  ``lens`` (int32, one length
per utterance) marks frames at and behind it as padding: never read, zero in every result, absent from every sum, and a state passes
them unchanged; lengths outside [0, T] are clamped.  Work is enqueued on the current stream of the tensors' device; sums run in a
fixed order, so two runs give the same bits.  A bad argument raises ``ValueError``, sizes that the library refuses ``AdenetError``;
without the HIP library the first call raises.
"""
import ctypes as C

import torch

from .. import _lib
from .._lib import ConvArgs, NormArgs, ScanArgs

_DTYPE = {torch.float32: 0, torch.bfloat16: 1}
_ACTIVATION = {None: 0, "linear": 0, "silu": 1}
_NO_SEQ = (None, 0, 0)
# the current stream's handle without the Stream object around it (2.7 us of the 12 of a small call), where this torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _fail(what):
    raise ValueError("ip_avsr_amd.custom.sequence: " + what)


def _activation(name, t, shape, like=None):
    """Checks an activation and returns its (pointer, utterance stride, frame stride)."""
    if like is not None:
        if not isinstance(t, torch.Tensor) or t.dtype is not like.dtype or t.get_device() != like.get_device():
            _fail("%s must be a %s tensor on %s" % (name, like.dtype, like.device))
        if t.shape != shape:
            _fail("%s must have the shape %s, got %s" % (name, tuple(shape), tuple(t.shape)))
    st = t.stride()
    if st[-1] != 1 and shape[-1] != 1:
        _fail("the channels of %s must be dense" % name)
    return t.data_ptr(), st[0], st[1] if len(st) == 3 else 0


def _param(name, t, shape, like, dtype=torch.float32):
    """Checks a dense float32 (or ``dtype``) tensor and returns its pointer; None stays None."""
    if t is None:
        return None
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == like.get_device() and t.shape == shape and t.is_contiguous()):
        _fail("%s must be a dense %s tensor of shape %s on %s" % (name, dtype, tuple(shape), like.device))
    return t.data_ptr()


def _first(name, x, dims):
    if not (isinstance(x, torch.Tensor) and x.is_cuda):
        _fail("%s must be a CUDA tensor" % name)
    if x.dtype not in _DTYPE:
        _fail("%s must be float32 or bfloat16, got %s" % (name, x.dtype))
    if x.dim() not in dims:
        _fail("%s must have %s dimensions, got %d" % (name, " or ".join(str(d) for d in dims), x.dim()))
    if not 0 < x.numel() < 1 << 31 and max(x.shape) >= 1 << 31:          # (the library's sizes are 32-bit, and ctypes would cut them off)
        _fail("a dimension of %s reaches 2^31" % name)


def _call(fn, args, x):
    """Runs an entry point on the current stream of x's device (the library launches on the current device)."""
    index = x.get_device()
    if index == torch.cuda.current_device():
        status = fn(args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(args, _raw_stream(index))
    if status != _lib.ADN_OK:
        _lib.check(status)


def _floats(n, x):
    """(n floats or None, their address)"""
    if n < 0:
        _fail("sizes out of range")
    ws = x.new_empty(n, dtype=torch.float32) if n else None
    return ws, (ws.data_ptr() if n else None)


# ----------------------------------------------------------------------------------------------------------------- layer norm
def layer_norm_forward(x, gamma=None, beta=None, lens=None, eps=1e-5):
    """Layer norm over the last dimension of ``x`` (rows, channels) or (batch, time, channels), at most 16384 channels:
    ``(x - mean) inv_std gamma + beta`` with ``inv_std = 1 / sqrt(var + eps)``.  Returns ``(y, mean, inv_std)``; the statistics
    (float32, the shape of the rows) are what the backward pass needs.  The sum of a row's squared deviations has to be a float32 number
    (rows that spread past about 1e17 are outside)."""
    _first("x", x, (2, 3))
    if x.dim() == 2:
        y, mean, inv = layer_norm_forward(x[None], gamma, beta, lens, eps)
        return y[0], mean[0], inv[0]
    B, T, D = x.shape
    y = x.new_empty((B, T, D))
    mean, inv = x.new_empty((B, T), dtype=torch.float32), x.new_empty((B, T), dtype=torch.float32)
    args = NormArgs(_DTYPE[x.dtype], B, T, D, eps, 0, _param("lens", lens, (B,), x, torch.int32), *_activation("x", x, x.shape),
                    y.data_ptr(), T * D, D, _param("gamma", gamma, (D,), x), _param("beta", beta, (D,), x), mean.data_ptr(), inv.data_ptr())
    _call(_lib.load().adn_op_layer_norm_forward, args, x)
    return y, mean, inv


def layer_norm_backward(dy, x, gamma, mean, inv_std, lens=None):
    """``(dx, dgamma, dbeta)`` for the gradient ``dy`` of ``layer_norm_forward``'s result, from its ``x`` and statistics."""
    _first("x", x, (2, 3))
    if x.dim() == 2:
        _first("dy", dy, (2,))
        for name, t in (("mean", mean), ("inv_std", inv_std)):
            if t is None:
                _fail("the backward pass needs %s" % name)
            _param(name, t, x.shape[:1], x)
        dx, dgamma, dbeta = layer_norm_backward(dy[None], x[None], gamma, mean[None], inv_std[None], lens)
        return dx[0], dgamma, dbeta
    B, T, D = x.shape
    lib = _lib.load()
    dx = x.new_empty((B, T, D))
    dgamma, dbeta = x.new_empty(D, dtype=torch.float32), x.new_empty(D, dtype=torch.float32)
    n = lib.adn_op_layer_norm_workspace(B, T, D)
    ws, at = _floats(n, x)
    args = NormArgs(_DTYPE[x.dtype], B, T, D, 0.0, 0, _param("lens", lens, (B,), x, torch.int32), *_activation("x", x, x.shape), *_NO_SEQ,
                    _param("gamma", gamma, (D,), x), None, _param("mean", mean, (B, T), x), _param("inv_std", inv_std, (B, T), x),
                    *_activation("dy", dy, x.shape, x), dx.data_ptr(), T * D, D, dgamma.data_ptr(), dbeta.data_ptr(), at, n)
    _call(lib.adn_op_layer_norm_backward, args, x)
    return dx, dgamma, dbeta


# ---------------------------------------------------------------------------------------------------- short causal convolution
def _conv_args(x, weight, bias, lens, activation):
    if activation not in _ACTIVATION:
        _fail("activation must be 'silu' or 'linear', got %r" % (activation,))
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not 1 <= weight.shape[0] <= 8:
        _fail("weight must be (taps, channels) with 1 to 8 taps")
    D, K = x.shape[-1], weight.shape[0]
    return K, _ACTIVATION[activation], _param("weight", weight, (K, D), x), _param("bias", bias, (D,), x)


def causal_conv_forward(x, weight, bias=None, state=None, lens=None, activation="silu"):
    """Convolution of every channel of ``x`` (batch, time, channels) with its own taps over the frames up to and including its own:
    ``act(bias + sum_k weight[k] x[t - (taps - 1) + k])``, ``weight`` (taps <= 8, channels), ``activation`` 'silu' or 'linear'.
    ``state`` (batch, taps - 1, channels), in the type of ``x``: the frames before the first (None: zeros).  Returns ``(y, state)``
    with the last taps - 1 frames seen, to go on from."""
    _first("x", x, (3,))
    B, T, D = x.shape
    K, act, w, b = _conv_args(x, weight, bias, lens, activation)
    y, out = x.new_empty((B, T, D)), x.new_empty((B, K - 1, D))
    args = ConvArgs(_DTYPE[x.dtype], B, T, D, K, act, _param("lens", lens, (B,), x, torch.int32), *_activation("x", x, x.shape),
                    y.data_ptr(), T * D, D, w, b, _param("state", state, (B, K - 1, D), x, x.dtype), out.data_ptr())
    _call(_lib.load().adn_op_causal_conv_forward, args, x)
    return y, out


def causal_conv_backward(dy, x, weight, bias=None, state=None, lens=None, activation="silu"):
    """``(dx, dweight, dbias, dstate)`` for the gradient ``dy`` of ``causal_conv_forward``'s ``y``; ``dstate`` is None without a
    ``state``.  (The returned history is a copy of frames: its gradient, if any, is the caller's to add.)"""
    _first("x", x, (3,))
    B, T, D = x.shape
    K, act, w, b = _conv_args(x, weight, bias, lens, activation)
    lib = _lib.load()
    dx = x.new_empty((B, T, D))
    dw, db = x.new_empty((K, D), dtype=torch.float32), x.new_empty(D, dtype=torch.float32)
    dstate = None if state is None else x.new_empty((B, K - 1, D))
    n = lib.adn_op_causal_conv_workspace(B, T, D, K)
    ws, at = _floats(n, x)
    args = ConvArgs(_DTYPE[x.dtype], B, T, D, K, act, _param("lens", lens, (B,), x, torch.int32), *_activation("x", x, x.shape), *_NO_SEQ, w, b,
                    _param("state", state, (B, K - 1, D), x, x.dtype), None, *_activation("dy", dy, x.shape, x), dx.data_ptr(), T * D, D,
                    dw.data_ptr(), db.data_ptr(), None if dstate is None else dstate.data_ptr(), at, n)
    _call(lib.adn_op_causal_conv_backward, args, x)
    return dx, dw, db, dstate


def causal_conv_step(x, state, weight, bias=None, activation="silu"):
    """One frame ``x`` (batch, channels): returns ``y`` and moves ``state`` (batch, taps - 1, channels) on by the frame in place."""
    _first("x", x, (2,))
    B, D = x.shape
    K, act, w, b = _conv_args(x, weight, bias, None, activation)
    y = x.new_empty((B, D))
    if state is None:
        _fail("a step needs the state it moves on")
    args = ConvArgs(_DTYPE[x.dtype], B, 1, D, K, act, None, *_activation("x", x, x.shape), y.data_ptr(), D, D, w, b,
                    None, _param("state", state, (B, K - 1, D), x, x.dtype))
    _call(_lib.load().adn_op_causal_conv_step, args, x)
    return y


# ------------------------------------------------------------------------------------------------------ selective state-space scan
def _scan_rows(name, m, lead, D, N, u):
    """Checks B or C, (..., states) or (..., groups, states) with dense groups and states; returns (groups, pointer and strides)."""
    if not isinstance(m, torch.Tensor) or m.dtype is not u.dtype or m.get_device() != u.get_device():
        _fail("%s must be a %s tensor on %s" % (name, u.dtype, u.device))
    shape, st, k = m.shape, m.stride(), len(lead)
    if len(shape) == k + 1:
        G = 1
    elif len(shape) == k + 2:
        G = shape[-2]
        if G > 1 and st[-2] != N:
            _fail("the groups of %s must be dense" % name)
        if G < 1 or D % G:
            _fail("%d channels cannot be shared out over the %d groups of %s" % (D, G, name))
    else:
        _fail("%s must be (..., states) or (..., groups, states)" % name)
    if shape[:k] != lead or shape[-1] != N:
        _fail("%s must hold %d states for each of %s frames, got %s" % (name, N, tuple(lead), tuple(shape)))
    if st[-1] != 1 and N != 1:
        _fail("the states of %s must be dense" % name)
    return G, (m.data_ptr(), st[0], st[1] if k == 2 else 0)


def _scan_head(u, delta, A, Bm, Cm, D, z, delta_bias, lens, softplus, steps):
    """What every scan call starts its arguments with: sizes, activations, y's place left open."""
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or not 1 <= A.shape[1] <= 32:
        _fail("A must be (channels, states) with 1 to 32 states")
    ch, N = u.shape[-1], A.shape[1]
    lead = u.shape[:-1]
    G, b = _scan_rows("Bm", Bm, lead, ch, N, u)
    G2, c = _scan_rows("Cm", Cm, lead, ch, N, u)
    if G != G2:
        _fail("Bm has %d groups, Cm %d" % (G, G2))
    sizes = (_DTYPE[u.dtype], u.shape[0], steps, ch, N, G, 1 if softplus else 0, 0, _param("lens", lens, (u.shape[0],), u, torch.int32))
    seqs = _activation("u", u, u.shape) + _activation("delta", delta, u.shape, u) + b + c + (_NO_SEQ if z is None else _activation("z", z, u.shape, u))
    return sizes, seqs, (_param("A", A, (ch, N), u), _param("D", D, (ch,), u), _param("delta_bias", delta_bias, (ch,), u))


def selective_scan_forward(u, delta, A, Bm, Cm, D=None, z=None, delta_bias=None, state=None, lens=None, softplus=True, save=False):
    """The selective scan over ``u``, ``delta`` (batch, time, channels) with decays ``A`` (channels, states <= 32; finite) and input / output
    rows ``Bm``, ``Cm`` (batch, time, states) or (batch, time, groups, states)::

        dt = softplus(delta + delta_bias)          (softplus=False: the sum itself)
        h  = exp(dt A) h + dt u Bm;   y = sum_n h Cm + D u;   y *= z sigmoid(z)  if z is given

    A scan may grow (``A`` > 0, or steps below 0), as long as ``exp(dt A)`` of a frame and the states are float32 numbers.
    ``state`` (batch, channels, states), float32: the state to start from (None: zeros).  Returns ``(y, state, saved)``: the state behind
    the last valid frame and, with ``save=True``, what ``selective_scan_backward`` needs (else None)."""
    _first("u", u, (3,))
    sizes, seqs, params = _scan_head(u, delta, A, Bm, Cm, D, z, delta_bias, lens, softplus, u.shape[1])
    B, T, ch = u.shape
    N, G = sizes[4], sizes[5]
    lib = _lib.load()
    y, out = u.new_empty((B, T, ch)), u.new_empty((B, ch, N), dtype=torch.float32)
    saved, n = None, 0
    if save:
        n = lib.adn_op_selective_scan_checkpoints(B, T, ch, N, G)
        saved = u.new_empty(max(n, 0), dtype=torch.float32)
    m = lib.adn_op_selective_scan_workspace(B, T, ch, N, G, 0)
    ws, at = _floats(m, u)
    args = ScanArgs(*sizes, *seqs, y.data_ptr(), T * ch, ch, *params, _param("state", state, (B, ch, N), u), out.data_ptr(),
                    saved.data_ptr() if n else None, n, at, m)
    _call(lib.adn_op_selective_scan_forward, args, u)
    return y, out, saved


def selective_scan_backward(dy, u, delta, A, Bm, Cm, saved, D=None, z=None, delta_bias=None, state=None, lens=None, softplus=True, dlast=None):
    """Gradients for ``dy`` (of ``selective_scan_forward``'s ``y``) and ``dlast`` (of its state, or None), from the forward call's
    arguments and its ``saved``: a dict with ``du``, ``ddelta``, ``dz`` (None without a gate), ``dB``, ``dC``, ``dA``, ``dD``,
    ``ddelta_bias`` and ``dstate`` (None without a ``state``)."""
    _first("u", u, (3,))
    sizes, seqs, params = _scan_head(u, delta, A, Bm, Cm, D, z, delta_bias, lens, softplus, u.shape[1])
    B, T, ch = u.shape
    N, G = sizes[4], sizes[5]
    lib = _lib.load()
    n = lib.adn_op_selective_scan_checkpoints(B, T, ch, N, G)
    if saved is None:
        _fail("the backward pass needs what the forward pass saved (save=True)")
    _param("saved", saved, (n,), u)
    _param("state", state, (B, ch, N), u)
    du, ddelta, dz = u.new_empty((B, T, ch)), u.new_empty((B, T, ch)), None if z is None else u.new_empty((B, T, ch))
    dB, dC = u.new_empty(Bm.shape), u.new_empty(Cm.shape)
    dA, dD, dbias = u.new_empty((ch, N), dtype=torch.float32), u.new_empty(ch, dtype=torch.float32), u.new_empty(ch, dtype=torch.float32)
    dstate = None if state is None else u.new_empty((B, ch, N), dtype=torch.float32)
    m = lib.adn_op_selective_scan_workspace(B, T, ch, N, G, 1)
    ws, at = _floats(m, u)
    args = ScanArgs(*sizes, *seqs, *_NO_SEQ, *params, None, None, saved.data_ptr() if n else None, n, at, m,
                    *_activation("dy", dy, u.shape, u), du.data_ptr(), T * ch, ch, ddelta.data_ptr(), T * ch, ch,
                    *(_NO_SEQ if z is None else (dz.data_ptr(), T * ch, ch)), _param("dlast", dlast, (B, ch, N), u), dB.data_ptr(), dC.data_ptr(),
                    dA.data_ptr(), dD.data_ptr(), dbias.data_ptr(), None if dstate is None else dstate.data_ptr())
    _call(lib.adn_op_selective_scan_backward, args, u)
    return {"du": du, "ddelta": ddelta, "dz": dz, "dB": dB, "dC": dC, "dA": dA, "dD": dD, "ddelta_bias": dbias, "dstate": dstate}


def selective_scan_step(u, delta, A, Bm, Cm, state, D=None, z=None, delta_bias=None, softplus=True):
    """One frame: ``u``, ``delta``, ``z`` (batch, channels), ``Bm``, ``Cm`` (batch, states) or (batch, groups, states).  Returns ``y`` and
    moves ``state`` (batch, channels, states) on in place."""
    _first("u", u, (2,))
    sizes, seqs, params = _scan_head(u, delta, A, Bm, Cm, D, z, delta_bias, None, softplus, 1)
    B, ch = u.shape
    if state is None:
        _fail("a step needs the state it moves on")
    y = u.new_empty((B, ch))
    args = ScanArgs(*sizes, *seqs, y.data_ptr(), ch, ch, *params, None, _param("state", state, (B, ch, sizes[4]), u))
    _call(_lib.load().adn_op_selective_scan_step, args, u)
    return y
