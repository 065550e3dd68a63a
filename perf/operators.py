"""The cases on which the sequence operators of ``ip_avsr_amd.custom.sequence`` are measured: layer norm, the short causal
convolution and the selective state-space scan, each forward, in training (forward and backward) and, for the two with a state,
for single frames.

``run`` computes an operator in its plain form -- elementary torch operations in float32, the recurrence as a doubling scan over
the time axis -- or, where ``own`` is true, through the package.  ``exact`` restates the definitions in float64 (the recurrence
frame by frame, gradients by differentiation), apart from both.

Activations are (batch, time, channels) with the channels dense; where a block's projection makes several of them at once they
are column ranges of one wider array, as they are here.  Frames at and behind an utterance's length (``lens``) are padding: never
read, zero in every result.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
MOST_SCAN = 8 * 2048 * 2048 * 16        # states of the largest listed scan, a drawn one has no more
MOST_ROWS = 8 * 4096 * 4096             # elements of the largest listed norm / convolution
EPS = 1e-5


# ---------------------------------------------------------------------------------------------------------------- cases
def _case(op, mode, dtype, batch, steps, channels, **more):
    c = {"op": op, "mode": mode, "dtype": dtype, "batch": batch, "steps": steps, "channels": channels, "ragged": False}
    c.update({"layer_norm": {}, "causal_conv": {"taps": 4, "carried": False},
              "selective_scan": {"states": 16, "groups": 1, "gated": True, "carried": False}}[op])
    c.update(more)
    return c


def listed():
    return [
        # the 50-unit bottleneck of the AVLetters encoders over one minibatch of the reference's size (26 utterances, 40 frames)
        dict(_case("layer_norm", "train", "float32", 26, 40, 50, ragged=True), name="norm_train_minibatch"),
        # held-out split at once (520 utterances): the widest encoder layer's output, inference
        dict(_case("layer_norm", "forward", "bfloat16", 520, 40, 2000), name="norm_forward_split"),
        # the benchmark's batch, lengths U[12, 40]: the 1000-unit layer, one training step
        dict(_case("layer_norm", "train", "float32", 520, 40, 1000, ragged=True), name="norm_train_split"),
        # long recordings through a wide model: the bandwidth of both directions
        dict(_case("layer_norm", "train", "bfloat16", 8, 4096, 4096), name="norm_train_wide"),
        # one minibatch of 500-unit features: the cost of a small call
        dict(_case("causal_conv", "forward", "float32", 26, 40, 500), name="conv_forward_minibatch"),
        # the benchmark's batch of 1000-unit features with its lengths, one training step
        dict(_case("causal_conv", "train", "bfloat16", 520, 40, 1000, ragged=True), name="conv_train_split"),
        # long recordings, a wide model, a carried history
        dict(_case("causal_conv", "train", "bfloat16", 4, 4096, 4096, carried=True), name="conv_train_wide"),
        # live recognition of one speaker: one frame at a time
        dict(_case("causal_conv", "step", "bfloat16", 1, 1, 2048, carried=True), name="conv_step_one"),
        # live recognition of 64 speakers
        dict(_case("selective_scan", "step", "bfloat16", 64, 1, 2048, carried=True), name="scan_step_batch"),
        # one minibatch of 250-unit features (the width of the reference's LSTMs) with its lengths, one training step
        dict(_case("selective_scan", "train", "float32", 26, 40, 250, ragged=True, gated=False), name="scan_train_minibatch"),
        # one long recording: few rows, a long axis
        dict(_case("selective_scan", "forward", "bfloat16", 1, 8192, 2048, carried=True), name="scan_forward_long"),
        # a training step of a wide model
        dict(_case("selective_scan", "train", "bfloat16", 8, 2048, 2048), name="scan_train_wide"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "causal_conv", "selective_scan", "selective_scan"])
    mode = rng.choice(["forward", "train"] if op == "layer_norm" else ["forward", "train", "train", "step"])
    more = {}
    if op == "causal_conv":
        more = {"taps": rng.randint(2, 8), "carried": mode == "step" or rng.random() < 0.3}
    if op == "selective_scan":
        more = {"states": rng.choice([4, 8, 16, 16, 16, 24, 32, rng.randint(1, 32)]), "groups": rng.choice([1, 1, 2]),
                "gated": rng.random() < 0.6, "carried": mode == "step" or rng.random() < 0.3}
    most = MOST_SCAN // more["states"] if op == "selective_scan" else MOST_ROWS
    steps = 1 if mode == "step" else _log_int(rng, 1, 8192)
    channels = _log_int(rng, 16, 4096)
    channels += channels % more.get("groups", 1)
    batch = _log_int(rng, 1, max(1, min(520, most // (steps * channels))))
    steps = min(steps, max(1, most // (batch * channels)))
    return _case(op, mode, rng.choice(["float32", "bfloat16"]), batch, steps, channels, ragged=mode != "step" and rng.random() < 0.5, **more)


# --------------------------------------------------------------------------------------------------------------- inputs
def _lens(case, g):
    """Lengths as a padded minibatch has them: U[0.3 T, T] (12 to 40 of 40 frames), the first utterance the longest."""
    if not case["ragged"]:
        return None
    T = case["steps"]
    lens = torch.randint(int(math.ceil(0.3 * T)), T + 1, (case["batch"],), generator=g, device="cuda")
    lens[0] = T
    return lens.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    B, T, D = case["batch"], case["steps"], case["channels"]
    rn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")         # noqa: E731
    uni = lambda *shape: torch.rand(*shape, generator=g, device="cuda")         # noqa: E731
    s = {"case": dict(case), "lens": _lens(case, g)}
    if case["op"] == "layer_norm":
        s["x"] = (1.5 * rn(B, T, D) + 0.3 * rn(D)).to(dt)
        s["gamma"], s["beta"] = 1 + 0.1 * rn(D), 0.1 * rn(D)
    elif case["op"] == "causal_conv":
        K = case["taps"]
        both = rn(B, T, 2 * D).to(dt)                                            # [convolved | gate] columns of one projection
        s["x"] = both[..., :D]
        s["weight"], s["bias"] = rn(K, D) / math.sqrt(K), 0.1 * rn(D)
        s["state"] = rn(B, K - 1, D).to(dt) if case["carried"] else None
        if case["mode"] == "step":
            s["x"] = s["x"][:, 0]
    else:
        N, G = case["states"], case["groups"]
        both = rn(B, T, 2 * D).to(dt)
        s["u"] = torch.nn.functional.silu(rn(B, T, D)).to(dt)                    # what the convolution leaves
        s["z"] = both[..., D:] if case["gated"] else None
        s["delta"] = (0.5 * rn(B, T, D)).to(dt)
        bc = rn(B, T, 2 * G * N).to(dt)                                          # [B | C] columns of one projection
        s["Bm"], s["Cm"] = bc[..., :G * N].unflatten(-1, (G, N)), bc[..., G * N:].unflatten(-1, (G, N))
        s["A"] = -torch.arange(1, N + 1, device="cuda", dtype=torch.float32) * (0.75 + 0.5 * uni(D, N))
        s["D"] = 1 + 0.1 * rn(D)
        step = torch.exp(math.log(1e-3) + uni(D) * (math.log(0.1) - math.log(1e-3)))
        s["delta_bias"] = step + torch.log(-torch.expm1(-step))                  # softplus of it is `step`
        s["state"] = rn(B, D, N) if case["carried"] else None
        if case["mode"] == "step":
            for k in ("u", "z", "delta", "Bm", "Cm"):
                s[k] = None if s[k] is None else s[k][:, 0]
    if case["mode"] == "train":
        s["dy"] = rn(B, T, D).to(dt)
    return s


# ----------------------------------------------------------------------------------------------------------- plain forms
def _valid(s, T):
    """(batch, time, 1) truth values of the frames that are no padding, or None."""
    return None if s["lens"] is None else (torch.arange(T, device="cuda") < s["lens"][:, None])[..., None]


def _keep(valid, x):
    return x if valid is None else torch.where(valid, x, torch.zeros((), dtype=x.dtype, device=x.device))


def _plain_layer_norm(s):
    case, dt = s["case"], s["x"].dtype
    valid = _valid(s, case["steps"])
    x = _keep(valid, s["x"].float())
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    inv = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    xhat = xc * inv
    y = _keep(valid, xhat * s["gamma"] + s["beta"]).to(dt)
    out = {"y": y, "mean": _keep(valid, mean)[..., 0], "inv_std": _keep(valid, inv)[..., 0]}
    if case["mode"] == "train":
        dy = _keep(valid, s["dy"].float())
        gdy = dy * s["gamma"]
        dx = inv * (gdy - gdy.mean(-1, keepdim=True) - xhat * (gdy * xhat).mean(-1, keepdim=True))
        out.update(dx=_keep(valid, dx).to(dt), dgamma=(dy * xhat).sum((0, 1)), dbeta=dy.sum((0, 1)))
    return out


def _plain_conv(s):
    case, dt = s["case"], s["x"].dtype
    K, w, bias = case["taps"], s["weight"], s["bias"]
    if case["mode"] == "step":
        frames = torch.cat([s["state"], s["x"][:, None]], 1)
        pre = (frames.float() * w).sum(1) + bias
        s["state"].copy_(frames[:, 1:])
        return {"y": (pre * torch.sigmoid(pre)).to(dt), "state": s["state"]}
    T = case["steps"]
    valid = _valid(s, T)
    x = _keep(valid, s["x"])
    past = x.new_zeros(x.shape[0], K - 1, x.shape[2]) if s["state"] is None else s["state"]
    xp = torch.cat([past, x], 1)
    at = (torch.full((x.shape[0],), T, device="cuda") if s["lens"] is None else s["lens"].long())[:, None] + torch.arange(K - 1, device="cuda")
    state = torch.gather(xp, 1, at[..., None].expand(-1, -1, x.shape[2]))
    xf = xp.float()
    pre = bias + sum(w[k] * xf[:, k:k + T] for k in range(K))
    sg = torch.sigmoid(pre)
    out = {"y": _keep(valid, pre * sg).to(dt), "state": state}
    if case["mode"] == "train":
        dpre = _keep(valid, s["dy"].float() * sg * (1 + pre * (1 - sg)))
        dxp = torch.zeros_like(xf)
        for k in range(K):
            dxp[:, k:k + T] += w[k] * dpre
        out.update(dx=_keep(valid, dxp[:, K - 1:]).to(dt), dweight=torch.stack([(dpre * xf[:, k:k + T]).sum((0, 1)) for k in range(K)]),
                   dbias=dpre.sum((0, 1)))
        if s["state"] is not None:
            out["dstate"] = dxp[:, :K - 1].to(dt)
    return out


def _doubling(a, b):
    """h[t] = a[t] h[t - 1] + b[t] along dim 1 with h[-1] = 0, in log2(T) passes over both arrays."""
    shift = 1
    while shift < b.shape[1]:
        b = torch.cat([b[:, :shift], torch.addcmul(b[:, shift:], a[:, shift:], b[:, :-shift])], 1)
        if 2 * shift < b.shape[1]:
            a = torch.cat([a[:, :shift], a[:, shift:] * a[:, :-shift]], 1)
        shift *= 2
    return b


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20))))


def _per_channel(m, D):
    """(..., groups, states) -> (..., channels, states), the group's row for each of its channels."""
    return m.float().repeat_interleave(D // m.shape[-2], dim=-2)


def _plain_scan(s):
    case, dt = s["case"], s["u"].dtype
    D, A = case["channels"], s["A"]
    if case["mode"] == "step":
        step = _softplus(s["delta"].float() + s["delta_bias"])
        u = s["u"].float()
        h = torch.exp(step[..., None] * A) * s["state"] + (step * u)[..., None] * _per_channel(s["Bm"], D)
        y = (h * _per_channel(s["Cm"], D)).sum(-1) + s["D"] * u
        if s["z"] is not None:
            z = s["z"].float()
            y = y * z * torch.sigmoid(z)
        s["state"].copy_(h)
        return {"y": y.to(dt), "state": s["state"]}
    valid = _valid(s, case["steps"])
    u = _keep(valid, s["u"].float())
    pre = _keep(valid, s["delta"].float()) + s["delta_bias"]
    step = _keep(valid, _softplus(pre))                                          # a padding frame leaves the state as it is
    bm = _keep(valid if valid is None else valid[..., None], _per_channel(s["Bm"], D))
    cm = _keep(valid if valid is None else valid[..., None], _per_channel(s["Cm"], D))
    a = torch.exp(step[..., None] * A)
    inp = (step * u)[..., None] * bm
    if s["state"] is not None:
        inp[:, 0] += a[:, 0] * s["state"]
    h = _doubling(a, inp)
    del inp
    y_scan = (h * cm).sum(-1) + s["D"] * u
    if s["z"] is not None:
        z = _keep(valid, s["z"].float())
        sg = torch.sigmoid(z)
        y = y_scan * z * sg
    else:
        y = y_scan
    out = {"y": y.to(dt), "state": h[:, -1].contiguous()}
    if case["mode"] == "train":
        G = case["groups"]
        dy = _keep(valid, s["dy"].float())
        if s["z"] is not None:
            out["dz"] = (dy * y_scan * sg * (1 + z * (1 - sg))).to(dt)
            dy = dy * z * sg
        # dh[t] = dy[t] C[t] + a[t + 1] dh[t + 1]
        after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1).flip(1)
        dh = _doubling(after, (dy[..., None] * cm).flip(1)).flip(1)
        del after
        before = torch.zeros_like(h[:, :1]) if s["state"] is None else s["state"][:, None]
        decay = dh * a * torch.cat([before, h[:, :-1]], 1)                       # d loss / d (step A)
        split = lambda m: m.unflatten(2, (G, D // G)).sum(3)                     # noqa: E731  over a group's channels
        dstep = (decay * A).sum(-1) + (dh * bm).sum(-1) * u
        ddelta = _keep(valid, dstep * torch.sigmoid(pre))
        out.update(du=_keep(valid, (dh * bm).sum(-1) * step + s["D"] * dy).to(dt), ddelta=ddelta.to(dt), ddelta_bias=ddelta.sum((0, 1)),
                   dA=(decay * step[..., None]).sum((0, 1)), dD=(dy * u).sum((0, 1)),
                   dB=split(dh * (step * u)[..., None]).to(dt), dC=split(h * dy[..., None]).to(dt))
        if s["state"] is not None:
            out["dstate"] = a[:, 0] * dh[:, 0]
    return out


# -------------------------------------------------------------------------------------------------- the package's operators
def _own_layer_norm(s):
    from ip_avsr_amd.custom import sequence as S
    y, mean, inv_std = S.layer_norm_forward(s["x"], s["gamma"], s["beta"], lens=s["lens"], eps=EPS)
    out = {"y": y, "mean": mean, "inv_std": inv_std}
    if s["case"]["mode"] == "train":
        out["dx"], out["dgamma"], out["dbeta"] = S.layer_norm_backward(s["dy"], s["x"], s["gamma"], mean, inv_std, lens=s["lens"])
    return out


def _own_conv(s):
    from ip_avsr_amd.custom import sequence as S
    if s["case"]["mode"] == "step":
        return {"y": S.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], activation="silu"), "state": s["state"]}
    more = dict(state=s["state"], lens=s["lens"], activation="silu")
    y, state = S.causal_conv_forward(s["x"], s["weight"], s["bias"], **more)
    out = {"y": y, "state": state}
    if s["case"]["mode"] == "train":
        out["dx"], out["dweight"], out["dbias"], dstate = S.causal_conv_backward(s["dy"], s["x"], s["weight"], s["bias"], **more)
        if s["state"] is not None:
            out["dstate"] = dstate
    return out


def _own_scan(s):
    from ip_avsr_amd.custom import sequence as S
    more = dict(D=s["D"], z=s["z"], delta_bias=s["delta_bias"], softplus=True)
    if s["case"]["mode"] == "step":
        return {"y": S.selective_scan_step(s["u"], s["delta"], s["A"], s["Bm"], s["Cm"], s["state"], **more), "state": s["state"]}
    train = s["case"]["mode"] == "train"
    more.update(state=s["state"], lens=s["lens"])
    y, state, saved = S.selective_scan_forward(s["u"], s["delta"], s["A"], s["Bm"], s["Cm"], save=train, **more)
    out = {"y": y, "state": state}
    if train:
        grads = S.selective_scan_backward(s["dy"], s["u"], s["delta"], s["A"], s["Bm"], s["Cm"], saved, **more)
        out.update({k: v for k, v in grads.items() if v is not None})
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"layer_norm": _own_layer_norm, "causal_conv": _own_conv, "selective_scan": _own_scan}[op](state)
    return {"layer_norm": _plain_layer_norm, "causal_conv": _plain_conv, "selective_scan": _plain_scan}[op](state)


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    B, T, D = case["batch"], case["steps"], case["channels"]
    rows = B * T * (0.65 if case["ragged"] else 1.0)            # mean of U[0.3 T, T]: padding is neither read nor computed
    pad = B * T - rows                                          # ... but its zeros are written
    train, step = case["mode"] == "train", case["mode"] == "step"
    if case["op"] == "layer_norm":
        n, b = rows * D, 8 * D + 8 * B * T
        b += e * (2 * n + pad * D) + ((e * (3 * n + pad * D) + 12 * D) if train else 0)
        return {"bytes": b, "flops": n * (8 + (13 if train else 0))}
    if case["op"] == "causal_conv":
        K, n = case["taps"], rows * D
        state = e * B * (K - 1) * D
        b = 4 * (K + 1) * D + e * (2 * n + pad * D) + state * (2 if case["carried"] else 1)
        b += (e * (3 * n + pad * D) + 8 * (K + 1) * D + (2 * state if case["carried"] else 0)) if train else 0
        return {"bytes": b, "flops": n * (2 * K + 6 + (4 * K + 2 * K + 12 if train else 0))}
    N, G, z = case["states"], case["groups"], int(case["gated"])
    n, state = rows * D, 4 * B * D * N
    b = 4 * (D * N + 2 * D) + e * ((3 + z) * n + pad * D + 2 * rows * G * N) + state * (2 if case["carried"] else 1)
    if train:
        b += e * ((3 + z) * n + (2 + z) * (n + pad * D) + 2 * (rows + B * T) * G * N) + 4 * (2 * D * N + 4 * D) + (2 * state if case["carried"] else 0)
    return {"bytes": b, "flops": n * N * (7 + (24 if train else 0)) + n * (12 + (20 if train else 0))}


# ---------------------------------------------------------------------------------------------------------------- exact
def _exact_forward(case, s, p):
    """The definitions in float64: outputs of one pass as a function of the leaves `p`."""
    T = case["steps"]
    lens = torch.full((case["batch"],), T, device="cuda") if s["lens"] is None else s["lens"].long()
    if case["op"] == "layer_norm":
        on = (torch.arange(T, device="cuda") < lens[:, None])[..., None]
        x = torch.where(on, p["x"], torch.zeros_like(p["x"]))
        mean = x.mean(-1, keepdim=True)
        var = (x * x).mean(-1, keepdim=True) - mean * mean
        inv = (var + EPS) ** -0.5
        y = (x - mean) * inv * p["gamma"] + p["beta"]
        return {"y": y * on, "mean": (mean * on)[..., 0], "inv_std": (inv * on)[..., 0]}
    if case["op"] == "causal_conv":
        K, frames = case["taps"], (p["x"] if case["mode"] != "step" else p["x"][:, None]).unbind(1)
        past = list(p["state"].unbind(1)) if "state" in p else [torch.zeros_like(frames[0])] * (K - 1)
        hist, ys = past + list(frames), []
        for t in range(T):
            pre = p["bias"]
            for k in range(K):
                pre = pre + p["weight"][k] * hist[t + k]
            ys.append(pre / (1 + torch.exp(-pre)) * (t < lens)[:, None])
        idx = lens[:, None] + torch.arange(K - 1, device="cuda")
        state = torch.stack(hist, 1)[torch.arange(len(lens), device="cuda")[:, None], idx]
        return {"y": torch.stack(ys, 1) if case["mode"] != "step" else ys[0], "state": state}
    D, N, G = case["channels"], case["states"], case["groups"]
    seq = {k: (p[k] if case["mode"] != "step" else p[k][:, None]) for k in ("u", "delta", "Bm", "Cm", "z") if k in p}
    x = seq["delta"] + p["delta_bias"]
    dts = torch.where(x > 40, x, torch.log1p(torch.exp(x))).unbind(1)
    us, bs, cs = seq["u"].unbind(1), seq["Bm"].unbind(1), seq["Cm"].unbind(1)
    h = p["state"] if "state" in p else torch.zeros(case["batch"], D, N, device="cuda", dtype=torch.float64)
    ys = []
    for t in range(T):
        on = (t < lens)[:, None, None]
        b, c = (m[:, :, None].expand(-1, -1, D // G, -1).reshape(-1, D, N) for m in (bs[t], cs[t]))
        new = torch.exp(dts[t][..., None] * p["A"]) * h + (dts[t] * us[t])[..., None] * b
        h = new if s["lens"] is None else torch.where(on, new, h)
        ys.append(((h * c).sum(-1) + p["D"] * us[t]) * on[..., 0])
    y = torch.stack(ys, 1)
    if "z" in seq:
        y = y * seq["z"] / (1 + torch.exp(-seq["z"]))
    return {"y": y if case["mode"] != "step" else y[:, 0], "state": h}


def exact(case, seed):
    s = prepare(case, seed)
    names = {"layer_norm": ("x", "gamma", "beta"), "causal_conv": ("x", "weight", "bias", "state"),
             "selective_scan": ("u", "delta", "A", "Bm", "Cm", "D", "z", "delta_bias", "state")}[case["op"]]
    p = {k: s[k].double() for k in names if s[k] is not None}
    if case["mode"] != "train":
        with torch.no_grad():
            return _exact_forward(case, s, p)
    for v in p.values():
        v.requires_grad_(True)
    out = _exact_forward(case, s, p)
    on = 1.0 if s["lens"] is None else (torch.arange(case["steps"], device="cuda") < s["lens"][:, None])[..., None]
    grads = torch.autograd.grad((out["y"] * s["dy"].double() * on).sum(), list(p.values()))
    out = {k: v.detach() for k, v in out.items()}
    out.update({"d" + {"Bm": "B", "Cm": "C"}.get(k, k): g for k, g in zip(p, grads)})
    return out
