"""Performance cases of the group norm and state space operators, through their public entry points.

  norm        ``group_norm`` over channels-last images and over rows of tokens
  norm_train  ``group_norm`` with its statistics, then ``group_norm_backward``: outputs and all gradients
  conv        ``causal_conv1d`` over prompts, with the state before and after them
  scan        ``selective_scan`` over prompts, with the state before and after them
  step        ``causal_conv1d_step`` and ``selective_scan_step`` for one token of each row, states updated in place

Where ``own`` is false the same is computed in its plain form, by elementary torch operations in 32 bits.
"""
import math

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZES = {"f16": 2, "bf16": 2, "f32": 4}
_EPS = 1e-5


def _norm(name, kind, dtype, n, c, h, w, groups, act):
    """h = w = 0: rows of tokens, x [n, c]."""
    return {"name": name, "kind": kind, "dtype": dtype, "n": n, "c": c, "h": h, "w": w, "groups": groups, "act": act}


def _conv(name, dtype, n, l, c, width, act, ragged):
    return {"name": name, "kind": "conv", "dtype": dtype, "n": n, "l": l, "c": c, "width": width, "act": act, "ragged": ragged}


def _scan(name, dtype, n, l, c, s, groups, gate, ragged):
    return {"name": name, "kind": "scan", "dtype": dtype, "n": n, "l": l, "c": c, "s": s, "groups": groups, "gate": gate,
            "ragged": ragged}


def _step(name, dtype, n, c, s, groups, width, slots):
    return {"name": name, "kind": "step", "dtype": dtype, "n": n, "c": c, "s": s, "groups": groups, "width": width, "slots": slots}


def listed():
    return [
        # one image behind a small layer: launches and host time are what it costs
        _norm("norm_one_image_f16", "norm", "f16", 1, 64, 14, 14, 16, "silu"),
        # a batch behind the wide convolutions of a network's second stage
        _norm("norm_images_bf16", "norm", "bf16", 32, 256, 56, 56, 32, "silu"),
        # channel counts and image sides that fit no tile, fp32
        _norm("norm_ragged_f32", "norm", "f32", 5, 90, 45, 37, 6, "none"),
        # a mixer's heads normalised per token, over many tokens
        _norm("norm_tokens_bf16", "norm", "bf16", 16384, 4096, 0, 0, 64, "none"),
        # a training step of an image network's layer
        _norm("norm_train_images_bf16", "norm_train", "bf16", 64, 256, 28, 28, 32, "silu"),
        # a training step of a mixer's norm, parameters in fp32 with the activations
        _norm("norm_train_tokens_f32", "norm_train", "f32", 4096, 2048, 0, 0, 32, "none"),
        # a batch of prompts
        _conv("conv_prompts_bf16", "bf16", 4, 2048, 4096, 4, "silu", False),
        # ragged continuations of earlier prompts
        _conv("conv_ragged_f32", "f32", 6, 777, 1000, 3, "none", True),
        # one long prompt
        _scan("scan_long_bf16", "bf16", 1, 8192, 4096, 16, 1, True, False),
        # ragged continuations, channels in two groups, fp32
        _scan("scan_ragged_f32", "f32", 7, 701, 1000, 16, 2, False, True),
        # one user's next token
        _step("step_one_row_bf16", "bf16", 1, 2048, 16, 1, 4, 8),
        # the next tokens of many users, whose states lie in a larger cache
        _step("step_many_rows_f16", "f16", 256, 4096, 16, 1, 4, 320),
    ]


def _log(rng, low, high):
    """An integer of [low, high], uniform in its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _channels(rng, low, high):
    """A channel count: mostly multiples of 8, as networks have them, one in four as it falls."""
    c = _log(rng, low, high)
    return c if rng.random() < 0.25 else max(8, c // 8 * 8)


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        # no larger than the largest listed case of its kind
        if case["kind"] == "scan":
            fits = case["n"] * case["l"] * case["c"] * case["s"] <= 8192 * 4096 * 16
        else:
            fits = w["bytes"] <= {"norm": 2.7e8, "norm_train": 1.7e8, "conv": 1.4e8, "step": 1.8e8}[case["kind"]]
        if fits:
            return case


def _draw(rng):
    kind = rng.choice(["norm", "norm", "norm_train", "norm_train", "conv", "conv", "scan", "scan", "scan", "step", "step"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("norm", "norm_train"):
        act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu", "silu"])
        if rng.random() < 0.4:
            groups = rng.choice([1, 4, 8, 32, 64])
            case = _norm("", kind, dtype, _log(rng, 1, 16384), groups * _channels(rng, 8, 512), 0, 0, groups, act)
        else:
            groups = rng.choice([4, 8, 16, 32])
            per = _log(rng, 1, 32)
            case = _norm("", kind, dtype, _log(rng, 1, 64), groups * per, _log(rng, 7, 112), _log(rng, 7, 112), groups, act)
    elif kind == "conv":
        case = _conv("", dtype, _log(rng, 1, 16), _log(rng, 1, 8192), _channels(rng, 64, 8192), rng.choice([2, 3, 4, 4]),
                     rng.choice(["none", "silu"]), rng.random() < 0.5)
    elif kind == "scan":
        groups = rng.choice([1, 1, 1, 2])
        case = _scan("", dtype, _log(rng, 1, 16), _log(rng, 1, 8192), groups * _channels(rng, 64, 4096), rng.choice([8, 16, 16, 16, 32, 64]),
                     groups, rng.random() < 0.7, rng.random() < 0.5)
    else:
        groups = rng.choice([1, 1, 1, 2])
        n = _log(rng, 1, 512)
        case = _step("", dtype, n, groups * _channels(rng, 64, 4096), rng.choice([8, 16, 16, 16, 32, 64]), groups, rng.choice([2, 3, 4, 4]),
                     n + rng.choice([0, 1, 64]))
    del case["name"]
    return case


def work(case):
    es, kind, n, c = _SIZES[case["dtype"]], case["kind"], case["n"], case["c"]
    if kind in ("norm", "norm_train"):
        values = n * c * max(1, case["h"] * case["w"])
        if kind == "norm":
            return {"bytes": float(es * (2 * values + 2 * c)), "flops": 8.0 * values}
        # forward x -> y, backward x, dy -> dx, and the gradients of the parameters
        return {"bytes": float(es * (5 * values + 6 * c) + 16 * n * case["groups"]), "flops": 24.0 * values}
    if kind == "conv":
        values, tail = n * case["l"] * c, n * (case["width"] - 1) * c
        return {"bytes": float(es * (2 * values + 2 * tail + c * (case["width"] + 1))), "flops": 2.0 * values * case["width"]}
    if kind == "scan":
        tokens, s = n * case["l"], case["s"]
        values = tokens * (c * (4 if case["gate"] else 3) + 2 * case["groups"] * s)
        return {"bytes": float(es * values + 4 * (2 * n * c * s + c * s + 2 * c)), "flops": 7.0 * tokens * c * s}
    s, width = case["s"], case["width"]
    values = n * (c * 6 + 2 * case["groups"] * s) + 2 * n * (width - 1) * c + c * (width + 1)
    return {"bytes": float(es * values + 4 * (2 * n * c * s + c * s + 2 * c)), "flops": 7.0 * n * c * s + 2.0 * n * c * width}


def prepare(case, seed):
    dtype = _DTYPES[case["dtype"]]
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(seed)
    kind, n, c = case["kind"], case["n"], case["c"]

    def normal(shape, std=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device=device).mul_(std).add_(mean)

    def uniform(shape, low, high):
        return torch.rand(shape, generator=g, device=device).mul_(high - low).add_(low)

    def lengths():
        # whole prompts, shorter ones, and where there are several an empty one
        v = torch.randint(max(1, case["l"] // 2), case["l"] + 1, (n,), generator=g, device=device, dtype=torch.int32)
        v[0] = case["l"]
        if n > 2:
            v[-1] = 0
        return v

    state = {"case": case}
    if kind in ("norm", "norm_train"):
        shape = (n, c, case["h"], case["w"]) if case["h"] else (n, c)
        fmt = torch.channels_last if case["h"] else torch.contiguous_format
        # activations with a mean of their own in every channel
        offset = normal((1, c) + (1,) * (len(shape) - 2), 0.5)
        state["x"] = (normal(shape) + offset).to(dtype).contiguous(memory_format=fmt)
        state["weight"] = normal((c,), 0.2, 1.0).to(dtype)
        state["bias"] = normal((c,), 0.2).to(dtype)
        if kind == "norm_train":
            state["dy"] = normal(shape).to(dtype).contiguous(memory_format=fmt)
        return state
    if kind == "conv":
        state["x"] = normal((n, case["l"], c)).to(dtype)
        state["weight"] = normal((c, case["width"]), case["width"] ** -0.5).to(dtype)
        state["bias"] = normal((c,), 0.1).to(dtype)
        state["before"] = normal((n, case["width"] - 1, c)).to(dtype)
        state["lengths"] = lengths() if case["ragged"] else None
        return state
    s, groups = case["s"], case["groups"]
    # decay rates 1 .. s and steps of 0.001 .. 0.1, as such layers begin their training with
    state["A"] = -torch.arange(1, s + 1, device=device, dtype=torch.float32).repeat(c, 1) * uniform((c, 1), 0.7, 1.3)
    state["D"] = normal((c,), 0.2, 1.0)
    dt = torch.exp(uniform((c,), math.log(1e-3), math.log(1e-1)))
    state["delta_bias"] = dt + torch.log(-torch.expm1(-dt))
    rows = (n, case["l"]) if kind == "scan" else (n,)
    state["u"] = normal(rows + (c,)).to(dtype)
    state["delta"] = normal(rows + (c,), 0.5).to(dtype)
    state["B"] = normal(rows + (groups, s)).to(dtype)
    state["C"] = normal(rows + (groups, s)).to(dtype)
    state["z"] = normal(rows + (c,)).to(dtype) if kind == "step" or case["gate"] else None
    if kind == "scan":
        state["before"] = normal((n, c, s), 0.5)
        state["lengths"] = lengths() if case["ragged"] else None
        return state
    width = case["width"]
    state["x"] = normal((n, c)).to(dtype)
    state["weight"] = normal((c, width), width ** -0.5).to(dtype)
    state["bias"] = normal((c,), 0.1).to(dtype)
    state["conv_state"] = normal((case["slots"], width - 1, c)).to(dtype)
    state["scan_state"] = normal((case["slots"], c, s), 0.5)
    state["slots"] = torch.randperm(case["slots"], generator=g, device=device)[:n].to(torch.int32)
    return state


def run(state):
    case = state["case"]
    return (_OWN if own else _PLAIN)[case["kind"]](state, case)


# ---- the framework's operators -------------------------------------------------------------------------------------


def _own_norm(s, case):
    import flagdnn_b200 as fd

    return fd.group_norm(s["x"], case["groups"], s["weight"], s["bias"], _EPS, activation=case["act"])


def _own_norm_train(s, case):
    import flagdnn_b200 as fd

    y, mean, rstd = fd.group_norm(s["x"], case["groups"], s["weight"], s["bias"], _EPS, activation=case["act"], return_stats=True)
    dx, dw, db = fd.group_norm_backward(s["dy"], s["x"], mean, rstd, case["groups"], s["weight"], s["bias"], activation=case["act"])
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db}


def _own_conv(s, case):
    import flagdnn_b200 as fd

    y, after = fd.causal_conv1d(s["x"], s["weight"], s["bias"], activation=case["act"], initial_state=s["before"],
                                lengths=s["lengths"], return_final_state=True)
    return {"y": y, "after": after}


def _own_scan(s, case):
    import flagdnn_b200 as fd

    y, after = fd.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], delta_bias=s["delta_bias"],
                                 delta_softplus=True, initial_state=s["before"], lengths=s["lengths"], return_final_state=True)
    return {"y": y, "after": after}


def _own_step(s, case):
    # (the products between the two are the program's own, so that each has inputs of its own here)
    import flagdnn_b200 as fd

    v = fd.causal_conv1d_step(s["x"], s["conv_state"], s["weight"], s["bias"], activation="silu", slots=s["slots"])
    y = fd.selective_scan_step(s["u"], s["delta"], s["A"], s["B"], s["C"], s["scan_state"], D=s["D"], z=s["z"],
                               delta_bias=s["delta_bias"], delta_softplus=True, slots=s["slots"])
    return {"v": v, "y": y, "conv_state": s["conv_state"], "scan_state": s["scan_state"]}


_OWN = {"norm": _own_norm, "norm_train": _own_norm_train, "conv": _own_conv, "scan": _own_scan, "step": _own_step}


# ---- the plain forms -----------------------------------------------------------------------------------------------

_SQRT_HALF, _SQRT_2_PI, _CUBIC = math.sqrt(0.5), math.sqrt(2 / math.pi), 0.044715


def _act(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * _SQRT_HALF))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(_SQRT_2_PI * (v + _CUBIC * v * v * v)))
    return v


def _act_slope(v, act):
    if act == "relu":
        return (v > 0).to(v.dtype)
    if act == "silu":
        p = 1 / (1 + torch.exp(-v))
        return p * (1 + v * (1 - p))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(v * _SQRT_HALF)) + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        t = torch.tanh(_SQRT_2_PI * (v + _CUBIC * v * v * v))
        return 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * _SQRT_2_PI * (1 + 3 * _CUBIC * v * v)
    return torch.ones_like(v)


def _split(x, case):
    """[n, c, h, w] or [n, c] as fp32 [n, pixels, groups, channels of a group]."""
    v = x.movedim(1, -1) if case["h"] else x
    return v.reshape(case["n"], -1, case["groups"], case["c"] // case["groups"]).float()


def _joined(v, like, case):
    v = v.to(like.dtype)
    return v.reshape(case["n"], case["h"], case["w"], case["c"]).movedim(-1, 1) if case["h"] else v.reshape(case["n"], case["c"])


def _plain_norm_parts(s, case):
    x = _split(s["x"], case)
    mean = x.mean((1, 3), keepdim=True)
    x = x - mean
    rstd = torch.rsqrt((x * x).mean((1, 3), keepdim=True) + _EPS)
    w = s["weight"].float().view(case["groups"], -1)
    normed = x * rstd
    return normed, rstd, w, normed * w + s["bias"].float().view(case["groups"], -1)


def _plain_norm(s, case):
    return _joined(_act(_plain_norm_parts(s, case)[3], case["act"]), s["x"], case)


def _plain_norm_train(s, case):
    normed, rstd, w, v = _plain_norm_parts(s, case)
    y = _act(v, case["act"])
    grad = _split(s["dy"], case) * _act_slope(v, case["act"])
    gw = grad * w
    dx = rstd * (gw - gw.mean((1, 3), keepdim=True) - normed * (gw * normed).mean((1, 3), keepdim=True))
    dw, db = (grad * normed).sum((0, 1)).view(-1), grad.sum((0, 1)).view(-1)
    return {"y": _joined(y, s["x"], case), "dx": _joined(dx, s["x"], case), "dweight": dw.to(s["weight"].dtype),
            "dbias": db.to(s["bias"].dtype)}


def _plain_conv(s, case):
    x, w = s["x"], s["weight"].float()
    n, l, c, width = case["n"], case["l"], case["c"], case["width"]
    if s["lengths"] is not None:
        inside = (torch.arange(l, device=x.device) < s["lengths"][:, None])[:, :, None]
        x = torch.where(inside, x, torch.zeros((), dtype=x.dtype, device=x.device))
    xs = torch.cat([s["before"], x], 1)
    y = _act((xs.unfold(1, width, 1).float() * w).sum(-1) + s["bias"].float(), case["act"])
    if s["lengths"] is None:
        return {"y": y.to(x.dtype), "after": xs[:, l:].contiguous()}
    at = s["lengths"].long()[:, None] + torch.arange(width - 1, device=x.device)
    after = torch.gather(xs, 1, at[:, :, None].expand(n, width - 1, c))
    return {"y": torch.where(inside, y, torch.zeros((), device=x.device)).to(x.dtype), "after": after}


def _plain_dt(s):
    dt = s["delta"].float() + s["delta_bias"]
    return dt.clamp_min(0) + torch.log1p(torch.exp(-dt.abs()))


def _plain_scan(s, case):
    n, l, c, groups = case["n"], case["l"], case["c"], case["groups"]
    u, dt = s["u"].float(), _plain_dt(s)
    if s["lengths"] is not None:
        inside = (torch.arange(l, device=u.device) < s["lengths"][:, None])[:, :, None]
        dt = torch.where(inside, dt, torch.zeros((), device=u.device))  # a step of no time leaves the state as it is
    per = c // groups
    rows = s["B"].float().repeat_interleave(per, 2) if groups > 1 else s["B"].float()
    decay = torch.exp(dt[..., None] * s["A"])
    h = (dt * u)[..., None] * rows
    h[:, 0] += decay[:, 0] * s["before"]
    # h_t = decay_t h_(t-1) + h_t over all t: spans of twice the length with each round
    span = 1
    while span < l:
        h = torch.cat([h[:, :span], h[:, span:] + decay[:, span:] * h[:, :-span]], 1)
        decay = torch.cat([decay[:, :span], decay[:, span:] * decay[:, :-span]], 1)
        span *= 2
    rows = s["C"].float().repeat_interleave(per, 2) if groups > 1 else s["C"].float()
    y = (h * rows).sum(-1) + s["D"] * u
    if s["z"] is not None:
        y = y * _act(s["z"].float(), "silu")
    if s["lengths"] is not None:
        y = torch.where(inside, y, torch.zeros((), device=u.device))
    return {"y": y.to(s["u"].dtype), "after": h[:, -1].contiguous()}


def _plain_step(s, case):
    slots, groups = s["slots"].long(), case["groups"]
    xs = torch.cat([s["conv_state"][slots], s["x"][:, None]], 1)
    v = _act((xs.float() * s["weight"].float().t()).sum(1) + s["bias"].float(), "silu")
    s["conv_state"][slots] = xs[:, 1:]
    u, dt = s["u"].float(), _plain_dt(s)
    per = case["c"] // groups
    decay = torch.exp(dt[..., None] * s["A"])
    h = decay * s["scan_state"][slots] + (dt * u)[..., None] * s["B"].float().repeat_interleave(per, 1)
    s["scan_state"][slots] = h
    y = (h * s["C"].float().repeat_interleave(per, 1)).sum(-1) + s["D"] * u
    y = y * _act(s["z"].float(), "silu")
    return {"v": v.to(s["x"].dtype), "y": y.to(s["u"].dtype), "conv_state": s["conv_state"], "scan_state": s["scan_state"]}


_PLAIN = {"norm": _plain_norm, "norm_train": _plain_norm_train, "conv": _plain_conv, "scan": _plain_scan, "step": _plain_step}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def exact(case, seed):
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in prepare(case, seed).items()}
    kind = case["kind"]
    if kind in ("norm", "norm_train"):
        return _exact_norm(case, s)
    if kind == "conv":
        return _exact_conv(case, s)
    if kind == "scan":
        return _exact_scan(case, s)
    return _exact_step(case, s)


def _exact_value_and_slope(v, act):
    one = torch.ones_like(v)
    if act == "relu":
        return torch.relu(v), torch.heaviside(v, 0 * one)
    if act == "silu":
        p = torch.sigmoid(v)
        return v * p, p + v * p * torch.sigmoid(-v)
    if act == "gelu":
        p = torch.special.ndtr(v)
        return v * p, p + v * torch.exp(-v.square() / 2) / (2 * math.pi) ** 0.5
    if act == "gelu_tanh":
        # (1 + tanh(a)) / 2 is the logistic function of 2 a
        a = 2 * (2 / math.pi) ** 0.5 * (v + 0.044715 * v ** 3)
        p = torch.sigmoid(a)
        return v * p, p + v * p * torch.sigmoid(-a) * 2 * (2 / math.pi) ** 0.5 * (1 + 3 * 0.044715 * v ** 2)
    return v, one


def _exact_norm(case, s):
    n, c, groups = case["n"], case["c"], case["groups"]
    shape = s["x"].shape
    x = s["x"].reshape(n, groups, -1)                      # logical order: a group's channels, then its pixels
    var, mean = torch.var_mean(x, 2, unbiased=False, keepdim=True)
    scale = (var + _EPS) ** -0.5
    normed = ((x - mean) * scale).reshape(n, c, -1)
    v, slope = _exact_value_and_slope(normed * s["weight"][None, :, None] + s["bias"][None, :, None], case["act"])
    if case["kind"] == "norm":
        return v.reshape(shape)
    grad = s["dy"].reshape(n, c, -1) * slope
    dw, db = torch.einsum("ncp,ncp->c", grad, normed), torch.einsum("ncp->c", grad)
    back = (grad * s["weight"][None, :, None]).reshape(n, groups, -1)
    normed = normed.reshape(n, groups, -1)
    m = back.shape[2]
    dx = scale * (back - back.sum(2, keepdim=True) / m - normed * (back * normed).sum(2, keepdim=True) / m)
    return {"y": v.reshape(shape), "dx": dx.reshape(shape), "dweight": dw, "dbias": db}


def _exact_conv(case, s):
    n, l, width = case["n"], case["l"], case["width"]
    y, after = torch.zeros_like(s["x"]), torch.empty_like(s["before"])
    for i in range(n):
        end = l if s["lengths"] is None else int(s["lengths"][i])
        line = torch.cat([s["before"][i], s["x"][i, :end]])
        v = s["bias"].expand(end, -1).clone()
        for j in range(width):
            v += line[j:j + end] * s["weight"][:, j]
        y[i, :end] = _exact_value_and_slope(v, case["act"])[0]
        after[i] = line[end:]
    return {"y": y, "after": after}


def _exact_scan(case, s):
    groups, per = case["groups"], case["c"] // case["groups"]
    h = s["before"].clone()
    dt = torch.nn.functional.softplus(s["delta"] + s["delta_bias"], threshold=1000)
    y = torch.zeros_like(s["u"])
    for t in range(case["l"]):
        d, u = dt[:, t, :, None], s["u"][:, t]
        new = h * torch.exp(d * s["A"]) + d * u[:, :, None] * s["B"][:, t].repeat_interleave(per, 1)
        out = torch.einsum("ngps,ngs->ngp", new.unflatten(1, (groups, per)), s["C"][:, t]).flatten(1) + s["D"] * u
        if s["z"] is not None:
            out = out * s["z"][:, t] * torch.sigmoid(s["z"][:, t])
        if s["lengths"] is None:
            h, y[:, t] = new, out
        else:
            live = (t < s["lengths"])[:, None]
            h, y[:, t] = torch.where(live[:, :, None], new, h), torch.where(live, out, 0 * out)
    return {"y": y, "after": h}


def _exact_step(case, s):
    conv_state, scan_state = s["conv_state"].clone(), s["scan_state"].clone()
    slots, per = s["slots"].long(), case["c"] // case["groups"]
    old = conv_state[slots]
    v = s["bias"] + s["x"] * s["weight"][:, -1] + torch.einsum("njc,cj->nc", old, s["weight"][:, :-1])
    conv_state[slots] = torch.cat([old[:, 1:], s["x"][:, None]], 1)
    dt = torch.nn.functional.softplus(s["delta"] + s["delta_bias"], threshold=1000)[:, :, None]
    h = scan_state[slots] * torch.exp(dt * s["A"]) + dt * s["u"][:, :, None] * s["B"].repeat_interleave(per, 1)
    scan_state[slots] = h
    y = torch.einsum("ncs,ncs->nc", h, s["C"].repeat_interleave(per, 1)) + s["D"] * s["u"]
    return {"v": v * torch.sigmoid(v), "y": y * s["z"] * torch.sigmoid(s["z"]), "conv_state": conv_state, "scan_state": scan_state}
