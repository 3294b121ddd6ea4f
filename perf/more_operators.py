"""Performance cases of the gated delta rule and of the product with its epilogue, through their public entry points.

  delta  ``gated_delta_rule`` over prompts, with the state before and after them
  step   ``gated_delta_rule_step`` for one token of each row, states updated in place
  mm     ``mm_bias_act``: a product with bias, residual and activation, from single rows to many

Where ``own`` is false the same is computed in its plain form, by elementary torch operations in 32 bits.
"""
import math

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZES = {"f16": 2, "bf16": 2, "f32": 4}
_NORM_EPS = 1e-6
_CHUNK = 64


def _delta(name, dtype, n, l, key_heads, heads, dk, dv, raw, norm, ragged):
    """raw: decays and step sizes as a projection leaves them (softplus and sigmoid within the call), else ready ones in fp32.
    norm: keys and queries of any length, normed within the call, else of length one."""
    return {"name": name, "kind": "delta", "dtype": dtype, "n": n, "l": l, "key_heads": key_heads, "heads": heads, "dk": dk, "dv": dv,
            "raw": raw, "norm": norm, "ragged": ragged}


def _step(name, dtype, n, key_heads, heads, dk, dv, raw, norm, slots):
    return {"name": name, "kind": "step", "dtype": dtype, "n": n, "key_heads": key_heads, "heads": heads, "dk": dk, "dv": dv,
            "raw": raw, "norm": norm, "slots": slots}


def _mm(name, dtype, m, k, n, linear, bias, residual, act):
    """linear: the second operand lies [n, k], as a linear layer's weight does, else [k, n]."""
    return {"name": name, "kind": "mm", "dtype": dtype, "m": m, "k": k, "n": n, "linear": linear, "bias": bias, "residual": residual,
            "act": act}


def listed():
    return [
        # a short question to a small model: launches, and the latency of two chunks
        _delta("delta_short_f16", "f16", 1, 100, 2, 4, 64, 64, True, True, False),
        # one long prompt
        _delta("delta_long_bf16", "bf16", 1, 8192, 16, 32, 128, 128, True, True, False),
        # ragged continuations of earlier prompts, a batch of them
        _delta("delta_batch_bf16", "bf16", 8, 1024, 16, 16, 128, 128, False, False, True),
        # heads that fit no tile, fp32
        _delta("delta_ragged_f32", "f32", 5, 333, 3, 6, 72, 100, True, True, True),
        # one user's next token
        _step("step_one_row_bf16", "bf16", 1, 16, 32, 128, 128, True, True, 8),
        # the next tokens of many users, whose states lie in a larger cache
        _step("step_many_rows_bf16", "bf16", 128, 16, 32, 128, 128, True, True, 160),
        # one user's next token through a mixer's last product, onto what goes around the mixer
        _mm("mm_one_row_bf16", "bf16", 1, 4096, 2048, False, False, True, "none"),
        # the next tokens of some users through a wide layer
        _mm("mm_few_rows_bf16", "bf16", 16, 4096, 8192, True, True, False, "gelu"),
        # sizes that fit no tile, fp32
        _mm("mm_ragged_f32", "f32", 5, 1001, 777, False, True, True, "relu"),
        # a short prompt through a mixer's first product
        _mm("mm_short_prompt_f16", "f16", 100, 2048, 4096, True, True, False, "none"),
        # long prompts through a wide layer
        _mm("mm_prompts_bf16", "bf16", 8192, 4096, 4096, False, True, True, "gelu_tanh"),
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
        # no larger than the largest listed case of its kind
        if case["kind"] == "delta":
            fits = case["n"] * case["l"] * case["heads"] * case["dk"] * case["dv"] <= 8192 * 32 * 128 * 128
        elif case["kind"] == "step":
            fits = case["n"] * case["heads"] * case["dk"] * case["dv"] <= 128 * 32 * 128 * 128
        else:
            fits = case["m"] * case["k"] * case["n"] <= 8192 * 4096 * 4096
        if fits:
            return case


def _draw(rng):
    kind = rng.choice(["delta", "delta", "delta", "step", "step", "mm", "mm"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "mm":
        case = _mm("", dtype, _log(rng, 1, 8192), _channels(rng, 64, 8192), _channels(rng, 64, 8192), rng.random() < 0.5, rng.random() < 0.6,
                   rng.random() < 0.5, rng.choice(["none", "none", "relu", "gelu", "gelu_tanh"]))
    else:
        key_heads, group = _log(rng, 1, 16), rng.choice([1, 1, 2, 4])
        dk, dv = (rng.choice([64, 128, 128, _channels(rng, 16, 128)]) for _ in range(2))
        raw, norm = rng.random() < 0.6, rng.random() < 0.6
        if kind == "delta":
            case = _delta("", dtype, _log(rng, 1, 16), _log(rng, 1, 8192), key_heads, key_heads * group, dk, dv, raw, norm, rng.random() < 0.5)
        else:
            n = _log(rng, 1, 512)
            case = _step("", dtype, n, key_heads, key_heads * group, dk, dv, raw, norm, n + rng.choice([0, 1, 64]))
    del case["name"]
    return case


def work(case):
    es = _SIZES[case["dtype"]]
    if case["kind"] == "mm":
        m, k, n = case["m"], case["k"], case["n"]
        values = m * k + k * n + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)
        return {"bytes": float(es * values), "flops": 2.0 * m * k * n}
    heads, dk, dv = case["heads"], case["dk"], case["dv"]
    tokens = case["n"] * case.get("l", 1)
    values = tokens * (2 * case["key_heads"] * dk + 2 * heads * dv)
    gates = tokens * 2 * heads * (es if case["raw"] else 4)
    # the state meets a key, takes a value times a key, and meets a query
    return {"bytes": float(es * values + gates + 2 * 4 * case["n"] * heads * dk * dv), "flops": 6.0 * tokens * heads * dk * dv}


def prepare(case, seed):
    dtype = _DTYPES[case["dtype"]]
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(shape, std=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device=device).mul_(std).add_(mean)

    def uniform(shape, low, high):
        return torch.rand(shape, generator=g, device=device).mul_(high - low).add_(low)

    state = {"case": case}
    if case["kind"] == "mm":
        m, k, n = case["m"], case["k"], case["n"]
        state["x"] = normal((m, k)).to(dtype)
        state["w"] = normal((n, k) if case["linear"] else (k, n), k ** -0.5).to(dtype)
        state["bias"] = normal((n,), 0.2).to(dtype) if case["bias"] else None
        state["residual"] = normal((m, n)).to(dtype) if case["residual"] else None
        return state
    n, heads, key_heads, dk, dv = (case[i] for i in ("n", "heads", "key_heads", "dk", "dv"))
    rows = (n, case["l"]) if case["kind"] == "delta" else (n,)
    for name in ("q", "k"):
        # keys of a head have something in common, as those behind an activation do
        x = normal((*rows, key_heads, dk)) + normal((key_heads, dk), 0.5)
        state[name] = (x if case["norm"] else x / (x * x).sum(-1, keepdim=True).sqrt()).to(dtype)
    state["v"] = normal((*rows, heads, dv)).to(dtype)
    if case["raw"]:
        # decay rates 1 .. 16 and steps of 0.001 .. 0.1, as such layers begin their training with
        dt = torch.exp(uniform((heads,), math.log(1e-3), math.log(1e-1)))
        state["delta_bias"] = dt + torch.log(-torch.expm1(-dt))
        state["A"] = -uniform((heads,), 1.0, 16.0)
        state["delta"], state["beta"] = normal((*rows, heads), 0.5).to(dtype), normal((*rows, heads)).to(dtype)
    else:
        state["delta_bias"] = state["A"] = None
        state["delta"], state["beta"] = -torch.exp(uniform((*rows, heads), -6.0, 0.5)), uniform((*rows, heads), 0.0, 1.0)
    if case["kind"] == "delta":
        state["before"] = normal((n, heads, dv, dk), 0.3)
        state["lengths"] = None
        if case["ragged"]:
            # whole prompts, shorter ones, and where there are several an empty one
            v = torch.randint(max(1, case["l"] // 2), case["l"] + 1, (n,), generator=g, device=device, dtype=torch.int32)
            v[0] = case["l"]
            if n > 2:
                v[-1] = 0
            state["lengths"] = v
    else:
        state["state"] = normal((case["slots"], heads, dv, dk), 0.3)
        state["slots"] = torch.randperm(case["slots"], generator=g, device=device)[:n].to(torch.int32)
    return state


def run(state):
    case = state["case"]
    return (_OWN if own else _PLAIN)[case["kind"]](state, case)


# ---- the framework's operators -------------------------------------------------------------------------------------


def _own_delta(s, case):
    import flagdnn_b200 as fd

    y, after = fd.gated_delta_rule(s["q"], s["k"], s["v"], s["delta"], s["beta"], A=s["A"], delta_bias=s["delta_bias"],
                                   delta_softplus=case["raw"], beta_sigmoid=case["raw"], qk_norm=case["norm"],
                                   initial_state=s["before"], lengths=s["lengths"], return_final_state=True)
    return {"y": y, "after": after}


def _own_step(s, case):
    import flagdnn_b200 as fd

    y = fd.gated_delta_rule_step(s["q"], s["k"], s["v"], s["delta"], s["beta"], s["state"], A=s["A"], delta_bias=s["delta_bias"],
                                 delta_softplus=case["raw"], beta_sigmoid=case["raw"], qk_norm=case["norm"], slots=s["slots"])
    return {"y": y, "state": s["state"]}


def _own_mm(s, case):
    import flagdnn_b200 as fd

    return fd.mm_bias_act(s["x"], s["w"].t() if case["linear"] else s["w"], s["bias"], residual=s["residual"], activation=case["act"])


_OWN = {"delta": _own_delta, "step": _own_step, "mm": _own_mm}


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _plain_gates(s, case):
    """Logarithms of the decays, and step sizes."""
    delta, beta = s["delta"].float(), s["beta"].float()
    if not case["raw"]:
        return delta, beta
    dt = delta + s["delta_bias"]
    return (dt.clamp_min(0) + torch.log1p(torch.exp(-dt.abs()))) * s["A"], 1 / (1 + torch.exp(-beta))


def _plain_heads(s, case):
    """q (scaled), k and v in fp32, one key and query per head."""
    q, k = s["q"].float(), s["k"].float()
    if case["norm"]:
        q, k = (x * torch.rsqrt((x * x).sum(-1, keepdim=True) + _NORM_EPS) for x in (q, k))
    group = case["heads"] // case["key_heads"]
    if group > 1:
        q, k = q.repeat_interleave(group, -2), k.repeat_interleave(group, -2)
    return q * case["dk"] ** -0.5, k, s["v"].float()


def _plain_delta(s, case):
    n, l, c = case["n"], case["l"], _CHUNK
    (q, k, v), (g, beta) = _plain_heads(s, case), _plain_gates(s, case)
    if s["lengths"] is not None:
        # a token that decays by nothing and writes nothing leaves the state as it is
        inside = (torch.arange(l, device=q.device) < s["lengths"][:, None])[:, :, None]
        g, beta = g * inside, beta * inside
    chunks = (l + c - 1) // c

    def cut(x):
        """[n, l, heads, ...] as [n, heads, chunks, c, ...], zeros behind the last token."""
        x = torch.cat([x, x.new_zeros(n, chunks * c - l, *x.shape[2:])], 1)
        return x.unflatten(1, (chunks, c)).movedim(3, 1)

    q, k, v, beta = cut(q), cut(k), cut(v), cut(beta)[..., None]
    total = cut(g).double().cumsum(-1)                       # far sums, near differences
    row = torch.arange(c, device=q.device)
    between = torch.exp(torch.where(row[:, None] >= row, total[..., :, None] - total[..., None, :], -math.inf).float())
    since, until = torch.exp(total.float())[..., None], between[..., -1, :, None]
    # u = beta (v - decayed state's answer to k - what the chunk's earlier tokens wrote): (1 + a) u = beta (v - ...), a strictly lower
    a = (k @ k.mT) * between * beta * (row[:, None] > row)
    inverse = torch.eye(c, device=q.device).expand_as(a)
    span = 1
    while span < c:                                          # diagonal blocks of twice the size with each round
        pairs = row // span
        below = (pairs[:, None] == pairs + 1) & (pairs % 2 == 0)
        inverse = inverse - inverse @ (a * below) @ inverse
        span *= 2
    u, w = inverse @ (beta * v), inverse @ (beta * since * k)
    # a chunk's end, [dk, dv]: keep @ the state before it + add
    late = k * until
    add = late.mT @ u
    keep = torch.eye(case["dk"], device=q.device) * since[..., -1:, :] - late.mT @ w
    add[:, :, 0] += keep[:, :, 0] @ s["before"].mT
    span = 1
    while span < chunks:                                     # all chunks behind spans of twice the length with each round
        add = torch.cat([add[:, :, :span], add[:, :, span:] + keep[:, :, span:] @ add[:, :, :-span]], 2)
        keep = torch.cat([keep[:, :, :span], keep[:, :, span:] @ keep[:, :, :-span]], 2)
        span *= 2
    first = torch.cat([s["before"].mT[:, :, None], add[:, :, :-1]], 2)
    y = (q * since) @ first + ((q @ k.mT) * between) @ (u - w @ first)
    y = y.movedim(1, 3).flatten(1, 2)[:, :l]
    if s["lengths"] is not None:
        y = y * inside[..., None]
    return {"y": y.to(s["v"].dtype), "after": add[:, :, -1].mT.contiguous()}


def _plain_step(s, case):
    (q, k, v), (g, beta) = _plain_heads(s, case), _plain_gates(s, case)
    slots = s["slots"].long()
    h = s["state"][slots] * torch.exp(g)[..., None, None]
    u = beta[..., None] * (v - (h @ k[..., None])[..., 0])
    h = h + u[..., None] * k[..., None, :]
    s["state"][slots] = h
    return {"y": (h @ q[..., None])[..., 0].to(s["v"].dtype), "state": s["state"]}


def _plain_mm(s, case):
    w = s["w"].float()
    y = s["x"].float() @ (w.t() if case["linear"] else w)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if case["act"] == "relu":
        y = y.clamp_min(0)
    elif case["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    elif case["act"] == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y.to(s["x"].dtype)


_PLAIN = {"delta": _plain_delta, "step": _plain_step, "mm": _plain_mm}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def exact(case, seed):
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in prepare(case, seed).items()}
    if case["kind"] == "mm":
        y = torch.einsum("mk,nk->mn" if case["linear"] else "mk,kn->mn", s["x"], s["w"])
        for term in (s["bias"], s["residual"]):
            if term is not None:
                y += term
        if case["act"] == "relu":
            return torch.relu(y)
        if case["act"] == "gelu":
            return y * torch.special.ndtr(y)
        if case["act"] == "gelu_tanh":
            # (1 + tanh(a)) / 2 is the logistic function of 2 a
            return y * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3))
        return y
    group = case["heads"] // case["key_heads"]
    q, k = s["q"], s["k"]
    if case["norm"]:
        q, k = q / (q.square().sum(-1, keepdim=True) + _NORM_EPS).sqrt(), k / (k.square().sum(-1, keepdim=True) + _NORM_EPS).sqrt()
    q, k = q.repeat_interleave(group, -2) / case["dk"] ** 0.5, k.repeat_interleave(group, -2)
    decay, beta = s["delta"], s["beta"]
    if case["raw"]:
        decay, beta = torch.nn.functional.softplus(decay + s["delta_bias"], threshold=1000) * s["A"], torch.sigmoid(beta)
    decay = decay.exp()
    if case["kind"] == "step":
        slots = s["slots"].long()
        y, s["state"][slots] = _exact_token(s["state"][slots], q, k, s["v"], decay, beta)
        return {"y": y, "state": s["state"]}
    h, y = s["before"], torch.zeros_like(s["v"])
    for t in range(case["l"]):
        out, new = _exact_token(h, q[:, t], k[:, t], s["v"][:, t], decay[:, t], beta[:, t])
        if s["lengths"] is None:
            y[:, t], h = out, new
        else:
            live = (t < s["lengths"])[:, None, None]
            y[:, t], h = torch.where(live, out, 0 * out), torch.where(live[..., None], new, h)
    return {"y": y, "after": h}


def _exact_token(h, q, k, v, decay, beta):
    """One token's output and the state after it, [.., dv, dk]."""
    h = h * decay[..., None, None]
    wrote = beta[..., None] * (v - torch.einsum("nhvk,nhk->nhv", h, k))
    h = h + torch.einsum("nhv,nhk->nhvk", wrote, k)
    return torch.einsum("nhvk,nhk->nhv", h, q), h
