"""causal_conv1d, selective_scan and their single-token forms against their definitions in 64 bits.

Tolerances.  Outputs are rounded once to their type (unit roundoff 2^-8 bf16, 2^-11 f16, 2^-24 f32).  A convolution adds up to
eight fp32 products: 2e-5 of the sum of their sizes, taken as 2e-5 (1 + |y|).  A scan multiplies a state by one rounded decay
a token (relative error 2^-21 with its exponent's rounding): l * 2^-21 of the state, at most, and the same of an output's sum of
terms; 2e-4 (l = 400), more for longer prompts."""
import pytest
import torch

from oracle import sequence_oracle as so

pytestmark = pytest.mark.gpu

ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "f16", "f32"]


@pytest.fixture(scope="module")
def fd(native_lib):
    import flagdnn_b200

    assert torch.cuda.is_available()
    return flagdnn_b200


def near(got, want, dtype, tol):
    got = got.double().cpu()
    assert got.shape == want.shape
    bad = (got - want).abs() > (1.02 * ROUND[dtype] + tol) * want.abs() + tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((got - want).abs().max())}"


def rand(gen, shape, dtype, std=1.0, wide=0, odd=False, spread=False):
    """A tensor whose last dimension is dense, a slice of `wide` more columns, at an odd address, or strided."""
    t = (torch.randn(shape, generator=gen) * std).to(dtype).cuda()
    if wide:
        big = torch.full((*shape[:-1], shape[-1] + wide), float("nan"), dtype=dtype, device="cuda")
        big[..., wide // 2:wide // 2 + shape[-1]] = t
        return big[..., wide // 2:wide // 2 + shape[-1]]
    if odd:
        flat = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        return flat[1:].view(shape)
    if spread:
        return t.transpose(-1, -2).contiguous().transpose(-1, -2)
    return t


LAYOUTS = {"dense": {}, "slice": {"wide": 16}, "ragged slice": {"wide": 6}, "odd": {"odd": True}, "strided": {"spread": True}}

CONVS = [   # n, l, c, width, layout, lengths
    (1, 1, 8, 4, "dense", None),
    (2, 37, 64, 4, "dense", None),
    (3, 130, 100, 3, "dense", [130, 0, 1]),
    (4, 65, 33, 2, "odd", [2, 64, 65, 1]),
    (2, 50, 72, 4, "slice", [50, 3]),
    (2, 50, 72, 4, "ragged slice", None),
    (2, 41, 24, 8, "strided", [41, 5]),
    (1, 300, 520, 4, "dense", None),
    (2, 9, 16, 1, "dense", [9, 4]),
    (5, 2, 256, 4, "dense", [2, 1, 0, 2, 1]),
    (2, 0, 16, 4, "dense", None),
    (2, 200, 2048, 4, "dense", [200, 77]),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("case", CONVS, ids=[f"{n}x{l}x{c}w{w}{k}" for n, l, c, w, k, _ in CONVS])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_causal_conv1d(fd, case, dtype, act):
    n, l, c, width, layout, lengths = case
    g = torch.Generator().manual_seed(l)
    x = rand(g, (n, l, c), dtype, **(LAYOUTS[layout] if l else {}))
    w, b = rand(g, (c, width), dtype, width ** -0.5), rand(g, (c,), dtype, 0.1)
    before = rand(g, (n, width - 1, c), dtype)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if lengths is not None:
        for i, end in enumerate(lengths):
            x[i, end:] = float("nan")            # padding is never read
    for initial, bias in ((before, b), (None, None)):
        want, final = so.causal_conv1d(x, w, bias, act, initial, lengths)
        y, got_final = fd.causal_conv1d(x, w, bias, act, initial, lens, return_final_state=True)
        near(y, want, dtype, 2e-5)
        assert torch.equal(got_final.double().cpu(), final)
        assert torch.equal(y, fd.causal_conv1d(x, w[:, None], bias, act, initial, lens))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,c,width,slots", [(1, 8, 4, None), (3, 100, 3, [4, 0, 2]), (4, 33, 2, [1, -1, 9, 0]), (2, 16, 1, None),
                                             (70, 520, 4, "all"), (5, 2048, 8, "all")])
def test_causal_conv1d_step(fd, n, c, width, slots, dtype):
    g = torch.Generator().manual_seed(c)
    cache = n + 3
    x, state = rand(g, (n, c), dtype, wide=6), rand(g, (cache, width - 1, c), dtype)
    w, b = rand(g, (c, width), dtype, width ** -0.5), rand(g, (c,), dtype, 0.1)
    at = list(range(n)) if slots is None else torch.randperm(cache, generator=g)[:n].tolist() if slots == "all" else slots
    where = None if slots is None else torch.tensor(at, dtype=torch.int32, device="cuda")
    before = state.clone()
    y = fd.causal_conv1d_step(x, state, w, b, "silu", where)
    live = [i for i in range(n) if 0 <= at[i] < cache]
    want, final = so.causal_conv1d(x[live][:, None], w, b, "silu", before[[at[i] for i in live]])
    near(y[live], want[:, 0], dtype, 2e-5)
    after = before.clone()
    after[[at[i] for i in live]] = final.to(dtype).cuda()
    assert torch.equal(state, after)
    idle = [i for i in range(n) if i not in live]
    assert not y[idle].any()


def scan_inputs(g, n, l, c, s, groups, dtype, layout="dense"):
    rows = (n, l) if l is not None else (n,)
    lay = LAYOUTS[layout] if l != 0 else {}
    v = {"u": rand(g, (*rows, c), dtype, **lay), "delta": rand(g, (*rows, c), dtype, 0.5, **lay), "z": rand(g, (*rows, c), dtype, **lay),
         "B": rand(g, (*rows, groups, s), dtype, **lay), "C": rand(g, (*rows, groups, s), dtype, **lay)}
    v["A"] = -(torch.arange(1, s + 1).float().repeat(c, 1) * (0.5 + torch.rand(c, 1, generator=g))).cuda()
    v["D"] = torch.randn(c, generator=g).cuda()
    v["delta_bias"] = (torch.rand(c, generator=g) * 4 - 6).cuda()
    return v


SCANS = [   # n, l, c, s, groups, layout, lengths
    (1, 1, 8, 16, 1, "dense", None),
    (2, 37, 64, 16, 1, "dense", None),
    (3, 130, 100, 16, 2, "dense", [130, 0, 1]),
    (4, 65, 33, 8, 1, "odd", [2, 64, 65, 1]),
    (2, 50, 72, 16, 1, "slice", [50, 3]),
    (2, 50, 72, 16, 3, "ragged slice", None),
    (2, 41, 24, 4, 1, "strided", [41, 5]),
    (1, 400, 40, 16, 1, "dense", None),
    (1, 390, 130, 16, 1, "dense", [333]),
    (2, 23, 20, 5, 1, "dense", None),
    (2, 30, 12, 32, 2, "dense", None),
    (1, 100, 6, 64, 1, "dense", None),
    (1, 20, 4, 100, 1, "dense", None),
    (1, 33, 3, 256, 1, "dense", None),
    (2, 15, 5, 1, 5, "dense", None),
    (2, 0, 16, 16, 1, "dense", None),
    (5, 129, 256, 16, 1, "dense", [129, 128, 127, 32, 33]),
    (1, 260, 1030, 16, 1, "dense", None),
    (2, 70, 72, 16, 2, "dense", [70, 40]),             # 36 channels a group: eights and four
    (2, 45, 40, 8, 2, "slice", None),
    (2, 2500, 40, 16, 1, "dense", [2500, 700]),       # rows in chunks
    (1, 2100, 24, 64, 2, "slice", None),
    (3, 1500, 9, 5, 1, "odd", [0, 1500, 130]),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("case", SCANS, ids=[f"{n}x{l}x{c}s{s}g{g}{k}" for n, l, c, s, g, k, _ in SCANS])
def test_selective_scan(fd, case, dtype):
    n, l, c, s, groups, layout, lengths = case
    g = torch.Generator().manual_seed(l + s)
    v = scan_inputs(g, n, l, c, s, groups, dtype, layout)
    before = torch.randn(n, c, s, generator=g).cuda()
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if lengths is not None:
        for i, end in enumerate(lengths):
            for name in ("u", "delta", "z", "B", "C"):
                v[name][i, end:] = float("nan")
    want, final = so.selective_scan(v["u"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], v["delta_bias"], True, before, lengths)
    y, got_final = fd.selective_scan(**v, delta_softplus=True, initial_state=before, lengths=lens, return_final_state=True)
    tol = max(2e-4, l * 2.0 ** -21)
    near(got_final, final, torch.float32, tol)
    near(y, want, dtype, tol * s ** 0.5)
    assert torch.equal(y, fd.selective_scan(**v, delta_softplus=True, initial_state=before, lengths=lens))
    # no options: steps as they come (positive ones), no gate, no skip, from zeros
    delta = (v["delta"].float().abs() * 0.1).to(dtype)
    if lengths is None:
        flat = (v["B"][..., 0, :], v["C"][..., 0, :]) if groups == 1 else (v["B"], v["C"])
        want, final = so.selective_scan(v["u"], delta, v["A"], v["B"], v["C"])
        y, got_final = fd.selective_scan(v["u"], delta, v["A"], *flat, return_final_state=True)
        near(got_final, final, torch.float32, tol)
        near(y, want, dtype, tol * s ** 0.5)


@pytest.mark.parametrize("steps", [False, True], ids=["prompt", "steps"])
def test_decays_have_no_drift(fd, steps):
    """Roundings of a slow decay cancel out over many steps: a mean error of 2e-8 a step, a cut one's, is 1e-6 after 50, which
    8192 states' mean shows (their scatter: sqrt(50) * 5e-8 / sqrt(8192) = 4e-9)."""
    l, c, s = 50, 512, 16
    g = torch.Generator().manual_seed(11)
    delta = torch.empty(1, l, c).uniform_(0.01, 0.03, generator=g).cuda()
    a = torch.empty(c, s).uniform_(-1.5, -0.5, generator=g).cuda()
    u, bc, state = torch.zeros(1, l, c, device="cuda"), torch.ones(1, l, s, device="cuda"), torch.ones(1, c, s, device="cuda")
    if steps:
        for t in range(l):
            fd.selective_scan_step(u[:, t], delta[:, t], a, bc[:, t], bc[:, t], state)
    else:
        state = fd.selective_scan(u, delta, a, bc, bc, initial_state=state, return_final_state=True)[1]
    want = torch.exp(delta.double().sum(1)[..., None] * a.double())
    drift = float((state.double() / want - 1).mean())
    assert abs(drift) < l * 1e-8, drift


def test_a_long_prompt_equals_its_parts(fd):
    """A prompt scanned whole, and in parts that hand their states on."""
    g = torch.Generator().manual_seed(1)
    v = scan_inputs(g, 2, 3001, 96, 16, 1, torch.float32)
    y, final = fd.selective_scan(**v, delta_softplus=True, return_final_state=True)
    state, parts = None, []
    seq = ("u", "delta", "z", "B", "C")
    for a, b in ((0, 1), (1, 700), (700, 2999), (2999, 3001)):
        part = {k: (t[:, a:b] if k in seq else t) for k, t in v.items()}
        out, state = fd.selective_scan(**part, delta_softplus=True, initial_state=state, return_final_state=True)
        parts.append(out)
    torch.testing.assert_close(torch.cat(parts, 1), y, rtol=2e-4, atol=2e-3)
    torch.testing.assert_close(state, final, rtol=2e-4, atol=2e-4)
    x, w = v["u"], torch.randn(96, 4, generator=g).cuda()
    whole, end = fd.causal_conv1d(x, w, return_final_state=True)
    first, mid = fd.causal_conv1d(x[:, :1], w, return_final_state=True)
    rest, last = fd.causal_conv1d(x[:, 1:], w, initial_state=mid, return_final_state=True)
    assert torch.equal(torch.cat([first, rest], 1), whole) and torch.equal(last, end)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,c,s,groups,slots", [(1, 8, 16, 1, None), (3, 100, 16, 2, [4, 0, 2]), (4, 33, 8, 1, [1, -1, 9, 0]),
                                                (2, 20, 5, 1, None), (3, 12, 32, 2, "all"), (2, 6, 64, 1, "all"), (2, 4, 100, 1, None),
                                                (1, 3, 256, 1, None), (70, 520, 16, 1, "all"), (2, 5, 1, 5, None), (9, 34, 4, 1, "all")])
def test_selective_scan_step(fd, n, c, s, groups, slots, dtype):
    g = torch.Generator().manual_seed(c)
    cache = n + 3
    v = scan_inputs(g, n, None, c, s, groups, dtype, "ragged slice")
    state = torch.randn(cache, c, s, generator=g).cuda()
    at = list(range(n)) if slots is None else torch.randperm(cache, generator=g)[:n].tolist() if slots == "all" else slots
    where = None if slots is None else torch.tensor(at, dtype=torch.int32, device="cuda")
    before = state.clone()
    y = fd.selective_scan_step(**v, state=state, delta_softplus=True, slots=where)
    live = [i for i in range(n) if 0 <= at[i] < cache]
    row = {k: v[k][live][:, None] for k in ("u", "delta", "B", "C", "z")}
    want, final = so.selective_scan(row["u"], row["delta"], v["A"], row["B"], row["C"], v["D"], row["z"], v["delta_bias"], True,
                                    before[[at[i] for i in live]])
    near(y[live], want[:, 0], dtype, 2e-5 * s ** 0.5)
    near(state[[at[i] for i in live]], final, torch.float32, 2e-5)
    untouched = [i for i in range(cache) if i not in [at[j] for j in live]]
    assert torch.equal(state[untouched], before[untouched])
    assert not y[[i for i in range(n) if i not in live]].any()


def test_steps_continue_a_prompt(fd):
    g = torch.Generator().manual_seed(3)
    v = scan_inputs(g, 2, 40, 48, 16, 1, torch.float32)
    x, w, b = v["u"], torch.randn(48, 4, generator=g).cuda(), torch.randn(48, generator=g).cuda()
    seq = ("u", "delta", "z", "B", "C")
    y, final = fd.selective_scan(**v, delta_softplus=True, return_final_state=True)
    conv, conv_final = fd.causal_conv1d(x, w, b, "silu", return_final_state=True)
    head = {k: (t[:, :35] if k in seq else t) for k, t in v.items()}
    _, state = fd.selective_scan(**head, delta_softplus=True, return_final_state=True)
    _, conv_state = fd.causal_conv1d(x[:, :35], w, b, "silu", return_final_state=True)
    for t in range(35, 40):
        token = {k: (a[:, t] if k in seq else a) for k, a in v.items()}
        torch.testing.assert_close(fd.selective_scan_step(**token, state=state, delta_softplus=True), y[:, t], rtol=2e-4, atol=2e-4)
        torch.testing.assert_close(fd.causal_conv1d_step(x[:, t], conv_state, w, b, "silu"), conv[:, t], rtol=2e-5, atol=2e-5)
    torch.testing.assert_close(state, final, rtol=2e-4, atol=2e-4)
    assert torch.equal(conv_state, conv_final)


def test_extreme_values(fd):
    """Steps that underflow every decay, steps of nothing, gates at their ends; a NaN stays in its channel and row."""
    g = torch.Generator().manual_seed(5)
    v = scan_inputs(g, 2, 150, 40, 16, 1, torch.float32)
    v["delta_bias"] = None
    v["delta"][:, 10] = 60.0        # exp(60 * -8) is no fp32 number
    v["delta"][:, 20:40] = -200.0   # softplus: nothing
    v["z"][:, 50] = 300.0
    v["z"][:, 51] = -300.0
    v["A"][:, 15] = -1e6
    v["A"][:, 14] = 0.0
    want, final = so.selective_scan(v["u"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], None, True)
    y, got = fd.selective_scan(**v, delta_softplus=True, return_final_state=True)
    # the state without decay grows to hundreds: sums of 150 terms of it
    near(got, final, torch.float32, 1e-3)
    near(y, want, torch.float32, 2e-2)
    v["u"][1, 70, 7] = float("nan")
    y, got = fd.selective_scan(**v, delta_softplus=True, return_final_state=True)
    bad = torch.zeros(2, 150, 40, dtype=torch.bool)
    bad[1, 70:, 7] = True
    assert torch.equal(torch.isnan(y).cpu(), bad)
    assert torch.isnan(got[1, 7]).all() and int(torch.isnan(got).sum()) == 16


def test_other_streams_and_captured_steps(fd):
    g = torch.Generator().manual_seed(6)
    v = scan_inputs(g, 2, 300, 64, 16, 1, torch.bfloat16)
    want = fd.selective_scan(**v, delta_softplus=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fd.selective_scan(**v, delta_softplus=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    token = {k: (t[:, 0] if k in ("u", "delta", "z", "B", "C") else t) for k, t in v.items()}
    state, conv_state = torch.zeros(2, 64, 16, device="cuda"), torch.zeros(2, 3, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(64, 4, generator=g).to(torch.bfloat16).cuda()

    def step():
        return fd.causal_conv1d_step(token["u"], conv_state, w), fd.selective_scan_step(**token, state=state, delta_softplus=True)

    first = step()
    second = step()
    state.zero_()
    conv_state.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    state.zero_()
    conv_state.zero_()
    for ref in (first, second):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])


def test_refusals(fd):
    g = torch.Generator().manual_seed(7)
    v = scan_inputs(g, 2, 6, 12, 16, 1, torch.float32)
    x, w = v["u"], torch.randn(12, 4).cuda()
    lens = torch.tensor([6, 6], dtype=torch.int32).cuda()
    state, conv_state = torch.zeros(2, 12, 16).cuda(), torch.zeros(2, 3, 12).cuda()
    token = {k: (t[:, 0] if k in ("u", "delta", "z", "B", "C") else t) for k, t in v.items()}
    with_ = lambda d, **k: {**d, **k}  # noqa: E731
    for call, exc, text in [
        (lambda: fd.causal_conv1d(x[0], w), RuntimeError, "3 dimensions"),
        (lambda: fd.causal_conv1d(x.double(), w.double()), NotImplementedError, "does not support dtype"),
        (lambda: fd.causal_conv1d(x, w[:5]), RuntimeError, "weight must have shape"),
        (lambda: fd.causal_conv1d(x, torch.randn(12, 9).cuda()), NotImplementedError, "1 to 8 taps"),
        (lambda: fd.causal_conv1d(x, w.half()), RuntimeError, "weight must be"),
        (lambda: fd.causal_conv1d(x, w, w[:, 0].cpu()), RuntimeError, "bias must be on"),
        (lambda: fd.causal_conv1d(x, w, initial_state=x), RuntimeError, "initial_state must have shape"),
        (lambda: fd.causal_conv1d(x, w, lengths=lens.long()), RuntimeError, "lengths must be"),
        (lambda: fd.causal_conv1d(x, w, activation="tanh"), RuntimeError, "activation must be one of"),
        (lambda: fd.causal_conv1d(x.clone().requires_grad_(), w), NotImplementedError, "computes no gradients"),
        (lambda: fd.causal_conv1d_step(x[:, 0], conv_state[:1], w), RuntimeError, "1 states for 2 rows"),
        (lambda: fd.causal_conv1d_step(x[:, 0], conv_state.transpose(1, 2).contiguous().transpose(1, 2), w), RuntimeError, "contiguous"),
        (lambda: fd.causal_conv1d_step(x[:, 0], conv_state.half(), w), RuntimeError, "conv_state must be"),
        (lambda: fd.causal_conv1d_step(x[:, 0], conv_state, w, slots=lens[:1]), RuntimeError, "slots must have shape"),
        (lambda: fd.selective_scan(**with_(v, A=v["A"][:6])), RuntimeError, "A must have shape"),
        (lambda: fd.selective_scan(**with_(v, A=v["A"].half())), RuntimeError, "A must be"),
        (lambda: fd.selective_scan(**with_(v, A=torch.zeros(12, 257).cuda())), NotImplementedError, "1 to 256 states"),
        (lambda: fd.selective_scan(**with_(v, B=v["B"].expand(2, 6, 5, 16))), RuntimeError, "groups dividing"),
        (lambda: fd.selective_scan(**with_(v, C=v["C"].half())), RuntimeError, "C must be"),
        (lambda: fd.selective_scan(**with_(v, delta=v["delta"][:, :5])), RuntimeError, "delta must have shape"),
        (lambda: fd.selective_scan(**with_(v, D=v["D"].half())), RuntimeError, "D must be"),
        (lambda: fd.selective_scan(**v, initial_state=state.half()), RuntimeError, "initial_state must be"),
        (lambda: fd.selective_scan(**v, lengths=lens[:1]), RuntimeError, "lengths must have shape"),
        (lambda: fd.selective_scan(**with_(v, u=v["u"].clone().requires_grad_())), NotImplementedError, "computes no gradients"),
        (lambda: fd.selective_scan_step(**token, state=state[:1]), RuntimeError, "1 states for 2 rows"),
        (lambda: fd.selective_scan_step(**token, state=state.bfloat16()), RuntimeError, "state must be"),
        (lambda: fd.selective_scan_step(**token, state=state[:, :, :8]), RuntimeError, "state must have shape"),
    ]:
        with pytest.raises(exc, match=text):
            call()
