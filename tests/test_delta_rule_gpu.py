"""gated_delta_rule and gated_delta_rule_step against their definition in 64 bits.

Tolerances.  Outputs are rounded once to their type (unit roundoff 2^-8 bf16, 2^-11 f16, 2^-24 f32).  A state is made of fp32 sums
of up to 64 + 256 terms whose factors are kept to 2^-21 or better: 320 * 2^-24 + 3 * 2^-21 < 2^-15 of the sum of their sizes,
which the oracle gives.  bf16 outputs take each of state, weight and written value to 11 bits: 3 * 2^-12 of that sum."""
import pytest
import torch

from oracle import delta_oracle as do
from test_sequence_gpu import DTYPES, IDS, LAYOUTS, ROUND, rand

pytestmark = pytest.mark.gpu

STATE_TOL = 2.0 ** -15


@pytest.fixture(scope="module")
def fd(native_lib):
    import flagdnn_b200

    assert torch.cuda.is_available()
    return flagdnn_b200


def near(got, want, size, dtype):
    got = got.double().cpu()
    assert got.shape == want.shape
    tol = STATE_TOL + (3 * 2.0 ** -12 if dtype == torch.bfloat16 else 0.0)
    least = {torch.float16: 2.0 ** -25}.get(dtype, 1e-38)       # half a step of the type's smallest numbers
    off = (got - want).abs()
    bad = ~(off <= 1.02 * ROUND[dtype] * want.abs() + tol * size + least)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off / (size + 1e-300)).max())} of the terms"


def inputs(g, n, l, key_heads, heads, dk, dv, dtype, raw, norm, layout="dense"):
    """Tensors and options of a call; l None: single tokens."""
    rows = (n,) if l is None else (n, l)
    lay = LAYOUTS[layout] if l != 0 else {}
    length = 1.0 if norm else dk ** -0.5
    common = torch.randn(key_heads, dk, generator=g).cuda() * 0.5 * length
    v = {}
    for name in ("q", "k"):
        v[name] = rand(g, (*rows, key_heads, dk), dtype, length, **lay)
        v[name].add_(common.to(dtype))
    v["v"] = rand(g, (*rows, heads, dv), dtype, **lay)
    gates = dtype if raw else torch.float32
    if raw:
        v["delta"], v["beta"] = rand(g, (*rows, heads), gates, 0.5, **lay), rand(g, (*rows, heads), gates, **lay)
        v["A"] = -(torch.rand(heads, generator=g) * 15 + 1).cuda()
        v["delta_bias"] = (torch.rand(heads, generator=g) * 4 - 6).cuda()
        return v, {"delta_softplus": True, "beta_sigmoid": True, "qk_norm": norm}
    v["delta"] = rand(g, (*rows, heads), gates, **lay).mul_(2).sub_(3).exp_().neg_()
    v["beta"] = rand(g, (*rows, heads), gates, **lay).sigmoid_()
    return v, {"qk_norm": norm}


RULES = [   # n, l, key heads, heads, dk, dv, layout, lengths
    (1, 1, 1, 1, 16, 16, "dense", None),
    (2, 37, 2, 2, 64, 64, "dense", None),
    (1, 64, 1, 2, 128, 128, "dense", None),
    (1, 65, 2, 2, 128, 128, "dense", None),
    (3, 130, 2, 4, 64, 32, "dense", [130, 0, 1]),
    (2, 100, 3, 3, 72, 100, "dense", [64, 100]),
    (4, 65, 1, 3, 33, 17, "odd", [2, 64, 65, 1]),
    (2, 150, 2, 2, 128, 64, "slice", [150, 3]),
    (2, 90, 1, 2, 40, 24, "ragged slice", None),
    (2, 41, 2, 2, 24, 40, "strided", [41, 5]),
    (1, 300, 1, 1, 128, 256, "dense", None),
    (1, 70, 2, 2, 200, 48, "dense", None),          # keys wider than the chunks' kernels take
    (2, 9, 1, 1, 256, 5, "dense", [9, 4]),
    (1, 400, 2, 6, 96, 80, "dense", [333]),
    (2, 0, 1, 2, 64, 64, "dense", None),
    (5, 129, 1, 1, 8, 8, "dense", [129, 128, 127, 64, 63]),
    (1, 20, 1, 1, 1, 1, "dense", None),
    (2, 66, 4, 4, 128, 128, "strided", [66, 65]),
    (1, 195, 1, 1, 64, 300, "dense", None),
]
IDS_R = [f"{n}x{l}h{g}-{h}k{dk}v{dv}{lay}" for n, l, g, h, dk, dv, lay, _ in RULES]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("case", RULES, ids=IDS_R)
@pytest.mark.parametrize("raw,norm", [(True, True), (False, False)], ids=["raw", "ready"])
def test_prompts(fd, case, dtype, raw, norm):
    n, l, key_heads, heads, dk, dv, layout, lengths = case
    g = torch.Generator().manual_seed(l + dk)
    v, options = inputs(g, n, l, key_heads, heads, dk, dv, dtype, raw, norm, layout)
    before = torch.randn(n, heads, dv, dk, generator=g).cuda()
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if lengths is not None:
        for i, end in enumerate(lengths):
            for name in ("q", "k", "v", "delta", "beta"):
                v[name][i, end:] = float("nan")            # padding is never read
    for initial in (before, None):
        want = do.gated_delta_rule(**v, **options, initial_state=initial, lengths=lengths)
        y, state = fd.gated_delta_rule(**v, **options, initial_state=initial, lengths=lens, return_final_state=True)
        near(state, want.state, want.state_size, torch.float32)
        near(y, want.y, want.y_size, dtype)
        assert torch.equal(y, fd.gated_delta_rule(**v, **options, initial_state=initial, lengths=lens))
        if lengths is not None:
            for i, end in enumerate(lengths):
                assert not y[i, end:].any()


LONG = [   # few rows of many chunks: in segments
    (2, 1500, 1, 2, 64, 48, "dense", [1500, 700]),
    (1, 2300, 1, 1, 128, 100, "dense", None),
    (3, 1300, 1, 1, 40, 20, "odd", [0, 1300, 65]),
    (1, 1100, 1, 3, 72, 24, "slice", [1031]),
    (2, 780, 2, 2, 128, 128, "dense", None),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("case", LONG, ids=[f"{n}x{l}h{g}-{h}k{dk}v{dv}{lay}" for n, l, g, h, dk, dv, lay, _ in LONG])
def test_long_prompts(fd, case, dtype):
    test_prompts(fd, case, dtype, True, True)


def test_long_prompts_of_few_and_of_many_rows(fd):
    """A row by itself, cut into segments, and among others, whole: the same but for roundings; where it forgets nothing, too."""
    g = torch.Generator().manual_seed(13)
    v, options = inputs(g, 40, 1000, 1, 2, 128, 128, torch.bfloat16, False, True)
    v["delta"][3] *= 1e-4
    before = torch.randn(40, 2, 128, 128, generator=g).cuda()
    y, state = fd.gated_delta_rule(**v, **options, initial_state=before, return_final_state=True)
    for i in (0, 3):
        alone = {name: t[i:i + 1] for name, t in v.items()}
        y1, state1 = fd.gated_delta_rule(**alone, **options, initial_state=before[i:i + 1], return_final_state=True)
        torch.testing.assert_close(state1, state[i:i + 1], rtol=1e-4, atol=2e-5 * float(state[i].abs().max()))
        torch.testing.assert_close(y1.float(), y[i:i + 1].float(), rtol=2.0 ** -7, atol=2.0 ** -10 * float(y[i].abs().max()))


STEPS = [   # n, key heads, heads, dk, dv, slots
    (1, 1, 1, 16, 16, None), (3, 2, 4, 64, 32, [4, 0, 2]), (4, 1, 3, 33, 17, [1, -1, 9, 0]), (2, 2, 2, 128, 128, None), (70, 1, 2, 72, 100, "all"),
    (5, 4, 4, 200, 48, "all"), (2, 1, 1, 256, 3, None), (3, 1, 2, 128, 1024, "all"), (2, 1, 1, 1, 1, None), (9, 2, 2, 32, 64, "all")]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("case", STEPS, ids=[f"{c[0]}h{c[1]}-{c[2]}k{c[3]}v{c[4]}" for c in STEPS])
@pytest.mark.parametrize("raw,norm", [(True, True), (False, False)], ids=["raw", "ready"])
def test_steps(fd, case, dtype, raw, norm):
    n, key_heads, heads, dk, dv, slots = case
    g = torch.Generator().manual_seed(dk + n)
    cache = n + 3
    for layout in ("dense", "ragged slice"):
        v, options = inputs(g, n, None, key_heads, heads, dk, dv, dtype, raw, norm, layout)
        state = torch.randn(cache, heads, dv, dk, generator=g).cuda()
        at = list(range(n)) if slots is None else torch.randperm(cache, generator=g)[:n].tolist() if slots == "all" else slots
        where = None if slots is None else torch.tensor(at, dtype=torch.int32, device="cuda")
        before = state.clone()
        y = fd.gated_delta_rule_step(**v, **options, state=state, slots=where)
        live = [i for i in range(n) if 0 <= at[i] < cache]
        places = [at[i] for i in live]
        token = {name: t if name in ("A", "delta_bias") else t[live][:, None] for name, t in v.items()}
        want = do.gated_delta_rule(**token, **options, initial_state=before[places])
        near(y[live], want.y[:, 0], want.y_size[:, 0], dtype)
        near(state[places], want.state, want.state_size, torch.float32)
        others = [i for i in range(cache) if i not in places]
        assert torch.equal(state[others], before[others])
        assert not y[[i for i in range(n) if i not in live]].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_a_prompt_equals_its_parts_and_its_tokens(fd, dtype):
    g = torch.Generator().manual_seed(3)
    v, options = inputs(g, 2, 150, 2, 4, 128, 64, dtype, True, True)
    whole = do.gated_delta_rule(**v, **options)
    rows = lambda a, b: {name: t if name in ("A", "delta_bias") else t[:, a:b] for name, t in v.items()}  # noqa: E731
    state, parts = None, []
    for a, b in ((0, 70), (70, 71), (71, 140)):
        y, state = fd.gated_delta_rule(**rows(a, b), **options, initial_state=state, return_final_state=True)
        parts.append(y)
    for t in range(140, 150):
        token = {name: x if name in ("A", "delta_bias") else x[:, 0] for name, x in rows(t, t + 1).items()}
        parts.append(fd.gated_delta_rule_step(**token, **options, state=state)[:, None])
    near(torch.cat(parts, 1), whole.y, whole.y_size, dtype)
    near(state, whole.state, whole.state_size, torch.float32)


def test_gates_at_their_ends(fd):
    """A decay of zero forgets all, beta = 0 writes nothing, a key of zeros answers nothing; also in a chunk's first and last token."""
    g = torch.Generator().manual_seed(4)
    v, options = inputs(g, 1, 140, 1, 2, 64, 48, torch.float32, False, False)
    before = torch.randn(1, 2, 48, 64, generator=g).cuda()
    v["delta"][:, (0, 20, 21, 63, 64, 100)] = -float("inf")
    v["delta"][:, 30:40] = 0.0
    v["delta"][:, 50] = -1e6
    v["beta"][:, 70:90] = 0.0
    v["beta"][:, 95] = 1.0
    v["k"][:, (5, 64, 127)] = 0.0
    v["q"][:, 11] = 0.0
    for norm in (False, True):
        options["qk_norm"] = norm
        want = do.gated_delta_rule(**v, **options, initial_state=before)
        y, state = fd.gated_delta_rule(**v, **options, initial_state=before, return_final_state=True)
        near(y, want.y, want.y_size, torch.float32)
        near(state, want.state, want.state_size, torch.float32)
        state = before.clone()
        for t in range(30):
            got = fd.gated_delta_rule_step(*(v[name][:, t] for name in ("q", "k", "v", "delta", "beta")), state, qk_norm=norm)
            near(got, want.y[:, t], want.y_size[:, t], torch.float32)


@pytest.mark.parametrize("k_size,v_size", [(1e-3, 1e-4), (1.0, 3e4), (1e2, 1.0), (1e-12, 1e20), (1.0, 1e-25)])
def test_values_of_any_size(fd, k_size, v_size):
    """Rows of one call whose sizes lie far apart: every value channel and every key has a scale of its own."""
    g = torch.Generator().manual_seed(5)
    v, options = inputs(g, 2, 100, 1, 1, 64, 32, torch.float32, False, False)
    v["beta"] *= min(1.0, k_size ** -2)                   # (a step of more than 2 / |k|^2 diverges)
    v["k"] *= k_size
    v["k"][1] *= 2.0 ** torch.randint(-8, 1, (100, 1, 1), generator=g).cuda()
    v["v"] *= v_size * 2.0 ** torch.randint(-20, 1, (32,), generator=g).cuda()
    want = do.gated_delta_rule(**v, **options)
    y, state = fd.gated_delta_rule(**v, **options, return_final_state=True)
    near(y, want.y, want.y_size, torch.float32)
    near(state, want.state, want.state_size, torch.float32)


def test_keys_that_repeat(fd):
    """The same key at every token: the solve within a chunk has its largest entries; what is written last is what is answered."""
    g = torch.Generator().manual_seed(6)
    v, options = inputs(g, 1, 192, 1, 2, 64, 32, torch.float32, False, True)
    v["k"][:] = v["k"][:, :1].clone()
    v["delta"].zero_()
    v["beta"].fill_(1.0)
    want = do.gated_delta_rule(**v, **options)
    y, state = fd.gated_delta_rule(**v, **options, return_final_state=True)
    near(y, want.y, want.y_size, torch.float32)
    near(state, want.state, want.state_size, torch.float32)


def test_heads_share_keys(fd):
    """Heads of one key head, against the same keys given to each."""
    g = torch.Generator().manual_seed(7)
    v, options = inputs(g, 2, 100, 2, 6, 64, 64, torch.bfloat16, True, True)
    y = fd.gated_delta_rule(**v, **options)
    wide = dict(v, q=v["q"].repeat_interleave(3, 2), k=v["k"].repeat_interleave(3, 2))
    assert torch.equal(y, fd.gated_delta_rule(**wide, **options))


def test_a_longer_scale(fd):
    g = torch.Generator().manual_seed(8)
    v, options = inputs(g, 1, 70, 1, 1, 32, 32, torch.float32, True, True)
    want = do.gated_delta_rule(**v, **options, scale=2.5)
    near(fd.gated_delta_rule(**v, **options, scale=2.5), want.y, want.y_size, torch.float32)


def test_captured_prompts_and_steps(fd):
    g = torch.Generator().manual_seed(9)
    v, options = inputs(g, 2, 130, 1, 2, 128, 128, torch.bfloat16, True, True)
    token, _ = inputs(g, 2, None, 1, 2, 128, 128, torch.bfloat16, True, True)
    cache = torch.zeros(2, 2, 128, 128, device="cuda")

    def both():
        y, state = fd.gated_delta_rule(**v, **options, return_final_state=True)
        cache.copy_(state)
        return y, fd.gated_delta_rule_step(**token, **options, state=cache)

    want = [t.clone() for t in (*both(), cache)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for _ in range(2):
        cache.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*out, cache), want))


def test_two_streams_at_once(fd):
    g = torch.Generator().manual_seed(10)
    calls = [inputs(g, 1, 500, 2, 2, 128, 128, torch.bfloat16, True, True) for _ in range(2)]
    want = [fd.gated_delta_rule(**v, **o) for v, o in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, (v, o) in enumerate(calls):
            with torch.cuda.stream(streams[i]):
                got[i] = fd.gated_delta_rule(**v, **o)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_python_route_gives_the_same(fd, monkeypatch):
    from flagdnn_b200 import conv_host

    g = torch.Generator().manual_seed(11)
    v, options = inputs(g, 2, 80, 1, 2, 64, 64, torch.float16, True, True)
    token, _ = inputs(g, 2, None, 1, 2, 64, 64, torch.float16, True, True)
    states = [torch.ones(2, 2, 64, 64, device="cuda") for _ in range(2)]
    first = fd.gated_delta_rule(**v, **options, return_final_state=True), fd.gated_delta_rule_step(**token, **options, state=states[0])
    monkeypatch.setattr(conv_host, "_fast", False)
    version = states[1]._version
    second = fd.gated_delta_rule(**v, **options, return_final_state=True), fd.gated_delta_rule_step(**token, **options, state=states[1])
    assert torch.equal(first[0][0], second[0][0]) and torch.equal(first[0][1], second[0][1]) and torch.equal(first[1], second[1])
    assert torch.equal(*states) and states[1]._version > version and states[0]._version > 0


def test_a_wait_that_runs_out_is_reported_and_the_device_stays_usable(fd, native_lib):
    """No copy is issued: the first wait for a chunk's operands runs out after some 0.1 ms of clocks, the launches return, and the next
    call is as before. A whole row and one in segments."""
    import ctypes

    from flagdnn_b200 import _native as nat

    g = torch.Generator().manual_seed(14)
    for rows, length in ((40, 130), (1, 1200)):
        v, options = inputs(g, rows, length, 1, 2, 64, 64, torch.bfloat16, True, True)
        good = fd.gated_delta_rule(**v, **options)
        torch.cuda.synchronize()
        assert fd.device_status() == 0
        nat.check(native_lib.fdnn_debug_set_wait_limit(200_000, 1))
        try:
            fd.gated_delta_rule(**v, **options)
            torch.cuda.synchronize()
        finally:
            nat.check(native_lib.fdnn_debug_set_wait_limit(0, 0))
        word = ctypes.c_uint32(0)
        assert native_lib.fdnn_device_status(ctypes.byref(word)) == nat.FDNN_DEVICE_TIMEOUT and word.value == 9
        assert native_lib.fdnn_device_status(ctypes.byref(word)) == nat.FDNN_OK
        assert torch.equal(fd.gated_delta_rule(**v, **options), good) and fd.device_status() == 0


def test_refusals(fd):
    g = torch.Generator().manual_seed(12)
    v, options = inputs(g, 2, 10, 1, 2, 16, 16, torch.float16, True, True)
    token, _ = inputs(g, 2, None, 1, 2, 16, 16, torch.float16, True, True)
    state = torch.zeros(2, 2, 16, 16, device="cuda")

    def refused(error, match, call=fd.gated_delta_rule, base=v, **change):
        with pytest.raises(error, match=match):
            call(**{**base, **options, **change})

    refused(RuntimeError, "q must have shape", q=v["q"][:, :9])
    refused(RuntimeError, "k must have shape", k=v["k"][..., :8])
    refused(RuntimeError, "share", q=v["q"].expand(2, 10, 3, 16), k=v["k"].expand(2, 10, 3, 16))
    refused(RuntimeError, "must be torch.float16", k=v["k"].float())
    refused(RuntimeError, "delta must be", delta=v["delta"].bfloat16(), beta=v["beta"].bfloat16())
    refused(RuntimeError, "beta must be", beta=v["beta"].float())
    refused(RuntimeError, "A must have shape", A=v["A"][:1])
    refused(RuntimeError, "delta_bias must be", delta_bias=v["delta_bias"].half())
    refused(RuntimeError, "initial_state must have shape", initial_state=state[:1])
    refused(RuntimeError, "lengths must be", lengths=torch.tensor([1, 2], device="cuda"))
    refused(RuntimeError, "4 dimensions", v=v["v"][0])
    refused(NotImplementedError, "keys of 1 to 256", q=torch.zeros(2, 10, 1, 257, device="cuda").half(), k=torch.zeros(2, 10, 1, 257, device="cuda").half())
    refused(NotImplementedError, "values of 1 to 1024", v=torch.zeros(2, 10, 2, 1025, device="cuda").half())
    refused(NotImplementedError, "does not support", v=v["v"].double())
    for name in ("q", "k", "v", "delta", "beta", "A", "delta_bias"):
        refused(NotImplementedError, "no gradients", **{name: v[name].clone().requires_grad_()})
    refused(NotImplementedError, "no gradients", initial_state=state.clone().requires_grad_())
    step = dict(call=fd.gated_delta_rule_step, base={**token, "state": state})
    refused(RuntimeError, "contiguous", **step, state=state.transpose(2, 3))
    refused(RuntimeError, "1 states for 2 rows", **step, state=state[:1])
    refused(RuntimeError, "state must be", **step, state=state.half())
    refused(RuntimeError, "slots must be", **step, slots=torch.tensor([0, 1], device="cuda"))
    refused(NotImplementedError, "no gradients", **step, state=state.clone().requires_grad_())
    with torch.no_grad():
        fd.gated_delta_rule_step(**{**token, "v": token["v"].clone().requires_grad_()}, **options, state=state)
