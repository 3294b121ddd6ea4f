"""gated_delta_rule where its inputs reach their ends: tokens that forget all, infinities, lengths, decays above one, long
sums of decays; and rows that are cut into segments, as their workspace tells.

Tolerances as in test_delta_rule_gpu.py."""
import ctypes
import math

import pytest
import torch

from flagdnn_b200 import _native as nat
from oracle import delta_oracle as do
from test_delta_rule_gpu import STATE_TOL, fd, inputs, near  # noqa: F401
from test_sequence_gpu import DTYPES, IDS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("resets", [1, 2, 8, 16, 32, 41])
@pytest.mark.parametrize("forget", [-float("inf"), -1e30, -3e4, -250.0])
def test_several_tokens_of_a_chunk_forget_all(fd, dtype, resets, forget):  # noqa: F811
    """Packed documents begin within a chunk, the last of them in its middle: what the tokens behind it write is kept as they say."""
    g = torch.Generator().manual_seed(resets)
    v, options = inputs(g, 1, 150, 1, 2, 64, 48, dtype, False, True)
    at = [40 - i * 40 // max(1, resets - 1) for i in range(resets)]
    assert len(set(at)) == resets and max(at) == 40
    for chunk in (0, 64):
        v["delta"][:, [chunk + i for i in at]] = forget
    before = torch.randn(1, 2, 48, 64, generator=g).cuda()
    for length in (64, 150):
        part = {name: t[:, :length] for name, t in v.items()}
        want = do.gated_delta_rule(**part, **options, initial_state=before)
        y, state = fd.gated_delta_rule(**part, **options, initial_state=before, return_final_state=True)
        near(state, want.state, want.state_size, torch.float32)
        near(y, want.y, want.y_size, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("name", ["v", "k", "q", "beta", "delta"])
@pytest.mark.parametrize("length,at", [(130, 40), (64, 63), (130, 64), (2304, 1400)])
def test_an_infinite_input_is_seen(fd, dtype, name, length, at):  # noqa: F811
    """Tokens before it in its chunk are right or not finite, never finite and wrong; those before the chunk are right."""
    g = torch.Generator().manual_seed(at)
    v, options = inputs(g, 1, length, 1, 2, 64, 40, dtype, False, False)
    v[name][0, at, 0, ...] = float("inf") if v[name].dim() == 3 else v[name][0, at, 0]
    if v[name].dim() == 4:
        v[name][0, at, 0, 7] = float("inf")
    y, state = fd.gated_delta_rule(**v, **options, return_final_state=True)
    y, state = y.double().cpu(), state.double().cpu()
    want = do.gated_delta_rule(**{n: t[:, :at] for n, t in v.items()}, **options)
    chunk = at // 64 * 64
    heads = 1 if name in ("beta", "delta") or (name == "v") else 2          # the two heads share keys and queries
    channels = slice(7, 8) if name == "v" else slice(0, 40)
    assert y[0, :chunk].isfinite().all()
    near(torch.where(y[0, :at].isfinite(), y[0, :at], want.y[0]), want.y[0], want.y_size[0], dtype)
    assert not y[0, at, :heads, channels].isfinite().any()
    others = torch.ones(2, 40, dtype=torch.bool)
    others[:heads, channels] = False
    assert y[0, :, others].isfinite().all()
    if name != "q":
        assert not y[0, at:, :heads, channels].isfinite().any() and not state[0, :heads, channels].isfinite().any()
        assert state[0][others].isfinite().all()
    else:
        assert y[0, at + 1:].isfinite().all() and state.isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("length", [9, 130, 2304])
def test_an_infinite_state_is_seen(fd, dtype, length):  # noqa: F811
    g = torch.Generator().manual_seed(length)
    v, options = inputs(g, 1, length, 1, 2, 64, 40, dtype, False, False)
    before = torch.randn(1, 2, 40, 64, generator=g).cuda()
    want = do.gated_delta_rule(**v, **options, initial_state=before)
    before[0, 1, 5, 3] = float("inf")
    y, state = fd.gated_delta_rule(**v, **options, initial_state=before, return_final_state=True)
    assert not y[0, :, 1, 5].isfinite().any() and not state[0, 1, 5].isfinite().any()
    keep = [i for i in range(80) if i != 45]
    near(y.flatten(2)[..., keep], want.y.flatten(2)[..., keep], want.y_size.flatten(2)[..., keep], dtype)
    near(state.flatten(1, 2)[:, keep], want.state.flatten(1, 2)[:, keep], want.state_size.flatten(1, 2)[:, keep], torch.float32)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("length", [10, 11, 12, 13, 16, 17])
@pytest.mark.parametrize("dk", [64, 128])
def test_lengths_between_the_two_ways(fd, dtype, length, dk):  # noqa: F811
    g = torch.Generator().manual_seed(length)
    v, options = inputs(g, 3, length, 1, 2, dk, 40, dtype, True, True)
    before = torch.randn(3, 2, 40, dk, generator=g).cuda()
    lengths = [length, 0, length - 3]
    want = do.gated_delta_rule(**v, **options, initial_state=before, lengths=lengths)
    y, state = fd.gated_delta_rule(**v, **options, initial_state=before, lengths=torch.tensor(lengths, dtype=torch.int32).cuda(),
                                   return_final_state=True)
    near(y, want.y, want.y_size, dtype)
    near(state, want.state, want.state_size, torch.float32)


def segments(native_lib, v):
    """Of each row of a call, by what its workspace holds beside its chunks: ends (of values and of a unit matrix) and starts."""
    n, length, heads, dv = v["v"].shape
    key_heads, dk = v["q"].shape[2:]
    d, nbytes = nat.DeltaRuleDesc(), ctypes.c_int64()
    d.dtype = {torch.float16: nat.F16, torch.bfloat16: nat.BF16, torch.float32: nat.F32}[v["v"].dtype]
    d.gate_dtype, d.n, d.key_heads, d.heads, d.dk, d.dv = d.dtype, n, key_heads, heads, dk, dv
    sizes = []
    for d.l in (64, length):
        nat.check(native_lib.fdnn_gated_delta_rule_workspace_bytes(ctypes.byref(d), ctypes.byref(nbytes)))
        sizes.append(nbytes.value)
    more, rest = divmod(sizes[1] - (length + 63) // 64 * sizes[0], n * heads * ((dv + 15) // 16 * 16 + dk + dv) * dk * 4)
    assert rest == 0
    return more + 1


CUT = [   # n, l, key heads, heads, dk, dv, layout, lengths
    (1, 1600, 1, 2, 128, 128, "dense", None), (1, 2300, 1, 2, 128, 128, "slice", [2222]), (2, 2304, 2, 2, 128, 128, "dense", [2304, 700]),
    (1, 3000, 2, 4, 128, 128, "strided", None), (4, 2500, 1, 1, 128, 128, "odd", [0, 2500, 65, 1999]), (1, 2300, 1, 2, 127, 100, "ragged slice", None),
    (1, 2000, 2, 2, 126, 96, "dense", [1]), (2, 1500, 1, 2, 64, 48, "dense", [1500, 700]), (1, 2300, 3, 3, 8, 300, "dense", None)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("case", CUT, ids=[f"{n}x{l}h{g}-{h}k{dk}v{dv}{lay}" for n, l, g, h, dk, dv, lay, _ in CUT])
def test_rows_in_segments(fd, native_lib, case, dtype):  # noqa: F811
    n, l, key_heads, heads, dk, dv, layout, lengths = case
    g = torch.Generator().manual_seed(l + dk)
    v, options = inputs(g, n, l, key_heads, heads, dk, dv, dtype, True, True, layout)
    v["A"][-1] = -1e-3                                       # a head that forgets next to nothing
    assert segments(native_lib, v) > 1
    before = torch.randn(n, heads, dv, dk, generator=g).cuda()
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for i, end in enumerate(lengths or []):
        for name in ("q", "k", "v", "delta", "beta"):
            v[name][i, end:] = float("nan")
    for initial in (before, None):
        want = do.gated_delta_rule(**v, **options, initial_state=initial, lengths=lengths)
        y, state = fd.gated_delta_rule(**v, **options, initial_state=initial, lengths=lens, return_final_state=True)
        near(state, want.state, want.state_size, torch.float32)
        near(y, want.y, want.y_size, dtype)
        assert torch.equal(y, fd.gated_delta_rule(**v, **options, initial_state=initial, lengths=lens))
        for i, end in enumerate(lengths or []):
            assert not y[i, end:].any()


def test_a_row_in_segments_and_among_others(fd, native_lib):  # noqa: F811
    """A row by itself is cut, among forty it is whole: the same but for roundings; where it forgets nothing, too."""
    g = torch.Generator().manual_seed(13)
    v, options = inputs(g, 40, 2304, 1, 2, 128, 128, torch.bfloat16, False, True)
    v["delta"][3] *= 1e-4
    assert segments(native_lib, v) == 1
    before = torch.randn(40, 2, 128, 128, generator=g).cuda()
    y, state = fd.gated_delta_rule(**v, **options, initial_state=before, return_final_state=True)
    for i in (0, 3):
        alone = {name: t[i:i + 1] for name, t in v.items()}
        assert segments(native_lib, alone) > 1
        y1, state1 = fd.gated_delta_rule(**alone, **options, initial_state=before[i:i + 1], return_final_state=True)
        want = do.gated_delta_rule(**alone, **options, initial_state=before[i:i + 1])
        for a, b in ((y1, state1), (y[i:i + 1], state[i:i + 1])):
            near(a, want.y, want.y_size, torch.bfloat16)
            near(b, want.state, want.state_size, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("length,grow", [(64, 0.19), (64, 1.3), (130, 0.19), (130, 0.6), (2304, 0.036)])
def test_decays_above_one(fd, native_lib, dtype, length, grow):  # noqa: F811
    """Products of decays up to 2^17.3 over chunks, and to e^83 over segments, next to the largest fp32 number; key channels that no key touches and
    states of zeros in them. What grows is the state; values are small. Past 2^18 within a chunk it is NaN, by the step it is not."""
    g = torch.Generator().manual_seed(length)
    v, options = inputs(g, 1, length, 1, 2, 64, 40, dtype, False, True)
    v["delta"].fill_(grow)
    for name in ("k", "q"):
        v[name][..., 40:] = 0.0
    assert (segments(native_lib, v) > 1) == (length == 2304)
    before = torch.randn(1, 2, 40, 64, generator=g).cuda() * 1e-6
    before[:, :, ::2, 40:] = 0.0
    v["v"] *= 1e-4
    y, state = fd.gated_delta_rule(**v, **options, initial_state=before, return_final_state=True)
    if grow > 0.2:
        assert y.isnan().all() and state.isnan().all()
        length = 10                                          # token by token
        v = {name: t[:, :length] for name, t in v.items()}
        y, state = fd.gated_delta_rule(**v, **options, initial_state=before, return_final_state=True)
    want = do.gated_delta_rule(**v, **options, initial_state=before)
    near(state, want.state, want.state_size, torch.float32)
    if dtype != torch.float16:
        near(y, want.y, want.y_size, dtype)


def least_steps(v, options, before):
    """What y can be off by because a channel's values of a chunk share a scale. Their largest is taken to 2^14 .. 2^15, and the second f16 part of
    one of them is off by half of f16's least step, 2^-25: by 2^-39 of the largest. That goes for v - e^G S k and for what is written, U. An
    error of the first is one of v; an error e of U does no more to y than a v of e / beta adds to the sums of sizes."""
    x = {name: t.double().cpu() for name, t in v.items()}
    norm = lambda t: t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() if options["qk_norm"] else t  # noqa: E731
    heads, length = x["v"].shape[2], x["v"].shape[1]
    keys = norm(x["k"])[0].repeat_interleave(heads // x["k"].shape[2], 1)
    most, state = torch.zeros_like(x["v"]), before.double().cpu()
    for c in range(0, length, 64):
        part = slice(c, min(length, c + 64))
        for h in range(heads):
            k, b, total = keys[part, h], x["beta"][0, part, h], x["delta"][0, part, h].clamp_min(-1e5).cumsum(0)
            rest = x["v"][0, part, h] - total.exp()[:, None] * (k @ state[0, h].T)
            a = b[:, None] * torch.exp((total[:, None] - total).clamp_max(700)).tril(-1) * (k @ k.T)
            written = torch.linalg.solve_triangular(torch.eye(len(k), dtype=k.dtype) + a.tril(-1), b[:, None] * rest, upper=False)
            most[0, part, h] = rest.abs().amax(0) + written.abs().amax(0) / b[:, None]
        state = do.gated_delta_rule(**{n: t[:, part] for n, t in x.items()}, **options, initial_state=state).state
    return 2.0 ** -39 * do.gated_delta_rule(**dict(x, v=most), **options).y_size


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("length", [200, 2304])
def test_decays_on_both_sides_of_one(fd, dtype, length):  # noqa: F811
    """Heads whose decays wander, grow within a chunk (too far in some) and shrink again, and forget all in between."""
    g = torch.Generator().manual_seed(length + 1)
    v, options = inputs(g, 1, length, 1, 6, 64, 24, dtype, False, True)
    t = torch.arange(length)
    v["delta"][0, :, 0] = torch.randn(length, generator=g).cuda() * 0.3
    v["delta"][0, :, 1] = torch.where(t % 40 < 20, 1.0, -1.0).cuda()
    v["delta"][0, :, 2] = torch.where(t % 64 == 31, -float("inf"), 0.3).cuda()
    v["delta"][0, :, 3] = torch.where(t % 64 < 63, 0.3, -19.0).cuda()
    v["delta"][0, :, 4] = torch.where(t % 40 < 20, 0.6, -0.6).cuda()
    v["delta"][0, :, 5] = torch.where(t % 64 == 31, -float("inf"), 0.18).cuda()
    before = torch.randn(1, 6, 24, 64, generator=g).cuda()
    total = (v["delta"][0].double().clamp_min(-1e5) / math.log(2)).cumsum(0).cpu()
    growth = [max(float((c[None] - c[:, None]).triu().max()) for c in total[:, h].split(64)) for h in range(6)]
    assert [x > 18 for x in growth] == [False, True, False, True, False, False]
    want = do.gated_delta_rule(**v, **options, initial_state=before)
    y, state = fd.gated_delta_rule(**v, **options, initial_state=before, return_final_state=True)
    y_size = want.y_size + least_steps(v, options, before) / STATE_TOL
    for h in range(6):
        if growth[h] > 18:
            assert y[0, :, h].isnan().all() and state[0, h].isnan().all()
            continue
        near(state[0, h], want.state[0, h], want.state_size[0, h], torch.float32)
        fits = want.y[0, :, h].abs() < 6e4                   # (past 65504 f16 has infinity)
        near(y[0, :, h].cpu()[fits], want.y[0, :, h][fits], y_size[0, :, h][fits], dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_values_far_below_their_chunks_largest(fd, dtype):  # noqa: F811
    """A token whose values are 2^24 times its neighbours'."""
    g = torch.Generator().manual_seed(21)
    v, options = inputs(g, 1, 64, 1, 2, 64, 40, dtype, False, True)
    v["v"][:, 50] *= 2.0 ** 24
    want = do.gated_delta_rule(**v, **options)
    y = fd.gated_delta_rule(**v, **options)
    near(y, want.y, want.y_size + least_steps(v, options, torch.zeros(1, 2, 40, 64)) / STATE_TOL, dtype)


@pytest.mark.parametrize("low,high", [(-8.0, -6.0), (-6.0, -4.0), (-4.0, -2.0), (-2.0, 0.0), (0.0, 2.0), (2.0, 6.0)])
def test_raw_decays_add_up(fd, low, high):  # noqa: F811
    """A state that forgets to e^-80 of itself, with nothing written, by tokens that are alike. A log decay's relative error: its softplus is a
    polynomial (1.3e-7) of a power by the special function unit (2^-22), whose argument, log2 e times |dt|, is rounded (2^-24, and 1.3e-8 of the
    constant: (2^-24 + 1.3e-8) |dt| of the power), then a product (2^-24). The state takes 2^-22 with a chunk's power and product, 3 * 2^-24
    with a token's."""
    g = torch.Generator().manual_seed(int(low) + 9)
    n, heads = 8, 16
    for length, by_step in ((1024, False), (64, True), (9, False)):
        rows = torch.rand(n, heads, generator=g).cuda() * (high - low) + low
        soft = torch.nn.functional.softplus(rows.double(), threshold=1000)
        A = -(80.0 / (soft.mean(0) * length)).float()
        total = soft * A.double() * length
        q, v = torch.zeros(n, length, 1, 8, device="cuda"), torch.zeros(n, length, heads, 8, device="cuda")
        delta, beta = rows[:, None].expand(n, length, heads).contiguous(), torch.full((n, length, heads), -200.0, device="cuda")
        state = torch.ones(n, heads, 8, 8, device="cuda")
        options = {"A": A, "delta_softplus": True, "beta_sigmoid": True}
        if by_step:
            for t in range(length):
                fd.gated_delta_rule_step(q[:, t], q[:, t], v[:, t], delta[:, t], beta[:, t], state, **options)
        else:
            _, state = fd.gated_delta_rule(q, q, v, delta, beta, **options, initial_state=state, return_final_state=True)
        want = total.exp()                                   # (of rates above the mean past fp32's normal numbers: steps of 2^-149 a product)
        off = (state.double() - want[..., None, None]).abs().amax((2, 3))
        each = 1.3e-7 + 2.0 ** -22 + (2.0 ** -24 + 1.3e-8) * rows.double().abs() + 2.0 ** -24
        bound = each * total.abs() + (length // 64 * 2.0 ** -22 if length == 1024 else length * 3 * 2.0 ** -24)
        assert (off <= bound * want + length * 2.0 ** -150).all(), float((off / (bound * want + length * 2.0 ** -150)).max())
