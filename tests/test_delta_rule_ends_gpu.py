"""gated_delta_rule where its inputs reach their ends: tokens that forget all, infinities, lengths; and rows that
are cut into segments, as their workspace tells.

Tolerances as in test_delta_rule_gpu.py."""
import ctypes

import pytest
import torch

from flagdnn_b200 import _native as nat
from oracle import delta_oracle as do
from test_delta_rule_gpu import fd, inputs, near  # noqa: F401
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
