"""group_norm and group_norm_backward against their definition in 64 bits, at the sizes, layouts and values where they can
go wrong.

Tolerances.  Values are rounded once to the tensor's type (unit roundoff 2^-8 bf16, 2^-11 f16, 2^-24 f32) after fp32
arithmetic; a normed value carries a few fp32 roundings of numbers of its own size and of sums over the group, taken as 2e-5
of the value plus 2e-5 (gradients: of the largest gradient).  Sums over many pixels (dweight, dbias) are taken as
2e-5 of the root of the sum of squares of what is summed, times its length's root at most."""
import pytest
import torch

from oracle import sequence_oracle as so

pytestmark = pytest.mark.gpu

ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
FP32 = 2e-5


@pytest.fixture(scope="module")
def fd(native_lib):
    import flagdnn_b200

    assert torch.cuda.is_available()
    return flagdnn_b200


def make(shape, dtype, layout, seed=0, offset=0.3):
    """x on the GPU in a layout: "cl" channels last, "nchw" contiguous, "slice" channels of a wider channels-last tensor,
    "odd" channels last at an odd address, "crop" a window of a wider image."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=g) + offset * torch.randn((1, shape[1]) + (1,) * (len(shape) - 2), generator=g)).to(dtype).cuda()
    if layout == "nchw" or (len(shape) == 2 and layout == "cl"):
        return x.contiguous()
    if len(shape) == 2 and layout == "t":
        return x.t().contiguous().t()
    order = (0, *range(2, len(shape)), 1)
    back = [order.index(i) for i in range(len(shape))]
    rows = x.permute(order).contiguous()
    if layout == "cl":
        return rows.permute(back)
    if layout == "slice":
        wide = torch.full((*rows.shape[:-1], shape[1] + 24), float("nan"), dtype=dtype, device="cuda")
        wide[..., 8:8 + shape[1]] = rows
        return wide[..., 8:8 + shape[1]].permute(back)
    if layout == "odd":
        flat = torch.empty(rows.numel() + 1, dtype=dtype, device="cuda")
        flat[1:] = rows.reshape(-1)
        return flat[1:].view(rows.shape).permute(back)
    assert layout == "crop" and len(shape) == 4
    wide = torch.full((rows.shape[0], rows.shape[1] + 2, rows.shape[2] + 3, rows.shape[3]), float("nan"), dtype=dtype, device="cuda")
    wide[:, 1:-1, 2:-1] = rows
    return wide[:, 1:-1, 2:-1].permute(back)


def params(c, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.2 * torch.randn(c, generator=g)).to(dtype).cuda(), (0.2 * torch.randn(c, generator=g)).to(dtype).cuda()


def near(got, want, dtype, atol=FP32, rtol=FP32):
    got = got.double().cpu()
    assert got.shape == want.shape
    bad = (got - want).abs() > (1.02 * ROUND[dtype] + rtol) * want.abs() + atol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((got - want).abs().max())}"


SHAPES = [   # shape, groups, layout
    ((1, 64, 14, 14), 16, "cl"),          # one image
    ((3, 32, 5, 7), 32, "cl"),            # a channel a group
    ((2, 90, 45, 37), 6, "cl"),           # channels that fill no vector
    ((2, 60, 9, 11), 4, "cl"),            # fifteen channels a group
    ((2, 40, 13, 3), 10, "cl"),           # four channels a group
    ((2, 7, 3, 5), 1, "cl"),              # an odd channel count
    ((2, 33, 4, 4), 3, "cl"),
    ((4, 128, 56, 56), 32, "cl"),         # larger than one block holds
    ((1, 64, 112, 112), 2, "cl"),         # a group of 401 408 values
    ((1, 16, 260, 260), 1, "cl"),         # larger than a cluster holds
    ((2, 8, 512, 300), 8, "cl"),
    ((1, 511, 13, 13), 1, "cl"),          # a group wider than a block of the two-launch form
    ((2, 300, 9, 10), 1, "odd"),
    ((2, 1026, 3, 3), 2, "cl"),
    ((3, 700, 1, 1), 1, "odd"),
    ((1, 2040, 6, 6), 8, "cl"),           # 255 channels a group: eight groups to a slab
    ((2, 2040, 1, 33), 8, "cl"),
    ((1, 1032, 12, 12), 8, "cl"),
    ((2, 1032, 13, 13), 8, "cl"),
    ((3, 4096, 1, 1), 1, "cl"),           # slabs as wide as they get
    ((2, 4096, 3, 5), 8, "cl"),
    ((2, 3968, 6, 6), 1, "cl"),
    ((40, 64, 28, 28), 8, "cl"),          # several images to a cluster
    ((700, 32, 4, 4), 4, "cl"),
    ((5, 96, 1, 1), 8, "cl"),             # one pixel
    ((2, 256, 1, 3), 32, "cl"),
    ((2, 48, 17), 6, "cl"),               # [N, C, L]
    ((3, 24, 1), 3, "nchw"),
    ((2, 64, 30, 31), 8, "slice"),
    ((2, 64, 30, 31), 8, "odd"),
    ((2, 64, 30, 31), 8, "crop"),
    ((2, 64, 30, 31), 8, "nchw"),
    ((2, 30, 12, 12), 5, "nchw"),
    ((70, 512), 8, "cl"),                 # rows of tokens
    ((1, 4096), 64, "cl"),
    ((1000, 200), 8, "cl"),               # 25 channels a group
    ((33, 1024), 1, "cl"),                # layer norm
    ((9, 12000), 1, "cl"),                # a group larger than a warp holds
    ((7, 6000), 5, "cl"),
    ((65, 100), 100, "cl"),
    ((1000, 128), 4, "cl"),               # several tokens to a block
    ((6455, 8), 1, "cl"),
    ((77, 12), 3, "cl"),
    ((3, 24), 2, "cl"),
    ((301, 1916), 4, "cl"),               # four groups of 479 channels: two tokens to a block
    ((123, 1024), 2, "cl"),
    ((21, 64 * 477), 64, "cl"),           # as long, and more of them than a block has warps
    ((61, 1024), 1, "cl"),
    ((5, 429), 1, "cl"),                  # an odd number of channels, more than a lane's of a warp
    ((40, 906), 3, "cl"),
    ((9, 1020), 1, "cl"),
    ((12, 36), 3, "t"),
    ((300, 640), 20, "slice"),
]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", SHAPES, ids=[f"{'x'.join(map(str, s))}g{g}{k}" for s, g, k in SHAPES])
def test_values_and_statistics(fd, case, dtype):
    shape, groups, layout = case
    x = make(shape, dtype, layout)
    w, b = params(shape[1], dtype)
    want, mean, rstd = so.group_norm(x, groups, w, b, 1e-5, "silu")
    y, got_mean, got_rstd = fd.group_norm(x, groups, w, b, 1e-5, activation="silu", return_stats=True)
    assert y.dtype == dtype and got_mean.dtype == got_rstd.dtype == torch.float32
    near(got_mean, mean, torch.float32)
    near(got_rstd, rstd, torch.float32, rtol=5e-5)
    near(y, want, dtype)
    assert torch.equal(y, fd.group_norm(x, groups, w, b, 1e-5, activation="silu"))
    if layout == "cl" and len(shape) == 4 and shape[1] > 1:
        assert y.is_contiguous(memory_format=torch.channels_last)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", SHAPES, ids=[f"{'x'.join(map(str, s))}g{g}{k}" for s, g, k in SHAPES])
def test_gradients(fd, case, dtype):
    shape, groups, layout = case
    x, dy = make(shape, dtype, layout), make(shape, dtype, "slice" if layout == "cl" else layout, seed=7)
    w, b = params(shape[1], dtype)
    _, mean, rstd = fd.group_norm(x, groups, w, b, return_stats=True)
    dx, dw, db = fd.group_norm_backward(dy, x, mean, rstd, groups, w, b, activation="silu")
    want = so.group_norm_grad(dy, x, groups, w, b, 1e-5, "silu")
    # rstd of a group of one value or of a few is large: its gradients are differences of large terms
    scale = float(so.group_norm(x, groups)[2].max().clamp_min(1.0))
    near(dx, want[0], dtype, atol=FP32 * scale * 5, rtol=FP32)
    terms = (x.numel() // shape[1]) ** 0.5
    near(dw, want[1], dtype, atol=FP32 * terms * 4)
    near(db, want[2], dtype, atol=FP32 * terms * 4)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), fd.group_norm_backward(dy, x, mean, rstd, groups, w, b, activation="silu")))


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("shape,groups", [((3, 48, 10, 9), 6), ((40, 256), 4)])
def test_activations_and_optional_parameters(fd, act, shape, groups):
    x, dy = make(shape, torch.float32, "cl"), make(shape, torch.float32, "cl", seed=3)
    w, b = params(shape[1], torch.float32)
    for weight, bias in ((w, b), (w, None), (None, b), (None, None)):
        y, mean, rstd = fd.group_norm(x, groups, weight, bias, 1e-3, act, return_stats=True)
        near(y, so.group_norm(x, groups, weight, bias, 1e-3, act)[0], torch.float32)
        got = fd.group_norm_backward(dy, x, mean, rstd, groups, weight, bias, act)
        want = so.group_norm_grad(dy, x, groups, weight, bias, 1e-3, act)
        near(got[0], want[0], torch.float32, atol=1e-4)
        for p, g, v in ((weight, got[1], want[1]), (bias, got[2], want[2])):
            if p is None:
                assert g is None
            else:
                near(g, v, torch.float32, atol=FP32 * 4 * (x.numel() // shape[1]) ** 0.5)


@pytest.mark.parametrize("shape,groups", [((3, 48, 10, 9), 6), ((2, 48, 10, 9), 48), ((40, 256), 4)])
def test_float32_parameters_with_16_bit_activations(fd, shape, groups):
    x, dy = make(shape, torch.bfloat16, "cl"), make(shape, torch.bfloat16, "cl", seed=3)
    w, b = params(shape[1], torch.float32)
    y, mean, rstd = fd.group_norm(x, groups, w, b, activation="gelu", return_stats=True)
    near(y, so.group_norm(x, groups, w, b, act="gelu")[0], torch.bfloat16)
    dx, dw, db = fd.group_norm_backward(dy, x, mean, rstd, groups, w, b, "gelu")
    want = so.group_norm_grad(dy, x, groups, w, b, act="gelu")
    assert dw.dtype == db.dtype == torch.float32
    near(dx, want[0], torch.bfloat16, atol=2e-4)
    terms = (x.numel() // shape[1]) ** 0.5
    near(dw, want[1], torch.float32, atol=FP32 * 4 * terms)
    near(db, want[2], torch.float32, atol=FP32 * 4 * terms)


@pytest.mark.parametrize("border", [False, True])
@pytest.mark.parametrize("shape,groups,layout", [((2, 64, 40, 40), 8, "cl"), ((2, 64, 40, 40), 8, "nchw"), ((50, 512), 4, "cl"),
                                                 ((1, 8, 400, 400), 1, "cl")])
def test_a_mean_far_from_zero_costs_no_precision(fd, shape, groups, layout, border):
    # the mean is held to a few fp32 roundings of 1000 (6e-5 apart): 1.5e-4 of a spread of one
    x = make(shape, torch.float32, layout) + 1000.0
    if border and len(shape) == 4:
        x[:, :, :1] = 0.0     # the first values are not like the others
    ref, mean, rstd = so.group_norm(x, groups)
    y, got_mean, got_rstd = fd.group_norm(x, groups, return_stats=True)
    near(y, ref, torch.float32, atol=1.5e-4)
    near(got_rstd, rstd, torch.float32, rtol=2e-4)


def test_constant_groups_and_nan_stay_in_their_group(fd):
    x = make((2, 32, 8, 8), torch.float32, "cl")
    x[0, :8] = 3.25
    x[1, 8:16, 3, 3] = float("nan")
    x[1, 16, 0, 0] = float("inf")
    y = fd.group_norm(x, 4)
    assert torch.equal(y[0, :8], torch.zeros_like(y[0, :8]))
    bad = torch.zeros(2, 32, dtype=torch.bool)
    bad[1, 8:24] = True
    assert torch.equal(torch.isnan(y).any(3).any(2).cpu(), bad)
    near(y[0], so.group_norm(x[:1], 4)[0][0], torch.float32)


def test_gradients_against_differences(fd):
    shape, groups = (2, 12, 4, 3), 3
    x, dy = make(shape, torch.float32, "cl"), make(shape, torch.float32, "cl", seed=5)
    w, b = params(12, torch.float32)
    for act in ("none", "gelu", "gelu_tanh", "silu"):
        _, mean, rstd = fd.group_norm(x, groups, w, b, return_stats=True)
        got = fd.group_norm_backward(dy, x, mean, rstd, groups, w, b, act)
        loss = lambda x_, w_, b_: float((so.group_norm(x_, groups, w_, b_, act=act)[0] * dy.double().cpu()).sum())  # noqa: E731
        for k, base in enumerate((x, w, b)):
            base = base.double().cpu()
            g = torch.Generator().manual_seed(k)
            for _ in range(4):
                d = torch.randn(base.shape, generator=g, dtype=torch.float64)
                h = 1e-5
                args = [t.double().cpu() for t in (x, w, b)]
                args[k] = base + h * d
                up = loss(*args)
                args[k] = base - h * d
                slope = (up - loss(*args)) / (2 * h)
                # central differences: h^2 and cancellation are below 1e-6 here, the gradient's own error FP32 of its size
                assert abs(float((got[k].double().cpu() * d).sum()) - slope) < 1e-3


def test_autograd(fd):
    x, dy = make((2, 24, 6, 6), torch.float32, "cl"), make((2, 24, 6, 6), torch.float32, "cl", seed=2)
    w, b = params(24, torch.float32)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
    fd.group_norm(leaves[0], 4, leaves[1], leaves[2], activation="silu").backward(dy)
    _, mean, rstd = fd.group_norm(x, 4, w, b, return_stats=True)
    for leaf, want in zip(leaves, fd.group_norm_backward(dy, x, mean, rstd, 4, w, b, "silu")):
        assert torch.equal(leaf.grad, want)
    only = w.clone().requires_grad_()
    fd.group_norm(x, 4, only, None).sum().backward()
    assert only.grad is not None and x.grad is None


def test_empty_inputs(fd):
    w, b = params(8, torch.float32)
    for shape in ((0, 8, 3, 3), (2, 8, 0, 3), (0, 8)):
        x = torch.empty(shape, device="cuda")
        y, mean, rstd = fd.group_norm(x, 2, w, b, return_stats=True)
        assert y.shape == x.shape and mean.shape == (shape[0], 2)
        dx, dw, db = fd.group_norm_backward(x, x, mean, rstd, 2, w, b)
        assert dx.shape == x.shape and not dw.any() and not db.any()


def test_another_stream_and_a_captured_graph(fd):
    x, dy = make((4, 64, 20, 20), torch.bfloat16, "cl"), make((4, 64, 20, 20), torch.bfloat16, "cl", seed=4)
    w, b = params(64, torch.bfloat16)

    def step():
        y, mean, rstd = fd.group_norm(x, 8, w, b, activation="silu", return_stats=True)
        return (y, *fd.group_norm_backward(dy, x, mean, rstd, 8, w, b, "silu"))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(captured, want))


def test_behind_a_convolution_in_a_compiled_graph(fd):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 16, 12, 12, generator=g).to(torch.bfloat16).cuda().contiguous(memory_format=torch.channels_last)
    w = (torch.randn(32, 16, 3, 3, generator=g) / 12).to(torch.bfloat16).cuda().contiguous(memory_format=torch.channels_last)
    gw, gb = params(32, torch.bfloat16)

    @fd.graph
    def block(x, w, gw, gb):
        return fd.group_norm(fd.conv2d(x, w, padding=1), 8, gw, gb, activation="silu")

    compiled = fd.compile(block, inputs=[x, w, gw, gb], options={"cache": None})
    assert [n.op_type for n in compiled.graph.nodes] == ["conv2d", "group_norm"]
    want = fd.group_norm(fd.conv2d(x, w, padding=1), 8, gw, gb, activation="silu")
    assert torch.equal(compiled.run(x, w, gw, gb), want)


def test_refusals(fd):
    x = make((2, 12, 4, 4), torch.float32, "cl")
    w, b = params(12, torch.float32)
    for call, exc, text in [
        (lambda: fd.group_norm(x, 5), RuntimeError, "divisible by num_groups"),
        (lambda: fd.group_norm(x, 0), RuntimeError, "divisible by num_groups"),
        (lambda: fd.group_norm(x, 4, w[:6]), RuntimeError, "weight shape mismatch"),
        (lambda: fd.group_norm(x, 4, w, b[None]), RuntimeError, "bias shape mismatch"),
        (lambda: fd.group_norm(x, 4, w.half()), RuntimeError, "weight must be of the input's type"),
        (lambda: fd.group_norm(x.half(), 4, w, b.half()), RuntimeError, "same dtype"),
        (lambda: fd.group_norm(x, 4, w.cpu()), RuntimeError, "input's device"),
        (lambda: fd.group_norm(x.double(), 4), NotImplementedError, "does not support dtype"),
        (lambda: fd.group_norm(x, 4, activation="tanh"), RuntimeError, "activation must be one of"),
        (lambda: fd.group_norm(x, 4, eps=-1.0), RuntimeError, "eps"),
        (lambda: fd.group_norm(x[None], 4), RuntimeError, "2 to 4 dimensions"),
        (lambda: fd.group_norm_backward(x[:1], x, x, x, 4), RuntimeError, "dy must have"),
        (lambda: fd.group_norm_backward(x, x, x, x, 4), RuntimeError, "mean must be"),
    ]:
        with pytest.raises(exc, match=text):
            call()
