"""mm_bias_act against its formula in 64 bits.

Tolerances.  fp32 sums of K products, of parts that leave out 2^-20 of a term at most: K * 2^-24 + 2^-20 of the sum of the terms'
sizes, with bias and residual among them; no activation is steeper than 1.13, and GELU by itself is off by 2^-20 of its argument at
most.  Then one rounding (2^-8 bf16, 2^-11 f16, 2^-24 f32)."""
import pytest
import torch

from oracle import delta_oracle as do
from test_sequence_gpu import DTYPES, IDS, ROUND

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "gelu", "gelu_tanh"]


@pytest.fixture(scope="module")
def fd(native_lib):
    import flagdnn_b200

    assert torch.cuda.is_available()
    return flagdnn_b200


def matrix(g, rows, cols, dtype, layout, std=1.0):
    """dense; a column slice of 16-byte columns, of odd ones; transposed; at an odd address."""
    t = (torch.randn(rows, cols, generator=g) * std).to(dtype)
    if layout == "t":
        return t.t().contiguous().cuda().t()
    if layout in ("slice", "ragged"):
        pad = 16 if layout == "slice" else 5
        big = torch.full((rows, cols + 2 * pad), float("nan"), dtype=dtype)
        big[:, pad:pad + cols] = t
        return big.cuda()[:, pad:pad + cols]
    if layout == "odd":
        flat = torch.zeros(rows * cols + 1, dtype=dtype)
        flat[1:] = t.reshape(-1)
        return flat.cuda()[1:].view(rows, cols)
    return t.cuda()


def check(fd, a, b, bias, residual, act):
    got = fd.mm_bias_act(a, b, bias, residual=residual, activation=act)
    want = do.mm_bias_act(a, b, bias, residual, act)
    size = a.double().cpu().abs() @ b.double().cpu().abs()
    for t in (bias, residual):
        if t is not None:
            size = size + t.double().cpu().abs()
    tol = 1.13 * (a.shape[1] * 2.0 ** -24 + 2.0 ** -20) + 2.0 ** -20
    least = 2.0 ** -25 if a.dtype == torch.float16 else 1e-38
    assert got.shape == want.shape and got.dtype == a.dtype and got.is_contiguous()
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= 1.02 * ROUND[a.dtype] * want.abs() + tol * size + least)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off / (size + 1e-300)).max())} of the terms"
    return got


PRODUCTS = [   # m, k, n, layout of a, of b
    (1, 64, 64, "dense", "dense"), (1, 1000, 333, "dense", "t"), (1, 4096, 2048, "dense", "dense"), (3, 72, 40, "slice", "slice"),
    (7, 1001, 777, "dense", "dense"), (8, 130, 70, "odd", "odd"), (16, 512, 520, "dense", "t"), (17, 33, 129, "ragged", "ragged"),
    (31, 256, 64, "t", "dense"), (33, 640, 200, "dense", "slice"), (64, 2048, 72, "dense", "t"), (65, 96, 88, "dense", "dense"),
    (100, 520, 264, "slice", "t"), (130, 1001, 96, "ragged", "dense"), (300, 64, 1032, "dense", "t"), (2, 1, 5, "dense", "dense"),
    (5, 7, 9, "dense", "t"), (1, 1, 1, "dense", "dense"), (200, 4, 64, "dense", "dense"), (500, 3, 8, "t", "t"), (1, 9000, 16, "dense", "t"),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("case", PRODUCTS, ids=[f"{m}x{k}x{n}{a}-{b}" for m, k, n, a, b in PRODUCTS])
def test_products(fd, case, dtype):
    m, k, n, la, lb = case
    g = torch.Generator().manual_seed(m + k)
    a, b = matrix(g, m, k, dtype, la), matrix(g, k, n, dtype, lb, k ** -0.5)
    bias = torch.randn(n, generator=g).to(dtype).cuda()
    residual = matrix(g, m, n, dtype, "dense")
    for i, act in enumerate(ACTS):
        check(fd, a, b, bias if i % 2 else None, residual if i < 2 else None, act)
    check(fd, a, b, bias, matrix(g, m, n, dtype, "ragged"), "gelu")
    check(fd, a, b, bias, matrix(g, m, n, dtype, "t"), "none")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_nothing_to_multiply(fd, dtype):
    g = torch.Generator().manual_seed(0)
    bias, residual = torch.randn(24, generator=g).to(dtype).cuda(), torch.randn(5, 24, generator=g).to(dtype).cuda()
    for m in (5, 0, 300):
        a, b = torch.empty(m, 0, dtype=dtype, device="cuda"), torch.empty(0, 24, dtype=dtype, device="cuda")
        r = residual[:m] if m <= 5 else None
        got = fd.mm_bias_act(a, b, bias, residual=r, activation="relu")
        want = torch.relu(bias.double() + (0 if r is None else r.double())).expand(m, 24)
        assert got.shape == (m, 24) and torch.equal(got, want.to(dtype))
    assert fd.mm_bias_act(torch.ones(3, 4, dtype=dtype, device="cuda"), torch.ones(4, 0, dtype=dtype, device="cuda")).shape == (3, 0)


def test_long_sums_do_not_drift(fd):
    """fp32 sums of many products of one sign: cut at every step they would be 1e-5 too small; rounded ones scatter."""
    g = torch.Generator().manual_seed(5)
    for m in (3, 40, 200):
        a, b = torch.rand(m, 8192, generator=g).cuda(), torch.rand(8192, 96, generator=g).cuda()
        want = a.double() @ b.double()
        drift = float((fd.mm_bias_act(a, b).double() / want - 1).mean())
        assert abs(drift) < 1e-6, drift


def test_infinite_columns_stay_in_their_columns(fd):
    """What stands beside a product's columns, rows and reduction is not multiplied."""
    g = torch.Generator().manual_seed(1)
    for m in (3, 90):
        for dtype in DTYPES:
            a, b = matrix(g, m, 200, dtype, "slice"), matrix(g, 200, 100, dtype, "slice")
            b[:, 7] = float("inf")
            a[1] = float("nan")
            got = fd.mm_bias_act(a, b)
            assert got[1].isnan().all()
            keep = [i for i in range(m) if i != 1]
            cols = [j for j in range(100) if j != 7]
            assert got[keep][:, cols].isfinite().all() and not got[keep][:, 7].isfinite().any()


def test_rounded_once(fd):
    """bias and residual meet the sum before it is rounded: 1 + 2^-9 - 1 is not zero in bf16."""
    for m in (4, 100):
        a, b = torch.zeros(m, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(64, 64, dtype=torch.bfloat16, device="cuda")
        a[:, 0], a[:, 1], b[0], b[1] = 1.0, 2.0 ** -9, 1.0, 1.0
        bias, residual = torch.zeros(64, device="cuda").bfloat16(), torch.full((m, 64), -1.0, device="cuda").bfloat16()
        assert (fd.mm_bias_act(a, b, bias, residual=residual).float() == 2.0 ** -9).all()


def test_captured_and_on_streams(fd):
    g = torch.Generator().manual_seed(2)
    calls = [(matrix(g, m, 512, torch.bfloat16, "dense"), matrix(g, 512, 640, torch.bfloat16, "t")) for m in (1, 40, 100)]
    want = [fd.mm_bias_act(a, b, activation="gelu") for a, b in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = []
    for s, (a, b) in zip(streams, calls):
        with torch.cuda.stream(s):
            got.append(fd.mm_bias_act(a, b, activation="gelu"))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [fd.mm_bias_act(a, b, activation="gelu") for a, b in calls]
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_the_python_route_gives_the_same(fd, monkeypatch):
    from flagdnn_b200 import conv_host

    g = torch.Generator().manual_seed(3)
    for m, k, lr in ((2, 300, "dense"), (90, 300, "dense"), (90, 300, "ragged"), (700, 5, "dense")):
        a, b, r = matrix(g, m, k, torch.float16, "dense"), matrix(g, k, 72, torch.float16, "t"), matrix(g, m, 72, torch.float16, lr)
        bias = torch.randn(72, generator=g).half().cuda()
        with monkeypatch.context() as mp:
            first = fd.mm_bias_act(a, b, bias, residual=r, activation="relu")
            mp.setattr(conv_host, "_fast", False)
            assert torch.equal(first, fd.mm_bias_act(a, b, bias, residual=r, activation="relu"))
            mp.setattr(conv_host, "_MOST_ROWS", 300)
            if k < 8:
                assert torch.equal(first, fd.mm_bias_act(a, b, bias, residual=r, activation="relu"))


def test_refusals(fd):
    a, b = torch.zeros(4, 8, device="cuda"), torch.zeros(8, 6, device="cuda")

    def refused(error, match, *args, **kw):
        with pytest.raises(error, match=match):
            fd.mm_bias_act(*args, **kw)

    refused(RuntimeError, "cannot be multiplied", a, a)
    refused(RuntimeError, "must be a matrix", a[0], b)
    refused(RuntimeError, "mat2 must be torch.float32", a, b.half())
    refused(RuntimeError, "bias must have shape", a, b, torch.zeros(4, device="cuda"))
    refused(RuntimeError, "bias must be on", a, b, torch.zeros(6))
    refused(RuntimeError, "residual must have shape", a, b, residual=a)
    refused(RuntimeError, "residual must be torch.float32", a, b, residual=torch.zeros(4, 6, device="cuda").half())
    refused(RuntimeError, "activation must be one of", a, b, activation="silu")
    refused(NotImplementedError, "does not support", a.double(), b.double())
    for i in range(2):
        args = [a, b]
        args[i] = args[i].clone().requires_grad_()
        refused(NotImplementedError, "no gradients", *args)
    refused(NotImplementedError, "no gradients", a, b, residual=torch.zeros(4, 6, device="cuda", requires_grad=True))
