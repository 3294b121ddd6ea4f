"""mm_bias_act at the ends of its range: the most rows, the largest numbers, wide blocks, vectors.

Tolerances as in test_mm_bias_act_gpu.py."""
import pytest
import torch

from oracle import delta_oracle as do
from test_mm_bias_act_gpu import ACTS, check, fd, matrix  # noqa: F401
from test_sequence_gpu import DTYPES, IDS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [65535 * 64, 65535 * 64 + 1, 1 << 22, (1 << 22) + 70])
@pytest.mark.parametrize("dtype,k,n", [(torch.float32, 2, 1), (torch.float32, 9, 3), (torch.bfloat16, 5, 1), (torch.float16, 8, 8)], ids=str)
def test_the_most_rows(fd, m, dtype, k, n):  # noqa: F811
    """As many rows as a call of the library takes, and more, which are cut."""
    g = torch.Generator().manual_seed(m)
    a, b = torch.randn(m, k, generator=g).to(dtype).cuda(), torch.randn(k, n, generator=g).to(dtype).cuda()
    bias = torch.randn(n, generator=g).to(dtype).cuda()
    check(fd, a, b, bias, None, "none")


LARGEST = torch.finfo(torch.float32).max


@pytest.mark.parametrize("m,k,n", [(1, 64, 64), (3, 1000, 72), (40, 130, 64), (130, 1100, 300)])
@pytest.mark.parametrize("layout", ["dense", "t"])
def test_the_largest_numbers(fd, m, k, n, layout):  # noqa: F811
    """fp32 operands up to the largest finite one have finite products with small ones, of either sign and in either operand."""
    g = torch.Generator().manual_seed(m)
    for swap in (False, True):
        big, small = (k, n) if swap else (m, k), (m, k) if swap else (k, n)
        x = matrix(g, *big, torch.float32, layout)
        x.copy_(torch.where(torch.rand(big, generator=g).cuda() < 0.5, LARGEST, -LARGEST) * (1 - 2.0 ** -24 * torch.randint(0, 5000, big, generator=g).cuda()))
        w = matrix(g, *small, torch.float32, layout, 2.0 ** -30 / k)
        check(fd, *((w, x) if swap else (x, w)), None, None, "none")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(1, 64, 64), (3, 200, 72), (130, 1100, 300)])
def test_infinite_operands(fd, m, k, n, dtype):  # noqa: F811
    """An infinity times a number of ordinary size is one, of the product's sign; times zero, or with its opposite beside it, NaN."""
    g = torch.Generator().manual_seed(m)
    a, b = matrix(g, m, k, dtype, "dense"), matrix(g, k, n, dtype, "dense")
    a[m // 2, 5] = float("inf")
    b[9, 3] = -float("inf")
    b[5, 7] = 0.0
    a[m // 2, 11] = 2.0
    got, want = fd.mm_bias_act(a, b).double().cpu(), do.mm_bias_act(a, b)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[got.isinf()], want[want.isinf()]) and torch.equal(got.isinf(), want.isinf())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("m,k,n", [(16, 4096, 8192), (15, 4096, 8192), (16, 4104, 7176), (8, 512, 18952), (4, 512, 18952)])
@pytest.mark.parametrize("layout", ["dense", "t", "ragged"])
def test_few_rows_of_wide_layers(fd, m, k, n, dtype, layout):  # noqa: F811
    """On either side of where the convolution is ahead."""
    g = torch.Generator().manual_seed(k + m)
    a, b = matrix(g, m, k, dtype, "dense"), matrix(g, k, n, dtype, layout, k ** -0.5)
    bias = torch.randn(n, generator=g).to(dtype).cuda()
    check(fd, a, b, bias, matrix(g, m, n, dtype, "dense"), "none")
    check(fd, a, b, bias, None, "gelu")


WIDE = [   # m, k, n, layout of a, of b: fp32 blocks of 64 x 128, several of them across, the last a part
    (70, 1100, 300, "dense", "dense"), (130, 1101, 333, "dense", "dense"), (70, 1100, 300, "slice", "t"), (130, 1101, 333, "odd", "ragged"),
    (96, 1100, 260, "t", "t"), (200, 1028, 516, "ragged", "slice"), (65, 4096, 130, "dense", "t"), (128, 1030, 257, "ragged", "t"),
    (1300, 64, 2000, "dense", "dense"), (5000, 33, 520, "dense", "t"),     # by the count of blocks
]


@pytest.mark.parametrize("case", WIDE, ids=[f"{m}x{k}x{n}{a}-{b}" for m, k, n, a, b in WIDE])
def test_wide_blocks(fd, case):  # noqa: F811
    m, k, n, la, lb = case
    g = torch.Generator().manual_seed(m + k)
    a, b = matrix(g, m, k, torch.float32, la), matrix(g, k, n, torch.float32, lb, k ** -0.5)
    bias = torch.randn(n, generator=g).cuda()
    for i, act in enumerate(ACTS):
        check(fd, a, b, bias if i % 2 else None, matrix(g, m, n, torch.float32, ("dense", "ragged", "t", "odd")[i]) if i < 3 else None, act)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(1, 4096, 1), (100, 4096, 1), (1, 520, 72), (5, 1, 1), (1, 1, 40), (300, 128, 1), (1, 129, 1)])
def test_vectors(fd, m, k, n, dtype):  # noqa: F811
    """Extents of one, whose strides say nothing."""
    g = torch.Generator().manual_seed(m + k)
    a, b = matrix(g, m, k, dtype, "dense"), matrix(g, k, n, dtype, "dense", k ** -0.5)
    bias = torch.randn(n, generator=g).to(dtype).cuda()
    want = check(fd, a, b, bias, matrix(g, m, n, dtype, "t"), "gelu_tanh")
    if n == 1:
        b = torch.as_strided(b, (k, 1), (1, 7))
    if m == 1:
        a = torch.as_strided(a, (1, k), (12345, 1))
    assert torch.equal(check(fd, a, b, bias, None, "none"), check(fd, a.clone(), b.clone(), bias, None, "none"))
    assert want.shape == (m, n)
