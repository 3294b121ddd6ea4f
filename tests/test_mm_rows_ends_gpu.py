"""mm_bias_act at the ends of its range: the most rows.

Tolerances as in test_mm_bias_act_gpu.py."""
import pytest
import torch

from test_mm_bias_act_gpu import check, fd, matrix  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [65535 * 64, 65535 * 64 + 1, 1 << 22, (1 << 22) + 70])
@pytest.mark.parametrize("dtype,k,n", [(torch.float32, 2, 1), (torch.float32, 9, 3), (torch.bfloat16, 5, 1), (torch.float16, 8, 8)], ids=str)
def test_the_most_rows(fd, m, dtype, k, n):  # noqa: F811
    """As many rows as a call of the library takes, and more, which are cut."""
    g = torch.Generator().manual_seed(m)
    a, b = torch.randn(m, k, generator=g).to(dtype).cuda(), torch.randn(k, n, generator=g).to(dtype).cuda()
    bias = torch.randn(n, generator=g).to(dtype).cuda()
    check(fd, a, b, bias, None, "none")
