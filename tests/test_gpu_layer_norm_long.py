"""Layer norm of the longest rows, against 64 bits."""
import pytest
import torch

from test_gpu_layer_norm import F32, check

pytestmark = pytest.mark.gpu


def test_sums_of_more_columns_than_one_launch_has():
    """2^25 columns and more: dw and db are added 16 columns to 1024 threads, and a
    launch has fewer than 2^32 of them."""
    N = 2 ** 25 + 24
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    check(r(2, N), r(N), r(N), r(2, N))
