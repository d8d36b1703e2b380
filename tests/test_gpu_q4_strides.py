"""Linears with 4-bit weights whose operands are views of buffers with very long rows: further apart than the kernels' 32-bit
offsets reach within a tile, so they are copied."""
import pytest
import torch

from test_gpu_q4_linear import DEV, check, rows, weights

pytestmark = pytest.mark.gpu


def far(t, ld):
    """t's values in rows ld elements apart."""
    buf = torch.empty(t.shape[0] * ld, dtype=t.dtype, device=DEV)
    view = buf.view(t.shape[0], ld)[:, :t.shape[1]]
    view.copy_(t)
    return view


@pytest.mark.parametrize("M", [3, 40])
def test_rows_far_apart(gpu_lib, M):
    from opendecider_amd import kernels
    N, K = 20, 96
    qs, d, w = weights(N, K)
    x = rows(M, K)
    here = [t.to(DEV) for t in (x, qs, d)]
    want = kernels.q4_linear(*here)
    check(want, x, w, d)
    for i, ld in enumerate(((1 << 21) + 8, (1 << 22) + 16, (1 << 21) + 1)):
        args = list(here)
        args[i] = far(args[i], ld)
        assert args[i].stride(0) == ld
        assert torch.equal(kernels.q4_linear(*args), want)
