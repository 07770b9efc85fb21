"""-m gpu test of the gradient of the norm (include/bof_f8.h): products of dw are added unrounded."""
import pytest
import torch

import bofhip
from test_gpu_f8 import at, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n", [(4097, 64), (4097, 640), (1025, 2048), (1025, 4096), (1025, 8192), (513, 9000), (513, 20000)])
def test_dw_adds_products_unrounded(dev, rows, n):
    """A team of waves takes every 2048th, 512th or 256th row: the last one of `rows` comes to the first one's sum, as 2^k rows of a
    team do.  The first row's product is -P, the last one's p, of which P is the nearest float32; the others are zero, rstd is 1.
    Added unrounded they leave p - P, which float32 holds (the error of a product is a float32); rounded first, zero."""
    g = torch.Generator(device=dev).manual_seed(rows + n)
    dy, h = (torch.zeros(rows, n, device=dev) for _ in range(2))
    dy[-1], h[-1] = (torch.rand(n, generator=g, device=dev) + 0.5 for _ in range(2))
    exact = dy[-1].double() * h[-1].double()
    dy[0], h[0] = -exact.float(), 1.0
    want = exact - exact.float().double()
    assert want.count_nonzero() > n // 2 and torch.equal(want.float().double(), want)
    w, rstd, dx, dw = torch.ones(n, device=dev), torch.ones(rows, device=dev), torch.empty_like(h), torch.empty(n, device=dev)
    work = torch.empty(bofhip.rmsnorm_grad_workspace_bytes(rows, n), dtype=torch.uint8, device=dev)
    bofhip.rmsnorm_grad(rows, n, bofhip.F32, at(dy), n, at(h), n, at(w), at(rstd), 0, 0, at(dx), n, 0.0, at(dw), at(work), work.numel(), stream())
    assert torch.equal(dw.double(), want)
