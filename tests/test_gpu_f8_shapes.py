"""-m gpu tests of bof_f8_gemm (include/bof_f8.h) on shapes that go every way through every one of its kernels (tests/f8_shapes.py), each
kernel with every pair of 8-bit types."""
import pytest

import f8_shapes
from test_gpu_f8 import Mat, check_product, gen

pytestmark = pytest.mark.gpu
TYPES = [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")]


@pytest.mark.parametrize("kernel,bits,aligned,m,n,k,parts,number", f8_shapes.each())
def test_product_every_way(dev, kernel, bits, aligned, m, n, k, parts, number):
    g, (a, b), ld = gen(m + n + k), TYPES[number % 4], f8_shapes.row_bytes(k, aligned)
    A = Mat(g, m, k, a, 1 if number & 4 else 128, ld=ld, lds=-(-k // 128) + 2)
    B = Mat(g, n, k, b, 128 if number & 8 else 1, ld=ld, lds=-(-k // 128) + 1)
    check_product(A, B, "f32" if bits == 32 else ("bf16", "f16")[number & 1], alpha=0.75, beta=1.0 if number & 2 else 0.0, ldc=n + 5)
