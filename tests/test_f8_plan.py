"""CPU tests of bof_f8_gemm_plan (include/bof_f8.h): which kernel a product takes."""
import itertools

import pytest

import bofhip
import f8_shapes

AT = 1 << 20   # an address, which nobody follows


def plan(m, n, k, c_type=bofhip.BF16, ld=None, at=AT, work=1 << 30):
    ld, nb = ld or k, -(-k // 128)
    return bofhip.f8_gemm_plan(m, n, k, at, ld, nb, at, ld, nb, c_type, work)


@pytest.mark.parametrize("m,n,k", [(2048, 2048, 1024), (2048, 2048, 4096), (1024, 4096, 14336), (2048, 2048, 16384)])
def test_one_round_of_128x128_stays_one_at_any_depth(m, n, k):
    """256 tiles for 256 CUs.  Tiles of 128 x 160 leave a fifth of them idle and take 12 to 40 % longer."""
    assert plan(m, n, k) == ("128x128", 1)


@pytest.mark.parametrize("m,n", [(2048, 2560), (1024, 5120)])
@pytest.mark.parametrize("k", [4096, 14336])
def test_one_round_of_128x160_that_takes_128x128_two(m, n, k):
    assert plan(m, n, k) == ("128x160", 1)


def test_long_sums_of_few_tiles_are_split():
    assert plan(512, 8192, 28672) == ("256x128", 2)   # 132 us; 128 x 160: 164
    assert plan(512, 8192, 28672, work=0)[1] == 1


def test_the_large_tiles_are_never_split():
    """Their kernel has no parts."""
    for m in (256, 300, 4096, 16384):
        for n in (256, 1000, 8192):
            for k in (128, 1000, 14336, 100000):
                assert plan(m, n, k)[0] != "256x256" or plan(m, n, k)[1] == 1


@pytest.mark.parametrize("kernel,bits,aligned,m,n,k,parts,number", f8_shapes.each())
def test_each_shape_takes_its_kernel(kernel, bits, aligned, m, n, k, parts, number):
    c_type = bofhip.F32 if bits == 32 else bofhip.BF16
    assert plan(m, n, k, c_type, f8_shapes.row_bytes(k, aligned), work=bofhip.f8_gemm_workspace_bytes(m, n, k)) == (kernel, parts)


def test_the_shapes_go_every_way_through_every_kernel():
    """(256 x 128 is split for long sums alone.)"""
    assert {k for k, _, _ in f8_shapes.SHAPES} == set(bofhip.F8_KERNELS)
    assert {k for k, _, aligned in f8_shapes.SHAPES if not aligned} == set(f8_shapes.STAGED)
    for (kernel, _, _), shapes in f8_shapes.SHAPES.items():
        ways = {f8_shapes.way(k, parts) for _, _, k, parts in shapes}
        if kernel == "any":
            assert all(k < 128 for _, _, k, _ in shapes) and len(shapes) == 4
            continue
        want = set(itertools.product([False, True] if kernel in f8_shapes.SPLIT else [False], [False, True], [False, True], [False, True]))
        if kernel == "256x128":
            want = {w for w in want if not w[0] or w[3]}
        assert ways == want, kernel


@pytest.mark.parametrize("wrong", [dict(m=0), dict(n=-1), dict(k=0), dict(k=2 ** 31), dict(c_type=bofhip.E4M3)])
def test_empty_products_have_no_plan(wrong):
    with pytest.raises(bofhip.BofError, match="rc=-1"):
        plan(**{**dict(m=8, n=8, k=300), **wrong})
