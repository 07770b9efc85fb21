"""-m gpu tests of the operators in 8-bit floating point (include/bof_f8.h) against plain forms in 64 bits.  Tolerances
are bounds: every rounding of the kernels counted at half a step (a cut at a whole one), see f8_util.product_bound."""
import pytest
import torch

import bofhip
import f8_util as f8
from f8_util import CODE, DENSE, F8, HALF, U

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def at(t):
    return 0 if t is None else t.data_ptr()


def padded(rows, cols, dtype, ld, offset=0, fill=0x5A):
    """(view, flat): rows x cols with ld elements from row to row, `offset` elements into its storage; every byte of the
    storage is `fill`, so that writes outside the view show."""
    z = torch.empty(0, dtype=dtype).element_size()
    flat = torch.full(((rows * ld + offset + 16) * z,), fill, dtype=torch.uint8, device="cuda")
    return flat.view(dtype).as_strided((rows, cols), (ld, 1), offset), flat


def outside_untouched(view, flat, fill=0x5A):
    mask = torch.ones_like(flat, dtype=torch.bool)
    z = view.element_size()
    inside = mask.view(-1, z).as_strided((*view.shape, z), (view.stride(0) * z, z, 1), view.storage_offset() * z)
    inside.fill_(False)
    return bool((flat[mask] == fill).all())


class Mat:
    """A matrix in 8 bits: random values quantised by the plain form, with strides of its own."""

    def __init__(self, g, rows, cols, f8t="e4m3", group=1, ld=None, lds=None, offset=0, x=None):
        x = torch.randn(rows, cols, generator=g, device="cuda") if x is None else x
        q, codes = f8.quantised(x.double(), f8t, group)
        ld, lds = ld or cols, lds or codes.shape[1]
        self.q, _ = padded(rows, cols, torch.uint8, ld, offset, fill=0x7F)   # NaN where nothing belongs
        self.q.copy_(q)
        self.s, _ = padded(codes.shape[0], codes.shape[1], torch.uint8, lds, offset, fill=0xFF)
        self.s.copy_(codes)
        self.type, self.group, self.shape = f8t, group, (rows, cols)

    def args(self):
        return at(self.q), self.q.stride(0), CODE[self.type], at(self.s), self.s.stride(0), self.group

    def values(self):
        return f8.decoded(self.q, self.s, self.type, self.group)


def product(A, B, c, c_type, alpha=1.0, beta=0.0, work=None, st=None):
    (m, k), n = A.shape, B.shape[0]
    bofhip.f8_gemm(m, n, k, alpha, *A.args(), *B.args(), beta, at(c), c.stride(0), CODE[c_type], at(work),
                   0 if work is None else work.numel(), stream() if st is None else st)


def check_product(A, B, c_type, alpha=1.0, beta=0.0, ldc=None, offset=0, work="full", seed=0):
    (m, k), n = A.shape, B.shape[0]
    c, flat = padded(m, n, DENSE[c_type], ldc or n, offset)
    c.copy_(torch.randn(m, n, generator=gen(seed + 1), device="cuda") * 3)
    c0 = c.double()
    if beta == 0:
        c.fill_(float("nan"))
    nbytes = bofhip.f8_gemm_workspace_bytes(m, n, k)
    w = torch.empty(nbytes if work == "full" else work, dtype=torch.uint8, device="cuda") if work and nbytes else None
    product(A, B, c, c_type, alpha, beta, w)
    torch.cuda.synchronize()
    a, b = A.values(), B.values()
    want = alpha * (a @ b.t()) + (beta * c0 if beta else 0)
    bound = f8.product_bound(a, b, c_type, alpha, beta, c0, want)
    err = (c.double() - want).abs()
    worst = (err - bound).max().item()
    assert worst <= 0, f"m {m} n {n} k {k} {A.type}/{A.group} x {B.type}/{B.group} -> {c_type}: {err.max().item()} off, {worst} over the bound"
    assert outside_untouched(c, flat)
    return c


# ---- product -----------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 16, 128), (1, 257, 129), (1, 4096, 2048), (2, 300, 1000), (16, 129, 256), (17, 100, 127), (31, 513, 640),
          (48, 640, 1000), (64, 256, 4096), (65, 128, 384), (100, 1000, 515), (128, 128, 128), (129, 255, 257), (250, 130, 3333),
          (256, 256, 1024), (257, 513, 144), (511, 300, 2048), (512, 512, 640), (1000, 100, 16), (768, 1024, 256)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("c_type", ["bf16", "f32"])
def test_product_sizes(dev, m, n, k, c_type):
    g = gen(m * 7 + n * 3 + k)
    check_product(Mat(g, m, k, group=1, ld=-(-k // 16) * 16), Mat(g, n, k, group=128, ld=-(-k // 16) * 16), c_type)


@pytest.mark.parametrize("m,n,k", [(1, 130, 520), (40, 130, 520), (300, 270, 520)])
@pytest.mark.parametrize("a,b", [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("ga,gb", [(1, 1), (1, 128), (128, 1), (128, 128)])
@pytest.mark.parametrize("c_type", ["f16", "f32"])
def test_product_types_and_groups(dev, m, n, k, a, b, ga, gb, c_type):
    g = gen(m + len(a + b) + ga + gb)
    check_product(Mat(g, m, k, a, ga), Mat(g, n, k, b, gb), c_type)


@pytest.mark.parametrize("m,n,k", [(1, 70, 300), (20, 300, 515), (300, 300, 515), (512, 256, 1024)])
@pytest.mark.parametrize("lda,ldb,lds,ldc,offset", [(0, 0, 0, 0, 0), (1, 3, 1, 1, 1), (16, 32, 4, 8, 0), (16, 16, 3, 5, 16), (5, 0, 7, 0, 2)])
def test_product_strides(dev, m, n, k, lda, ldb, lds, ldc, offset):
    g = gen(m + lda)
    A = Mat(g, m, k, group=1, ld=k + lda, lds=-(-k // 128) + lds, offset=offset)
    B = Mat(g, n, k, group=128, ld=k + ldb, lds=-(-k // 128) + lds, offset=offset)
    for c_type in ("bf16", "f32"):
        check_product(A, B, c_type, ldc=n + ldc, offset=offset, beta=0.5)


@pytest.mark.parametrize("alpha,beta", [(1.0, 1.0), (-2.5, 0.0), (0.5, -1.5), (0.0, 2.0), (0.0, 0.0), (0.0, 1.0)])
@pytest.mark.parametrize("m", [1, 33, 300])
@pytest.mark.parametrize("c_type", ["bf16", "f16", "f32"])
def test_product_alpha_beta(dev, alpha, beta, m, c_type):
    g = gen(m)
    check_product(Mat(g, m, 700), Mat(g, 290, 700, group=128), c_type, alpha, beta)


@pytest.mark.parametrize("c_type", ["bf16", "f32"])
def test_product_without_k(dev, c_type):
    c = torch.randn(5, 7, device="cuda").to(DENSE[c_type])
    c0 = c.clone()
    bofhip.f8_gemm(5, 7, 0, 1.0, 0, 0, bofhip.E4M3, 0, 0, 1, 0, 0, bofhip.E4M3, 0, 0, 1, 2.0, at(c), 7, CODE[c_type], 0, 0, stream())
    assert torch.equal(c, c0 * 2)
    c.fill_(float("nan"))
    bofhip.f8_gemm(5, 7, 0, 1.0, 0, 0, bofhip.E4M3, 0, 0, 1, 0, 0, bofhip.E4M3, 0, 0, 1, 0.0, at(c), 7, CODE[c_type], 0, 0, stream())
    assert torch.equal(c, torch.zeros_like(c))


@pytest.mark.parametrize("alpha", [float("inf"), float("nan")])
def test_product_without_k_and_any_alpha(dev, alpha):
    c = torch.randn(5, 8, device="cuda")
    c0 = c.clone()
    bofhip.f8_gemm(5, 8, 0, alpha, 0, 0, bofhip.E4M3, 0, 0, 1, 0, 0, bofhip.E4M3, 0, 0, 1, -3.0, at(c), 8, bofhip.F32, 0, 0, stream())
    assert torch.equal(c, c0 * -3)


@pytest.mark.parametrize("m,n,k,c_type", [(3, 300, 500, "bf16"), (40, 200, 300, "f16"), (300, 1000, 700, "bf16"), (7, 90, 300, "f32"), (100, 300, 400, "f32")])
def test_product_of_mapped_host_memory(dev, m, n, k, c_type):
    g = gen(k)
    A, B = Mat(g, m, k, ld=k), Mat(g, n, k, group=128, ld=k)
    want = check_product(A, B, c_type)
    for x in (A, B):
        x.q = torch.empty(x.q.shape, dtype=torch.uint8, pin_memory=True).copy_(x.q)
        x.s = torch.empty(x.s.shape, dtype=torch.uint8, pin_memory=True).copy_(x.s)
    c = torch.zeros_like(want)
    product(A, B, c, c_type)
    torch.cuda.synchronize()
    ref = torch.zeros_like(want)
    for x in (A, B):
        x.q, x.s = x.q.cuda(), x.s.cuda()
    product(A, B, ref, c_type)
    assert torch.equal(c, ref)


@pytest.mark.parametrize("m,n,k", [(2048, 2048, 512), (2048, 2304, 1024), (2100, 2300, 1100), (4000, 1300, 640), (2111, 2048, 1920), (2500, 2056, 2047), (4096, 4100, 256), (2048, 2050, 6500),
                                   (3000, 3700, 1100), (3001, 3703, 640), (2999, 3750, 6500), (1500, 1500, 385), (1501, 1400, 4500),
                                   (1600, 4000, 700), (1601, 4096, 1281), (1800, 4001, 5000), (4096, 4000, 2100), (5000, 1000, 700)])
@pytest.mark.parametrize("a,ga,b,gb", [("e4m3", 1, "e4m3", 128), ("e5m2", 1, "e4m3", 1), ("e4m3", 128, "e5m2", 1), ("e5m2", 128, "e5m2", 128)])
def test_product_many_tiles(dev, m, n, k, a, ga, b, gb):
    """Outputs of many tiles, with whole and cut tiles at the edges, odd numbers of blocks and a short last one."""
    g = gen(m + k)
    up = -(-k // 16) * 16
    A, B = Mat(g, m, k, a, ga, ld=up), Mat(g, n, k, b, gb, ld=up, lds=-(-k // 128) + 3)
    check_product(A, B, "bf16")
    check_product(Mat(g, m, k, a, ga, ld=k + 1), B, "bf16")
    check_product(Mat(g, m, k, a, ga, ld=up + 4, offset=8), B, "bf16")
    check_product(A, B, "f16", alpha=0.5, beta=1.0, ldc=n + 1)
    check_product(A, B, "f32", beta=1.0)


@pytest.mark.parametrize("m,n,k", [(128, 128, 129), (300, 400, 300), (333, 129, 6000), (130, 200, 12345), (256, 257, 4096), (700, 1030, 385), (100, 300, 2500), (127, 64, 5000),
                                   (400, 2900, 8200)])
@pytest.mark.parametrize("pad", [0, 1, 4, 16])
def test_product_few_tiles(dev, m, n, k, pad):
    """Outputs of some tiles of 128, rows aligned or not, whole or split along k, with and without a short last block."""
    g = gen(m + k)
    up = -(-k // pad) * pad if pad > 1 else k + pad
    A, B = Mat(g, m, k, ld=up), Mat(g, n, k, "e5m2", 128, ld=up)
    for c_type in ("bf16", "f16", "f32"):
        check_product(A, B, c_type, alpha=-0.5, beta=0.25, ldc=n + 3)
        check_product(A, B, c_type, work=None)


@pytest.mark.parametrize("m,n,k", [(1, 256, 8192), (16, 64, 16384), (128, 128, 16384), (256, 256, 8192), (130, 140, 9000)])
@pytest.mark.parametrize("c_type", ["bf16", "f32"])
def test_product_split_along_k(dev, m, n, k, c_type):
    """Few output tiles: with the whole workspace, with room for two parts and with none; each within the bound, and the
    same call gives the same bits."""
    g = gen(k)
    A, B = Mat(g, m, k, "e5m2"), Mat(g, n, k, group=1)
    full = check_product(A, B, c_type, beta=1.0)
    assert torch.equal(full, check_product(A, B, c_type, beta=1.0))
    check_product(A, B, c_type, beta=1.0, work=2 * 4 * m * n + 64)
    check_product(A, B, c_type, beta=1.0, work=None)


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("c_type", ["bf16", "f32"])
@pytest.mark.parametrize("what", ["a NaN", "b NaN", "a scale NaN", "b scale NaN", "inf"])
def test_product_carries_nans_to_their_row_or_column_only(dev, m, c_type, what):
    g = gen(9)
    n, k = 290, 400
    A, B = Mat(g, m, k, "e5m2"), Mat(g, n, k, "e4m3", 128)
    if what == "a NaN":
        A.q[m - 1, k - 1] = 0x7F
    elif what == "inf":
        A.q[m - 1, 200] = 0x7C
        B.q[:, 200] = 0x38   # 1.0
    elif what == "b NaN":
        B.q[289, 129] = 0x7F
    elif what == "a scale NaN":
        A.s[m - 1, 3] = 255
    else:
        B.s[2, 0] = 255
    c = torch.zeros(m, n, dtype=DENSE[c_type], device="cuda")
    product(A, B, c, c_type)
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    if what.startswith("a") or what == "inf":
        bad[m - 1] = True
    elif what == "b NaN":
        bad[:, 289] = True
    else:
        bad[:, 256:] = True
    assert torch.equal(bad, torch.isinf(c) if what == "inf" else torch.isnan(c))


@pytest.mark.parametrize("c_type", ["bf16", "f32"])
@pytest.mark.parametrize("m", [3, 200])
def test_product_scales_far_apart(dev, m, c_type):
    """Blocks whose scales differ by 2^80, and operands whose scales cancel: 2^-60 against 2^60."""
    g = gen(4)
    n, k = 140, 512
    x = torch.randn(m, k, generator=g, device="cuda") * 2.0 ** -60
    x[:, 128:256] *= 2.0 ** 80
    y = torch.randn(n, k, generator=g, device="cuda") * 2.0 ** 60
    y[:, 128:256] *= 2.0 ** -80
    check_product(Mat(g, m, k, x=x), Mat(g, n, k, group=128, x=y), c_type)


def test_product_beyond_four_gigabytes(dev):
    """Rows 1.5 and 0.75 GiB apart: offsets of A, B and C past 32 bits."""
    g = gen(2)
    m, n, k, far = 4, 20, 300, 3 << 29
    A, B = Mat(g, m, k), Mat(g, n, k, group=128)
    big = torch.empty((m - 1) * far + k, dtype=torch.uint8, device="cuda").as_strided((m, k), (far, 1))
    big.copy_(A.q)
    A.q = big
    check_product(A, B, "bf16")
    out = torch.empty((m - 1) * (far // 2) + n, dtype=torch.bfloat16, device="cuda").as_strided((m, n), (far // 2, 1))
    ref = check_product(A, B, "bf16")
    product(A, B, out, "bf16")
    assert torch.equal(out, ref)
    del big
    B.q, q = torch.empty((n - 1) * (far // 4) + k, dtype=torch.uint8, device="cuda").as_strided((n, k), (far // 4, 1)), B.q
    B.q.copy_(q)
    assert torch.equal(check_product(A, B, "bf16"), ref)


# ---- quantiser ---------------------------------------------------------------------------------------------------
def run_quant(x, x_type, f8t, group, both, pad=0, offset=0, only_t=False):
    rows, cols = x.shape
    q = qf = s = sf = qt = qtf = st = stf = None
    if not only_t:
        q, qf = padded(rows, cols, torch.uint8, cols + pad, offset)
        s, sf = padded(-(-rows // group), -(-cols // 128), torch.uint8, -(-cols // 128) + pad, offset)
    if both or only_t:
        qt, qtf = padded(cols, rows, torch.uint8, rows + pad, offset)
        st, stf = padded(-(-cols // group), -(-rows // 128), torch.uint8, -(-rows // 128) + pad, offset)
    ld = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    bofhip.f8_quant(rows, cols, at(x), x.stride(0), CODE[x_type], CODE[f8t], group, at(q), ld(q), at(s), ld(s), at(qt), ld(qt), at(st), ld(st),
                    stream())
    torch.cuda.synchronize()
    for v, f in ((q, qf), (s, sf), (qt, qtf), (st, stf)):
        assert v is None or outside_untouched(v, f)
    return q, s, qt, st


def same_bytes(got, want):
    """Equal codes; any NaN is as good as another."""
    nan = (want & 0x7F) > 0x7C if want.dtype == torch.uint8 and same_bytes.e5m2 else (want & 0x7F) == 0x7F
    gnan = (got & 0x7F) > 0x7C if same_bytes.e5m2 else (got & 0x7F) == 0x7F
    return torch.equal(nan, gnan) and torch.equal(got[~nan], want[~nan])


def check_quant(x, x_type, f8t, group, **kw):
    same_bytes.e5m2 = f8t == "e5m2"
    q, s, qt, st = run_quant(x, x_type, f8t, group, **kw)
    for got, codes, v in ((q, s, x.double()), (qt, st, x.double().t())):
        if got is not None:
            wq, wc = f8.quantised(v, f8t, group)
            assert torch.equal(codes.long(), wc), "scales"
            assert same_bytes(got.contiguous(), wq), "elements"


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (1, 1000), (3, 129), (64, 256), (127, 128), (128, 127), (129, 4096), (300, 515), (1000, 96),
                                       (513, 130), (256, 512), (1, 20000), (2000, 1)])
@pytest.mark.parametrize("x_type", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("group", [1, 128])
def test_quant_sizes(dev, rows, cols, x_type, group):
    x = (torch.randn(rows, cols, generator=gen(rows + cols), device="cuda") * 5).to(DENSE[x_type])
    check_quant(x, x_type, "e4m3", group, both=True)
    check_quant(x, x_type, "e5m2", group, both=False)
    check_quant(x, x_type, "e4m3", group, both=False, only_t=True)


@pytest.mark.parametrize("pad,offset,ldx", [(0, 0, 8), (1, 1, 1), (16, 16, 16), (3, 5, 0), (8, 0, 3), (4, 4, 4)])
@pytest.mark.parametrize("x_type", ["bf16", "f32"])
@pytest.mark.parametrize("group", [1, 128])
def test_quant_strides(dev, pad, offset, ldx, x_type, group):
    rows, cols = 140, 400
    x, _ = padded(rows, cols, DENSE[x_type], cols + ldx, offset)
    x.copy_(torch.randn(rows, cols, generator=gen(pad), device="cuda"))
    check_quant(x, x_type, "e4m3", group, both=True, pad=pad, offset=offset)
    check_quant(x, x_type, "e4m3", group, both=False, pad=pad, offset=offset)


@pytest.mark.parametrize("f8t", ["e4m3", "e5m2"])
@pytest.mark.parametrize("x_type", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("group", [1, 128])
def test_quant_special_values(dev, f8t, x_type, group):
    """Zero blocks, subnormals, the type's largest value, the borders of the scale, NaN and infinities among others."""
    x = torch.randn(200, 600, generator=gen(1), device="cuda")
    x[:, 128:256] = 0
    x[5:, 130] = -0.0
    x[0, 256:384] *= 1e-30
    x[1, :128] = 2.0 ** -149
    x[2, :128] = torch.finfo(DENSE[x_type]).max
    x[3, :128] = torch.finfo(DENSE[x_type]).smallest_normal
    top = f8.LARGEST[f8t]
    for i in range(128):   # on the border of two scales, and next to it
        x[4, i] = top * 2.0 ** -10 if i == 0 else 0.001
    x[5, 0] = top * 2.0 ** -10 * (1 + torch.finfo(DENSE[x_type]).eps)
    x[6, 0:128] = torch.linspace(-1.9, 1.9, 128) * top * 2.0 ** -12
    x[7, 7], x[8, 300], x[9, 599] = float("nan"), float("inf"), -float("inf")
    x[10, :] = float("nan")
    x[11, 384:512] = float("inf")
    x[150:, 512:] = float("nan")
    check_quant(x.to(DENSE[x_type]), x_type, f8t, group, both=True)


def test_quant_beyond_four_gigabytes(dev):
    rows, cols, far = 5, 300, 1 << 30
    x = torch.empty((rows - 1) * far + cols, dtype=torch.float32, device="cuda").as_strided((rows, cols), (far, 1))
    x.copy_(torch.randn(rows, cols, generator=gen(3), device="cuda"))
    check_quant(x, "f32", "e4m3", 1, both=True)


# ---- norm --------------------------------------------------------------------------------------------------------
def sum_error(n):
    """Relative error of a sum of n squares or products in fp32: at most n / 64 in a row, then a tree; the rest is the
    handful of operations around it."""
    return (n / 64 + 40) * U


def run_norm(x, r, w, t, eps=1e-6, f8t="e4m3", pad=0, offset=0, h="new", want="qyr", st=None):
    rows, n = x.shape
    q, qf = padded(rows, n, torch.uint8, n + pad, offset) if "q" in want else (None, None)
    s, sf = padded(rows, -(-n // 128), torch.uint8, -(-n // 128) + pad, offset) if "q" in want else (None, None)
    y, yf = padded(rows, n, DENSE[t], n + pad, offset) if "y" in want else (None, None)
    hh, hf = padded(rows, n, DENSE[t], n + pad, offset) if isinstance(h, str) else (h, None)
    rstd = torch.empty(rows, device="cuda") if "r" in want else None
    ld = lambda a: 0 if a is None else a.stride(0)  # noqa: E731
    bofhip.rmsnorm_f8(rows, n, CODE[t], at(x), ld(x), at(r), ld(r), at(w), eps, at(hh), ld(hh), CODE[f8t], at(q), ld(q), at(s), ld(s), at(y),
                      ld(y), at(rstd), stream() if st is None else st)
    torch.cuda.synchronize()
    for v, f in ((q, qf), (s, sf), (y, yf), (hh, hf)):
        assert f is None or outside_untouched(v, f)
    return hh, q, s, y, rstd


def check_norm(x, r, w, t, eps=1e-6, f8t="e4m3", **kw):
    n = x.shape[1]
    h64, rstd64, y64 = f8.rms_norm(x.clone(), None if r is None else r.clone(), w, eps)
    hh, q, s, y, rstd = run_norm(x, r, w, t, eps, f8t, **kw)
    e = sum_error(n)
    if hh is not None:
        assert ((hh.double() - h64).abs() <= (HALF[t] + U) * h64.abs() + torch.finfo(DENSE[t]).smallest_normal * HALF[t] * 2).all()
    if rstd is not None:
        assert ((rstd.double() - rstd64).abs() <= e * rstd64).all()
    tiny = torch.finfo(DENSE[t]).smallest_normal * HALF[t] * 2
    if y is not None:
        assert ((y.double() - y64).abs() <= (HALF[t] + 2 * e) * y64.abs() + tiny).all()
    if q is not None:
        codes = s.long()
        lo, hi = f8.block_codes(y64 * (1 - 2 * e), f8t, 1), f8.block_codes(y64 * (1 + 2 * e), f8t, 1)
        assert ((codes == lo) | (codes == hi)).all(), "scales"
        got, sc = f8.decoded(q, codes, f8t, 1), f8.spread(codes, 1, *x.shape)
        assert ((got - y64).abs() <= torch.maximum((HALF[f8t] + 4 * e) * y64.abs(), sc * f8.SMALLEST[f8t] / 2 + 4 * e * y64.abs())).all()


@pytest.mark.parametrize("rows,n", [(1, 1), (1, 4096), (3, 127), (5, 129), (2, 640), (7, 1000), (1, 8192), (300, 256), (4, 5001), (2, 16384), (2, 33000),
                                    (1, 100001), (70, 2048)])
@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("res", [False, True])
def test_norm_sizes(dev, rows, n, t, res):
    g = gen(rows + n)
    x = torch.randn(rows, n, generator=g, device="cuda").to(DENSE[t])
    r = (torch.randn(rows, n, generator=g, device="cuda") * 3).to(DENSE[t]) if res else None
    w = (1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(DENSE[t])
    check_norm(x, r, w, t)
    check_norm(x, r, w, t, f8t="e5m2", want="q", h=None)


@pytest.mark.parametrize("pad,offset", [(0, 1), (1, 0), (8, 8), (16, 16), (3, 5), (4, 4)])
@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("n", [520, 2048])
def test_norm_strides(dev, pad, offset, t, n):
    g = gen(pad + n)
    x, r = (padded(6, n, DENSE[t], n + pad, offset)[0] for _ in range(2))
    x.copy_(torch.randn(6, n, generator=g, device="cuda"))
    r.copy_(torch.randn(6, n, generator=g, device="cuda"))
    w = torch.randn(n + 1, generator=g, device="cuda").to(DENSE[t])[1:]
    check_norm(x, r, w, t, pad=pad, offset=offset)


@pytest.mark.parametrize("n", [700, 1024, 4096, 40000])
@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("over", ["x", "r"])
@pytest.mark.parametrize("want", ["q", "y", "qyr", "r"])
def test_norm_in_place_and_single_outputs(dev, n, t, over, want):
    g = gen(n)
    x = torch.randn(5, n, generator=g, device="cuda").to(DENSE[t])
    r = torch.randn(5, n, generator=g, device="cuda").to(DENSE[t])
    w = torch.randn(n, generator=g, device="cuda").to(DENSE[t])
    ref = run_norm(x, r, w, t, want=want)
    x2, r2 = x.clone(), r.clone()
    got = run_norm(x2, r2, w, t, h=x2 if over == "x" else r2, want=want)
    for a, b in zip(got, ref):
        assert (a is None and b is None) or torch.equal(a, b)
    check_norm(x, r, w, t, want=want, h=None)


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("n", [640, 4096])
def test_norm_special_rows(dev, t, n):
    """Zero rows, with and without eps; rows with a NaN or an infinity spoil themselves alone; tiny rows."""
    x = torch.randn(6, n, generator=gen(n), device="cuda")
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 6] = float("inf")
    x[4] *= 1e-15
    x = x.to(DENSE[t])
    w = torch.ones(n, device="cuda").to(DENSE[t])
    for eps in (1e-6, 0.0):
        hh, q, s, y, rstd = run_norm(x, None, w, t, eps)
        h64, rstd64, y64 = f8.rms_norm(x, None, w, eps)
        for row in (0, 4, 5):
            assert ((y[row].double() - y64[row]).abs() <= (HALF[t] + 2 * sum_error(n)) * y64[row].abs() + 1e-40).all()
            assert torch.isfinite(f8.decoded(q, s, "e4m3", 1)[row]).all()
        if eps:
            assert not y[1].any() and not q[1].any() and (s[1] == 127).all()
        else:
            assert torch.isnan(y[1]).all() and (s[1] == 127).all() and ((q[1] & 0x7F) == 0x7F).all()
        assert torch.isnan(y[2]).all() and ((q[2] & 0x7F) == 0x7F).all()
        assert torch.isnan(y[3, 6]) and ((q[3, 6] & 0x7F) == 0x7F)
        assert not y[3, :6].any()   # an infinite mean: 1 / sqrt(inf) = 0


# ---- gradient of the norm ----------------------------------------------------------------------------------------
def run_grad(dy, h, w, rstd, dh, t, beta=0.0, dw=None, pad=0, offset=0, dx=None, st=None, work=None):
    rows, n = h.shape
    flat = None
    if dx is None:
        dx, flat = padded(rows, n, DENSE[t], n + pad, offset)
    need = bofhip.rmsnorm_grad_workspace_bytes(rows, n) if dw is not None else 0
    work = torch.empty(need, dtype=torch.uint8, device="cuda") if work is None else work
    bofhip.rmsnorm_grad(rows, n, CODE[t], at(dy), dy.stride(0), at(h), h.stride(0), at(w), at(rstd), at(dh), 0 if dh is None else dh.stride(0),
                        at(dx), dx.stride(0), beta, at(dw), at(work), work.numel(), stream() if st is None else st)
    torch.cuda.synchronize()
    assert flat is None or outside_untouched(dx, flat)
    return dx


def check_grad(dy, h, w, rstd, dh, t, beta=0.0, **kw):
    rows, n = h.shape
    dw = torch.randn(n, generator=gen(n), device="cuda") if beta else torch.full((n,), float("nan"), device="cuda")
    dw0 = dw.double()
    dx64, dw64 = f8.rms_norm_grad(dy, h, w, rstd, dh)
    terms_w = (dy.double() * h.double() * rstd.double()[:, None]).abs().sum(0)
    g, xhat, rs = dy.double() * w.double(), h.double() * rstd.double()[:, None], rstd.double()[:, None]
    e = sum_error(n)
    spread = rs * (g.abs() + xhat.abs() * (g * xhat).abs().mean(1, keepdim=True)) + (dh.double().abs() if dh is not None else 0)
    dx = run_grad(dy, h, w, rstd, dh, t, beta, dw, **kw)
    tiny = torch.finfo(DENSE[t]).smallest_normal * HALF[t] * 2
    assert ((dx.double() - dx64).abs() <= HALF[t] * dx64.abs() + e * (1 + HALF[t]) * spread + tiny).all()
    want = dw64 + (beta * dw0 if beta else 0)
    assert ((dw.double() - want).abs() <= (rows + 8) * U * (terms_w + (abs(beta) * dw0.abs() if beta else 0))).all()
    return dx, dw


def grad_inputs(rows, n, t, dh=True, seed=0):
    g = gen(rows * 3 + n + seed)
    d = DENSE[t]
    h = torch.randn(rows, n, generator=g, device="cuda").to(d)
    dy = (0.1 * torch.randn(rows, n, generator=g, device="cuda")).to(d)
    w = (1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(d)
    e = (0.1 * torch.randn(rows, n, generator=g, device="cuda")).to(d) if dh else None
    return dy, h, w, (h.double().square().mean(1) + 1e-6).rsqrt().float(), e


@pytest.mark.parametrize("rows,n", [(1, 1), (1, 4096), (3, 127), (5, 129), (2, 640), (700, 130), (300, 1000), (260, 8192), (129, 5001), (3, 16384),
                                    (5, 33000), (1, 100001), (2000, 64)])
@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dh", [False, True])
def test_grad_sizes(dev, rows, n, t, dh):
    dy, h, w, rstd, e = grad_inputs(rows, n, t, dh)
    a = check_grad(dy, h, w, rstd, e, t)
    b = check_grad(dy, h, w, rstd, e, t)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])          # the same call, the same bits
    check_grad(dy, h, w, rstd, e, t, beta=-0.5)
    assert torch.equal(run_grad(dy, h, w, rstd, e, t), a[0])            # dw not wanted


@pytest.mark.parametrize("pad,offset", [(0, 1), (1, 0), (8, 8), (3, 5), (4, 4)])
@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("n", [520, 4096])
def test_grad_strides(dev, pad, offset, t, n):
    src = grad_inputs(9, n, t)
    dy, h, e = (padded(9, n, DENSE[t], n + pad, offset)[0] for _ in range(3))
    for dst, s in ((dy, src[0]), (h, src[1]), (e, src[4])):
        dst.copy_(s)
    check_grad(dy, h, src[2], src[3], e, t, pad=pad, offset=offset)


@pytest.mark.parametrize("n", [700, 4096, 40000])
@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("over", ["dy", "dh"])
def test_grad_in_place(dev, n, t, over):
    dy, h, w, rstd, e = grad_inputs(40, n, t)
    dw, dw2 = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    ref = run_grad(dy, h, w, rstd, e, t, dw=dw)
    dy2, e2 = dy.clone(), e.clone()
    got = run_grad(dy2, h, w, rstd, e2, t, dw=dw2, dx=dy2 if over == "dy" else e2)
    assert torch.equal(got, ref) and torch.equal(dw, dw2)


def test_grad_without_rows(dev):
    dw = torch.ones(10, device="cuda")
    bofhip.rmsnorm_grad(0, 10, bofhip.BF16, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0.5, at(dw), 0, 0, stream())
    assert torch.equal(dw, torch.full_like(dw, 0.5))


def test_grad_agrees_with_differences_of_the_norm(dev):
    """d/dx of sum(dy * Y) by central differences of the 64-bit norm, at the point the kernel was given."""
    dy, h, w, _, _ = grad_inputs(3, 200, "f32", False)
    eps, d = 1e-3, 1e-5
    rstd = f8.rms_norm(h, None, w, eps)[1].float()
    dw = torch.zeros(200, device="cuda")
    dx = run_grad(dy, h, w, rstd, None, "f32", dw=dw).double()
    loss = lambda h, w: (f8.rms_norm(h, None, w, eps)[2] * dy.double()).sum()  # noqa: E731
    for r, c in ((0, 0), (1, 17), (2, 199), (0, 100)):
        e = torch.zeros(3, 200, dtype=torch.float64, device="cuda")
        e[r, c] = d
        assert abs((loss(h.double() + e, w) - loss(h.double() - e, w)) / (2 * d) - dx[r, c]) < 1e-5
        f = torch.zeros(200, dtype=torch.float64, device="cuda")
        f[c] = d
        assert abs((loss(h, w.double() + f) - loss(h, w.double() - f)) / (2 * d) - dw[c]) < 1e-5


# ---- together ----------------------------------------------------------------------------------------------------
class Layer:
    """One linear layer behind a norm, forward and backward, as a program uses the operators: buffers made once, a step
    is a handful of calls on one stream."""

    def __init__(self, tokens, n, out, seed=0):
        g = gen(seed)
        e = lambda *s, d=torch.uint8: torch.empty(*s, dtype=d, device="cuda")  # noqa: E731
        nb = lambda c: -(-c // 128)  # noqa: E731
        self.t, self.n, self.o = tokens, n, out
        self.x, self.r = (torch.randn(tokens, n, generator=g, device="cuda").bfloat16() for _ in range(2))
        self.gamma = (1 + 0.1 * torch.randn(n, generator=g, device="cuda")).bfloat16()
        self.W = torch.randn(out, n, generator=g, device="cuda") * 0.05
        self.dz = (torch.randn(tokens, out, generator=g, device="cuda") * 0.01).bfloat16()
        self.dh = (torch.randn(tokens, n, generator=g, device="cuda") * 0.01).bfloat16()
        self.h, self.y, self.dy, self.dx = (e(tokens, n, d=torch.bfloat16) for _ in range(4))
        self.z, self.rstd = e(tokens, out, d=torch.bfloat16), e(tokens, d=torch.float32)
        self.yq, self.ys = e(tokens, n), e(tokens, nb(n))
        self.yqt, self.yst = e(n, tokens), e(n, nb(tokens))
        self.wq, self.ws, self.wqt, self.wst = e(out, n), e(nb(out), nb(n)), e(n, out), e(nb(n), nb(out))
        self.zq, self.zs, self.zqt, self.zst = e(tokens, out), e(tokens, nb(out)), e(out, tokens), e(out, nb(tokens))
        self.dW, self.dgamma = torch.zeros(out, n, device="cuda"), torch.zeros(n, device="cuda")
        size = [bofhip.f8_gemm_workspace_bytes(*s) for s in ((tokens, out, n), (tokens, n, out), (out, n, tokens))]
        self.work = e(max(size + [bofhip.rmsnorm_grad_workspace_bytes(tokens, n), 16]))

    def step(self):
        t, n, o, st, L = self.t, self.n, self.o, stream(), bofhip
        nb, w, wb = lambda c: -(-c // 128), at(self.work), self.work.numel()  # noqa: E731
        L.f8_quant(o, n, at(self.W), n, L.F32, L.E4M3, 128, at(self.wq), n, at(self.ws), nb(n), at(self.wqt), o, at(self.wst), nb(o), st)
        L.rmsnorm_f8(t, n, L.BF16, at(self.x), n, at(self.r), n, at(self.gamma), 1e-6, at(self.h), n, L.E4M3, at(self.yq), n, at(self.ys), nb(n),
                     at(self.y), n, at(self.rstd), st)
        L.f8_gemm(t, o, n, 1.0, at(self.yq), n, L.E4M3, at(self.ys), nb(n), 1, at(self.wq), n, L.E4M3, at(self.ws), nb(n), 128, 0.0, at(self.z), o,
                  L.BF16, w, wb, st)
        L.f8_quant(t, o, at(self.dz), o, L.BF16, L.E5M2, 1, at(self.zq), o, at(self.zs), nb(o), at(self.zqt), t, at(self.zst), nb(t), st)
        L.f8_quant(t, n, at(self.y), n, L.BF16, L.E4M3, 1, 0, 0, 0, 0, at(self.yqt), t, at(self.yst), nb(t), st)
        L.f8_gemm(t, n, o, 1.0, at(self.zq), o, L.E5M2, at(self.zs), nb(o), 1, at(self.wqt), o, L.E4M3, at(self.wst), nb(o), 128, 0.0, at(self.dy),
                  n, L.BF16, w, wb, st)
        L.f8_gemm(o, n, t, 1.0, at(self.zqt), t, L.E5M2, at(self.zst), nb(t), 1, at(self.yqt), t, L.E4M3, at(self.yst), nb(t), 1, 1.0, at(self.dW),
                  n, L.F32, w, wb, st)
        L.rmsnorm_grad(t, n, L.BF16, at(self.dy), n, at(self.h), n, at(self.gamma), at(self.rstd), at(self.dh), n, at(self.dx), n, 1.0,
                       at(self.dgamma), w, wb, st)

    def outputs(self):
        return [self.h, self.z, self.dx, self.dW, self.dgamma]


@pytest.mark.parametrize("tokens,n,out", [(1, 256, 384), (37, 640, 300), (300, 512, 1000)])
def test_a_layer_forward_and_backward(dev, tokens, n, out):
    """Every product against 64 bits on the very operands it was given, and the whole against the layer in 64 bits
    without 8-bit roundings, whose relative distance is what the operands' roundings can amount to."""
    L = Layer(tokens, n, out, seed=tokens)
    L.step()
    torch.cuda.synchronize()
    W, Wt = f8.decoded(L.wq, L.ws, "e4m3", 128), f8.decoded(L.wqt, L.wst, "e4m3", 128)
    assert torch.equal(W, Wt.t())                                        # one block, one scale, both layouts
    yq, yqt = f8.decoded(L.yq, L.ys, "e4m3", 1), f8.decoded(L.yqt, L.yst, "e4m3", 1)
    zq, zqt = f8.decoded(L.zq, L.zs, "e5m2", 1), f8.decoded(L.zqt, L.zst, "e5m2", 1)
    for got, a, b, t in ((L.z, yq, W, "bf16"), (L.dy, zq, Wt, "bf16"), (L.dW, zqt, yqt, "f32")):
        want = a @ b.t()
        assert ((got.double() - want).abs() <= f8.product_bound(a, b, t, 1.0, 0.0, None, want)).all()
    h, rstd, y = f8.rms_norm(L.x, L.r, L.gamma, 1e-6)
    dy = L.dz.double() @ L.W.double()
    dx, dgamma = f8.rms_norm_grad(dy, h, L.gamma, rstd, L.dh)
    rel = lambda got, want: ((got.double() - want).norm() / want.norm()).item()  # noqa: E731
    assert rel(L.h, h) <= HALF["bf16"]
    # two operands, each off by at most half a step of its type (plus what its subnormals lose: below a step's tenth)
    for got, want, halves in ((L.z, y @ L.W.double().t(), ("e4m3", "e4m3")), (L.dW, L.dz.double().t() @ y, ("e5m2", "e4m3")),
                              (L.dx, dx, ("e5m2", "e4m3")), (L.dgamma, dgamma, ("e5m2", "e4m3"))):
        assert rel(got, want) <= 1.1 * sum(HALF[t] for t in halves)


def test_a_captured_step_replays(dev):
    """The step captured into a graph and replayed, with eager work and new inputs in between: every replay has the bits
    of the eager step on the same inputs; a second graph with its own buffers, on its own stream, beside it."""
    L, E = Layer(130, 512, 384, seed=1), Layer(130, 512, 384, seed=1)
    other = Layer(40, 640, 256, seed=2)
    E.step()
    torch.cuda.synchronize()
    graphs = []
    for layer in (L, other):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            layer.step()
            s.synchronize()
            layer.dW.zero_()
            layer.dgamma.zero_()
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                layer.dW.zero_()
                layer.dgamma.zero_()
                layer.step()
        graphs.append((g, s))
    for rep in range(4):
        x = torch.randn(130, 512, generator=gen(50 + rep), device="cuda").bfloat16()
        for layer in (L, E):
            layer.x.copy_(x)
        E.dW.zero_()
        E.dgamma.zero_()
        E.step()
        torch.cuda.synchronize()
        for g, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(L.outputs(), E.outputs()):
            assert torch.equal(a, b), rep
    ref = Layer(40, 640, 256, seed=2)
    ref.step()
    torch.cuda.synchronize()
    for a, b in zip(other.outputs(), ref.outputs()):
        assert torch.equal(a, b)


def enough_memory(gib):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of device memory")


def test_norm_of_more_rows_than_a_grid_dimension_holds(dev):
    """2^22 rows of a workgroup of 1024 threads each are 2^32 threads."""
    enough_memory(70)
    rows, n = (1 << 22) + 5, 8200
    x = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    x[:2], x[-7:] = 0.5, 2.0
    w = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    rstd = torch.full((rows + 3,), 7.0, device="cuda")
    bofhip.rmsnorm_f8(rows, n, bofhip.BF16, at(x), n, 0, 0, at(w), 0.0, 0, 0, bofhip.E4M3, 0, 0, 0, 0, rstd=at(rstd), stream=stream())
    torch.cuda.synchronize()
    assert rstd[:2].tolist() == [2.0, 2.0] and rstd[rows - 7:].tolist() == [0.5] * 7 + [7.0] * 3


def test_gradient_of_a_row_longer_than_a_grid_dimension_holds(dev):
    """2^29 columns are 2^32 threads of the join."""
    enough_memory(12)
    n = (1 << 29) + 40
    h = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    dy, dx, rstd = torch.zeros_like(h), torch.empty_like(h), torch.full((1,), 0.5, device="cuda")
    places = torch.tensor([0, 31, 5000, (1 << 29) - 1, 1 << 29, n - 1], device="cuda")
    dy[places] = torch.arange(1, 7, device="cuda").bfloat16()
    dw = torch.full((n + 8,), 9.0, device="cuda")
    work = torch.empty(bofhip.rmsnorm_grad_workspace_bytes(1, n), dtype=torch.uint8, device="cuda")
    bofhip.rmsnorm_grad(1, n, bofhip.BF16, at(dy), n, at(h), n, at(h), at(rstd), 0, 0, at(dx), n, 0.0, at(dw), at(work), work.numel(), stream())
    torch.cuda.synchronize()
    assert torch.equal(dw[places], torch.arange(1, 7, device="cuda") * 0.5)
    assert dw[:n].count_nonzero() == 6 and torch.equal(dw[n:], torch.full((8,), 9.0, device="cuda"))


def test_two_streams_at_once(dev):
    """Two layers stepping on two streams, without waiting for one another, each with its own workspace."""
    layers = [Layer(64, 512, 512, seed=s) for s in (1, 2)]
    refs = [Layer(64, 512, 512, seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in layers]
    for r in refs:
        for _ in range(5):
            r.step()
        torch.cuda.synchronize()
    for _ in range(5):
        for layer, s in zip(layers, streams):
            with torch.cuda.stream(s):
                layer.step()
    torch.cuda.synchronize()
    for layer, r in zip(layers, refs):
        for a, b in zip(layer.outputs(), r.outputs()):
            assert torch.equal(a, b)


def test_memory_the_device_cannot_reach_is_refused(dev):
    x = torch.zeros(64, dtype=torch.float32)     # pageable host memory
    d = torch.zeros(64, dtype=torch.float32, device="cuda")
    with pytest.raises(bofhip.BofError, match="X is not memory"):
        bofhip.f8_quant(1, 16, at(x), 16, bofhip.F32, bofhip.E4M3, 1, at(d), 16, at(d) + 64, 1, stream=stream())
    with pytest.raises(bofhip.BofError, match="q is not memory"):
        bofhip.f8_quant(1, 16, at(d), 16, bofhip.F32, bofhip.E4M3, 1, at(x), 16, at(d) + 64, 1, stream=stream())
    with pytest.raises(bofhip.BofError, match="work is not memory"):
        bofhip.rmsnorm_grad(1, 4, bofhip.F32, at(d), 4, at(d) + 16, 4, at(d) + 32, at(d) + 48, 0, 0, at(d) + 64, 4, 0.0, at(d) + 80,
                            x.data_ptr() // 16 * 16 + 16, 16, stream())
    p = torch.arange(16, dtype=torch.float32, pin_memory=True)   # host memory that the device maps
    q = torch.zeros(16, dtype=torch.uint8, device="cuda")
    s = torch.zeros(1, dtype=torch.uint8, device="cuda")
    bofhip.f8_quant(1, 16, at(p), 16, bofhip.F32, bofhip.E4M3, 1, at(q), 16, at(s), 1, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(f8.decoded(q[None], s[None], "e4m3", 1).cpu()[0], torch.arange(16).double())
