"""CPU tests of the 8-bit operators' host side (include/bof_f8.h): every declared symbol is exported and bound, wrong
arguments are refused before a device is looked for, empty results need none, and the tests' own 64-bit forms agree
with a gradient taken by differences."""
import os
import re

import pytest
import torch

import bofhip
import f8_util as f8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_declared_symbol_is_exported_and_bound():
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "bof_f8.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(bof_[a-z0-9_]+)\s*\(", src)))
    assert sorted(s[0] for s in bofhip.SYMBOLS_F8) == names
    for n in names:
        assert hasattr(bofhip.lib(), n)


# host addresses that the checks below never follow
AT = 1 << 20


def gemm(**kw):
    a = dict(m=8, n=8, k=300, alpha=1.0, a=AT, lda=300, a_type=bofhip.E4M3, sa=AT, ldsa=3, ga=1, b=AT, ldb=300, b_type=bofhip.E4M3, sb=AT,
             ldsb=3, gb=128, beta=0.0, c=AT, ldc=8, c_type=bofhip.BF16, work=0, work_bytes=0)
    a.update(kw)
    bofhip.f8_gemm(**a)


def quant(**kw):
    a = dict(rows=200, cols=300, x=AT, ldx=300, x_type=bofhip.BF16, f8_type=bofhip.E4M3, group=1, q=AT, ldq=300, s=AT, lds=3, qt=AT, ldqt=200,
             st=AT, ldst=2)
    a.update(kw)
    bofhip.f8_quant(**a)


def norm(**kw):
    a = dict(rows=4, n=300, type_=bofhip.BF16, x=AT, ldx=300, r=2 * AT, ldr=300, w=AT, eps=1e-6, h=3 * AT, ldh=300, f8_type=bofhip.E4M3, q=AT,
             ldq=300, s=AT, lds=3, y=AT, ldy=300, rstd=AT)
    a.update(kw)
    bofhip.rmsnorm_f8(**a)


def grad(**kw):
    a = dict(rows=4, n=300, type_=bofhip.BF16, dy=AT, lddy=300, h=2 * AT, ldh=300, w=AT, rstd=AT, dh=3 * AT, lddh=300, dx=4 * AT, lddx=300,
             beta=0.0, dw=AT, work=AT, work_bytes=1 << 20)
    a.update(kw)
    bofhip.rmsnorm_grad(**a)


@pytest.mark.parametrize("call,wrong", [
    (gemm, dict(m=-1)), (gemm, dict(n=2 ** 31)), (gemm, dict(k=-5)), (gemm, dict(a_type=bofhip.BF16)), (gemm, dict(b_type=7)),
    (gemm, dict(c_type=bofhip.E4M3)), (gemm, dict(ga=64)), (gemm, dict(gb=0)), (gemm, dict(lda=299)), (gemm, dict(ldb=0)),
    (gemm, dict(ldsa=2)), (gemm, dict(ldsb=2)), (gemm, dict(ldc=7)), (gemm, dict(a=0)), (gemm, dict(b=0)), (gemm, dict(sa=0)),
    (gemm, dict(sb=0)), (gemm, dict(c=0)), (gemm, dict(c=AT + 1)), (gemm, dict(c=AT + 2, c_type=bofhip.F32)),
    (gemm, dict(work=AT + 4, work_bytes=1 << 20)),
    (quant, dict(rows=-1)), (quant, dict(cols=2 ** 31)), (quant, dict(x_type=bofhip.E4M3)), (quant, dict(f8_type=bofhip.F16)),
    (quant, dict(group=2)), (quant, dict(q=0)), (quant, dict(s=0)), (quant, dict(qt=0)), (quant, dict(st=0)),
    (quant, dict(q=0, s=0, qt=0, st=0)), (quant, dict(x=0)), (quant, dict(ldx=299)), (quant, dict(x=AT + 1)), (quant, dict(ldq=299)),
    (quant, dict(lds=2)), (quant, dict(ldqt=199)), (quant, dict(ldst=1)),
    (norm, dict(rows=-1)), (norm, dict(n=-1)), (norm, dict(rows=1 << 24)), (norm, dict(type_=bofhip.E5M2)), (norm, dict(f8_type=bofhip.F32)),
    (norm, dict(q=0)), (norm, dict(s=0)), (norm, dict(q=0, s=0, y=0, h=0, rstd=0)), (norm, dict(x=0)), (norm, dict(w=0)),
    (norm, dict(ldx=299)), (norm, dict(ldr=299)), (norm, dict(ldh=299)), (norm, dict(ldq=299)), (norm, dict(lds=2)), (norm, dict(ldy=299)),
    (norm, dict(x=AT + 1)), (norm, dict(rstd=AT + 2)), (norm, dict(eps=-1.0)), (norm, dict(eps=float("nan"))), (norm, dict(h=AT, ldh=304)),
    (norm, dict(h=2 * AT, ldr=304)),
    (grad, dict(rows=-1)), (grad, dict(n=-1)), (grad, dict(rows=1 << 24)), (grad, dict(type_=5)), (grad, dict(dy=0)), (grad, dict(h=0)),
    (grad, dict(w=0)), (grad, dict(rstd=0)), (grad, dict(dx=0)), (grad, dict(lddy=299)), (grad, dict(ldh=299)), (grad, dict(lddh=299)),
    (grad, dict(lddx=299)), (grad, dict(dx=AT + 1)), (grad, dict(dw=AT + 2)), (grad, dict(work=0)), (grad, dict(work=AT + 4)),
    (grad, dict(work_bytes=100)), (grad, dict(dx=AT, lddx=304)), (grad, dict(dx=3 * AT, lddx=304)), (grad, dict(dx=2 * AT)),
])
def test_wrong_arguments_are_refused(call, wrong):
    with pytest.raises(bofhip.BofError, match="rc=-1"):
        call(**wrong)


def test_empty_results_need_no_device():
    gemm(m=0)
    gemm(n=0)
    quant(rows=0)
    quant(cols=0, ldx=0)
    norm(rows=0)
    norm(n=0)
    grad(n=0)
    grad(rows=0, dw=0)
    grad(rows=0, beta=1.0)
    gemm(m=0, k=0, a=0, b=0, sa=0, sb=0, c=0)


@pytest.mark.skipif(torch.cuda.is_available(), reason="what a box without a GPU does")
@pytest.mark.parametrize("call", [gemm, quant, norm, grad])
def test_without_a_device_the_calls_fail(call):
    with pytest.raises(bofhip.BofError, match="rc=-4"):
        call()


def test_workspace_sizes():
    assert bofhip.f8_gemm_workspace_bytes(0, 5, 5) == 0 and bofhip.f8_gemm_workspace_bytes(-1, 5, 5) == 0
    assert bofhip.f8_gemm_workspace_bytes(8192, 8192, 8192) == 0        # tiles enough: not split
    small = bofhip.f8_gemm_workspace_bytes(128, 128, 16384)
    assert small > 0 and small % (4 * 128 * 128) == 0
    assert bofhip.rmsnorm_grad_workspace_bytes(0, 5) == 0
    assert bofhip.rmsnorm_grad_workspace_bytes(3, 100) >= 400


@pytest.mark.parametrize("f8t", ["e4m3", "e5m2"])
def test_the_plain_quantiser_keeps_what_it_can(f8t):
    """The tests' own reference: the scale is the smallest that fits, and an element is off by half a step at most."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(130, 300, generator=g).double() * torch.exp2(torch.randint(-30, 30, (130, 1), generator=g).double())
    for group in (1, 128):
        q, codes = f8.quantised(x, f8t, group)
        s = f8.spread(codes, group, *x.shape)
        top = f8.spread(f8.block_codes(x, f8t, group), group, *x.shape) * f8.LARGEST[f8t]
        assert (x.abs() <= top).all()
        back = f8.decoded(q, codes, f8t, group)
        assert ((back - x).abs() <= torch.maximum(f8.HALF[f8t] * x.abs(), s * f8.SMALLEST[f8t] / 2)).all()
    for v, want in ((448.0, 127), (448.0001, 128), (224.0, 126), (0.0, 127), (1e-45, 1), (float("nan"), 127), (float("inf"), 127)):
        assert f8.block_codes(torch.tensor([[v]], dtype=torch.float32).double(), "e4m3", 1).item() == want, v


def test_the_plain_gradient_agrees_with_differences():
    g = torch.Generator().manual_seed(5)
    x, dy, w = (torch.randn(3, 40, generator=g).double() for _ in range(2)), None, torch.randn(40, generator=g).double()
    x, dy = x
    eps, d = 1e-3, 1e-6
    h, rstd, _ = f8.rms_norm(x, None, w, eps)
    dx, dw = f8.rms_norm_grad(dy, h, w, rstd, None)
    loss = lambda x, w: (f8.rms_norm(x, None, w, eps)[2] * dy).sum()  # noqa: E731
    for r in range(3):
        for c in range(40):
            e = torch.zeros_like(x)
            e[r, c] = d
            assert abs((loss(x + e, w) - loss(x - e, w)) / (2 * d) - dx[r, c]) < 1e-7
    for c in range(40):
        e = torch.zeros_like(w)
        e[c] = d
        assert abs((loss(x, w + e) - loss(x, w - e)) / (2 * d) - dw[c]) < 1e-7
