"""Products whose every partial sum fp32 holds exactly, in whatever order it is made: bof_f8_gemm (include/bof_f8.h) has to return the exact
value, rounded once to C's type.  A bound on rounding errors grows with k faster than a random result does, so that beyond some
hundred k it would let a dropped chunk or cut products pass; equality does not.

Elements are -1, 0, 1 and scales 2^-1, 1, 2 on either side.  For a 32-bit C, in up to 24 places along k, both operands also hold +-128: a
product of 2^14 beside products of 1, of which the f8 instructions would leave nothing (they cut at 2^-13 of the largest of eight).
All terms are multiples of 2^-2, and the sum of their magnitudes stays below 2^22: k * 4 + 24 * 2^16 <= 1.65e6 for k <= 17000."""
import pytest
import torch

import bofhip
import f8_shapes
import f8_util as f8

TYPES = [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")]


def operand(rows, k, f8t, group, places, ld, seed, dev):
    """(bytes, codes, values in 64 bits); bytes between the rows are NaN"""
    g = torch.Generator(device=dev).manual_seed(seed)
    v = torch.randint(-1, 2, (rows, k), generator=g, device=dev).float()
    v[:, places] = 128.0 * (1 - 2 * torch.randint(0, 2, (rows, len(places)), generator=g, device=dev).float())
    q = torch.full((rows, ld), 0x7F, dtype=torch.uint8, device=dev)
    q[:, :k] = v.to(f8.F8[f8t]).view(torch.uint8)
    codes = torch.randint(126, 129, (-(-rows // group), -(-k // 128)), generator=g, device=dev)
    return q, codes.to(torch.uint8), v.double() * f8.spread(codes, group, rows, k)


def places_of(k, bits):
    """columns of the large elements: the first and the last, and some between, neighbours of small ones"""
    return sorted({0, k - 1, *(k * i // 22 for i in range(22))}) if bits == 32 and k > 100 else []


def cut_product(a, b):
    """What an instruction that adds eight neighbouring products, cut at 2^-13 of the largest, makes of two rows (64 bits)."""
    p = torch.nn.functional.pad(a * b, (0, -len(a) % 8)).reshape(-1, 8)
    step = torch.exp2(torch.floor(torch.log2(p.abs().amax(1, keepdim=True).clamp(min=1e-30))) - 13)
    return (torch.trunc(p / step) * step).sum()


@pytest.mark.parametrize("k", [129, 4096, 16384])
def test_cut_products_and_dropped_chunks_show(k):
    places = places_of(k, 32)
    assert len(places) <= 24
    _, _, a = operand(3, k, "e4m3", 1, places, k, 1, "cpu")
    _, _, b = operand(4, k, "e5m2", 128, places, k, 2, "cpu")
    assert (a.abs() @ b.abs().t()).max() < 2 ** 22 and ((a @ b.t()) * 4 % 1 == 0).all()
    want = a @ b.t()
    # (what is lost of one element may come to nothing by chance -- a few terms of either sign --, of most it does not)
    assert sum(bool(cut_product(a[i], b[j]) != want[i, j]) for i in range(3) for j in range(4)) >= 6
    assert ((a[:, :k - 16] @ b[:, :k - 16].t()) != want).sum() >= 6


def test_small_products_are_not_cut():
    _, _, a = operand(3, 1000, "e4m3", 1, [], 1000, 1, "cpu")
    _, _, b = operand(4, 1000, "e5m2", 128, [], 1000, 2, "cpu")
    assert all(cut_product(a[i], b[j]) == (a @ b.t())[i, j] for i in range(3) for j in range(4))


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,bits,aligned,m,n,k,parts,number", f8_shapes.each())
def test_product_is_exact(dev, kernel, bits, aligned, m, n, k, parts, number):
    (ta, tb), ld, places = TYPES[(number + number // 4) % 4], f8_shapes.row_bytes(k, aligned), places_of(k, bits)
    ga, gb = 1 if number & 1 else 128, 128 if number & 2 else 1
    qa, sa, a = operand(m, k, ta, ga, places, ld, m, dev)
    qb, sb, b = operand(n, k, tb, gb, places, ld, n + 1, dev)
    dtype, code = (torch.float32, bofhip.F32) if bits == 32 else (torch.float16, bofhip.F16) if number & 1 else (torch.bfloat16, bofhip.BF16)
    c0 = torch.randint(-8, 9, (m, n), generator=torch.Generator(device=dev).manual_seed(k), device=dev)
    c = c0.to(dtype)
    work = torch.empty(bofhip.f8_gemm_workspace_bytes(m, n, k) + 16, dtype=torch.uint8, device=dev)
    bofhip.f8_gemm(m, n, k, 1.0, qa.data_ptr(), ld, bofhip.E4M3 if ta == "e4m3" else bofhip.E5M2, sa.data_ptr(), sa.stride(0), ga, qb.data_ptr(),
                   ld, bofhip.E4M3 if tb == "e4m3" else bofhip.E5M2, sb.data_ptr(), sb.stride(0), gb, 1.0, c.data_ptr(), n, code, work.data_ptr(),
                   work.numel(), torch.cuda.current_stream().cuda_stream)
    want = (a @ b.t() + c0).to(dtype)
    wrong = c != want
    assert not wrong.any(), f"{int(wrong.sum())} of {wrong.numel()}, the first at {wrong.nonzero()[0].tolist()}: {c[wrong][0]} for {want[wrong][0]}"
