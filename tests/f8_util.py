"""Plain 64-bit forms of the operators of include/bof_f8.h, for the tests (CPU or GPU tensors alike)."""
import torch

import bofhip

DENSE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
CODE = {"f32": bofhip.F32, "bf16": bofhip.BF16, "f16": bofhip.F16, "e4m3": bofhip.E4M3, "e5m2": bofhip.E5M2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11, "e4m3": 2.0 ** -4, "e5m2": 2.0 ** -3}  # half a step: finfo(t).eps / 2
SMALLEST = {"e4m3": 2.0 ** -9, "e5m2": 2.0 ** -16}  # step of the subnormals
U = 2.0 ** -23                                      # one operation in fp32, rounded or cut


def exp2(e):
    return torch.exp2(e.double())


def block_codes(x, f8, group):
    """E8M0 codes (int64) of the group x 128 blocks of x (float64): the smallest power of two >= 2^-126 that brings the
    largest finite magnitude into the type's range; 127 for a block without any."""
    rows, cols = x.shape
    gr, gc = -(-rows // group), -(-cols // 128)
    a = torch.zeros(gr * group, gc * 128, dtype=torch.float64, device=x.device)
    a[:rows, :cols] = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    top = a.reshape(gr, group, gc, 128).amax((1, 3))
    f, e = torch.frexp(top / LARGEST[f8])           # the division by 7 * 2^j is the only rounding: settled below
    e = e.double()
    e = torch.where(exp2(e - 1) * LARGEST[f8] >= top, e - 1, e)
    e = torch.where(exp2(e) * LARGEST[f8] < top, e + 1, e)
    e = torch.where(top > 0, e.clamp(min=-126), torch.zeros_like(e))
    return (e + 127).long()


def spread(codes, group, rows, cols):
    """2^(code - 127) of every element; code 255: NaN."""
    s = torch.where(codes == 255, torch.full_like(codes, 0, dtype=torch.float64) * float("nan"), exp2(codes.double() - 127))
    return s.repeat_interleave(group, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def quantised(x, f8, group):
    """(bytes, codes) of x (float64 holding float32 values): x / scale is exact, then one rounding."""
    codes = block_codes(x, f8, group)
    v = x / spread(codes, group, *x.shape)
    return v.float().to(F8[f8]).view(torch.uint8), codes


def decoded(q, codes, f8, group):
    return q.contiguous().view(F8[f8]).double() * spread(codes.long(), group, *q.shape)


def rms_norm(x, r, w, eps):
    h = x.double() + r.double() if r is not None else x.double()
    rstd = (h.square().mean(1) + eps).rsqrt()
    return h, rstd, h * rstd[:, None] * w.double()


def rms_norm_grad(dy, h, w, rstd, dh):
    dy, h, w, rstd = dy.double(), h.double(), w.double(), rstd.double()[:, None]
    g, xhat = dy * w, h * rstd
    dx = rstd * (g - xhat * (g * xhat).mean(1, keepdim=True))
    return (dx + dh.double() if dh is not None else dx), (dy * xhat).sum(0)


def group8(x):
    """Largest magnitude of every eight neighbours along a row."""
    rows, cols = x.shape
    a = torch.zeros(rows, -(-cols // 8) * 8, dtype=torch.float64, device=x.device)
    a[:, :cols] = x.abs()
    return a.reshape(rows, -1, 8).amax(2)


def product_bound(a, b, c_type, alpha, beta, c0, want):
    """Largest error of bof_f8_gemm for the decoded operands a, b.  fp32 sums of k terms in any order: k operations, two
    more for alpha and beta.  A 16-bit C: every product of a group of eight is cut at 2^-13 of the largest, which is at
    most the product of the group's largest factors: 8 * 2^-13 of that, and its own rounding (half a step, or half the
    smallest step where C is subnormal)."""
    k = a.shape[1]
    terms = a.abs() @ b.abs().t()
    bound = (k + 4) * U * terms
    if c_type != "f32":
        bound = bound + 2.0 ** -10 * (group8(a) @ group8(b).t())
    bound = abs(alpha) * bound + 4 * U * (abs(alpha) * terms + (abs(beta) * c0.abs() if beta else 0))
    return bound * (1 + 2 * HALF[c_type]) + HALF[c_type] * want.abs() + {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -25}[c_type]
