"""Cases and plain forms of the 8-bit floating-point operators of libbof_hip.so.

The operators are the parts of a linear layer of a language model whose products run in 8-bit floating point: the
product itself (bofhip.f8_gemm), the quantiser that makes its operands (f8_quant), and the root-mean-square norm
that feeds it (rmsnorm_f8) with its backward pass (rmsnorm_grad).

A matrix in 8 bits is `q` (float8_e4m3fn or float8_e5m2, row-major, rows along the contracted dimension) with one
scale for each block of 128 along a row, shared by `group` rows (1: activations and gradients, 128: weights).  A scale
is a power of two (float8_e8m0fnu): the smallest one that brings the block's largest magnitude into the type's range.
The value of an element is q * s.
"""
import math
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DENSE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
TOP = {"e4m3": 9, "e5m2": 16}  # the largest value of either type is 0.875 * 2^TOP
SCRATCH = 64 << 20  # bytes of workspace that a program keeps for its products and its norm gradients
EPS = 1e-6


# ---- cases ---------------------------------------------------------------------------------------------------------
def _product(name, m, n, k, a="e4m3", b="e4m3", ga=1, gb=128, out="bf16", beta=0.0, tight=False):
    return {"name": name, "kind": "product", "m": m, "n": n, "k": k, "a": a, "b": b, "ga": ga, "gb": gb, "out": out, "beta": beta, "tight": tight}


def _quant(name, rows, cols, x="bf16", f8="e4m3", group=1, both=False, tight=False):
    return {"name": name, "kind": "quant", "rows": rows, "cols": cols, "x": x, "f8": f8, "group": group, "both": both, "tight": tight}


def _norm(name, rows, n, x="bf16", res=True, train=False, tight=False):
    return {"name": name, "kind": "norm", "rows": rows, "n": n, "x": x, "res": res, "train": train, "tight": tight}


def _grad(name, rows, n, x="bf16", dres=True):
    return {"name": name, "kind": "norm grad", "rows": rows, "n": n, "x": x, "dres": dres}


def listed():
    return [
        _product("product, one token", 1, 4096, 4096),  # serving: the next token of one request, bound by the weights' bytes
        _product("product, few tokens", 48, 8192, 4096),  # serving: one new token for each of a batch of requests
        _product("product, ragged", 1021, 5000, 4100, out="f16", tight=True),  # a prompt of odd length, rows without padding
        _product("product, large", 8192, 8192, 8192),  # training forward or a batch of long prompts
        _product("input gradient", 4096, 4096, 8192, a="e5m2"),  # training: the output's gradient times the weights
        _product("weight gradient", 4096, 2048, 16384, a="e5m2", gb=1, out="f32", beta=1.0),  # summed over 16384 tokens, added to what is there
        _quant("quantise weights", 4096, 4096, x="f32", group=128, both=True),  # after an optimiser step: both layouts of the master weights
        _quant("quantise activations", 16384, 4096, both=True),  # for the forward product and, transposed, the weight gradient
        _norm("norm, one token", 1, 4096),  # serving: a layer's input for one new token
        _norm("norm, long batch", 8192, 8192, train=True),  # training forward: keeps what the backward pass reads
        _grad("norm gradient", 8192, 8192),  # its backward pass, with the gradient of the residual path
        _grad("norm gradient, odd", 129, 5001, x="f32", dres=False),  # a short batch of odd width
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm; every third one a multiple of 128 where there is room."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, v // 128 * 128) if v >= 256 and rng.random() < 0.34 else v


def draw(rng):
    kind = rng.choice(["product"] * 5 + ["quant"] * 2 + ["norm"] * 2 + ["norm grad"] * 2)
    if kind == "product":
        use = rng.choice(["forward", "forward", "serving", "input gradient", "weight gradient"])
        while True:
            m, n, k = _spread(rng, 1, 64 if use == "serving" else 16384), _spread(rng, 64, 16384), _spread(rng, 64, 16384)
            if m * n * k <= 8192 ** 3:
                break
        c = _product("", m, n, k, out=rng.choice(["bf16", "bf16", "f16", "f32"]), tight=rng.random() < 0.25)
        if use.endswith("gradient"):
            c["a"] = rng.choice(["e4m3", "e5m2"])
        if use == "weight gradient":
            c.update(gb=1, out="f32", beta=rng.choice([0.0, 1.0]))
    elif kind == "quant":
        while True:
            rows, cols = _spread(rng, 1, 32768), _spread(rng, 64, 16384)
            if rows * cols <= 16384 * 4096:
                break
        c = _quant("", rows, cols, x=rng.choice(["bf16", "f16", "f32"]), f8=rng.choice(["e4m3", "e4m3", "e5m2"]), group=rng.choice([1, 1, 128]),
                   both=rng.random() < 0.5, tight=rng.random() < 0.25)
    else:
        while True:
            rows, n = _spread(rng, 1, 16384), _spread(rng, 64, 16384)
            if rows * n <= 8192 * 8192:
                break
        x = rng.choice(["bf16", "bf16", "f16", "f32"])
        c = _norm("", rows, n, x=x, res=rng.random() < 0.7, train=rng.random() < 0.5, tight=rng.random() < 0.25) if kind == "norm" else \
            _grad("", rows, n, x=x, dres=rng.random() < 0.7)
    del c["name"]
    return c


# ---- inputs --------------------------------------------------------------------------------------------------------
def _up(x, to):
    return -(-x // to) * to


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _rows(rows, cols, dtype, tight):
    """A matrix whose rows begin at multiples of 16 elements, or one without padding."""
    return torch.empty(rows, cols if tight else _up(cols, 16), dtype=dtype, device=DEV)[:, :cols]


def _values(g, rows, cols, size):
    """Normal values, with some channels 16 times as large, as activations and gradients have them."""
    x = torch.randn(rows, cols, generator=g, device=DEV) * size
    loud = torch.rand(cols, generator=g, device=DEV) < 0.005
    return x * (1 + 15 * loud.float())


def _operand(g, rows, cols, f8, group, tight, size):
    """A matrix in 8 bits, as a program holds it."""
    q8, s8 = _quantised(_values(g, rows, cols, size), f8, group)
    q = _rows(rows, cols, torch.uint8, tight)
    q.copy_(q8.view(torch.uint8))
    return {"q": q.view(F8[f8]), "s": s8.contiguous()}


def prepare(case, seed):
    g, c = _gen(seed), dict(case)
    st = {"case": c, "work": torch.empty(SCRATCH, dtype=torch.uint8, device=DEV)}
    if c["kind"] == "product":
        m, n, k, tight = c["m"], c["n"], c["k"], c["tight"]
        st["a"] = _operand(g, m, k, c["a"], c["ga"], tight, 1.0 if c["a"] == "e4m3" else 1e-3)
        st["b"] = _operand(g, n, k, c["b"], c["gb"], tight, 0.02 if c["gb"] == 128 else 1.0)
        st["c"] = torch.randn(m, n, generator=g, device=DEV).to(DENSE[c["out"]])
    elif c["kind"] == "quant":
        rows, cols, group, tight = c["rows"], c["cols"], c["group"], c["tight"]
        x = _rows(rows, cols, DENSE[c["x"]], tight)
        x.copy_(_values(g, rows, cols, 0.02 if group == 128 else 1.0))
        st["x"] = x
        st["q"] = _rows(rows, cols, F8[c["f8"]], tight)
        st["s"] = torch.empty(-(-rows // group), -(-cols // 128), dtype=torch.float8_e8m0fnu, device=DEV)
        if c["both"]:
            st["qt"] = _rows(cols, rows, F8[c["f8"]], tight)
            st["st"] = torch.empty(-(-cols // group), -(-rows // 128), dtype=torch.float8_e8m0fnu, device=DEV)
    else:
        rows, n, d = c["rows"], c["n"], DENSE[c["x"]]
        st["w"] = (1 + 0.1 * torch.randn(n, generator=g, device=DEV)).to(d)
        if c["kind"] == "norm":
            tight = c["tight"]
            st["x"] = _values(g, rows, n, 1.0).to(d)
            st["res"] = (3 * torch.randn(rows, n, generator=g, device=DEV)).to(d) if c["res"] else None
            st["h"] = torch.empty(rows, n, dtype=d, device=DEV) if c["res"] else None
            st["q"] = _rows(rows, n, F8["e4m3"], tight)
            st["s"] = torch.empty(rows, -(-n // 128), dtype=torch.float8_e8m0fnu, device=DEV)
            st["y"] = torch.empty(rows, n, dtype=d, device=DEV) if c["train"] else None
            st["rstd"] = torch.empty(rows, dtype=torch.float32, device=DEV) if c["train"] else None
        else:
            st["h"] = _values(g, rows, n, 1.0).to(d)
            st["dy"] = (1e-2 * torch.randn(rows, n, generator=g, device=DEV)).to(d)
            st["dres"] = (1e-2 * torch.randn(rows, n, generator=g, device=DEV)).to(d) if c["dres"] else None
            st["rstd"] = (st["h"].double().square().mean(1) + EPS).rsqrt().float()
            st["dx"] = torch.empty(rows, n, dtype=d, device=DEV)
            st["dw"] = torch.empty(n, dtype=torch.float32, device=DEV)
    return st


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _spread_scales(s, group, rows, cols):
    return s.float().repeat_interleave(group, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def _scales(x, f8, group):
    """The smallest power of two for each block of group x 128 that brings it into the type's range; 1 for a block of zeros."""
    rows, cols = x.shape
    gr, gc = -(-rows // group), -(-cols // 128)
    a = torch.zeros(gr * group, gc * 128, device=x.device)
    a[:rows, :cols] = x.abs()
    top = a.view(gr, group, gc, 128).amax((1, 3))
    part, exp = torch.frexp(top)
    e = (exp - TOP[f8] + (part > 0.875).int()).clamp(min=-126)
    return torch.exp2(torch.where(top > 0, e, torch.zeros_like(e)).double()).float()


def _quantised(x, f8, group):
    """(q, s) of a matrix of float32."""
    s = _scales(x, f8, group)
    return (x / _spread_scales(s, group, *x.shape)).to(F8[f8]), s.to(torch.float8_e8m0fnu)


def _value(mat, group):
    return mat["q"].float() * _spread_scales(mat["s"], group, *mat["q"].shape)


def _plain(st):
    c = st["case"]
    if c["kind"] == "product":
        p = torch.matmul(_value(st["a"], c["ga"]), _value(st["b"], c["gb"]).t())
        if c["beta"]:
            p += c["beta"] * st["c"].float()
        st["c"].copy_(p)
        return st["c"]
    if c["kind"] == "quant":
        x = st["x"].float()
        out = list(_quantised(x, c["f8"], c["group"]))
        return out + list(_quantised(x.t().contiguous(), c["f8"], c["group"])) if c["both"] else out
    d, w = DENSE[c["x"]], st["w"].float()
    if c["kind"] == "norm":
        h = st["x"].float() + st["res"].float() if c["res"] else st["x"].float()
        rstd = torch.rsqrt((h * h).mean(1) + EPS)
        y = h * rstd[:, None] * w
        out = list(_quantised(y, "e4m3", 1))
        if c["res"]:
            out.append(h.to(d))
        return out + [y.to(d), rstd] if c["train"] else out
    h, dy, rstd = st["h"].float(), st["dy"].float(), st["rstd"][:, None]
    xhat, g = h * rstd, dy * w
    dx = rstd * (g - xhat * (g * xhat).mean(1, keepdim=True))
    if c["dres"]:
        dx = dx + st["dres"].float()
    return [dx.to(d), (dy * xhat).sum(0)]


# ---- the framework's calls -----------------------------------------------------------------------------------------
def _library():
    if "bofhip" not in sys.modules:
        sys.path.insert(0, "blas-on-flash_amd")
    import bofhip
    return bofhip


def _kernels(st):
    L, c = _library(), st["case"]
    code = {"f32": L.F32, "bf16": L.BF16, "f16": L.F16, "e4m3": L.E4M3, "e5m2": L.E5M2}
    stream = torch.cuda.current_stream().cuda_stream
    at = lambda t: t.data_ptr() if t is not None else 0  # noqa: E731
    ld = lambda t: t.stride(0) if t is not None else 0  # noqa: E731
    if c["kind"] == "product":
        a, b, o = st["a"], st["b"], st["c"]
        L.f8_gemm(c["m"], c["n"], c["k"], 1.0, at(a["q"]), ld(a["q"]), code[c["a"]], at(a["s"]), ld(a["s"]), c["ga"],
                  at(b["q"]), ld(b["q"]), code[c["b"]], at(b["s"]), ld(b["s"]), c["gb"], c["beta"], at(o), ld(o), code[c["out"]],
                  at(st["work"]), SCRATCH, stream)
        return o
    if c["kind"] == "quant":
        x, qt, t = st["x"], st.get("qt"), st.get("st")
        L.f8_quant(c["rows"], c["cols"], at(x), ld(x), code[c["x"]], code[c["f8"]], c["group"], at(st["q"]), ld(st["q"]), at(st["s"]), ld(st["s"]),
                   at(qt), ld(qt), at(t), ld(t), stream)
        return [st["q"], st["s"], qt, t] if c["both"] else [st["q"], st["s"]]
    if c["kind"] == "norm":
        x, r, h, q, s, y = st["x"], st["res"], st["h"], st["q"], st["s"], st["y"]
        L.rmsnorm_f8(c["rows"], c["n"], code[c["x"]], at(x), ld(x), at(r), ld(r), at(st["w"]), EPS, at(h), ld(h), L.E4M3, at(q), ld(q), at(s), ld(s),
                     at(y), ld(y), at(st["rstd"]), stream)
        return [t for t in (q, s, h, y, st["rstd"]) if t is not None]
    dy, h, r, dx = st["dy"], st["h"], st["dres"], st["dx"]
    L.rmsnorm_grad(c["rows"], c["n"], code[c["x"]], at(dy), ld(dy), at(h), ld(h), at(st["w"]), at(st["rstd"]), at(r), ld(r), at(dx), ld(dx),
                   0.0, at(st["dw"]), at(st["work"]), SCRATCH, stream)
    return [dx, st["dw"]]


def run(state):
    if own:
        return _kernels(state)
    return _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    c = case
    size = {"f32": 4, "bf16": 2, "f16": 2}
    blocks = lambda rows, cols, group: -(-rows // group) * -(-cols // 128)  # noqa: E731
    if c["kind"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        b = m * k + n * k + blocks(m, k, c["ga"]) + blocks(n, k, c["gb"]) + m * n * size[c["out"]] * (2 if c["beta"] else 1)
        return {"bytes": b, "flops": 2 * m * n * k}
    if c["kind"] == "quant":
        rows, cols = c["rows"], c["cols"]
        b = rows * cols * (size[c["x"]] + 1) + blocks(rows, cols, c["group"])
        if c["both"]:
            b += rows * cols + blocks(cols, rows, c["group"])
        return {"bytes": b, "flops": 3 * rows * cols}
    rows, n, z = c["rows"], c["n"], size[c["x"]]
    if c["kind"] == "norm":
        b = rows * n * (z * (1 + 2 * c["res"] + c["train"]) + 1) + blocks(rows, n, 1) + n * z + (4 * rows if c["train"] else 0)
        return {"bytes": b, "flops": 8 * rows * n}
    return {"bytes": rows * n * z * (3 + c["dres"]) + n * (z + 4) + 4 * rows, "flops": 12 * rows * n}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------
def _decoded(mat, group):
    """q * s in 64 bits, block by block of the contracted dimension."""
    q, s = mat["q"].double(), mat["s"].float().double()
    rows, cols = q.shape
    block = torch.arange(cols, device=q.device) // 128
    return q * s[torch.arange(rows, device=q.device) // group][:, block]


def _unrounded(x, f8, group):
    """What q stands for before its rounding, and the scales, from a matrix in 64 bits."""
    x = x.cpu().numpy() if x.numel() < 4096 else x
    if isinstance(x, np.ndarray):
        x = torch.from_numpy(x).to(DEV)
    rows, cols = x.shape
    row, col = torch.arange(rows, device=DEV) // group, torch.arange(cols, device=DEV) // 128
    tops = torch.zeros(int(row[-1]) + 1, cols, dtype=torch.float64, device=DEV)
    tops.index_reduce_(0, row, x.abs(), "amax")
    top = torch.zeros(int(row[-1]) + 1, int(col[-1]) + 1, dtype=torch.float64, device=DEV)
    top.index_reduce_(1, col, tops, "amax")
    limit = 448.0 if f8 == "e4m3" else 57344.0
    e = torch.ceil(torch.log2(top / limit))
    e = torch.where(torch.exp2(e - 1) * limit >= top, e - 1, e)  # the logarithm may land on the wrong side of a border
    e = torch.where(torch.exp2(e) * limit < top, e + 1, e)
    s = torch.where(top > 0, torch.exp2(e.clamp(min=-126.0)), torch.ones_like(top))
    return x / s[row][:, col], s


def exact(case, seed):
    st, c = prepare(case, seed), case
    if c["kind"] == "product":
        p = _decoded(st["a"], c["ga"]) @ _decoded(st["b"], c["gb"]).t()
        return p + c["beta"] * st["c"].double() if c["beta"] else p
    if c["kind"] == "quant":
        x = st["x"].double()
        out = list(_unrounded(x, c["f8"], c["group"]))
        return out + list(_unrounded(x.t().contiguous(), c["f8"], c["group"])) if c["both"] else out
    w = st["w"].double()
    if c["kind"] == "norm":
        h = st["x"].double() + st["res"].double() if c["res"] else st["x"].double()
        rstd = 1.0 / torch.sqrt(torch.sum(h ** 2, 1) / c["n"] + EPS)
        y = w * (h * rstd[:, None])
        # the scales jump by two at a border that sums of either width may pass: no value in 64 bits to be met
        out = [_unrounded(y, "e4m3", 1)[0], None]
        if c["res"]:
            out.append(h)
        return out + [y, rstd] if c["train"] else out
    h, dy, r = st["h"].double(), st["dy"].double(), st["rstd"].double()
    dot = torch.sum(dy * w * h, 1) * r ** 3 / c["n"]
    dx = r[:, None] * dy * w - dot[:, None] * h
    if c["dres"]:
        dx = dx + st["dres"].double()
    return [dx, torch.sum(dy * h * r[:, None], 0)]
