"""Cases that time and check the library's operators of a pre-norm block in 16 bits: the RMS norm with
the residual's addition (forward, straight into FP8, backward), the matrix product with bias, activation
and residual in its epilogue (alone, and as the training step of a linear layer), and the global gradient
norm with clipping.

`run` computes each case either with `neuroflow_b200.ops` (`own` true) or in its plain form, elementary
torch operations in 32 bits.  `exact` is the definition in 64 bits.
"""
import random

import torch
import torch.nn.functional as F

own = False

DEV = "cuda"
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "none": 0}
E4M3 = torch.float8_e4m3fn
TOP = 448.0          # largest E4M3 value
LEAST = 2.0 ** -126  # smallest scale
EPS = 1e-5
CLIP_EPS = 1e-6
GELU, RELU = 1, 2


def listed():
    return [
        # one decoded token between two sub-layers: launch latency
        dict(name="rms 1x4096 bf16 + residual", op="rms", rows=1, d=4096, x="bf16", res="bf16", g="bf16"),
        # training: a full batch of wide tokens whose residual stream is kept in fp32
        dict(name="rms 16384x4096 bf16 + f32", op="rms", rows=16384, d=4096, x="bf16", res="f32", g="f32"),
        # an odd width, whose rows start anywhere
        dict(name="rms 5003x1031 f16 + residual", op="rms", rows=5003, d=1031, x="f16", res="f16", g="f16"),
        # the norm in front of an FP8 linear layer, a ragged batch of tokens
        dict(name="rms to fp8 8191x2048 bf16", op="rms_fp8", rows=8191, d=2048, x="bf16", res="bf16", g="f32"),
        # training: the norm's gradient joined with the one that comes down the residual stream
        dict(name="rms grad 16384x4096 bf16", op="rms_grad", rows=16384, d=4096, x="bf16", res="bf16", g="f32"),
        # one token through a square layer: the weight's bytes
        dict(name="gemm 1x4096x4096 + residual", op="gemm", m=1, n=4096, k=4096, x="bf16", out="bf16", bias=True, act=0, res=True, t=False),
        # a small batch, odd in every direction
        dict(name="gemm 333x1001x1543 f16 relu", op="gemm", m=333, n=1001, k=1543, x="f16", out="f16", bias=True, act=RELU, res=False, t=False),
        # a full batch into the feed-forward's wide side
        dict(name="gemm 8192x16384x4096 gelu", op="gemm", m=8192, n=16384, k=4096, x="bf16", out="bf16", bias=True, act=GELU, res=False, t=False),
        # a weight gradient: both operands run along the tokens, fp32 result
        dict(name="gemm wgrad 4096x2048x8192", op="gemm", m=4096, n=2048, k=8192, x="bf16", out="f32", bias=False, act=0, res=False, t=True),
        # forward and backward of one linear layer with everything in its epilogue, ragged tokens
        dict(name="linear step 4095x2048x8192", op="linear", m=4095, n=2048, k=8192, x="bf16", act=GELU),
        # the gradients of a small feed-forward block: launch latency
        dict(name="clip 6 tensors f32", op="clip", tensors=6, total=66000, x="f32", out="f32", tight=True),
        # the gradients of a deep model in bf16, clipped into the optimizer's fp32 buffer
        dict(name="clip 290 tensors bf16 to f32", op="clip", tensors=290, total=1 << 27, x="bf16", out="f32", tight=True),
    ]


def draw(rng):
    def log(a, b):
        return max(a, min(b, int(round(a * (b / a) ** rng.random()))))

    op = rng.choice(["rms", "rms_fp8", "rms_grad", "gemm", "gemm", "gemm", "linear", "clip", "clip"])
    if op in ("rms", "rms_fp8", "rms_grad"):
        d = log(32, 16384)
        x = rng.choice(["bf16", "f32", "f16"])
        return dict(op=op, rows=log(1, max(1, min(131072, (1 << 26) // d))), d=d, x=x, res=rng.choice([x, x, "f32", "none"]),
                    g=rng.choice([x, "f32"]))
    if op == "clip":
        tensors = log(1, 600)
        x = rng.choice(["bf16", "f32", "f16"])
        return dict(op=op, tensors=tensors, total=log(4096, 1 << 26), x=x, out=rng.choice([x, "f32"]), tight=rng.random() < 0.8)
    step = rng.choice([1, 8, 8, 8, 64])  # odd widths, and the multiples of eight and 64 that models have
    n, k = (max(1, log(24, 16384) // step) * step for _ in range(2))
    if op == "gemm":
        x = rng.choice(["bf16", "bf16", "f16"])
        return dict(op=op, m=log(1, max(1, min(16384, (1 << 39) // (n * k)))), n=n, k=k, x=x, out=rng.choice([x, x, "f32"]),
                    bias=rng.random() < 0.6, act=rng.choice([0, 0, GELU, RELU]), res=rng.random() < 0.4, t=rng.random() < 0.25)
    return dict(op=op, m=log(16, max(16, min(16384, (1 << 37) // (n * k)))), n=n, k=k, x="bf16", act=rng.choice([0, GELU, RELU]))


def up(a, b):
    return -(-a // b)


def work(c):
    op = c["op"]
    if op in ("rms", "rms_fp8", "rms_grad"):
        rows, d, e = c["rows"], c["d"], SIZE[c["x"]]
        r = SIZE[c["res"]]  # the residual is read and the sum written
        par = d * SIZE[c["g"]]
        if op == "rms":
            return {"bytes": rows * d * (2 * e + 2 * r) + par + 4 * rows, "flops": 5 * rows * d}
        if op == "rms_fp8":
            return {"bytes": rows * d * (e + 2 * r + 1) + 4 * rows * up(d, 128) + par + 4 * rows, "flops": 7 * rows * d}
        # dy, the sum and the stream's gradient read; the gradient written (twice where the types differ)
        h = r if r else e
        return {"bytes": rows * d * (2 * e + (3 * h if h != e else 2 * h if r else h)) + 2 * par + 4 * rows, "flops": 9 * rows * d}
    if op == "clip":
        return {"bytes": c["total"] * (SIZE[c["x"]] + SIZE[c["out"]]), "flops": 3 * c["total"]}
    m, n, k, e = c["m"], c["n"], c["k"], SIZE[c["x"]]
    if op == "gemm":
        return {"bytes": e * (m * k + n * k) + m * n * SIZE[c["out"]] * (2 if c["res"] else 1) + (4 * n if c["bias"] else 0),
                "flops": 2 * m * n * k}
    # x, w, b, residual, dy read; y, dx, dw, db written
    return {"bytes": e * (2 * m * k + 2 * n * k + 3 * m * n + 2 * n), "flops": 6 * m * n * k}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def activations(gen, rows, cols, dt):
    """Tokens as a mixer has them: channels of unlike size, a few of them large."""
    return (normal(gen, rows, cols) * torch.exp(0.7 * normal(gen, 1, cols))).to(dt)


def parts(tensors, total, seed):
    """`tensors` sizes that add up to `total`, from a few elements (biases, norms) to most of it (weights)."""
    rng = random.Random(seed)
    w = [10.0 ** rng.uniform(-3, 0) for _ in range(tensors)]
    sizes = [max(1, int(total * v / sum(w))) for v in w]
    sizes[sizes.index(max(sizes))] += total - sum(sizes)
    return sizes


def prepare(case, seed):
    c, gen = dict(case), torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": c}
    op = c["op"]
    if op in ("rms", "rms_fp8", "rms_grad"):
        rows, d, dt = c["rows"], c["d"], DT[c["x"]]
        s["g"] = (1 + 0.1 * normal(gen, d)).to(DT[c["g"]])
        s["x"] = activations(gen, rows, d, dt)
        s["res"] = None if c["res"] == "none" else (2 * normal(gen, rows, d)).to(DT[c["res"]])
        if op == "rms_grad":
            # what the forward pass left behind: the sum and 1 / its root mean square
            _, h, s["rstd"] = plain_rms(s["x"], s["res"], s["g"])
            s["h"] = s["x"] if h is None else h
            s["dy"] = (0.02 * normal(gen, rows, d)).to(dt)
            s["dsum"] = None if c["res"] == "none" else (0.02 * normal(gen, rows, d)).to(DT[c["res"]])
            del s["x"], s["res"]
    elif op == "gemm":
        m, n, k, dt = c["m"], c["n"], c["k"], DT[c["x"]]
        if c["t"]:  # as the forward pass left them, along the tokens
            s["a"] = (0.02 * normal(gen, k, m)).to(dt).t()
            s["b"] = activations(gen, k, n, dt).t()
        else:
            s["a"] = activations(gen, m, k, dt)
            s["b"] = (normal(gen, n, k) / k ** 0.5).to(dt)
        s["bias"] = 0.1 * normal(gen, n) if c["bias"] else None
        s["res"] = normal(gen, m, n).to(DT[c["out"]]) if c["res"] else None
    elif op == "linear":
        m, n, k, dt = c["m"], c["n"], c["k"], DT[c["x"]]
        s["x"] = activations(gen, m, k, dt).requires_grad_()
        s["w"] = (normal(gen, n, k) / k ** 0.5).to(dt).requires_grad_()
        s["b"] = (0.1 * normal(gen, n)).to(dt).requires_grad_()
        s["res"] = normal(gen, m, n).to(dt).requires_grad_()
        s["dy"] = (0.02 * normal(gen, m, n)).to(dt)
    else:
        dt = DT[c["x"]]
        sizes = parts(c["tensors"], c["total"], c["tensors"] * 7919 + c["total"])
        s["grads"] = [(normal(gen, n) * 0.01).to(dt) for n in sizes]
        s["flat"] = torch.empty(c["total"], device=DEV, dtype=DT[c["out"]])  # the optimizer's buffer
        s["out"] = list(s["flat"].split(sizes))
        s["max_norm"] = 0.001 * c["total"] ** 0.5 if c["tight"] else c["total"] ** 0.5
    return s


# ---------------------------------------------------------------------------------------------
# plain forms: elementary torch operations in 32 bits
# ---------------------------------------------------------------------------------------------
def plain_rms(x, res, g):
    """(y in fp32, the sum in the residual's type, rstd); the norm is that of the sum as it is stored."""
    h = None if res is None else (x.float() + res.float()).to(res.dtype)
    v = x.float() if res is None else h.float()
    rstd = 1.0 / torch.sqrt((v * v).mean(1) + EPS)
    return v * rstd[:, None] * g.float(), h, rstd


def plain_rms_grad(dy, h, rstd, g, dsum):
    dy, xh = dy.float(), h.float() * rstd[:, None]
    a = dy * g.float()
    dh = rstd[:, None] * (a - xh * (a * xh).mean(1, keepdim=True))
    if dsum is not None:
        dh = dh + dsum.float()
    return dh, (dy * xh).sum(0)


def plain_quantise(x):
    """(codes as E4M3, scales) of groups of 128 along the rows."""
    r, k = x.shape
    g = F.pad(x, (0, up(k, 128) * 128 - k)).reshape(r, up(k, 128), 128)
    scale = torch.clamp_min(g.abs().amax(2) / torch.full((), TOP, device=DEV), LEAST)
    v = g * (1.0 / scale)[:, :, None]
    # the library's encoder keeps what lies under the smallest normal number at the largest subnormal one
    v = torch.where((v.abs() < 2.0 ** -6) & (v.abs() > 7 * 2.0 ** -9), torch.copysign(torch.full_like(v, 7 * 2.0 ** -9), v), v)
    return torch.clamp(v, -TOP, TOP).to(E4M3).reshape(r, -1)[:, :k], scale


def plain_act(z, act):
    if act == GELU:
        return 0.5 * z * (1.0 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z)))
    return torch.clamp_min(z, 0.0) if act == RELU else z


def plain_slope(z, act):
    """The activation's derivative."""
    if act == GELU:
        t = torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * 0.7978845608028654 * (1.0 + 3 * 0.044715 * z * z)
    return (z > 0).float() if act == RELU else torch.ones_like(z)


def plain(s):
    c = s["case"]
    op = c["op"]
    if op in ("rms", "rms_fp8"):
        y, h, rstd = plain_rms(s["x"], s["res"], s["g"])
        out = {"rstd": rstd} if h is None else {"sum": h, "rstd": rstd}
        if op == "rms":
            return out | {"y": y.to(s["x"].dtype)}
        codes, scales = plain_quantise(y)
        return out | {"codes": codes, "scales": scales}
    if op == "rms_grad":
        dh, dg = plain_rms_grad(s["dy"], s["h"], s["rstd"], s["g"], s["dsum"])
        return {"dx": dh.to(s["dy"].dtype), "dres": dh.to(s["h"].dtype), "dg": dg.to(s["g"].dtype)}
    if op == "gemm":
        z = s["a"].float() @ s["b"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"]
        y = plain_act(z, c["act"])
        if s["res"] is not None:
            y = y + s["res"].float()
        return y.to(DT[c["out"]])
    if op == "linear":
        with torch.no_grad():
            x, w, dy, dt = s["x"].float(), s["w"].float(), s["dy"].float(), DT[c["x"]]
            z = x @ w.t() + s["b"].float()
            dz = dy * plain_slope(z, c["act"])
            return {"y": (plain_act(z, c["act"]) + s["res"].float()).to(dt), "dx": (dz @ w).to(dt), "dw": (dz.t() @ x).to(dt),
                    "db": dz.sum(0).to(dt), "dres": s["dy"]}
    flat = torch.cat([g.float() for g in s["grads"]])
    norm = torch.sqrt((flat * flat).sum(dtype=torch.float64))
    scale = torch.clamp_max(s["max_norm"] / (norm + CLIP_EPS), 1.0).float()
    return {"norm": norm.float(), "clipped": (flat * scale).to(DT[c["out"]])}


# ---------------------------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------------------------
def library(s):
    from neuroflow_b200 import ops
    c = s["case"]
    op = c["op"]
    if op in ("rms", "rms_fp8"):
        call = ops.rms_norm if op == "rms" else ops.rms_norm_fp8
        got = call(s["x"], s["g"], EPS, residual=s["res"], stats=True)
        out = {"rstd": got[-1]} if s["res"] is None else {"sum": got[1], "rstd": got[-1]}
        return out | ({"y": got[0]} if op == "rms" else {"codes": got[0].codes, "scales": got[0].scales})
    if op == "rms_grad":
        dx, dres, dg = ops.rms_norm_backward(s["dy"], s["h"], s["rstd"], s["g"], dsum=s["dsum"])
        return {"dx": dx, "dres": dres, "dg": dg}
    if op == "gemm":
        return ops.gemm(s["a"], s["b"], bias=s["bias"], act=c["act"], residual=s["res"], out_dtype=DT[c["out"]])
    if op == "linear":
        y = ops.linear(s["x"], s["w"], s["b"], act=c["act"], residual=s["res"])
        dx, dw, db, dres = torch.autograd.grad(y, (s["x"], s["w"], s["b"], s["res"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db, "dres": dres}
    norm = ops.clip_grad_norm(s["grads"], s["max_norm"], CLIP_EPS, out=s["out"])
    return {"norm": norm, "clipped": s["flat"]}


def run(state):
    return library(state) if own else plain(state)


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def nearest_e4m3(v):
    """v (64 bits) on the E4M3 grid: three fraction bits, ties to even, steps of 2^-9 under 2^-6 and
    there no further than 7 steps, nothing above 448."""
    size = torch.abs(v)
    _, e = torch.frexp(size)
    step = torch.ldexp(torch.ones_like(size), torch.clamp_min(e - 1, -6) - 3)
    q = torch.round(size / step) * step
    low = torch.clamp_max(torch.round(size * 512.0), 7.0) / 512.0
    return torch.sign(v) * torch.clamp_max(torch.where(size < 2.0 ** -6, low, q), TOP)


def exact_quantise(x):
    """(E4M3 values, scales) of x in 64 bits; the scale, its reciprocal and their product with an element
    are numbers of 32 bits by definition."""
    r, k = x.shape
    cols = -(-k // 128)
    padded = torch.zeros(r, cols * 128, dtype=torch.float64, device=x.device)
    padded[:, :k] = x
    cells = padded.view(r, cols, 128)
    scale = torch.maximum(cells.abs().amax(2) / 448.0, torch.full((r, cols), 2.0 ** -126, dtype=torch.float64, device=x.device))
    scale = scale.float().double()
    inverse = (1.0 / scale).float().double()
    scaled = (cells * inverse[:, :, None]).float().double()
    return nearest_e4m3(scaled).reshape(r, -1)[:, :k], scale


def exact_gelu(z):
    """(gelu, its derivative) by the logistic function: gelu = z s(2u), u = sqrt(2 / pi) (z + 0.044715 z^3)."""
    c = (2.0 / torch.pi) ** 0.5
    sg = torch.sigmoid(2.0 * c * (z + 0.044715 * z ** 3))
    return z * sg, sg + z * sg * (1.0 - sg) * 2.0 * c * (1.0 + 0.134145 * z ** 2)


def exact_act(z, act):
    if act == GELU:
        return exact_gelu(z)
    on = torch.where(z > 0, torch.ones_like(z), torch.zeros_like(z))
    return (z * on, on) if act == RELU else (z, torch.ones_like(z))


def exact(case, seed):
    s = prepare(case, seed)
    c, op = s["case"], case["op"]
    D = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and k != "flat"}
    if op in ("rms", "rms_fp8"):
        out = {}
        h = D["x"]
        if "res" in D:
            h = out["sum"] = (D["x"] + D["res"]).to(s["res"].dtype).double()  # the stored sum is what is normalised
        rstd = out["rstd"] = (torch.einsum("rd,rd->r", h, h) / c["d"] + EPS) ** -0.5
        y = h * D["g"] * rstd[:, None]
        if op == "rms":
            return out | {"y": y}
        codes, scales = exact_quantise(y)
        return out | {"codes": codes, "scales": scales}
    if op == "rms_grad":
        # the derivative of sum(dy * y) by the quotient rule: y = g h / n, n = sqrt(mean(h^2) + eps)
        h, dy, r = D["h"], D["dy"], D["rstd"][:, None]
        dyg = dy * D["g"]
        dh = dyg * r - h * (torch.einsum("rd,rd->r", dyg, h)[:, None] / c["d"]) * r ** 3
        if "dsum" in D:
            dh = dh + D["dsum"]
        return {"dx": dh, "dres": dh, "dg": torch.einsum("rd,rd->d", dy, h * r)}
    if op == "gemm":
        z = torch.mm(D["a"], D["b"].t())
        if c["bias"]:
            z += D["bias"]
        y = exact_act(z, c["act"])[0]
        return y + D["res"] if c["res"] else y
    if op == "linear":
        y, slope = exact_act(torch.addmm(D["b"], D["x"], D["w"].t()), c["act"])
        dz = D["dy"] * slope
        return {"y": y + D["res"], "dx": torch.mm(dz, D["w"]), "dw": torch.mm(dz.t(), D["x"]), "db": dz.sum(0), "dres": D["dy"]}
    grads = torch.cat([g.double() for g in s["grads"]])
    norm = torch.linalg.vector_norm(grads)
    return {"norm": norm, "clipped": grads * min(1.0, s["max_norm"] / (float(norm) + CLIP_EPS))}
