"""Cases that measure the layer norm and the 4-bit microscaled (MXFP4) operators: their plain forms in elementary torch
operations, and the calls a user makes of the framework's kernels (``own``).

An MXFP4 matrix (rows x cols) is held as the framework's ``MX4Tensor`` documents it: ``data`` uint8 (rows, 16 * nb), two e2m1 codes
per byte, the even column in the low half, nb = ceil(cols / 32) blocks per row, zeros behind the last column; ``scales`` uint8
(ceil(rows / 128), ceil(nb / 4), 32, 4, 4): the power-of-two exponent (bias 127) of block b of row r stands at
[r // 128, b // 4, r % 32, r % 128 // 32, b % 4].
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5


def listed():
    return [
        # one token of a language model between two layers: nothing but latency
        {"name": "ln one token", "op": "ln", "dtype": "bf16", "rows": 1, "cols": 1024, "train": False},
        # a feature map of 64 video streams, 14x14 pixels of 576 channels (the framework's own benchmark shape), inference
        {"name": "ln maps 576ch 14x14 x64", "op": "ln", "dtype": "f16", "rows": 12544, "cols": 576, "train": False},
        # a training step's norm over 16384 tokens, forward and backward
        {"name": "ln train 16384x4096", "op": "ln", "dtype": "bf16", "rows": 16384, "cols": 4096, "train": True},
        # full precision and a width that no vector access divides
        {"name": "ln train odd 2500x1001", "op": "ln", "dtype": "f32", "rows": 2500, "cols": 1001, "train": True},
        # delta form: 64 streams, 28x28 pixels of 192 channels, a third of the pixels updated
        {"name": "ln delta 192ch 28x28 x64", "op": "lnd", "dtype": "f16", "n": 64, "h": 28, "w": 28, "cols": 192, "density": 0.35},
        # delta form: the detector's map (136x240, 64 channels, 32 streams), a tenth of the pixels updated
        {"name": "ln delta 64ch 136x240 x32", "op": "lnd", "dtype": "f16", "n": 32, "h": 136, "w": 240, "cols": 64, "density": 0.1},
        # quantising the activations of a decoding batch
        {"name": "quantize 16x4096", "op": "quant", "dtype": "bf16", "rows": 16, "cols": 4096, "both": False},
        # quantising a training step's gradient for both products that read it (blocks along rows and along columns)
        {"name": "quantize both 8192x5120", "op": "quant", "dtype": "bf16", "rows": 8192, "cols": 5120, "both": True},
        # the classifier of 64 video streams (MobileNetV2's head), weights packed once
        {"name": "linear 64x1280-1000", "op": "lin", "dtype": "f16", "rows": 64, "cols": 1280, "outs": 1000, "train": False},
        # one token through a wide layer: bound by the weight's bytes
        {"name": "linear 1x4096-14336", "op": "lin", "dtype": "bf16", "rows": 1, "cols": 4096, "outs": 14336, "train": False},
        # a prompt of 8192 tokens
        {"name": "linear 8192x4096-14336", "op": "lin", "dtype": "bf16", "rows": 8192, "cols": 4096, "outs": 14336, "train": False},
        # a training step's layer: three products, every operand quantised on the way, ragged in every direction
        {"name": "linear train 4100x2050-4010", "op": "lin", "dtype": "bf16", "rows": 4100, "cols": 2050, "outs": 4010, "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ln", "ln", "lnd", "quant", "lin", "lin"])
    if op == "ln":
        cols = _log(rng, 24, 16000)
        return {"op": op, "dtype": rng.choice(list(DTYPES)), "rows": min(_log(rng, 1, 30000), 2 ** 25 // cols), "cols": cols,
                "train": rng.random() < 0.6}
    if op == "lnd":
        cols = _log(rng, 16, 1280)
        n, h, w = _log(rng, 1, 64), _log(rng, 7, 136), _log(rng, 7, 240)
        n = max(1, min(n, 2 ** 25 // (cols * h * w)))
        return {"op": op, "dtype": rng.choice(["f32", "f16"]), "n": n, "h": h, "w": w, "cols": cols, "density": round(rng.uniform(0.02, 1.0), 3)}
    if op == "quant":
        cols = _log(rng, 20, 10000)
        return {"op": op, "dtype": rng.choice(list(DTYPES)), "rows": min(_log(rng, 1, 30000), 2 ** 25 // cols), "cols": cols,
                "both": rng.random() < 0.5}
    train = rng.random() < 0.4
    cols, outs = _log(rng, 40, 8000), _log(rng, 24, 14336)
    rows = max(1, min(_log(rng, 1, 8192), 2 ** 36 // (cols * outs)))
    return {"op": op, "dtype": rng.choice(list(DTYPES)), "rows": rows, "cols": cols, "outs": outs, "train": train}


# ---- inputs ----------------------------------------------------------------------------------------------------

def _activations(shape, dtype, g):
    """What a layer hands on: a normal body, channels that are ten times larger, an offset."""
    x = torch.randn(shape, generator=g, device="cuda")
    wide = torch.rand(shape[-1], generator=g, device="cuda") < 0.02
    return (x * (1.0 + 9.0 * wide) + 0.3).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, op, c = DTYPES[case["dtype"]], case["op"], case["cols"]
    s = dict(case)
    if op == "ln":
        s["x"] = _activations((case["rows"], c), dtype, g)
        s["weight"] = (1.0 + 0.2 * torch.randn(c, generator=g, device="cuda")).to(dtype)
        s["bias"] = (0.2 * torch.randn(c, generator=g, device="cuda")).to(dtype)
        if case["train"]:
            s["dy"] = torch.randn((case["rows"], c), generator=g, device="cuda").to(dtype)
            for k in ("x", "weight", "bias"):
                s[k].requires_grad_()
    elif op == "lnd":
        # a video that goes one frame on and back again; pixels are N,C,H,W in channels-last memory, held here as N,H,W,C
        n, h, w = case["n"], case["h"], case["w"]
        x = _activations((n, h, w, c), dtype, g)
        s["weight"] = (1.0 + 0.2 * torch.randn(c, generator=g, device="cuda")).to(dtype)
        s["bias"] = (0.2 * torch.randn(c, generator=g, device="cuda")).to(dtype)
        wide = x.float()
        wide = wide - wide.mean(-1, keepdim=True)
        y = wide * torch.rsqrt(wide.square().mean(-1, keepdim=True) + EPS) * s["weight"].float() + s["bias"].float()
        mask = torch.rand((n, h, w), generator=g, device="cuda") < case["density"]
        moved = torch.rand((n, h, w), generator=g, device="cuda") < 0.8        # the others change by less than the threshold
        step = torch.randn((n, h, w, c), generator=g, device="cuda") * torch.where(moved, 1.0, 1e-4)[..., None]
        step[..., 0] = torch.where(moved, 2.0 * wide.abs().amax(-1) + 3.0, step[..., 0])      # one channel moves far: never next to the threshold
        delta = torch.where(mask[..., None], step, torch.zeros((), device="cuda")).to(dtype)
        s["frames"] = [delta.permute(0, 3, 1, 2), (-delta).permute(0, 3, 1, 2)]
        s["mask"] = mask.to(torch.int32)[:, None]
        s["prev_in"], s["prev_out"] = x.permute(0, 3, 1, 2), y.to(dtype).permute(0, 3, 1, 2)
        s["out"] = torch.zeros_like(s["prev_in"])
        s["out_mask"] = torch.zeros_like(s["mask"])
        s["threshold"], s["step"] = 0.05, 0
    elif op == "quant":
        x = _activations((case["rows"], c), torch.float32, g)
        s["x"] = (x * torch.exp(2.0 * torch.randn((case["rows"], 1), generator=g, device="cuda"))).to(dtype)
    else:
        o = case["outs"]
        s["x"] = _activations((case["rows"], c), dtype, g)
        w = torch.randn((o, c), generator=g, device="cuda") * c ** -0.5
        s["bias"] = torch.randn(o, generator=g, device="cuda").to(dtype)
        if case["train"]:
            s["w"], s["dy"] = w.to(dtype), torch.randn((case["rows"], o), generator=g, device="cuda").to(dtype)
            for k in ("x", "w", "bias"):
                s[k].requires_grad_()
        else:       # a checkpoint's packed weight
            s["wdata"], s["wscales"] = _pack(*_codes(w))
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------

def _norm(x, weight, bias):
    """y and what the backward pass reads again, in 32 bits."""
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt(xc.square().mean(-1, keepdim=True) + EPS)
    xh = xc * rstd
    return xh * weight + bias, xh, rstd


def _codes(x):
    """e2m1 codes (rows, cols) and scale bytes (rows, ceil(cols / 32)) of a float32 matrix, blocks along the columns."""
    rows, cols = x.shape
    nb = -(-cols // 32)
    b = torch.nn.functional.pad(x, (0, nb * 32 - cols)).view(rows, nb, 32)
    top = b.abs().amax(-1)
    field = top.view(torch.int32) >> 23                                         # biased exponent of the largest value
    finite = field < 255
    scale = torch.where(finite, (field - 2).clamp(min=0), 255)
    factor = ((254 - scale.clamp(max=253)) << 23).view(torch.float32)            # 2 ** (127 - scale)
    v = torch.where(finite[..., None], b * factor[..., None], torch.zeros((), device=x.device))
    a = v.abs().clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))             # spacing of e2m1 around a
    m = torch.round(a / step) * step                                             # ties to even, as the spacing's parity is the mantissa's
    code = torch.where(m < 2.0, m * 2, torch.where(m < 4.0, m + 2, m / 2 + 4)).to(torch.uint8)
    code = code | ((v < 0) & (code > 0)).to(torch.uint8) * 8
    return code.view(rows, nb * 32), scale.to(torch.uint8)


def _pack(code, scale):
    rows, nb = scale.shape
    data = code[:, 0::2] | (code[:, 1::2] << 4)
    rt, bt = -(-rows // 128), -(-nb // 4)
    full = torch.zeros((rt * 128, bt * 4), dtype=torch.uint8, device=code.device)
    full[:rows, :nb] = scale
    return data.contiguous(), full.view(rt, 4, 32, bt, 4).permute(0, 3, 2, 1, 4).contiguous()


def _values(code, scale, cols):
    """The matrix that codes and scale bytes stand for."""
    rows, nb = scale.shape
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
    s = torch.where(scale == 255, torch.full((), math.nan, device=code.device), torch.exp2(scale.float() - 127))
    return (table[code.int()].view(rows, nb, 32) * s[..., None]).view(rows, nb * 32)[:, :cols]


def _unpack(data, scales, rows):
    nb = data.shape[1] // 16
    code = torch.stack((data & 15, data >> 4), -1).view(rows, nb * 32)
    rt, bt = scales.shape[:2]
    return code, scales.permute(0, 3, 2, 1, 4).reshape(rt * 128, bt * 4)[:rows, :nb]


def _fake(x):
    """x rounded to MXFP4 along its rows, in 32 bits."""
    x = x.float()
    return _values(*_codes(x), x.shape[1])


def _run_plain(s):
    op = s["op"]
    if op == "ln":
        with torch.no_grad():
            dtype, w = s["x"].dtype, s["weight"].float()
            y, xh, rstd = _norm(s["x"].float(), w, s["bias"].float())
            if not s["train"]:
                return y.to(dtype)
            dy = s["dy"].float()
            gr = dy * w
            dx = rstd * (gr - gr.mean(-1, keepdim=True) - xh * (gr * xh).mean(-1, keepdim=True))
            return y.to(dtype), dx.to(dtype), (dy * xh).sum(0).to(dtype), dy.sum(0).to(dtype)
    if op == "lnd":
        delta = s["frames"][s["step"] % 2].permute(0, 2, 3, 1)
        s["step"] += 1
        prev_in, prev_out, out = (s[k].permute(0, 2, 3, 1) for k in ("prev_in", "prev_out", "out"))
        on = s["mask"][:, 0, :, :, None] != 0
        u = torch.where(on, (prev_in.float() + delta.float()).to(delta.dtype), prev_in)
        y = _norm(u.float(), s["weight"].float(), s["bias"].float())[0].to(delta.dtype)
        e = (y.float() - prev_out.float()).to(delta.dtype)
        keep = on & (e.float().abs() > s["threshold"]).any(-1, keepdim=True)
        prev_in.copy_(u)
        out.copy_(torch.where(keep, e, out))
        prev_out.copy_(torch.where(keep, (prev_out.float() + e.float()).to(delta.dtype), prev_out))
        s["out_mask"].copy_(keep[..., 0][:, None])
        return s["out"], s["out_mask"], s["prev_in"], s["prev_out"]
    if op == "quant":
        x = s["x"]
        v = _fake(x).to(x.dtype)
        return (v, _fake(x.t().contiguous()).to(x.dtype)) if s["both"] else v
    with torch.no_grad():
        dtype, bias = s["x"].dtype, s["bias"].float()
        if not s["train"]:
            w = _values(*_unpack(s["wdata"], s["wscales"], s["outs"]), s["cols"])
            return (_fake(s["x"]) @ w.t() + bias).to(dtype)
        x, w, dy = s["x"], s["w"], s["dy"]
        y = _fake(x) @ _fake(w).t() + bias
        dx = _fake(dy) @ _fake(w.t().contiguous()).t()
        dw = _fake(dy.t().contiguous()) @ _fake(x.t().contiguous()).t()
        return y.to(dtype), dx.to(dtype), dw.to(dtype), dy.float().sum(0).to(dtype)


# ---- the framework's calls -------------------------------------------------------------------------------------

def _run_own(s):
    import deltacnn_b200 as dc
    op = s["op"]
    if op == "ln":
        y = dc.layer_norm(s["x"], s["weight"], s["bias"], EPS)
        return (y, *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])) if s["train"] else y
    if op == "lnd":
        delta = s["frames"][s["step"] % 2]
        s["step"] += 1
        dc.layer_norm_delta(delta, s["mask"], s["prev_in"], s["prev_out"], s["weight"], s["bias"], s["threshold"], EPS,
                            out=s["out"], out_mask=s["out_mask"])
        return s["out"], s["out_mask"], s["prev_in"], s["prev_out"]
    if op == "quant":
        if not s["both"]:
            return dc.mx4_dequantize(dc.mx4_quantize(s["x"]), s["x"].dtype)
        q, qt = dc.mx4_quantize_both(s["x"])
        return dc.mx4_dequantize(q, s["x"].dtype), dc.mx4_dequantize(qt, s["x"].dtype)
    if not s["train"]:
        return dc.mx4_linear(s["x"], dc.MX4Tensor(s["wdata"], s["wscales"], (s["outs"], s["cols"])), s["bias"])
    y = dc.mx4_linear(s["x"], s["w"], s["bias"])
    return (y, *torch.autograd.grad(y, (s["x"], s["w"], s["bias"]), s["dy"]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def work(case):
    b, c, op = BYTES[case["dtype"]], case["cols"], case["op"]
    if op == "ln":
        n = case["rows"] * c
        return {"bytes": (5 if case["train"] else 2) * n * b + (4 if case["train"] else 2) * c * b, "flops": (18 if case["train"] else 8) * n}
    if op == "lnd":
        pixels = case["n"] * case["h"] * case["w"]
        active, kept = pixels * case["density"], pixels * case["density"] * 0.8
        return {"bytes": 8 * pixels + (4 * active + 2 * kept) * c * b + 2 * c * b, "flops": 11 * active * c}
    if op == "quant":
        n = case["rows"] * c
        return {"bytes": (3 if case["both"] else 2) * n * b, "flops": (8 if case["both"] else 4) * n}
    m, o = case["rows"], case["outs"]
    if case["train"]:
        return {"bytes": (2 * m * c + 2 * m * o + 2 * o * c + 2 * o) * b, "flops": 6.0 * m * c * o}
    return {"bytes": (m * c + m * o + o) * b + o * c * (0.5 + 1 / 32), "flops": 2.0 * m * c * o}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------

def _mx4_64(x):
    """MXFP4 along the rows, by its definition: X = 2 ** (floor(log2 max|v|) - 2), values to the nearest of the e2m1 grid, ties to even."""
    x = x.double()
    rows, cols = x.shape
    nb = -(-cols // 32)
    full = torch.zeros((rows, nb * 32), dtype=torch.float64, device=x.device)
    full[:, :cols] = x
    full = full.view(rows, nb, 32)
    top = full.abs().amax(2, keepdim=True)
    _, e = torch.frexp(top)                               # top = f * 2 ** e with f in [1/2, 1)
    e = torch.where(top > 0, e - 3, -127).clamp(min=-127).double()
    v = full * torch.exp2(-e)
    # a border between neighbours of the grid that is met exactly goes to the neighbour whose last bit is 0
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    borders = (grid[1:] + grid[:-1]) / 2
    a = v.abs()
    up, down = torch.bucketize(a, borders, right=True), torch.bucketize(a, borders)
    k = torch.where(up % 2 == 0, up, down)
    return (grid[k] * torch.sign(v) * torch.exp2(e)).view(rows, nb * 32)[:, :cols]


def _packed_64(data, scales, rows, cols):
    """The packed matrix in 64 bits, bit by bit: sign, two exponent bits (bias 1, 0 for 0 and 1/2), one mantissa bit."""
    k = torch.arange(cols, device=data.device)
    c = (data[:, k // 2].int() >> (4 * (k % 2)).int()) & 15
    e, m = (c >> 1) & 3, (c & 1).double()
    v = torch.where(e > 0, (1 + m / 2) * torch.exp2(e.double() - 1), m / 2) * (1 - 2 * (c >> 3)).double()
    r, b = torch.arange(rows, device=data.device)[:, None], (k // 32)[None]
    return torch.ldexp(v, scales[r // 128, b // 4, r % 32, r % 128 // 32, b % 4].int() - 127)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        op = case["op"]
        if op in ("ln", "lnd"):
            w, b = s["weight"].double(), s["bias"].double()

            def norm(x):
                mu = x.sum(-1, keepdim=True) / x.shape[-1]
                var = ((x - mu) ** 2).sum(-1, keepdim=True) / x.shape[-1]
                return (x - mu) / torch.sqrt(var + EPS), torch.sqrt(var + EPS)
        if op == "ln":
            xh, sd = norm(s["x"].double())
            y = xh * w + b
            if not case["train"]:
                return y
            dy = s["dy"].double()
            q = dy * w
            dx = (q - (q.sum(-1, keepdim=True) + xh * (q * xh).sum(-1, keepdim=True)) / case["cols"]) / sd
            return y, dx, (dy * xh).sum(0), dy.sum(0)
        if op == "lnd":
            delta, old, was, out = (t.permute(0, 2, 3, 1).double() for t in (s["frames"][0], s["prev_in"], s["prev_out"], s["out"]))
            on = (s["mask"][:, 0] != 0)[..., None]
            u = old + on * delta
            e = norm(u)[0] * w + b - was
            keep = (on & (e.abs() > s["threshold"])).any(-1, keepdim=True)
            back = lambda t: t.permute(0, 3, 1, 2)      # noqa: E731
            return back(torch.where(keep, e, out)), keep[..., 0].int()[:, None], back(u), back(torch.where(keep, was + e, was))
        if op == "quant":
            x = s["x"]
            return (_mx4_64(x), _mx4_64(x.t())) if case["both"] else _mx4_64(x)
        bias = s["bias"].double()
        if not case["train"]:
            w = _packed_64(s["wdata"], s["wscales"], case["outs"], case["cols"])
            return _mx4_64(s["x"]) @ w.t() + bias
        x, w, dy = s["x"], s["w"], s["dy"].double()
        return (_mx4_64(x) @ _mx4_64(w).t() + bias, _mx4_64(dy) @ _mx4_64(w.t()).t(), _mx4_64(dy.t()) @ _mx4_64(x.t()).t(), dy.sum(0))
