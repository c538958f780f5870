"""Cases of three operators that belong together: the token-wise half of a
transformer block whose activations are kept for the backward pass in 8 bits.

- ``norm``:   root-mean-square norm with the residual's addition, and the
              normalised rows also in 8 bits with scales;
- ``gelu``:   exact GELU whose input is kept in 8 bits for the backward pass;
- ``linear``: masked matrix product with bias, GELU and residual in its
              epilogue, and its gradients, from 8-bit or 16-bit kept inputs.

"8 bits" is one format throughout: e4m3 codes with one power-of-two scale
for every 32 neighbouring values of a row, the smallest power that keeps the
block's largest magnitude at 448 or less.

``own`` selects between the operators' plain form (elementary torch
operations in 32 bits) and the framework's entry points.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16,
          "fp32": torch.float32}
BLOCK = 32


def listed():
    return [
        # one token of a DeiT-base stream, answered alone: latency only
        {"name": "norm_one_token", "op": "norm", "rows": 1, "cols": 768,
         "dtype": "bf16", "res": "same", "keep": True, "train": False},
        # inference on 64 images: 197 tokens each, DeiT-small width, with the
        # 8-bit rows that the next product keeps
        {"name": "norm_serve_small", "op": "norm", "rows": 12608,
         "cols": 384, "dtype": "bf16", "res": "same", "keep": True,
         "train": False},
        # odd rows and columns, full precision, training
        {"name": "norm_train_odd", "op": "norm", "rows": 4099, "cols": 1001,
         "dtype": "fp32", "res": "none", "keep": False, "train": True},
        # DeiT-base training, 256 images a GPU, the stream held in 32 bits
        {"name": "norm_train_base", "op": "norm", "rows": 50432,
         "cols": 768, "dtype": "bf16", "res": "fp32", "keep": True,
         "train": True},
        # one image's MLP in DeiT-tiny
        {"name": "gelu_train_tiny", "op": "gelu", "rows": 197, "cols": 768,
         "dtype": "bf16", "train": True},
        # DeiT-small's MLP, 256 images
        {"name": "gelu_train_small", "op": "gelu", "rows": 50432,
         "cols": 1536, "dtype": "bf16", "train": True},
        # classifier head for one image
        {"name": "linear_one_row", "op": "linear", "rows": 1, "cols": 384,
         "out": 1000, "dtype": "bf16", "act": False, "res": "none",
         "keep": False, "train": False, "density": 0.2},
        # eight images through the attention projection, with its residual
        {"name": "linear_serve_proj", "op": "linear", "rows": 1576,
         "cols": 768, "out": 768, "dtype": "bf16", "act": False,
         "res": "same", "keep": False, "train": False, "density": 0.5},
        # DeiT-small's first MLP product, 256 images: GELU, kept in 8 bits
        {"name": "linear_train_fc1", "op": "linear", "rows": 50432,
         "cols": 384, "out": 1536, "dtype": "bf16", "act": True,
         "res": "none", "keep": True, "train": True, "density": 0.5},
        # its second: residual in 32 bits, no activation
        {"name": "linear_train_fc2", "op": "linear", "rows": 50432,
         "cols": 1536, "out": 384, "dtype": "bf16", "act": False,
         "res": "fp32", "keep": True, "train": True, "density": 0.5},
        # nothing a multiple of a tile, half precision, everything at once
        {"name": "linear_train_odd", "op": "linear", "rows": 2051,
         "cols": 333, "out": 1001, "dtype": "fp16", "act": True,
         "res": "same", "keep": True, "train": True, "density": 0.8},
        # a wide MLP: compute-bound, kept in 16 bits
        {"name": "linear_train_wide", "op": "linear", "rows": 25216,
         "cols": 1024, "out": 4096, "dtype": "bf16", "act": True,
         "res": "none", "keep": False, "train": True, "density": 0.5},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm; every
    other one is rounded to a multiple of 64 where that stays in range."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if v >= 64 and rng.random() < 0.5:
        v = v // 64 * 64
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(("norm", "gelu", "linear"))
    train = rng.random() < 0.6
    if op == "norm":
        cols = _spread(rng, 48, 8192)
        dtype = rng.choice(("bf16", "fp16", "fp32"))
        return {"op": op, "rows": _spread(rng, 1, 38000000 // max(768, cols)),
                "cols": cols, "dtype": dtype,
                "res": rng.choice(("none", "same", "fp32")),
                "keep": rng.random() < 0.5, "train": train}
    if op == "gelu":
        cols = _spread(rng, 48, 8192)
        return {"op": op, "rows": _spread(rng, 1, 77000000 // max(1536, cols)),
                "cols": cols, "dtype": rng.choice(("bf16", "fp16", "fp32")),
                "train": True}
    cols, out = _spread(rng, 48, 4096), _spread(rng, 48, 4096)
    most = min(50432, 25216 * 1024 * 4096 // max(cols * out, 1024 * 1024))
    return {"op": op, "rows": _spread(rng, 1, most), "cols": cols, "out": out,
            "dtype": rng.choice(("bf16", "fp16")),
            "act": rng.random() < 0.5,
            "res": rng.choice(("none", "same", "fp32")),
            "keep": rng.random() < 0.5, "train": train,
            "density": rng.choice((0.2, 0.5, 1.0))}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]
    rows, cols = case["rows"], case["cols"]

    def normal(*shape, std=1.0, mean=0.0, dtype=t):
        v = torch.randn(*shape, generator=gen, device="cuda")
        return v.mul_(std).add_(mean).to(dtype)

    train = case["train"]
    # a few channels of a trained stream are much larger than the others
    loud = 1.0 + 7.0 * (torch.rand(cols, generator=gen, device="cuda")
                        < 0.02)
    s = {"case": case, "x": (normal(rows, cols) * loud).to(t)}
    res = case.get("res", "none")
    if case["op"] == "norm":
        s["weight"] = normal(cols, std=0.2, mean=1.0, dtype=torch.float32)
        s["res"] = None if res == "none" else \
            normal(rows, cols, std=2.0,
                   dtype=torch.float32 if res == "fp32" else t)
        h_type = t if s["res"] is None else s["res"].dtype
        if train:
            s["dy"] = normal(rows, cols)
            s["dh"] = normal(rows, cols, dtype=h_type)
            s["weight"].requires_grad_()
    elif case["op"] == "gelu":
        s["res"] = None
        if train:
            s["dy"] = normal(rows, cols)
    else:
        out = case["out"]
        s["weight"] = normal(out, cols, std=cols ** -0.5)
        s["mask"] = (torch.rand(out, cols, generator=gen, device="cuda")
                     < case["density"]).float()
        # the masked compute weight, which the optimizer step keeps
        s["cache"] = torch.where(s["mask"] != 0, s["weight"],
                                 torch.zeros_like(s["weight"]))
        s["bias"] = normal(out, std=0.1)
        s["res"] = None if res == "none" else \
            normal(rows, out, std=2.0,
                   dtype=torch.float32 if res == "fp32" else t)
        if train:
            s["dy"] = normal(rows, out,
                             dtype=t if s["res"] is None
                             else s["res"].dtype)
            s["weight"].requires_grad_()
            s["bias"].requires_grad_()
    if train:
        s["x"].requires_grad_()
        if s["res"] is not None:
            s["res"].requires_grad_()
    return s


# ------------------------------------------------------------- plain form
def _through_8_bits(v):
    """What 32-bit values along the last axis stand for once held in the
    8-bit format."""
    cols = v.shape[-1]
    pad = -cols % BLOCK
    b = torch.nn.functional.pad(v, (0, pad))
    b = b.reshape(*v.shape[:-1], -1, BLOCK)
    mant, expo = torch.frexp(b.abs().amax(-1, keepdim=True))
    # amax = 2 mant * 2^(expo-1); 2 mant * 2^8 <= 448 where 2 mant <= 1.75
    expo = expo - 9 + (mant > 0.875).to(expo.dtype)
    expo = torch.where(mant == 0, torch.full_like(expo, -126), expo)
    scale = ((expo.clamp(-126, 126) + 127) << 23).view(torch.float32)
    q = (b / scale).to(torch.float8_e4m3fn).float() * scale
    return q.reshape(*v.shape[:-1], -1)[..., :cols]


def _gelu(z):
    return 0.5 * z * (1.0 + torch.erf(z * 0.5 ** 0.5))


def _gelu_slope(z):
    cdf = 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5))
    return cdf + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5


def _plain_norm(s, case):
    x, res, w = s["x"], s["res"], s["weight"].detach()
    t = x.dtype
    # the stream as it is handed on, which is also what is normalised
    h = x.detach() if res is None else \
        (x.detach().float() + res.detach().float()).to(res.dtype)
    hf = h.float()
    r = torch.rsqrt(hf.square().mean(-1, keepdim=True) + 1e-6)
    hat = hf * r
    yf = hat * w
    o = {"y": yf.to(t)}
    if res is not None:
        o["h"] = h
    if case["keep"]:
        o["kept"] = _through_8_bits(yf).bfloat16()
    if case["train"]:
        g = s["dy"].float() * w
        d = r * (g - hat * (g * hat).mean(-1, keepdim=True))
        if res is not None:
            d = d + s["dh"].float()
            o["dres"] = d.to(res.dtype)
        o["dx"] = d.to(t)
        o["dweight"] = (s["dy"].float() * hat).sum(0)
    return o


def _plain_gelu(s, case):
    x = s["x"].detach().float()
    o = {"y": _gelu(x).to(s["x"].dtype)}
    if case["train"]:
        o["dx"] = (s["dy"].float() * _gelu_slope(_through_8_bits(x))
                   ).to(s["x"].dtype)
    return o


def _plain_linear(s, case):
    t = s["x"].dtype
    x, w = s["x"].detach().float(), s["cache"].float()
    res = s["res"]
    z = x @ w.t() + s["bias"].detach().float()
    y = _gelu(z) if case["act"] else z
    if res is not None:
        y = y + res.detach().float()
    o = {"y": y.to(t if res is None else res.dtype)}
    if case["train"]:
        dz = s["dy"].float()
        if res is not None:
            o["dres"] = s["dy"]
        if case["act"]:
            dz = dz * _gelu_slope(_through_8_bits(z) if case["keep"] else z)
        kept = _through_8_bits(x) if case["keep"] else x
        o["dx"] = (dz @ w).to(t)
        o["dweight"] = ((dz.t() @ kept) * s["mask"]).to(t)
        o["dbias"] = dz.sum(0).to(t)
    return o


# ------------------------------------------------------ the framework's way
def _own_norm(s, case):
    from turboprune_amd.ops.norm_act import add_rms_norm
    x, res, w = s["x"], s["res"], s["weight"]
    if not case["train"]:
        with torch.no_grad():
            y, h, kept = add_rms_norm(x, res, w, 1e-6,
                                      keep="e4m3" if case["keep"] else None)
            o = {"y": y}
            if res is not None:
                o["h"] = h
            if case["keep"]:
                o["kept"] = kept.dequantize(torch.bfloat16)
        return o
    y, h, kept = add_rms_norm(x, res, w, 1e-6,
                              keep="e4m3" if case["keep"] else None)
    o = {"y": y.detach()}
    if case["keep"]:
        o["kept"] = kept.dequantize(torch.bfloat16)
    if res is None:
        o["dx"], o["dweight"] = torch.autograd.grad(y, (x, w), s["dy"])
        return o
    o["h"] = h.detach()
    o["dx"], o["dres"], o["dweight"] = torch.autograd.grad(
        (y, h), (x, res, w), (s["dy"], s["dh"]))
    return o


def _own_gelu(s, case):
    from turboprune_amd.ops.norm_act import gelu
    y = gelu(s["x"], keep="e4m3")
    o = {"y": y.detach()}
    if case["train"]:
        o["dx"], = torch.autograd.grad(y, s["x"], s["dy"])
    return o


def _own_linear(s, case):
    from turboprune_amd.ops.functional import masked_linear_act
    x, res = s["x"], s["res"]
    act = "gelu" if case["act"] else None
    if not case["train"]:
        with torch.no_grad():
            return {"y": masked_linear_act(
                x, s["weight"], s["mask"], s["bias"], residual=res, act=act,
                cache=s["cache"])}
    y = masked_linear_act(x, s["weight"], s["mask"], s["bias"], residual=res,
                          act=act, cache=s["cache"],
                          keep="e4m3" if case["keep"] else None)
    leaves = [x, s["weight"], s["bias"]] + ([] if res is None else [res])
    grads = torch.autograd.grad(y, leaves, s["dy"])
    o = {"y": y.detach(), "dx": grads[0], "dweight": grads[1],
         "dbias": grads[2]}
    if res is not None:
        o["dres"] = grads[3]
    return o


def run(state):
    case = state["case"]
    if own:
        return {"norm": _own_norm, "gelu": _own_gelu,
                "linear": _own_linear}[case["op"]](state, case)
    return {"norm": _plain_norm, "gelu": _plain_gelu,
            "linear": _plain_linear}[case["op"]](state, case)


# ------------------------------------------------------------------- work
def work(case):
    b = DTYPES[case["dtype"]].itemsize
    m, k = case["rows"], case["cols"]
    eight = 1.0 + 1.0 / BLOCK        # a code and its share of a scale
    res = {"none": 0, "same": b, "fp32": 4}[case.get("res", "none")]
    if case["op"] == "norm":
        # x, [residual] in; y, [h] out; the 8-bit rows written and read back
        # as values where they are asked for
        per = 2 * b + 2 * res + (2 * eight + b if case["keep"] else 0)
        flops = 5.0
        if case["train"]:
            per += b + b + (3 * res if res else b)   # dy, dx, [dh, h, dres]
            flops += 9.0
        return {"bytes": m * k * per + 4 * k * (2 if case["train"] else 1),
                "flops": m * k * flops}
    if case["op"] == "gelu":
        return {"bytes": m * k * (4 * b + 2 * eight), "flops": m * k * 60.0}
    n = case["out"]
    out = res or b
    size = m * k * b + n * k * b + n * b + m * n * (out + res)
    flops = 2.0 * m * n * k
    if case["train"]:
        kept = eight if case["keep"] else b
        if case["keep"]:             # the kept input, written and read
            size += 2 * m * k * eight
        else:
            size += m * k * b
        if case["act"]:              # the kept pre-activation
            size += 2 * m * n * kept
        size += m * n * out + n * k * b          # dy, w
        size += m * k * b + n * k * (b + 4) + n * b   # dx, dw with its mask
        flops *= 3.0
    return {"bytes": size, "flops": flops}


# -------------------------------------------- the definition, in 64 bits
def _power(e):
    """2^e in 64 bits, exactly, for whole e."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest_e4m3(u):
    """Round to the nearest e4m3 value, ties to the even one: 3 bits behind
    the leading one, and steps of 2^-9 below 2^-6."""
    _, expo = torch.frexp(u)
    step = _power((expo - 1).clamp(min=-6) - 3)
    return torch.round(u / step) * step


def _held(v):
    rows, cols = v.shape
    out = torch.empty_like(v)
    whole = cols // BLOCK * BLOCK
    for part in (slice(0, whole), slice(whole, cols)):
        p = v[:, part]
        if p.shape[1] == 0:
            continue
        p = p.reshape(rows, -1, BLOCK) if part.start == 0 and whole else \
            p.reshape(rows, 1, -1)
        top = p.abs().max(dim=2, keepdim=True).values
        power = torch.ceil(torch.log2(top / 448.0)).clamp(-126, 126)
        # the logarithm may be a hair off where top / 448 is a power
        power = torch.where(top <= 448.0 * _power(power - 1),
                            power - 1, power).clamp(-126, 126)
        power = torch.where(top > 448.0 * _power(power),
                            power + 1, power).clamp(-126, 126)
        unit = _power(power)
        out[:, part] = (_nearest_e4m3(p / unit) * unit).reshape(rows, -1)
    return out


def _phi(z):
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))


def _bell(z):
    return torch.exp(-z * z / 2.0) / math.sqrt(2.0 * math.pi)


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items()
         if isinstance(v, torch.Tensor)}
    op, train = case["op"], case["train"]
    if op == "gelu":
        z = d["x"]
        o = {"y": z * _phi(z)}
        if train:
            q = _held(z)
            o["dx"] = d["dy"] * (_phi(q) + q * _bell(q))
        return o
    if op == "norm":
        res = s["res"]
        h = d["x"] if res is None else \
            (d["x"] + d["res"]).to(res.dtype).double()
        n = case["cols"]
        size = ((h * h).sum(1, keepdim=True) / n + 1e-6).sqrt()
        y = h / size * d["weight"]
        o = {"y": y}
        if res is not None:
            o["h"] = h
        if case["keep"]:
            o["kept"] = _held(y)
        if train:
            gw = d["dy"] * d["weight"]
            dx = gw / size - h * (gw * h).sum(1, keepdim=True) / (n * size ** 3)
            if res is not None:
                dx = dx + d["dh"]
                o["dres"] = dx
            o["dx"] = dx
            o["dweight"] = (d["dy"] * h / size).sum(0)
        return o
    w = torch.where(s["mask"] != 0, d["weight"], torch.zeros_like(d["weight"]))
    z = torch.addmm(d["bias"], d["x"], w.t())
    y = z * _phi(z) if case["act"] else z.clone()
    if s["res"] is not None:
        y += d["res"]
    o = {"y": y}
    if train:
        if s["res"] is not None:
            o["dres"] = d["dy"]
        g = d["dy"]
        if case["act"]:
            q = _held(z) if case["keep"] else z
            g = g * (_phi(q) + q * _bell(q))
        o["dx"] = torch.mm(g, w)
        x = _held(d["x"]) if case["keep"] else d["x"]
        o["dweight"] = torch.where(s["mask"] != 0, torch.mm(g.t(), x),
                                   torch.zeros_like(w))
        o["dbias"] = g.sum(0)
    return o
