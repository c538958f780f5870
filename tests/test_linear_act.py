"""Masked linear layer with bias, GELU and residual in the epilogue, and its
gradients from inputs kept in 16 or 8 bits, against the formulas in 64 bits.

The gradients are taken at the kept values, so the reference reads those back
from the operator (their own distance from the exact ones is tested
separately). Bounds: products of 16-bit values are exact in fp32; a sum of n
of them is off by n 2^-23 of the sum of magnitudes at most, whatever the
matrix instructions' rounding; each rounding to 16 bits adds half a step."""

import math

import pytest
import torch

from turboprune_amd.ops import functional as TF
from turboprune_amd.ops.act8 import Act8, quantize_act8
from turboprune_amd.ops.mask_layers import Conv1dMask, LinearMask
from turboprune_amd.ops.norm_act import add_rms_norm

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
F32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16
ACC = 2.0 ** -23


def half(t):
    return torch.finfo(t).eps / 2


def low(t):
    return 2.0 ** -25 if t == FP16 else 1e-38


def gelu64(z):
    """(value, bound, slope, bound) of the kernel's GELU at z. Its forward
    tail |z| Phi(-|z|) is off by its fit, 5e-6 of itself up to |z| = 4 and 5e-5
    up to 6.5, by 3e-10 behind that, and by the exponent's roundings, below
    8 2^-24 (1 + z^2) of itself; the slope's tail by (1.5e-6 + 1e-7 z^2) of
    itself, see test_act8."""
    cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
    q = 0.5 * torch.special.erfc(z.abs() / math.sqrt(2))
    phi = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    rel = 1.5e-6 + 1e-7 * z * z
    s = cdf + z * phi
    fwd = torch.where(z.abs() <= 4, 5e-6, 5e-5) + 2.0 ** -21 * (1 + z * z)
    return (z * cdf, (z * cdf).abs() * 2.0 ** -22 + z.abs() * q * fwd + 3e-10,
            s, s.abs() * 2.0 ** -22 + (q + z.abs() * phi) * rel)


def make(M, K, N, t=BF16, res=None, dev="cpu", density=0.6, seed=0,
         bias=F32, weight=F32):
    g = torch.Generator().manual_seed(seed)
    d = {"x": torch.randn(M, K, generator=g).to(t),
         "weight": (torch.randn(N, K, generator=g) * 1.5
                    / math.sqrt(K)).to(weight),
         "mask": (torch.rand(N, K, generator=g) < density).float(),
         "bias": None if bias is None
         else (0.3 * torch.randn(N, generator=g)).to(bias),
         "residual": None if res is None
         else (2 * torch.randn(M, N, generator=g)).to(res)}
    d["dy"] = torch.randn(M, N, generator=g).to(res or t)
    return {k: None if v is None else v.to(dev) for k, v in d.items()}


def kept_z(d, t, act, keep, compute):
    """The pre-activation as the operator keeps it."""
    if act is None:
        return None, None
    w = torch.where(d["mask"] != 0, d["weight"],
                    torch.zeros_like(d["weight"])).to(compute)
    x = d["x"].to(compute).reshape(-1, w.shape[1])
    bias = d["bias"]
    if bias is not None and bias.dtype not in (compute, F32):
        bias = bias.to(compute)
    if x.is_cuda:
        from turboprune_amd.ops._backend import extension
        # the same call as the operator's: the order of a sum goes by it
        return extension().linear_act_fwd(x, w, bias, None, True,
                                          2 if keep else 1, bool(keep))[1:3]
    return TF._linear_act_fwd_plain(x, w, bias, None, "gelu",
                                    2 if keep else 1)[1:]


def check(d, t, act=None, keep=None, compute=None):
    leaf = {k: d[k].detach().requires_grad_() for k in
            ("x", "weight", "bias", "residual") if d[k] is not None}
    y = TF.masked_linear_act(
        leaf["x"], leaf["weight"], d["mask"], leaf.get("bias"),
        leaf.get("residual"), act, compute_dtype=compute or t, keep=keep)
    M, N = y.numel() // y.shape[-1], y.shape[-1]
    K = d["x"].shape[-1]
    ot = t if d["residual"] is None else d["residual"].dtype
    assert y.dtype == ot and y.shape == d["x"].shape[:-1] + (N,)
    dbl = lambda v: v.detach().double().cpu()  # noqa: E731
    w = torch.where(d["mask"] != 0, d["weight"],
                    torch.zeros_like(d["weight"])).to(t)
    X, W = dbl(d["x"].to(t)).reshape(M, K), dbl(w)
    B = 0 if d["bias"] is None else dbl(d["bias"])
    R = 0 if d["residual"] is None else dbl(d["residual"]).reshape(M, N)
    z = X @ W.t() + B
    zerr = (K + 4) * ACC * (X.abs() @ W.abs().t() + abs(B))
    if act is None:
        want, tol = z, zerr
    else:
        want, tol, _, _ = gelu64(z)
        tol = tol + 1.13 * zerr            # |slope| < 1.13
    want = want + R
    tol = tol + want.abs() * (half(ot) + ACC) * 1.001 + low(ot)
    if not isinstance(R, int):
        tol = tol + R.abs() * ACC
    got = dbl(y).reshape(M, N)
    assert ((got - want).abs() <= tol).all()

    grads = dict(zip(leaf, torch.autograd.grad(
        y, list(leaf.values()), d["dy"].reshape(y.shape),
        retain_graph=True)))
    for k, v in grads.items():
        assert v.shape == leaf[k].shape and v.dtype == leaf[k].dtype
    G = dbl(d["dy"]).reshape(M, N)
    zk, zs = kept_z(d, t, act, keep, compute or t)
    gerr = G.abs() * half(t)
    if act is not None:
        if keep:
            zq = dbl(Act8(zk, zs).dequantize(F32))
            pad = torch.nn.functional.pad(z.abs() + zerr, (0, -N % 32))
            top = pad.reshape(M, -1, 32).amax(-1)
            top = top.repeat_interleave(32, -1)[:, :N]
            tol = zerr * 1.07 + z.abs() * 2.0 ** -4 + top * 2.0 ** -10 / 223
        else:
            assert zs is None
            zq = dbl(zk)
            tol = zerr + z.abs() * half(t) * 1.001 + low(t)
        assert ((zq - z).abs() <= tol).all()
        _, _, s, serr = gelu64(zq)
        gerr = G.abs() * (s.abs() * half(t) * 1.01 + serr) + low(t)
        G = G * s
    if keep:
        X = dbl(quantize_act8(d["x"].to(t)).dequantize(F32)).reshape(M, K)
        if t == FP16:
            X = X.clamp(-65504, 65504)
    want = G @ W
    tol = gerr @ W.abs() + (N + 4) * ACC * (G.abs() @ W.abs())
    xt = d["x"].dtype
    tol = tol + want.abs() * (half(t) + half(xt)) * 1.01 + low(t)
    assert ((dbl(grads["x"]).reshape(M, K) - want).abs() <= tol).all()
    dead = dbl(d["mask"]) == 0
    want = (G.t() @ X).masked_fill(dead, 0)
    wt = d["weight"].dtype
    tol = gerr.t() @ X.abs() + (M + 4) * ACC * (G.abs().t() @ X.abs())
    tol = tol + want.abs() * half(wt) * 1.001 + low(wt)
    got = dbl(grads["weight"])
    assert ((got - want).abs() <= tol).all() and (got[dead] == 0).all()
    if d["bias"] is not None:
        want = G.sum(0)
        bt = d["bias"].dtype
        serr = 0 if act is None else (dbl(d["dy"]).reshape(M, N).abs()
                                      * gelu64(zq)[3]).sum(0)
        tol = serr + (M + 4) * 2.0 ** -24 * G.abs().sum(0) \
            + want.abs() * half(bt) * 1.001 + low(bt)
        assert ((dbl(grads["bias"]) - want).abs() <= tol).all()
    if d["residual"] is not None:
        assert torch.equal(grads["residual"],
                           d["dy"].reshape(grads["residual"].shape))
    return y


SIZES = [(1, 1, 1), (1, 8, 8), (2, 16, 5), (3, 33, 47), (15, 64, 32),
         (16, 96, 100), (17, 72, 129), (63, 128, 64), (65, 200, 96),
         (127, 63, 130), (130, 136, 257), (197, 192, 192), (200, 333, 1001),
         (257, 64, 65), (1000, 48, 48)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("act,keep,res", [
    (None, None, None), ("gelu", "e4m3", F32), ("gelu", None, BF16)])
def test_sizes(dev, M, K, N, act, keep, res):
    check(make(M, K, N, res=res, dev=dev), BF16, act, keep)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("keep", [None, "e4m3"])
@pytest.mark.parametrize("res", ["none", "same", "fp32"])
def test_types(dev, t, act, keep, res):
    r = {"none": None, "same": t, "fp32": F32}[res]
    check(make(90, 104, 72, t, r, dev), t, act, keep)
    check(make(90, 51, 70, t, r, dev, bias=t, weight=t), t, act, keep)
    check(make(40, 64, 64, t, r, dev, bias=None), t, act, keep)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [
    (5000, 192, 768), (4100, 768, 192), (12608, 384, 384), (3000, 1100, 520),
    (2000, 2048, 1000), (20000, 64, 64), (40, 4096, 4096), (8, 4000, 4000),
    (1, 2048, 1000), (700, 4104, 136)])
@pytest.mark.parametrize("act,keep", [("gelu", "e4m3"), ("gelu", None),
                                      (None, "e4m3")])
def test_larger(M, K, N, act, keep):
    check(make(M, K, N, res=F32, dev="cuda"), BF16, act, keep)


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [None, F32])
@pytest.mark.parametrize("res", [None, BF16, F32])
@pytest.mark.parametrize("M,K,N", [(2000, 2048, 1000), (20000, 200, 40),
                                   (9000, 384, 1536), (41000, 66, 1)])
def test_weight_turned_over(M, K, N, res, bias):
    """Input gradients long enough for it, with a dz pass that does it on the
    way and without one, and narrow outputs."""
    check(make(M, K, N, BF16, res, "cuda", bias=bias), BF16, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("db", [BF16, FP16, F32])
@pytest.mark.parametrize("dw", [BF16, FP16, F32])
def test_gradient_types(db, dw):
    for t in (BF16, FP16):
        check(make(700, 100, 300, t, t, "cuda", bias=db if db in (t, F32)
                   else t, weight=dw), t, "gelu", "e4m3")


@pytest.mark.parametrize("dev", DEVICES)
def test_strides_and_leading_dimensions(dev):
    d = make(24, 80, 40, BF16, F32, dev)
    ref = check(d, BF16, "gelu", "e4m3").detach()
    e = dict(d)
    wide = torch.zeros(24, 200, dtype=BF16, device=dev)
    for at in (8, 3):                       # an aligned slice, and one not
        wide.zero_()[:, at:at + 80] = d["x"]
        e["x"] = wide[:, at:at + 80]
        assert torch.equal(check(e, BF16, "gelu", "e4m3"), ref)
        assert torch.equal(check(e, BF16, "gelu"), ref)
    e["x"] = d["x"].t().contiguous().t()
    assert torch.equal(check(e, BF16, "gelu"), ref)
    e = dict(d, residual=d["residual"].t().contiguous().t())
    assert torch.equal(check(e, BF16, "gelu", "e4m3"), ref)
    e = {k: v.reshape(2, 3, 4, -1) if k in ("x", "residual", "dy") else v
         for k, v in d.items()}
    assert torch.equal(check(e, BF16, "gelu", "e4m3").reshape(24, 40), ref)
    e = dict(d, x=d["x"][:1].expand(24, 80))
    check(e, BF16, "gelu", "e4m3")


@pytest.mark.parametrize("dev", DEVICES)
def test_unusual_arguments(dev):
    """A vector for x, a weight in columns, x as its own residual, a cache
    that asks for gradients, kept rows cut from a larger tensor, a fp16 weight
    under a bf16 product."""
    d = make(1, 40, 24, BF16, F32, dev)
    ref = check(d, BF16, "gelu", "e4m3").detach()
    v = {k: t.reshape(-1) if k in ("x", "residual", "dy") else t
         for k, t in d.items()}
    assert torch.equal(check(v, BF16, "gelu", "e4m3"), ref.reshape(-1))
    d = make(30, 48, 56, BF16, BF16, dev)
    ref = check(d, BF16, "gelu").detach()
    cols = dict(d, weight=d["weight"].t().contiguous().t(),
                mask=d["mask"].t().contiguous().t())
    assert torch.equal(check(cols, BF16, "gelu"), ref)
    d = make(30, 48, 48, BF16, BF16, dev)
    x = d["x"].clone().requires_grad_()
    y = TF.masked_linear_act(x, d["weight"], d["mask"], residual=x,
                             compute_dtype=BF16)
    g, = torch.autograd.grad(y, x, d["dy"])
    two = d["x"].clone().requires_grad_()
    y2 = TF.masked_linear_act(two, d["weight"], d["mask"],
                              residual=d["x"], compute_dtype=BF16)
    h, = torch.autograd.grad(y2, two, d["dy"])
    assert torch.equal(y, y2)
    assert ((g.double() - (h.double() + d["dy"].double())).abs()
            <= (h.abs() + d["dy"].abs()).double() * 2.0 ** -8).all()
    cache = TF.mask_apply(d["weight"], d["mask"], BF16).requires_grad_()
    w = d["weight"].clone().requires_grad_()
    y = TF.masked_linear_act(d["x"], w, d["mask"], cache=cache)
    a, b = torch.autograd.grad(y, (w, cache), d["dy"], allow_unused=True)
    assert a is not None and b is None
    big = quantize_act8(torch.cat((d["x"], d["x"]), 1).reshape(60, 48))
    part = Act8(big.codes[::2], big.scales[::2])
    whole = quantize_act8(d["x"])
    gs = []
    for k in (part, whole):
        y = TF.masked_linear_act(d["x"], w, d["mask"], cache=cache,
                                 keep="e4m3", kept=k)
        gs.append(torch.autograd.grad(y, w, d["dy"])[0])
    assert torch.equal(*gs)
    check(dict(d, weight=d["weight"].half()), BF16, "gelu", "e4m3")


@pytest.mark.parametrize("dev", DEVICES)
def test_cast_inputs_and_cache(dev):
    """A float32 stream into a bfloat16 layer, as under autocast; a cache in
    place of weight and mask."""
    d = make(50, 64, 96, BF16, F32, dev)
    d["x"] = d["x"].float() + 1e-3
    y = check(d, BF16, "gelu", "e4m3")
    cache = TF.mask_apply(d["weight"], d["mask"], BF16)
    wrong = torch.zeros_like(d["weight"])
    leaf = d["x"].clone().requires_grad_()
    got = TF.masked_linear_act(leaf, wrong, d["mask"], d["bias"],
                               d["residual"], "gelu", cache=cache,
                               keep="e4m3")
    assert torch.equal(got, y)
    # without a gradient to come the sum may be taken in another order
    with torch.no_grad():
        x = d["x"].clone().requires_grad_()
        z = TF.masked_linear_act(
            x, d["weight"], d["mask"], d["bias"], d["residual"], "gelu",
            compute_dtype=BF16)
    mag = d["x"].abs().double() @ cache.abs().double().t() + 2
    assert ((z.double() - y.double()).abs()
            <= 2 * 1.13 * 68 * ACC * mag + 8 * ACC).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_without_a_mask(dev):
    d = make(20, 64, 48, BF16, None, dev, density=2.0)
    a = TF.masked_linear_act(d["x"], d["weight"], None, d["bias"],
                             compute_dtype=BF16)
    b = TF.masked_linear_act(d["x"], d["weight"], d["mask"], d["bias"],
                             compute_dtype=BF16)
    assert torch.equal(a, b)
    w = d["weight"].requires_grad_()
    y = TF.masked_linear_act(d["x"], w, None, compute_dtype=BF16)
    g, = torch.autograd.grad(y, w, d["dy"])
    assert (g != 0).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_some_gradients_only(dev):
    d = make(40, 64, 96, BF16, BF16, dev, bias=BF16, weight=BF16)
    names = ("x", "weight", "bias", "residual")
    full = {k: d[k].clone().requires_grad_() for k in names}
    args = lambda v: (v["x"], v["weight"], d["mask"], v["bias"],  # noqa: E731
                      v["residual"], "gelu")
    y = TF.masked_linear_act(*args(full), keep="e4m3")
    ref = dict(zip(names, torch.autograd.grad(y, [full[k] for k in names],
                                              d["dy"])))
    for only in names:
        v = {k: d[k].clone().requires_grad_(k == only) for k in names}
        y = TF.masked_linear_act(*args(v), keep="e4m3")
        g, = torch.autograd.grad(y, v[only], d["dy"])
        assert torch.equal(g, ref[only])
    # an expanded gradient, as a sum's backward gives
    y = TF.masked_linear_act(*args(full), keep="e4m3")
    a = torch.autograd.grad(y, list(full.values()),
                            d["dy"][:1, :1].expand(40, 96),
                            retain_graph=True)
    b = torch.autograd.grad(y, list(full.values()),
                            d["dy"][:1, :1].expand(40, 96).contiguous())
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dev", DEVICES)
def test_kept_from_the_norm(dev):
    """The norm's 8-bit rows in place of a second quantisation: the run of
    operators of a transformer block's MLP."""
    torch.manual_seed(0)
    C, H, M = 96, 200, 70
    x = torch.randn(M, C, device=dev).to(BF16)
    r = torch.randn(M, C, device=dev)
    nw = torch.rand(C, device=dev) + 0.5
    w1 = torch.randn(H, C, device=dev) * C ** -0.5
    w2 = torch.randn(C, H, device=dev) * H ** -0.5
    m1, m2 = ((torch.rand_like(w) < 0.7).float() for w in (w1, w2))
    dy = torch.randn(M, C, device=dev)
    leaves = [t.requires_grad_() for t in (x, r, nw, w1, w2)]

    def block(kept_rows):
        y, h, k = add_rms_norm(x, r, nw, keep="e4m3")
        a = TF.masked_linear_act(y, w1, m1, act="gelu", compute_dtype=BF16,
                                 keep="e4m3", kept=k if kept_rows else None)
        return TF.masked_linear_act(a, w2, m2, residual=h,
                                    compute_dtype=BF16, keep="e4m3")
    out = block(True)
    assert out.dtype == F32
    grads = torch.autograd.grad(out, leaves, dy)

    # the same run in 64 bits, without 8-bit keeping: the kept values are off
    # by 2^-4 at most each, independently, so whole gradients by a few percent
    L = [t.detach().double().requires_grad_() for t in leaves]
    H64 = L[0] + L[1]
    Y = H64 * (H64.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * L[2]
    A = torch.nn.functional.gelu(Y @ (L[3] * m1.double()).t())
    O = A @ (L[4] * m2.double()).t() + H64
    ref = torch.autograd.grad(O, L, dy.double())
    assert (out.double() - O).norm() < 2.0 ** -7 * O.norm()
    for got, want in zip(grads, ref):
        assert (got.double() - want).norm() < 2.0 ** -4 * want.norm()
    # quantising the rounded y instead of y: the same but for ties
    g2 = torch.autograd.grad(block(False), leaves, dy)
    for a, b in zip(grads, g2):
        assert (a.double() - b.double()).norm() < 2.0 ** -4 * b.double().norm()


@pytest.mark.parametrize("dev", DEVICES)
def test_gradient_against_differences(dev):
    """Along random directions, in 64 bits: with 16-bit inputs the gradients
    are those of the exact function up to their own roundings."""
    d = make(30, 40, 24, BF16, F32, dev, bias=F32)
    w = d["weight"].to(BF16).float()
    leaves = [t.clone().requires_grad_() for t in
              (d["x"], w, d["bias"], d["residual"])]
    y = TF.masked_linear_act(leaves[0], leaves[1], d["mask"], leaves[2],
                             leaves[3], "gelu", compute_dtype=BF16)
    grads = torch.autograd.grad(y, leaves, d["dy"])
    base = [t.detach().double() for t in leaves]

    def loss(X, W, B, R):
        z = X @ (W * d["mask"].double()).t() + B
        return ((torch.nn.functional.gelu(z) + R) * d["dy"].double()
                ).sum().item()
    g = torch.Generator().manual_seed(3)
    for k, got in enumerate(grads):
        u = torch.randn(got.shape, generator=g, dtype=torch.float64).to(dev)
        up, down = list(base), list(base)
        up[k], down[k] = base[k] + 1e-6 * u, base[k] - 1e-6 * u
        num = (loss(*up) - loss(*down)) / 2e-6
        # dz, z kept and the gradient are each rounded to bf16 once: 3 2^-9 of
        # the terms' magnitudes at most, times slope' |z| < 1.2
        ana = (got.double() * u).sum().item()
        assert abs(num - ana) < 4 * 2.0 ** -9 * (
            got.double().abs() * u.abs()).sum() + 1e-3


@pytest.mark.parametrize("dev", DEVICES)
def test_bad_values_stay_in_their_row(dev):
    d = make(40, 72, 50, BF16, None, dev)
    ref = TF.masked_linear_act(d["x"], d["weight"], d["mask"], d["bias"],
                               act="gelu", compute_dtype=BF16)
    x = d["x"].clone()
    x[7, 71] = float("nan")
    x[39, 3] = float("inf")
    y = TF.masked_linear_act(x, d["weight"], d["mask"], d["bias"],
                             act="gelu", compute_dtype=BF16)
    rest = [i for i in range(40) if i not in (7, 39)]
    assert torch.equal(y[rest], ref[rest]) and y[7].isnan().all()


@pytest.mark.parametrize("dev", DEVICES)
def test_no_rows(dev):
    d = make(4, 16, 8, BF16, F32, dev)
    x = torch.empty(0, 16, dtype=BF16, device=dev, requires_grad=True)
    w = d["weight"].requires_grad_()
    r = torch.empty(0, 8, device=dev, requires_grad=True)
    y = TF.masked_linear_act(x, w, d["mask"], d["bias"], r, "gelu",
                             compute_dtype=BF16, keep="e4m3")
    assert y.shape == (0, 8) and y.dtype == F32
    gx, gw, gr = torch.autograd.grad(y, (x, w, r), torch.empty_like(y))
    assert gx.shape == (0, 16) and (gw == 0).all() and gr.shape == (0, 8)


def test_refusals():
    x, w, m = torch.randn(4, 16), torch.randn(8, 16), torch.ones(8, 16)
    f = TF.masked_linear_act
    k = quantize_act8(x)
    for err, call in [
            (ValueError, lambda: f(x, torch.randn(8, 17), m)),
            (ValueError, lambda: f(x, w.reshape(8, 16, 1), m)),
            (ValueError, lambda: f(x, w, m[:1])),
            (ValueError, lambda: f(x, w, m, torch.zeros(16))),
            (ValueError, lambda: f(x, w, m, residual=torch.zeros(1, 8))),
            (ValueError, lambda: f(x, w, m, act="relu")),
            (ValueError, lambda: f(x, w, m, keep="fp8")),
            (ValueError, lambda: f(x, w, m, cache=w[:4])),
            (ValueError, lambda: f(x, w, m, kept=k)),
            (ValueError, lambda: f(x, w, m, keep="e4m3",
                                   kept=quantize_act8(x[:2]))),
            (TypeError, lambda: f(x.double(), w, m)),
            (TypeError, lambda: f(x, w.double(), m)),
            (TypeError, lambda: f(x, w, m.bool())),
            (TypeError, lambda: f(x, w, m, residual=torch.zeros(4, 8).half())),
            (TypeError, lambda: f(x, w, m, compute_dtype=torch.float64))]:
        with pytest.raises(err):
            call()


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    x, w = torch.randn(4, 16, device="cuda"), torch.randn(8, 16)
    m = torch.ones(8, 16, device="cuda")
    with pytest.raises(ValueError):
        TF.masked_linear_act(x, w, m)
    with pytest.raises(TypeError):          # float32 products
        TF.masked_linear_act(x, w.cuda(), m)
    from turboprune_amd.ops._backend import extension
    ext = extension()
    xb, wb = x.bfloat16(), w.cuda().bfloat16()
    for bad in (lambda: ext.linear_act_fwd(xb, wb[:, :8], None, None, False,
                                           0, False),
                lambda: ext.linear_act_fwd(xb, wb.half(), None, None, False,
                                           0, False),
                lambda: ext.linear_act_fwd(xb, wb, m[0], None, False, 0,
                                           False),
                lambda: ext.linear_act_fwd(xb, wb, None, xb, False, 0, False),
                lambda: ext.linear_act_fwd(xb[:0], wb, None, None, False, 0,
                                           False),
                lambda: ext.linear_act_bwd(xb, None, None, xb, None, wb,
                                           None, True, None, None),
                lambda: ext.linear_act_bwd(
                    torch.zeros(4, 8, device="cuda").bfloat16(), None, None,
                    xb[:3], None, wb, None, True, torch.float32, None)):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("cls", [LinearMask, Conv1dMask])
def test_layers(dev, cls):
    torch.manual_seed(0)
    layer = cls(in_features=64, out_features=48, bias=True).to(dev)
    layer.set_er_mask(0.5)
    layer.enable_cache(BF16)
    x = torch.randn(5, 7, 64, device=dev, dtype=BF16)
    r = torch.randn(5, 7, 48, device=dev)
    y = layer.fused(x, residual=r, act="gelu", keep="e4m3")
    with torch.no_grad():
        want = torch.nn.functional.gelu(
            x.double() @ layer.weight_masked.squeeze(-1).double().t()
            + layer.bias.double()) + r.double()
    assert (y.double() - want).abs().max() < 1e-4
    y.sum().backward()
    assert layer.weight.grad.shape == layer.weight.shape
    assert (layer.weight.grad[layer.mask == 0] == 0).all()
    assert layer.weight.grad.dtype == F32
    assert layer.bias.grad.shape == (48,)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 32, 33, 48, 63, 64, 65])
@pytest.mark.parametrize("K,N", [(1, 1), (7, 40), (31, 31), (64, 33),
                                 (333, 64), (1024, 1000), (2875, 70)])
def test_few_rows(dev, t, M, K, N):
    """The forward pass alone, as inference calls it, from single rows on."""
    for act, res in (("gelu", F32), (None, None)):
        d = make(M, K, N, t, res, dev, seed=M)
        x = torch.zeros(M, K + 3, dtype=t, device=dev)[:, 1:K + 1]
        x.copy_(d["x"])                       # rows at odd addresses
        with torch.no_grad():
            y = TF.masked_linear_act(x, d["weight"], d["mask"], d["bias"],
                                     d["residual"], act, compute_dtype=t)
        w = torch.where(d["mask"] != 0, d["weight"],
                        torch.zeros_like(d["weight"])).to(t).double()
        X, B = d["x"].double(), d["bias"].double()
        z = X @ w.t() + B
        zerr = (K + 10) * ACC * (X.abs() @ w.abs().t() + B.abs())
        if act is None:
            want, tol = z, zerr
        else:
            want, tol, _, _ = gelu64(z)
            tol = tol + 1.13 * zerr
        if res is not None:
            want = want + d["residual"].double()
            tol = tol + d["residual"].double().abs() * ACC
        tol = tol + want.abs() * (half(y.dtype) + ACC) * 1.001 + low(y.dtype)
        assert ((y.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("M,K,N", [
    (100, 768, 384), (197, 384, 1536), (200, 97, 1100), (256, 300, 2048),
    (128, 64, 4096), (300, 131, 1000), (4096, 34, 31), (4097, 34, 31),
    (16, 72, 9000), (32, 71, 9000), (40, 72, 9000)])
def test_rows_in_groups(dev, t, M, K, N):
    """Few outputs in all, whatever their rows and columns."""
    test_few_rows(dev, t, M, K, N)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("M,K,N", [
    (1, 8, 8), (3, 33, 47), (65, 200, 300), (130, 1000, 700), (70, 64, 2000),
    (5000, 384, 1000), (20000, 72, 400), (52000, 520, 256)])
def test_input_kept_by_the_product(t, M, K, N):
    """The codes that the product writes of its input are quantise_act8's, in
    each of the tile sizes."""
    from turboprune_amd.ops._backend import extension
    d = make(M, K, N, t, None, "cuda")
    x = d["x"] * torch.exp2(torch.randint(-9, 9, (M, 1), device="cuda")).to(t)
    x[M // 2, K // 3] = float("nan")
    x[M // 3, K // 2] = float("inf")
    _, _, _, c, s = extension().linear_act_fwd(
        x, d["weight"].to(t), None, None, False, 0, True)
    ref = quantize_act8(x)
    assert torch.equal(c.view(torch.uint8) & 127,
                       ref.codes.view(torch.uint8) & 127)
    assert torch.equal(c.float().nan_to_num(0), ref.codes.float().nan_to_num(0))
    assert torch.equal(s.view(torch.uint8), ref.scales.view(torch.uint8))


@pytest.mark.gpu
def test_the_same_bits_every_time():
    d = make(9000, 384, 512, BF16, F32, "cuda")
    leaves = [d[k].requires_grad_() for k in ("x", "weight", "bias",
                                              "residual")]
    first = None
    for _ in range(3):
        y = TF.masked_linear_act(leaves[0], leaves[1], d["mask"], leaves[2],
                                 leaves[3], "gelu", compute_dtype=BF16,
                                 keep="e4m3")
        got = (y,) + torch.autograd.grad(y, leaves, d["dy"])
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


@pytest.mark.gpu
def test_two_streams_and_a_graph():
    def setup(seed):
        d = make(600, 192, 256, BF16, F32, "cuda", seed=seed)
        d["leaves"] = [d[k].requires_grad_() for k in
                       ("x", "weight", "bias", "residual")]
        return d

    def step(d):
        x, w, b, r = d["leaves"]
        y = TF.masked_linear_act(x, w, d["mask"], b, r, "gelu",
                                 compute_dtype=BF16, keep="e4m3")
        return (y,) + torch.autograd.grad(y, d["leaves"], d["dy"])
    a, b = setup(1), setup(2)
    ref = [[v.detach().clone() for v in step(t)] for t in (a, b)]
    got = []
    for t in (a, b):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([step(t) for _ in range(10)][-1])
    torch.cuda.synchronize()
    for g, r in zip(got, ref):
        assert all(torch.equal(u, v) for u, v in zip(g, r))
    del got, g
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a)
    names = ("x", "weight", "bias", "residual", "mask", "dy")
    saved = [{k: t[k].detach().clone() for k in names} for t in (a, b)]
    for i in (1, 0, 1):
        with torch.no_grad():
            for k in names:
                a[k].copy_(saved[i][k])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, ref[i]))


@pytest.mark.gpu
def test_rows_past_32_bit_offsets():
    """Outputs and inputs longer than 2^32 bytes: the last rows."""
    M, K, N = 2200000, 64, 1024
    x = torch.zeros(M, K, device="cuda", dtype=BF16)
    d = make(100, K, N, BF16, None, "cuda")
    x[-100:] = d["x"]
    y = TF.masked_linear_act(x, d["weight"], d["mask"], d["bias"],
                             act="gelu", compute_dtype=BF16)
    # a call with gradients: 100 rows alone would be added in another order
    ref = TF.masked_linear_act(d["x"], d["weight"].clone().requires_grad_(),
                               d["mask"], d["bias"], act="gelu",
                               compute_dtype=BF16).detach()
    assert torch.equal(y[-100:], ref)
    assert torch.equal(y[:1].expand(1000, N), y[:1000])
    del y
    w = d["weight"].requires_grad_()
    xr = x.requires_grad_()
    y = TF.masked_linear_act(xr, w, d["mask"], d["bias"], act="gelu",
                             compute_dtype=BF16, keep="e4m3")
    dy = torch.zeros_like(y)
    dy[-100:] = d["dy"]
    dx, dw = torch.autograd.grad(y, (xr, w), dy)
    xs = d["x"].clone().requires_grad_()
    y = TF.masked_linear_act(xs, w, d["mask"], d["bias"], act="gelu",
                             compute_dtype=BF16, keep="e4m3")
    sx, sw = torch.autograd.grad(y, (xs, w), d["dy"])
    assert torch.equal(dx[-100:], sx) and (dx[:-100] == 0).all()
    # other slabs, another order of the same 100 products
    assert (dw - sw).abs().max() <= 104 * ACC * (
        sw.abs().max() * 10 + 1)
