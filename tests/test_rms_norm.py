"""Root-mean-square norm with the residual's addition and an 8-bit output,
against its formulas in 64 bits. Bounds: half a step of the output's type,
and n 2^-24 for an fp32 sum of n dependent additions."""

import pytest
import torch

from turboprune_amd.ops.norm_act import FusedRMSNorm, add_rms_norm

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
F32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16
# x, residual (None: without one), output
TYPES = [(F32, None, F32), (F32, F32, F32), (F32, F32, BF16),
         (F32, None, FP16), (BF16, None, BF16), (BF16, BF16, BF16),
         (BF16, F32, BF16), (FP16, FP16, FP16), (FP16, F32, FP16)]
SHAPES = [(1, 1), (3, 7), (1, 48), (9, 128), (5, 129), (17, 192), (4, 333),
          (6, 512), (2, 577), (33, 768), (3, 1001), (5, 2048), (2, 2056),
          (3, 5000), (2, 16384), (2, 16385), (1, 20001)]


def half(t):
    return torch.finfo(t).eps / 2


def low(t):
    """Half a step of the type's subnormals."""
    return 2.0 ** -25 if t == FP16 else 1e-38


def make(rows, C, tx, tr, ty, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, C, generator=g) * 2).to(tx)
    x[:, C // 3] *= 8
    r = None if tr is None else (torch.randn(rows, C, generator=g) * 3).to(tr)
    w = 1 + 0.3 * torch.randn(C, generator=g)
    dy = torch.randn(rows, C, generator=g).to(ty)
    dh = None if tr is None else torch.randn(rows, C, generator=g).to(tr)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    return [to(t) for t in (x, r, w, dy, dh)]


def check(x, r, w, dy, dh, ty, eps=1e-6, keep="e4m3"):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    r = None if r is None else r.detach().requires_grad_()
    y, h, kept = add_rms_norm(x, r, w, eps, keep, ty)
    C = x.shape[-1]
    # the sum handed on: one rounding of an fp32 sum
    if r is None:
        assert h is x
        hd = x.detach()
    else:
        hd = (x.detach().float() + r.detach().float()).to(r.dtype)
        assert h.dtype == r.dtype and torch.equal(h.detach(), hd)
    assert y.dtype == ty and y.shape == x.shape
    H, W = hd.double().cpu(), w.detach().double().cpu()
    rstd = (H.square().mean(-1, keepdim=True) + eps).rsqrt()
    want = H * rstd * W
    # squares: each lane adds at most C/256 + 64 of them one after the other,
    # the join a dozen; rsqrt halves it; a division, rsqrt and two products
    rel = (C / 256 + 76) * 2.0 ** -25 + 6 * 2.0 ** -24
    got = y.detach().double().cpu()
    tol = want.abs() * (rel + half(ty)) * 1.001 + low(ty)
    assert ((got - want).abs() <= tol).all()
    if keep:
        v = kept.dequantize(F32).double().cpu()
        pad = torch.nn.functional.pad(want, (0, -C % 32))
        top = pad.reshape(*want.shape[:-1], -1, 32).abs().amax(-1)
        top = top.repeat_interleave(32, -1)[..., :C]
        # half a step of e4m3; below 2^-6 of the scale 2^-10 of it, and the
        # scale is less than top / 224
        tol = want.abs() * (2.0 ** -4 + 2 * rel) + top * 2.0 ** -10 / 223
        assert ((v - want).abs() <= tol).all()
    else:
        assert kept is None
    outs = [y] if r is None else [y, h]
    gs = [dy] if r is None else [dy, dh]
    leaves = [x, w] + ([] if r is None else [r])
    grads = torch.autograd.grad(outs, leaves, gs)
    G = dy.double().cpu()
    hat, gw = H * rstd, G * W
    m = (gw * hat).mean(-1, keepdim=True)
    d = rstd * (gw - hat * m)
    mag = rstd * (gw.abs() + hat.abs() * (gw * hat).abs().mean(-1, True))
    if r is not None:
        d = d + dh.double().cpu()
        mag = mag + dh.double().cpu().abs()
    # three factors carry the forward's error, the mean its own sum
    err = mag * (4 * rel + (C / 256 + 76) * 2.0 ** -24)
    for got, t in ((grads[0], x.dtype),) + (
            () if r is None else ((grads[2], r.dtype),)):
        assert got.dtype == t and got.shape == x.shape
        tol = err + d.abs() * half(t) * 1.001 + low(t)
        assert ((got.double().cpu() - d).abs() <= tol).all()
    dw = (G * hat).reshape(-1, C).sum(0)
    n = G.numel() // C
    mag = (G * hat).abs().reshape(-1, C).sum(0)
    assert grads[1].dtype == w.dtype
    tol = mag * (2 * rel + (n + 8) * 2.0 ** -24) + dw.abs() * (
        half(w.dtype) if w.dtype != F32 else 0) + 1e-30
    assert ((grads[1].double().cpu() - dw).abs() <= tol).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("rows,C", [(3, 7), (17, 192), (5, 1001)])
def test_types(dev, types, rows, C):
    check(*make(rows, C, *types, dev), types[2])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("rows,C", SHAPES)
@pytest.mark.parametrize("types", [TYPES[0], TYPES[6]], ids=str)
def test_lengths(dev, rows, C, types):
    check(*make(rows, C, *types, dev), types[2])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 4, 5, 63, 1023, 4097, 9000])
@pytest.mark.parametrize("C", [64, 200, 384, 3001])
def test_many_rows(rows, C):
    check(*make(rows, C, BF16, BF16, BF16, "cuda"), BF16, keep=None)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("tw", [BF16, FP16])
def test_weight_types(dev, tw):
    x, r, w, dy, dh = make(40, 96, BF16, BF16, BF16, dev)
    check(x, r, w.to(tw), dy, dh, BF16)


@pytest.mark.parametrize("dev", DEVICES)
def test_strided_rows_and_leading_dimensions(dev):
    x, r, w, dy, dh = make(24, 100, BF16, F32, BF16, dev)
    wide = torch.zeros(24, 260, dtype=BF16, device=dev)
    wide[:, 7:107] = x
    wider = torch.zeros(24, 301, dtype=F32, device=dev)
    wider[:, 1:101] = r
    ref = add_rms_norm(x, r, w, keep="e4m3")
    got = add_rms_norm(wide[:, 7:107], wider[:, 1:101], w, keep="e4m3")
    for a, b in ((got[0], ref[0]), (got[1], ref[1]),
                 (got[2].codes.view(torch.uint8),
                  ref[2].codes.view(torch.uint8)),
                 (got[2].scales.view(torch.uint8),
                  ref[2].scales.view(torch.uint8))):
        assert torch.equal(a, b)
    check(wide[:, 7:107], wider[:, 1:101], w, dy, dh, BF16)
    cols = x.t().contiguous().t()                 # column by column
    assert torch.equal(add_rms_norm(cols, r, w)[0], ref[0])
    one = x[:1].expand(24, 100)                   # one row, shown 24 times
    assert torch.equal(add_rms_norm(one, r, w)[0],
                       add_rms_norm(one.contiguous(), r, w)[0])
    s = (2, 3, 4, 100)
    check(x.reshape(s), r.reshape(s), w, dy.reshape(s), dh.reshape(s), BF16)
    check(x[0], r[0], w, dy[0], dh[0], BF16)      # a vector is one row


@pytest.mark.parametrize("dev", DEVICES)
def test_expanded_gradients_and_unused_outputs(dev):
    x, r, w, _, _ = make(6, 64, BF16, F32, BF16, dev)
    x, r, w = (t.requires_grad_() for t in (x, r, w))
    y, h, _ = add_rms_norm(x, r, w)
    one = torch.ones_like(y)
    a = torch.autograd.grad(y, (x, r, w), one[:1, :1].expand(6, 64),
                            retain_graph=True)
    b = torch.autograd.grad(y, (x, r, w), one, retain_graph=True)
    for u, v in zip(a, b):
        assert torch.equal(u, v)
    # only the sum is used: it is an addition, and the weight takes no part
    gx, gr, gw = torch.autograd.grad(h, (x, r, w), torch.ones_like(h),
                                     allow_unused=True)
    assert (gx == 1).all() and (gr == 1).all() and gw is None


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_of_zeros_and_bad_values(dev):
    x, r, w, dy, dh = make(5, 70, F32, F32, F32, dev)
    x[1] = 0
    r[1] = 0
    ref = add_rms_norm(x, r, w, keep="e4m3")
    assert (ref[0][1] == 0).all()
    assert (ref[2].dequantize()[1] == 0).all()
    check(x, r, w, dy, dh, F32)
    bad = x.clone()
    bad[3, 5] = float("nan")
    bad[4, 6] = float("inf")
    y, _, k = add_rms_norm(bad, r, w, keep="e4m3")
    assert y[3].isnan().all() and k.dequantize()[3].isnan().all()
    assert y[4, 6].isnan() and (y[4, :6] == 0).all()   # inf * 0, x * 0
    assert torch.equal(y[:3], ref[0][:3])


@pytest.mark.parametrize("dev", DEVICES)
def test_no_rows(dev):
    x = torch.empty(0, 64, device=dev, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    y, h, k = add_rms_norm(x, torch.empty(0, 64, device=dev), w, keep="e4m3")
    assert y.shape == h.shape == k.codes.shape == (0, 64)
    gx, gw = torch.autograd.grad(y, (x, w), torch.empty(0, 64, device=dev))
    assert gx.shape == (0, 64) and (gw == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_gradient_against_differences(dev):
    """d/dt of L(x + t u) by central differences in 64 bits, from the
    gradient that the operator returns."""
    x, r, w, dy, dh = make(4, 90, F32, F32, F32, dev)
    leaves = [t.requires_grad_() for t in (x, r, w)]
    y, h, _ = add_rms_norm(x, r, w)
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))

    def loss(X, R, W):
        H = X + R
        Y = H * (H.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * W
        return ((Y * dy.double()).sum() + (H * dh.double()).sum()).item()
    g = torch.Generator().manual_seed(3)
    base = [t.detach().double() for t in leaves]
    for k, got in enumerate(grads):
        u = torch.randn(got.shape, generator=g, dtype=torch.float64).to(dev)
        t = 1e-6
        up, down = list(base), list(base)
        up[k], down[k] = base[k] + t * u, base[k] - t * u
        num = (loss(*up) - loss(*down)) / (2 * t)
        ana = (got.double() * u).sum().item()
        # fp32 gradients: 1e-5 of the terms' magnitudes; cancellation in the
        # loss of ~1e3 over 2e-6: 1e-7
        assert abs(num - ana) < 1e-5 * (got.double() * u).abs().sum() + 1e-5


@pytest.mark.parametrize("dev", DEVICES)
def test_module(dev):
    m = FusedRMSNorm(64, eps=1e-5).to(dev)
    assert list(m.state_dict()) == ["weight"]
    x = torch.randn(3, 5, 64, device=dev)
    with torch.no_grad():
        m.weight.uniform_(0.5, 2.0)
        assert torch.equal(m(x), add_rms_norm(x, None, m.weight, 1e-5)[0])
        y, h, k = m.add(x, x, "e4m3")
        assert torch.equal(h, 2 * x) and k.codes.shape == x.shape
        with torch.autocast(device_type=dev, dtype=BF16):
            assert m(x).dtype == BF16
            assert m.add(x.bfloat16(), x)[1].dtype == F32
    m(x).sum().backward()
    assert m.weight.grad.shape == (64,)


def test_refusals():
    x, w = torch.randn(4, 64), torch.ones(64)
    bf = x.bfloat16()
    for err, call in [
            (ValueError, lambda: add_rms_norm(x, None, torch.ones(63))),
            (ValueError, lambda: add_rms_norm(x, None, torch.ones(1, 64))),
            (ValueError, lambda: add_rms_norm(x, x[:1], w)),
            (ValueError, lambda: add_rms_norm(x, None, w, keep="int8")),
            (ValueError, lambda: add_rms_norm(torch.tensor(1.), None, w)),
            (ValueError, lambda: add_rms_norm(torch.empty(3, 0), None,
                                              torch.empty(0))),
            (TypeError, lambda: add_rms_norm(x.double(), None, w)),
            (TypeError, lambda: add_rms_norm(x, None, w.double())),
            (TypeError, lambda: add_rms_norm(x, bf, w)),
            (TypeError, lambda: add_rms_norm(bf, x.half(), w)),
            (TypeError, lambda: add_rms_norm(bf, None, w, out_dtype=F32)),
            (TypeError, lambda: add_rms_norm(x, None, w,
                                             out_dtype=torch.float64))]:
        with pytest.raises(err):
            call()


@pytest.mark.gpu
def test_refuses_other_devices():
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64)
    with pytest.raises(ValueError):
        add_rms_norm(x, None, w)
    with pytest.raises(ValueError):
        add_rms_norm(x, x.cpu(), w.cuda())


@pytest.mark.gpu
def test_the_same_bits_every_time():
    args = make(5000, 384, BF16, F32, BF16, "cuda")
    x, r, w = (t.requires_grad_() for t in args[:3])
    first = None
    for _ in range(3):
        y, h, _ = add_rms_norm(x, r, w)
        got = torch.autograd.grad((y, h), (x, r, w), args[3:])
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


@pytest.mark.gpu
def test_two_streams_and_a_graph():
    a = make(300, 384, BF16, F32, BF16, "cuda", seed=1)
    b = make(300, 384, BF16, F32, BF16, "cuda", seed=2)

    def step(t):
        y, h, _ = add_rms_norm(t[0], t[1], t[2])
        return (y, h) + torch.autograd.grad((y, h), t[:3], t[3:])
    for t in a[:3] + b[:3]:
        t.requires_grad_()
    ref = [[v.detach().clone() for v in step(t)] for t in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, t in zip(streams, (a, b)):
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
    for t in (b, a, b):
        for dst, src in zip(a, t):
            if dst is not src:
                with torch.no_grad():
                    dst.copy_(src)
        want = [v.detach().clone() for v in step(a)] if t is a else ref[1]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, want))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,C", [(12608, 384), (700, 20000)])
def test_codes_are_those_of_the_formula(rows, C):
    """A code is the one nearest to the formula's value but for one in a
    million. The row's scale is off by half of what the sum's parts of 8 are
    (2^-24 at most each, as often up as down, and 48 of them or more to a
    row): some 2e-9 of a value, and the edges between codes are 1/12 of it
    apart: one in ten million or fewer."""
    x, r, w, _, _ = make(rows, C, BF16, F32, BF16, "cuda")
    _, h, kept = add_rms_norm(x, r, w, keep="e4m3")
    h = h.double()
    y = h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    scale = torch.exp2(kept.scales.view(torch.uint8).double() - 127)
    scale = scale.repeat_interleave(32, -1)[:, :C]
    v = y / scale
    step = torch.exp2(v.abs().log2().floor().clamp(min=-6) - 3)
    want = torch.round(v / step) * step
    got = kept.dequantize(F32).double() / scale
    assert (got != want).sum() <= 1e-6 * y.numel()
    assert ((got - want).abs() <= step).all()
