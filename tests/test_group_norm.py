"""Group norm with an activation or an activated gate: the kernels against the
formula in 64 bits, and the refusals.

Bounds, for groups of d channels.  The fp32 mean is off by at most (d / 8 + 16)
2^-24 of the mean of absolute values (8 or more chains of sums), the differences
from it by that and their own rounding, the root of their mean square by half of
(d / 8 + 20) 2^-24 of itself and by what the differences are off, in the mean.  A
bf16 output is rounded once (half a step, 2^-8)."""

import pytest
import torch
from torch.autograd import forward_ad

import trainium_linear_attention_b200 as T
from trainium_linear_attention_b200 import _native as N

gpu = pytest.mark.gpu
EPS = 1e-5
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F = 2.0 ** -20


def make(shape, groups, dtype, gate=True, silu=True, affine=True, wtype=None, seed=0,
         device="cuda"):
    gen = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=gen)

    c = shape[-1]
    s = dict(x=(2 * normal(*shape) + 1).to(dtype), groups=groups, weight=None, bias=None, gate=None,
             activation="silu" if silu else None)
    if affine:
        s.update(weight=(1 + 0.3 * normal(c)).to(wtype or dtype),
                 bias=(0.3 * normal(c)).to(wtype or dtype))
    if gate:
        s["gate"] = normal(*shape).to(dtype)
    return {n: v.to(device) if isinstance(v, torch.Tensor) else v for n, v in s.items()}


def plain(s):
    return {n: v.detach() if isinstance(v, torch.Tensor) else v for n, v in s.items()}


def normed(s):
    """n and the bound of its error, the reciprocal deviations, in 64 bits and groups."""
    x = s["x"].detach().double().unflatten(-1, (s["groups"], -1))
    d = x.shape[-1]
    diff = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(diff.square().mean(-1, keepdim=True) + EPS)
    off = (d / 8 + 18) * 2.0 ** -24 * x.abs().mean(-1, keepdim=True) + 2.0 ** -24 * diff.abs()
    n = diff * rstd
    root = (d / 16 + 14) * 2.0 ** -24 + rstd * (n.abs() * off).mean(-1, keepdim=True)
    return n, 1.1 * (rstd * off + n.abs() * root), rstd


def act(v):
    return v * torch.sigmoid(v)


def slope(v):
    r = torch.sigmoid(v)
    return r * (1 + v * (1 - r))


def terms(s):
    """z, its error's bound, act(gate) (or None)."""
    n, en, _ = normed(s)
    n, en = n.flatten(-2), en.flatten(-2)
    one = torch.ones(1, dtype=torch.float64, device=n.device)
    w = one if s["weight"] is None else s["weight"].detach().double()
    b = 0 * one if s["bias"] is None else s["bias"].detach().double()
    gate = None if s["gate"] is None else s["gate"].detach().double()
    z = n * w + b
    ez = en * w.abs() + 2.0 ** -23 * ((n * w).abs() + b.abs())
    return n, en, w, z, ez, gate


def check_forward(s):
    y = T.group_norm(**plain(s), eps=EPS)
    _, _, _, z, ez, gate = terms(s)
    silu = s["activation"] is not None
    if gate is None:
        want, near = (act(z), 1.1 * ez + F * act(z).abs()) if silu else (z, ez)
    else:
        a = act(gate) if silu else gate
        want, near = z * a, a.abs() * (ez + F * z.abs())
    assert y.dtype == s["x"].dtype and y.is_contiguous()
    assert ((y.double() - want).abs() <= near + HALF[y.dtype] * 1.01 * want.abs()).all()
    return y


SHAPES = [((1, 1), 1), ((3, 8), 1), ((5, 24), 3), ((7, 57 * 7), 7), ((2, 5, 64), 4), ((33, 96), 2),
          ((129, 1024), 16), ((4, 1000), 8), ((3, 1040), 13), ((65, 2048), 4), ((9, 1536), 3),
          ((17, 2047), 1), ((6, 4096), 1), ((5, 8192), 1), ((3, 8184), 2), ((4, 8000), 1),
          ((2, 8191), 1), ((40, 512), 64), ((3, 2, 3, 48), 3), ((1200, 40), 5), ((2, 4096), 128)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_forward(shape, groups, dtype):
    for gate in (True, False):
        check_forward(make(shape, groups, dtype, gate))
        check_forward(make(shape, groups, dtype, gate, silu=False, affine=False, seed=1))
    check_forward(make(shape, groups, dtype, wtype=torch.float32, seed=2))
    s = make(shape, groups, dtype, seed=3)
    check_forward({**s, "weight": None})
    check_forward({**s, "bias": None})


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    s = make((3, 10, 64), 4, dtype, seed=3)
    want = check_forward(s)
    joined = torch.cat([s["x"], s["gate"]], -1)
    turned = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    for change in ({"x": joined[..., :64], "gate": joined[..., 64:]},
                   {"x": turned(s["x"])}, {"gate": turned(s["gate"])},
                   {"x": s["x"].transpose(1, 2).contiguous().transpose(1, 2)},
                   {"weight": torch.stack([s["weight"]] * 2, 1)[:, 0]}):
        assert torch.equal(T.group_norm(**{**s, **change}, eps=EPS), want)
    flat = {**s, "x": s["x"].flatten(0, 1), "gate": s["gate"].flatten(0, 1)}
    assert torch.equal(T.group_norm(**flat, eps=EPS), want.flatten(0, 1))
    one = s["gate"][:, :1].expand(-1, 10, -1)
    assert torch.equal(T.group_norm(**{**s, "gate": one}, eps=EPS),
                       T.group_norm(**{**s, "gate": one.contiguous()}, eps=EPS))
    odd = torch.cat([s["x"][..., :1], s["x"]], -1)[..., 1:]  # summed in another order
    check_forward({**s, "x": odd})
    check_forward({**s, "x": s["x"][0, 0], "gate": s["gate"][0, 0]})
    five = make((2, 3, 2, 5, 16), 2, dtype)
    t = lambda v: v.transpose(1, 3)
    got = T.group_norm(**{**five, "x": t(five["x"]), "gate": t(five["gate"])})
    assert torch.equal(got, T.group_norm(**{**five, "x": t(five["x"]).contiguous(),
                                            "gate": t(five["gate"]).contiguous()}))


@gpu
def test_extremes():
    x = torch.zeros(5, 64, device="cuda")
    x[1] = 1e18
    x[2, ::2] = 1e-18
    x[3, 5] = float("nan")
    x[4] = 1e4
    x[4, ::2] += 1
    y = T.group_norm(x, 2, eps=EPS)
    assert (y[:2] == 0).all() and (y[2].abs() <= 1e-15).all()
    assert torch.isnan(y[3, :32]).all() and (y[3, 32:] == 0).all()
    # differences of 1 on a mean of 10^4 keep their variance: 0.25 in both groups
    want = torch.where(torch.arange(64, device="cuda") % 2 == 0, 0.5, -0.5) / (0.25 + EPS) ** 0.5
    assert ((y[4] - want).abs() <= 2.0 ** -24 * 1e4 * 8).all()
    silu = T.group_norm(torch.randn(4, 64, device="cuda"), 2, gate=torch.full(
        (4, 64), -200.0, device="cuda"), activation="silu")
    assert (silu.abs() <= 1e-30).all()
    assert T.group_norm(torch.zeros(0, 64, device="cuda"), 4).shape == (0, 64)
    w = torch.ones(64, device="cuda").requires_grad_()
    y = T.group_norm(torch.zeros(3, 0, 64, device="cuda"), 4, w)
    assert y.shape == (3, 0, 64) and (torch.autograd.grad(y.sum(), [w])[0] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", SHAPES + [((3000, 96), 2), ((5000, 30), 5),
                                                   ((2500, 1024), 16)])
def test_gradients(shape, groups, dtype):
    for i, (gate, silu, affine) in enumerate([(True, True, True), (False, True, True),
                                              (True, False, False), (False, False, True)]):
        check_gradients(make(shape, groups, dtype, gate, silu, affine,
                             wtype=torch.float32 if i == 1 else None, seed=i))


def check_gradients(s):
    dtype, groups = s["x"].dtype, s["groups"]
    names = [n for n in ("x", "weight", "bias", "gate") if s[n] is not None]
    for n in names:
        s[n].requires_grad_()
    gen = torch.Generator().manual_seed(9)
    up = torch.randn(s["x"].shape, generator=gen).to(dtype).cuda()
    got = dict(zip(names, torch.autograd.grad(T.group_norm(**s, eps=EPS), [s[n] for n in names], up)))
    w64 = {n: s[n].detach().double().requires_grad_() for n in names}
    want = dict(zip(names, torch.autograd.grad(T.ref_group_norm(**{**s, **w64}, eps=EPS),
                                               [w64[n] for n in names], up.double())))
    n, en, w, z, ez, gate = terms(s)
    silu, up = s["activation"] is not None, up.double().abs()
    near = {}
    if gate is None:
        g = up * slope(z).abs() if silu else up
        eg = up * (0.5 * ez + 1.1 * F * (1 + z.abs())) if silu else 0 * up
    else:
        a, d = (act(gate), slope(gate)) if silu else (gate, torch.ones_like(gate))
        near["gate"] = up * (d.abs() * (ez + F * z.abs()) + z.abs() * F * (1 + gate.abs()))
        g, eg = up * a.abs(), F * up * a.abs()
    rows = n.numel() // n.shape[-1]
    many = (rows / 8 + 128) * 2.0 ** -24  # 8 rows or more at a time, then the CTAs' sums
    over = tuple(range(n.dim() - 1))
    near["weight"] = (eg * n.abs() + g * en + many * g * n.abs()).sum(over)
    near["bias"] = (eg + many * g).sum(over)
    split = lambda v: v.unflatten(-1, (groups, -1))
    n, en, g, eg = (split(v) for v in (n, en, (g * w.abs()), (eg * w.abs())))
    _, _, rstd = normed(s)
    d = n.shape[-1]
    mean = lambda v: v.mean(-1, keepdim=True)
    sums = (d / 8 + 20) * 2.0 ** -24
    size = g + mean(g) + n.abs() * mean(g * n.abs())
    e = (eg + mean(eg) + sums * mean(g) + en * mean(g * n.abs())
         + n.abs() * mean(eg * n.abs() + g * en + sums * g * n.abs()) + 4 * 2.0 ** -24 * size)
    # rstd is off by what n is (relatively), times what the result is
    x = split(s["x"].detach().double())
    off = ((d / 16 + 20) * 2.0 ** -24 + rstd * (d / 8 + 18) * 2.0 ** -24 * x.abs().mean(
        -1, keepdim=True))
    near["x"] = (rstd * (e + off * size)).flatten(-2)
    for name in names:
        assert got[name].dtype == s[name].dtype and got[name].shape == s[name].shape
        diff = (got[name].double() - want[name]).abs()
        assert (diff <= near[name] + HALF[got[name].dtype] * 1.01 * want[name].abs()).all(), name


@gpu
@pytest.mark.parametrize("gate", [True, False])
def test_gradients_and_differences(gate):
    """The gradient along a direction against the quotient of the definition's differences in
    64 bits (step 2^-12: off by its square times third derivatives, far below 2^-10)."""
    s = make((6, 48), 3, torch.float32, gate, seed=5)
    names = [n for n in ("x", "weight", "bias", "gate") if s[n] is not None]
    base = {n: v.double() if isinstance(v, torch.Tensor) else v for n, v in s.items()}
    for n in names:
        s[n].requires_grad_()
    gen = torch.Generator().manual_seed(3)
    up = torch.randn(6, 48, generator=gen).cuda()
    grads = torch.autograd.grad(T.group_norm(**s, eps=EPS), [s[n] for n in names], up)
    for n, g in zip(names, grads):
        d = torch.randn(s[n].shape, generator=gen).cuda().double()
        ends = [T.ref_group_norm(**{**base, n: base[n] + h * d}, eps=EPS) * up
                for h in (2.0 ** -12, -2.0 ** -12)]
        quotient = (ends[0] - ends[1]).sum() * 2.0 ** 11
        assert (quotient - (g * d).sum()).abs() <= 2.0 ** -10 * (g * d).abs().sum(), n


@gpu
def test_parts_and_broadcasts():
    s = make((4, 10, 64), 4, torch.bfloat16, seed=7)
    names = ("x", "weight", "bias", "gate")
    for n in names:
        s[n].requires_grad_()
    y = T.group_norm(**s)
    up = torch.randn_like(y)
    every = torch.autograd.grad(y, [s[n] for n in names], up, retain_graph=True)
    for n, g in zip(names, every):
        assert torch.equal(torch.autograd.grad(y, [s[n]], up, retain_graph=True)[0], g)
    a = torch.autograd.grad(y.float().sum(), [s["x"]], retain_graph=True)[0]
    b = torch.autograd.grad(y, [s["x"]], torch.ones_like(y), retain_graph=True)[0]
    assert torch.equal(a, b)
    row = s["gate"].detach()[:, :1].clone().requires_grad_()
    g, = torch.autograd.grad(T.group_norm(**{**s, "gate": row.expand(-1, 10, -1)}), [row], up)
    full = row.detach().expand(-1, 10, -1).contiguous().requires_grad_()
    f, = torch.autograd.grad(T.group_norm(**{**s, "gate": full}), [full], up)
    assert torch.equal(g, f.sum(1, keepdim=True))
    g, = torch.autograd.grad(T.group_norm(s["x"], 4, gate=s["x"]), [s["x"]], up)
    assert torch.isfinite(g).all()  # the same tensor twice
    slices = torch.cat([s["x"], s["gate"]], -1).detach().requires_grad_()
    g, = torch.autograd.grad(T.group_norm(**{**s, "x": slices[..., :64], "gate": slices[..., 64:]}),
                             [slices], up)
    assert torch.equal(g, torch.cat([every[0], every[3]], -1))


@gpu
def test_streams_and_graphs():
    s = make((700, 256), 4, torch.bfloat16, seed=19)
    leaves = [s[n].requires_grad_() for n in ("x", "weight", "bias", "gate")]
    up = torch.randn(700, 256, device="cuda").bfloat16()

    def step():
        y = T.group_norm(**s)
        return [y.detach(), *torch.autograd.grad(y, leaves, up)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals_on_the_cpu():
    s = make((2, 8), 2, torch.float32, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        T.group_norm(**s)
    with pytest.raises(TypeError):
        T.group_norm(**{**s, "groups": 2.0})
    with forward_ad.dual_level():
        x = forward_ad.make_dual(s["x"], s["x"])
        with pytest.raises(NotImplementedError):
            T.group_norm(**{**s, "x": x})
    lib, one, bad = N.lib(), 16, N.LA_ERR_INVALID_ARGUMENT
    strides = (N.ctypes.c_int64 * 2)(8, 8)
    shape = (N.ctypes.c_int64 * 2)(1, 3)
    st, sh = N.ctypes.addressof(strides), N.ctypes.addressof(shape)
    fwd = lambda x=one, c=8, g=2, dtype=0, wd=0, out=one, sh=sh, st=st: lib.la_group_norm_fwd(
        x, st, None, None, None, None, wd, out, None, sh, c, g, 0, dtype, 1e-5, None)
    assert fwd(x=None) == fwd(c=0) == fwd(g=0) == fwd(g=3) == fwd(dtype=5) == fwd(wd=5) == bad
    assert fwd(sh=None) == fwd(st=None) == fwd(out=None) == bad
    assert fwd(c=8193, g=1) == N.LA_ERR_UNSUPPORTED
    assert strides[0] == 8 and shape[1] == 3


def test_c_refuses_pointers_between_elements():
    """Numbers in place of pointers, which no call gets as far as reading."""
    lib, bad = N.lib(), N.LA_ERR_INVALID_ARGUMENT
    strides, shape = (N.ctypes.c_int64 * 2)(8, 8), (N.ctypes.c_int64 * 2)(1, 3)
    st, sh = N.ctypes.addressof(strides), N.ctypes.addressof(shape)

    def fwd(x=16, gate=16, w=16, b=16, out=16, stats=16, dtype=0, wd=0):
        return lib.la_group_norm_fwd(x, st, gate, st, w, b, wd, out, stats, sh, 8, 2, 0, dtype,
                                     1e-5, None)

    assert fwd(x=18) == fwd(gate=18) == fwd(w=18) == fwd(b=18) == fwd(out=18) == bad
    assert fwd(stats=20) == fwd(x=17, dtype=1) == fwd(w=17, wd=1) == bad
    bwd = lambda d=16, dx=16, dg=16, dw=16: lib.la_group_norm_bwd(
        16, st, 16, st, 16, 16, 0, 16, d, st, dx, dg, dw, None, sh, 8, 2, 0, 0, None, 0, None)
    assert bwd(d=18) == bwd(dx=18) == bwd(dg=18) == bwd(dw=18) == bad


@gpu
def test_refusals():
    s = make((2, 5, 8), 2, torch.bfloat16)
    for change, error, text in [
            (dict(groups=3), ValueError, "divide"), (dict(groups=0), ValueError, "divide"),
            (dict(groups=-1), ValueError, "divide"), (dict(x=s["x"].half()), TypeError, "float16"),
            (dict(weight=s["weight"][:4]), ValueError, "weight"),
            (dict(weight=s["weight"].float()), TypeError, "differ"),
            (dict(bias=s["bias"].cpu()), ValueError, "bias"),
            (dict(gate=s["gate"][:1]), ValueError, "gate"),
            (dict(gate=s["gate"].float()), ValueError, "gate"),
            (dict(gate=3), TypeError, "gate"),
            (dict(activation="relu"), ValueError, "activation")]:
        with pytest.raises(error, match=text):
            T.group_norm(**{**s, **change})
    with pytest.raises(N.LaError):
        T.group_norm(torch.zeros(2, 9000, device="cuda"), 1)


@gpu
@pytest.mark.parametrize("shape,groups", [((3, 64), 2), ((5, 33), 1), ((7, 60), 6), ((9, 96), 4),
                                          ((40, 1000), 2), ((3, 2047), 1), ((2, 4096), 1),
                                          ((1200, 40), 5)])
def test_a_common_part_costs_the_gradient_nothing(shape, groups):
    """Values on a grid of 2^-10 below 8, and the same with 2^13 added, are both exact in fp32,
    and so are their differences: outputs and gradients are the same bits."""
    for gate, silu in ((True, True), (False, True), (False, False)):
        s = make(shape, groups, torch.float32, gate, silu, seed=21)
        s["x"] = torch.round(s["x"].clamp(-7, 7) * 1024) / 1024
        names = [n for n in ("x", "weight", "bias", "gate") if s[n] is not None]
        up = torch.randn(shape, generator=torch.Generator().manual_seed(2)).cuda()
        got = []
        for common in (0.0, 8192.0):
            leaves = {n: (s[n] + common if n == "x" else s[n].detach()).requires_grad_()
                      for n in names}
            y = T.group_norm(**{**s, **leaves}, eps=EPS)
            got.append([y.detach(), *torch.autograd.grad(y, list(leaves.values()), up)])
        for n, a, b in zip(["y", *names], *got):
            assert torch.equal(a, b), n


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((3, 48), 2), ((3, 30), 1), ((3, 33), 1), ((2, 1032), 1)])
def test_gradients_of_equal_large_values(shape, groups, dtype):
    """Equal values have n = 0 and rstd = 1 / sqrt(eps) = 316: finite gradients, whatever the
    value (its product with rstd is not), in groups that leave threads without values too."""
    for affine, silu in ((True, True), (False, True), (False, False)):
        s = make(shape, groups, dtype, False, silu, affine, seed=25)
        s["x"] = torch.full_like(s["x"], 2.0 ** 122).requires_grad_()
        y = T.group_norm(**s, eps=EPS)
        up = torch.randn(shape, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
        g, = torch.autograd.grad(y, [s["x"]], up)
        w64 = s["x"].detach().double().requires_grad_()
        args = {n: v.double() if isinstance(v, torch.Tensor) else v for n, v in s.items()}
        want, = torch.autograd.grad(T.ref_group_norm(**{**args, "x": w64}, eps=EPS), [w64],
                                    up.double())
        # up to 1032 terms in a row at most in the mean, a few roundings beside it
        size = 316.3 * 1.6 * 1.1 * up.double().abs().max()
        near = 1100 * 2.0 ** -24 * size + F * size
        assert ((g.double() - want).abs() <= near + HALF[dtype] * 1.01 * want.abs()).all()
