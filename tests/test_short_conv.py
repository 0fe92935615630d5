"""Short causal convolution: the kernels against the definition in 64 bits, and the
refusals.

Bounds.  A sum of at most 4 products and a bias is off by 5 2^-24 of the sum of
absolute values; the activation by a few 2^-22 of itself and its slope (at most
1.1) times that.  An output is rounded once (half a step).  Sums over n tokens
for the weights' gradients: at most (n / 8 + 64) 2^-24 of the absolute sum (runs
of 32 tokens, 8 of them joined, then rows of those)."""

import pytest
import torch
from torch.autograd import forward_ad

import trainium_linear_attention_b200 as T
from trainium_linear_attention_b200 import _native as N

gpu = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F = 2.0 ** -20


def make(b, t, c, taps, dtype, bias=True, state=True, lengths=False, silu=True, wtype=None, seed=0,
         device="cuda"):
    gen = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=gen)

    s = dict(x=normal(b, t, c).to(dtype), weight=normal(c, taps).to(wtype or dtype), bias=None,
             activation="silu" if silu else None, initial_state=None, lengths=None)
    if bias:
        s["bias"] = normal(c).to(wtype or dtype)
    if state:
        s["initial_state"] = normal(b, taps - 1, c).to(dtype)
    if lengths:
        s["lengths"] = torch.randint(0, t + 1, (b,), generator=gen)
    return {n: v.to(device) if isinstance(v, torch.Tensor) else v for n, v in s.items()}


def formula(s, absolute=False):
    """z, the windows (b, t, c, taps), which tokens are inside; in 64 bits."""
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    b, t, c = x.shape
    taps = w.shape[1]
    first = (x.new_zeros(b, taps - 1, c) if s["initial_state"] is None
             else s["initial_state"].detach().double())
    win = torch.cat([first, x], 1).unfold(1, taps, 1)
    if absolute:
        win, w = win.abs(), w.abs()
    z = (win * w).sum(-1)
    if s["bias"] is not None:
        z = z + (s["bias"].detach().double().abs() if absolute else s["bias"].detach().double())
    n = (torch.full((b,), t, device=x.device) if s["lengths"] is None
         else s["lengths"].clamp(0, t))
    return z, win, (torch.arange(t, device=x.device) < n[:, None])[..., None], n


def check_forward(s):
    out, state = T.causal_conv(**{n: v.detach() if isinstance(v, torch.Tensor) else v
                                  for n, v in s.items()}, return_state=True)
    z, _, inside, _ = formula(s)
    size, _, _, _ = formula(s, absolute=True)
    want = torch.where(inside, z if s["activation"] is None else z * torch.sigmoid(z), 0.0)
    near = 1.1 * 6 * 2.0 ** -24 * size + F * want.abs()
    assert out.dtype == s["x"].dtype and out.is_contiguous()
    diff = (out.double() - want).abs()
    assert (diff <= torch.where(inside, near + HALF[s["x"].dtype] * 1.01 * want.abs(), 0.0)).all()
    assert torch.equal(state, T.ref_causal_conv(**{
        n: v.detach() if isinstance(v, torch.Tensor) else v for n, v in s.items()})[1])
    return out, state


SIZES = [(1, 1, 1, 2), (2, 1, 5, 4), (1, 2, 64, 4), (1, 3, 64, 4), (3, 8, 33, 3), (2, 9, 66, 4),
         (1, 64, 128, 4), (2, 255, 96, 2), (4, 257, 72, 3), (1, 1024, 64, 4), (2, 2500, 20, 4),
         (300, 7, 64, 4), (1, 700, 1030, 4)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,c,taps", SIZES)
def test_forward(b, t, c, taps, dtype):
    check_forward(make(b, t, c, taps, dtype))
    check_forward(make(b, t, c, taps, dtype, bias=False, state=False, silu=False, seed=1))
    check_forward(make(b, t, c, taps, dtype, lengths=True, wtype=torch.float32, seed=2))


@gpu
def test_long_rows():
    """A tensor beyond 2^31 elements."""
    n, t, c = 2, 40000, 32000
    x = torch.zeros(n, t, c, dtype=torch.bfloat16, device="cuda")
    x[1, -100:, -40:] = torch.randn(100, 40, device="cuda").bfloat16()
    w = torch.randn(c, 4, device="cuda").bfloat16()
    out = T.causal_conv(x, w)
    assert (out[0] == 0).all() and (out[1, :-100] == 0).all()
    small = T.causal_conv(x[1:, -100:, -40:], w[-40:])
    assert torch.equal(out[1, -100:, -40:], small[0])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts_and_padding(dtype):
    s = make(3, 50, 40, 4, dtype, lengths=True, seed=3)
    want, state = check_forward(s)
    x = s["x"]
    for view in (torch.cat([x, x], -1)[..., 40:], torch.cat([x[..., :3], x], -1)[..., 3:],
                 torch.cat([x[..., :2], x], -1)[..., 2:], x.transpose(0, 1).contiguous().transpose(0, 1),
                 x.transpose(1, 2).contiguous().transpose(1, 2)):
        got = T.causal_conv(**{**s, "x": view}, return_state=True)
        assert torch.equal(got[0], want) and torch.equal(got[1], state)
    got = T.causal_conv(**{**s, "weight": s["weight"].t().contiguous().t(),
                           "lengths": s["lengths"].int()}, return_state=True)
    assert torch.equal(got[0], want) and torch.equal(got[1], state)
    behind = (torch.arange(50, device="cuda") >= s["lengths"][:, None])[..., None]
    s["x"] = torch.where(behind, float("nan"), x).requires_grad_()
    out, end = T.causal_conv(**s, return_state=True)
    assert torch.equal(out, want) and torch.equal(end, state)
    g, = torch.autograd.grad(out, [s["x"]], torch.ones_like(out))
    assert (torch.where(behind, g, 0.0) == 0).all() and torch.isfinite(g).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,c,taps", SIZES)
def test_gradients(b, t, c, taps, dtype):
    check_gradients(make(b, t, c, taps, dtype))
    check_gradients(make(b, t, c, taps, dtype, bias=False, state=False, silu=False, seed=1))
    check_gradients(make(b, t, c, taps, dtype, lengths=True, wtype=torch.float32, seed=2))


def check_gradients(s):
    dtype = s["x"].dtype
    b, t, c = s["x"].shape
    taps = s["weight"].shape[1]
    names = [n for n in ("x", "weight", "bias", "initial_state") if s[n] is not None]
    for n in names:
        s[n].requires_grad_()
    out, state = T.causal_conv(**s, return_state=True)
    gen = torch.Generator().manual_seed(5)
    dy = torch.randn(out.shape, generator=gen).to(dtype).cuda()
    ds = torch.randn(state.shape, generator=gen).to(dtype).cuda()
    got = dict(zip(names, torch.autograd.grad((out, state), [s[n] for n in names], (dy, ds))))
    w64 = {n: s[n].detach().double().requires_grad_() for n in names}
    ref = T.ref_causal_conv(**{**s, **w64})
    want = dict(zip(names, torch.autograd.grad(ref, [w64[n] for n in names],
                                               (dy.double(), ds.double()))))
    z, win, inside, n = formula(s)
    size, _, _, _ = formula(s, absolute=True)
    # dz: the activation's slope (below 1.1, itself of slope 0.5 at most) at a z off by ez
    ez = 6 * 2.0 ** -24 * size
    g = torch.where(inside, dy.double().abs(), 0.0)
    if s["activation"] is not None:
        eg = g * (0.5 * ez + 1.1 * F * (1 + z.abs()))
        g = g * 1.1
    else:
        eg = 0.0 * g
    w = s["weight"].detach().double().abs()
    sums = torch.zeros(b, t + taps - 1, c, dtype=torch.float64, device="cuda")
    off = torch.zeros_like(sums)
    for j in range(taps):
        sums[:, j:j + t] += w[:, j] * g
        off[:, j:j + t] += w[:, j] * eg
    at = n[:, None] + torch.arange(taps - 1, device="cuda")
    sums.scatter_add_(1, at[..., None].expand(-1, -1, c), ds.double().abs())
    off = off + 6 * 2.0 ** -24 * sums
    many = (b * t / 8 + 64) * 2.0 ** -24
    near = {"x": off[:, taps - 1:], "initial_state": off[:, :taps - 1],
            "weight": ((eg[..., None] + many * g[..., None]) * win.abs()).sum((0, 1)),
            "bias": (eg + many * g).sum((0, 1))}
    for name in names:
        assert got[name].dtype == s[name].dtype and got[name].shape == s[name].shape
        diff = (got[name].double() - want[name]).abs()
        assert (diff <= near[name] + HALF[got[name].dtype] * 1.01 * want[name].abs()).all(), name


@gpu
def test_gradients_and_differences():
    """The kernel's quotients of differences against its gradients: the outputs are off by
    6 2^-24 of their terms, twice, over a step of 2^-7; the third derivative of the activation
    is below 1, so the quotient is off by step^2 / 6 of the cubes besides."""
    s = make(2, 40, 12, 4, torch.float32, seed=9)
    names = ["x", "weight", "bias", "initial_state"]
    gen = torch.Generator().manual_seed(3)
    up = torch.randn(2, 40, 12, generator=gen).cuda()
    plain = dict(s)
    for n in names:
        s[n] = s[n].clone().requires_grad_()
    grads = dict(zip(names, torch.autograd.grad(T.causal_conv(**s), [s[n] for n in names], up)))
    step = 2.0 ** -7
    for n in names:
        d = torch.rand(s[n].shape, generator=gen).cuda() * 2 - 1
        ends = [T.causal_conv(**{**plain, n: plain[n] + sign * step * d}).double() for sign in (1, -1)]
        quotient = ((ends[0] - ends[1]) * up).sum() / (2 * step)
        slope = (grads[n].double() * d.double()).sum()
        size, win, _, _ = formula(plain, absolute=True)
        w = plain["weight"].double().abs().sum(-1) if n in ("x", "initial_state") else (
            win.sum(-1) if n == "weight" else torch.ones(1, dtype=torch.float64, device="cuda"))
        near = (up.abs() * (8 * 2.0 ** -24 * (size + 1) / step + step ** 2 / 6 * w ** 3)).sum()
        assert (quotient - slope).abs() <= near, n
        assert near <= 0.5 * (grads[n].double() * d.double()).abs().sum() or n == "bias"


@gpu
def test_parts_of_the_gradient():
    s = make(2, 30, 16, 4, torch.bfloat16, seed=13)
    for n in ("x", "weight", "bias", "initial_state"):
        s[n].requires_grad_()
    out, state = T.causal_conv(**s, return_state=True)
    up = torch.randn_like(out)
    every = torch.autograd.grad(out, [s["x"], s["weight"], s["bias"]], up, retain_graph=True)
    for i, n in enumerate(("x", "weight", "bias")):
        assert torch.equal(torch.autograd.grad(out, [s[n]], up, retain_graph=True)[0], every[i])
    gx, gs = torch.autograd.grad(state, [s["x"], s["initial_state"]], torch.ones_like(state),
                                 retain_graph=True)
    assert (gx[:, -3:] == 1).all() and (gx[:, :-3] == 0).all() and (gs == 0).all()
    a = torch.autograd.grad(out.float().sum(), [s["x"]], retain_graph=True)[0]
    b = torch.autograd.grad(out, [s["x"]], torch.ones_like(out), retain_graph=True)[0]
    assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,c,taps", [(1, 1, 2), (1, 4, 4), (5, 7, 3), (3, 64, 4), (257, 130, 4)])
def test_pieces_and_steps(b, c, taps, dtype):
    """Pieces and single tokens give the whole's bits: the sums are the same."""
    s = make(b, 12, c, taps, dtype, seed=17)
    want, end = check_forward(s)
    state, outs, at = s["initial_state"], [], 0
    for n in (1, 6, 0, 2):
        out, state = T.causal_conv(s["x"][:, at:at + n], s["weight"], s["bias"], s["activation"],
                                   state, return_state=True)
        outs.append(out)
        at += n
    wide = torch.zeros(b, taps + 2, c, dtype=dtype, device="cuda")
    wide[:, :taps - 1] = state
    state = wide[:, :taps - 1]
    version = state._version
    for t in range(at, 12):
        outs.append(T.causal_conv_step(s["x"][:, t], s["weight"], state, s["bias"],
                                       s["activation"])[:, None])
    assert state._version > version and (wide[:, taps - 1:] == 0).all()
    assert torch.equal(torch.cat(outs, 1), want) and torch.equal(state, end)


@gpu
def test_empty():
    z = lambda *s: torch.zeros(*s, device="cuda")
    first = torch.randn(2, 3, 5, device="cuda").requires_grad_()
    w = torch.randn(5, 4, device="cuda").requires_grad_()
    out, state = T.causal_conv(z(2, 0, 5), w, initial_state=first, return_state=True)
    assert out.shape == (2, 0, 5) and torch.equal(state, first)
    g, gw = torch.autograd.grad(state, [first, w], torch.ones_like(state))
    assert (g == 1).all() and (gw == 0).all()
    assert (T.causal_conv(z(2, 0, 5), w.detach(), return_state=True)[1] == 0).all()
    y = T.causal_conv(z(0, 3, 5), w)
    assert y.shape == (0, 3, 5) and (torch.autograd.grad(y.sum(), [w])[0] == 0).all()
    assert T.causal_conv_step(z(0, 5), w.detach(), z(0, 3, 5)).shape == (0, 5)
    nothing = T.causal_conv(torch.ones(2, 6, 5, device="cuda"), w.detach(), z(5) + 1, "silu",
                            lengths=torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert (nothing == 0).all()


@gpu
def test_streams_and_graphs():
    s = make(2, 700, 64, 4, torch.bfloat16, seed=19)
    leaves = [s[n].requires_grad_() for n in ("x", "weight", "bias")]
    up = torch.randn(2, 700, 64, device="cuda").bfloat16()

    def step():
        out = T.causal_conv(**s)
        return [out.detach(), *torch.autograd.grad(out, leaves, up)]

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
    s = make(2, 5, 8, 4, torch.float32, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        T.causal_conv(**s)
    with pytest.raises(ValueError, match="CUDA"):
        T.causal_conv_step(s["x"][:, 0], s["weight"], s["initial_state"])
    with forward_ad.dual_level():
        w = forward_ad.make_dual(s["weight"], s["weight"])
        with pytest.raises(NotImplementedError):
            T.causal_conv(**{**s, "weight": w})
    lib, one, bad = N.lib(), 16, N.LA_ERR_INVALID_ARGUMENT
    strides = (N.ctypes.c_int64 * 2)(8, 8)
    st = N.ctypes.addressof(strides)
    fwd = lambda x=one, w=one, out=one, t=1, c=8, taps=4, dtype=0, wd=0, bits=0, lens=None: (
        lib.la_short_conv_fwd(x, st, w, None, wd, None, lens, bits, out, None, 1, t, c, taps, 0,
                              dtype, None))
    assert fwd(x=None) == fwd(w=None) == fwd(c=0) == fwd(dtype=3) == fwd(wd=3) == fwd(t=-1) == bad
    assert fwd(lens=one, bits=8) == bad
    assert fwd(taps=1) == fwd(taps=5) == fwd(c=2 ** 40) == N.LA_ERR_UNSUPPORTED
    step = lambda state=one, stride=24, taps=4: lib.la_short_conv_step(
        one, 8, one, None, 0, state, stride, one, 2, 8, taps, 0, 0, None)
    assert step(state=None) == step(stride=23) == bad
    assert step(taps=7) == N.LA_ERR_UNSUPPORTED
    assert strides[0] == 8


def test_c_refuses_pointers_between_elements():
    """Numbers in place of pointers, which no call gets as far as reading."""
    lib, bad = N.lib(), N.LA_ERR_INVALID_ARGUMENT
    strides = (N.ctypes.c_int64 * 2)(8, 8)
    st = N.ctypes.addressof(strides)
    fwd = lambda x=16, w=16, b=16, init=16, lens=None, dtype=0, wd=0: lib.la_short_conv_fwd(
        x, st, w, b, wd, init, lens, 32, 16, None, 1, 1, 8, 4, 0, dtype, None)
    assert fwd(x=18) == fwd(w=18) == fwd(b=18) == fwd(init=18) == fwd(lens=18) == bad
    assert fwd(x=17, dtype=1) == fwd(w=17, wd=1) == bad
    step = lambda x=16, w=16, state=16, out=16: lib.la_short_conv_step(
        x, 8, w, None, 0, state, 24, out, 2, 8, 4, 0, 0, None)
    assert step(x=18) == step(w=18) == step(state=18) == step(out=18) == bad


@gpu
def test_refusals():
    s = make(2, 5, 8, 4, torch.bfloat16)
    for change, error, text in [
            (dict(weight=None), TypeError, "weight"),
            (dict(weight=s["weight"][:, :1]), ValueError, "taps"),
            (dict(weight=s["weight"][:4]), ValueError, "weight"),
            (dict(weight=s["weight"].cpu()), ValueError, "weight"),
            (dict(weight=s["weight"].float()), TypeError, "differ"),
            (dict(bias=s["bias"][:4]), ValueError, "bias"),
            (dict(activation="gelu"), ValueError, "activation"),
            (dict(initial_state=s["initial_state"][:, :2]), ValueError, "initial_state"),
            (dict(initial_state=s["initial_state"].float()), ValueError, "initial_state"),
            (dict(lengths=torch.ones(3, dtype=torch.int32, device="cuda")), ValueError, "lengths"),
            (dict(x=s["x"].half()), TypeError, "float16")]:
        with pytest.raises(error, match=text):
            T.causal_conv(**{**s, **change})
    with pytest.raises(ValueError, match="dense"):
        T.causal_conv_step(s["x"][:, 0], s["weight"],
                           s["initial_state"].transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(ValueError, match="in place"):
        T.causal_conv_step(s["x"][:, 0], s["weight"], s["initial_state"].clone().requires_grad_())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("silu", [True, False])
def test_infinite_values_end_with_their_sequence(dtype, silu):
    """An infinite last token (or state, of an empty sequence): nothing of it behind the
    sequence, where gradients are zero and from which the weights get nothing."""
    inf = float("inf")
    s = make(5, 70, 40, 4, dtype, silu=silu, seed=31)
    ends = [0, 1, 15, 40, 64]
    s["lengths"] = torch.tensor(ends, device="cuda")
    s["initial_state"][0] = inf
    for i, n in enumerate(ends[1:], 1):
        s["x"][i, n - 1] = inf
    names = ["x", "weight", "bias", "initial_state"]
    for n in names:
        s[n].requires_grad_()
    out, state = T.causal_conv(**s, return_state=True)
    up = torch.randn(out.shape, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    d_state = torch.ones_like(state)
    dx, dw, db, dh = torch.autograd.grad((out, state), [s[n] for n in names], (up, d_state))
    behind = torch.arange(70, device="cuda") >= s["lengths"][:, None]
    assert (out[behind] == 0).all() and (dx[behind] == 0).all()
    assert (dh[0] == 1).all()
    if silu:
        return  # (the slope at an infinite z is 0 * inf, as PyTorch's)
    assert torch.isfinite(dx).all() and torch.isfinite(db).all() and torch.isfinite(dh).all()
    # the last tap alone meets the infinite tokens
    first = s["initial_state"].detach().double()
    whole = torch.cat([first, s["x"].detach().double()], 1).unfold(1, 4, 1)
    g = up.double()[..., None]
    for j in range(3):
        terms = torch.where(behind[..., None], 0.0, whole[..., j] * g[..., 0])
        want, size = terms.sum((0, 1)), terms.abs().sum((0, 1))
        near = (5 * 70 / 8 + 64) * 2.0 ** -24 * size + HALF[dtype] * 1.01 * want.abs()
        assert ((dw[:, j].double() - want).abs() <= near).all()
