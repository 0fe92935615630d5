"""Root-mean-square norm with the residual's addition, its gradient and its
8-bit form: the kernels against the formula in 64 bits, and the refusals.

Bounds.  The fp32 mean of d squares is off by at most (d / 8 + 16) 2^-24 of it
(8 or more chains of sums), the root by half of that; a product of a few fp32
factors by a few 2^-24.  A bf16 output is rounded once (half a step, 2^-8)."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import trainium_linear_attention_b200 as T
from trainium_linear_attention_b200 import _native as N
from trainium_linear_attention_b200 import ops

gpu = pytest.mark.gpu
EPS = 1e-5
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def relative(d):
    return (d / 8 + 40) * 2.0 ** -24


def make(shape, dtype, residual, weight, seed=0, device="cuda"):
    gen = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=gen)

    x = normal(*shape).to(dtype).to(device)
    r = (normal(*shape) * 2).to(dtype).to(device) if residual else None
    w = None if weight is None else (1 + 0.3 * normal(shape[-1])).to(weight).to(device)
    return x, r, w


def formula(x, w, r):
    s = x.double() if r is None else x.double() + r.double()
    rstd = 1 / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS)
    y = s * rstd
    return (y if w is None else y * w.double()), s, rstd


def check(x, w, r):
    d = x.shape[-1]
    y, total, rstd = ops.rms_norm(x, w, r, EPS, want_rstd=True)
    want, s, want_rstd = formula(x, w, r)
    # the sum of two bf16 or fp32 values is itself rounded to fp32 first
    near = relative(d) * want.abs() + (0 if r is None else 2.0 ** -24 * (
        (x.double().abs() + r.double().abs()) * want_rstd
        * (1 if w is None else w.double().abs())))
    assert ((y.double() - want).abs() <= near * 1.01 + HALF[x.dtype] * want.abs()).all()
    assert ((rstd.double()[..., None] - want_rstd).abs()
            <= 2 * relative(d) * want_rstd).all()
    if r is not None:
        assert torch.equal(total, (x.float() + r.float()).to(x.dtype))
    return y


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [1, 7, 8, 64, 65, 100, 128, 256, 264, 512, 1000, 1024, 2048, 2049,
                               4096, 5000, 5001, 8192, 9003, 16382, 16384])
def test_widths(d, dtype):
    for rows in (1, 5, 33):
        x, r, w = make((rows, d), dtype, rows != 5, dtype if rows != 33 else torch.float32, d)
        check(x, w, r)
        x, _, _ = make((rows, d), dtype, False, None, d)
        check(x, None, None)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    x, r, w = make((2, 5, 33, 64), dtype, True, dtype)
    xt = x.transpose(1, 2)
    y = check(xt, w, None)
    assert y.is_contiguous() and torch.equal(y, ops.rms_norm(xt.contiguous(), w, None, EPS)[0])
    a = ops.rms_norm(xt, w, r.transpose(1, 2), EPS)
    b = ops.rms_norm(xt.contiguous(), w, r.transpose(1, 2).contiguous(), EPS)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    wide = torch.randn(6, 80).to(dtype).cuda()
    for view in (wide[:, :64], wide.T, wide[:1].expand(4, -1), wide[0]):
        y = check(view, None, None)
        assert torch.equal(y, ops.rms_norm(view.contiguous().clone(), None, None, EPS)[0])
    check(wide[:, 1:65], None, None)  # single elements, summed in another order
    five = torch.randn(2, 3, 2, 5, 16).to(dtype).cuda().transpose(1, 3)
    assert torch.equal(ops.rms_norm(five)[0], ops.rms_norm(five.contiguous())[0])


@gpu
def test_extremes():
    x = torch.zeros(4, 64, device="cuda")
    x[1] = 1e18
    x[2] = 1e-18
    x[3, 5] = float("nan")
    y = T.rms_norm(x, eps=EPS)
    assert (y[0] == 0).all() and torch.isfinite(y[:3]).all() and torch.isnan(y[3]).all()
    assert ((y[1] - 1).abs() <= 100 * 2.0 ** -24).all()
    assert T.rms_norm(torch.zeros(0, 64, device="cuda")).shape == (0, 64)
    y, s = T.rms_norm(torch.zeros(3, 0, 64, device="cuda"),
                      residual=torch.zeros(3, 0, 64, device="cuda"))
    assert y.shape == s.shape == (3, 0, 64)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d,residual", [(1, 64, True), (700, 64, False), (4097, 128, True),
                                             (37, 1000, True), (2500, 1024, True), (65, 2049, True),
                                             (9, 8192, False), (3, 16384, True), (5000, 7, True),
                                             (20000, 37, True), (3001, 1279, False),
                                             (1500, 2297, True), (700, 5002, True),
                                             (400, 9003, True)])
def test_gradients(rows, d, residual, dtype):
    x, r, w = make((rows, d), dtype, residual, dtype, rows)
    leaves = [t.requires_grad_() for t in (x, w, r) if t is not None]
    gen = torch.Generator().manual_seed(9)
    dy = torch.randn(rows, d, generator=gen).to(dtype).cuda()
    dt = torch.randn(rows, d, generator=gen).to(dtype).cuda()
    out = T.rms_norm(x, w, residual=r, eps=EPS)
    outs, ups = (out, (dy, dt)) if residual else ((out,), (dy,))
    got = torch.autograd.grad(outs, leaves, ups)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    s = wide[0] if not residual else wide[0] + wide[2]
    y = s / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS) * wide[1]
    loss = (y * dy.double()).sum() + ((s * dt.double()).sum() if residual else 0.0)
    want = torch.autograd.grad(loss, wide)
    s, w64 = s.detach(), wide[1].detach()
    rstd = 1 / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS)
    g = dy.double() * w64
    dot = (g * s).abs().mean(-1, keepdim=True)
    # sizes of the terms: the saved sum is rounded to the dtype with a residual
    held = HALF[dtype] if residual else 0.0
    size = rstd * (g.abs() + s.abs() * rstd * rstd * dot) + (dt.double().abs() if residual else 0)
    through = rstd * s.abs() * rstd * rstd * dot
    near = 4 * relative(d) * size + 2.1 * held * through + HALF[dtype] * want[0].abs()
    assert ((got[0].double() - want[0]).abs() <= 1.01 * near).all()
    if residual:
        assert torch.equal(got[0], got[2])
    size = (dy.double() * s * rstd).abs().sum(0)
    near = (relative(d) + relative(rows) + 1.01 * held) * size + HALF[dtype] * want[1].abs()
    assert ((got[1].double() - want[1]).abs() <= 1.01 * near).all()


@gpu
def test_gradient_against_differences():
    x, r, w = make((6, 96), torch.float32, True, torch.float32)
    leaves = [t.requires_grad_() for t in (x, r, w)]
    gen = torch.Generator().manual_seed(4)
    dy, dt = (torch.randn(6, 96, generator=gen).cuda() for _ in range(2))

    def loss(x, r, w):
        y, s = T.rms_norm(x, w, residual=r, eps=EPS)
        return (y.double() * dy).sum() + (s.double() * dt).sum()

    grads = torch.autograd.grad(loss(*leaves), leaves)
    h = 2.0 ** -7
    for i, t in enumerate(leaves):
        step = torch.randn(t.shape, generator=gen).cuda()
        args = [[u.detach() if j != i else (u + f * h * step).detach()
                 for j, u in enumerate(leaves)] for f in (1, -1)]
        high, low = loss(*args[0]), loss(*args[1])
        slope = (grads[i].double() * step).sum()
        # fp32 rounding of both losses over 2h, and the third derivative's h^2
        size = (dy.abs() * 3).sum() + (dt.abs() * 8).sum()
        cubic = 20 * h * h * step.abs().max() ** 3 * dy.abs().sum()
        assert abs((high - low) / (2 * h) - slope) <= 16 * 2.0 ** -24 / h * size + cubic


@gpu
def test_gradient_parts():
    """Unused outputs, frozen weights, strided and expanded gradients, the same
    tensor as input and residual."""
    x, r, w = make((2, 3, 40, 64), torch.bfloat16, True, torch.bfloat16)
    for t in (x, r, w):
        t.requires_grad_()
    y, s = T.rms_norm(x, w, residual=r, eps=EPS)
    up = torch.randn_like(s)
    assert torch.equal(torch.autograd.grad(s, x, up, retain_graph=True)[0], up)
    dw = torch.autograd.grad(s, w, up, retain_graph=True, allow_unused=True)[0]
    assert dw is None or not dw.any()
    a = torch.autograd.grad(y, (x, w), torch.ones(1, device="cuda").bfloat16().expand_as(y),
                            retain_graph=True)
    b = torch.autograd.grad(y, (x, w), torch.ones_like(y), retain_graph=True)
    c = torch.autograd.grad(y, (x, w), torch.ones(2, 40, 3, 64, device="cuda").bfloat16()
                            .transpose(1, 2))
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and all(
        torch.equal(p, q) for p, q in zip(a, c))
    both, _ = T.rms_norm(x, w.detach(), residual=x, eps=EPS)
    g = torch.autograd.grad(both.float().sum(), x)[0]
    assert g.shape == x.shape and torch.isfinite(g).all()
    empty = torch.zeros(0, 64, device="cuda").bfloat16().requires_grad_()
    dx, dw = torch.autograd.grad(T.rms_norm(empty, w).sum(), (empty, w))
    assert dx.shape == (0, 64) and not dw.any()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d,group", [(1, 1024, None), (33, 64, 16), (33, 64, 64), (5, 100, None),
                                          (40, 4096, 128), (7, 1000, None), (3, 8192, 256),
                                          (3, 16384, 32), (65, 96, 32), (9, 16, 16),
                                          (50, 77, None), (9, 2297, None), (5, 6001, None)])
def test_fp8(rows, d, group, dtype):
    x, r, w = make((rows, d), dtype, True, dtype, rows)
    x[0, :group or d] = 0
    r[0, :group or d] = 0
    got = T.rms_norm_fp8(x, w, residual=r, eps=EPS, group_size=group)
    y8, scales, total = got
    want, s, rstd = formula(x, w, r)
    blocks = want.reshape(rows, -1, group or d)
    amax = blocks.abs().amax(-1).clamp(min=2.0 ** -96)
    near = relative(d) + 2.0 ** -22
    absolute = (x.double().abs() + r.double().abs()) * rstd * (w.double().abs())
    # the sum's own fp32 rounding, as a part of the group's largest value
    lost = 2.0 ** -24 * absolute.reshape(rows, -1, group or d).amax(-1)
    assert scales.shape == (rows, d // (group or d)) and y8.dtype == torch.float8_e4m3fn
    assert ((scales.double() * 448 - amax).abs() <= near * amax + lost).all()
    held = y8.double().reshape(blocks.shape) * scales.double()[..., None]
    # half a step of e4m3: 2^-4 of the value, or half of its smallest step 2^-9
    step = torch.maximum(2.0 ** -4 * blocks.abs(), 2.0 ** -10 * scales.double()[..., None])
    assert ((held - blocks).abs() <= step * (1 + 2 * near) + 2 * near * blocks.abs()
            + lost[..., None]).all()
    assert torch.equal(total, (x.float() + r.float()).to(dtype))
    assert (y8.float()[0, :group or d] == 0).all()
    if group in (None, d):  # odd rows are summed in another order; with groups they are copied
        return
    wide = torch.zeros(rows, d + 1, dtype=dtype, device="cuda")  # rows at odd offsets
    wide[:, 1:] = x
    again = T.rms_norm_fp8(wide[:, 1:], w, residual=r, eps=EPS, group_size=group)
    assert torch.equal(again[0].view(torch.uint8), y8.view(torch.uint8))
    assert torch.equal(again[1], scales)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d", [(1184, 1024), (1185, 1024), (2500, 1000), (592, 2048),
                                    (593, 2040), (1301, 1032), (296, 4096), (297, 4096),
                                    (701, 2056), (1000, 520), (260, 8200)])
def test_many_rows(rows, d, dtype):
    """Around the number of rows from which a thread takes several packs."""
    x, r, w = make((rows, d), dtype, True, dtype, rows)
    check(x, w, r)
    test_gradients(rows, d, True, dtype)
    test_fp8(rows, d, None, dtype)
    if d % 128 == 0:
        test_fp8(rows, d, 128, dtype)


@gpu
def test_fp8_not_finite():
    x = torch.randn(3, 64, device="cuda")
    x[1, 3] = float("nan")
    x[2, 3] = float("inf")
    y, scales = T.rms_norm_fp8(x, group_size=16)
    assert torch.isfinite(scales[0]).all() and torch.isfinite(y[0].float()).all()
    assert torch.isnan(scales[1]).all() and torch.isnan(y[1].float()).all()
    assert torch.isnan(y[2, 3].float())


@gpu
def test_repeats_and_graph():
    x, r, w = make((3000, 1024), torch.bfloat16, True, torch.bfloat16)
    dy = torch.randn_like(x)

    def call():
        y, s, rstd = ops.rms_norm(x, w, r, EPS, want_rstd=True)
        return (y, s, *ops.rms_norm_backward(s, w, rstd, dy, dy),
                *(t.view(torch.uint8) for t in ops.rms_norm_fp8(x, w, r, EPS, 128)[:1]))

    first = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, out))
    assert all(torch.equal(a, b) for a, b in zip(first, call()))


@gpu
def test_streams_and_threads():
    """The same bits on another stream, and from a thread without a context of its
    own, forward, backward and to e4m3, while the default stream works too."""
    import threading

    x, r, w = make((3000, 1024), torch.bfloat16, True, torch.bfloat16)
    dy, ds = torch.randn_like(x), torch.randn_like(x)

    def call():
        y, s, rstd = ops.rms_norm(x, w, r, EPS, want_rstd=True)
        y8, scales, _ = ops.rms_norm_fp8(x, w, r, EPS, 128)
        return (y, s, rstd, *ops.rms_norm_backward(s, w, rstd, dy, ds), y8.view(torch.uint8),
                scales)

    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    others = []
    with torch.cuda.stream(side):
        others.append(call())
    here = call()
    torch.cuda.synchronize()
    worker = threading.Thread(target=lambda: others.append(call()))
    worker.start()
    worker.join()
    torch.cuda.synchronize()
    assert len(others) == 2
    for got in (here, *others):
        assert all(torch.equal(a, b) for a, b in zip(first, got))


# --------------------------------------------------------------------- CPU
def test_refusals():
    x = torch.randn(4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        T.rms_norm(x)
    with pytest.raises(ValueError, match="CUDA"):
        T.rms_norm_fp8(x)
    with pytest.raises(TypeError):
        T.rms_norm([1.0])
    with pytest.raises(ValueError):
        ops._check_rows(torch.zeros(()), "x")
    y, s = T.ref_rms_norm(x.double(), torch.ones(64).double(), x.double(), EPS)
    assert torch.allclose(s, 2 * x.double()) and torch.allclose(
        y.square().mean(-1), torch.ones(4).double(), rtol=1e-4)


def test_forward_mode_is_refused():
    """A dual tensor requires no gradient; its tangent may not be lost."""
    args = make((4, 64), torch.float32, True, torch.float32, device="cpu")
    with forward_ad.dual_level():
        for call in (T.rms_norm, T.rms_norm_fp8):
            for i, x in enumerate(args):
                x, r, w = (*args[:i], forward_ad.make_dual(x, torch.ones_like(x)), *args[i + 1:])
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(x, w, r)
            with pytest.raises(ValueError, match="CUDA"):
                call(args[0], args[2], args[1])  # none of them dual


@gpu
def test_refusals_on_the_gpu():
    x = torch.randn(4, 64, device="cuda")
    for bad in (dict(weight=torch.ones(32, device="cuda")), dict(weight=torch.ones(64)),
                dict(residual=x.bfloat16()), dict(residual=x[:2])):
        with pytest.raises(ValueError):
            T.rms_norm(x, **bad)
    for group in (24, 8, 512, 0):
        with pytest.raises(ValueError, match="group_size"):
            T.rms_norm_fp8(x, group_size=group)
    with pytest.raises(TypeError):
        T.rms_norm(x.half())
    with pytest.raises(T.LaError):
        T.rms_norm(torch.zeros(1, 16385, device="cuda"))


def test_c_entry_points_refuse():
    lib, p = N.lib(), ctypes.c_void_p(256)
    s = (ctypes.c_int64 * 3)(0, 0, 64)

    def shape(*v):
        return (ctypes.c_int64 * 3)(*v)

    def fwd(x=p, xs=s, sh=shape(1, 1, 4), d=64, dtype=1, wtype=1, r=None):
        return lib.la_rms_norm_fwd(x, xs, r, None, None, p, None, None, sh, d, dtype, wtype, 1e-6,
                                   None)

    bad = N.LA_ERR_INVALID_ARGUMENT
    assert fwd(sh=shape(1, -1, 4)) == fwd(d=0) == fwd(dtype=9) == fwd(wtype=-1) == bad
    assert fwd(d=16385) == N.LA_ERR_UNSUPPORTED
    assert fwd(sh=shape(1, 1, 0)) == N.LA_OK
    if torch.cuda.is_available():
        assert fwd(x=None) == fwd(xs=None) == fwd(r=p) == bad
    else:
        assert fwd() == N.LA_ERR_NO_DEVICE
    assert lib.la_rms_norm_bwd_workspace_size(4, 0, ctypes.byref(ctypes.c_size_t(0))) == bad
