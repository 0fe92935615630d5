"""Linear attention with a decay for each head: the kernels against the
definition in 64 bits, the gradients against the formulas and differences, and
the refusals.

Bounds.  Let A be the definition applied to |q|, |k|, |v| and |S_0|.  A product
of fp32 sums over at most n terms is off by at most n 2^-24 A; a weight
lambda^m by a few ulp, and by a few more for each tile that carried it.  With
bf16 inputs the weights that multiply v and the state that multiplies q are
rounded once to bf16 (half a step: 2^-8), and so is the output.
"""

import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

import trainium_linear_attention_b200 as T
from trainium_linear_attention_b200 import _native as N
from trainium_linear_attention_b200 import ops

gpu = pytest.mark.gpu


# ------------------------------------------------------------------ definition
def recurrence(q, k, v, g, scale, state):
    """Token by token in float64 (b, h, t, d); returns (out, state)."""
    lam = torch.exp(g.double())[:, None, None]
    outs = []
    for t in range(q.shape[2]):
        state = lam * state + k[:, :, t, :, None] * v[:, :, t, None, :]
        outs.append((q[:, :, t, None, :] @ state).squeeze(-2) * scale)
    out = torch.stack(outs, 2) if outs else q.new_zeros((*q.shape[:2], 0, v.shape[-1]))
    return out, state


def definition(q, k, v, g, scale, state):
    """The same, 64 tokens at a time."""
    outs = []
    for at in range(0, q.shape[2], 64):
        qi, ki, vi = (x[:, :, at:at + 64] for x in (q, k, v))
        out, end = T.ref_decay_attn(qi, ki, vi, g.double(), scale, state)
        outs.append(out)
        state = end
    out = torch.cat(outs, 2) if outs else q.new_zeros((*q.shape[:2], 0, v.shape[-1]))
    return out, state


def bound(dtype, out, absolute, t, d):
    terms = (2 * d + 128 + 8 * (t // 64 + 1) + 64) * 2.0 ** -24
    if dtype == torch.float32 or out.dim() == 0:
        return terms * absolute + 1e-30
    return 2.0 ** -8 * 1.01 * (out.abs() + absolute) + 1e-30


def make(b, h, t, dk, dv, dtype, layout="bhtd", seed=0, device="cuda"):
    gen = torch.Generator().manual_seed(seed)

    def heads(d):
        if layout == "bthd":
            return torch.randn(b, t, h, d, generator=gen).to(dtype).to(device).transpose(1, 2)
        if layout == "sliced":  # rows inside wider ones, an odd token stride
            wide = torch.randn(b, h, t, d + 8, generator=gen).to(dtype).to(device)
            return wide[..., :d]
        if layout == "odd":  # rows that start at no 16-byte boundary
            wide = torch.randn(b, h, t, d + 3, generator=gen).to(dtype).to(device)
            return wide[..., 1:d + 1]
        return torch.randn(b, h, t, d, generator=gen).to(dtype).to(device)

    q, k, v = heads(dk), heads(dk), heads(dv)
    g = -torch.exp2(-8.0 * torch.arange(1, h + 1) / h).float().to(device)
    state = (torch.randn(b, h, dk, dv, generator=gen) * 3).to(device)
    return q, k, v, g, state


def check_forward(q, k, v, g, scale, state, segments=0):
    t, d = q.shape[2], q.shape[3]
    s0 = torch.zeros(*q.shape[:2], d, v.shape[-1], device=q.device) if state is None else state
    out, end = ops.decay_attention(q, k, v, g, scale=scale, initial_state=state,
                                   return_state=True, segments=segments)
    wide = [x.double() for x in (q, k, v)]
    want, want_end = definition(*wide, g, scale, s0.double())
    a_out, a_end = definition(*(x.abs() for x in wide), g, abs(scale), s0.double().abs())
    assert out.dtype == q.dtype and out.shape == want.shape
    assert ((out.double() - want).abs() <= bound(q.dtype, want, a_out, t, d)).all()
    # bf16 inputs: lambda^m k v enters as two bf16 terms, off by 2^-17 of it
    slack = 0.0 if q.dtype == torch.float32 else 2.0 ** -17
    assert ((end.double() - want_end).abs()
            <= bound(torch.float32, want_end, a_end, t, d) + slack * a_end).all()
    return out, end


# --------------------------------------------------------------------- CPU
def test_reference_is_the_recurrence():
    q, k, v, g, state = make(2, 3, 150, 8, 5, torch.float64, device="cpu")
    want = recurrence(q, k, v, g, 0.3, state.double())
    for got in (T.ref_decay_attn(q, k, v, g.double(), 0.3, state.double()),
                definition(q, k, v, g, 0.3, state.double())):
        for x, y in zip(got, want):
            assert (x - y).abs().max() <= 1e-12 * y.abs().max()
    # no memory at all: every token sees itself
    gone = torch.full((3,), float("-inf"), dtype=torch.float64)
    out, end = T.ref_decay_attn(q, k, v, gone, 1.0)
    assert torch.allclose(out, (q * k).sum(-1, keepdim=True) * v, rtol=1e-12, atol=0)
    assert torch.allclose(end, k[:, :, -1, :, None] * v[:, :, -1, None, :], rtol=1e-12, atol=0)


def test_refusals():
    q, k, v, g, state = make(1, 2, 8, 16, 16, torch.float32, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        T.decay_linear_attention(q, k, v, g)
    with pytest.raises(ValueError, match="CUDA"):
        T.decay_linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g, state)
    with pytest.raises(ValueError):
        T.decay_linear_attention_step(q, k, v, g, state)
    with pytest.raises(TypeError):
        T.decay_linear_attention(q, k.double(), v, g)
    for bad in (g[:1], g.double(), g.clone().requires_grad_()):
        with pytest.raises(ValueError, match="log_decay"):
            ops._check_log_decay(bad, 2, q.device)
    with pytest.raises(TypeError):
        ops._check_log_decay(-0.5, 2, q.device)
    with pytest.raises(ValueError, match="state"):
        ops._check_state(state.double(), (1, 2, 16, 16), q.device, "state")


def test_trained_decay_is_refused():
    """Also where other inputs are trained: inside an autograd function gradients
    are off, so the check has to come before it."""
    q, k, v, g, state = make(1, 2, 8, 16, 16, torch.float32, device="cpu")
    g.requires_grad_()
    for i in range(4):
        inputs = [x.clone().requires_grad_(i == j) for j, x in enumerate((q, k, v, state))]
        with pytest.raises(ValueError, match="log_decay"):
            T.decay_linear_attention(*inputs[:3], g, initial_state=inputs[3])
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        T.decay_linear_attention(q, k, v, g)  # the decay itself is accepted


def test_forward_mode_is_refused():
    """A dual tensor requires no gradient; its tangent may not be lost."""
    q, k, v, g, state = make(1, 2, 8, 16, 16, torch.float32, device="cpu")
    calls = [(q, k, v, g, state), tuple(x[:, :, 0] for x in (q, k, v)) + (g, state)]
    with forward_ad.dual_level():
        for call, args in zip((lambda q, k, v, g, s: T.decay_linear_attention(
                q, k, v, g, initial_state=s), T.decay_linear_attention_step), calls):
            for i, x in enumerate(args):
                dual = forward_ad.make_dual(x, torch.ones_like(x))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*args[:i], dual, *args[i + 1:])
            with pytest.raises(ValueError, match="CUDA"):
                call(*args)  # none of them dual


def test_c_entry_points_refuse():
    import ctypes

    from trainium_linear_attention_b200 import _native as N

    lib, p, s = N.lib(), ctypes.c_void_p(256), (ctypes.c_int64 * 3)(1, 1, 1)
    n, ws = ctypes.c_int(0), ctypes.c_size_t(0)
    plan = [ctypes.byref(n), ctypes.byref(ws)]
    assert lib.la_decay_plan(2, 4, 4096, 64, 64, 1, 0, 4, *plan) == N.LA_OK
    assert n.value == 4 and ws.value == 2 * 4 * 4 * 64 * 64 * 4
    assert lib.la_decay_plan(2, 4, 4096, 64, 64, 1, 1, 4, *plan) == N.LA_OK
    assert ws.value == 2 * 2 * 4 * 4 * 64 * 64 * 4
    assert lib.la_decay_plan(2, 4, 100, 64, 64, 1, 0, 4, *plan) == N.LA_OK
    assert n.value == 1 and ws.value == 0
    assert lib.la_decay_plan(2, 4, 4096, 129, 64, 1, 0, 1, *plan) == N.LA_ERR_UNSUPPORTED
    assert lib.la_decay_plan(2, 4, -1, 64, 64, 1, 0, 1, *plan) == N.LA_ERR_INVALID_ARGUMENT
    assert lib.la_decay_plan(1 << 15, 4, 8, 64, 64, 1, 0, 1, *plan) == N.LA_ERR_UNSUPPORTED

    def fwd(q=p, qs=s, dtype=1, b=1, t=8, dk=64, g=p, segments=0):
        return lib.la_decay_chunked_fwd(q, qs, p, s, p, s, p, s, g, b, 2, t, dk, 64, dtype, 1.0,
                                        None, None, None, 0, segments, None)

    assert fwd(q=None) == fwd(qs=None) == fwd(dtype=5) == fwd(g=None) == N.LA_ERR_INVALID_ARGUMENT
    assert fwd(segments=-1) == fwd(dk=0) == N.LA_ERR_INVALID_ARGUMENT
    assert fwd(dk=130) == N.LA_ERR_UNSUPPORTED
    assert fwd(b=0) == fwd(t=0) == N.LA_OK  # nothing to do
    if not torch.cuda.is_available():
        assert fwd() == N.LA_ERR_NO_DEVICE
    assert lib.la_decay_step(p, s, p, s, p, s, p, None, s, p, 1, 2, 64, 64, 1, 1.0, None) == \
        N.LA_ERR_INVALID_ARGUMENT
    assert lib.la_decay_step(p, s, p, s, p, s, p, p, s, p, 0, 2, 64, 64, 1, 1.0, None) == N.LA_OK


# --------------------------------------------------------------------- GPU
WIDTHS = [(16, 64), (24, 32), (32, 128), (64, 64), (128, 128), (64, 128), (40, 72), (128, 8), (57, 33), (1, 1)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t", [1, 2, 63, 64, 65, 127, 128, 129, 300])
def test_lengths(t, dtype):
    q, k, v, g, state = make(2, 3, t, 64, 64, dtype, seed=t)
    check_forward(q, k, v, g, 0.125, state)
    check_forward(q, k, v, g, 0.125, None)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk,dv", WIDTHS)
def test_widths(dk, dv, dtype):
    q, k, v, g, state = make(2, 5, 261, dk, dv, dtype, "bthd", seed=dk + dv)
    check_forward(q, k, v, g, 1.0 / math.sqrt(dk), state)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["bthd", "sliced", "odd"])
def test_layouts(layout, dtype):
    q, k, v, g, state = make(2, 3, 200, 64, 64, dtype, layout)
    out, end = check_forward(q, k, v, g, 0.125, state)
    plain = ops.decay_attention(*(x.contiguous() for x in (q, k, v)), g, scale=0.125,
                                initial_state=state, return_state=True)
    assert torch.equal(out, plain[0]) and torch.equal(end, plain[1])
    if layout == "bthd":
        assert out.transpose(1, 2).is_contiguous()
    # a broadcast head
    one = q[:, :1].expand(-1, 3, -1, -1)
    a = ops.decay_attention(one, k, v, g, scale=0.125)
    assert torch.equal(a, ops.decay_attention(one.contiguous(), k, v, g, scale=0.125))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,segments", [(1000, 2), (1000, 3), (1024, 8), (2049, 5)])
def test_segments(t, segments, dtype):
    q, k, v, g, state = make(1, 4, t, 64, 128, dtype, seed=segments)
    check_forward(q, k, v, g, 0.125, state, segments)
    check_forward(q, k, v, g, 0.125, None, segments)


@gpu
@pytest.mark.parametrize("segments", [2, 3, 8])
@pytest.mark.parametrize("dk,dv", [(128, 64), (128, 128), (64, 128)])
def test_segments_of_wide_heads(dk, dv, segments):
    """Keys or values of 128: the joined state's last two rows lie where the copies
    of the state are written, and every row counts (a large state, slow decays)."""
    q, k, v, _, state = make(2, 4, 2000, dk, dv, torch.bfloat16, "bthd", seed=segments)
    g = torch.tensor([0.0, -1e-4, -1e-3, -1e-2], device="cuda")
    first = check_forward(q, k, v, g, dk ** -0.5, 40 * state, segments)
    again = ops.decay_attention(q, k, v, g, scale=dk ** -0.5, initial_state=40 * state,
                                return_state=True, segments=segments)
    assert all(torch.equal(x, y) for x, y in zip(first, again))
    test_gradients(2000, dk, dv, segments, torch.bfloat16)


@gpu
@pytest.mark.parametrize("dk,dv", [(16, 64), (64, 64), (64, 128), (128, 128)])
@pytest.mark.parametrize("t,segments", [(3, 0), (45, 0), (128, 0), (300, 2), (384, 1), (384, 0)])
def test_final_state_is_held_in_fp32(t, segments, dk, dv):
    """What decoding goes on from, and its gradient, do not keep bf16's roundings.
    In units of 2^-24 of the absolute sums: a weight and each tile that carries it 8
    (expf and its products), the products' split 2 and their sums 16 (8 steps of one
    rounding, cut), joins 6: 56 for three tiles, so 64.  What decays below 2^-16 may
    hold two bf16 terms: 2^-14 of it, 2^-30 of what entered."""
    q, k, v, _, state = make(2, 8, t, dk, dv, torch.bfloat16, "bthd", seed=t)
    g = torch.tensor([-5.0, -1.0, -0.4, -0.1, -0.03, -0.01, -1e-3, 0.0], device="cuda")
    do = torch.randn(v.shape, generator=torch.Generator().manual_seed(1)).to(v.dtype).cuda()
    end = ops.decay_attention(q, k, v, g, initial_state=state, return_state=True,
                              segments=segments)[1]
    first = ops.decay_attention_backward(q, k, v, g, do, scale=0.3, initial_state=state,
                                         d_state=state, want_d_initial=True, segments=segments)[3]
    i = torch.arange(t, device="cuda")
    for got, a, b, left, scale in ((end, k, v, t - 1 - i, 1.0), (first, q, do, i + 1, 0.3)):
        a, b = a.double(), scale * b.double()
        weight = torch.exp(g.double()[:, None] * left)[..., None]

        def total(a, b, s):
            return (torch.exp(g.double() * t)[:, None, None] * s
                    + (a * weight).transpose(-1, -2) @ b)

        s = state.double()
        near = 64 * 2.0 ** -24 * total(a.abs(), b.abs(), s.abs())
        far = 2.0 ** -30 * (a.abs().transpose(-1, -2) @ b.abs())
        assert ((got.double() - total(a, b, s)).abs() <= near + far).all()


@gpu
def test_some_heads_split():
    """More heads than SMs: whole ones fill a wave, the rest share the next in
    segments (the default split; seen by its smaller workspace)."""
    import ctypes

    from trainium_linear_attention_b200 import _native as N

    b, h, t = 4, 16, 4000
    q, k, v, g, state = make(b, h, t, 64, 64, torch.bfloat16, "bthd")
    n, ws = ctypes.c_int(0), ctypes.c_size_t(0)
    assert N.lib().la_decay_plan(b, h, t, 64, 64, 1, 1, 0, ctypes.byref(n), ctypes.byref(ws)) == 0
    every = 2 * b * h * n.value * 64 * 64 * 4
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert n.value > 1 and 0 < ws.value < every
    do, ds = torch.randn_like(v), torch.randn_like(state)
    got = ops.decay_attention_backward(q, k, v, g, do, scale=0.2, initial_state=state, d_state=ds,
                                       want_d_initial=True)
    pick = torch.tensor([0, 17, 48, 49, 55, 63], device="cuda")  # whole and split ones

    def heads(x):
        return x.flatten(0, 1)[pick][None]

    def formulas(absolute):
        leaves = [heads(x).double() for x in (q, k, v, state)]
        up = [heads(x).double() for x in (do, ds)]
        if absolute:
            leaves, up = [x.abs() for x in leaves], [x.abs() for x in up]
        leaves = [x.requires_grad_() for x in leaves]
        out, end = definition(*leaves[:3], g[pick % h], 0.2, leaves[3])
        return torch.autograd.grad((out, end), leaves, up)

    for i, (x, y, a) in enumerate(zip(got, formulas(False), formulas(True))):
        kind = torch.float32 if i == 3 else torch.bfloat16
        slack = 2.0 ** -17 if i == 3 else 0.0
        assert ((heads(x).double() - y).abs() <= bound(kind, y, a, t, 64) + slack * a).all(), i


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decays(dtype):
    """No decay, none of the past, and everything between; an infinite decay is
    the limit of a large one."""
    q, k, v, _, state = make(1, 6, 333, 64, 64, dtype)
    g = torch.tensor([0.0, -1e-4, -0.1, -3.0, -90.0, -200.0], device="cuda")
    check_forward(q, k, v, g, 0.125, state)
    g[4:] = float("-inf")
    out, end = ops.decay_attention(q, k, v, g, scale=0.125, initial_state=state, return_state=True)
    assert torch.isfinite(out).all()
    near = torch.tensor([0.0, -1e-4, -0.1, -3.0, -200.0, -200.0], device="cuda")
    same = ops.decay_attention(q, k, v, near, scale=0.125, initial_state=state, return_state=True)
    assert torch.equal(out, same[0]) and torch.equal(end, same[1])


@gpu
@pytest.mark.parametrize("d", [16, 64, 128])
def test_small_values_under_strong_decays(d):
    """A token's own weight is one however strong the decay: scores of 1e-21 may not
    meet a power of it on the way there.  Gradients scale with d_out (a step of
    bf16 where a sum's last bits change, and what falls below fp32 at 2^-126)."""
    q, k, v, _, state = make(1, 4, 300, d, 64, torch.bfloat16, seed=d)
    g = torch.tensor([-3.95, -3.0, -2.0, -1.0], device="cuda")
    small = 2.0 ** -70
    check_forward(q * small, k, v, g, 0.125, None)
    check_forward(q * small, k, v, g, 0.125, state)
    do = torch.randn(v.shape, generator=torch.Generator().manual_seed(1)).to(v.dtype).cuda()
    grads = [ops.decay_attention_backward(q, k, v, g, up, scale=0.125)[:3]
             for up in (do, do * small)]
    for x, y in zip(*(map(torch.Tensor.double, part) for part in grads)):
        assert ((y / small - x).abs() <= 2.0 ** -7 * x.abs() + 2.0 ** -40 * x.abs().max()).all()


@gpu
def test_empty_and_zero_tokens():
    q, k, v, g, state = make(2, 3, 0, 16, 64, torch.bfloat16)
    out, end = T.decay_linear_attention(q, k, v, g, initial_state=state, return_state=True)
    assert out.shape == (2, 3, 0, 64) and torch.equal(end, state)
    _, end = T.decay_linear_attention(q, k, v, g, return_state=True)
    assert not end.any()
    q, k, v, g, state = make(0, 3, 5, 16, 64, torch.bfloat16)
    assert T.decay_linear_attention(q, k, v, g).shape == (0, 3, 5, 64)
    s = torch.zeros(0, 3, 16, 64, device="cuda")
    assert T.decay_linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g, s).shape == (0, 3, 64)
    q, k, v, g, state = make(2, 3, 0, 57, 33, torch.bfloat16)  # (widened)
    out, end = T.decay_linear_attention(q, k, v, g, initial_state=state, return_state=True)
    assert out.shape == (2, 3, 0, 33) and torch.equal(end, state)
    q, k, v, g, state = make(1, 2, 0, 16, 64, torch.bfloat16)
    state.requires_grad_()
    _, end = T.decay_linear_attention(q, k, v, g, initial_state=state, return_state=True)
    assert torch.equal(torch.autograd.grad(end.sum(), state)[0], torch.ones_like(state))


def test_empty_inputs_have_no_strides():
    """A tensor without elements is contiguous whatever its strides say: a copy
    does not change them, so they are not looked at."""
    for shape in ((2, 3, 0, 16), (0, 3, 5, 16), (2, 0, 5, 16)):
        for x in (torch.zeros(1).expand(shape), torch.zeros(1).bfloat16().expand(shape),
                  torch.zeros(shape[0], shape[1], shape[3], shape[2]).transpose(2, 3)):
            assert ops._heads_strides(x) is not None


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,h,t", [(2, 3, 0), (0, 3, 5), (2, 0, 5)])
def test_empty_inputs_of_any_strides(b, h, t, dtype):
    one = torch.zeros(1, dtype=dtype, device="cuda")
    g = torch.zeros(h, device="cuda")
    state = torch.ones(b, h, 16, 64, device="cuda")
    q, v = one.expand(b, h, t, 16), one.expand(b, h, t, 64)
    out, end = T.decay_linear_attention(q, q, v, g, initial_state=state, return_state=True)
    assert out.shape == (b, h, t, 64) and torch.equal(end, state)
    leaves = [torch.zeros(x.shape, dtype=dtype, device="cuda", requires_grad=True)
              for x in (q, q, v)]
    T.decay_linear_attention(*leaves, g).sum().backward()  # an expanded gradient
    assert all(x.grad.shape == x.shape for x in leaves)
    if t:
        qs, vs = one.expand(b, h, 16), torch.zeros(b, 64, h, dtype=dtype, device="cuda").transpose(1, 2)
        assert T.decay_linear_attention_step(qs, qs, vs, g, state).shape == (b, h, 64)


@gpu
def test_long_sequence_many_tiles():
    """Slow decays over many tiles: the carried state and its power stay exact."""
    q, k, v, g, state = make(1, 2, 20000, 16, 64, torch.float32)
    g = torch.tensor([-1e-4, -2e-3], device="cuda")
    check_forward(q, k, v, g, 0.25, state)
    check_forward(*(x.bfloat16() for x in (q, k, v)), g, 0.25, state)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,dk,dv,segments", [(1, 16, 64, 0), (70, 64, 64, 0), (129, 40, 72, 0),
                                              (300, 128, 64, 0), (1000, 64, 128, 3),
                                              (333, 57, 33, 0), (2049, 64, 64, 5), (700, 24, 32, 3),
                                              (260, 32, 16, 0)])
def test_gradients(t, dk, dv, segments, dtype):
    q, k, v, g, state = make(2, 2, t, dk, dv, dtype, "bthd", seed=t)
    do = torch.randn(2, 2, t, dv, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    ds = torch.randn(2, 2, dk, dv, generator=torch.Generator().manual_seed(2)).cuda()
    got = ops.decay_attention_backward(q, k, v, g, do, scale=0.2, initial_state=state, d_state=ds,
                                       want_d_initial=True, segments=segments)

    def formulas(absolute):
        leaves = [x.double() for x in (q, k, v, state)]
        up = [x.double() for x in (do, ds)]
        if absolute:
            leaves, up = [x.abs() for x in leaves], [x.abs() for x in up]
        leaves = [x.requires_grad_() for x in leaves]
        out, end = definition(*leaves[:3], g, 0.2, leaves[3])
        return torch.autograd.grad((out, end), leaves, up)

    for i, (x, y, a) in enumerate(zip(got, formulas(False), formulas(True))):
        kind = torch.float32 if i == 3 else dtype
        slack = 2.0 ** -17 if i == 3 and dtype == torch.bfloat16 else 0.0
        assert ((x.double() - y).abs() <= bound(kind, y, a, t, max(dk, dv)) + slack * a).all(), i


@gpu
@pytest.mark.parametrize("heads,t,dk,dv,backward", [
    (48, 1024, 64, 64, False), (24, 1000, 64, 64, False), (30, 1023, 128, 128, False),
    (50, 300, 32, 16, False), (40, 1300, 16, 64, False), (16, 1001, 64, 64, True),
    (16, 1024, 32, 24, True), (20, 129, 64, 64, True)])
def test_two_parts(heads, t, dk, dv, backward):
    """Few heads are walked in two parts without a state pass: the same steps as
    one walk, and so the same bits."""
    q, k, v, g, state = make(1, heads, t, dk, dv, torch.bfloat16, "bthd", seed=t)
    n, size = ctypes.c_int(0), ctypes.c_size_t(1)
    assert N.lib().la_decay_plan(1, heads, t, dk, dv, N.LA_DTYPE_BFLOAT16, int(backward), 0,
                                 ctypes.byref(n), ctypes.byref(size)) == N.LA_OK
    assert (n.value, size.value) == (2, 0)
    if backward:
        do = torch.randn(v.shape, generator=torch.Generator().manual_seed(1)).to(v.dtype).cuda()
        ds = torch.randn(state.shape, generator=torch.Generator().manual_seed(2)).cuda()

        def run(segments):
            return ops.decay_attention_backward(q, k, v, g, do, initial_state=state, d_state=ds,
                                                want_d_initial=True, segments=segments)
    else:
        check_forward(q, k, v, g, 0.125, state)

        def run(segments):
            return ops.decay_attention(q, k, v, g, initial_state=state, return_state=True,
                                       segments=segments)
    for x, y in zip(run(0), run(1)):
        assert torch.equal(x, y)


@gpu
@pytest.mark.parametrize("dk,dv", [(57, 33), (20, 100), (3, 5), (125, 60)])
@pytest.mark.parametrize("b,t", [(1, 55), (1, 450), (42, 320), (42, 450), (1, 4097)])
def test_odd_widths(b, t, dk, dv):
    """bf16 widths without 16-byte packs: taken as they are where that is a few
    tiles (the first two), widened where it is more."""
    q, k, v, g, state = make(b, 3, t, dk, dv, torch.bfloat16, seed=t)
    check_forward(q, k, v, g, 0.125, state)
    check_forward(q, k, v, g, 0.125, None)
    if b == 1:
        test_gradients(t, dk, dv, 0, torch.bfloat16)


@gpu
def test_odd_widths_take_their_paths():
    """Which of test_odd_widths' cases are widened; empty inputs never are."""
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the number of tiles that count as few goes by the SMs")
    widened = {  # (d_qk, d_v): forward, backward, by (batch, tokens) below
        (57, 33): ((0, 0, 0, 1, 1), (0, 0, 1, 1, 1)),
        (20, 100): ((0, 0, 1, 1, 1), (0, 0, 1, 1, 1)),
        (3, 5): ((0, 0, 0, 1, 1), (0, 0, 1, 1, 1)),
        (125, 60): ((0, 0, 1, 1, 1), (0, 0, 1, 1, 1))}
    for (dk, dv), want in widened.items():
        for i, (b, t) in enumerate([(1, 55), (1, 450), (42, 320), (42, 450), (1, 4097)]):
            q, k, v, g, _ = make(b, 3, t, dk, dv, torch.bfloat16)
            for up, pads in zip((None, v), want):
                plan = ops._decay_plan(q, k, v, g, None, None, up, 0)
                assert plan.pad == ((-dk % 8, -dv % 8) if pads[i] else None), (dk, dv, b, t)
    q, k, v, g, _ = make(2, 3, 0, 57, 33, torch.bfloat16)
    assert ops._decay_plan(q, k, v, g, None, None, None, 0).pad is None


@gpu
def test_gradients_against_differences():
    """The loss is linear in each input alone, so a central difference of any
    length is the directional derivative, up to the forward pass's rounding."""
    q, k, v, g, state = make(1, 3, 200, 40, 24, torch.float32)
    leaves = [x.clone().requires_grad_() for x in (q, k, v, state)]
    gen = torch.Generator().manual_seed(3)
    do = torch.randn(1, 3, 200, 24, generator=gen).cuda()
    ds = torch.randn(1, 3, 40, 24, generator=gen).cuda()

    def loss(*x):
        out, end = T.decay_linear_attention(*x[:3], g, initial_state=x[3], return_state=True)
        return (out.double() * do).sum() + (end.double() * ds).sum()

    grads = torch.autograd.grad(loss(*leaves), leaves)
    for i, x in enumerate(leaves):
        step = torch.randn(x.shape, generator=gen).cuda()
        up, down = ([y.detach() if j != i else (y + s * step).detach()
                     for j, y in enumerate(leaves)] for s in (1, -1))
        high, low = loss(*up), loss(*down)
        slope = (grads[i].double() * step).sum()
        # both sides are fp32 sums of these sizes
        size = high.abs() + low.abs() + (grads[i].double().abs() * step.abs()).sum()
        assert abs((high - low) / 2 - slope) <= 400 * 2.0 ** -24 * size


@gpu
def test_autograd_needs_and_nones():
    q, k, v, g, state = make(1, 2, 50, 16, 16, torch.bfloat16)
    q.requires_grad_()
    out, end = T.decay_linear_attention(q, k, v, g, initial_state=state, return_state=True)
    only = torch.autograd.grad(end.sum(), q, retain_graph=True, allow_unused=True)[0]
    assert not only.any()  # the final state does not depend on q
    dq = torch.autograd.grad(out.sum(), q)[0]  # an expanded gradient
    want = ops.decay_attention_backward(q.detach(), k, v, g, torch.ones_like(out),
                                        initial_state=state)[0]
    assert torch.equal(dq, want)
    with torch.no_grad():
        assert not T.decay_linear_attention(q, k, v, g).requires_grad
    out = T.decay_linear_attention(q, k, v, g)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(out.sum(), q, create_graph=True)[0].sum(), q)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,h,dk,dv", [(1, 1, 1, 1), (3, 5, 64, 64), (2, 4, 128, 128),
                                       (2, 3, 40, 72), (2, 3, 57, 33), (300, 2, 16, 64)])
def test_step(b, h, dk, dv, dtype):
    q, k, v, g, state = make(b, h, 1, dk, dv, dtype)
    q, k, v = (x[:, :, 0] for x in (q, k, v))
    lam = torch.exp(g.double())[:, None, None]
    want = lam * state.double() + k.double()[..., None] * v.double()[..., None, :]
    held = lam * state.double().abs() + (k.double()[..., None] * v.double()[..., None, :]).abs()
    out_want = (q.double()[..., None, :] @ want).squeeze(-2) * 0.3
    size = (q.double().abs()[..., None, :] @ held).squeeze(-2) * 0.3
    before = state.clone()
    out = T.decay_linear_attention_step(q, k, v, g, state, scale=0.3)
    assert ((state.double() - want).abs() <= 4 * 2.0 ** -24 * held).all()
    last = 2.0 ** -8 * out_want.abs() if dtype == torch.bfloat16 else 0.0
    assert ((out.double() - out_want).abs() <= (dk + 8) * 2.0 ** -24 * size * 1.01 + last).all()
    # a view of a larger pool, strided vectors: the same bits, the rest untouched
    pool = torch.full((b + 2, h, dk, dv), 7.0, device="cuda")
    pool[1:b + 1] = before
    wide = torch.empty(b, h + 1, dk, dtype=dtype, device="cuda")
    wide[:, :h] = q
    again = T.decay_linear_attention_step(wide[:, :h], k, v, g, pool[1:b + 1], scale=0.3)
    assert torch.equal(out, again) and torch.equal(pool[1:b + 1], state)
    assert (pool[0] == 7).all() and (pool[b + 1] == 7).all()


@gpu
def test_step_refuses():
    q, k, v, g, state = make(2, 3, 1, 16, 16, torch.float32)
    q, k, v = (x[:, :, 0] for x in (q, k, v))
    for bad in (state[:1].expand(2, -1, -1, -1), state.transpose(2, 3), state[:, :, :8],
                state.clone().requires_grad_()):
        with pytest.raises(ValueError):
            T.decay_linear_attention_step(q, k, v, g, bad)
    with pytest.raises(ValueError):
        T.decay_linear_attention_step(q, k, v[:1], g, state)
    with pytest.raises(ValueError, match="state"):
        T.decay_linear_attention(*(x[:, :, None] for x in (q, k, v)), g, initial_state=state[:1])
    with pytest.raises(T.LaError):
        T.decay_linear_attention(*(torch.zeros(1, 3, 4, 160, device="cuda"),) * 3, g)
    # the state may not be rewritten under a backward pass that needs it
    q4, k4, v4 = (x[:, :, None].clone().requires_grad_() for x in (q, k, v))
    out = T.decay_linear_attention(q4, k4, v4, g, initial_state=state)
    T.decay_linear_attention_step(q, k, v, g, state)
    with pytest.raises(RuntimeError, match="modified"):
        out.sum().backward()


@gpu
def test_widths_of_zero_are_refused():
    for dk, dv in ((0, 16), (16, 0), (0, 0)):
        q, k, v, g, state = make(1, 2, 3, dk, dv, torch.float32)
        with pytest.raises(T.LaError):
            T.decay_linear_attention(q, k, v, g)
        with pytest.raises((T.LaError, ValueError)):
            T.decay_linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g, state)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_left_padded_batch(dtype):
    """Sequences of different lengths, padded on the left with zero keys, end in
    their own states and outputs."""
    q, k, v, g, _ = make(3, 2, 300, 64, 64, dtype)
    lengths = (300, 131, 1)
    for i, n in enumerate(lengths):
        k[i, :, :300 - n] = 0
    out, end = T.decay_linear_attention(q, k, v, g, scale=0.125, return_state=True)
    for i, n in enumerate(lengths):
        one = [x[i:i + 1, :, 300 - n:].double() for x in (q, k, v)]
        s0 = torch.zeros(1, 2, 64, 64, device="cuda", dtype=torch.float64)
        want, want_end = definition(*one, g, 0.125, s0)
        a_out, a_end = definition(*(x.abs() for x in one), g, 0.125, s0)
        got = out[i:i + 1, :, 300 - n:].double()
        assert ((got - want).abs() <= bound(dtype, want, a_out, 300, 64)).all()
        assert ((end[i:i + 1].double() - want_end).abs()
                <= bound(torch.float32, want_end, a_end, 300, 64) + 2.0 ** -17 * a_end).all()


@gpu
def test_without_gradients():
    """Inference mode, and a decay that some other code trains."""
    q, k, v, g, _ = make(2, 3, 9, 16, 16, torch.bfloat16)
    want = T.decay_linear_attention(q, k, v, g, return_state=True)
    g = g.clone().requires_grad_()
    with pytest.raises(ValueError, match="log_decay"):
        T.decay_linear_attention(q, k, v, g)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            out, state = T.decay_linear_attention(q, k, v, g, return_state=True)
            assert torch.equal(out, want[0]) and torch.equal(state, want[1])
            y = T.decay_linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g, state)
            assert torch.isfinite(y).all()


@gpu
def test_step_refuses_a_trained_decay_always():
    """Also after the same call without gradients, whose checks are kept."""
    q, k, v, g, state = make(1, 2, 1, 16, 24, torch.float32)
    q, k, v = (x[:, :, 0] for x in (q, k, v))
    g.requires_grad_()
    with torch.no_grad():
        T.decay_linear_attention_step(q, k, v, g, state)
    before = state.clone()
    with pytest.raises(ValueError, match="log_decay"):
        T.decay_linear_attention_step(q, k, v, g, state)
    assert torch.equal(state, before)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_in_pieces_then_tokens(dtype):
    """A prompt read at once, in pieces, and token by token end in one state."""
    q, k, v, g, _ = make(2, 4, 300, 64, 64, dtype)
    whole, end = check_forward(q, k, v, g, 0.125, None)
    state, outs = None, []
    for a, b in ((0, 100), (100, 101), (101, 290)):
        out, state = T.decay_linear_attention(q[:, :, a:b], k[:, :, a:b], v[:, :, a:b], g,
                                              initial_state=state, return_state=True)
        outs.append(out)
    for t in range(290, 300):
        outs.append(T.decay_linear_attention_step(q[:, :, t], k[:, :, t], v[:, :, t], g,
                                                  state)[:, :, None])
    got = torch.cat(outs, 2).double()
    wide = [x.double() for x in (q, k, v)]
    s0 = torch.zeros(2, 4, 64, 64, device="cuda", dtype=torch.float64)
    want, want_end = definition(*wide, g, 0.125, s0)
    a_out, a_end = definition(*(x.abs() for x in wide), g, 0.125, s0)
    assert ((got - want).abs() <= bound(dtype, want, a_out, 300, 64)).all()
    assert ((state.double() - want_end).abs()
            <= bound(torch.float32, want_end, a_end, 300, 64) + 2.0 ** -17 * a_end).all()


@gpu
def test_first_call_of_a_thread():
    """A thread without a CUDA context of its own (as an autograd worker's is),
    whose allocations come from the cache."""
    import threading

    q, k, v, g, state = make(1, 3, 400, 64, 64, torch.bfloat16)
    do = torch.randn_like(v)
    want = ops.decay_attention_backward(q, k, v, g, do)
    got = []
    worker = threading.Thread(target=lambda: got.extend(
        ops.decay_attention_backward(q, k, v, g, do)))
    torch.cuda.synchronize()
    worker.start()
    worker.join()
    torch.cuda.synchronize()
    assert len(got) == 4 and all(torch.equal(x, y) for x, y in zip(got[:3], want))


@gpu
def test_repeats_streams_and_graphs():
    """The same bits on every call, on another stream, and replayed from graphs
    whose captures share the allocator."""
    q, k, v, g, state = make(1, 3, 4000, 64, 64, torch.bfloat16)
    do = torch.randn_like(v)

    def call():
        return (*ops.decay_attention(q, k, v, g, initial_state=state, return_state=True),
                *ops.decay_attention_backward(q, k, v, g, do, initial_state=state,
                                              want_d_initial=True))

    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    q0 = q.clone()
    q.copy_(torch.randn_like(q))
    for graph, _ in graphs:
        graph.replay()
    other = call()
    q.copy_(q0)
    assert all(torch.equal(x, y) for x, y in zip(graphs[0][1], other))
    for graph, _ in reversed(graphs):
        graph.replay()
    torch.cuda.synchronize()
    for got in (second, graphs[0][1], graphs[1][1]):
        assert all(torch.equal(x, y) for x, y in zip(first, got))
    assert ops.N.lib().la_take_device_error(None) == 0
