"""Gated linear recurrence: the kernels against the definition in 64 bits, and the
refusals.

Bounds.  a - 1, beta and u are products of a few fp32 functions, each within a
few 2^-22 of itself (2^-19 in all, F below).  A token's state is off by the old
one's error, decayed, a rounding of the sum (2^-23 of the terms' size M, with M
the recurrence of absolute values) and what a - 1 and b are off by:

    E_t = a_t E_{t-1} + 2^-23 M_t + F ((1 - a_t) M_{t-1} + |b_t u_t x_t|)

The order of the sums (tokens in groups, the groups' products) adds the same
terms once more: 4 E in all.  The gradient's recurrence is the same with a of
the next token.  An output is rounded once (half a step)."""

import pytest
import torch
from torch.autograd import forward_ad

import trainium_linear_attention_b200 as T
from trainium_linear_attention_b200 import _native as N

gpu = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F = 2.0 ** -19


def make(b, t, c, dtype, decay=True, input_gate=True, state=True, lengths=False, seed=0,
         device="cuda"):
    gen = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=gen)

    s = dict(x=normal(b, t, c).to(dtype), gate=(2 * normal(b, t, c)).to(dtype),
             log_decay=None, input_gate=None, initial_state=None, lengths=None)
    if decay:  # half-lives from a token to thousands
        s["log_decay"] = -torch.exp(torch.rand(c, generator=gen) * 9 - 8)
    if input_gate:
        s["input_gate"] = normal(b, t, c).to(dtype)
    if state:
        s["initial_state"] = 2 * normal(b, c)
    if lengths:
        s["lengths"] = torch.randint(0, t + 1, (b,), generator=gen)
    return {n: v if v is None else v.to(device) for n, v in s.items()}


def wide(s):
    return {n: v if v is None or n == "lengths" else v.detach().double() for n, v in s.items()}


def parts(s):
    """a, 1 - a, beta, u, sigmoid(gate) in 64 bits; what lies behind the lengths keeps the state."""
    w = wide(s)
    r = torch.sigmoid(w["gate"])
    u = torch.ones_like(r) if w["input_gate"] is None else torch.sigmoid(w["input_gate"])
    if w["log_decay"] is None:
        a, am1, beta = r, torch.sigmoid(-w["gate"]), torch.sigmoid(-w["gate"])
    else:
        la = w["log_decay"] * r
        a, am1, beta = la.exp(), -torch.expm1(la), (-torch.expm1(2 * la)).sqrt()
    inside = torch.ones_like(r, dtype=torch.bool)
    if w["lengths"] is not None:
        inside &= (torch.arange(r.shape[1], device=r.device) < w["lengths"][:, None])[..., None]
    zero = torch.zeros_like(r)
    return (torch.where(inside, a, 1 + zero), torch.where(inside, am1, zero),
            torch.where(inside, beta, zero), u, r, inside)


def chain(a, b, first):
    outs, h = [], first
    for ai, bi in zip(a.unbind(1), b.unbind(1)):
        h = ai * h + bi
        outs.append(h)
    return torch.stack(outs, 1) if outs else b.clone()


def before(h, first):
    return torch.cat([first[:, None], h[:, :-1]], 1)


def errors(a, am1, b, first):
    """The recurrence, that of absolute values, and the bound of the first's error."""
    zero = torch.zeros_like(first)
    h, m = chain(a, b, first), chain(a, b.abs(), first.abs())
    e = chain(a, 2.0 ** -23 * m + F * (am1 * before(m, first.abs()) + b.abs()), zero)
    return h, m, 4 * e


def forward_bounds(s):
    a, am1, beta, u, r, inside = parts(s)
    x = s["x"].detach().double()
    first = (x.new_zeros(x.shape[0], x.shape[2]) if s["initial_state"] is None
             else s["initial_state"].detach().double())
    h, _, e = errors(a, am1, torch.where(inside, beta * u * x, 0.0), first)
    return h, e, inside, first


def check_forward(s):
    out, state = T.gated_recurrence(**{n: v if v is None else v.detach() for n, v in s.items()},
                                    return_state=True)
    h, e, inside, first = forward_bounds(s)
    assert out.is_contiguous() and out.dtype == s["x"].dtype and state.dtype == torch.float32
    diff = (out.double() - torch.where(inside, h, 0.0)).abs()
    assert (diff <= torch.where(inside, e + HALF[s["x"].dtype] * 1.01 * h.abs(), 0.0)).all()
    want, near = (h[:, -1], e[:, -1]) if h.shape[1] else (first, 0.0)
    assert ((state.double() - want).abs() <= near + 2.0 ** -24 * want.abs()).all()
    return out, state


SIZES = [(1, 1, 1), (2, 1, 5), (1, 7, 64), (3, 16, 33), (2, 17, 66), (1, 64, 128), (2, 65, 96),
         (1, 129, 200), (4, 300, 72), (1, 1024, 64), (1, 1025, 40), (2, 5000, 48), (300, 33, 64),
         (1, 2100, 1031)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,c", SIZES)
def test_forward(b, t, c, dtype):
    for i, (decay, gate) in enumerate([(True, True), (True, False), (False, True), (False, False)]):
        check_forward(make(b, t, c, dtype, decay, gate, state=i % 2 == 0, lengths=i in (0, 3),
                           seed=i))


@gpu
def test_many_channels_and_long_rows():
    """More CTAs than fit at once, clusters of one; a tensor beyond 2^31 elements."""
    check_forward(make(2, 70, 32768, torch.bfloat16))
    n, t, c = 2, 40000, 32000
    x = torch.zeros(n, t, c, dtype=torch.bfloat16, device="cuda")
    x[1, -1000:, -40:] = torch.randn(1000, 40, device="cuda").bfloat16()
    out = T.gated_recurrence(x, x)
    small = T.gated_recurrence(x[1:, -1000:, -40:], x[1:, -1000:, -40:])
    assert (out[0] == 0).all() and (out[1, :-1000] == 0).all()
    # (the groups of tokens are others, so the last bit may be)
    assert ((out[1, -1000:, -40:].float() - small[0].float()).abs()
            <= 2.0 ** -7 * small[0].float().abs() + 1e-6).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    s = make(3, 100, 40, dtype, seed=3)
    want, state = check_forward(s)
    joined = torch.cat([s["x"], s["gate"], s["input_gate"]], -1)  # slices of one projection
    parts_ = dict(zip(("x", "gate", "input_gate"), joined.split(40, -1)))
    for change in (parts_, {"x": s["x"].transpose(0, 1).contiguous().transpose(0, 1)},
                   {"gate": s["gate"].transpose(1, 2).contiguous().transpose(1, 2)},
                   {"x": torch.cat([s["x"], s["x"]], -1)[..., 40:]},
                   {"input_gate": torch.cat([s["input_gate"][..., :3], s["input_gate"]],
                                            -1)[..., 3:]}):
        got = T.gated_recurrence(**{**s, **change}, return_state=True)
        assert torch.equal(got[0], want) and torch.equal(got[1], state)
    one = s["gate"][:1, :1].expand(3, 100, 40)  # strides of zero
    got = T.gated_recurrence(**{**s, "gate": one})
    assert torch.equal(got, T.gated_recurrence(**{**s, "gate": one.contiguous()}))
    lengths = torch.tensor([100, 0, 37], device="cuda")
    a = T.gated_recurrence(**{**s, "lengths": lengths}, return_state=True)
    b = T.gated_recurrence(**{**s, "lengths": lengths.int()}, return_state=True)
    c = T.gated_recurrence(**{**s, "lengths": torch.stack([lengths, lengths], 1)[:, 0]},
                           return_state=True)
    for other in (b, c):
        assert torch.equal(a[0], other[0]) and torch.equal(a[1], other[1])
    beyond = T.gated_recurrence(**{**s, "lengths": torch.tensor([10 ** 12, -5, 37], device="cuda")},
                                return_state=True)
    assert torch.equal(a[0], beyond[0]) and torch.equal(a[1], beyond[1])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_padding_is_not_read(dtype):
    s = make(4, 300, 48, dtype, lengths=True, seed=5)
    want = T.gated_recurrence(**s, return_state=True)
    behind = torch.arange(300, device="cuda") >= s["lengths"][:, None]
    for n in ("x", "gate", "input_gate"):
        s[n] = torch.where(behind[..., None], float("nan"), s[n])
    got = T.gated_recurrence(**s, return_state=True)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    leaves = [s[n].requires_grad_() for n in ("x", "gate", "log_decay", "input_gate")]
    grads = torch.autograd.grad(T.gated_recurrence(**s), leaves, torch.ones_like(want[0]))
    assert all(torch.isfinite(g).all() for g in grads)
    assert all((g[behind] == 0).all() for g in (grads[0], grads[1], grads[3]))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinite_gates(dtype):
    """A gate of -inf (with a decay; +inf without) keeps the state, the other sign forgets."""
    inf = float("inf")
    for decay in (True, False):
        s = make(1, 40, 34, dtype, decay, seed=7)
        s["gate"][:, 10:20] = -inf if decay else inf
        # within the bound of a constant; to the bit within a group of 16 tokens (the next
        # group's state comes as A h + E from the groups' summaries: other roundings, the
        # second part of the bound's 4 E)
        out, _ = check_forward(s)
        assert (out[:, 10:16] == out[:, 9:10]).all() and (out[:, 17:20] == out[:, 16:17]).all()
        s["gate"][:, 10:20] = inf if decay else -inf
        check_forward(s) if decay else None
        s["gate"][0, 25, 3] = float("nan")
        out = T.gated_recurrence(**s)
        assert torch.isnan(out[0, 25:, 3]).all() and torch.isfinite(out[0, :, 4:]).all()
        if not decay:  # a gate of -inf takes the input itself
            u = torch.sigmoid(s["input_gate"][0, 15].double())
            assert torch.allclose(out[0, 15].double(), u * s["x"][0, 15].double(),
                                  rtol=HALF[dtype] * 1.01 + 2.0 ** -20, atol=0)
    s = make(1, 40, 34, dtype, seed=8)
    s["input_gate"][:] = -inf
    s["initial_state"] = None
    assert (T.gated_recurrence(**s) == 0).all()


@gpu
@pytest.mark.parametrize("b,t,c", [(4, 300, 1024), (8, 300, 1024), (1, 1100, 2048), (4, 289, 1016),
                                   (1, 4100, 128), (700, 40, 72)])
def test_shapes_of_launches(b, t, c):
    """Channel groups of each width by CTAs of 16 warps, a cluster of 8, CTAs of 2 warps."""
    for i, (decay, gate) in enumerate([(True, True), (True, False), (False, True)]):
        s = make(b, t, c, torch.bfloat16, decay, gate, state=i != 1, lengths=i == 1, seed=i)
        check_forward(s)
        check_gradients(s, seed=i)
        if i == 1:  # sequences that end in the first and last tokens of a step's tiles
            ends = [0, 1, t, t - 1, 255, 256, 257, 129]
            s["lengths"] = torch.tensor([min(ends[j % 8], t) for j in range(b)], device="cuda")
            check_forward(s)
            check_gradients(s, seed=i)


@gpu
def test_slow_decays():
    """1 - a below fp32's step next to 1: the memory is 2^30 tokens long."""
    n = 20000
    x = torch.zeros(1, n, 2, device="cuda")
    gate = torch.zeros(1, n, 2, device="cuda")
    log_decay = torch.full((2,), -2.0 ** -29, device="cuda")
    first = torch.ones(1, 2, device="cuda") * 2.0 ** 20
    # Not the 1.9e-5 that is lost in all: a token's 2^-30 of the state is below half a step
    # of fp32 (2^-25 of it at least), so a state held in fp32 cannot show it, and the bound
    # for the token's rounding (2^-23 M_t, n times) is what holds.
    check_forward(dict(x=x, gate=gate, log_decay=log_decay, input_gate=None, lengths=None,
                       initial_state=first))
    s = make(1, n, 2, torch.float32, decay=False)
    s["log_decay"] = log_decay
    check_forward(s)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,c", SIZES)
def test_gradients(b, t, c, dtype):
    for i, (decay, gate) in enumerate([(True, True), (True, False), (False, True), (False, False)]):
        s = make(b, t, c, dtype, decay, gate, state=i % 2 == 0, lengths=i in (0, 3), seed=i)
        check_gradients(s, seed=i)


def check_gradients(s, seed=0):
    dtype = s["x"].dtype
    half = HALF[dtype] * 1.01
    gen = torch.Generator().manual_seed(100 + seed)
    names = [n for n in ("x", "gate", "log_decay", "input_gate", "initial_state")
             if s[n] is not None]
    for n in names:
        s[n].requires_grad_()
    out, state = T.gated_recurrence(**s, return_state=True)
    dy = torch.randn(out.shape, generator=gen).to(dtype).cuda()
    ds = torch.randn(state.shape, generator=gen).cuda()
    got = dict(zip(names, torch.autograd.grad((out, state), [s[n] for n in names], (dy, ds))))

    h, eh, inside, first = forward_bounds(s)
    a, am1, beta, u, r, _ = parts(s)
    x, lam = s["x"].detach().double(), s["log_decay"]
    lam = None if lam is None else lam.detach().double()
    hp, ehp = before(h, first), before(eh, torch.zeros_like(first))
    # the gradient's recurrence in c_t = a_t H_t, what H_{t-1} gets
    d = torch.where(inside, dy.double(), 0.0)
    back = lambda v: v.flip(1)
    zero = torch.zeros_like(first)
    c_ = back(chain(back(a), back(a * d), ds.double()))
    m = back(chain(back(a), back(a * d.abs()), ds.double().abs()))
    after = lambda v, end: torch.cat([v[:, 1:], end[:, None]], 1)
    big, h_grad = after(m, ds.double().abs()) + d.abs(), after(c_, ds.double()) + d
    ec = 4 * back(chain(back(a), back(2.0 ** -23 * big + F * am1 * big), zero))
    eg = after(ec, zero) + 2.0 ** -23 * big
    ab = torch.where(inside, 1.0, 0.0)
    want = {"x": h_grad * beta * u}
    near = {"x": beta * u * (eg + F * h_grad.abs())}
    if s["input_gate"] is not None:
        f = beta * x * u * (1 - u)
        want["input_gate"], near["input_gate"] = h_grad * f, f.abs() * (eg + 2 * F * h_grad.abs())
    if lam is None:
        f, w = r * (1 - r) * ab, u * x
        log_grad = h_grad * (hp - w)
        e_log = eg * (hp - w).abs() + h_grad.abs() * (ehp + F * (hp.abs() + w.abs()))
    else:
        f, w = lam * r * (1 - r) * ab, torch.where(inside, a * u * x / beta, 0.0)
        log_grad = a * h_grad * (hp - w)
        e_log = a * (eg * (hp - w).abs() + h_grad.abs() * (ehp + 2 * F * (hp.abs() + w.abs())))
        want["log_decay"] = (log_grad * r * ab).sum((0, 1))
        near["log_decay"] = ((e_log + 2 * F * log_grad.abs()) * r * ab).sum((0, 1))
    want["gate"], near["gate"] = log_grad * f, f.abs() * (e_log + 2 * F * log_grad.abs())
    if s["initial_state"] is not None:
        want["initial_state"] = c_[:, 0]
        near["initial_state"] = ec[:, 0]
    for n in names:
        rounding = half if n in ("x", "gate", "input_gate") else 2.0 ** -23
        assert got[n].shape == s[n].shape and got[n].dtype == s[n].dtype
        diff = (got[n].double() - want[n]).abs()
        # (below 2^-120 products of small factors may be flushed to zero)
        assert (diff <= near[n] + rounding * want[n].abs() + 2.0 ** -120).all(), n


@gpu
@pytest.mark.parametrize("decay,gate", [(True, True), (False, False)])
def test_gradients_are_the_definitions_and_differences(decay, gate):
    """The formula above is autograd's of the definition, and the kernel's own
    quotient of differences is the definition's."""
    s = make(2, 70, 6, torch.float32, decay, gate, seed=11)
    names = [n for n in ("x", "gate", "log_decay", "input_gate", "initial_state")
             if s[n] is not None]
    w = {n: v if v is None else v.double().requires_grad_() for n, v in s.items()}
    gen = torch.Generator().manual_seed(1)
    up = torch.randn(2, 70, 6, generator=gen).cuda()
    want = torch.autograd.grad(T.ref_gated_recurrence(**w)[0], [w[n] for n in names], up.double())
    for n in names:
        s[n].requires_grad_()
    got = torch.autograd.grad(T.gated_recurrence(**s), [s[n] for n in names], up)
    step = 2.0 ** -8
    for n, g, g64 in zip(names, got, want):
        assert float((g.double() - g64).norm() / g64.norm()) <= 2.0 ** -18, n
        direction = torch.randn(s[n].shape, generator=gen).cuda() * s[n].detach().abs().clamp(max=1)

        def moved(f, base, sign):
            to = base[n].detach() + sign * step * direction.to(base[n].dtype)
            args = {k: v if v is None else v.detach() for k, v in {**base, n: to}.items()}
            return f(args).double() * up

        ours = moved(lambda v: T.gated_recurrence(**v), s, 1) - moved(
            lambda v: T.gated_recurrence(**v), s, -1)
        theirs = moved(lambda v: T.ref_gated_recurrence(**v)[0], w, 1) - moved(
            lambda v: T.ref_gated_recurrence(**v)[0], w, -1)
        # both sides of a difference are off by the forward bound
        _, e, _, _ = forward_bounds(s)
        assert abs(float(ours.sum() - theirs.sum())) <= float(
            (3 * (e + 2.0 ** -23 * out_size(s)) * up.abs()).sum())
        quotient = float(theirs.sum()) / (2 * step)
        slope = float((g64 * direction).sum())
        size = float((g64 * direction).abs().sum())
        assert abs(quotient - slope) <= 2.0 ** -8 * size, n


def out_size(s):
    h, _, _, _ = forward_bounds(s)
    return h.abs()


@gpu
def test_parts_of_the_gradient():
    s = make(2, 90, 40, torch.bfloat16, seed=13)
    for n in ("x", "gate", "log_decay", "input_gate", "initial_state"):
        s[n].requires_grad_()
    out, state = T.gated_recurrence(**s, return_state=True)
    up = torch.randn_like(out)
    all_ = torch.autograd.grad(out, [s["x"], s["gate"], s["log_decay"], s["initial_state"]], up,
                               retain_graph=True)
    again = torch.autograd.grad(out, [s["log_decay"]], up, retain_graph=True)
    assert torch.equal(all_[2], again[0])
    only = torch.autograd.grad(state, [s["x"], s["initial_state"]], torch.ones_like(state),
                               retain_graph=True)
    assert torch.isfinite(only[0]).all() and (only[1] != 0).any()
    expanded = torch.autograd.grad(out.float().sum(), [s["x"]], retain_graph=True)[0]
    ones = torch.autograd.grad(out, [s["x"]], torch.ones_like(out), retain_graph=True)[0]
    assert torch.equal(expanded, ones)
    # a shared input's gradients add up, and a broadcast gate's are summed
    g = torch.autograd.grad(T.gated_recurrence(s["x"], s["x"]), [s["x"]], up)[0]
    assert g.shape == s["x"].shape
    row = s["gate"].detach()[:, :1].clone().requires_grad_()
    g = torch.autograd.grad(T.gated_recurrence(s["x"], row.expand(-1, 90, -1), s["log_decay"]),
                            [row], up)[0]
    full = row.detach().expand(-1, 90, -1).contiguous().requires_grad_()
    f = torch.autograd.grad(T.gated_recurrence(s["x"], full, s["log_decay"]), [full], up)[0]
    assert torch.equal(g, f.sum(1, keepdim=True))
    with pytest.raises(RuntimeError):
        y = T.gated_recurrence(**s)
        first, = torch.autograd.grad(y, [s["x"]], torch.ones_like(y), create_graph=True)
        torch.autograd.grad(first.float().sum(), [s["gate"]])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pieces_and_steps(dtype):
    """A prompt in pieces and single tokens against the whole: each within its bound."""
    s = make(3, 90, 52, dtype, seed=17)
    h, e, _, _ = forward_bounds(s)
    state, at, outs = s["initial_state"], 0, []
    piece = lambda n, i, j: None if s[n] is None else s[n][:, i:j]
    for n in (1, 40, 30, 0):
        out, state = T.gated_recurrence(
            piece("x", at, at + n), piece("gate", at, at + n), s["log_decay"],
            piece("input_gate", at, at + n), state, return_state=True)
        outs.append(out)
        at += n
    state = state.clone()
    version = state._version
    for t in range(at, 90):
        outs.append(T.gated_recurrence_step(s["x"][:, t], s["gate"][:, t], state, s["log_decay"],
                                            s["input_gate"][:, t])[:, None])
    assert state._version > version
    got = torch.cat(outs, 1)
    assert ((got.double() - h).abs() <= 2 * e + HALF[dtype] * 1.01 * h.abs()).all()
    assert ((state.double() - h[:, -1]).abs() <= 2 * e[:, -1] + 2.0 ** -23 * h[:, -1].abs()).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,c", [(1, 1), (1, 4), (5, 7), (3, 64), (257, 130)])
def test_step(b, c, dtype):
    for i, (decay, gate) in enumerate([(True, True), (True, False), (False, True), (False, False)]):
        s = make(b, 1, c, dtype, decay, gate, seed=i)
        h, e, _, _ = forward_bounds(s)
        state = s["initial_state"].clone()
        wide_state = torch.randn(b, c + 3, device="cuda")
        kept = wide_state[:, c:].clone()
        wide_state[:, :c] = state
        args = (s["log_decay"], None if s["input_gate"] is None else s["input_gate"][:, 0])
        out = T.gated_recurrence_step(s["x"][:, 0], s["gate"][:, 0], state, *args)
        assert ((out.double() - h[:, 0]).abs() <= e[:, 0] + HALF[dtype] * 1.01 * h[:, 0].abs()).all()
        assert ((state.double() - h[:, 0]).abs() <= e[:, 0] + 2.0 ** -24 * h[:, 0].abs()).all()
        again = T.gated_recurrence_step(s["x"][:, 0], s["gate"][:, 0], wide_state[:, :c], *args)
        assert torch.equal(wide_state[:, :c], state) and torch.equal(wide_state[:, c:], kept)
        assert torch.equal(again, out)
        slices = torch.cat([s["x"][:, 0], s["gate"][:, 0]], -1)
        third = s["initial_state"].clone()
        assert torch.equal(out, T.gated_recurrence_step(slices[:, :c], slices[:, c:], third, *args))


@gpu
def test_empty():
    z = lambda *s: torch.zeros(*s, device="cuda")
    first = torch.randn(2, 5, device="cuda").requires_grad_()
    lam = torch.full((5,), -1.0, device="cuda").requires_grad_()
    out, state = T.gated_recurrence(z(2, 0, 5), z(2, 0, 5), lam, initial_state=first,
                                    return_state=True)
    assert out.shape == (2, 0, 5) and torch.equal(state, first)
    g, gl = torch.autograd.grad(state, [first, lam], torch.ones_like(state))
    assert (g == 1).all() and (gl == 0).all()
    assert (T.gated_recurrence(z(2, 0, 5), z(2, 0, 5), return_state=True)[1] == 0).all()
    assert T.gated_recurrence(z(0, 3, 5), z(0, 3, 5)).shape == (0, 3, 5)
    assert T.gated_recurrence_step(z(0, 5), z(0, 5), z(0, 5)).shape == (0, 5)


@gpu
def test_streams_and_graphs():
    s = make(2, 700, 64, torch.bfloat16, seed=19)
    leaves = [s[n].requires_grad_() for n in ("x", "gate", "log_decay", "input_gate",
                                              "initial_state")]
    up = torch.randn(2, 700, 64, device="cuda").bfloat16()

    def step():
        out, state = T.gated_recurrence(**s, return_state=True)
        return [out.detach(), state.detach(),
                *torch.autograd.grad((out, state), leaves, (up, torch.ones_like(state)))]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graphs = []
    for _ in range(2):  # two graphs replayed one after the other share nothing
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
    for graph, _ in graphs:
        graph.replay()
    for _, got in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    with torch.no_grad():
        s["x"].mul_(0.5)
    again = step()
    graphs[0][0].replay()
    assert all(torch.equal(a, b) for a, b in zip(again, graphs[0][1]))


def on_cpu(**change):
    s = make(2, 5, 8, torch.float32, device="cpu")
    return {**s, **change}


def test_refusals_on_the_cpu():
    with pytest.raises(ValueError, match="CUDA"):
        T.gated_recurrence(**on_cpu())
    with pytest.raises(TypeError, match="x must be"):
        T.gated_recurrence(**on_cpu(x=3.0))
    with pytest.raises(ValueError, match="batch, tokens, channels"):
        T.gated_recurrence(**on_cpu(x=torch.zeros(5, 8)))
    with pytest.raises(ValueError, match="CUDA"):
        T.gated_recurrence_step(torch.zeros(2, 8), torch.zeros(2, 8), torch.zeros(2, 8))
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.zeros(2, 5, 8), torch.ones(2, 5, 8))
        with pytest.raises(NotImplementedError):
            T.gated_recurrence(**on_cpu(x=x))


def test_c_refusals():
    lib = N.lib()
    one = 16  # never read
    i64 = N.ctypes.c_int64 * 2
    st = N.ctypes.addressof(strides := i64(8, 8))
    fwd = lambda x=one, g=one, out=one, b=1, t=1, c=8, dtype=0, bits=0, lengths=None, s=st: (
        lib.la_recurrence_fwd(x, s, g, s, None, None, None, None, lengths, bits, out, None, None,
                              b, t, c, dtype, None))
    bad, unsupported = N.LA_ERR_INVALID_ARGUMENT, N.LA_ERR_UNSUPPORTED
    assert fwd(x=None) == fwd(g=None) == fwd(out=None) == fwd(c=0) == fwd(b=-1) == bad
    assert fwd(t=-1) == fwd(dtype=2) == fwd(lengths=one, bits=16) == fwd(s=None) == bad
    assert fwd(c=2 ** 40) == fwd(t=2 ** 40, b=2 ** 30) == unsupported
    assert fwd(b=0) == N.LA_OK
    negative = i64(-8, 8)
    assert fwd(s=N.ctypes.addressof(negative)) == bad
    step = lambda state=one, stride=8, b=2: lib.la_recurrence_step(
        one, 8, one, 8, None, 0, None, state, stride, one, b, 8, 0, None)
    assert step(state=None) == step(stride=4) == step(stride=0) == bad
    assert step(b=0) == N.LA_OK
    a, w = N.ctypes.c_size_t(), N.ctypes.c_size_t()
    plan = lambda b, t, c: lib.la_recurrence_plan(b, t, c, N.ctypes.byref(a), N.ctypes.byref(w))
    assert plan(1, 1, 0) == bad and plan(0, 5, 8) == N.LA_OK and a.value == 0
    assert strides[0] == 8


def test_c_refuses_pointers_between_elements():
    """Numbers in place of pointers, which no call gets as far as reading."""
    lib, bad = N.lib(), N.LA_ERR_INVALID_ARGUMENT
    strides = (N.ctypes.c_int64 * 2)(8, 8)
    st = N.ctypes.addressof(strides)

    def calls(odd, dtype, at):
        p = [odd if i == at else 16 for i in range(9)]
        x, g, u, lam, init, out, final, saved, lengths = p
        return (lib.la_recurrence_fwd(x, st, g, st, u, st, lam, init, lengths, 64, out, final,
                                      saved, 1, 1, 8, dtype, None),
                lib.la_recurrence_bwd(x, st, g, st, u, st, lam, saved, lengths, 64, out, st, init,
                                      16, 16, 16, final, None, 1, 1, 8, dtype, None, 0, None))

    for at in range(9):
        odd, dtype = (20 if at == 8 else 18, 0)  # lengths of 8 bytes, all else of 4
        assert calls(odd, dtype, at) == (bad, bad), at
    for at in (0, 1, 2, 5):
        assert calls(17, 1, at) == (bad, bad), at
    step = lambda x=16, g=16, u=16, lam=16, state=16, out=16: lib.la_recurrence_step(
        x, 8, g, 8, u, 8, lam, state, 8, out, 2, 8, 0, None)
    assert step(x=18) == step(g=18) == step(u=18) == step(lam=18) == step(state=18) == step(
        out=18) == bad


@gpu
def test_refusals():
    s = make(2, 5, 8, torch.bfloat16)
    call = lambda **change: T.gated_recurrence(**{**s, **change})
    for change, error, text in [
            (dict(gate=None), TypeError, "gate"), (dict(gate=s["gate"][:, :4]), ValueError, "gate"),
            (dict(gate=s["gate"].float()), ValueError, "gate"),
            (dict(x=s["x"].half()), TypeError, "float16"),
            (dict(input_gate=s["gate"].cpu()), ValueError, "input_gate"),
            (dict(log_decay=s["log_decay"].bfloat16()), ValueError, "log_decay"),
            (dict(log_decay=s["log_decay"][:4]), ValueError, "log_decay"),
            (dict(initial_state=s["initial_state"].bfloat16()), ValueError, "initial_state"),
            (dict(initial_state=s["initial_state"][:1]), ValueError, "initial_state"),
            (dict(lengths=[1, 2]), TypeError, "lengths"),
            (dict(lengths=torch.ones(2, device="cuda")), ValueError, "lengths"),
            (dict(lengths=torch.ones(2, dtype=torch.int64)), ValueError, "lengths"),
            (dict(x=s["x"][..., :0], gate=s["gate"][..., :0]), ValueError, "channels")]:
        with pytest.raises(error, match=text):
            call(**change)
    x, g, state = s["x"][:, 0], s["gate"][:, 0], s["initial_state"]
    step = T.gated_recurrence_step
    with pytest.raises(ValueError, match="overlap"):
        step(x, g, torch.zeros(1, 8, device="cuda").expand(2, 8))
    with pytest.raises(ValueError, match="dense"):
        step(x, g, torch.zeros(8, 2, device="cuda").t())
    with pytest.raises(ValueError, match="state"):
        step(x, g, state.bfloat16())
    with pytest.raises(TypeError, match="state"):
        step(x, g, None)
    with pytest.raises(ValueError, match="in place"):
        step(x, g, state.clone().requires_grad_())
    with pytest.raises(ValueError, match="batch, channels"):
        step(s["x"], g, state)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,c", [(2, 100, 40), (1, 70, 33), (1, 300, 1030), (8, 1400, 1024)])
def test_nearly_closed_input_gates(b, t, c, dtype):
    """sigmoid of -40 to -75 is far from 0 (e-18 to e-33) and reaches the outputs, with a
    decay and without, among open gates and by itself.  The bound holds: exp's argument in
    units of ln 2 is below 128, so its rounding (half of 2^-17) and the constant's (2^-26
    of it) are below 2^-18 of u, F's fourfold is 2^-17."""
    for decay in (True, False):
        s = make(b, t, c, dtype, decay, state=False, seed=23)
        gen = torch.Generator().manual_seed(24)
        low = (-40 - 35 * torch.rand(b, t, c, generator=gen)).to(dtype).cuda()
        s["x"] = s["x"].abs().clamp(min=2.0 ** -6) * 2.0 ** 20
        mixed = torch.where(torch.rand(b, t, c, generator=gen).cuda() < 0.9, s["input_gate"], low)
        for gates in (low, mixed):
            s["input_gate"] = gates
            out, _ = check_forward(s)
            assert (out != 0).all()
        s["input_gate"] = low
        state = torch.zeros(b, c, device="cuda")
        one = T.gated_recurrence_step(s["x"][:, 0], s["gate"][:, 0], state, s["log_decay"], low[:, 0])
        h, e, _, _ = forward_bounds({n: v if v is None or v.dim() < 3 else v[:, :1]
                                     for n, v in s.items()})
        assert (one != 0).all()
        assert ((one.double() - h[:, 0]).abs() <= e[:, 0] + HALF[dtype] * 1.01 * h[:, 0].abs()).all()
