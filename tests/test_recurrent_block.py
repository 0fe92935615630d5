"""The block of the convolution, the recurrence and the group norm together:
training, prompts in pieces and of unlike lengths, single tokens, a captured step."""

import pytest
import torch

import trainium_linear_attention_b200 as T

gpu = pytest.mark.gpu


def plain(m, x, residual, state=None, lengths=None, p=None):
    """GatedRecurrence's definition on its parameters, in float64."""
    p = p or {n: v.detach().double() for n, v in m.named_parameters()}
    y, stream = T.ref_rms_norm(x, p["norm_weight"], residual, m.eps)
    y, out_gate = (y @ p["in_proj.weight"].T).chunk(2, -1)
    before, h0 = (None, None) if state is None else state
    y, tail = T.ref_causal_conv(y, p["conv_weight"], p["conv_bias"], "silu", before, lengths)
    gate, input_gate = (y @ p["gate_proj.weight"].T).chunk(2, -1)
    h, end = T.ref_gated_recurrence(y, gate, -torch.nn.functional.softplus(p["decay"]), input_gate,
                                    h0, lengths)
    h = T.ref_group_norm(h, m.num_heads, p["head_norm_weight"], p["head_norm_bias"], out_gate,
                         "silu", m.eps)
    return h @ p["o_proj.weight"].T, stream, tail, end


def make(dim=256, heads=4, dtype=torch.float32, seed=0):
    torch.manual_seed(seed)
    m = T.GatedRecurrence(dim, heads)
    with torch.no_grad():
        for w in (m.norm_weight, m.head_norm_weight):
            w.uniform_(0.5, 1.5)
        m.conv_bias.uniform_(-0.2, 0.2)
        m.head_norm_bias.uniform_(-0.2, 0.2)
    return m.to(dtype).cuda() if torch.cuda.is_available() else m.to(dtype)


def rel(x, y):
    return float((x.double() - y).norm() / y.norm())


# Compared in the 2-norm.  fp32: three products of at most 256 terms in a row and four
# operators, each off by at most (256 + 40) 2^-24 of sums of absolute values, which random
# signs make sqrt(256) times their norm at most: 7 * 296 * 2^-24 * 16 = 2e-3 would be sure; the
# errors are random too, so a sixteenth of it is asked for.  bf16: eight roundings in a row
# (norm, input, convolution, gates, recurrence, head norm, output, and the decay's own in the
# module's cast, which both sides have), 2^-8 each at most; the head norm divides by what the
# heads vary by, of which a mean of the same size is taken first: twice that.
BOUND = {torch.float32: 1.3e-4, torch.bfloat16: 16 * 2.0 ** -8}


def test_block_on_the_cpu_refuses():
    m = T.GatedRecurrence(64, 4)
    with pytest.raises(ValueError, match="CUDA"):
        m(torch.zeros(1, 3, 64))
    with pytest.raises(ValueError, match="heads"):
        T.GatedRecurrence(64, 5)
    with pytest.raises(ValueError, match="taps"):
        T.GatedRecurrence(64, 4, taps=5)
    keep = torch.exp(0.5 * m._log_decay())
    assert abs(float(keep.min()) - 0.9) < 1e-5 and abs(float(keep.max()) - 0.999) < 1e-5


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_step(dtype):
    m = make(dtype=dtype)
    x = torch.randn(2, 300, 256, device="cuda").to(dtype).requires_grad_()
    r = torch.randn(2, 300, 256, device="cuda").to(dtype).requires_grad_()
    tail = torch.randn(2, 3, 256, device="cuda").to(dtype).requires_grad_()
    h0 = torch.randn(2, 256, device="cuda").requires_grad_()
    out, stream, end = m(x, r, (tail, h0), return_state=True)
    outs = (out, stream, *end)
    up = [torch.randn_like(t) for t in outs]
    params = dict(m.named_parameters())
    got = torch.autograd.grad(outs, [x, r, tail, h0, *params.values()], up)
    wide = [t.detach().double().requires_grad_() for t in (x, r, tail, h0)]
    p = {n: t.detach().double().requires_grad_() for n, t in params.items()}
    want = plain(m, wide[0], wide[1], (wide[2], wide[3]), p=p)
    grads = torch.autograd.grad(want, [*wide, *p.values()], [u.double() for u in up])
    for a, b in zip(outs, want):
        assert rel(a.detach(), b.detach()) <= BOUND[dtype]
    # a gradient passes the block's roundings twice, forward and back
    for name, a, b in zip(["x", "residual", "tail", "h0", *params], got, grads):
        assert rel(a, b) <= 2 * BOUND[dtype], name


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_tokens(dtype):
    """Prompts of unlike lengths, padded, then four single tokens each, against each
    sequence by itself."""
    m = make(dtype=dtype, seed=1)
    lengths = torch.tensor([130, 1, 57], device="cuda")
    x = torch.randn(3, 134, 256, device="cuda").to(dtype)
    r = torch.randn(3, 134, 256, device="cuda").to(dtype)
    with torch.no_grad():
        first, _, state = m(x[:, :130], r[:, :130], return_state=True, lengths=lengths)
    row = torch.arange(3, device="cuda")
    steps = []
    for i in range(4):
        y, stream = m.step(x[row, lengths + i], state, r[row, lengths + i])
        steps.append(y)
        assert torch.equal(stream, (x + r)[row, lengths + i])
    for i, n in enumerate(lengths.tolist()):
        want = plain(m, x[i:i + 1, :n + 4].double(), r[i:i + 1, :n + 4].double())[0][0]
        got = torch.cat([first[i, :n], torch.stack([y[i] for y in steps])])
        assert rel(got, want) <= BOUND[dtype]
        with torch.no_grad():  # in two pieces, by itself
            k = n // 2
            a, _, s = m(x[i:i + 1, :k], r[i:i + 1, :k], return_state=True)
            b, _, s = m(x[i:i + 1, k:n + 4], r[i:i + 1, k:n + 4], s, return_state=True)
        assert rel(torch.cat([a, b], 1)[0], want) <= BOUND[dtype]


@gpu
def test_captured_step_and_training():
    """Decoding and a training step replayed from graphs give what eager calls do."""
    m = make(dtype=torch.bfloat16, seed=2)
    x = torch.randn(5, 2, 256, device="cuda").bfloat16()
    eager = m.empty_state(2)
    outs = [m.step(t, eager)[0] for t in x]
    state, static = m.empty_state(2), torch.empty_like(x[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.step(static.zero_(), m.empty_state(2))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = m.step(static, state)
    for t, want in zip(x, outs):
        static.copy_(t)
        graph.replay()
        assert torch.equal(out, want)
    assert all(torch.equal(a, b) for a, b in zip(state, eager))

    x = torch.randn(2, 70, 256, device="cuda").bfloat16()
    params = list(m.parameters())

    def train():
        out, _ = m(x)
        return [out.detach(), *torch.autograd.grad(out, params, torch.ones_like(out))]

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = train()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = train()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_training_runs():
    """A few optimiser steps run and leave finite parameters that have moved."""
    m = make(64, 4, torch.bfloat16, seed=3)
    before = {n: p.detach().clone() for n, p in m.named_parameters()}
    optimiser = torch.optim.SGD(m.parameters(), lr=0.1)
    for i in range(3):
        x = torch.randn(2, 50, 64, device="cuda").bfloat16()
        optimiser.zero_grad()
        out, stream = m(x, x)
        (out + stream).float().square().mean().backward()
        optimiser.step()
    for n, p in m.named_parameters():
        assert torch.isfinite(p).all() and p.grad.abs().sum() > 0, n
    assert any(not torch.equal(p, before[n]) for n, p in m.named_parameters())


@gpu
def test_autocast():
    """fp32 parameters under autocast to bf16: prompts, and tokens from a new sequence's state,
    within a bf16 block's bound; a training step's gradients are fp32 and finite."""
    m = make(seed=4)
    x = torch.randn(2, 6, 256, device="cuda")
    want = plain(m, x.double(), None)[0]
    with torch.autocast("cuda", torch.bfloat16), torch.no_grad():
        out, _ = m(x)
        state = m.empty_state(2)
        steps = torch.stack([m.step(t, state)[0] for t in x.unbind(1)], 1)
    assert rel(out, want) <= BOUND[torch.bfloat16] and rel(steps, want) <= BOUND[torch.bfloat16]
    with torch.autocast("cuda", torch.bfloat16):
        out, _ = m(x)
    grads = torch.autograd.grad(out.float().square().mean(), list(m.parameters()))
    assert all(g.dtype == torch.float32 and torch.isfinite(g).all() for g in grads)
    assert m.empty_state(1)[0].dtype == torch.float32
