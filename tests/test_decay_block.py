"""The blocks that use the decayed linear attention and the norms together:
training, prompts in pieces, single tokens, a captured step."""

import pytest
import torch

import trainium_linear_attention_b200 as T

gpu = pytest.mark.gpu


class Plain(torch.nn.Module):
    """DecayLinearAttention's definition on its parameters, in float64."""

    def __init__(self, m):
        super().__init__()
        self.m, self.p = m, {n: x.detach().double() for n, x in m.named_parameters()}

    def forward(self, x, residual, state):
        m, p = self.m, self.p
        b, t, dim = x.shape
        y, stream = T.ref_rms_norm(x, p["norm_weight"], residual, m.eps)

        def heads(name):
            return (y @ p[name].T).view(b, t, m.num_heads, m.head_dim).transpose(1, 2)

        o, end = T.ref_decay_attn(heads("q_proj.weight"), heads("k_proj.weight"),
                                  heads("v_proj.weight"), m.log_decay.double(), None, state)
        o, _ = T.ref_rms_norm(o.transpose(1, 2), p["head_norm_weight"], None, m.eps)
        return o.reshape(b, t, dim) @ p["o_proj.weight"].T, stream, end


def make(dim=256, heads=4, dtype=torch.float32, seed=0):
    torch.manual_seed(seed)
    m = T.DecayLinearAttention(dim, heads)
    with torch.no_grad():
        m.norm_weight.uniform_(0.5, 1.5)
        m.head_norm_weight.uniform_(0.5, 1.5)
    return m.to(dtype).cuda() if torch.cuda.is_available() else m.to(dtype)


def rel(x, y):
    return float((x.double() - y).norm() / y.norm())


# The whole block is compared in the 2-norm.  fp32: six products of at most 256
# terms in a row and two norms, each off by at most (256 + 40) 2^-24 of sums of
# absolute values, which random signs make sqrt(256) times their norm at most:
# 8 * 296 * 2^-24 * 16 = 2.3e-3 would be sure; the errors are random too, so a
# sixteenth of it is asked for.  bf16: nine roundings in a row (norm, q, k, v, P
# or S, o, head norm, output), each 2^-8 at most: 9 * 2^-8.
BOUND = {torch.float32: 1.5e-4, torch.bfloat16: 9 * 2.0 ** -8}


def test_block_on_the_cpu_refuses():
    m = T.DecayLinearAttention(64, 4)
    assert sorted(m.state_dict()) == ["head_norm_weight", "k_proj.weight", "log_decay",
                                      "norm_weight", "o_proj.weight", "q_proj.weight",
                                      "v_proj.weight"]
    before = m.log_decay.clone()
    assert m.to(torch.bfloat16).log_decay.dtype == torch.float32
    assert torch.equal(m.log_decay, before) and m.norm_weight.dtype == torch.bfloat16
    assert not any(n == "log_decay" for n, _ in m.named_parameters())
    with pytest.raises(ValueError, match="CUDA"):
        m(torch.zeros(1, 3, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="log_decay"):
        T.DecayLinearAttention(64, 4, log_decay=[-1.0])
    with pytest.raises(ValueError, match="head dim"):
        T.DecayLinearAttention(512, 2)
    with pytest.raises(ValueError, match="residual"):
        T.TrainiumBasedLinearAttentionNKI(64, 4)(torch.zeros(1, 3, 64), torch.zeros(1, 3, 64))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_step(dtype):
    m = make(dtype=dtype)
    ref = Plain(m)
    x = torch.randn(2, 300, 256, device="cuda").to(dtype).requires_grad_()
    r = torch.randn(2, 300, 256, device="cuda").to(dtype).requires_grad_()
    s = torch.randn(2, 4, 64, 64, device="cuda").requires_grad_()
    out, stream, end = m(x, r, s, return_state=True)
    up = [torch.randn_like(t) for t in (out, stream, end)]
    params = dict(m.named_parameters())
    got = torch.autograd.grad((out, stream, end), [x, r, s, *params.values()], up)
    wide = [t.detach().double().requires_grad_() for t in (x, r, s)]
    ref.p = {n: t.requires_grad_() for n, t in ref.p.items()}
    want = ref(*wide)
    grads = torch.autograd.grad(want, [*wide, *(ref.p[n] for n in params)],
                                [u.double() for u in up])
    for a, b in zip((out, stream, end), want):
        assert rel(a.detach(), b.detach()) <= BOUND[dtype]
    # a gradient passes the block's roundings twice, forward and back
    for name, a, b in zip(["x", "residual", "state", *params], got, grads):
        assert rel(a, b) <= 2 * BOUND[dtype], name


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_tokens(dtype):
    """A prompt in two pieces and four single tokens against the whole at once."""
    m = make(dtype=dtype, seed=1)
    x = torch.randn(3, 200, 256, device="cuda").to(dtype)
    r = torch.randn(3, 200, 256, device="cuda").to(dtype)
    with torch.no_grad():
        whole, stream = m(x, r)
        a, _, state = m(x[:, :130], r[:, :130], return_state=True)
        b, _, state = m(x[:, 130:196], r[:, 130:196], state=state, return_state=True)
    outs = [a, b]
    for t in range(196, 200):
        y, st = m.step(x[:, t], state, r[:, t])
        assert torch.equal(st, stream[:, t])
        outs.append(y[:, None])
    want = Plain(m)(x.double(), r.double(), None)[0]
    assert rel(torch.cat(outs, 1), want) <= BOUND[dtype]
    assert rel(whole, want) <= BOUND[dtype]


@gpu
def test_captured_step():
    """Decoding replayed from a graph: the state advances as in eager calls."""
    m = make(dtype=torch.bfloat16, seed=2)
    x = torch.randn(5, 2, 256, device="cuda").bfloat16()
    eager = torch.zeros(2, 4, 64, 64, device="cuda")
    outs = [m.step(t, eager)[0] for t in x]
    state, static = torch.zeros_like(eager), torch.empty_like(x[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.step(static.zero_(), torch.zeros_like(state))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = m.step(static, state)
    for t, want in zip(x, outs):
        static.copy_(t)
        graph.replay()
        assert torch.equal(out, want)
    assert torch.equal(state, eager)


@gpu
def test_based_module_with_pre_norm():
    """The BASED module normed ahead of its projections is the module behind the
    norm, and without the option what it was."""
    torch.manual_seed(3)
    m = T.TrainiumBasedLinearAttentionNKI(128, 8, window_size=16, pre_norm=True).cuda()
    plain = T.TrainiumBasedLinearAttentionNKI(128, 8, window_size=16).cuda()
    state = m.state_dict()
    state.pop("norm_weight")
    plain.load_state_dict(state)
    x, r = torch.randn(2, 70, 128, device="cuda"), torch.randn(2, 70, 128, device="cuda")
    with torch.no_grad():
        out, stream = m(x, r)
        y, total = T.rms_norm(x, m.norm_weight, residual=r, eps=m.eps)
        assert torch.equal(stream, total) and torch.equal(out, plain(y))
        out, stream = m(x)
        assert stream is x and torch.equal(out, plain(T.rms_norm(x, m.norm_weight, eps=m.eps)))
