"""The recurrence and the convolution where a warp's ring of tiles goes round several times:
every kind of launch, and sequences that end around the tiles' and the runs' ends."""

import pytest
import test_gated_recurrence as recurrence
import test_short_conv as conv
import torch

import trainium_linear_attention_b200 as T

gpu = pytest.mark.gpu


# ---- convolution --------------------------------------------------------------------
# A run is 128 tokens, 8 tiles of 16, halved until the launch has 222 CTAs of 64 channels
# and 8 runs: runs of 128 in all of these but the second (64).  Rows by TMA, by 4- and 8-byte
# copies, and by shifted pieces (bf16) or single values (fp32).
#
# The bounds of a sum over n = b t tokens allow (n / 8 + 64) roundings in a row.  There are 128
# at most in a run, 8 for its CTA, (b t / 1024 + b) / 32 + 6 for the CTAs' rows: fewer, from n
# = 1024 on.
RUNS = [(240, 300, 64, 4), (100, 600, 70, 3), (8, 1100, 2048, 4), (16, 1100, 1030, 4),
        (16, 1100, 1023, 2)]
ENDS = [0, 1, 2, 3, 4, 15, 16, 17, 18, 19, 20, 31, 32, 33, 35, 127, 128, 129, 130, 131, 132, 143,
        144, 145, 147, 255, 256, 257, 259, 272]


def ends(b, t, seed):
    """b lengths around the ends of tiles and runs, those near t among them."""
    most = [n for n in (*ENDS, 1023, 1024, 1025, 1027, t - 17, t - 16, t - 1, t) if n <= t]
    order = torch.randperm(len(most), generator=torch.Generator().manual_seed(seed)).tolist()
    return torch.tensor([most[order[i % len(most)]] for i in range(b)], device="cuda")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,c,taps", RUNS)
def test_convolution(b, t, c, taps, dtype):
    s = conv.make(b, t, c, taps, dtype, seed=41)
    conv.check_forward(s)
    conv.check_gradients(s)
    s = conv.make(b, t, c, taps, dtype, bias=False, state=False, silu=False, seed=42)
    conv.check_forward(s)
    conv.check_gradients(s)
    for seed in range(3):
        s = conv.make(b, t, c, taps, dtype, state=seed != 1, wtype=torch.float32, seed=43 + seed)
        s["lengths"] = ends(b, t, seed)
        conv.check_forward(s)
        conv.check_gradients(s)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,c,taps", RUNS)
def test_convolution_without_a_final_states_gradient(b, t, c, taps, dtype):
    """Where it is left out other tiles are whole ones; zeros in its place give the same bits."""
    for seed in range(2):
        s = conv.make(b, t, c, taps, dtype, seed=51 + seed)
        if seed:
            s["lengths"] = ends(b, t, seed)
        leaves = [s[n].requires_grad_() for n in ("x", "weight", "bias", "initial_state")]
        out, state = T.causal_conv(**s, return_state=True)
        up = torch.randn(out.shape, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
        without = torch.autograd.grad(out, leaves, up, retain_graph=True)
        zeros = torch.autograd.grad((out, state), leaves, (up, torch.zeros_like(state)))
        assert all(torch.equal(a, b) for a, b in zip(without, zeros))


# ---- recurrence ---------------------------------------------------------------------
# Tokens of a step (of all warps of a channel group), forward and in the gradient, where a GPU
# has 148 SMs: 256 (64 channels, 16 warps) and 128; 512 and 256 (32 channels, 16 warps); 1024
# and 512 (16 channels, 16 warps); 4096 and 2048 (clusters of 8 CTAs of 8 warps); fp32 the same
# but for 16 warps.  Five steps and more of each.  Odd widths: by copies and shifted pieces.
STEPS = [(8, 1400, 1024), (4, 2700, 1024), (1, 5300, 2048), (1, 21000, 128), (2, 4200, 1030),
         (2, 4200, 1023)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("decay,gate", [(True, True), (False, False)])
@pytest.mark.parametrize("b,t,c", STEPS)
def test_recurrence(b, t, c, decay, gate, dtype):
    s = recurrence.make(b, t, c, dtype, decay, gate, seed=61)
    recurrence.check_forward(s)
    recurrence.check_gradients(s)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,c,back", [(8, 1400, 1024, (0, 1, 120, 121, 128, 376, 377, 700)),
                                        (4, 2700, 1024, (1, 140, 141, 652)),
                                        (3, 5300, 672, (1, 181, 1205)),
                                        (1, 21000, 128, (521,)), (1, 21000, 128, (4617,)),
                                        (2, 4200, 1023, (105, 617))])
def test_recurrence_that_ends_in_the_last_steps(b, t, c, back, dtype):
    """(`back`: tokens that a sequence is shorter by; at, before and behind a step's first.)"""
    s = recurrence.make(b, t, c, dtype, True, True, seed=71)
    s["lengths"] = torch.tensor([t - n for n in back], device="cuda")
    recurrence.check_forward(s)
    recurrence.check_gradients(s)


@gpu
@pytest.mark.parametrize("b,t,c", [(4, 300, 1024), (8, 300, 1024), (1, 1100, 2048), (4, 289, 1016),
                                   (1, 4100, 128), (700, 40, 72)])
def test_shapes_of_launches_in_fp32(b, t, c):
    for i, (decay, gate) in enumerate([(True, True), (True, False), (False, True)]):
        s = recurrence.make(b, t, c, torch.float32, decay, gate, state=i != 1, lengths=i == 1, seed=i)
        recurrence.check_forward(s)
        recurrence.check_gradients(s, seed=i)


# ---- transforms ---------------------------------------------------------------------
@gpu
def test_transforms_of_functions_are_refused():
    """A batched or wrapped tensor has no memory that a kernel could be given."""
    x, w = torch.ones(4, 2, 3, 8, device="cuda"), torch.ones(8, 4, device="cuda")
    state = torch.zeros(2, 8, device="cuda")
    for call in (lambda v: T.gated_recurrence(v, v), lambda v: T.causal_conv(v, w),
                 lambda v: T.group_norm(v, 2)):
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(x)
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda v: call(v).sum())(x[0])
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: T.gated_recurrence_step(v[:, 0], v[:, 0], state))(x)
