"""Workloads of the gated linear recurrence, the short causal convolution and
the group norm.

Each case is one call, or one training step, of

* the gated linear recurrence ``h_t = a_t h_{t-1} + b_t u_t x_t`` on each channel
  of (batch, tokens, channels), with ``u = sigmoid(input_gate)`` (1 without one)
  and, with a decay, ``a = exp(log_decay * sigmoid(gate))``, ``b = sqrt(1 - a^2)``,
  without one ``a = sigmoid(gate)``, ``b = 1 - a`` -- a prompt ("recur"), a
  training step ("recur train"), one token of every sequence ("recur step");
* the causal convolution of each channel with a few taps, and an activation:
  ``y_t = act(bias + sum_j weight_j x_{t - taps + 1 + j})`` -- the same three;
* the group norm of each token's channels, times an activated gate:
  ``y = act(gate) * ((x - mean) / sqrt(var + eps) * weight + bias)``, or
  ``act`` of the normed value without a gate -- a call, or a training step.

``run`` computes them in elementary torch operations, or, with ``own`` set,
calls this repository's operators.
"""

import math

import torch

own = False

_EPS = 1e-5


# --------------------------------------------------------------------- cases
def listed():
    recur = {"op": "recur", "dtype": "bfloat16", "decay": True, "input_gate": True,
             "state": False, "lengths": False, "sliced": False}
    conv = {"op": "conv", "dtype": "bfloat16", "taps": 4, "silu": True, "bias": True,
            "state": False, "lengths": False, "sliced": False}
    norm = {"op": "norm", "dtype": "bfloat16", "gate": True, "silu": True, "affine": True}
    return [
        # the long-context shape of the framework's own benchmark, 16 heads of 64 wide
        dict(recur, name="recur t32768 c1024", b=8, t=32768, c=1024),
        # one long prompt whose state the decoding starts from, gates as slices of one product
        dict(recur, name="recur b1 t16384 c2048", b=1, t=16384, c=2048, state=True, sliced=True),
        # an ordinary training step
        dict(recur, name="recur train t4096 c1024", op="recur train", b=4, t=4096, c=1024),
        # full precision, an odd width, sequences of unlike lengths, the gate alone as the decay
        dict(recur, name="recur train fp32 t333 c57", op="recur train", b=3, t=333, c=57,
             dtype="float32", decay=False, input_gate=False, state=True, lengths=True),
        # one token of one sequence: latency
        dict(recur, name="recur step b1 c1024", op="recur step", b=1, c=1024),
        # one token of every sequence of a full server
        dict(recur, name="recur step b256 c4096", op="recur step", b=256, c=4096),
        # the convolution ahead of the recurrence: a training step, a ragged batch of prompts
        dict(conv, name="conv train t4096 c1024", op="conv train", b=4, t=4096, c=1024),
        dict(conv, name="conv t1000 c1300", b=5, t=1000, c=1300, state=True, lengths=True,
             sliced=True),
        # its single token
        dict(conv, name="conv step b64 c2048", op="conv step", b=64, c=2048),
        # the norm of the heads' outputs with the block's gate: a training step
        dict(norm, name="norm train 16384x1024", op="norm train", rows=16384, c=1024, groups=16),
        # decoding: a few rows
        dict(norm, name="norm 8x1024", rows=8, c=1024, groups=16),
        # an activation without a gate, odd groups, full precision
        dict(norm, name="norm train fp32 2000x399", op="norm train", rows=2000, c=399, groups=7,
             dtype="float32", gate=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, most):
    """A number of channels: every other one a multiple of 64, the others any."""
    c = _log_int(rng, 16, most)
    return max(64, c // 64 * 64) if rng.random() < 0.5 else c


def draw(rng):
    op = rng.choice(["recur", "recur train", "recur step", "conv", "conv train", "conv step",
                     "norm", "norm train"])
    case = {"op": op, "dtype": rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])}
    if op.startswith("norm"):
        groups = _log_int(rng, 1, 64)
        size = _log_int(rng, 4, 4096 // groups)
        if rng.random() < 0.5:
            size = max(8, size // 8 * 8)
        c = groups * size
        return dict(case, rows=_log_int(rng, 1, min(32768, (1 << 25) // c)), c=c, groups=groups,
                    gate=rng.random() < 0.7, silu=rng.random() < 0.7, affine=rng.random() < 0.7)
    case["sliced"] = rng.random() < 0.3
    if op.endswith("step"):
        case.update(b=_log_int(rng, 1, 512), c=_width(rng, 8192))
    else:
        t = _log_int(rng, 1, 8192 if op.endswith("train") else 32768)
        c = _width(rng, 4096)
        case.update(t=t, c=c, b=_log_int(rng, 1, max(1, min(64, (1 << 25) // (t * c)))),
                    state=rng.random() < 0.5, lengths=rng.random() < 0.3)
    if op.startswith("recur"):
        return dict(case, decay=rng.random() < 0.7, input_gate=rng.random() < 0.7)
    return dict(case, taps=rng.choice([2, 3, 4, 4, 4]), silu=rng.random() < 0.7,
                bias=rng.random() < 0.7)


# -------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(to)

    op, c = case["op"], case["c"]
    s = {"op": op, "names": []}
    if op.startswith("norm"):
        rows = case["rows"]
        s.update(x=normal(rows, c, scale=2.0), groups=case["groups"], names=["x"],
                 weight=None, bias=None, gate=None, activation="silu" if case["silu"] else None)
        if case["affine"]:
            s["weight"] = (1.0 + normal(c, scale=0.2, to=torch.float32)).to(dtype)
            s["bias"] = normal(c, scale=0.2)
            s["names"] += ["weight", "bias"]
        if case["gate"]:
            s["gate"] = normal(rows, c)
            s["names"].append("gate")
        if op == "norm train":
            s["d_out"] = normal(rows, c)
            for n in s["names"]:
                s[n].requires_grad_()
        return s
    b = case["b"]
    step, train = op.endswith("step"), op.endswith("train")
    shape = (b, c) if step else (b, case["t"], c)

    def rows_of(n):
        """n tensors of the tokens, or of them as slices of one projection's output."""
        if case.get("sliced"):
            return list(normal(*shape[:-1], n * c).split(c, -1))
        return [normal(*shape) for _ in range(n)]

    if op.startswith("recur"):
        n = 3 if case["input_gate"] else 2
        s.update(zip(("x", "gate", "input_gate"), rows_of(n) + [None] * (3 - n)))
        s.update(log_decay=None, state=None, names=["x", "gate"])
        if case["input_gate"]:
            s["names"].append("input_gate")
        if case["decay"]:
            # half-open gates keep 0.9 to 0.999 of the state for each token
            keep = 0.9 + 0.099 * torch.rand(c, generator=gen, device="cuda")
            s["log_decay"] = 2.0 * torch.log(keep)
            s["names"].append("log_decay")
        if step or case["state"]:
            s["state"] = normal(b, c, to=torch.float32)
            if not step:
                s["names"].append("state")
    else:
        taps = case["taps"]
        s.update(x=rows_of(1)[0], weight=normal(c, taps, scale=taps ** -0.5), bias=None,
                 state=None, activation="silu" if case["silu"] else None, names=["x", "weight"])
        if case["bias"]:
            s["bias"] = normal(c, scale=0.2)
            s["names"].append("bias")
        if step or case["state"]:
            s["state"] = normal(b, taps - 1, c)
            if not step:
                s["names"].append("state")
    if step:
        return s
    s["want_state"], s["lengths"] = case["state"], None
    if case["lengths"]:
        s["lengths"] = torch.randint(case["t"] // 2, case["t"] + 1, (b,), generator=gen,
                                     device="cuda")
    if train:
        s["d_out"] = normal(*shape)
        s["d_state"] = None if s["state"] is None else normal(*s["state"].shape, to=s["state"].dtype)
        for n in s["names"]:
            s[n] = s[n].detach().requires_grad_()
    return s


# --------------------------------------------------------------- plain forms
def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t over dimension 1, in place of b: by doubling
    within blocks of 64 tokens, and again over the blocks' ends."""
    t = b.shape[1]
    if t > 64:
        n = -(-t // 64)
        pad = (0, 0, 0, n * 64 - t)
        a, b = (torch.nn.functional.pad(x, pad).unflatten(1, (n, 64)).flatten(0, 1).clone()
                for x in (a, b))
        a, b = _doubled(a, b)
        a, b = (x.unflatten(0, (-1, n)) for x in (a, b))
        end = _scan(a[:, :, -1].clone(), b[:, :, -1].clone())
        b[:, 1:] += a[:, 1:] * end[:, :-1, None]
        return b.flatten(1, 2)[:, :t]
    return _doubled(a.clone(), b.clone())[1]


def _doubled(a, b):
    d = 1
    while d < b.shape[1]:
        b[:, d:] += a[:, d:] * b[:, :-d]
        a[:, d:] = a[:, d:] * a[:, :-d]
        d *= 2
    return a, b


def _sigmoid(x):
    return 1.0 / (1.0 + torch.exp(-x))


def _gates(s):
    """a, b, u and sigmoid(gate) in fp32."""
    r = _sigmoid(s["gate"].detach().float())
    u = 1.0 if s["input_gate"] is None else _sigmoid(s["input_gate"].detach().float())
    if s["log_decay"] is None:
        return r, 1.0 - r, u, r
    la = s["log_decay"].detach() * r
    return torch.exp(la), torch.sqrt(-torch.expm1(2.0 * la)), u, r


def _inside(s):
    """Which tokens a sequence has, (b, t, 1), or None for all."""
    if s["lengths"] is None:
        return None
    return (torch.arange(s["x"].shape[1], device="cuda") < s["lengths"][:, None])[..., None]


def _recur(s):
    x = s["x"].detach().float()
    dtype = s["x"].dtype
    a, b, u, r = _gates(s)
    ux = u * x
    add, inside = b * ux, _inside(s)
    if inside is not None:
        a = torch.where(inside, a, 1.0)
        add = torch.where(inside, add, 0.0)
    if s["state"] is not None:
        add[:, 0] += a[:, 0] * s["state"].detach()
    h = _scan(a, add)
    del add
    got = {"out": (h if inside is None else torch.where(inside, h, 0.0)).to(dtype)}
    if s["want_state"]:
        got["state"] = h[:, -1].clone()
    if s["op"] == "recur":
        return got
    g = s["d_out"].to(torch.float32, copy=True)  # (the final state's gradient is added to it)
    if inside is not None:
        g = torch.where(inside, g, 0.0)
    if s["d_state"] is not None:
        g[:, -1] += s["d_state"]
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)  # h_t's part in h_{t+1}
    g = _scan(after.flip(1), g.flip(1)).flip(1)
    before = torch.zeros_like(h[:, 0]) if s["state"] is None else s["state"].detach()
    before = torch.cat([before[:, None], h[:, :-1]], 1)
    d_state = a[:, 0] * g[:, 0]
    if inside is not None:
        g = torch.where(inside, g, 0.0)
    if s["log_decay"] is None:
        d_gate = g * (before - ux) * r * (1.0 - r)
    else:
        d_log = g * (a * before - a * a * ux / b)
        d_gate = d_log * s["log_decay"].detach() * r * (1.0 - r)
        got["d_log_decay"] = (d_log * r).sum((0, 1), dtype=torch.float64).float()
    got.update(dx=(g * b * u).to(dtype), d_gate=d_gate.to(dtype))
    if s["input_gate"] is not None:
        got["d_input_gate"] = (g * b * ux * (1.0 - u)).to(dtype)
    if s["d_state"] is not None:
        got["d_state"] = d_state
    return got


def _act(z, name):
    return z if name is None else z * _sigmoid(z)


def _d_act(z, name):
    if name is None:
        return torch.ones_like(z)
    r = _sigmoid(z)
    return r * (1.0 + z * (1.0 - r))


def _conv(s):
    x, w = s["x"].detach(), s["weight"].detach().float()
    b, t, c = x.shape
    dtype, taps = x.dtype, w.shape[1]
    before = x.new_zeros(b, taps - 1, c) if s["state"] is None else s["state"].detach()
    whole = torch.cat([before, x], 1).float()
    inside = _inside(s)
    z = sum(w[:, j] * whole[:, j:j + t] for j in range(taps))
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    y = _act(z, s["activation"])
    got = {"out": (y if inside is None else torch.where(inside, y, 0.0)).to(dtype)}
    at = (torch.full((b,), t, device="cuda") if s["lengths"] is None else s["lengths"])
    at = (at[:, None] + torch.arange(taps - 1, device="cuda"))[..., None].expand(-1, -1, c)
    if s["want_state"]:
        got["state"] = whole.gather(1, at).to(dtype)
    if s["op"] == "conv":
        return got
    g = s["d_out"].float() * _d_act(z, s["activation"])
    if inside is not None:
        g = torch.where(inside, g, 0.0)
    d_whole = torch.zeros_like(whole)
    for j in range(taps):
        d_whole[:, j:j + t] += w[:, j] * g
    if s["d_state"] is not None:
        d_whole.scatter_add_(1, at, s["d_state"].float())
    got["dx"] = d_whole[:, taps - 1:].to(dtype)
    got["d_weight"] = torch.stack(
        [(g * whole[:, j:j + t]).sum((0, 1), dtype=torch.float64) for j in range(taps)],
        -1).to(dtype)
    if s["bias"] is not None:
        got["d_bias"] = g.sum((0, 1), dtype=torch.float64).to(dtype)
    if s["d_state"] is not None:
        got["d_state"] = d_whole[:, :taps - 1].to(dtype)
    return got


def _norm(s):
    x = s["x"].detach().float().unflatten(-1, (s["groups"], -1))
    dtype, act = s["x"].dtype, s["activation"]
    x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    n = (x * r).flatten(-2)
    w = 1.0 if s["weight"] is None else s["weight"].detach().float()
    z = n * w
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    gate = None if s["gate"] is None else s["gate"].detach().float()
    got = {"out": (_act(z, act) if gate is None else z * _act(gate, act)).to(dtype)}
    if s["op"] == "norm":
        return got
    g = s["d_out"].float()
    if gate is None:
        g = g * _d_act(z, act)
    else:
        got["d_gate"] = (g * z * _d_act(gate, act)).to(dtype)
        g = g * _act(gate, act)
    if s["weight"] is not None:
        got["d_weight"] = (g * n).sum(0, dtype=torch.float64).to(dtype)
        got["d_bias"] = g.sum(0, dtype=torch.float64).to(dtype)
    g, n = ((g * w).unflatten(-1, (s["groups"], -1)), n.unflatten(-1, (s["groups"], -1)))
    dx = r * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    got["dx"] = dx.flatten(-2).to(dtype)
    return got


def _plain(s):
    op = s["op"]
    if op == "recur step":
        a, b, u, _ = _gates(s)
        s["state"].mul_(a).add_(b * u * s["x"].float())
        return {"out": s["state"].to(s["x"].dtype), "state": s["state"]}
    if op == "conv step":
        whole = torch.cat([s["state"], s["x"][:, None]], 1)
        z = (whole.float() * s["weight"].float().T).sum(1)
        if s["bias"] is not None:
            z = z + s["bias"].float()
        s["state"].copy_(whole[:, 1:])
        return {"out": _act(z, s["activation"]).to(s["x"].dtype), "state": s["state"]}
    return {"r": _recur, "c": _conv, "n": _norm}[op[0]](s)


# ---------------------------------------------------------------------- run
_GRADS = {"x": "dx", "state": "d_state"}


def run(s):
    if not own:
        return _plain(s)
    import trainium_linear_attention_b200 as T

    op = s["op"]
    if op == "recur step":
        out = T.gated_recurrence_step(s["x"], s["gate"], s["state"], log_decay=s["log_decay"],
                                      input_gate=s["input_gate"])
        return {"out": out, "state": s["state"]}
    if op == "conv step":
        out = T.causal_conv_step(s["x"], s["weight"], s["state"], bias=s["bias"],
                                 activation=s["activation"])
        return {"out": out, "state": s["state"]}
    if op.startswith("norm"):
        outs = T.group_norm(s["x"], s["groups"], weight=s["weight"], bias=s["bias"],
                            gate=s["gate"], activation=s["activation"], eps=_EPS),
    else:
        if op.startswith("recur"):
            got = T.gated_recurrence(s["x"], s["gate"], log_decay=s["log_decay"],
                                     input_gate=s["input_gate"], initial_state=s["state"],
                                     return_state=s["want_state"], lengths=s["lengths"])
        else:
            got = T.causal_conv(s["x"], s["weight"], bias=s["bias"], activation=s["activation"],
                                initial_state=s["state"], return_state=s["want_state"],
                                lengths=s["lengths"])
        outs = got if s["want_state"] else (got,)
    got = {n: y.detach() for n, y in zip(("out", "state"), outs)}
    if op.endswith("train"):
        ups = (s["d_out"], s["d_state"]) if len(outs) == 2 else (s["d_out"],)
        grads = torch.autograd.grad(outs, [s[n] for n in s["names"]], ups)
        got.update((_GRADS.get(n, "d_" + n), g) for n, g in zip(s["names"], grads))
    return got


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    op, c = case["op"], case["c"]
    train = op.endswith("train")
    if op.startswith("norm"):
        n = case["rows"] * c
        # x, y, the gate; in training d_y, dx, the gate's gradient
        tensors = (5 if case["gate"] else 4) + (1 if case["gate"] else 0) if train else \
            (3 if case["gate"] else 2)
        affine = 2 * c * size * (2 if train else 1) if case["affine"] else 0
        return {"bytes": n * size * tensors + affine, "flops": n * (30 if train else 12)}
    n = case["b"] * case.get("t", 1) * c
    gates = 1 + case["input_gate"] if op.startswith("recur") else 0
    # x and the gates, the output; in training its gradient and those of the inputs
    tensors = (1 + gates) * (2 if train else 1) + (2 if train else 1)
    if op.startswith("recur"):
        entry, fixed, flops = 4, 4 * c * (2 if train else 1) if case["decay"] else 0, 24
        entries = case["b"] * c
    else:
        entry, flops = size, 2 * case["taps"] + 4
        fixed = c * size * (case["taps"] + case["bias"]) * (2 if train else 1)
        entries = case["b"] * c * (case["taps"] - 1)
    states = 0
    if op.endswith("step") or case["state"]:  # read, written; their gradients
        states = 2 * entry * entries * (2 if train else 1)
    return {"bytes": n * size * tensors + fixed + states, "flops": n * flops * (3 if train else 1)}


# -------------------------------------------------------------------- exact
def _token_by_token(x, gate, input_gate, log_decay, state, lengths):
    """The recurrence as it is defined, one token after another, in 64 bits."""
    keep = torch.sigmoid(gate)
    if log_decay is None:
        add = (1.0 - keep) * x
    else:
        log_keep = log_decay * keep
        keep = log_keep.exp()
        add = (-torch.expm1(2.0 * log_keep)).sqrt() * x
    if input_gate is not None:
        add = add * torch.sigmoid(input_gate)
    h, outs = state, []
    for i, (a, b) in enumerate(zip(keep.unbind(1), add.unbind(1))):
        new = torch.addcmul(b, a, h)
        if lengths is None:
            h = new
            outs.append(h)
        else:
            live = (i < lengths)[:, None]
            h = torch.where(live, new, h)
            outs.append(torch.where(live, new, 0.0))
    return torch.stack(outs, 1), h


def _convolved(x, weight, bias, state, silu, lengths):
    b, t, c = x.shape
    taps = weight.shape[1]
    whole = torch.cat([state, x], 1)
    y = torch.einsum("btcj,cj->btc", whole.unfold(1, taps, 1), weight)
    if bias is not None:
        y = y + bias
    if silu:
        y = torch.nn.functional.silu(y)
    if lengths is None:
        return y, whole[:, t:]
    ends = [whole[i, n:n + taps - 1] for i, n in enumerate(lengths.tolist())]
    live = torch.arange(t, device=x.device)[None] < lengths[:, None]
    return torch.where(live[..., None], y, 0.0), torch.stack(ends)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    wide = {n: v.detach().double() for n, v in s.items()
            if isinstance(v, torch.Tensor) and n != "lengths"}
    step, train = op.endswith("step"), op.endswith("train")
    if train:
        for n in s["names"]:
            wide[n].requires_grad_()
    if op.startswith("norm"):
        y = torch.nn.functional.group_norm(wide["x"], case["groups"], wide.get("weight"),
                                           wide.get("bias"), _EPS)
        act = torch.nn.functional.silu if case["silu"] else (lambda v: v)
        outs = (y * act(wide["gate"]) if case["gate"] else act(y),)
    else:
        x, lengths = wide["x"], s.get("lengths")
        if step:
            x = x[:, None]
        if op.startswith("recur"):
            gate, input_gate = (None if wide.get(n) is None else wide[n].view(x.shape)
                                for n in ("gate", "input_gate"))
            state = wide.get("state")
            if state is None:
                state = x.new_zeros(x.shape[0], x.shape[2])
            outs = _token_by_token(x, gate, input_gate, wide.get("log_decay"), state, lengths)
        else:
            state = wide.get("state")
            if state is None:
                state = x.new_zeros(x.shape[0], case["taps"] - 1, x.shape[2])
            outs = _convolved(x, wide["weight"], wide.get("bias"), state, case["silu"], lengths)
        if step:
            outs = (outs[0][:, 0], outs[1])
        elif not s["want_state"]:
            outs = outs[:1]
    got = {n: y.detach() for n, y in zip(("out", "state"), outs)}
    if train:
        ups = [wide["d_out"]] + ([wide["d_state"]] if len(outs) == 2 else [])
        grads = torch.autograd.grad(outs, [wide[n] for n in s["names"]], ups)
        got.update((_GRADS.get(n, "d_" + n), g) for n, g in zip(s["names"], grads))
    return got
