"""Workloads of the decayed linear attention and RMS norm operators.

Each case is one call, or one training step, of

* linear attention with a decay for each head: ``o_t = scale * q_t S_t`` with
  ``S_t = exp(g_h) S_{t-1} + k_t v_t^T`` -- a prompt at once ("prompt"), a
  training step with all gradients ("train"), one token per sequence ("step");
* the root-mean-square norm with the residual's addition -- a training step
  ("norm"), and a call whose output is held in e4m3 with fp32 scales ("fp8").

``run`` computes them in elementary fp32 torch operations, or, with ``own``
set, calls this repository's operators.
"""

import math

import torch

own = False

_EPS = 1e-6
_E4M3_MAX = 448.0
_AMAX_MIN = 2.0 ** -96


# --------------------------------------------------------------------- cases
def listed():
    attend = {"dtype": "bfloat16", "layout": "bhtd", "state": False}
    return [
        # the long-context shape of the framework's own benchmark: narrow keys, 128 heads
        dict(attend, name="prompt d16/64 t32768", op="prompt", b=8, h=16, t=32768, dk=16, dv=64),
        # a batch of ordinary prompts, heads as a projection leaves them
        dict(attend, name="prompt d64 t2048", op="prompt", b=4, h=16, t=2048, dk=64, dv=64,
             layout="bthd"),
        # one long prompt with wide heads, whose state the decoding starts from
        dict(attend, name="prompt d128 t16384", op="prompt", b=1, h=16, t=16384, dk=128, dv=128,
             layout="bthd", state=True),
        # the next piece of prompts that are read in pieces: short, ragged, seeded with a state
        dict(attend, name="prompt d64/128 t1000", op="prompt", b=3, h=5, t=1000, dk=64, dv=128,
             state=True),
        # an ordinary training step
        dict(attend, name="train d64 t4096", op="train", b=4, h=16, t=4096, dk=64, dv=64,
             layout="bthd"),
        # a step in full precision on a piece of a longer sequence (gradient of the state too)
        dict(attend, name="train fp32 d40/72 t333", op="train", b=2, h=3, t=333, dk=40, dv=72,
             dtype="float32", state=True),
        # one token of one sequence: latency
        dict(name="step b1 d64", op="step", dtype="bfloat16", b=1, h=16, dk=64, dv=64),
        # one token of every sequence of a full server: the states' traffic
        dict(name="step b256 d128", op="step", dtype="bfloat16", b=256, h=16, dk=128, dv=128),
        # the block's norm with its residual stream in training: 4 x 4096 tokens, 16 heads of 64
        dict(name="norm 16384x1024", op="norm", dtype="bfloat16", rows=16384, d=1024,
             residual=True, b=0, h=0),
        # the norm of each head's attention output, read through the transposed view
        dict(name="norm heads 64", op="norm", dtype="bfloat16", rows=4 * 2048 * 16, d=64,
             residual=False, b=4, h=16),
        # decoding: a few rows ahead of an 8-bit product
        dict(name="fp8 8x1024", op="fp8", dtype="bfloat16", rows=8, d=1024, group=0,
             residual=True),
        # a long prompt's rows ahead of an 8-bit product, a scale for each 128 values
        dict(name="fp8 32768x4096", op="fp8", dtype="bfloat16", rows=32768, d=4096, group=128,
             residual=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "train", "train", "step", "norm", "fp8"])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    if op in ("prompt", "train"):
        dk, dv = (rng.choice([16, 24, 32, 40, 57, 64, 64, 80, 96, 128, 128]) for _ in range(2))
        t = _log_int(rng, 1, 32768 if op == "prompt" else 8192)
        if dtype == "float32":
            t = min(t, 4096)
        # tokens times heads of all sequences, within the largest listed case
        most = max(1, (1 << 21 if op == "prompt" else 1 << 18) // t)
        bh = min(256, _log_int(rng, 1, most))
        h = rng.randint(1, min(bh, 32))
        return {"op": op, "dtype": dtype, "layout": rng.choice(["bhtd", "bthd"]),
                "state": rng.random() < 0.5, "b": max(1, bh // h), "h": h, "t": t,
                "dk": dk, "dv": dv}
    if op == "step":
        return {"op": op, "dtype": dtype, "b": _log_int(rng, 1, 256), "h": rng.randint(1, 16),
                "dk": rng.choice([16, 40, 57, 64, 96, 128]),
                "dv": rng.choice([16, 40, 57, 64, 96, 128])}
    if op == "norm":
        if rng.random() < 0.4:
            b, h, t = rng.randint(1, 4), rng.randint(1, 16), _log_int(rng, 1, 2048)
            return {"op": op, "dtype": dtype, "rows": b * h * t, "d": rng.choice([16, 40, 64, 128]),
                    "residual": False, "b": b, "h": h}
        return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, 8192),
                "d": _log_int(rng, 32, 8192), "residual": rng.random() < 0.7, "b": 0, "h": 0}
    group = rng.choice([0, 32, 64, 128])
    d = _log_int(rng, 64, 8192)
    if group:
        d = max(group, d // group * group)
    return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, 8192), "d": d, "group": group,
            "residual": rng.random() < 0.7}


# -------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(to)

    op = case["op"]
    s = {"op": op}
    if op in ("prompt", "train", "step"):
        b, h, dk, dv = case["b"], case["h"], case["dk"], case["dv"]
        # geometric slopes, from half a token's memory to hundreds of tokens
        s["log_decay"] = -torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda") / h).float()
        s["scale"] = 1.0 / math.sqrt(dk)
        if op == "step":
            s.update(q=normal(b, h, dk), k=normal(b, h, dk), v=normal(b, h, dv),
                     state=normal(b, h, dk, dv, scale=3.0, to=torch.float32))
            return s
        t = case["t"]

        def heads(d):
            if case["layout"] == "bthd":
                return normal(b, t, h, d).transpose(1, 2)
            return normal(b, h, t, d)

        s.update(q=heads(dk), k=heads(dk), v=heads(dv), state=None, want_state=case["state"])
        if case["state"]:
            s["state"] = normal(b, h, dk, dv, scale=3.0, to=torch.float32)
        if op == "train":
            s["d_out"] = heads(dv)
            s["d_state"] = (normal(b, h, dk, dv, to=torch.float32) if case["state"] else None)
            for n in ("q", "k", "v", "state"):
                if s[n] is not None:
                    s[n].requires_grad_()
        return s
    rows, d = case["rows"], case["d"]
    if op == "norm" and case["b"]:
        b, h = case["b"], case["h"]
        x = normal(b, h, rows // (b * h), d).transpose(1, 2)
    else:
        x = normal(rows, d)
    s.update(x=x, residual=normal(*x.shape, scale=2.0) if case["residual"] else None,
             weight=(1.0 + normal(d, scale=0.2, to=torch.float32)).to(dtype))
    if op == "norm":
        s.update(d_y=normal(*x.shape), d_sum=normal(*x.shape) if case["residual"] else None)
        for n in ("x", "weight", "residual"):
            if s[n] is not None:
                s[n].requires_grad_()
    else:
        s["group"] = case["group"] or None
    return s


# --------------------------------------------------------------- plain forms
def _attend(q, k, v, log_decay, scale, state, late):
    """Chunked form in fp32.  ``late`` = 1: the state holds the tokens before
    the chunk and decays once more before it is read; 0: it is read as it is
    (the reversed sums of the gradients).  Returns (out, final state)."""
    b, h, t, dk = q.shape
    dv = v.shape[-1]
    c = 128
    n = -(-t // c)
    g = log_decay.double()

    def power(exponent):  # (h, *exponent.shape), from 64-bit exponents
        e = exponent.double()
        return torch.exp(g.view(-1, *([1] * e.dim())) * e).float()

    def chunks(x):
        return torch.nn.functional.pad(x, (0, 0, 0, n * c - t)).reshape(b, h, n, c, x.shape[-1])

    i = torch.arange(c, device=q.device)
    lag = i[:, None] - i[None, :]
    inside = power(lag.clamp(min=0)) * (lag >= 0)
    qc, kc, vc = chunks(q), chunks(k), chunks(v)
    out = (qc @ kc.transpose(-1, -2) * inside[:, None]) @ vc
    added = (kc * power(c - late - i)[:, None, :, None]).transpose(-1, -2) @ vc
    m = torch.arange(n, device=q.device)
    gap = m[:, None] - m[None, :] - 1
    carry = power(gap.clamp(min=0) * c) * (gap >= 0)
    before = (carry @ added.reshape(b, h, n, dk * dv)).reshape(b, h, n, dk, dv)
    if state is not None:
        before = before + power(m * c)[:, :, None, None] * state[:, :, None]
    out = out + power(i + late)[:, None, :, None] * (qc @ before)
    out = (out * scale).reshape(b, h, n * c, dv)[:, :, :t]
    j = torch.arange(t, device=q.device)
    final = (k * power(t - late - j)[:, :, None]).transpose(-1, -2) @ v
    if state is not None:
        final = final + power(torch.tensor(t, device=q.device))[:, None, None] * state
    return out, final


def _attend_gradients(s):
    q, k, v, do = (s[n].detach().float() for n in ("q", "k", "v", "d_out"))
    state = None if s["state"] is None else s["state"].detach()
    d_state = s["d_state"]
    g, scale = s["log_decay"], s["scale"]

    def turned(x):
        return None if x is None else x.transpose(-1, -2)

    dq, _ = _attend(do, v, k, g, scale, turned(state), 1)
    qr, kr, vr, dor = (x.flip(2) for x in (q, k, v, do))
    dv, d_first = _attend(kr, qr * scale, dor, g, 1.0, d_state, 0)
    dk, _ = _attend(vr, dor * scale, qr, g, 1.0, turned(d_state), 0)
    return dq, dk.flip(2), dv.flip(2), d_first


def _norm(s):
    x = s["x"].detach().float()
    if s["residual"] is not None:
        x = x + s["residual"].detach().float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    return x, r, x * r * s["weight"].detach().float()


def _plain(s):
    op = s["op"]
    if op in ("prompt", "train"):
        dtype = s["q"].dtype
        state = None if s["state"] is None else s["state"].detach()
        out, final = _attend(*(s[n].detach().float() for n in ("q", "k", "v")), s["log_decay"],
                             s["scale"], state, 1)
        r = {"out": out.to(dtype)}
        if s["want_state"]:
            r["state"] = final
        if op == "train":
            dq, dk, dv, d_first = _attend_gradients(s)
            r.update(dq=dq.to(dtype), dk=dk.to(dtype), dv=dv.to(dtype))
            if s["want_state"]:
                r["d_state"] = d_first
        return r
    if op == "step":
        q, k, v = (s[n].float() for n in ("q", "k", "v"))
        lam = torch.exp(s["log_decay"].double()).float()
        state = s["state"]
        state.mul_(lam[:, None, None]).add_(k[..., :, None] * v[..., None, :])
        out = (q[..., None, :] @ state).squeeze(-2) * s["scale"]
        return {"out": out.to(s["q"].dtype), "state": state}
    x, r, y = _norm(s)
    dtype = s["x"].dtype
    if op == "norm":
        w, dy = s["weight"].detach().float(), s["d_y"].float()
        wdy = w * dy
        dx = r * (wdy - x * (r * r) * (wdy * x).mean(-1, keepdim=True))
        dw = (dy * x * r).reshape(-1, x.shape[-1]).sum(0)
        got = {"y": y.to(dtype), "dw": dw.to(dtype)}
        if s["residual"] is not None:
            dx = dx + s["d_sum"].float()
            got.update(sum=x.to(dtype), dr=dx.to(dtype))
        return dict(got, dx=dx.to(dtype))
    group = s["group"] or y.shape[-1]
    yg = y.reshape(*y.shape[:-1], -1, group)
    scales = yg.abs().amax(-1).clamp(min=_AMAX_MIN) / _E4M3_MAX
    y8 = (yg / scales[..., None]).reshape(y.shape).to(torch.float8_e4m3fn)
    got = {"y": y8, "scales": scales}
    if s["residual"] is not None:
        got["sum"] = x.to(dtype)
    return got


# ---------------------------------------------------------------------- run
def run(s):
    if not own:
        return _plain(s)
    import trainium_linear_attention_b200 as T

    op = s["op"]
    if op in ("prompt", "train"):
        r = T.decay_linear_attention(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"],
                                     initial_state=s["state"], return_state=s["want_state"])
        out, final = r if s["want_state"] else (r, None)
        got = {"out": out.detach()}
        if final is not None:
            got["state"] = final.detach()
        if op == "train":
            if final is None:
                grads = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["d_out"])
            else:
                grads = torch.autograd.grad((out, final), (s["q"], s["k"], s["v"], s["state"]),
                                            (s["d_out"], s["d_state"]))
                got["d_state"] = grads[3]
            got.update(dq=grads[0], dk=grads[1], dv=grads[2])
        return got
    if op == "step":
        out = T.decay_linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"],
                                            scale=s["scale"])
        return {"out": out, "state": s["state"]}
    if op == "norm":
        if s["residual"] is None:
            y = T.rms_norm(s["x"], s["weight"], eps=_EPS)
            dx, dw = torch.autograd.grad(y, (s["x"], s["weight"]), s["d_y"])
            return {"y": y.detach(), "dx": dx, "dw": dw}
        y, total = T.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=_EPS)
        dx, dr, dw = torch.autograd.grad((y, total), (s["x"], s["residual"], s["weight"]),
                                         (s["d_y"], s["d_sum"]))
        return {"y": y.detach(), "sum": total.detach(), "dx": dx, "dr": dr, "dw": dw}
    r = T.rms_norm_fp8(s["x"], s["weight"], residual=s["residual"], eps=_EPS,
                       group_size=s["group"])
    return dict(zip(("y", "scales", "sum"), r))


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    op = case["op"]
    if op in ("prompt", "train", "step"):
        b, h, dk, dv = case["b"], case["h"], case["dk"], case["dv"]
        state = b * h * dk * dv
        tokens = b * h * case.get("t", 1)
        if op == "step":  # the state read and written; decay, outer product, read-out
            return {"bytes": tokens * 2 * (dk + dv) * size + 8 * state, "flops": 5 * state}
        states = 4 * state if case["state"] else 0
        if op == "prompt":  # q, k, v, out; the recurrence's update and read-out
            return {"bytes": tokens * 2 * (dk + dv) * size + 2 * states,
                    "flops": 4 * tokens * dk * dv}
        # also d_out, dq, dk, dv; a second state for the reversed sums, three read-outs
        return {"bytes": tokens * 4 * (dk + dv) * size + 4 * states,
                "flops": 14 * tokens * dk * dv}
    n, d = case["rows"] * case["d"], case["d"]
    if op == "norm":  # x, y, d_y, dx (with a residual also it, the sum and its gradient)
        return {"bytes": n * size * (7 if case["residual"] else 4) + 2 * d * size, "flops": 12 * n}
    scales = 4 * case["rows"] * (d // case["group"] if case["group"] else 1)
    return {"bytes": n * (size * (3 if case["residual"] else 1) + 1) + d * size + scales,
            "flops": 6 * n}


# -------------------------------------------------------------------- exact
def _recurrence(q, k, v, g, scale, state):
    """The definition, 64 tokens at a time, in 64 bits; differentiable."""
    t, outs = q.shape[2], []
    for at in range(0, t, 64):
        qi, ki, vi = (x[:, :, at:at + 64] for x in (q, k, v))
        m = qi.shape[2]
        i = torch.arange(m, device=q.device, dtype=torch.float64)
        lag = i[:, None] - i[None, :]
        weight = torch.where(lag >= 0, torch.exp(g[:, None, None] * lag.clamp(min=0)), 0.0)
        o = torch.einsum("bhij,hij,bhjv->bhiv", torch.einsum("bhid,bhjd->bhij", qi, ki), weight, vi)
        o = o + torch.einsum("bhid,hi,bhdv->bhiv", qi, torch.exp(g[:, None] * (i + 1)), state)
        state = (torch.exp(g * m)[:, None, None] * state
                 + torch.einsum("bhjd,hj,bhjv->bhdv", ki, torch.exp(g[:, None] * (m - 1 - i)), vi))
        outs.append(o * scale)
    return torch.cat(outs, 2), state


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op in ("prompt", "train"):
        leaves = {n: s[n].detach().double() for n in ("q", "k", "v")}
        b, h = s["q"].shape[:2]
        leaves["state"] = (torch.zeros(b, h, case["dk"], case["dv"], device="cuda",
                                       dtype=torch.float64)
                           if s["state"] is None else s["state"].detach().double())
        if op == "train":
            for x in leaves.values():
                x.requires_grad_()
        out, final = _recurrence(leaves["q"], leaves["k"], leaves["v"], s["log_decay"].double(),
                                 s["scale"], leaves["state"])
        r = {"out": out.detach()}
        if s["want_state"]:
            r["state"] = final.detach()
        if op == "train":
            loss = (out * s["d_out"].double()).sum()
            if s["want_state"]:
                loss = loss + (final * s["d_state"].double()).sum()
            grads = torch.autograd.grad(loss, list(leaves.values()))
            r.update(zip(("dq", "dk", "dv"), grads))
            if s["want_state"]:
                r["d_state"] = grads[3]
        return r
    if op == "step":
        q, k, v, state = (s[n].double() for n in ("q", "k", "v", "state"))
        state = (torch.exp(s["log_decay"].double())[:, None, None] * state
                 + torch.einsum("bhd,bhv->bhdv", k, v))
        return {"out": torch.einsum("bhd,bhdv->bhv", q, state) * s["scale"], "state": state}
    x = s["x"].detach().double().requires_grad_()
    w = s["weight"].detach().double().requires_grad_()
    total = x if s["residual"] is None else x + s["residual"].detach().double()
    y = total / torch.sqrt(total.square().mean(-1, keepdim=True) + _EPS) * w
    if op == "norm":
        loss = (y * s["d_y"].double()).sum()
        if s["residual"] is not None:
            loss = loss + (total * s["d_sum"].double()).sum()
        dx, dw = torch.autograd.grad(loss, (x, w))
        r = {"y": y.detach(), "dx": dx, "dw": dw}
        if s["residual"] is not None:
            r.update(sum=total.detach(), dr=dx)
        return r
    y, total = y.detach(), total.detach()
    blocks = y.unflatten(-1, (-1, case["group"] or case["d"]))
    scales = blocks.abs().amax(-1).clamp(min=_AMAX_MIN) / _E4M3_MAX
    r = {"y": (blocks / scales.unsqueeze(-1)).flatten(-2), "scales": scales}
    if s["residual"] is not None:
        r["sum"] = total
    return r
