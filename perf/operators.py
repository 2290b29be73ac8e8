"""Performance cases of the selective state space operators and of distillation.

``listed()`` names the cases, ``draw(rng)`` makes one more of the same ranges,
``prepare(case, seed)`` makes what a program has in hand before the call,
``run(state)`` is one pass and ``work(case)`` what a pass cannot do without.
With ``own`` false the operators are computed in plain form: elementary torch
operations in 32 bits, each output rounded once.  With ``own`` true ``run``
calls ``causal_conv``, ``causal_conv_step``, ``selective_scan`` and
``selective_step`` of ``bayes_ssm.selective`` and
``bayes_ssm.distill.distillation_loss``.  ``exact(case, seed)`` computes
the same outputs in 64 bits by other means.

The operators, per sequence and channel:

* ``conv`` / ``conv_step``: depthwise causal convolution of a few taps,
  optional bias and SiLU, with the last inputs as its state;
* ``scan`` / ``step``: ``d = softplus(step + bias)``, ``h = exp(d A) h + d x k``,
  ``y = (q . h + skip x) silu(gate)`` with a state of N values per channel;
* ``distill``: ``tau^2 KL(p || q)`` of a teacher's softmax over its top logits
  against the student's softmax over the vocabulary, with its gradient.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _package():
    root = str(Path(__file__).resolve().parents[1] / "bayes-ssm_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from bayes_ssm import distill, selective
    return selective, distill


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _conv(name, dtype, batch, tokens, channels, taps, *, silu, bias, state, train, packed=0):
    return dict(name=name, op="conv", dtype=dtype, batch=batch, tokens=tokens, channels=channels, taps=taps,
                silu=silu, bias=bias, state=state, train=train, packed=packed)


def _scan(name, dtype, batch, tokens, channels, states, groups, *, gate, skip, state, train, packed=0):
    return dict(name=name, op="scan", dtype=dtype, batch=batch, tokens=tokens, channels=channels, states=states,
                groups=groups, gate=gate, skip=skip, state=state, train=train, packed=packed)


def listed():
    return [
        # one layer's convolution in a training step: 8 sequences of 2,048 tokens, 2,048 channels
        _conv("conv_train", "bf16", 8, 2048, 2048, 4, silu=True, bias=True, state=False, train=True),
        # prompts of uneven length (some empty) packed one after the other, an odd channel count, continued
        # from the states that earlier chunks of the same prompts left
        _conv("conv_prompts", "f32", 37, 700, 771, 3, silu=False, bias=False, state=True, train=False, packed=1),
        # one new token for each of 64 sequences
        dict(name="conv_token", op="conv_step", dtype="f16", batch=64, channels=2048, taps=4, silu=True, bias=True),
        # one long prompt: few rows and a long axis
        _scan("scan_prompt", "bf16", 1, 8192, 1024, 16, 1, gate=True, skip=True, state=False, train=False),
        # a batch of uneven prompts packed one after the other, continued from their states
        _scan("scan_prompts", "bf16", 24, 1500, 2048, 16, 1, gate=True, skip=True, state=True, train=False,
              packed=2),
        # one layer's scan in a training step, forward and backward
        _scan("scan_train", "bf16", 8, 2048, 1024, 16, 1, gate=True, skip=True, state=False, train=True),
        # a small odd model in full precision: two groups of keys and queries, 10 states, a given start
        _scan("scan_train_odd", "f32", 3, 333, 202, 10, 2, gate=False, skip=True, state=True, train=True),
        # one new token of a single sequence: latency
        dict(name="token_one", op="step", dtype="bf16", batch=1, channels=1024, states=16, groups=1, gate=True,
             skip=True),
        # one new token for each of 256 sequences of a wide layer: the states' traffic
        dict(name="token_batch", op="step", dtype="bf16", batch=256, channels=4096, states=16, groups=1, gate=True,
             skip=True),
        # a training step's logits in 16 bits: 8,192 tokens, vocabulary 32,000
        dict(name="distill_train", op="distill", dtype="bf16", rows=8192, vocab=32000, top=64, temperature=2.0,
             empty=0.05),
        # the 32-bit logits of the tied head
        dict(name="distill_head", op="distill", dtype="f32", rows=2048, vocab=32000, top=32, temperature=1.0,
             empty=0.0),
        # a handful of rows of a large odd vocabulary: latency, split rows
        dict(name="distill_few", op="distill", dtype="bf16", rows=4, vocab=50001, top=8, temperature=1.5,
             empty=0.25),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random):
    op = rng.choice(["conv", "conv_step", "scan", "scan", "step", "distill", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    if op == "conv":
        channels = _log_int(rng, 32, 4096)
        batch = _log_int(rng, 1, 64)
        tokens = _log_int(rng, 1, max(1, min(4096, 8 * 2048 * 2048 // (batch * channels))))
        return dict(op=op, dtype=dtype, batch=batch, tokens=tokens, channels=channels, taps=rng.choice([2, 3, 4, 4]),
                    silu=rng.random() < 0.7, bias=rng.random() < 0.5, state=rng.random() < 0.5,
                    train=rng.random() < 0.5, packed=rng.choice([0, rng.randint(1, 1000)]))
    if op == "conv_step":
        return dict(op=op, dtype=dtype, batch=_log_int(rng, 1, 512), channels=_log_int(rng, 32, 4096),
                    taps=rng.choice([2, 3, 4, 4]), silu=rng.random() < 0.7, bias=rng.random() < 0.5)
    if op == "scan":
        states = rng.choice([4, 8, 10, 16, 16, 16, 32, 64])
        groups = rng.choice([1, 1, 1, 2, 4])
        channels = groups * _log_int(rng, 16, 2048 // groups)
        batch = _log_int(rng, 1, 32)
        room = 8 * 2048 * 1024 * 16 // (batch * channels * states)
        train = rng.random() < 0.5
        tokens = _log_int(rng, 1, max(1, min(2048 if train else 8192, room)))
        return dict(op=op, dtype=dtype, batch=batch, tokens=tokens, channels=channels, states=states, groups=groups,
                    gate=rng.random() < 0.7, skip=rng.random() < 0.8, state=rng.random() < 0.5, train=train,
                    packed=rng.choice([0, rng.randint(1, 1000)]))
    if op == "step":
        states = rng.choice([4, 8, 10, 16, 16, 16, 32, 64])
        groups = rng.choice([1, 1, 1, 2, 4])
        channels = groups * _log_int(rng, 16, 4096 // groups)
        batch = _log_int(rng, 1, max(1, min(512, 256 * 4096 * 16 // (channels * states))))
        return dict(op=op, dtype=dtype, batch=batch, channels=channels, states=states, groups=groups,
                    gate=rng.random() < 0.7, skip=rng.random() < 0.8)
    vocab = _log_int(rng, 500, 130000)
    rows = _log_int(rng, 1, max(1, min(8192, 8192 * 32000 // (vocab * (2 if dtype == "f32" else 1)))))
    return dict(op=op, dtype=dtype, rows=rows, vocab=vocab, top=_log_int(rng, 1, 256),
                temperature=rng.choice([1.0, 1.0, 1.5, 2.0, 4.0]), empty=rng.choice([0.0, 0.1, 0.5]))


def _lengths(case):
    """Tokens of each sequence; uneven, zero and one among them, where the case is packed."""
    if not case["packed"]:
        return [case["tokens"]] * case["batch"]
    rng = random.Random(case["packed"] * 7919 + case["batch"])
    out = []
    for i in range(case["batch"]):
        if i % 8 == 3:
            out.append(0)
        elif i % 8 == 6:
            out.append(1)
        else:
            out.append(rng.randint(max(1, case["tokens"] // 4), case["tokens"]))
    return out


def work(case):
    op, e = case["op"], _BYTES[case["dtype"]]
    if op == "conv":
        n = sum(_lengths(case)) * case["channels"]
        states = case["batch"] * (case["taps"] - 1) * case["channels"] * e
        per = 2 * e + (2 * e if case["train"] else 0)  # x, y; the gradients of y and of x
        side = case["channels"] * (case["taps"] + int(case["bias"])) * e
        scale = 2 if case["train"] else 1
        return {"bytes": n * per + scale * (states * (2 if case["state"] else 1) + side),
                "flops": n * (2 * case["taps"] + (4 if case["silu"] else 0)) * (3 if case["train"] else 1)}
    if op == "conv_step":
        n = case["batch"] * case["channels"]
        return {"bytes": n * e * (2 + 2 * (case["taps"] - 1)) + case["channels"] * (case["taps"] + int(case["bias"])) * e,
                "flops": n * (2 * case["taps"] + (4 if case["silu"] else 0))}
    if op in ("scan", "step"):
        ch, n_states = case["channels"], case["states"]
        tokens = case["batch"] if op == "step" else sum(_lengths(case))
        n = tokens * ch
        io = n * e * (3 + int(case["gate"])) + tokens * case["groups"] * n_states * 2 * e  # x, steps, y, gate; k, q
        state = case["batch"] * ch * n_states * 4
        side = ch * n_states * 4 + ch * 4 * (1 + int(case["skip"]))
        if op == "step":
            return {"bytes": io + 2 * state + side, "flops": n * n_states * 7}
        total = io + side + state * (2 if case["state"] else 1)
        flops = n * n_states * 7
        if case["train"]:
            # gradients of x, steps, gate, keys and queries written, that of y read
            total += io + side + state * (1 if case["state"] else 0)
            flops += n * n_states * 16
        return {"bytes": total, "flops": flops}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * 2 * e + case["rows"] * case["top"] * (e + 8), "flops": n * 6}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _generator(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)
    return g


def prepare(case, seed):
    g = _generator(case, seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(to)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    op = case["op"]
    st = dict(case=case)
    if op in ("conv", "conv_step"):
        ch, taps = case["channels"], case["taps"]
        st["weight"] = normal(ch, taps, scale=taps ** -0.5)
        st["bias"] = normal(ch, scale=0.1) if case["bias"] else None
        if op == "conv_step":
            st["x"] = normal(case["batch"], ch)
            st["state"] = normal(case["batch"], taps - 1, ch)
            return st
        shape = (sum(_lengths(case)), ch) if case["packed"] else (case["batch"], case["tokens"], ch)
        st["x"] = normal(*shape)
        st["state"] = normal(case["batch"], taps - 1, ch) if case["state"] else None
        if case["train"]:
            st["grad"] = normal(*shape)
        leaves = ("x", "weight", "bias", "state")
    elif op in ("scan", "step"):
        ch, n, groups = case["channels"], case["states"], case["groups"]
        if op == "step":
            lead = (case["batch"],)
        else:
            lead = (sum(_lengths(case)),) if case["packed"] else (case["batch"], case["tokens"])
        st["values"] = torch.nn.functional.silu(normal(*lead, ch, to=torch.float32)).to(dtype)
        st["steps"] = normal(*lead, ch, scale=0.5)
        st["keys"] = normal(*lead, groups, n)
        st["queries"] = normal(*lead, groups, n)
        st["gate"] = normal(*lead, ch) if case["gate"] else None
        st["skip"] = 1.0 + 0.1 * normal(ch, to=torch.float32) if case["skip"] else None
        # decay rates 1..N per state, spread a little; steps of 1e-3..1e-1 after the softplus
        st["rates"] = -(1.0 + torch.arange(n, device="cuda", dtype=torch.float32)) * (0.75 + 0.5 * uniform(ch, n))
        base = torch.exp(uniform(ch) * math.log(100.0) + math.log(1e-3))
        st["step_bias"] = base + torch.log(-torch.expm1(-base))
        if op == "step":
            st["state"] = normal(case["batch"], ch, n, to=torch.float32)
            return st
        st["state"] = normal(case["batch"], ch, n, to=torch.float32) if case["state"] else None
        if case["train"]:
            st["grad"] = normal(*lead, ch)
            st["grad_state"] = normal(case["batch"], ch, n, scale=0.1, to=torch.float32) if case["state"] else None
        leaves = ("values", "steps", "rates", "keys", "queries", "skip", "gate", "step_bias", "state")
    else:
        rows, vocab, top = case["rows"], case["vocab"], min(case["top"], case["vocab"])
        logits = torch.empty(rows, vocab, device="cuda", dtype=dtype)
        values = torch.empty(rows, top, device="cuda", dtype=dtype)
        indices = torch.empty(rows, top, device="cuda", dtype=torch.int64)
        for lo in range(0, rows, 1024):
            part = torch.randn(min(1024, rows - lo), vocab, generator=g, device="cuda") * 2.5
            logits[lo:lo + 1024] = part.to(dtype)
            # the teacher agrees with the student in part: its top logits of a noisy copy
            v, i = torch.topk(part + torch.randn(part.shape, generator=g, device="cuda"), top, dim=-1)
            values[lo:lo + 1024], indices[lo:lo + 1024] = v.to(dtype), i
        # rows without a teacher (prompt positions): every entry is empty
        indices[uniform(rows) < case["empty"]] = -1
        st.update(logits=logits, teacher=values, indices=indices)
        leaves = ("logits",)
    if own:
        if case.get("packed"):
            st["sequences"] = _package()[0].PackedSequences(_lengths(case), device="cuda")
        if op == "distill" or case["train"]:
            st["leaves"] = [k for k in leaves if st[k] is not None]
            for k in st["leaves"]:
                st[k].requires_grad_(True)
    elif case.get("packed"):
        st["padded"] = _pad_index(case)
    return st


# ---------------------------------------------------------------------------
# The framework's operators
# ---------------------------------------------------------------------------

def _own(st):
    case = st["case"]
    selective, distill = _package()
    op = case["op"]
    if op == "conv_step":
        y = selective.causal_conv_step(st["x"], st["state"], st["weight"], st["bias"],
                                       activation="silu" if case["silu"] else None)
        return y, st["state"]
    if op == "step":
        y = selective.selective_step(st["values"], st["steps"], st["rates"], st["keys"], st["queries"], st["state"],
                                     skip=st["skip"], gate=st["gate"], step_bias=st["step_bias"], softplus=True)
        return y, st["state"]
    if op == "distill":
        loss = distill.distillation_loss(st["logits"], st["teacher"], st["indices"],
                                           temperature=case["temperature"])
        return loss, torch.autograd.grad(loss, st["logits"])[0]
    if op == "conv":
        out = selective.causal_conv(st["x"], st["weight"], st["bias"], activation="silu" if case["silu"] else None,
                                    initial_state=st["state"], sequences=st.get("sequences"))
        upstream = [st.get("grad"), None]
    else:
        out = selective.selective_scan(st["values"], st["steps"], st["rates"], st["keys"], st["queries"],
                                       skip=st["skip"], gate=st["gate"], step_bias=st["step_bias"], softplus=True,
                                       initial_state=st["state"], sequences=st.get("sequences"))
        upstream = [st.get("grad"), st.get("grad_state")]
    if not case["train"]:
        return tuple(out)
    ends = [(o, u) for o, u in zip(out, upstream) if u is not None]
    grads = torch.autograd.grad([o for o, _ in ends], [st[k] for k in st["leaves"]], [u for _, u in ends])
    return {"y": out[0].detach(), "final": out[1].detach(), **dict(zip(st["leaves"], grads))}


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def _pad_index(case):
    """Row of each (sequence, token) in the packed rows, and which of them exist."""
    lengths = torch.tensor(_lengths(case))
    starts = torch.cumsum(lengths, 0) - lengths
    t = torch.arange(max(1, int(lengths.max())))
    live = (t[None, :] < lengths[:, None]).cuda()
    index = (starts[:, None] + t[None, :]).clamp(max=max(0, int(lengths.sum()) - 1)).cuda()
    return index, live, lengths.cuda()


def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _silu_slope(x):
    s = 1.0 / (1.0 + torch.exp(-x))
    return s * (1.0 + x * (1.0 - s))


def _plain_conv(st):
    case = st["case"]
    dtype, taps = st["x"].dtype, case["taps"]
    x = st["x"].float()
    live = None
    if case["packed"]:
        index, live, lengths = st["padded"]
        x = torch.where(live[..., None], x[index], 0.0)
    else:
        lengths = torch.full((case["batch"],), case["tokens"], device="cuda")
    b, t, ch = x.shape
    past = st["state"].float() if st["state"] is not None else torch.zeros(b, taps - 1, ch, device="cuda")
    wide = torch.cat([past, x], 1)
    w = st["weight"].float()
    u = sum(wide[:, j:j + t] * w[:, j] for j in range(taps))
    if st["bias"] is not None:
        u = u + st["bias"].float()
    y = _silu(u) if case["silu"] else u
    # the last inputs of each sequence, older ones from the state it began with
    tail = (lengths[:, None] + torch.arange(taps - 1, device="cuda")[None, :])[..., None].expand(b, taps - 1, ch)
    final = torch.gather(wide, 1, tail)

    def rows(z):
        return z[live] if live is not None else z

    if not case["train"]:
        return rows(y).to(dtype), final.to(dtype)
    dy = st["grad"].float()
    if live is not None:
        dy = torch.where(live[..., None], dy[index], 0.0)
    du = dy * _silu_slope(u) if case["silu"] else dy
    dwide = torch.zeros_like(wide)
    for j in range(taps):
        dwide[:, j:j + t] += du * w[:, j]
    out = {"y": rows(y).to(dtype), "final": final.to(dtype), "x": rows(dwide[:, taps - 1:]).to(dtype),
           "weight": torch.stack([(du * wide[:, j:j + t]).sum((0, 1)) for j in range(taps)], 1).to(dtype)}
    if st["bias"] is not None:
        out["bias"] = du.sum((0, 1)).to(dtype)
    if st["state"] is not None:
        out["state"] = dwide[:, :taps - 1].to(dtype)
    return out


def _plain_conv_step(st):
    case = st["case"]
    wide = torch.cat([st["state"], st["x"][:, None]], 1)
    u = (wide.float() * st["weight"].float().t()).sum(1)
    if st["bias"] is not None:
        u = u + st["bias"].float()
    y = _silu(u) if case["silu"] else u
    st["state"].copy_(wide[:, 1:])
    return y.to(st["x"].dtype), st["state"]


def _softplus(x):
    return torch.clamp(x, min=0.0) + torch.log1p(torch.exp(-torch.abs(x)))


def _spread(z, channels):
    """Keys or queries [..., G, N] as each channel sees them, [..., C, N]."""
    return z.repeat_interleave(channels // z.shape[-2], dim=-2)


def _gather_groups(z, groups):
    """Sum of [..., C, N] over the channels of each group: [..., G, N]."""
    return z.reshape(*z.shape[:-2], groups, z.shape[-2] // groups, z.shape[-1]).sum(-2)


def _plain_scan(st):
    case = st["case"]
    dtype, ch, groups = st["values"].dtype, case["channels"], case["groups"]
    names = ("values", "steps", "keys", "queries", "gate", "grad")
    x, s, k, q, z, dy = (st[n].float() if st.get(n) is not None else None for n in names)
    live = None
    if case["packed"]:
        index, live, _ = st["padded"]
        x, s, k, q, z, dy = (None if v is None else v[index] for v in (x, s, k, q, z, dy))
    b, t = x.shape[:2]
    raw = s + st["step_bias"]
    d = _softplus(raw)
    if live is not None:
        d = d * live[..., None]  # a step of zero keeps the state
    rates, skip = st["rates"], st["skip"]
    h = st["state"].clone() if st["state"] is not None else torch.zeros(b, ch, case["states"], device="cuda")
    r = torch.empty_like(x)
    history = torch.empty(t + 1, *h.shape, device="cuda") if case["train"] else None
    if case["train"]:
        history[0] = h
    dx_in = d * x
    for i in range(t):
        h = torch.exp(d[:, i, :, None] * rates) * h + dx_in[:, i, :, None] * _spread(k[:, i], ch)
        r[:, i] = (h * _spread(q[:, i], ch)).sum(-1)
        if case["train"]:
            history[i + 1] = h
    if skip is not None:
        r = r + skip * x
    y = r if z is None else r * _silu(z)

    def rows(v):
        return v[live] if live is not None else v

    if not case["train"]:
        return rows(y).to(dtype), h
    if live is not None:
        dy = torch.where(live[..., None], dy, 0.0)
    dr = dy if z is None else dy * _silu(z)
    dx = torch.zeros_like(x) if skip is None else dr * skip
    dd = torch.empty_like(x)
    dk, dq = torch.empty_like(k), torch.empty_like(q)
    drates = torch.zeros_like(rates)
    carry = st["grad_state"].clone() if st["grad_state"] is not None else torch.zeros_like(h)
    for i in range(t - 1, -1, -1):
        kk, qq = _spread(k[:, i], ch), _spread(q[:, i], ch)
        a = torch.exp(d[:, i, :, None] * rates)
        gh = carry + qq * dr[:, i, :, None]
        dq[:, i] = _gather_groups(dr[:, i, :, None] * history[i + 1], groups)
        dk[:, i] = _gather_groups(gh * dx_in[:, i, :, None], groups)
        gk = (gh * kk).sum(-1)
        moved = gh * a * history[i]
        dx[:, i] += d[:, i] * gk
        dd[:, i] = (moved * rates).sum(-1) + x[:, i] * gk
        drates += (moved * d[:, i, :, None]).sum(0)
        carry = a * gh
    draw_ = dd / (1.0 + torch.exp(-raw))
    if live is not None:
        draw_ = draw_ * live[..., None]
    out = {"y": rows(y).to(dtype), "final": h, "values": rows(dx).to(dtype), "steps": rows(draw_).to(dtype),
           "rates": drates, "keys": rows(dk).to(dtype), "queries": rows(dq).to(dtype)}
    if skip is not None:
        out["skip"] = (dr * x).sum((0, 1))
    if z is not None:
        out["gate"] = rows(dy * r * _silu_slope(z)).to(dtype)
    out["step_bias"] = draw_.sum((0, 1))
    if st["state"] is not None:
        out["state"] = carry
    return out


def _plain_step(st):
    case = st["case"]
    ch = case["channels"]
    x, k, q = st["values"].float(), st["keys"].float(), st["queries"].float()
    d = _softplus(st["steps"].float() + st["step_bias"])
    h = torch.exp(d[..., None] * st["rates"]) * st["state"] + (d * x)[..., None] * _spread(k, ch)
    st["state"].copy_(h)
    r = (h * _spread(q, ch)).sum(-1)
    if st["skip"] is not None:
        r = r + st["skip"] * x
    if st["gate"] is not None:
        r = r * _silu(st["gate"].float())
    return r.to(st["values"].dtype), st["state"]


def _plain_distill(st):
    case = st["case"]
    tau = case["temperature"]
    live = st["indices"] >= 0
    counted = live.any(-1)
    index = st["indices"].clamp(min=0)
    t = torch.where(live, st["teacher"].float() / tau, -math.inf)
    top = t.amax(-1, keepdim=True)
    e = torch.where(live, torch.exp(t - torch.where(counted[:, None], top, 0.0)), 0.0)
    total = torch.where(counted[:, None], e.sum(-1, keepdim=True), 1.0)
    p = e / total
    log_p = torch.where(live, t - torch.where(counted[:, None], top, 0.0) - torch.log(total), 0.0)
    s = st["logits"].float() / tau
    m = s.amax(-1, keepdim=True)
    w = torch.exp(s - m)
    z = w.sum(-1, keepdim=True)
    log_q = torch.gather(s, 1, index) - m - torch.log(z)
    loss = (p * (log_p - log_q)).sum(-1) * tau * tau
    n = counted.sum().clamp(min=1)
    grad = w / z * (counted[:, None] * tau)
    grad.scatter_add_(1, index, p * -tau)
    return loss.sum() / n, (grad / n).to(st["logits"].dtype)


def run(state):
    if own:
        return _own(state)
    return {"conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan, "step": _plain_step,
            "distill": _plain_distill}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------

def _exact_sequences(case, st, name):
    """The rows of each sequence of one input, in 64 bits."""
    v = st[name]
    if v is None:
        return None
    v = v.detach().double()
    if case["packed"]:
        return list(torch.split(v, _lengths(case)))
    return list(v)


def _exact_conv(case, st):
    w = st["weight"].detach().double().requires_grad_(case["train"])
    bias = None if st["bias"] is None else st["bias"].detach().double().requires_grad_(case["train"])
    ys, finals, dxs, dstates = [], [], [], []
    grads = _exact_sequences(case, st, "grad") if case["train"] else None
    for i, x in enumerate(_exact_sequences(case, st, "x")):
        past = torch.zeros(case["taps"] - 1, case["channels"], device="cuda", dtype=torch.float64) \
            if st["state"] is None else st["state"][i].detach().double()
        x, past = x.requires_grad_(case["train"]), past.requires_grad_(case["train"])
        wide = torch.cat([past, x])
        u = torch.einsum("tcj,cj->tc", wide.unfold(0, case["taps"], 1), w) if x.shape[0] else x * 1.0
        if bias is not None:
            u = u + bias
        y = torch.nn.functional.silu(u) if case["silu"] else u
        if case["train"]:
            y.backward(grads[i])
            dxs.append(torch.zeros_like(x) if x.grad is None else x.grad)
            dstates.append(torch.zeros_like(past) if past.grad is None else past.grad)
        ys.append(y.detach())
        finals.append(wide.detach()[x.shape[0]:])
    join = torch.cat if case["packed"] else torch.stack
    y, final = join(ys), torch.stack(finals)
    if not case["train"]:
        return y, final
    out = {"y": y, "final": final, "x": join(dxs), "weight": w.grad if w.grad is not None else torch.zeros_like(w)}
    if bias is not None:
        out["bias"] = bias.grad if bias.grad is not None else torch.zeros_like(bias)
    if st["state"] is not None:
        out["state"] = torch.stack(dstates)
    return out


def _exact_recurrence(decay, inflow, h0):
    """All states of h_t = decay_t h_{t-1} + inflow_t by pairwise doubling over time."""
    inflow = torch.cat([inflow[:1] + decay[:1] * h0, inflow[1:]])
    span = 1
    while span < inflow.shape[0]:
        inflow = torch.cat([inflow[:span], inflow[span:] + decay[span:] * inflow[:-span]])
        decay = torch.cat([decay[:span], decay[span:] * decay[:-span]])
        span *= 2
    return inflow


def _exact_scan(case, st):
    train, ch, groups, n = case["train"], case["channels"], case["groups"], case["states"]
    width = ch // groups
    shared = {k: None if st[k] is None else st[k].detach().double().requires_grad_(train)
              for k in ("rates", "skip", "step_bias")}
    per = {k: _exact_sequences(case, st, k) for k in ("values", "steps", "keys", "queries", "gate")}
    grads = _exact_sequences(case, st, "grad") if train else None
    outs = {k: [] for k in ("y", "final", "values", "steps", "keys", "queries", "gate", "state")}
    for i in range(case["batch"]):
        leaf = {k: None if v is None else v[i].clone().requires_grad_(train) for k, v in per.items()}
        h0 = torch.zeros(ch, n, device="cuda", dtype=torch.float64) if st["state"] is None \
            else st["state"][i].detach().double()
        h0.requires_grad_(train)
        t = leaf["values"].shape[0]
        y_all = torch.empty(t, ch, device="cuda", dtype=torch.float64)
        last = h0.detach().clone()
        block = max(1, min(width, (1 << 24) // max(1, t * n)))
        for grp in range(groups):
            for lo in range(grp * width, (grp + 1) * width, block):
                c = slice(lo, min(lo + block, (grp + 1) * width))
                if t == 0:
                    if train and st["grad_state"] is not None:
                        h0[c].backward(st["grad_state"][i, c].double())
                    continue
                x, rate = leaf["values"][:, c], shared["rates"][c]
                d = torch.nn.functional.softplus(leaf["steps"][:, c] + shared["step_bias"][c], threshold=1000.0)
                h = _exact_recurrence(torch.exp(d[..., None] * rate),
                                      (d * x)[..., None] * leaf["keys"][:, grp, None, :], h0[c])
                r = torch.einsum("tcn,tn->tc", h, leaf["queries"][:, grp])
                if shared["skip"] is not None:
                    r = r + shared["skip"][c] * x
                y = r if leaf["gate"] is None else r * torch.nn.functional.silu(leaf["gate"][:, c])
                y_all[:, c] = y.detach()
                last[c] = h[-1].detach()
                if train:
                    ends, ups = [y], [grads[i][:, c]]
                    if st["grad_state"] is not None:
                        ends.append(h[-1])
                        ups.append(st["grad_state"][i, c].double())
                    torch.autograd.backward(ends, ups)
        outs["y"].append(y_all)
        outs["final"].append(last)
        if train:
            for k, v in leaf.items():
                if v is not None:
                    outs[k].append(torch.zeros_like(v) if v.grad is None else v.grad)
            outs["state"].append(torch.zeros_like(h0) if h0.grad is None else h0.grad)
    join = torch.cat if case["packed"] else torch.stack
    y, final = join(outs["y"]), torch.stack(outs["final"])
    if not train:
        return y, final
    out = {"y": y, "final": final}
    for k in ("values", "steps", "rates", "keys", "queries", "skip", "gate", "step_bias", "state"):
        if st[k] is None:
            continue
        if k in shared:
            out[k] = torch.zeros_like(shared[k]) if shared[k].grad is None else shared[k].grad
        else:
            out[k] = torch.stack(outs[k]) if k == "state" else join(outs[k])
    return out


def _exact_distill(case, st):
    tau = case["temperature"]
    rows, vocab = st["logits"].shape
    n = max(1, int((st["indices"] >= 0).any(-1).sum()))
    total = torch.zeros((), device="cuda", dtype=torch.float64)
    grad = torch.empty(rows, vocab, device="cuda", dtype=torch.float64)
    for lo in range(0, rows, 512):
        hi = min(rows, lo + 512)
        live = st["indices"][lo:hi] >= 0
        s = st["logits"][lo:hi].detach().double() / tau
        log_q = s - torch.logsumexp(s, -1, keepdim=True)
        t = torch.where(live, st["teacher"][lo:hi].double() / tau, -math.inf)
        log_p = torch.where(live, t - torch.logsumexp(t, -1, keepdim=True), 0.0)
        p = torch.where(live, torch.exp(log_p), 0.0)
        index = st["indices"][lo:hi].clamp(min=0)
        total += tau * tau * (p * (log_p - torch.gather(log_q, 1, index))).sum()
        dense = torch.zeros_like(s).scatter_add_(1, index, p)
        grad[lo:hi] = tau / n * (torch.exp(log_q) * live.any(-1, keepdim=True) - dense)
    return total / n, grad


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "conv":
        return _exact_conv(case, st)
    if op == "conv_step":
        wide = torch.cat([st["state"], st["x"][:, None]], 1).double()
        u = torch.einsum("bjc,cj->bc", wide, st["weight"].double())
        if st["bias"] is not None:
            u = u + st["bias"].double()
        return (torch.nn.functional.silu(u) if case["silu"] else u), wide[:, 1:]
    if op == "step":
        one = {k: st[k][:, None] for k in ("values", "steps", "keys", "queries") if st[k] is not None}
        one["gate"] = None if st["gate"] is None else st["gate"][:, None]
        y, final = _exact_scan(dict(case, train=False, packed=0), dict(st, **one))
        return y[:, 0], final
    if op == "scan":
        return _exact_scan(case, st)
    return _exact_distill(case, st)
