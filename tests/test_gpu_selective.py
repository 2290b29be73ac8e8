"""GPU: causal convolution and selective scan kernels vs plain 64-bit loops.

Outputs, final states and every gradient (autograd of the plain form in
float64 on the same inputs) are compared in relative L2.  Tolerances: an
output rounded once to bfloat16 (float16) is off by at most half an ulp,
2^-9 (2^-12) of itself, so 2.5e-3 (6e-4); in float32 a decay is good to
2^-22 (the multifunction unit's exp2) plus the rounding of its exponent, about
3.6e-7, and T of them multiply up, as a random walk sqrt(300) * 3.6e-7 = 6e-6
at the longest case: 2e-5 allows three times that.  The cases cover one token
to many tiles, odd channel and state counts, channel groups, every lane count
(N of 1..4, 5..8, 9..16, 17..32, 33..64), the alignments of the convolution's
vectors, empty and one-token sequences, and strided and broadcast operands.
"""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import plain_selective as plain
from bayes_ssm.selective import (PackedSequences, causal_conv, causal_conv_step, selective_scan, selective_step)

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-5, torch.bfloat16: 2.5e-3, torch.float16: 6e-4}
RAGGED = [0, 5, 1, 0, 40, 16, 17, 33, 0]


def close(got, want, tol, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    got, want = got.detach().double(), want.detach().double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    err = float((got - want).norm() / want.norm().clamp_min(1e-30)) if want.numel() else 0.0
    assert err <= tol, f"{what}: relative L2 error {err:.3e} above {tol:.1e}"


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rand(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def leaves64(*tensors):
    return [None if t is None else t.detach().double().requires_grad_() for t in tensors]


def leaves(*tensors):
    return [None if t is None else t.detach().requires_grad_() for t in tensors]


def grads(outs, ups, wrt):
    live = [w for w in wrt if w is not None]
    if isinstance(outs, tuple):  # an output that depends on none of them has no graph
        ends = [(o, u) for o, u in zip(outs, ups) if o.requires_grad]
        outs, ups = [o for o, _ in ends], [u for _, u in ends]
    got = iter(torch.autograd.grad(outs, live, ups, allow_unused=True))
    return [None if w is None else next(got) for w in wrt]


# ---------------------------------------------------------------------------
# convolution
# ---------------------------------------------------------------------------

# (lead or lengths, C, taps)
CONV = [((2, 37), 64, 4), ((1, 1), 8, 2), ((3, 2), 20, 4), ((2, 130), 33, 3), ((1, 70), 12, 4), ((5, 16), 256, 2),
        (RAGGED, 24, 4), (RAGGED, 7, 3), ([0, 0], 16, 4), ([3], 10, 2)]


def conv_inputs(shape, c, taps, dtype, seed, wdtype=None):
    g = gen(seed)
    lengths = shape if isinstance(shape, list) else None
    lead = (sum(shape),) if lengths is not None else shape
    count = len(shape) if lengths is not None else shape[0]
    x = rand(g, *lead, c, dtype=dtype)
    w = rand(g, c, taps, dtype=wdtype or dtype, scale=0.5)
    b = rand(g, c, dtype=wdtype or dtype, scale=0.2)
    s = rand(g, count, taps - 1, c, dtype=dtype)
    return x, w, b, s, lengths


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("silu,bias,state", [(True, True, True), (False, False, False), (True, False, True)])
@pytest.mark.parametrize("shape,c,taps", CONV)
def test_conv_forward_and_gradients(shape, c, taps, silu, bias, state, dtype):
    x, w, b, s, lengths = conv_inputs(shape, c, taps, dtype, 3 * c + taps)
    b, s = b if bias else None, s if state else None
    seqs = None if lengths is None else PackedSequences(lengths, device="cuda")
    act = "silu" if silu else None
    xr, wr, br, sr = leaves64(x, w, b, s)
    want, want_final = plain.conv(xr, wr, br, silu, sr, lengths)
    y, final = causal_conv(x, w, b, activation=act, initial_state=s, sequences=seqs)
    assert not y.requires_grad and y.dtype == dtype and final.dtype == dtype
    close(y, want, TOL[dtype], "y")
    assert torch.equal(final.double(), want_final.detach())
    g = gen(5)
    gy, gf = rand(g, *y.shape, dtype=dtype), rand(g, *final.shape, dtype=dtype)
    xk, wk, bk, sk = leaves(x, w, b, s)
    outs = causal_conv(xk, wk, bk, activation=act, initial_state=sk, sequences=seqs)
    got = grads(outs, (gy, gf), (xk, wk, bk, sk))
    ref = grads((want, want_final), (gy.double(), gf.double()), (xr, wr, br, sr))
    assert torch.equal(outs[0].detach(), y)
    for name, a, r in zip(("x", "weight", "bias", "state"), got, ref):
        if a is not None:
            r = torch.zeros_like(a, dtype=torch.float64) if r is None else r
            close(a, r, TOL[dtype], f"grad {name}")


def test_conv_weight_types_and_conv1d_shape():
    x, w, b, s, _ = conv_inputs((2, 50), 48, 4, torch.bfloat16, 1, wdtype=torch.float32)
    wk = w[:, None].detach().requires_grad_()
    y, _ = causal_conv(x, wk, b, activation="silu")
    want, _ = plain.conv(x.double(), w.double(), b.double(), True, None)
    close(y, want, TOL[torch.bfloat16], "y")
    (gw,) = torch.autograd.grad(y.float().sum(), wk)
    assert gw.shape == wk.shape and gw.dtype == torch.float32


def test_conv_only_final_state_used():
    x, w, b, s, _ = conv_inputs((2, 9), 16, 4, torch.float32, 2)
    xk, sk = leaves(x, s)
    _, final = causal_conv(xk, w, b, initial_state=sk)
    gx, gs = torch.autograd.grad(final.sum(), (xk, sk))
    want = torch.zeros_like(gx)
    want[:, -3:] = 1
    assert torch.equal(gx, want) and not gs.any()


def test_conv_strided_and_broadcast_rows():
    g = gen(8)
    wide = rand(g, 2, 40, 100)
    w, b = rand(g, 32, 4), rand(g, 32)
    for x in (wide[..., 4:36], wide[..., 5:37], wide.transpose(0, 1)[..., :32], wide[:1, :, :32].expand(3, 40, 32),
              wide[:, ::2, 8:40]):
        want, _ = plain.conv(x.double(), w.double(), b.double(), True, None)
        close(causal_conv(x, w, b, activation="silu")[0], want, 2e-5, f"strides {x.stride()}")
        xk = x.detach().requires_grad_()
        close(causal_conv(xk, w, b, activation="silu")[0], want, 2e-5, f"strides {x.stride()}")


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("c,taps", [(64, 4), (33, 3), (2, 2)])
def test_conv_steps_continue_a_prompt(c, taps, dtype):
    x, w, b, s, _ = conv_inputs((3, 23), c, taps, dtype, 4)
    want, want_final = causal_conv(x, w, b, activation="silu", initial_state=s)
    first, state = causal_conv(x[:, :10], w, b, activation="silu", initial_state=s)
    got = [first]
    for t in range(10, 23):
        got.append(causal_conv_step(x[:, t], state, w, b, activation="silu")[:, None])
    assert torch.equal(torch.cat(got, 1), want) and torch.equal(state, want_final)


# ---------------------------------------------------------------------------
# scan
# ---------------------------------------------------------------------------

# (lead or lengths, C, N, G)
SCAN = [((2, 37), 40, 16, 1), ((1, 1), 5, 1, 1), ((3, 33), 130, 10, 2), ((2, 65), 64, 4, 1), ((1, 100), 24, 64, 3),
        ((2, 17), 300, 3, 1), ((1, 300), 33, 32, 1), ((4, 16), 17, 8, 1), ((2, 48), 96, 40, 2), ((1, 31), 520, 7, 2),
        (RAGGED, 70, 16, 1), (RAGGED, 9, 5, 3), ([0, 0], 16, 16, 1), ([1, 1, 1], 64, 16, 2)]
NAMES = ("values", "steps", "rates", "keys", "queries", "skip", "gate", "step_bias", "state")


def scan_inputs(shape, c, n, groups, dtype, seed):
    g = gen(seed)
    lengths = shape if isinstance(shape, list) else None
    lead = (sum(shape),) if lengths is not None else shape
    count = len(shape) if lengths is not None else shape[0]
    rates = -torch.rand(c, n, generator=g, device="cuda") * n - 0.05
    return dict(values=rand(g, *lead, c, dtype=dtype), steps=rand(g, *lead, c, dtype=dtype), rates=rates,
                keys=rand(g, *lead, groups, n, dtype=dtype), queries=rand(g, *lead, groups, n, dtype=dtype),
                skip=rand(g, c), gate=rand(g, *lead, c, dtype=dtype), step_bias=rand(g, c) - 3.0,
                state=rand(g, count, c, n)), lengths


def call(i, softplus, seqs):
    return selective_scan(i["values"], i["steps"], i["rates"], i["keys"], i["queries"], skip=i["skip"],
                          gate=i["gate"], step_bias=i["step_bias"], softplus=softplus, initial_state=i["state"],
                          sequences=seqs)


def call_plain(i, softplus, lengths):
    return plain.scan(*(i[k] for k in NAMES[:8]), softplus, i["state"], lengths)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("parts", ("all", "bare", "gate", "skip+state"))
@pytest.mark.parametrize("shape,c,n,groups", SCAN)
def test_scan_forward_and_gradients(shape, c, n, groups, parts, dtype):
    i, lengths = scan_inputs(shape, c, n, groups, dtype, c + n)
    softplus = parts != "bare"
    if parts == "bare":  # steps are used as they are: make them small and positive
        i["steps"] = (i["steps"].float().abs() * 0.1).to(dtype)
    for k, kept in (("skip", ("all", "skip+state")), ("gate", ("all", "gate")), ("step_bias", ("all", "gate")),
                    ("state", ("all", "skip+state"))):
        if parts not in kept:
            i[k] = None
    seqs = None if lengths is None else PackedSequences(lengths, device="cuda")
    r = dict(zip(NAMES, leaves64(*(i[k] for k in NAMES))))
    want, want_final = call_plain(r, softplus, lengths)
    y, final = call(i, softplus, seqs)
    assert not y.requires_grad and y.dtype == dtype and final.dtype == torch.float32
    close(y, want, TOL[dtype], "read")
    close(final, want_final, TOL[torch.float32], "final state")
    k = dict(zip(NAMES, leaves(*(i[k] for k in NAMES))))
    outs = call(k, softplus, seqs)
    assert torch.equal(outs[0].detach(), y) and torch.equal(outs[1].detach(), final)
    g = gen(6)
    gy, gf = rand(g, *y.shape, dtype=dtype), rand(g, *final.shape)
    ups = (gy, gf) if parts != "gate" else (gy,)
    got = grads(outs[:len(ups)], ups, [k[n_] for n_ in NAMES])
    ref = grads((want, want_final)[:len(ups)], [u.double() for u in ups], [r[n_] for n_ in NAMES])
    for name, a, b in zip(NAMES, got, ref):
        if a is not None:
            b = torch.zeros_like(a, dtype=torch.float64) if b is None else b
            tol = TOL[dtype] if name in ("values", "steps", "keys", "queries", "gate") else TOL[torch.float32]
            close(a, b, tol, f"grad {name}")


@pytest.mark.parametrize("shape,c,n", [((1, 3400), 24, 16), ([3300, 0, 130, 1700, 1], 40, 6), ((2, 700), 33, 16)])
def test_scan_long_axis_split(shape, c, n):
    """Few channels and many tokens: the axis is split over many CTAs, chained
    by each of them (a few chunks) or by a launch of its own (more than 24, as
    in the first two), in both directions.  A state remembers 1 / (0.05 d) of
    these tokens at most, a few hundred, so the tolerance is that of the shorter
    cases."""
    i, lengths = scan_inputs(shape, c, n, 1, torch.float32, 31)
    seqs = None if lengths is None else PackedSequences(lengths, device="cuda")
    r = dict(zip(NAMES, leaves64(*(i[k] for k in NAMES))))
    k = dict(zip(NAMES, leaves(*(i[k] for k in NAMES))))
    want, want_final = call_plain(r, True, lengths)
    y, final = call(k, True, seqs)
    close(y, want, 2e-5, "read")
    close(final, want_final, 2e-5, "final state")
    g = gen(32)
    gy, gf = rand(g, *y.shape), rand(g, *final.shape)
    got = grads((y, final), (gy, gf), [k[n_] for n_ in NAMES])
    ref = grads((want, want_final), (gy.double(), gf.double()), [r[n_] for n_ in NAMES])
    for name, a, b in zip(NAMES, got, ref):
        close(a, b, 2e-5, f"grad {name}")


def test_a_step_of_zero_keeps_the_state():
    """Exactly: the decay of a zero step is 1, also with the exponent's bias."""
    i, _ = scan_inputs((2, 33), 40, 16, 1, torch.float32, 33)
    i["steps"].zero_()
    i["step_bias"] = None
    _, final = call(i, False, None)
    assert torch.equal(final, i["state"])
    selective_step(i["values"][:, 0], i["steps"][:, 0], i["rates"], i["keys"][:, 0], i["queries"][:, 0], final,
                   skip=i["skip"])
    assert torch.equal(final, i["state"])


def test_scan_gradients_against_differences():
    """<grad, direction> of the kernels against central differences of the
    plain form along random directions of every input."""
    i, _ = scan_inputs((2, 40), 18, 12, 2, torch.float32, 11)
    k = dict(zip(NAMES, leaves(*(i[n] for n in NAMES))))
    y, final = call(k, True, None)
    g = gen(12)
    gy, gf = rand(g, *y.shape), rand(g, *final.shape)
    got = torch.autograd.grad((y, final), [k[n] for n in NAMES], (gy, gf))
    for name, grad in zip(NAMES, got):
        direction = torch.randn(grad.shape, generator=g, device="cuda").double()

        def value(h):
            j = {n: v.double() for n, v in i.items()}
            j[name] = j[name] + h * direction
            a, b = call_plain(j, True, None)
            return float((a * gy.double()).sum() + (b * gf.double()).sum())
        want = (value(1e-6) - value(-1e-6)) / 2e-6
        size = float(grad.double().norm() * direction.norm())
        assert abs(float((grad.double() * direction).sum()) - want) <= 2e-5 * size, name


def test_scan_only_final_state_used():
    i, _ = scan_inputs((2, 21), 20, 16, 1, torch.float32, 13)
    r = dict(zip(NAMES, leaves64(*(i[n] for n in NAMES))))
    k = dict(zip(NAMES, leaves(*(i[n] for n in NAMES))))
    got = grads(call(k, True, None)[1].sum(), None, [k[n] for n in NAMES])
    ref = grads(call_plain(r, True, None)[1].sum(), None, [r[n] for n in NAMES])
    for name, a, b in zip(NAMES, got, ref):
        if b is None:
            assert a is None or not a.any(), name
        else:
            close(a, b, 2e-5, name)


def test_scan_strided_and_broadcast_rows():
    g = gen(14)
    i, _ = scan_inputs((2, 40), 24, 8, 2, torch.float32, 15)
    fused = rand(g, 2, 40, 3 * 24 + 2 * 16 + 3)
    i["values"], i["steps"], i["gate"] = fused[..., 1:25], fused[..., 25:49], fused[..., 49:73]
    i["keys"], i["queries"] = fused[..., 73:89].unflatten(-1, (2, 8)), fused[..., 89:105].unflatten(-1, (2, 8))
    for change in ({}, {"keys": i["keys"][:, :1].expand(2, 40, 2, 8)}, {"values": i["values"][:1].expand(2, 40, 24)},
                   {"queries": i["queries"].transpose(2, 3).contiguous().transpose(2, 3)}):
        j = dict(i, **change)
        want, want_final = call_plain({n: v.double() for n, v in j.items()}, True, None)
        y, final = call(j, True, None)
        close(y, want, 2e-5, f"read {list(change)}")
        close(final, want_final, 2e-5, f"state {list(change)}")
    # gradients of broadcast operands are summed over what they were broadcast to
    base = i["keys"][:, :1].detach().clone().requires_grad_()
    base64 = base.detach().double().requires_grad_()
    y, _ = call(dict(i, keys=base.expand(2, 40, 2, 8)), True, None)
    want, _ = call_plain(dict({n: v.double() for n, v in i.items()}, keys=base64.expand(2, 40, 2, 8)), True, None)
    close(torch.autograd.grad(y.sum(), base)[0], torch.autograd.grad(want.sum(), base64)[0], 2e-5, "broadcast keys")


def test_scan_large_and_negative_steps():
    """Softplus over its whole range, decays that vanish, steps that are zero."""
    i, _ = scan_inputs((1, 64), 16, 16, 1, torch.float32, 16)
    i["steps"] = torch.linspace(-60, 60, 64, device="cuda")[None, :, None].expand(1, 64, 16).contiguous()
    i["step_bias"] = None
    r = dict(zip(NAMES, leaves64(*(i[n] for n in NAMES))))
    k = dict(zip(NAMES, leaves(*(i[n] for n in NAMES))))
    want, want_final = call_plain(r, True, None)
    y, final = call(k, True, None)
    close(y, want, 2e-5, "read")
    close(final, want_final, 2e-5, "state")
    gy = rand(gen(1), *y.shape)
    names = [n for n in NAMES if i[n] is not None]
    for name, a, b in zip(names, torch.autograd.grad(y, [k[n] for n in names], gy),
                          torch.autograd.grad(want, [r[n] for n in names], gy.double())):
        close(a, b, 2e-5, f"grad {name}")


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("b,c,n,groups", [(1, 40, 16, 1), (5, 33, 10, 3), (2, 64, 64, 1), (3, 7, 1, 1), (4, 96, 20, 2)])
def test_steps_continue_a_prompt(b, c, n, groups, dtype):
    i, _ = scan_inputs((b, 20), c, n, groups, dtype, 17)
    r = {name: v.double() for name, v in i.items()}
    want, want_final = call_plain(r, True, None)
    head = {name: v[:, :12] if name in ("values", "steps", "keys", "queries", "gate") else v for name, v in i.items()}
    y, state = call(head, True, None)
    got = [y]
    for t in range(12, 20):
        got.append(selective_step(i["values"][:, t], i["steps"][:, t], i["rates"], i["keys"][:, t],
                                  i["queries"][:, t], state, skip=i["skip"], gate=i["gate"][:, t],
                                  step_bias=i["step_bias"], softplus=True)[:, None])
    close(torch.cat(got, 1), want, TOL[dtype], "read")
    close(state, want_final, TOL[torch.float32], "state")


def test_pieces_of_a_prompt_and_empty_pieces():
    i, _ = scan_inputs((2, 50), 24, 16, 1, torch.float32, 18)
    want, want_final = call_plain({n: v.double() for n, v in i.items()}, True, None)
    state, got = i["state"], []
    for lo, hi in ((0, 17), (17, 17), (17, 18), (18, 50)):
        piece = {n: v[:, lo:hi] if n in ("values", "steps", "keys", "queries", "gate") else v for n, v in i.items()}
        y, state = call(dict(piece, state=state), True, None)
        got.append(y)
    close(torch.cat(got, 1), want, 2e-5, "read")
    close(state, want_final, 2e-5, "state")


def test_nothing_at_all():
    for shape in ((0, 5), (2, 0)):
        i, _ = scan_inputs(shape, 16, 8, 1, torch.float32, 19)
        k = dict(zip(NAMES, leaves(*(i[n] for n in NAMES))))
        y, final = call(k, True, None)
        assert y.shape == (*shape, 16) and torch.equal(final.detach(), i["state"])
        got = torch.autograd.grad(y.sum() + final.sum(), [k["rates"], k["skip"], k["state"]])
        assert not got[0].any() and not got[1].any() and (got[2] == 1).all()
        x, w, b, s, _ = conv_inputs(shape, 16, 4, torch.float32, 20)
        xk, wk, sk = leaves(x, w, s)
        y, final = causal_conv(xk, wk, b, initial_state=sk)
        assert torch.equal(final.detach(), s)
        gw, gs = torch.autograd.grad(y.sum() + final.sum(), [wk, sk])
        assert not gw.any() and (gs == 1).all()


def test_runs_are_identical():
    i, _ = scan_inputs((3, 200), 200, 16, 2, torch.bfloat16, 21)
    k = dict(zip(NAMES, leaves(*(i[n] for n in NAMES))))
    x, w, b, s, _ = conv_inputs((3, 300), 200, 4, torch.bfloat16, 22)
    ck = leaves(x, w, b, s)
    first = None
    for _ in range(3):
        outs = call(k, True, None)
        got = [*outs, *torch.autograd.grad(outs, [k[n] for n in NAMES], [torch.ones_like(o) for o in outs])]
        couts = causal_conv(ck[0], ck[1], ck[2], activation="silu", initial_state=ck[3])
        got += [*couts, *torch.autograd.grad(couts, ck, [torch.ones_like(o) for o in couts])]
        if first is None:
            first = got
        assert all(torch.equal(a, b_) for a, b_ in zip(got, first))


def test_another_stream():
    i, _ = scan_inputs((2, 100), 64, 16, 1, torch.float32, 23)
    want, _ = call(i, True, None)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        k = dict(zip(NAMES, leaves(*(i[n] for n in NAMES))))
        y, _ = call(k, True, None)
        y.sum().backward()
    stream.synchronize()
    assert torch.equal(y.detach(), want) and torch.isfinite(k["rates"].grad).all()


def test_refusals_on_the_gpu():
    i, _ = scan_inputs((2, 5), 16, 8, 1, torch.float32, 24)
    with pytest.raises(NotImplementedError, match="at most 64"):
        selective_scan(i["values"], i["steps"], i["rates"].repeat(1, 9), i["keys"].repeat(1, 1, 1, 9),
                       i["queries"].repeat(1, 1, 1, 9))
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        selective_scan(*(i[n].double() for n in NAMES[:5]))
    with pytest.raises(ValueError, match="same device"):
        selective_scan(i["values"], i["steps"], i["rates"].cpu(), i["keys"], i["queries"])
    with pytest.raises(RuntimeError, match="no gradient"):
        selective_step(i["values"][:, 0], i["steps"][:, 0], i["rates"].requires_grad_(), i["keys"][:, 0],
                       i["queries"][:, 0], i["state"])
    i["rates"].requires_grad_(False)
    with pytest.raises(ValueError, match="contiguous"):
        selective_step(i["values"][:, 0], i["steps"][:, 0], i["rates"], i["keys"][:, 0], i["queries"][:, 0],
                       i["state"].transpose(1, 2).contiguous().transpose(1, 2))
    x, w, b, s, _ = conv_inputs((2, 5), 16, 4, torch.float32, 25)
    with pytest.raises(NotImplementedError, match="taps"):
        causal_conv(x, w.repeat(1, 2), b)
    with pytest.raises(ValueError, match="contiguous"):
        causal_conv_step(x[:, 0], s.transpose(1, 2).contiguous().transpose(1, 2), w)
    with pytest.raises(ValueError, match="same device"):
        causal_conv(x, w, b, sequences=None, initial_state=s.cpu())
    with pytest.raises(ValueError, match="same device"):
        causal_conv(x[0], w, b, sequences=PackedSequences([5], device="cpu"))


@pytest.mark.parametrize("shape,c", [((2, 37), 40), ((1, 5), 3), ((1, 64), 16), ([3300, 0, 130, 1700, 1], 24),
                                     ([700, 3, 90], 24)])
def test_rates_of_minus_infinity(shape, c):
    """A state that keeps nothing from token to token, whatever the lengths: the tokens that fill a tile up have a step
    of zero, and so do the chunks past a short sequence's end."""
    i, lengths = scan_inputs(shape, c, 16, 1, torch.float32, 45)
    i["rates"][::2, 1::3] = -torch.inf
    i["rates"][1, 4] = torch.finfo(torch.float32).min
    seqs = None if lengths is None else PackedSequences(lengths, device="cuda")
    names = ("values", "keys", "queries", "skip", "gate")  # the others' gradients are products of infinity and zero
    r = {n: v.double().requires_grad_(n in names) for n, v in i.items()}
    k = {n: v.clone().requires_grad_(n in names) for n, v in i.items()}
    want, want_final = call_plain(r, True, lengths)
    y, final = call(k, True, seqs)
    close(y, want, 2e-5, "read")
    close(final, want_final, 2e-5, "state")
    g = gen(46)
    gy, gf = rand(g, *y.shape), rand(g, *final.shape)
    got = torch.autograd.grad((y, final), [k[n] for n in names], (gy, gf))
    ref = torch.autograd.grad((want, want_final), [r[n] for n in names], (gy.double(), gf.double()))
    for name, a, b in zip(names, got, ref):
        close(a, b, 2e-5, f"grad {name}")


@pytest.mark.parametrize("shape,n", [((1, 3400), 16), ((2, 700), 6)])
def test_growing_states_that_are_still_zero(shape, n):
    """Positive rates: a state (or an adjoint) of zero stays zero over a chunk whose growth float32 cannot hold.  The
    values begin 20 tokens before the end (the reads' gradients end 20 tokens after the start), which grow as exp(40)."""
    i, _ = scan_inputs(shape, 24, n, 1, torch.float32, 47)
    i["rates"] = torch.full_like(i["rates"], 2.0)
    i["steps"] = torch.full_like(i["steps"], 1.0)
    i["state"] = i["step_bias"] = None
    late = dict(i, values=i["values"].clone())
    late["values"][:, :-20] = 0
    want, want_final = call_plain({k: None if v is None else v.double() for k, v in late.items()}, False, None)
    y, final = call(late, False, None)
    close(y, want, 2e-5, "read")
    close(final, want_final, 2e-5, "state")
    early = dict(i, values=torch.zeros_like(i["values"]))
    r = dict(zip(NAMES, leaves64(*(early[k] for k in NAMES))))
    k = dict(zip(NAMES, leaves(*(early[k] for k in NAMES))))
    gy = rand(gen(48), *y.shape)
    gy[:, 20:] = 0
    want = torch.autograd.grad(call_plain(r, False, None)[0], r["values"], gy.double())[0]
    close(torch.autograd.grad(call(k, False, None)[0], k["values"], gy)[0], want, 2e-5, "grad values")


def test_forward_mode_is_refused():
    """A tangent that came in must not be lost without a word."""
    i, _ = scan_inputs((2, 9), 16, 8, 1, torch.float32, 41)
    x, w, b, s, _ = conv_inputs((2, 9), 16, 4, torch.float32, 42)
    conv = dict(x=x, weight=w, bias=b, initial_state=s)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for keep in (True, False):
            with torch.set_grad_enabled(keep):
                for name in NAMES:
                    with pytest.raises(NotImplementedError, match="forward mode AD"):
                        call(dict(i, **{name: dual(i[name])}), True, None)
                for name in conv:
                    with pytest.raises(NotImplementedError, match="forward mode AD"):
                        causal_conv(**dict(conv, **{name: dual(conv[name])}))
                for name in ("x", "weight", "bias"):
                    one = dict(x=x[:, 0], weight=w, bias=b)
                    with pytest.raises(RuntimeError, match="no gradient"):
                        causal_conv_step(state=s.clone(), **dict(one, **{name: dual(one[name])}))
                for name in NAMES:
                    one = {n: v[:, 0] if n in ("values", "steps", "keys", "queries", "gate") else v.clone()
                           for n, v in i.items()}
                    one[name] = dual(one[name])
                    with pytest.raises(RuntimeError, match="no gradient"):
                        selective_step(*(one[n] for n in NAMES[:5]), one["state"], skip=one["skip"], gate=one["gate"],
                                       step_bias=one["step_bias"], softplus=True)
        call(i, True, None)
        causal_conv(**conv)


def test_steps_in_place_are_seen_by_autograd():
    """A backward that still needs the state a step has moved on says so instead of using the moved one."""
    x, w, b, s, _ = conv_inputs((2, 9), 16, 4, torch.float32, 43)
    wk = w.detach().requires_grad_()
    y, _ = causal_conv(x, wk, b, activation="silu", initial_state=s)
    causal_conv_step(x[:, 0], s, w, b, activation="silu")
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    i, _ = scan_inputs((2, 9), 16, 8, 1, torch.float32, 44)
    scale = torch.ones((), device="cuda", requires_grad=True)
    used = i["state"] * scale  # keeps the state for its backward
    head = {n: v[:, 0] if n in ("values", "steps", "keys", "queries", "gate") else v for n, v in i.items()}
    selective_step(*(head[n] for n in NAMES[:5]), i["state"], skip=head["skip"], gate=head["gate"],
                   step_bias=head["step_bias"], softplus=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        used.sum().backward()
    with torch.inference_mode():  # states without a version are moved on all the same
        y, state = causal_conv(x, w, b)
        _, hidden = call(i, True, None)
        causal_conv_step(x[:, 0], state, w, b)
    kept = state.clone(), hidden.clone()
    with torch.no_grad():
        causal_conv_step(x[:, 0], state, w, b)
        selective_step(*(head[n] for n in NAMES[:5]), hidden, softplus=True)
    assert not torch.equal(state, kept[0]) and not torch.equal(hidden, kept[1])


# ---------------------------------------------------------------------------
# sizes that the small cases above do not reach
# ---------------------------------------------------------------------------

def conv_wide(x, weight, bias, silu, state, lengths):
    """The plain form of a convolution, all tokens at a time."""
    taps, ys, finals = weight.shape[1], [], []
    for r, past in zip(plain.runs(x, lengths), state):
        wide = torch.cat([past, r])
        u = sum(wide[j:j + r.shape[0]] * weight[:, j] for j in range(taps)) + bias
        ys.append(u * torch.sigmoid(u) if silu else u)
        finals.append(wide[r.shape[0]:])
    return (torch.stack(ys) if lengths is None else torch.cat(ys)), torch.stack(finals)


# a thread's run of tokens grows from 4 with the number of elements: 8 (2.7 million), 32 (10 and 11) and, backward, 64
# (20), over odd and even channel counts
@pytest.mark.parametrize("shape,c,taps,dtype", [
    ((7, 391), 1001, 3, torch.bfloat16), ((5, 521), 4000, 4, torch.bfloat16), ((3, 1663), 4002, 2, torch.float32),
    ((5, 521), 4000, 3, torch.float32), ([0, 700, 1, 37, 2000, 0, 3], 4001, 3, torch.float16),
    ([0, 700, 1, 37, 2000, 0, 3], 4000, 4, torch.float32), ((2, 2500), 4001, 4, torch.bfloat16)])
def test_conv_long_runs(shape, c, taps, dtype):
    x, w, b, s, lengths = conv_inputs(shape, c, taps, dtype, 51, wdtype=torch.float32)
    seqs = None if lengths is None else PackedSequences(lengths, device="cuda")
    r, k = leaves64(x, w, b, s), leaves(x, w, b, s)
    want = conv_wide(*r[:3], True, r[3], lengths)
    outs = causal_conv(k[0], k[1], k[2], activation="silu", initial_state=k[3], sequences=seqs)
    close(outs[0], want[0], TOL[dtype], "y")
    assert torch.equal(outs[1].detach().double(), want[1].detach())
    assert torch.equal(causal_conv(x, w, b, activation="silu", initial_state=s, sequences=seqs)[0], outs[0].detach())
    g = gen(52)
    ups = [rand(g, *o.shape, dtype=dtype) for o in outs]
    got = torch.autograd.grad(outs, k, ups)
    ref = torch.autograd.grad(want, r, [u.double() for u in ups])
    for name, a, v in zip(("x", "weight", "bias", "state"), got, ref):
        close(a, v, TOL[a.dtype], f"grad {name}")


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("b,c,n,groups", [(1500, 40, 16, 1), (200, 300, 10, 3), (400, 64, 64, 2), (700, 300, 1, 1),
                                          (1300, 17, 4, 1)])
def test_steps_of_many_sequences(b, c, n, groups, dtype):
    """More sequences than one wave of CTAs takes: a lane walks several of them."""
    i, _ = scan_inputs((b, 1), c, n, groups, dtype, 53)
    want, want_final = call_plain({name: v.double() for name, v in i.items()}, True, None)
    one = {name: v[:, 0] if name in ("values", "steps", "keys", "queries", "gate") else v for name, v in i.items()}
    got = selective_step(*(one[name] for name in NAMES[:5]), one["state"], skip=one["skip"], gate=one["gate"],
                         step_bias=one["step_bias"], softplus=True)
    close(got[:, None], want, TOL[dtype], "read")
    close(one["state"], want_final, TOL[torch.float32], "state")
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("shape,c,n,groups", [((2, 70), 300, 1, 1), ((1, 90), 512, 2, 2), ((2, 48), 256, 2, 1),
                                              ([33, 0, 1, 100], 257, 1, 1), ((1, 800), 20, 2, 1)])
def test_scan_of_one_and_two_states(shape, c, n, groups, dtype):
    """A lane to a channel, over several tiles and segments, with and without channels left over."""
    i, lengths = scan_inputs(shape, c, n, groups, dtype, 54)
    seqs = None if lengths is None else PackedSequences(lengths, device="cuda")
    r = dict(zip(NAMES, leaves64(*(i[k] for k in NAMES))))
    k = dict(zip(NAMES, leaves(*(i[k] for k in NAMES))))
    want, want_final = call_plain(r, True, lengths)
    y, final = call(k, True, seqs)
    close(y, want, TOL[dtype], "read")
    close(final, want_final, 2e-5, "state")
    g = gen(55)
    gy, gf = rand(g, *y.shape, dtype=dtype), rand(g, *final.shape)
    got = torch.autograd.grad((y, final), [k[name] for name in NAMES], (gy, gf))
    ref = torch.autograd.grad((want, want_final), [r[name] for name in NAMES], (gy.double(), gf.double()))
    for name, a, b in zip(NAMES, got, ref):
        close(a, b, TOL[a.dtype], f"grad {name}")
