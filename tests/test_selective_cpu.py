"""CPU: the PyTorch forms of the selective operators and of distillation vs the
plain 64-bit loops, the checks of arguments, the model on them, and the C ABI's
refusals (no GPU needed).  float64 inputs run in float64 on both sides, so the
comparisons are to 1e-12; gradients are also tested against differences."""
from __future__ import annotations

import math

import pytest
import torch

import plain_selective as plain
from bayes_ssm import _capi
from bayes_ssm.distill import distillation_loss
from bayes_ssm.selective import (PackedSequences, causal_conv, causal_conv_step, selective_scan, selective_step)
from bayes_ssm.selective_lm import SelectiveLM, distill_step, generate
from bayes_ssm.six_layer import make_optimizer

RAGGED = [0, 5, 1, 0, 7]


def rel(a, b):
    return float((a.detach().double() - b.detach().double()).norm() / b.detach().double().norm().clamp_min(1e-30))


def scan_inputs(lead, count, c=6, n=5, groups=2, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, dtype=dtype)
    return dict(values=rand(*lead, c), steps=rand(*lead, c), rates=-torch.rand(c, n, generator=g, dtype=dtype) * n,
                keys=rand(*lead, groups, n), queries=rand(*lead, groups, n), skip=rand(c), gate=rand(*lead, c),
                step_bias=rand(c) - 2, state=rand(count, c, n))


def call(i, softplus=True, sequences=None):
    return selective_scan(i["values"], i["steps"], i["rates"], i["keys"], i["queries"], skip=i["skip"],
                          gate=i["gate"], step_bias=i["step_bias"], softplus=softplus, initial_state=i["state"],
                          sequences=sequences)


@pytest.mark.parametrize("lengths", (None, RAGGED))
def test_scan_and_conv_match_the_plain_forms(lengths):
    lead, count = ((2, 9), 2) if lengths is None else ((sum(lengths),), len(lengths))
    seqs = None if lengths is None else PackedSequences(lengths, device="cpu")
    i = scan_inputs(lead, count)
    y, final = call(i, sequences=seqs)
    want, want_final = plain.scan(*(i[k] for k in ("values", "steps", "rates", "keys", "queries", "skip", "gate",
                                                   "step_bias")), True, i["state"], lengths)
    assert rel(y, want) <= 1e-12 and rel(final, want_final) <= 1e-12
    g = torch.Generator().manual_seed(1)
    w = torch.randn(6, 3, generator=g, dtype=torch.float64)
    b = torch.randn(6, generator=g, dtype=torch.float64)
    s = torch.randn(count, 2, 6, generator=g, dtype=torch.float64)
    y, final = causal_conv(i["values"], w, b, activation="silu", initial_state=s, sequences=seqs)
    want, want_final = plain.conv(i["values"], w, b, True, s, lengths)
    assert rel(y, want) <= 1e-12 and torch.equal(final, want_final)


def test_gradients_against_differences():
    i = {k: v.requires_grad_() for k, v in scan_inputs((2, 6), 2, c=4, n=3).items()}
    names = list(i)
    assert torch.autograd.gradcheck(lambda *a: call(dict(zip(names, a))), tuple(i.values()))
    x = torch.randn(2, 5, 3, dtype=torch.float64, requires_grad=True)
    w = torch.randn(3, 4, dtype=torch.float64, requires_grad=True)
    s = torch.randn(2, 3, 3, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda *a: causal_conv(a[0], a[1], activation="silu", initial_state=a[2]),
                                    (x, w, s))
    logits = torch.randn(4, 7, dtype=torch.float64, requires_grad=True)
    teacher = torch.randn(4, 3, dtype=torch.float64)
    indices = torch.tensor([[0, 3, 6], [2, 2, 1], [-1, -1, -1], [5, -1, 4]])
    for reduction in ("mean", "sum", "none"):
        assert torch.autograd.gradcheck(lambda z: distillation_loss(z, teacher, indices, temperature=1.5,
                                                                    reduction=reduction), (logits,))


def test_steps_continue_a_prompt():
    i = scan_inputs((2, 9), 2)
    want, want_final = call(i)
    rows = ("values", "steps", "keys", "queries", "gate")
    y, state = call({k: v[:, :4] if k in rows else v for k, v in i.items()})
    got = [y]
    for t in range(4, 9):
        z = {k: i[k][:, t] for k in rows}
        got.append(selective_step(z["values"], z["steps"], i["rates"], z["keys"], z["queries"], state, skip=i["skip"],
                                  gate=z["gate"], step_bias=i["step_bias"], softplus=True)[:, None])
    assert rel(torch.cat(got, 1), want) <= 1e-12 and rel(state, want_final) <= 1e-12
    x, w = i["values"], torch.randn(6, 4, dtype=torch.float64)
    want, want_final = causal_conv(x, w)
    y, state = causal_conv(x[:, :4], w)
    got = [y] + [causal_conv_step(x[:, t], state, w)[:, None] for t in range(4, 9)]
    assert rel(torch.cat(got, 1), want) <= 1e-12 and torch.equal(state, want_final)


def test_distillation_matches_the_plain_form():
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(5, 11, generator=g, dtype=torch.float64)
    teacher = torch.randn(5, 4, generator=g, dtype=torch.float64)
    indices = torch.tensor([[0, 3, 6, 1], [2, 2, 1, 2], [-1, -1, -1, -1], [5, -1, 4, -9], [10, 9, 8, 7]])
    teacher[4, 1:] = -math.inf
    losses, counted = plain.distill(logits, teacher, indices, 1.7)
    assert rel(distillation_loss(logits, teacher, indices, temperature=1.7, reduction="none"), losses) <= 1e-12
    got = distillation_loss(logits, teacher, indices, temperature=1.7)
    assert abs(float(got - losses.sum() / sum(counted))) <= 1e-12
    indices[0, 0] = 11
    bad = distillation_loss(logits, teacher, indices, reduction="none")
    assert torch.isnan(bad[0]) and torch.isfinite(bad[1:]).all()
    indices[0, 0] = -1
    logits[0, 3] = -math.inf
    assert distillation_loss(logits, teacher, indices, reduction="none")[0] == math.inf
    none = distillation_loss(logits, teacher, torch.full_like(indices, -1))
    assert float(none) == 0.0


def test_packed_sequences():
    s = PackedSequences([3, 0, 2], device="cpu")
    assert (s.count, s.tokens, s.longest) == (3, 5, 3) and s.offsets.tolist() == [0, 3, 3, 5]
    assert PackedSequences(torch.tensor([1, 2]), device="cpu").tokens == 3
    assert PackedSequences([], device="cpu").tokens == 0
    for bad in ([1, -1], [1.5], [True], torch.tensor([[1]]), torch.tensor([1.0])):
        with pytest.raises(ValueError):
            PackedSequences(bad, device="cpu")


@pytest.mark.parametrize("change,error,match", [
    (dict(steps=torch.zeros(2, 9, 5)), ValueError, "values' shape"),
    (dict(gate=torch.zeros(2, 8, 6)), ValueError, "values' shape"),
    (dict(rates=torch.zeros(5, 5)), ValueError, r"rates must be \[6, N\]"),
    (dict(keys=torch.zeros(2, 9, 4, 5), queries=torch.zeros(2, 9, 4, 5)), ValueError, "divide the channels"),
    (dict(keys=torch.zeros(2, 9, 2, 4)), ValueError, "keys and queries"),
    (dict(keys=torch.zeros(2, 8, 2, 5), queries=torch.zeros(2, 8, 2, 5)), ValueError, "keys and queries"),
    (dict(skip=torch.zeros(5)), ValueError, r"skip must be \[6\]"),
    (dict(step_bias=torch.zeros(7)), ValueError, r"step_bias must be \[6\]"),
    (dict(state=torch.zeros(2, 6, 4)), ValueError, "initial_state"),
    (dict(steps=torch.zeros(2, 9, 6, dtype=torch.float64)), TypeError, "one dtype"),
    (dict(values=torch.zeros(2, 9, 6, dtype=torch.int64)), TypeError, "floating-point"),
])
def test_scan_refusals(change, error, match):
    i = {k: v.float() for k, v in scan_inputs((2, 9), 2).items()}
    with pytest.raises(error, match=match):
        call(dict(i, **change))


def test_other_refusals():
    i = {k: v.float() for k, v in scan_inputs((2, 9), 2).items()}
    seqs = PackedSequences([9, 9], device="cpu")
    with pytest.raises(ValueError, match="for these sequences"):
        call(i, sequences=seqs)
    with pytest.raises(TypeError, match="PackedSequences"):
        call(i, sequences=[9, 9])
    with pytest.raises(ValueError, match="with sequences"):
        flat = {k: v.flatten(0, 1) if v.ndim > 2 and k != "state" else v for k, v in i.items()}
        call(flat)
    x, w = i["values"], torch.zeros(6, 4)
    for args, kw, match in (((x, torch.zeros(5, 4)), {}, "weight must be"), ((x, w, torch.zeros(5)), {}, "bias"),
                            ((x, w), dict(activation="relu"), "activation"),
                            ((x, w), dict(initial_state=torch.zeros(2, 2, 6)), "initial_state"),
                            ((x, torch.zeros(6, 1)), {}, "taps")):
        with pytest.raises(ValueError, match=match):
            causal_conv(*args, **kw)
    with pytest.raises(TypeError, match="dtype"):
        causal_conv(x, w, initial_state=torch.zeros(2, 3, 6, dtype=torch.float64))
    with pytest.raises(ValueError, match="state must be"):
        causal_conv_step(x[:, 0], torch.zeros(2, 2, 6), w)
    with pytest.raises(RuntimeError, match="no gradient"):
        causal_conv_step(x[:, 0], torch.zeros(2, 3, 6), w.requires_grad_())
    with pytest.raises(RuntimeError, match="no gradient"):
        selective_step(x[:, 0], x[:, 0], i["rates"].requires_grad_(), i["keys"][:, 0], i["queries"][:, 0], i["state"])


@pytest.mark.parametrize("kwargs,error,match", [
    (dict(temperature=0.0), ValueError, "temperature"), (dict(temperature=math.inf), ValueError, "temperature"),
    (dict(temperature=True), ValueError, "temperature"), (dict(reduction="avg"), ValueError, "reduction"),
    (dict(teacher_indices=torch.zeros(3, 2, dtype=torch.int16)), TypeError, "int32 or int64"),
    (dict(teacher_indices=torch.zeros(3, 1, dtype=torch.int64)), ValueError, "teacher_logits' shape"),
    (dict(teacher_logits=torch.zeros(2, 2)), ValueError, "leading dimensions"),
    (dict(teacher_logits=torch.zeros(3, 0), teacher_indices=torch.zeros(3, 0, dtype=torch.int64)), ValueError,
     "empty"),
    (dict(logits=torch.zeros(3, 4, dtype=torch.int64)), TypeError, "floating-point"),
])
def test_distillation_refusals(kwargs, error, match):
    args = dict(logits=torch.zeros(3, 4), teacher_logits=torch.zeros(3, 2),
                teacher_indices=torch.zeros(3, 2, dtype=torch.int64))
    args.update(kwargs)
    with pytest.raises(error, match=match):
        distillation_loss(**args)


def test_c_abi_refusals_without_a_gpu():
    lib = _capi.load()
    conv = [None, 0, 16, 8, 16, 4, None, 0, None, 0, 0, None, 2, None, None, None, None]

    def error():
        return lib.bssm_last_error().decode()
    assert lib.bssm_causal_conv(*conv) == 1 and "null" in error()
    assert lib.bssm_causal_conv(*conv[:5], 5, *conv[6:]) == 2 and "taps" in error()
    assert lib.bssm_causal_conv(None, 7, *conv[2:]) == 2 and "dtype" in error()
    assert lib.bssm_causal_conv(None, 0, 16, 9, *conv[4:]) == 1  # 9 rows are not 2 sequences
    scan = [None, 8] * 5 + [0, None, None, None, 1, 8, 8, 16, 1, None, 2, 4] + [None] * 4 + [0, None, 0, None]
    assert lib.bssm_selective_scan(*scan) == 1 and "null" in error()
    assert lib.bssm_selective_scan(*scan[:17], 65, *scan[18:]) == 2 and "states" in error()
    assert lib.bssm_selective_scan(*scan[:18], 3, *scan[19:]) == 1 and "sizes" in error()
    step = [None, 8] * 5 + [0, None, None, None, 1, 2, 8, 16, 1, None, None, None]
    assert lib.bssm_selective_step(*step) == 1 and "null" in error()
    distill = [None, 0, 4, 10, 10, None, 0, None, 8, 3, 1.0, 1] + [None] * 6
    assert lib.bssm_distillation(*distill) == 1 and "null" in error()
    assert lib.bssm_distillation(*distill[:9], 2000, *distill[10:]) == 2 and "teacher logits" in error()
    assert lib.bssm_distillation(*distill[:10], -1.0, *distill[11:]) == 1 and "temperature" in error()
    assert lib.bssm_distillation(*distill[:8], 2, *distill[9:]) == 2
    # sizes of what the caller keeps: never negative, and enough for the saved states
    assert lib.bssm_selective_saved_floats(100, 3, 8, 16) >= 3 * math.ceil(100 / 3 / 16) * 8 * 16
    assert lib.bssm_selective_scan_floats(8, 2, 4, 8, 16, 1) == 0
    assert lib.bssm_selective_backward_floats(8, 2, 4, 8, 16, 1) > 0


def test_model_trains_from_a_teacher_and_generates():
    torch.manual_seed(0)
    model = SelectiveLM(vocab_size=40, width=16, layers=2, mlp_width=32, states=4, dtype=torch.float32)
    optimizer = make_optimizer(model, lr=3e-3)
    tokens = torch.randint(0, 40, (2, 12))
    teacher, indices = torch.topk(torch.randn(2, 12, 40) * 3, 4, -1)
    indices[:, :3] = -1  # no teacher over the prompt
    losses = [float(distill_step(model, optimizer, tokens, teacher, indices)) for _ in range(8)]
    assert all(math.isfinite(v) for v in losses) and losses[-1] < losses[0]
    # prompts of several lengths, then token by token: the logits of the whole sequences
    logits, state = model.prefill(tokens[:, :7])
    full = model(tokens)
    assert rel(logits, full[:, 6]) <= 1e-5
    for t in range(7, 12):
        assert rel(model.step(tokens[:, t], state), full[:, t]) <= 1e-5
    seqs = PackedSequences([3, 7], device="cpu")
    packed, _ = model.prefill(torch.cat([tokens[0, :3], tokens[1, :7]]), seqs)
    assert rel(packed, torch.stack([full[0, 2], full[1, 6]])) <= 1e-5
    out = generate(model, [[1, 2, 3], [4]], 5)
    assert out.shape == (2, 5)
    again = torch.tensor([[1, 2, 3] + out[0, :4].tolist()])
    assert torch.equal(model(again)[0, 2:].argmax(-1), out[0])
    with pytest.raises(ValueError, match="at least one token"):
        model.prefill(tokens[:, :0])


@pytest.mark.parametrize("dtype", (torch.float32, torch.float64))
def test_an_entry_past_the_vocabulary_makes_the_gradient_nan(dtype):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, 7, generator=g, dtype=dtype).requires_grad_()
    teacher = torch.randn(4, 3, generator=g, dtype=dtype)
    indices = torch.tensor([[0, 7, 2], [1, 2, 3], [-1, -1, -1], [6, 5, -1]])
    for reduction in ("mean", "sum", "none"):
        loss = distillation_loss(x, teacher, indices, reduction=reduction)
        grad = torch.autograd.grad(loss.sum(), x)[0]
        assert torch.isnan(loss).any() and torch.isnan(grad[0]).all(), reduction
        assert torch.isfinite(grad[1:]).all() and not grad[2].any() and grad[1].any(), reduction
    assert torch.isfinite(loss[1:]).all() and torch.isnan(loss[0])
