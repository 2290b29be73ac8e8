"""GPU: distillation kernels vs the plain 64-bit form.

Tolerances: a float32 logit's exponent (at most about 40 in magnitude here) is
rounded to 2^-24 of itself and exp2 to 2 ulp, so a probability is good to 40 *
2^-24 + 2^-22 = 2.6e-6 and the loss and gradient, sums and differences of
them, to 1e-5 in relative L2; a gradient rounded to bfloat16 (float16) is off
by at most 2^-9 (2^-12) of itself: 2.5e-3, and 6e-4 plus float16's subnormal
spacing.
"""
from __future__ import annotations

import gc
import math

import pytest
import torch
import torch.utils.checkpoint
from torch.autograd import forward_ad

import plain_selective as plain
from bayes_ssm.distill import distillation_loss, distillation_loss_torch

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1e-5, torch.bfloat16: 2.5e-3, torch.float16: 1e-3}


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def inputs(rows, vocab, top, dtype, seed, index_dtype=torch.int64, scale=2.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    logits = torch.randn(rows, vocab, generator=g, device="cuda") * scale
    teacher, indices = torch.topk(logits + torch.randn(rows, vocab, generator=g, device="cuda"), top, -1)
    return logits.to(dtype), teacher.to(dtype), indices.to(index_dtype)


def reference(logits, teacher, indices, temperature, reduction):
    x = logits.detach().double().requires_grad_()
    losses, counted = plain.distill(x, teacher.double(), indices, temperature)
    if reduction == "none":
        return losses, x
    total = losses.sum()
    return (total / max(1, sum(counted)) if reduction == "mean" else total), x


SHAPES = [(5, 1000, 8), (1, 7, 7), (3, 1, 1), (4, 4099, 33), (2, 50001, 16), (9, 513, 300), (2, 32000, 64),
          (150, 40, 3), (1, 130000, 5)]


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("temperature,reduction", [(1.0, "mean"), (2.5, "sum"), (0.7, "none")])
@pytest.mark.parametrize("rows,vocab,top", SHAPES)
def test_loss_and_gradient(rows, vocab, top, temperature, reduction, dtype):
    logits, teacher, indices = inputs(rows, vocab, top, dtype, rows + vocab)
    if rows > 2:
        indices[1] = -1                    # a row without a teacher
        teacher[2, top // 2:] = -math.inf  # one that gives fewer logits
        if top == 1:
            indices[2] = 0
    want, x64 = reference(logits, teacher, indices, temperature, reduction)
    x = logits.detach().requires_grad_()
    loss = distillation_loss(x, teacher, indices, temperature=temperature, reduction=reduction)
    assert loss.dtype == torch.float32 and loss.shape == want.shape
    g = torch.Generator(device="cuda").manual_seed(3)
    up = torch.randn(want.shape, generator=g, device="cuda")
    plain_loss = distillation_loss(logits, teacher, indices, temperature=temperature, reduction=reduction)
    assert torch.equal(plain_loss, loss.detach()) and not plain_loss.requires_grad
    # a loss near zero is a difference of logarithms of the size of log V
    assert float((loss.detach().double() - want.detach()).abs().max()) <= \
        1e-5 * (float(want.detach().abs().max()) + temperature ** 2 * (rows if reduction == "sum" else 1))
    if vocab == 1:
        got = torch.autograd.grad(loss, x, up)[0]
        assert not got.any()
        return
    got = torch.autograd.grad(loss, x, up)[0]
    ref = torch.autograd.grad(want, x64, up.double())[0]
    assert got.dtype == dtype and rel(got, ref) <= TOL[dtype]
    if rows > 2:
        assert not got[1].any()


def test_gradient_against_differences():
    logits, teacher, indices = inputs(3, 40, 6, torch.float32, 5)
    x = logits.requires_grad_()
    grad = torch.autograd.grad(distillation_loss(x, teacher, indices, temperature=1.7), x)[0].double()
    g = torch.Generator(device="cuda").manual_seed(4)
    direction = torch.randn(3, 40, generator=g, device="cuda").double()

    def value(h):
        losses, counted = plain.distill(logits.detach().double() + h * direction, teacher.double(), indices, 1.7)
        return float(losses.sum()) / sum(counted)
    want = (value(1e-6) - value(-1e-6)) / 2e-6
    assert abs(float((grad * direction).sum()) - want) <= 1e-5 * float(grad.norm() * direction.norm())


def test_upstream_factor_and_second_backward():
    logits, teacher, indices = inputs(6, 300, 9, torch.float32, 6)
    x = logits.requires_grad_()
    loss = distillation_loss(x, teacher, indices)
    once = torch.autograd.grad(loss, x, retain_graph=True)[0]
    again = torch.autograd.grad(loss * 3.0, x, retain_graph=True)[0]
    third = torch.autograd.grad(loss * -0.5, x)[0]
    assert rel(again, 3.0 * once) <= 1e-6 and rel(third, -0.5 * once) <= 1e-6
    assert once.data_ptr() != again.data_ptr()
    loss = distillation_loss(x, teacher, indices)
    assert rel(torch.autograd.grad(loss * 3.0, x)[0], 3.0 * once) <= 1e-6


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_entries_named_twice_and_narrow_indices(dtype):
    logits, teacher, indices = inputs(4, 100, 6, dtype, 7, index_dtype=torch.int32)
    indices[0] = 5
    indices[1, 3] = indices[1, 0]
    indices[2, 1] = -7
    want, x64 = reference(logits, teacher, indices, 1.0, "mean")
    x = logits.requires_grad_()
    loss = distillation_loss(x, teacher, indices)
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * (1 + abs(float(want.detach())))
    assert rel(torch.autograd.grad(loss, x)[0], torch.autograd.grad(want, x64)[0]) <= TOL[dtype]


@pytest.mark.parametrize("level", (-3000.0, 3000.0))
@pytest.mark.parametrize("top", (3, 40, 700))
def test_logits_far_from_zero(level, top):
    """Only differences of logits matter, on either side."""
    logits, teacher, indices = inputs(3, 3000, top, torch.float32, 15)
    teacher = teacher + level
    indices[1, 1:] = -1
    logits[2] += level
    want, x64 = reference(logits, teacher, indices, 1.0, "sum")
    x = logits.requires_grad_()
    loss = distillation_loss(x, teacher, indices, reduction="sum")
    # float32 logits of this size are 2^-13 apart, which both sides share
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * (3 + abs(float(want.detach())))
    assert rel(torch.autograd.grad(loss, x)[0], torch.autograd.grad(want, x64)[0]) <= 1e-5


def test_teacher_of_another_type():
    logits, teacher, indices = inputs(4, 2000, 6, torch.bfloat16, 8)
    teacher = teacher.float() + 0.01
    want, x64 = reference(logits, teacher, indices, 1.0, "sum")
    x = logits.requires_grad_()
    loss = distillation_loss(x, teacher, indices, reduction="sum")
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * (4 + abs(float(want.detach())))
    assert rel(torch.autograd.grad(loss, x)[0], torch.autograd.grad(want, x64)[0]) <= TOL[torch.bfloat16]


@pytest.mark.parametrize("low", (-math.inf, torch.finfo(torch.bfloat16).min))
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_masked_student_entries(dtype, low):
    """Vocabulary entries masked with -inf or the lowest value have no
    probability and no gradient; long stretches of them are skipped over."""
    logits, teacher, indices = inputs(4, 3000, 6, dtype, 9)
    mask = torch.ones(4, 3000, dtype=torch.bool, device="cuda")
    mask.scatter_(1, indices, False)
    mask[:, 2900:] = False
    mask[3] = False
    logits = logits.masked_fill(mask, low)
    want, x64 = reference(logits, teacher, indices, 1.0, "mean")
    x = logits.requires_grad_()
    loss = distillation_loss(x, teacher, indices)
    got = torch.autograd.grad(loss, x)[0]
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * (1 + abs(float(want.detach())))
    ref = torch.autograd.grad(want, x64)[0]
    assert torch.isfinite(got).all() and not got[mask].any()
    assert rel(got, ref) <= TOL[dtype]


def test_impossible_entries_and_not_a_number():
    logits, teacher, indices = inputs(8, 500, 4, torch.float32, 10)
    logits[0, indices[0, 0]] = -math.inf   # the teacher asks for what the student rules out
    indices[1, 2] = 500                    # past the vocabulary
    logits[2, 17] = math.nan
    logits[3] = -math.inf
    logits[4, 3] = math.inf
    teacher[5, 1] = math.nan
    logits[6] = math.nan
    indices[6] = -1                        # no teacher: whatever the logits are
    x = logits.requires_grad_()
    loss = distillation_loss(x, teacher, indices, reduction="none")
    grad = torch.autograd.grad(loss, x, torch.ones_like(loss))[0]
    assert loss[0] == math.inf and torch.isfinite(grad[0]).all()
    for r in (1, 2, 3, 4, 5):
        assert torch.isnan(loss[r]), r
    for r in (1, 2, 3, 4):
        assert torch.isnan(grad[r]).all(), r
    assert torch.isnan(grad[5, indices[5]]).all()
    assert loss[6] == 0 and not grad[6].any()
    want, x64 = reference(logits.detach()[7:], teacher[7:], indices[7:], 1.0, "sum")
    assert abs(float(loss[7].detach()) - float(want.detach())) <= 1e-5 * (1 + abs(float(want.detach())))
    assert rel(grad[7:], torch.autograd.grad(want, x64)[0]) <= 1e-5


def test_no_row_has_a_teacher():
    logits, teacher, indices = inputs(3, 100, 4, torch.float32, 11)
    indices.fill_(-1)
    x = logits.requires_grad_()
    loss = distillation_loss(x, teacher, indices)
    assert float(loss.detach()) == 0.0 and not torch.autograd.grad(loss, x)[0].any()
    empty = torch.zeros(0, 100, device="cuda", requires_grad=True)
    loss = distillation_loss(empty, teacher[:0], indices[:0])
    assert float(loss.detach()) == 0.0 and torch.autograd.grad(loss, empty)[0].shape == (0, 100)


def test_rows_of_a_padded_vocabulary_and_leading_dimensions():
    g = torch.Generator(device="cuda").manual_seed(12)
    wide = torch.randn(2, 5, 1032, generator=g, device="cuda", dtype=torch.bfloat16)
    for lo, hi in ((0, 1000), (3, 1003), (8, 1032)):
        logits = wide[..., lo:hi]
        teacher, indices = torch.topk(logits.float(), 7, -1)
        want, x64 = reference(logits.reshape(10, -1), teacher.reshape(10, -1), indices.reshape(10, -1), 1.0, "mean")
        x = logits.detach().requires_grad_()
        loss = distillation_loss(x, teacher, indices)
        assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * (1 + abs(float(want.detach())))
        got = torch.autograd.grad(loss, x)[0]
        assert rel(got.reshape(10, -1), torch.autograd.grad(want, x64)[0]) <= TOL[torch.bfloat16]


def test_runs_are_identical_and_match_the_torch_form():
    logits, teacher, indices = inputs(300, 5000, 20, torch.float32, 13)
    x = logits.requires_grad_()
    first = None
    for _ in range(3):
        loss = distillation_loss(x, teacher, indices, temperature=2.0)
        got = (loss.detach(), torch.autograd.grad(loss, x)[0])
        first = first or got
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])
    loss = distillation_loss_torch(x, teacher, indices, temperature=2.0)
    assert rel(first[0], loss) <= 1e-5 and rel(first[1], torch.autograd.grad(loss, x)[0]) <= 1e-5


def test_refusals_on_the_gpu():
    logits, teacher, indices = inputs(2, 3000, 4, torch.float32, 14)
    with pytest.raises(NotImplementedError, match="at most 1024"):
        distillation_loss(logits, logits[:, :2000], torch.arange(2000, device="cuda").expand(2, 2000))
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        distillation_loss(logits.double(), teacher, indices)
    with pytest.raises(ValueError, match="same device"):
        distillation_loss(logits, teacher, indices.cpu())


# rows of up to 8 KB, of up to 32 KB and longer ones (64, 128 and 256 threads a row), around the lengths where the form
# changes; 16 rows count those with a teacher themselves, 17 do not
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("rows,vocab,top", [(16, 2048, 20), (17, 2049, 20), (40, 4096, 100), (16, 4097, 1000),
                                            (17, 8192, 5), (33, 8193, 64), (16, 16384, 256), (17, 16385, 257)])
def test_row_lengths_where_the_form_changes(rows, vocab, top, dtype):
    logits, teacher, indices = inputs(rows, vocab, top, dtype, 3 * rows + vocab)
    indices[rows // 2] = -1
    indices[0, top // 2] = indices[0, 0]  # named twice
    for reduction in ("mean", "none"):
        want, x64 = reference(logits, teacher, indices, 1.5, reduction)
        x = logits.detach().requires_grad_()
        loss = distillation_loss(x, teacher, indices, temperature=1.5, reduction=reduction)
        assert float((loss.detach().double() - want.detach()).abs().max()) <= \
            1e-5 * (float(want.detach().abs().max()) + 1.5 ** 2)
        up = torch.ones_like(want)
        got = torch.autograd.grad(loss, x, up.float(), retain_graph=True)[0]
        ref = torch.autograd.grad(want, x64, up)[0]
        assert rel(got, ref) <= TOL[dtype] and not got[rows // 2].any()
        again = torch.autograd.grad(loss, x, up.float())[0]  # from the rows' statistics
        assert rel(again, ref) <= TOL[dtype]


def grad64(logits, teacher, indices, temperature):
    """The gradient of every row's loss in 64 bits (every row has a teacher, no entry is empty)."""
    q = torch.softmax(logits.double() / temperature, -1)
    p = torch.softmax(teacher.double() / temperature, -1)
    return temperature * q.scatter_add(1, indices, -p)


# an entry of the gradient differs from the 64-bit one's rounding only where that lies within its float32 error, 2.6e-6
# of itself outside the teacher's entries, of a boundary between two numbers of the type: these are at least 2^-8
# (bfloat16) and 2^-11 (float16) of it apart, so 2 * 2.6e-6 * 2^8 = 0.14 % and 1.1 % of the entries
@pytest.mark.parametrize("dtype,differ", [(torch.bfloat16, 1.4e-3), (torch.float16, 1.1e-2)])
@pytest.mark.parametrize("vocab", (2001, 2048))
@pytest.mark.parametrize("reduction,factor", [("mean", 65536.0), ("sum", 0.3), ("mean", -5000.0)])
def test_upstream_factor_before_the_one_rounding(reduction, factor, vocab, dtype, differ):
    """A loss scale reaches the gradient before it is rounded: unscaled, most of this one is below float16's least."""
    rows = 4096
    logits, teacher, indices = inputs(rows, vocab, 16, dtype, 21)
    up = torch.tensor(factor, device="cuda")
    ref = grad64(logits, teacher, indices, 2.0) * up.double() / (rows if reduction == "mean" else 1)
    x = logits.requires_grad_()
    loss = distillation_loss(x, teacher, indices, temperature=2.0, reduction=reduction)
    got = torch.autograd.grad(loss, x, up, retain_graph=True)[0]
    others = torch.ones_like(logits, dtype=torch.bool).scatter_(1, indices, False)
    assert float((got != ref.to(dtype))[others].double().mean()) <= differ
    assert rel(got, ref) <= TOL[dtype]
    assert torch.equal(torch.autograd.grad(loss, x, up)[0], got)  # a second walk


def test_upstream_factor_of_every_form():
    """The factor at few rows (split over clusters), many, rows without a teacher, and factors that are not finite."""
    for rows, vocab, top in ((2, 50001, 16), (3000, 300, 4), (20, 20000, 9), (5, 1, 1)):
        logits, teacher, indices = inputs(rows, vocab, top, torch.float32, 22)
        ref = grad64(logits, teacher, indices, 1.0) * 7.0
        indices[1] = -1
        x = logits.requires_grad_()
        loss = distillation_loss(x, teacher, indices, reduction="sum")
        got = torch.autograd.grad(loss, x, torch.tensor(7.0, device="cuda"), retain_graph=True)[0]
        ref[1] = 0
        if vocab > 1:
            assert rel(got, ref) <= 1e-5
        assert not got[1].any()
        nan = torch.autograd.grad(loss, x, torch.tensor(math.nan, device="cuda"))[0]
        assert torch.isnan(nan[0]).all() and not nan[1].any()


@pytest.mark.parametrize("value", (math.nan, math.inf))
@pytest.mark.parametrize("rows,vocab", [(3, 500), (2, 50001)])
def test_teacher_without_a_distribution(rows, vocab, value):
    """A teacher's NaN or +inf leaves no softmax: the row's loss and whole gradient are NaN, as in PyTorch operations."""
    logits, teacher, indices = inputs(rows, vocab, 4, torch.float32, 23)
    teacher[1, 2] = value
    x = logits.requires_grad_()
    for form in (distillation_loss, distillation_loss_torch):
        loss = form(x, teacher, indices, reduction="sum")
        first = torch.autograd.grad(loss, x, retain_graph=True)[0]
        second = torch.autograd.grad(loss, x)[0]
        for grad in (first, second):
            assert torch.isnan(grad[1]).all() and torch.isfinite(grad[0]).all() and torch.isfinite(grad[2:]).all()


def test_forward_mode_is_refused():
    """A tangent of the logits must not be lost without a word; the teacher is taken as a constant, as on the CPU."""
    logits, teacher, indices = inputs(3, 50, 4, torch.float32, 26)
    want = distillation_loss(logits, teacher, indices)
    with forward_ad.dual_level():
        for keep in (True, False):
            with torch.set_grad_enabled(keep), pytest.raises(NotImplementedError, match="forward mode AD"):
                distillation_loss(forward_ad.make_dual(logits, torch.ones_like(logits)), teacher, indices)
        assert torch.equal(distillation_loss(logits, teacher, indices), want)
        dual = forward_ad.make_dual(teacher, torch.ones_like(teacher))
        for device in ("cuda", "cpu"):
            loss = distillation_loss(logits.to(device), dual.to(device), indices.to(device))
            assert forward_ad.unpack_dual(loss).tangent is None


def test_nothing_of_the_logits_size_is_kept_past_the_hooks():
    """Recomputation and offloading of what a graph saves reach the gradient that the forward wrote."""
    g = torch.Generator(device="cuda").manual_seed(24)
    h = torch.randn(512, 64, generator=g, device="cuda").requires_grad_()
    w = (torch.randn(20000, 64, generator=g, device="cuda") * 0.3).requires_grad_()
    teacher, indices = torch.topk(torch.randn(512, 20000, generator=g, device="cuda"), 8, -1)

    def head(a, b):
        return distillation_loss(a @ b.t(), teacher, indices)
    want = torch.autograd.grad(head(h, w), (h, w))
    size = 512 * 20000 * 4
    for way in ("recomputed", "offloaded"):
        gc.collect()
        before = torch.cuda.memory_allocated()
        if way == "recomputed":
            loss = torch.utils.checkpoint.checkpoint(head, h, w, use_reentrant=False)
        else:
            with torch.autograd.graph.save_on_cpu():
                loss = head(h, w)
        assert torch.cuda.memory_allocated() - before < size // 4, way
        got = torch.autograd.grad(loss * 2.0, (h, w))
        assert all(rel(a, 2.0 * b) <= 1e-5 for a, b in zip(got, want)), way


def test_a_gradient_changed_in_place_between_two_walks():
    logits, teacher, indices = inputs(5, 200, 4, torch.float32, 25)
    x = logits.requires_grad_()
    loss = distillation_loss(x, teacher, indices)
    want = torch.autograd.grad(distillation_loss(x, teacher, indices), x)[0]
    loss.backward(retain_graph=True)
    x.grad.mul_(0.25)
    loss.backward(retain_graph=True)
    assert rel(x.grad, 1.25 * want) <= 1e-6
    x.grad.zero_()
    loss.backward()
    assert rel(x.grad, want) <= 1e-6


# a stretch too long for the bitmap of named entries; rows over 8 CTAs whose doubled entries lie in the first stretch, in
# the last one and on both sides of a boundary (6,252 float32, 6,256 bfloat16 logits)
@pytest.mark.parametrize("dtype,rows,vocab", [(torch.float32, 2, 400003), (torch.float32, 3, 50001),
                                              (torch.bfloat16, 3, 50001), (torch.bfloat16, 1, 800000)])
def test_doubled_entries_over_several_ctas(rows, vocab, dtype):
    logits, _, _ = inputs(rows, vocab, 4, dtype, 27)
    named = [0, 0, 5, 6251, 6252, 6251, 6252, 6255, 6256, 6256, 12503, 12504, 12504, 12512, 12511, vocab - 1, vocab - 1,
             vocab - 2, 7, -1]
    indices = torch.tensor(named, device="cuda").repeat(rows, 1)
    g = torch.Generator(device="cuda").manual_seed(28)
    teacher = torch.randn(rows, len(named), generator=g, device="cuda")
    want, x64 = reference(logits, teacher, indices, 1.0, "sum")
    x = logits.requires_grad_()
    loss = distillation_loss(x, teacher, indices, reduction="sum")
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * (rows + abs(float(want.detach())))
    ref = torch.autograd.grad(want, x64)[0]
    for keep in (True, False):  # written by the forward, then from the rows' statistics
        got = torch.autograd.grad(loss, x, retain_graph=keep)[0]
        assert rel(got, ref) <= TOL[dtype]
        at = indices[0, :-1]
        assert rel(got[:, at], ref[:, at]) <= TOL[dtype]
