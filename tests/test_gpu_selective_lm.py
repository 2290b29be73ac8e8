"""GPU: the selective language model on its kernels vs the same model on the
CPU (float32, the PyTorch forms), and the single-token path against the whole
sequence.  The tolerance is float32 GEMMs' (TF32 is off): 1e-4 in relative L2."""
from __future__ import annotations

import copy

import pytest
import torch

from bayes_ssm.selective import PackedSequences
from bayes_ssm.selective_lm import SelectiveLM, distill_step, generate
from bayes_ssm.six_layer import make_optimizer

pytestmark = pytest.mark.gpu


def rel(a, b):
    return float((a.detach().double().cpu() - b.detach().double().cpu()).norm() / b.detach().double().norm().cpu())


def make(groups=2):
    torch.manual_seed(0)
    cpu = SelectiveLM(vocab_size=101, width=48, layers=2, mlp_width=64, states=10, groups=groups,
                      dtype=torch.float32)
    return cpu, copy.deepcopy(cpu).cuda()


def test_forward_and_training_step_match_the_cpu():
    cpu, gpu = make()
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, 101, (3, 37), generator=g)
    teacher, indices = torch.topk(torch.randn(3, 37, 101, generator=g) * 2, 5, -1)
    indices[:, :4] = -1
    assert rel(gpu(tokens.cuda()), cpu(tokens)) <= 1e-4
    for model, dev in ((cpu, "cpu"), (gpu, "cuda")):
        loss = distill_step(model, make_optimizer(model), tokens.to(dev), teacher.to(dev), indices.to(dev),
                            temperature=2.0, grad_clip=0.0)
        model.loss = float(loss)
    assert abs(gpu.loss - cpu.loss) <= 1e-4 * abs(cpu.loss)
    for (name, a), b in zip(cpu.named_parameters(), gpu.parameters()):
        assert rel(b.grad, a.grad) <= 1e-4, name


def test_packed_prompts_then_tokens_match_the_whole_sequences():
    _, gpu = make()
    g = torch.Generator().manual_seed(2)
    tokens = torch.randint(0, 101, (3, 30), generator=g).cuda()
    full = gpu(tokens)
    lengths = [5, 1, 20]
    logits, state = gpu.prefill(torch.cat([tokens[i, :n] for i, n in enumerate(lengths)]),
                                PackedSequences(lengths, device="cuda"))
    for t in range(10):
        want = torch.stack([full[i, n + t - 1] for i, n in enumerate(lengths)])
        assert rel(logits, want) <= 1e-4
        logits = gpu.step(torch.stack([tokens[i, n + t] for i, n in enumerate(lengths)]), state)


def test_a_captured_token_step_replays():
    """The single-token path in a CUDA graph: static token and state buffers,
    moved on by every replay."""
    _, gpu = make()
    g = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, 101, (2, 14), generator=g).cuda()
    full = gpu(tokens)
    _, state = gpu.prefill(tokens[:, :6])
    start = copy.deepcopy(state)
    token = tokens[:, 6].clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        gpu.step(token, state)  # warm-up
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = gpu.step(token, state)
    for kept, s in zip(start, state):
        s.conv.copy_(kept.conv)
        s.scan.copy_(kept.scan)
    for t in range(6, 14):
        token.copy_(tokens[:, t])
        graph.replay()
        assert rel(logits, full[:, t]) <= 1e-4


def test_generate_and_bf16_training():
    torch.manual_seed(0)
    model = SelectiveLM(vocab_size=256, width=256, layers=2, mlp_width=256, device="cuda")
    optimizer = make_optimizer(model, lr=1e-3)
    tokens = torch.randint(0, 256, (4, 64), device="cuda")
    teacher, indices = torch.topk(torch.randn(4, 64, 256, device="cuda") * 3, 8, -1)
    losses = [float(distill_step(model, optimizer, tokens, teacher, indices)) for _ in range(6)]
    assert losses[-1] < losses[0]
    out = generate(model, [[1, 2, 3, 4], [7], [9, 9]], 12)
    assert out.shape == (3, 12) and int(out.min()) >= 0 and int(out.max()) < 256
