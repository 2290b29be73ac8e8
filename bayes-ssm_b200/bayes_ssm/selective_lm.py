"""A language model of selective state space blocks: trained from a teacher's
top logits, run over prompts and then token by token.

:class:`SelectiveMixer` takes the place of a :class:`bayes_ssm.mixer.BayesianMixer`
in a block: RMSNorm -> projection to values and gate -> short causal convolution
with SiLU -> projection to step, keys and queries -> the selective scan -> output
projection.  :class:`SelectiveLM` stacks such blocks with the SwiGLU MLPs and the
tied FP32 head of :mod:`bayes_ssm.six_layer`.

* :func:`distill_step` is one optimisation step on a teacher's top logits
  (:func:`bayes_ssm.distill.distillation_loss`).
* :meth:`SelectiveLM.prefill` runs prompts (of one length, or packed) and
  returns the logits after each one's last token and the state;
  :meth:`SelectiveLM.step` moves that state on by one token per sequence, at a
  cost that does not grow with the length.  :func:`generate` does both.

The convolution, the scan, their single-token forms and the loss run in this
package's kernels on CUDA tensors; the projections are PyTorch's GEMMs.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Sequence

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from .distill import distillation_loss
from .selective import PackedSequences, causal_conv, causal_conv_step, selective_scan, selective_step
from .six_layer import RMSNorm, SwiGLU


@dataclass
class MixerState:
    """What a mixer keeps of the tokens so far: the convolution's last inputs
    ``[B, taps - 1, inner]`` and the scan's state ``[B, inner, N]`` (float32)."""

    conv: Tensor
    scan: Tensor


class SelectiveMixer(nn.Module):
    def __init__(self, width: int, *, expand: int = 2, states: int = 16, groups: int = 1, taps: int = 4,
                 rank: Optional[int] = None, dtype: torch.dtype = torch.bfloat16, device=None) -> None:
        super().__init__()
        self.inner, self.states, self.groups = expand * width, states, groups
        if self.inner % groups:
            raise ValueError("groups must divide expand * width")
        self.rank = rank or max(1, math.ceil(width / 16))
        kw = dict(dtype=dtype, device=device)
        self.norm = RMSNorm(width, **kw)
        self.in_proj = nn.Linear(width, 2 * self.inner, bias=False, **kw)
        self.conv = nn.Conv1d(self.inner, self.inner, kernel_size=taps, groups=self.inner, **kw)
        self.x_proj = nn.Linear(self.inner, self.rank + 2 * groups * states, bias=False, **kw)
        self.step_proj = nn.Linear(self.rank, self.inner, bias=False, **kw)
        self.out_proj = nn.Linear(self.inner, width, bias=False, **kw)
        f32 = dict(dtype=torch.float32, device=device)
        # decay rates 1..N and steps spread over 1e-3..1e-1 after the softplus
        self.log_rates = nn.Parameter(torch.log(torch.arange(1, states + 1, **f32)).repeat(self.inner, 1))
        self.skip = nn.Parameter(torch.ones(self.inner, **f32))
        first = torch.exp(torch.linspace(math.log(1e-3), math.log(1e-1), self.inner, **f32))
        self.step_bias = nn.Parameter(first + torch.log(-torch.expm1(-first)))

    def _project(self, u: Tensor):
        low, keys, queries = self.x_proj(u).split([self.rank, self.groups * self.states, self.groups * self.states],
                                                  dim=-1)
        shape = (self.groups, self.states)
        return self.step_proj(low), keys.unflatten(-1, shape), queries.unflatten(-1, shape)

    def forward(self, x: Tensor, state: Optional[MixerState] = None,
                sequences: Optional[PackedSequences] = None) -> tuple[Tensor, MixerState]:
        values, gate = self.in_proj(self.norm(x)).chunk(2, dim=-1)
        u, conv = causal_conv(values, self.conv.weight, self.conv.bias, activation="silu",
                              initial_state=None if state is None else state.conv, sequences=sequences)
        steps, keys, queries = self._project(u)
        read, scan = selective_scan(u, steps, -torch.exp(self.log_rates), keys, queries, skip=self.skip, gate=gate,
                                    step_bias=self.step_bias, softplus=True,
                                    initial_state=None if state is None else state.scan, sequences=sequences)
        return self.out_proj(read), MixerState(conv, scan)

    def step(self, x: Tensor, state: MixerState) -> Tensor:
        """One token per sequence, ``x [B, width]``; ``state`` is moved on in place."""
        values, gate = self.in_proj(self.norm(x)).chunk(2, dim=-1)
        u = causal_conv_step(values, state.conv, self.conv.weight, self.conv.bias, activation="silu")
        steps, keys, queries = self._project(u)
        read = selective_step(u, steps, -torch.exp(self.log_rates), keys, queries, state.scan, skip=self.skip,
                              gate=gate, step_bias=self.step_bias, softplus=True)
        return self.out_proj(read)


class SelectiveBlock(nn.Module):
    def __init__(self, width: int, mlp_width: int, *, dtype, device, **mixer) -> None:
        super().__init__()
        self.mixer = SelectiveMixer(width, dtype=dtype, device=device, **mixer)
        self.ffn = SwiGLU(width, mlp_width, dtype=dtype, device=device)

    def forward(self, x: Tensor, state=None, sequences=None) -> tuple[Tensor, MixerState]:
        y, state = self.mixer(x, state, sequences)
        x = x + y
        return x + self.ffn(x), state

    def step(self, x: Tensor, state: MixerState) -> Tensor:
        x = x + self.mixer.step(x, state)
        return x + self.ffn(x)


class SelectiveLM(nn.Module):
    def __init__(self, vocab_size: int = 32_000, width: int = 512, layers: int = 6, mlp_width: int = 2048, *,
                 dtype: torch.dtype = torch.bfloat16, device=None, **mixer) -> None:
        super().__init__()
        self.vocab_size, self.width = vocab_size, width
        self.embedding = nn.Embedding(vocab_size, width, dtype=dtype, device=device)
        nn.init.normal_(self.embedding.weight, mean=0.0, std=0.02)
        self.blocks = nn.ModuleList(SelectiveBlock(width, mlp_width, dtype=dtype, device=device, **mixer)
                                    for _ in range(layers))
        self.final_norm = RMSNorm(width, dtype=dtype, device=device)

    def _head(self, x: Tensor) -> Tensor:
        return self.final_norm(x).float() @ self.embedding.weight.float().t()

    def forward(self, tokens: Tensor) -> Tensor:
        """Logits ``[B, T, V]`` (float32) of ``tokens [B, T]``."""
        x = self.embedding(tokens)
        for block in self.blocks:
            x, _ = block(x)
        return self._head(x)

    @torch.no_grad()
    def prefill(self, tokens: Tensor, sequences: Optional[PackedSequences] = None,
                state: Optional[list[MixerState]] = None) -> tuple[Tensor, list[MixerState]]:
        """Prompts ``tokens [B, T]``, or ``[tokens]`` packed: the logits after
        each one's last token ``[B, V]`` and the state, which a later call or
        :meth:`step` continues from.  No prompt may be empty."""
        if (sequences is None and tokens.shape[-1] == 0) or (sequences is not None and 0 in sequences.lengths):
            raise ValueError("prefill needs at least one token of every prompt")
        x = self.embedding(tokens)
        states = []
        for i, block in enumerate(self.blocks):
            x, s = block(x, None if state is None else state[i], sequences)
            states.append(s)
        last = x[:, -1] if sequences is None else x[sequences.offsets[1:] - 1]
        return self._head(last), states

    @torch.no_grad()
    def step(self, tokens: Tensor, state: list[MixerState]) -> Tensor:
        """One token per sequence, ``tokens [B]``: logits ``[B, V]``; ``state`` is moved on in place."""
        x = self.embedding(tokens)
        for block, s in zip(self.blocks, state):
            x = block.step(x, s)
        return self._head(x)


def distill_step(model: nn.Module, optimizer: torch.optim.Optimizer, inputs: Tensor, teacher_logits: Tensor,
                 teacher_indices: Tensor, *, temperature: float = 1.0, grad_clip: float = 1.0) -> Tensor:
    """One optimisation step on a teacher's top logits ``[B, T, K]`` at every
    position of ``inputs [B, T]`` (positions without a teacher have every index
    negative); returns the loss (on the device)."""
    optimizer.zero_grad(set_to_none=False)
    loss = distillation_loss(model(inputs), teacher_logits, teacher_indices, temperature=temperature)
    loss.backward()
    if grad_clip > 0:
        nn.utils.clip_grad_norm_(model.parameters(), grad_clip)
    optimizer.step()
    return loss.detach()


@torch.no_grad()
def generate(model: SelectiveLM, prompts: Sequence[Sequence[int]], new_tokens: int) -> Tensor:
    """Greedy continuations ``[len(prompts), new_tokens]`` of prompts of any
    lengths (one token at least): packed through :meth:`SelectiveLM.prefill`,
    then one :meth:`SelectiveLM.step` per token."""
    device = model.embedding.weight.device
    sequences = PackedSequences([len(p) for p in prompts], device=device)
    tokens = torch.tensor([t for p in prompts for t in p], device=device)
    logits, state = model.prefill(tokens, sequences)
    out = [logits.argmax(-1)]
    for _ in range(new_tokens - 1):
        out.append(model.step(out[-1], state).argmax(-1))
    return torch.stack(out[:new_tokens], 1) if new_tokens > 0 else tokens.new_zeros(len(prompts), 0)


__all__ = ["MixerState", "SelectiveMixer", "SelectiveBlock", "SelectiveLM", "distill_step", "generate"]
