"""Selective state space operators: a short causal convolution and the scan.

Per channel, the scan keeps a state of ``N`` values that decays by its own
rates at a step size chosen token by token:

* ``d_t = softplus(steps_t + step_bias)`` (or the sum itself);
* ``h_t = exp(d_t * rates) * h_{t-1} + d_t * values_t * keys_t``;
* ``read_t = (queries_t . h_t + skip * values_t) * silu(gate_t)``.

Keys and queries are shared by the channels of a group.  The convolution in
front of it is depthwise over the last few tokens.  Both take equal-length
rows ``[B, T, ...]`` or, with :class:`PackedSequences`, the rows of uneven
sequences one after the other ``[tokens, ...]``; both begin from a given state
or zeros and return the state after the last token, so a prompt can be
continued in pieces with the same call, or token by token with
:func:`causal_conv_step` and :func:`selective_step`, which move the states on
in place.

On CUDA the work runs in this package's sm_100a kernels (``csrc/bssm_conv.cu``,
``csrc/bssm_selective.cu``) on the current stream, with gradients for every
input of :func:`causal_conv` and :func:`selective_scan`; sums and states are
float32 whatever the rows' type, and results do not differ from run to run.
Forward-mode derivatives are refused.  On CPU tensors the same formulas run as
PyTorch operations.
"""
from __future__ import annotations

from numbers import Integral
from typing import Optional, Sequence

import torch
import torch.nn.functional as F
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _capi

_DTYPES = {torch.float32: _capi.BSSM_F32, torch.bfloat16: _capi.BSSM_BF16, torch.float16: _capi.BSSM_F16}
MAX_STATES = 64


class PackedSequences:
    """The lengths of sequences whose rows lie one after the other.

    ``lengths`` are whole numbers (zero is allowed), known on the host; the
    offsets the kernels read are put on ``device`` once.  One object serves
    every layer and call that takes rows of these sequences.
    """

    def __init__(self, lengths: Sequence[int], *, device) -> None:
        if isinstance(lengths, Tensor):
            if lengths.ndim != 1 or lengths.is_floating_point() or lengths.is_complex() or lengths.dtype == torch.bool:
                raise ValueError("lengths must be a one-dimensional tensor of whole numbers")
            lengths = lengths.tolist()
        self.lengths = list(lengths)
        if any(isinstance(n, bool) or not isinstance(n, Integral) or n < 0 for n in self.lengths):
            raise ValueError("lengths must be whole numbers, zero or more")
        starts = [0]
        for n in self.lengths:
            starts.append(starts[-1] + int(n))
        self.count, self.tokens = len(self.lengths), starts[-1]
        self.longest = max(self.lengths, default=0)
        self.starts = starts
        self.offsets = torch.tensor(starts, dtype=torch.int64).to(device)


def _rows(x: Tensor, trailing: int) -> tuple[Tensor, int]:
    """``x`` with its trailing dimensions contiguous and its rows evenly
    spaced (a copy where they are not), and the spacing in elements."""
    inner = x.shape[-1] if trailing == 1 else x.shape[-1] * x.shape[-2]
    if x.is_contiguous():
        return x, inner
    sizes, strides = x.shape, x.stride()
    even = sizes[-1] == 1 or strides[-1] == 1
    if trailing == 2:
        even &= sizes[-2] == 1 or strides[-2] == sizes[-1]
    row = expect = None
    for size, stride in zip(reversed(sizes[:-trailing]), reversed(strides[:-trailing])):
        if size == 1:
            continue
        if row is None:
            row = expect = stride
        even &= stride == expect
        expect = stride * size
    if row is None:
        row = inner
    if not even or row < inner:
        return x.contiguous(), inner
    return x, row


def _empty_like(x: Tensor) -> Tensor:
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, device=x.device, dtype=x.dtype)


def _check_devices(first: Tensor, **others) -> None:
    device = first.device
    for name, x in others.items():
        if x is not None and x.device != device:
            raise ValueError(f"{name} must be on the same device as the rows")


def _layout(lead: torch.Size, sequences: Optional[PackedSequences], device) -> tuple[int, int, int, Optional[int]]:
    """Number of sequences, of token rows, the longest sequence, and the offsets' address."""
    if sequences is None:
        if len(lead) != 2:
            raise ValueError("rows must be [B, T, ...], or [tokens, ...] with sequences")
        return lead[0], lead[0] * lead[1], lead[1], None
    if not isinstance(sequences, PackedSequences):
        raise TypeError("sequences must be PackedSequences")
    if len(lead) != 1 or lead[0] != sequences.tokens:
        raise ValueError(f"rows must be [{sequences.tokens}, ...] for these sequences")
    if sequences.offsets.device != device:
        raise ValueError("sequences must be on the same device as the rows")
    return sequences.count, sequences.tokens, sequences.longest, sequences.offsets.data_ptr()


def _gradients_wanted(*tensors) -> bool:
    if torch.is_grad_enabled():
        for x in tensors:
            if x is not None and x.requires_grad:
                return True
    return False


def _carries_tangent(*tensors) -> bool:
    """Whether a tensor is a dual one, of forward-mode differentiation (which no grad mode turns off).  The kernels
    have none: the autograd functions raise on such a tensor, where the bare calls would drop its tangent."""
    if forward_ad._current_level < 0:
        return False
    return any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in tensors)


def _written(x: Tensor) -> None:
    """Tells autograd that a kernel wrote ``x``: a backward that saved it must not read it any more."""
    if not x.is_inference():  # has no version to count
        torch.autograd.graph.increment_version(x)


# ---------------------------------------------------------------------------
# Causal convolution
# ---------------------------------------------------------------------------

def _conv_arguments(x, weight, bias, activation):
    channels = x.shape[-1]
    if weight.ndim == 3 and weight.shape[1] == 1:
        weight = weight.reshape(weight.shape[0], weight.shape[2])
    if weight.ndim != 2 or weight.shape[0] != channels:
        raise ValueError(f"weight must be [{channels}, taps] or [{channels}, 1, taps]")
    if bias is not None and bias.shape != (channels,):
        raise ValueError(f"bias must be [{channels}]")
    if activation not in (None, "silu"):
        raise ValueError("activation must be None or 'silu'")
    if not (x.is_floating_point() and weight.is_floating_point() and (bias is None or bias.is_floating_point())):
        raise TypeError("x, weight and bias must have floating-point dtype")
    _check_devices(x, weight=weight, bias=bias)
    if x.is_cuda:
        if x.dtype not in _DTYPES or weight.dtype not in _DTYPES or (bias is not None and bias.dtype not in _DTYPES):
            raise TypeError("causal_conv on CUDA takes float32, bfloat16 or float16 tensors")
        if not 2 <= weight.shape[1] <= 4:
            raise NotImplementedError(f"causal_conv on CUDA needs 2, 3 or 4 taps (got {weight.shape[1]}); "
                                      "use causal_conv_torch")
    elif weight.shape[1] < 2:
        raise ValueError("weight must have at least 2 taps")
    return weight


def causal_conv_torch(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, activation: Optional[str] = None,
                      initial_state: Optional[Tensor] = None,
                      sequences: Optional[PackedSequences] = None) -> tuple[Tensor, Tensor]:
    """:func:`causal_conv` in PyTorch operations, computed in float32 (float64
    for float64 rows)."""
    weight = weight.reshape(weight.shape[0], weight.shape[-1])
    wide = torch.promote_types(x.dtype, torch.float32)
    taps, channels = weight.shape[1], x.shape[-1]
    rows = list(x) if sequences is None else list(torch.split(x, sequences.lengths)) if sequences.count else []
    ys, states = [], []
    for i, r in enumerate(rows):
        past = r.new_zeros(taps - 1, channels) if initial_state is None else initial_state[i]
        w = torch.cat([past, r])
        u = sum(w[j:j + r.shape[0]].to(wide) * weight[:, j].to(wide) for j in range(taps))
        if bias is not None:
            u = u + bias.to(wide)
        ys.append((F.silu(u) if activation == "silu" else u).to(x.dtype))
        states.append(w[r.shape[0]:])
    if not rows:
        return torch.zeros_like(x), x.new_zeros(0, taps - 1, channels)
    return (torch.stack(ys) if sequences is None else torch.cat(ys)), torch.stack(states)


def _conv_forward(x, weight, bias, silu, state, count, tokens, offsets):
    channels, taps = weight.shape
    x, stride = _rows(x, 1)
    weight = weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    state = None if state is None else state.contiguous()
    y = _empty_like(x)
    final = torch.empty(count, taps - 1, channels, device=x.device, dtype=x.dtype)
    _capi.launch(x.device, "bssm_causal_conv", x.data_ptr(), _DTYPES[x.dtype], stride, tokens, channels, taps,
                 weight.data_ptr(), _DTYPES[weight.dtype], _capi.ptr(bias),
                 0 if bias is None else _DTYPES[bias.dtype], silu, offsets, count, _capi.ptr(state), y.data_ptr(),
                 final.data_ptr())
    return y, final


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, silu, count, tokens, sequences):
        offsets = None if sequences is None else sequences.offsets.data_ptr()
        ctx.save_for_backward(x, weight, bias, state)
        ctx.layout = (silu, count, tokens, sequences)
        ctx.set_materialize_grads(False)
        return _conv_forward(x, weight, bias, silu, state, count, tokens, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gfinal):
        x, weight, bias, state = ctx.saved_tensors
        silu, count, tokens, sequences = ctx.layout
        channels, taps = weight.shape
        dev = x.device
        gy = torch.zeros(x.shape, device=dev, dtype=x.dtype) if gy is None else gy.to(x.dtype).contiguous()
        gfinal = None if gfinal is None else gfinal.to(x.dtype).contiguous()
        rows, stride = _rows(x, 1)
        wt = weight.contiguous()
        b = None if bias is None else bias.contiguous()
        past = None if state is None else state.contiguous()
        gx, gw = _empty_like(rows), _empty_like(wt)
        gb = None if b is None else torch.empty_like(b)
        gs = None if past is None else torch.empty_like(past)
        room = _capi.load().bssm_causal_conv_partial_floats(tokens, channels, taps)
        ws = torch.empty(room, device=dev, dtype=torch.float32)
        _capi.launch(dev, "bssm_causal_conv_backward", rows.data_ptr(), _DTYPES[x.dtype], stride, tokens, channels,
                     taps, wt.data_ptr(), _DTYPES[wt.dtype], _capi.ptr(b), 0 if b is None else _DTYPES[b.dtype], silu,
                     None if sequences is None else sequences.offsets.data_ptr(), count, _capi.ptr(past),
                     gy.data_ptr(), _capi.ptr(gfinal), gx.data_ptr(), gw.data_ptr(), _capi.ptr(gb), _capi.ptr(gs),
                     ws.data_ptr(), room)
        return gx, gw, gb, gs, None, None, None, None


def causal_conv(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, activation: Optional[str] = None,
                initial_state: Optional[Tensor] = None,
                sequences: Optional[PackedSequences] = None) -> tuple[Tensor, Tensor]:
    """Depthwise causal convolution; returns ``(y, final_state)``.

    ``x`` is ``[B, T, C]``, or ``[tokens, C]`` with ``sequences``; ``weight``
    ``[C, taps]`` (or a Conv1d's ``[C, 1, taps]``), its last tap the current
    token's; ``activation`` None or ``"silu"``.  ``initial_state``
    ``[B, taps - 1, C]`` holds the inputs before the first token, oldest first
    (zeros without it), in ``x``'s dtype, and ``final_state`` the last ones
    after it.  CUDA takes 2, 3 or 4 taps; weight and bias may have another
    floating dtype than ``x``.
    """
    weight = _conv_arguments(x, weight, bias, activation)
    count, tokens, _, offsets = _layout(x.shape[:-1], sequences, x.device)
    if initial_state is not None:
        if initial_state.shape != (count, weight.shape[1] - 1, x.shape[-1]):
            raise ValueError(f"initial_state must be [{count}, {weight.shape[1] - 1}, {x.shape[-1]}]")
        if initial_state.dtype != x.dtype:
            raise TypeError("initial_state must have x's dtype")
        _check_devices(x, initial_state=initial_state)
    if not x.is_cuda:
        return causal_conv_torch(x, weight, bias, activation=activation, initial_state=initial_state,
                                 sequences=sequences)
    silu = int(activation == "silu")
    if _gradients_wanted(x, weight, bias, initial_state) or _carries_tangent(x, weight, bias, initial_state):
        return _CausalConv.apply(x, weight, bias, initial_state, silu, count, tokens, sequences)
    return _conv_forward(x, weight, bias, silu, initial_state, count, tokens, offsets)


def causal_conv_step(x: Tensor, state: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *,
                     activation: Optional[str] = None) -> Tensor:
    """One token of :func:`causal_conv` for each of B sequences: ``x [B, C]``;
    ``state [B, taps - 1, C]`` is moved on in place.  No gradients."""
    if x.ndim != 2:
        raise ValueError("x must be [B, C]")
    weight = _conv_arguments(x, weight, bias, activation)
    if state.shape != (x.shape[0], weight.shape[1] - 1, x.shape[1]):
        raise ValueError(f"state must be [{x.shape[0]}, {weight.shape[1] - 1}, {x.shape[1]}]")
    if state.dtype != x.dtype:
        raise TypeError("state must have x's dtype")
    _check_devices(x, state=state)
    if _gradients_wanted(x, weight, bias, state):
        raise RuntimeError("causal_conv_step has no gradient: call it under torch.no_grad(), or causal_conv")
    if not x.is_cuda:
        y, final = causal_conv_torch(x[:, None], weight, bias, activation=activation, initial_state=state)
        state.copy_(final)
        return y[:, 0]
    if _carries_tangent(x, weight, bias, state):
        raise RuntimeError("causal_conv_step has no gradient, in forward mode either: call causal_conv")
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is moved on in place")
    x, stride = _rows(x, 1)
    weight = weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    y = _empty_like(x)
    _capi.launch(x.device, "bssm_causal_conv_step", x.data_ptr(), _DTYPES[x.dtype], stride, x.shape[0], x.shape[1],
                 weight.shape[1], weight.data_ptr(), _DTYPES[weight.dtype], _capi.ptr(bias),
                 0 if bias is None else _DTYPES[bias.dtype], int(activation == "silu"), state.data_ptr(),
                 y.data_ptr())
    _written(state)
    return y


# ---------------------------------------------------------------------------
# Selective scan
# ---------------------------------------------------------------------------

def _scan_arguments(values, steps, rates, keys, queries, skip, gate, step_bias):
    """Checks shapes, dtypes and devices; returns the groups of keys and queries, and the per-channel tensors in
    float32 (on CUDA)."""
    shape, dtype, lead = values.shape, values.dtype, values.ndim - 1
    channels = shape[-1]
    for x in (values, steps, rates, keys, queries, skip, gate, step_bias):
        if x is not None and not x.is_floating_point():
            raise TypeError("selective_scan takes floating-point tensors")
    if steps.shape != shape or (gate is not None and gate.shape != shape):
        raise ValueError("steps and gate must have the values' shape")
    if rates.ndim != 2 or rates.shape[0] != channels or rates.shape[1] < 1:
        raise ValueError(f"rates must be [{channels}, N]")
    n = rates.shape[1]
    groups = keys.shape[-2] if keys.ndim == lead + 2 else 1
    if keys.shape != queries.shape or keys.ndim not in (lead + 1, lead + 2) or keys.shape[:lead] != shape[:lead] \
            or keys.shape[-1] != n:
        raise ValueError(f"keys and queries must be [..., {n}] or [..., G, {n}] with the values' leading dimensions")
    if groups < 1 or channels % groups:
        raise ValueError("the groups of keys and queries must divide the channels")
    if skip is not None and skip.shape != (channels,):
        raise ValueError(f"skip must be [{channels}]")
    if step_bias is not None and step_bias.shape != (channels,):
        raise ValueError(f"step_bias must be [{channels}]")
    if steps.dtype != dtype or keys.dtype != dtype or queries.dtype != dtype or (gate is not None
                                                                                and gate.dtype != dtype):
        raise TypeError("values, steps, keys, queries and gate must have one dtype")
    _check_devices(values, steps=steps, rates=rates, keys=keys, queries=queries, skip=skip, gate=gate,
                   step_bias=step_bias)
    if values.is_cuda:
        if dtype not in _DTYPES:
            raise TypeError("selective_scan on CUDA takes float32, bfloat16 or float16 rows")
        if n > MAX_STATES:
            raise NotImplementedError(f"selective_scan on CUDA needs at most {MAX_STATES} states (got {n}); "
                                      "use selective_scan_torch")
        rates = rates.float()
        skip = None if skip is None else skip.float()
        step_bias = None if step_bias is None else step_bias.float()
    return groups, rates, skip, step_bias


def selective_scan_torch(values: Tensor, steps: Tensor, rates: Tensor, keys: Tensor, queries: Tensor, *,
                         skip: Optional[Tensor] = None, gate: Optional[Tensor] = None,
                         step_bias: Optional[Tensor] = None, softplus: bool = False,
                         initial_state: Optional[Tensor] = None,
                         sequences: Optional[PackedSequences] = None) -> tuple[Tensor, Tensor]:
    """:func:`selective_scan` in PyTorch operations, token by token, computed in
    float32 (float64 for float64 rows)."""
    wide = torch.promote_types(values.dtype, torch.float32)
    channels, n = rates.shape
    if keys.ndim == values.ndim:
        keys, queries = keys.unsqueeze(-2), queries.unsqueeze(-2)
    repeat = channels // keys.shape[-2]
    d = steps.to(wide) if step_bias is None else steps.to(wide) + step_bias.to(wide)
    if softplus:
        d = F.softplus(d)
    rates = rates.to(wide)

    def runs(x):
        if sequences is None:
            return list(x)
        return list(torch.split(x, sequences.lengths)) if sequences.count else []

    reads, states = [], []
    for i, (x, dt, k, q) in enumerate(zip(runs(values.to(wide)), runs(d), runs(keys.to(wide)),
                                          runs(queries.to(wide)))):
        h = x.new_zeros(channels, n) if initial_state is None else initial_state[i].to(wide)
        out = []
        for t in range(x.shape[0]):
            h = torch.exp(dt[t, :, None] * rates) * h \
                + (dt[t] * x[t])[:, None] * k[t].repeat_interleave(repeat, dim=0)
            out.append((h * q[t].repeat_interleave(repeat, dim=0)).sum(-1))
        reads.append(torch.stack(out) if out else x)
        states.append(h)
    if not reads:
        return torch.zeros_like(values), rates.new_zeros(0, channels, n)
    r = torch.stack(reads) if sequences is None else torch.cat(reads)
    if skip is not None:
        r = r + skip.to(wide) * values.to(wide)
    if gate is not None:
        r = r * F.silu(gate.to(wide))
    return r.to(values.dtype), torch.stack(states)


def _scan_rows(values, steps, keys, queries, gate):
    """The row arguments (kept alive by the caller) and, for the C call, their addresses and spacings."""
    trailing = keys.ndim - values.ndim + 1
    x, xs = _rows(values, 1)
    s, ss = _rows(steps, 1)
    k, ks = _rows(keys, trailing)
    q, qs = _rows(queries, trailing)
    z, zs = (None, 0) if gate is None else _rows(gate, 1)
    return (x, s, k, q, z), (x.data_ptr(), xs, s.data_ptr(), ss, k.data_ptr(), ks, q.data_ptr(), qs, _capi.ptr(z), zs)


def _scan_forward(values, steps, rates, keys, queries, skip, gate, step_bias, state, groups, softplus, count, tokens,
                  longest, offsets, save):
    dev = values.device
    channels, n = rates.shape
    lib = _capi.load()
    kept, flat = _scan_rows(values, steps, keys, queries, gate)
    rates, state = rates.contiguous(), None if state is None else state.contiguous()
    skip = None if skip is None else skip.contiguous()
    step_bias = None if step_bias is None else step_bias.contiguous()
    out = _empty_like(values)
    final = torch.empty(count, channels, n, device=dev, dtype=torch.float32)
    room = lib.bssm_selective_scan_floats(tokens, count, longest, channels, n, groups)
    ws = torch.empty(room, device=dev, dtype=torch.float32) if room else None
    saved, saved_room = None, 0
    if save:
        saved_room = lib.bssm_selective_saved_floats(tokens, count, channels, n)
        saved = torch.empty(saved_room, device=dev, dtype=torch.float32)
    _capi.launch(dev, "bssm_selective_scan", *flat, _DTYPES[values.dtype], rates.data_ptr(), _capi.ptr(skip),
                 _capi.ptr(step_bias), softplus, tokens, channels, n, groups, offsets, count, longest,
                 _capi.ptr(state), out.data_ptr(), final.data_ptr(), _capi.ptr(saved), saved_room, _capi.ptr(ws), room)
    del kept
    return out, final, saved


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, values, steps, rates, keys, queries, skip, gate, step_bias, state, groups, softplus, count,
                tokens, longest, sequences):
        offsets = None if sequences is None else sequences.offsets.data_ptr()
        out, final, saved = _scan_forward(values, steps, rates, keys, queries, skip, gate, step_bias, state, groups,
                                          softplus, count, tokens, longest, offsets, True)
        ctx.save_for_backward(values, steps, rates, keys, queries, skip, gate, step_bias, saved)
        ctx.layout = (groups, softplus, count, tokens, longest, sequences, state is not None)
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @once_differentiable
    def backward(ctx, gout, gfinal):
        values, steps, rates, keys, queries, skip, gate, step_bias, saved = ctx.saved_tensors
        groups, softplus, count, tokens, longest, sequences, has_state = ctx.layout
        dev, dtype = values.device, values.dtype
        channels, n = rates.shape
        kept, flat = _scan_rows(values, steps, keys, queries, gate)
        a = rates.contiguous()
        sk = None if skip is None else skip.contiguous()
        sb = None if step_bias is None else step_bias.contiguous()
        gout = None if gout is None else gout.to(dtype).contiguous()
        gfinal = None if gfinal is None else gfinal.float().contiguous()
        gv, gs, gk, gq = _empty_like(values), _empty_like(steps), _empty_like(keys), _empty_like(queries)
        gz = None if gate is None else _empty_like(gate)
        ga = torch.empty_like(a)
        gskip = None if sk is None else torch.empty_like(sk)
        gbias = None if sb is None else torch.empty_like(sb)
        g0 = torch.empty(count, channels, n, device=dev, dtype=torch.float32) if has_state else None
        room = _capi.load().bssm_selective_backward_floats(tokens, count, longest, channels, n, groups)
        ws = torch.empty(room, device=dev, dtype=torch.float32)
        _capi.launch(dev, "bssm_selective_scan_backward", *flat, _DTYPES[dtype], a.data_ptr(), _capi.ptr(sk),
                     _capi.ptr(sb), softplus, tokens, channels, n, groups,
                     None if sequences is None else sequences.offsets.data_ptr(), count, longest, saved.data_ptr(),
                     _capi.ptr(gout), _capi.ptr(gfinal), gv.data_ptr(), gs.data_ptr(), ga.data_ptr(), gk.data_ptr(),
                     gq.data_ptr(), _capi.ptr(gskip), _capi.ptr(gz), _capi.ptr(gbias), _capi.ptr(g0), ws.data_ptr(),
                     room)
        del kept
        return gv, gs, ga, gk, gq, gskip, gz, gbias, g0, None, None, None, None, None, None


def selective_scan(values: Tensor, steps: Tensor, rates: Tensor, keys: Tensor, queries: Tensor, *,
                   skip: Optional[Tensor] = None, gate: Optional[Tensor] = None, step_bias: Optional[Tensor] = None,
                   softplus: bool = False, initial_state: Optional[Tensor] = None,
                   sequences: Optional[PackedSequences] = None) -> tuple[Tensor, Tensor]:
    """The selective scan; returns ``(read, final_state)`` (see the module docstring).

    ``values``, ``steps`` and ``gate`` are ``[B, T, C]`` (``[tokens, C]`` with
    ``sequences``), ``keys`` and ``queries`` ``[B, T, N]`` or ``[B, T, G, N]``
    where the C channels divide evenly into G groups, all of one dtype, which
    ``read`` has too.  ``rates [C, N]`` (negative for states that decay),
    ``skip [C]`` and ``step_bias [C]`` are used in float32.  ``initial_state``
    and ``final_state`` are float32 ``[B, C, N]``.  CUDA takes up to 64 states.
    A token whose step is zero leaves the state as it is.
    """
    groups, rates, skip, step_bias = _scan_arguments(values, steps, rates, keys, queries, skip, gate, step_bias)
    count, tokens, longest, offsets = _layout(values.shape[:-1], sequences, values.device)
    if initial_state is not None:
        if initial_state.shape != (count, *rates.shape):
            raise ValueError(f"initial_state must be [{count}, {rates.shape[0]}, {rates.shape[1]}]")
        _check_devices(values, initial_state=initial_state)
    if not values.is_cuda:
        return selective_scan_torch(values, steps, rates, keys, queries, skip=skip, gate=gate, step_bias=step_bias,
                                    softplus=softplus, initial_state=initial_state, sequences=sequences)
    if initial_state is not None:
        initial_state = initial_state.float()
    args = (values, steps, rates, keys, queries, skip, gate, step_bias, initial_state)
    if _gradients_wanted(*args) or _carries_tangent(*args):
        return _SelectiveScan.apply(*args, groups, int(softplus), count, tokens, longest, sequences)
    return _scan_forward(*args, groups, int(softplus), count, tokens, longest, offsets, False)[:2]


def selective_step(values: Tensor, steps: Tensor, rates: Tensor, keys: Tensor, queries: Tensor, state: Tensor, *,
                   skip: Optional[Tensor] = None, gate: Optional[Tensor] = None, step_bias: Optional[Tensor] = None,
                   softplus: bool = False) -> Tensor:
    """One token of :func:`selective_scan` for each of B sequences.

    ``values``, ``steps`` and ``gate`` are ``[B, C]``, ``keys`` and ``queries``
    ``[B, N]`` or ``[B, G, N]``; ``state`` (float32 ``[B, C, N]``, contiguous)
    is moved on in place.  Returns the read ``[B, C]``.  No gradients.
    """
    if values.ndim != 2:
        raise ValueError("values must be [B, C]")
    groups, rates, skip, step_bias = _scan_arguments(values, steps, rates, keys, queries, skip, gate, step_bias)
    b, (channels, n) = values.shape[0], rates.shape
    if state.shape != (b, channels, n):
        raise ValueError(f"state must be [{b}, {channels}, {n}]")
    _check_devices(values, state=state)
    if _gradients_wanted(values, steps, rates, keys, queries, state, skip, gate, step_bias):
        raise RuntimeError("selective_step has no gradient: call it under torch.no_grad(), or selective_scan")
    if not values.is_cuda:
        def one(x):
            return None if x is None else x[:, None]
        read, final = selective_scan_torch(one(values), one(steps), rates, one(keys), one(queries), skip=skip,
                                           gate=one(gate), step_bias=step_bias, softplus=softplus,
                                           initial_state=state)
        state.copy_(final)
        return read[:, 0]
    if _carries_tangent(values, steps, rates, keys, queries, state, skip, gate, step_bias):
        raise RuntimeError("selective_step has no gradient, in forward mode either: call selective_scan")
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError("state must be float32 and contiguous: it is moved on in place")
    kept, flat = _scan_rows(values, steps, keys, queries, gate)
    rates = rates.contiguous()
    skip = None if skip is None else skip.contiguous()
    step_bias = None if step_bias is None else step_bias.contiguous()
    out = _empty_like(values)
    _capi.launch(values.device, "bssm_selective_step", *flat, _DTYPES[values.dtype], rates.data_ptr(),
                 _capi.ptr(skip), _capi.ptr(step_bias), int(softplus), b, channels, n, groups, state.data_ptr(),
                 out.data_ptr())
    _written(state)
    del kept
    return out


__all__ = ["PackedSequences", "causal_conv", "causal_conv_torch", "causal_conv_step", "selective_scan",
           "selective_scan_torch", "selective_step"]
