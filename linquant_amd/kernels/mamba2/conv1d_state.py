"""Causal depthwise conv1d (+ SiLU) that carries its last inputs from call to call (HIP): prompts of any lengths and single tokens.
The reference's convolution (linquant/quantized_mamba2.py:262-268, ``causal_conv1d.py`` here) starts every prompt from zeros and
keeps nothing.  No gradients."""

from __future__ import annotations

import torch

from linquant_amd import _lib

_CODES = {torch.float16: _lib.LQ_DT_F16, torch.bfloat16: _lib.LQ_DT_BF16}


def check_slots(slots, n, num_slots, x):
    """``slots``: (n,) int32 or None, which stands for 0 .. n - 1."""
    if slots is None:
        assert n <= num_slots, f"{n} sequences, {num_slots} slots"
        return None
    assert slots.dtype == torch.int32 and slots.shape == (n,), f"slots: ({n},) int32"
    _lib.same_device(x, slots)
    return slots.contiguous()


def check_starts(seq_starts, x):
    assert seq_starts.dtype == torch.int32 and seq_starts.dim() == 1 and seq_starts.numel() >= 1, "seq_starts: (n + 1,) int32"
    _lib.same_device(x, seq_starts)
    return seq_starts.contiguous()


def _taps(x, weight, bias, activation):
    assert activation in (None, "silu", "swish") and x.dtype in _CODES
    D, W = weight.shape
    assert x.shape[-1] == D and 2 <= W <= 4 and D % 8 == 0, f"{x.shape[-1]} channels, weight {tuple(weight.shape)}"
    assert bias is None or bias.shape == (D,)
    _lib.below_2_31(*x.shape)
    _lib.same_device(x, weight, bias)
    weight = _lib.aligned(weight.to(x.dtype).contiguous())
    return weight, None if bias is None else _lib.aligned(bias.to(x.dtype).contiguous())


def _check_state(state, x, W):
    assert state.dim() == 3 and state.shape[1:] == (W - 1, x.shape[-1]) and state.dtype == x.dtype, \
        f"state: (slots, {W - 1}, {x.shape[-1]}) {x.dtype}, got {tuple(state.shape)} {state.dtype}"
    assert state.stride(2) == 1 and state.stride(0) % 8 == 0 and state.stride(1) % 8 == 0 and state.data_ptr() % 16 == 0
    _lib.same_device(x, state)


def conv1d_prompt(x, weight, bias=None, activation=None, *, state=None, slots=None, seq_starts=None):
    """y[t] = act(bias + sum_j weight[:, j] x[t - (W-1) + j]) over each prompt.  ``x`` fp16 or bf16: (B, L, D), or (T, D) with
    ``seq_starts`` (n + 1 int32, ascending) for packed prompts of any lengths; tokens outside them keep undefined outputs.
    ``weight`` (D, W), W 2 to 4, D a multiple of 8; taps and bias of another type are rounded to x's, as in ``causal_conv1d_fn``.  ``state`` (slots, W-1, D): the inputs in front of each prompt, oldest first,
    read and then replaced by its last W-1 (a prompt of no tokens leaves them); None: zeros in front, nothing kept.  ``slots``
    (n,) int32: each prompt's place in the state, all different; negative: zeros in front, nothing kept; beyond the state: NaN
    outputs.  Returns y, dense, in the shape of x."""
    if state is not None:
        out = _lib.native().conv1d_prompt(x, weight, bias, activation, state, slots, seq_starts)
        if out is not None:
            return out
    weight, bias = _taps(x, weight, bias, activation)
    D, W = weight.shape
    if seq_starts is None:
        assert x.dim() == 3, "x: (B, L, D), or (T, D) with seq_starts"
        n, L = x.shape[:2]
        x = _lib.rows16(x)
        dims = dict(x_stride_b=x.stride(0), x_stride_l=x.stride(1), seqlen=L)
    else:
        assert x.dim() == 2, "x: (T, D) with seq_starts"
        seq_starts = check_starts(seq_starts, x)
        n, L = seq_starts.numel() - 1, x.shape[0]
        x = _lib.rows16(x)
        dims = dict(x_stride_l=x.stride(0), tokens=L)
    num_slots = 0
    if state is not None:
        _check_state(state, x, W)
        num_slots = state.shape[0]
    slots = check_slots(slots, n, num_slots, x) if state is not None or slots is not None else None
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if n and L:
        _lib.call("lq_conv1d_prompt", x.device, x=_lib.ptr(x), dtype=_CODES[x.dtype], weight=_lib.ptr(weight), bias=_lib.ptr(bias),
                  out=_lib.ptr(out), state=_lib.ptr(state), state_stride_s=0 if state is None else state.stride(0),
                  state_stride_w=0 if state is None else state.stride(1), slots=_lib.ptr(slots if state is not None else None),
                  seq_starts=_lib.ptr(seq_starts), num_slots=num_slots, nseq=n, dim=D, width=W, silu=int(activation is not None), **dims)
    return out


def conv1d_step(x, state, weight, bias=None, activation=None, *, slots=None):
    """The same for one token of each sequence: ``x`` (B, D) -> (B, D), ``state`` moved on by it.  ``slots`` (B,) int32, all different;
    negative marks a padding entry (zeros out, no state touched), beyond the state: NaN outputs."""
    out = _lib.native().conv1d_step(x, state, weight, bias, activation, slots)
    if out is not None:
        return out
    weight, bias = _taps(x, weight, bias, activation)
    D, W = weight.shape
    assert x.dim() == 2, "x: (B, D)"
    _check_state(state, x, W)
    slots = check_slots(slots, x.shape[0], state.shape[0], x)
    x = _lib.rows16(x)
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.shape[0]:
        _lib.call("lq_conv1d_step", x.device, x=_lib.ptr(x), x_stride=x.stride(0), dtype=_CODES[x.dtype], weight=_lib.ptr(weight),
                  bias=_lib.ptr(bias), out=_lib.ptr(out), state=_lib.ptr(state), state_stride_s=state.stride(0), state_stride_w=state.stride(1),
                  slots=_lib.ptr(slots), num_slots=state.shape[0], batch=x.shape[0], dim=D, width=W, silu=int(activation is not None))
    return out
