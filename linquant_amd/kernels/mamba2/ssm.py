"""The selective state space scan of Mamba-2 with 16-bit activations and an fp32 state that a call starts from and ends in (HIP):
prompts of any lengths and single tokens.  It stands beside the INT8 forward of ``ssd_combined.py``
(linquant/kernels/mamba2/ssd_combined.py:19-131), which starts every prompt from zero and keeps no state.  No gradients."""

from __future__ import annotations

import ctypes
import functools

import torch

from linquant_amd import _lib

from .conv1d_state import check_slots, check_starts

_ACT = {torch.float16: _lib.LQ_DT_F16, torch.bfloat16: _lib.LQ_DT_BF16}
_FLOAT = {**_ACT, torch.float32: _lib.LQ_DT_F32}


def _params(x, dt, A, B, C, D, dt_bias, dt_softplus, dt_limit, lead):
    """Checks what both forms share; the fields of either args struct.  ``lead``: the token dimensions of x."""
    H, P = x.shape[-2:]
    G, N = B.shape[-2:]
    assert x.dtype in _ACT and B.dtype == x.dtype and C.dtype == x.dtype, "x, B and C: one type, fp16 or bf16"
    assert dt.dtype in _FLOAT and dt.shape == (*lead, H), f"dt: {(*lead, H)}, got {tuple(dt.shape)} {dt.dtype}"
    assert B.shape == (*lead, G, N) and C.shape == B.shape, f"B, C: {(*lead, 'G', 'N')}, got {tuple(B.shape)}, {tuple(C.shape)}"
    assert G >= 1 and H % G == 0 and P % 8 == 0 and N % 8 == 0 and 8 <= N <= 256, f"H {H} P {P} G {G} N {N}"
    assert A.shape == (H,) and (dt_bias is None or dt_bias.shape == (H,)) and (D is None or D.shape in ((H,), (H, P)))
    _lib.below_2_31(*x.shape)
    _lib.same_device(x, dt, A, B, C, D, dt_bias)
    A, D, dt_bias = (None if t is None else _lib.f32(t).contiguous() for t in (A, D, dt_bias))
    fields = dict(dtype=_ACT[x.dtype], dt_dtype=_FLOAT[dt.dtype], A=_lib.ptr(A), D=_lib.ptr(D), D_has_hdim=int(D is not None and D.dim() == 2),
                  dt_bias=_lib.ptr(dt_bias), dt_softplus=int(bool(dt_softplus)), dt_min=float(dt_limit[0]), dt_max=float(dt_limit[1]),
                  nheads=H, headdim=P, ngroups=G, dstate=N)
    return fields, (A, D, dt_bias)


def _check_state(state, x, N):
    H, P = x.shape[-2:]
    assert state.dtype == torch.float32 and state.dim() == 4 and state.shape[1:] == (H, P, N), \
        f"state: (slots, {H}, {P}, {N}) float32, got {tuple(state.shape)} {state.dtype}"
    assert state.shape[0] == 0 or (state[0].is_contiguous() and state.stride(0) % 4 == 0 and state.data_ptr() % 16 == 0), "state: dense slots"
    _lib.same_device(x, state)


@functools.lru_cache(maxsize=256)
def prompt_workspace_bytes(nseq, seqlen, tokens, packed, nheads, headdim, ngroups, dstate, dtype):
    st = _lib.fill("lq_ssm_prompt_args", nseq=nseq, seqlen=seqlen, tokens=tokens, seq_starts=16 if packed else None, nheads=nheads,
                   headdim=headdim, ngroups=ngroups, dstate=dstate, dtype=dtype)
    n = ctypes.c_int64(0)
    rc = _lib.load().lq_ssm_prompt_workspace_bytes(ctypes.byref(st), ctypes.byref(n))
    if rc != 0:
        _lib.raise_failed("lq_ssm_prompt_workspace_bytes", rc)
    return n.value


def ssm_prompt(x, dt, A, B, C, D=None, *, dt_bias=None, dt_softplus=True, dt_limit=(0.0, float("inf")), state=None, slots=None,
               seq_starts=None):
    """S = exp(d A) S + d x B^T,  y = S C + D x  over each prompt, d = clamp(softplus(dt + dt_bias), *dt_limit) (``dt_softplus``
    False: without the softplus).  ``x`` (B, L, H, P) fp16 or bf16, ``dt`` (B, L, H), ``B``, ``C`` (B, L, G, N), or each without
    its first dimension and with T tokens with ``seq_starts`` (n + 1 int32, ascending) for packed prompts of any lengths; tokens
    outside them keep undefined outputs.  ``A`` (H,) negative, ``D`` (H,) or (H, P).  P and N multiples of 8, N up to 256.  (A ``dt_limit``
    that lets steps be negative lets the state grow.)
    ``state`` (slots, H, P, N) fp32: what each prompt starts from, replaced by what it ends in (a prompt of no tokens leaves it);
    None: zero, nothing kept.  ``slots`` (n,) int32: each prompt's place in the state, all different; negative: from zero, nothing
    kept; beyond the state: NaN outputs.  An infinity in x, dt, B, C or the state counts as a NaN: it reaches the outputs and states that the formula
    has it reach, as one or the other.  Returns y, dense, in the shape and type of x."""
    if state is not None:
        out = _lib.native().ssm_prompt(x, dt, A, B, C, D, dt_bias, dt_softplus, dt_limit, state, slots, seq_starts)
        if out is not None:
            return out
    packed = seq_starts is not None
    assert x.dim() == (3 if packed else 4), "x: (B, L, H, P), or (T, H, P) with seq_starts"
    lead = x.shape[:-2]
    fields, keep = _params(x, dt, A, B, C, D, dt_bias, dt_softplus, dt_limit, lead)
    H, P = x.shape[-2:]
    N = B.shape[-1]
    if packed:
        seq_starts = check_starts(seq_starts, x)
        n, L, T = seq_starts.numel() - 1, 0, x.shape[0]
    else:
        (n, L), T = lead, 0
    num_slots = 0
    if state is not None:
        _check_state(state, x, N)
        num_slots = state.shape[0]
    slots = check_slots(slots, n, num_slots, x) if state is not None or slots is not None else None
    x, B, C = (_lib.rows16(t) for t in (x, B, C))
    if x.stride(-3) >= 1 << 24:
        x = x.contiguous()
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if n == 0 or L + T == 0 or H == 0 or P == 0:
        return out
    st = lambda t: (0, *t.stride()) if packed else t.stride()  # noqa: E731
    xs, ds, bs, cs = st(x), st(dt), st(B), st(C)
    nbytes = prompt_workspace_bytes(n, L, T, packed, H, P, B.shape[-2], N, fields["dtype"])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    _lib.call("lq_ssm_prompt", x.device, x=_lib.ptr(x), x_stride_b=xs[0], x_stride_l=xs[1], x_stride_h=xs[2], dt=_lib.ptr(dt),
              dt_stride_b=ds[0], dt_stride_l=ds[1], dt_stride_h=ds[2], B=_lib.ptr(B), B_stride_b=bs[0], B_stride_l=bs[1],
              B_stride_g=bs[2], C=_lib.ptr(C), C_stride_b=cs[0], C_stride_l=cs[1], C_stride_g=cs[2], out=_lib.ptr(out),
              state=_lib.ptr(state), state_stride_s=0 if state is None else state.stride(0),
              slots=_lib.ptr(slots if state is not None else None), seq_starts=_lib.ptr(seq_starts), num_slots=num_slots, nseq=n,
              seqlen=L, tokens=T, workspace=_lib.ptr(ws), workspace_bytes=nbytes, **fields)
    del keep
    return out


def ssm_step(state, x, dt, A, B, C, D=None, *, dt_bias=None, dt_softplus=True, dt_limit=(0.0, float("inf")), slots=None):
    """The same for one token of each of up to 65535 sequences: ``x`` (B, H, P), ``dt`` (B, H), ``B``, ``C`` (B, G, N) -> y (B, H, P), ``state``
    (slots, H, P, N) fp32 moved on by it.  ``slots`` (B,) int32, all different; negative marks a padding entry (zeros out, no
    state touched), beyond the state: NaN outputs."""
    out = _lib.native().ssm_step(x, dt, A, B, C, D, dt_bias, dt_softplus, dt_limit, state, slots)
    if out is not None:
        return out
    assert x.dim() == 3, "x: (B, H, P)"
    fields, keep = _params(x, dt, A, B, C, D, dt_bias, dt_softplus, dt_limit, x.shape[:1])
    n, H, P = x.shape
    _check_state(state, x, B.shape[-1])
    slots = check_slots(slots, n, state.shape[0], x)
    B, C = _lib.rows16(B), _lib.rows16(C)
    x = x if x.stride(2) == 1 else x.contiguous()
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if n and H and P:
        _lib.call("lq_ssm_step", x.device, x=_lib.ptr(x), x_stride_b=x.stride(0), x_stride_h=x.stride(1), dt=_lib.ptr(dt), dt_stride_b=dt.stride(0),
                  dt_stride_h=dt.stride(1), B=_lib.ptr(B), B_stride_b=B.stride(0), B_stride_g=B.stride(1), C=_lib.ptr(C),
                  C_stride_b=C.stride(0), C_stride_g=C.stride(1), out=_lib.ptr(out), state=_lib.ptr(state), state_stride_s=state.stride(0),
                  slots=_lib.ptr(slots), num_slots=state.shape[0], batch=n, **fields)
    del keep
    return out
