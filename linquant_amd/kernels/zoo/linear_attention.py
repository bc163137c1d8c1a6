"""Linear attention with no decay, one for each head, or one for each head and token, with 16-bit activations and an fp32 state that a
call starts from and ends in (HIP): prompts of any lengths and single tokens.  It stands beside the INT8 chunk forward of
``simple_gla.py`` (linquant/kernels/zoo/simple_gla.py:175-212), which starts every prompt from zero and takes whole chunks.  No gradients."""

from __future__ import annotations

import ctypes
import functools

import torch

from linquant_amd import _lib
from linquant_amd.kernels.mamba2.conv1d_state import check_slots, check_starts

_ACT = {torch.float16: _lib.LQ_DT_F16, torch.bfloat16: _lib.LQ_DT_BF16}
_FLOAT = {**_ACT, torch.float32: _lib.LQ_DT_F32}


def _check(q, k, v, g, scale, lead):
    """Checks what both forms share; the fields of either args struct.  ``lead``: the token dimensions of v."""
    H, V = v.shape[-2:]
    K = q.shape[-1]
    assert v.dtype in _ACT and q.dtype == v.dtype and k.dtype == v.dtype, "q, k and v: one type, fp16 or bf16"
    assert q.shape == (*lead, H, K) and k.shape == q.shape, f"q, k: {(*lead, H, 'K')}, got {tuple(q.shape)}, {tuple(k.shape)}"
    assert K % 8 == 0 and 8 <= K <= 256 and V % 8 == 0, f"K {K} V {V}: multiples of 8, K up to 256"
    assert g is None or (g.dtype in _FLOAT and g.shape in ((H,), (*lead, H))), f"g: {(H,)} or {(*lead, H)}, got {None if g is None else tuple(g.shape)}"
    _lib.below_2_31(*q.shape, V)
    _lib.same_device(q, k, v, g)
    return dict(dtype=_ACT[v.dtype], scale=float(K ** -0.5 if scale is None else scale),
                nheads=H, kdim=K, vdim=V)


def _check_state(state, q, V):
    H, K = q.shape[-2:]
    assert state.dtype == torch.float32 and state.dim() == 4 and state.shape[1:] == (H, K, V), \
        f"state: (slots, {H}, {K}, {V}) float32, got {tuple(state.shape)} {state.dtype}"
    n = state.shape[0]
    assert n == 0 or (state[0].is_contiguous() and state.stride(0) % 4 == 0 and state.data_ptr() % 16 == 0), "state: dense slots"
    assert n <= 1 or state.stride(0) >= state[0].numel(), "state: slots that do not overlap"
    _lib.same_device(q, state)


@functools.lru_cache(maxsize=256)
def prompt_workspace_bytes(nseq, seqlen, tokens, packed, nheads, kdim, vdim, dtype):
    st = _lib.fill("lq_linear_attention_prompt_args", nseq=nseq, seqlen=seqlen, tokens=tokens, seq_starts=16 if packed else None, nheads=nheads,
                   kdim=kdim, vdim=vdim, dtype=dtype)
    n = ctypes.c_int64(0)
    rc = _lib.load().lq_linear_attention_prompt_workspace_bytes(ctypes.byref(st), ctypes.byref(n))
    if rc != 0:
        _lib.raise_failed("lq_linear_attention_prompt_workspace_bytes", rc)
    return n.value


def linear_attention_prompt(q, k, v, g=None, *, scale=None, state=None, slots=None, seq_starts=None):
    """S = exp(g) S + k v^T,  o = scale S^T q  over each prompt.  ``q``, ``k`` (B, L, H, K) and ``v`` (B, L, H, V) fp16 or bf16, or each
    without its first dimension and with T tokens with ``seq_starts`` (n + 1 int32, ascending) for packed prompts of any lengths;
    tokens outside them keep undefined outputs.  ``g``: log decays, (H,) or one for each token like q without K, fp16, bf16 or fp32;
    one above zero counts as zero; None: no decay.  K and V multiples of 8, K up to 256; ``scale`` K ** -0.5 by default.
    ``state`` (slots, H, K, V) fp32, dense slots that do not overlap: what each prompt starts from, replaced by what it ends in (a prompt of no tokens leaves it);
    None: zero, nothing kept.  ``slots`` (n,) int32: each prompt's place in the state, all different; negative: from zero, nothing
    kept; beyond the state: NaN outputs.  An infinity in q, k, v or the state counts as a NaN: it reaches the outputs and states that the
    formula has it reach, as one or the other.  Returns o, dense, in the shape and type of v."""
    if state is not None:
        out = _lib.native().linear_attention_prompt(q, k, v, g, scale, state, slots, seq_starts)
        if out is not None:
            return out
    packed = seq_starts is not None
    assert v.dim() == (3 if packed else 4), "v: (B, L, H, V), or (T, H, V) with seq_starts"
    lead = v.shape[:-2]
    fields = _check(q, k, v, g, scale, lead)
    H, V = v.shape[-2:]
    K = q.shape[-1]
    if packed:
        seq_starts = check_starts(seq_starts, v)
        n, L, T = seq_starts.numel() - 1, 0, v.shape[0]
    else:
        (n, L), T = lead, 0
    num_slots = 0
    if state is not None:
        _check_state(state, q, V)
        num_slots = state.shape[0]
    slots = check_slots(slots, n, num_slots, v) if state is not None or slots is not None else None
    q, k, v = (_lib.rows16(t) for t in (q, k, v))
    q, k, v = (t if 0 <= t.stride(-3) < 1 << 24 else t.contiguous() for t in (q, k, v))
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    if n == 0 or L + T == 0 or H == 0 or V == 0:
        return out
    st = lambda t: (0, *t.stride()) if packed else t.stride()  # noqa: E731
    qs, ks, vs = st(q), st(k), st(v)
    g = _lib.f32(g)
    if g is not None and g.dim() > 1 and not 0 <= g.stride(-2) < 1 << 24:
        g = g.contiguous()
    gs = (0, 0, 0) if g is None else (0, 0, g.stride(0)) if g.dim() == 1 else st(g)
    nbytes = prompt_workspace_bytes(n, L, T, packed, H, K, V, fields["dtype"])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=v.device) if nbytes else None
    _lib.call("lq_linear_attention_prompt", v.device, q=_lib.ptr(q), q_stride_b=qs[0], q_stride_l=qs[1], q_stride_h=qs[2], k=_lib.ptr(k),
              k_stride_b=ks[0], k_stride_l=ks[1], k_stride_h=ks[2], v=_lib.ptr(v), v_stride_b=vs[0], v_stride_l=vs[1], v_stride_h=vs[2],
              g=_lib.ptr(g), g_stride_b=gs[0], g_stride_l=gs[1], g_stride_h=gs[2], out=_lib.ptr(out), state=_lib.ptr(state),
              state_stride_s=0 if state is None else state.stride(0), slots=_lib.ptr(slots if state is not None else None),
              seq_starts=_lib.ptr(seq_starts), num_slots=num_slots, nseq=n, seqlen=L, tokens=T, workspace=_lib.ptr(ws), workspace_bytes=nbytes,
              **fields)
    return out


def linear_attention_step(state, q, k, v, g=None, *, scale=None, slots=None):
    """The same for one token of each of up to 65535 sequences: ``q``, ``k`` (B, H, K), ``v`` (B, H, V), ``g`` (H,) or (B, H) -> o (B, H, V),
    ``state`` (slots, H, K, V) fp32 moved on by it.  ``slots`` (B,) int32, all different; negative marks a padding entry (zeros out, no
    state touched), beyond the state: NaN outputs."""
    out = _lib.native().linear_attention_step(q, k, v, g, scale, state, slots)
    if out is not None:
        return out
    assert v.dim() == 3, "v: (B, H, V)"
    fields = _check(q, k, v, g, scale, v.shape[:1])
    n, H, V = v.shape
    _check_state(state, q, V)
    slots = check_slots(slots, n, state.shape[0], v)
    v = _lib.rows16(v)
    q, k = (t if t.stride(2) == 1 else t.contiguous() for t in (q, k))
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    if n and H and V:
        gs = (0, 0) if g is None else (0, g.stride(0)) if g.dim() == 1 else g.stride()
        _lib.call("lq_linear_attention_step", v.device, q=_lib.ptr(q), q_stride_b=q.stride(0), q_stride_h=q.stride(1), k=_lib.ptr(k), k_stride_b=k.stride(0),
                  k_stride_h=k.stride(1), v=_lib.ptr(v), v_stride_b=v.stride(0), v_stride_h=v.stride(1), g=_lib.ptr(g),
                  g_dtype=0 if g is None else _FLOAT[g.dtype], g_stride_b=gs[0], g_stride_h=gs[1],
                  out=_lib.ptr(out), state=_lib.ptr(state), state_stride_s=state.stride(0), slots=_lib.ptr(slots), num_slots=state.shape[0],
                  batch=n, **fields)
    return out
