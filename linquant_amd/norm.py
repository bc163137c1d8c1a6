"""Gated RMSNorm behind the Mamba-2 SSD (HIP): the `self.norm(y, z)` step at linquant/quantized_mamba2.py:354-358,
i.e. RMSNormGated with norm_before_gate = False and group_size = d_ssm / ngroups, and its fusion with the Hadamard +
INT8 quantizer of the out_proj input (linquant/quantized_mamba2.py:364).  Also the residual stream between two blocks
(``residual_rmsnorm``), which the reference leaves to the surrounding model."""

from __future__ import annotations

import torch
import torch.nn as nn

from linquant_amd import _lib
from linquant_amd.hadamard_utils import _device_matrix, _kernel_scale

_W_CODES = {torch.float16: _lib.LQ_DT_F16, torch.float32: _lib.LQ_DT_F32}


def _rows(t, dim):
    t2 = t.reshape(-1, dim)
    if t2.stride(1) != 1 or t2.stride(0) % 8 != 0:
        t2 = t2.contiguous()
    return t2


def rmsnorm_gated(x, z, weight, eps=1e-5, group_size=None):
    """out = fp16(v * rsqrt(mean_group(v^2) + eps) * weight) with v = x * silu(z) (v = x when z is None), in fp32."""
    assert x.dtype == torch.float16 and weight.dtype in _W_CODES
    dim = x.shape[-1]
    group_size = dim if group_size is None else group_size
    x2 = _rows(x, dim)
    z2 = None if z is None else _rows(z, dim)
    assert z2 is None or (z2.dtype == torch.float16 and z2.shape == x2.shape)
    weight = weight.contiguous()
    out = torch.empty(x2.shape, dtype=torch.float16, device=x.device)
    if x2.shape[0]:
        _lib.call("lq_rmsnorm_gated", x.device, x=_lib.ptr(x2), x_stride=x2.stride(0), z=_lib.ptr(z2),
                  z_stride=0 if z2 is None else z2.stride(0), weight=_lib.ptr(weight),
                  weight_dtype=_W_CODES[weight.dtype], out=_lib.ptr(out), rows=x2.shape[0], dim=dim,
                  group_size=group_size, eps=float(eps))
    return out.reshape(x.shape)


def rmsnorm_gated_qhad(x, z, weight, input_scale, eps=1e-5, group_size=None, return_norm=False):
    """``qhad_transform(rmsnorm_gated(x, z, weight), input_scale)`` in one launch.
    Returns (int8, input_scale) or (int8, input_scale, fp16 normalized rows) with ``return_norm``."""
    assert x.dtype == torch.float16 and weight.dtype in _W_CODES
    dim = x.shape[-1]
    group_size = dim if group_size is None else group_size
    x2 = _rows(x, dim)
    z2 = None if z is None else _rows(z, dim)
    weight = weight.contiguous()
    out = torch.empty(x2.shape, dtype=torch.int8, device=x.device)
    normed = torch.empty(x2.shape, dtype=torch.float16, device=x.device) if return_norm else None
    if x2.shape[0]:
        _lib.call("lq_rmsnorm_gated_qhad", x.device, x=_lib.ptr(x2), x_stride=x2.stride(0), z=_lib.ptr(z2),
                  z_stride=0 if z2 is None else z2.stride(0), weight=_lib.ptr(weight),
                  weight_dtype=_W_CODES[weight.dtype], norm_out=_lib.ptr(normed), rows=x2.shape[0], dim=dim,
                  group_size=group_size, eps=float(eps), had=_lib.ptr(_device_matrix(dim, x.device)),
                  out=_lib.ptr(out), scale=_kernel_scale(dim, input_scale))
    if return_norm:
        return out.reshape(x.shape), input_scale, normed.reshape(x.shape)
    return out.reshape(x.shape), input_scale


_CODES = {torch.float16: _lib.LQ_DT_F16, torch.bfloat16: _lib.LQ_DT_BF16, torch.float32: _lib.LQ_DT_F32}


def _row_view(t, dim):
    """(rows, dim) of ``t`` with unit stride along dim, without a copy where its strides allow it."""
    t2 = t.reshape(-1, dim)
    return t2 if t2.stride(1) == 1 else t2.contiguous()


def residual_rmsnorm(x, weight, residual=None, eps=1e-5, *, gate=None, scale=1.0, post_weight=None, quantize=None,
                     residual_dtype=None):
    """The residual stream between two blocks, in fp32 with one rounding at each output (no gradients)::

        u = x                                                    # the block's output
        u = x * rsqrt(mean(x^2) + eps) * post_weight             # with post_weight: a norm after the block
        r = residual + scale * gate * u
        y = r * rsqrt(mean(r^2) + eps) * weight                  # the next block's input, from the unrounded r

    ``x`` (..., dim) fp16 or bf16; ``residual`` like x, or fp32 (None: zero, then r has ``residual_dtype``, x's by default);
    ``gate`` of x's type: (dim,), the shape of x, or (B, 1, dim) for x (B, L, dim); weights (dim,) fp16, bf16 or fp32; dim up to
    16384.  Returns (y, r), or (codes, scale, r) with ``quantize``: "rows" for INT8 codes on a scale of each row (fp32, the
    shape of x without dim; a row of zeros has 0, one with an infinity or a NaN has NaN), a 0-dim fp32 tensor for codes
    clamp(rint(y / quantize), -128, 127)."""
    if residual_dtype is None and not isinstance(quantize, torch.Tensor) and quantize in (None, "rows"):
        out = _lib.native().residual_rmsnorm(x, weight, residual, eps, gate, scale, post_weight, quantize is not None)
        if out is not None:
            return out
    assert x.dtype in (torch.float16, torch.bfloat16) and x.dim() >= 1
    dim = x.shape[-1]
    assert 1 <= dim <= 16384 and weight.shape == (dim,) and weight.dtype in _CODES
    assert post_weight is None or (post_weight.shape == (dim,) and post_weight.dtype in _CODES)
    assert residual is None or (residual.shape == x.shape and residual.dtype in (x.dtype, torch.float32))
    rdt = residual.dtype if residual is not None else (residual_dtype or x.dtype)
    assert rdt in (x.dtype, torch.float32) and residual_dtype in (None, rdt)
    static = isinstance(quantize, torch.Tensor)
    assert quantize is None or quantize == "rows" if not static else quantize.numel() == 1 and quantize.dtype == torch.float32
    _lib.same_device(x, weight, residual, gate, post_weight, quantize if static else None)
    rows = x.numel() // dim
    _lib.below_2_31(rows)
    x2 = _row_view(x, dim)
    r2 = None if residual is None else _row_view(residual, dim)
    gate_rows, gate_stride = 1, 0
    if gate is not None:
        assert gate.dtype == x.dtype
        if gate.shape == (dim,):
            gate, gate_rows = gate.contiguous(), 1
        elif gate.shape == x.shape:
            gate = _row_view(gate, dim)
            gate_stride = gate.stride(0)
        else:
            assert x.dim() == 3 and gate.shape == (x.shape[0], 1, dim), "gate: (dim,), the shape of x, or (B, 1, dim)"
            gate, gate_rows = _row_view(gate, dim), x.shape[1]
            gate_stride = gate.stride(0)
    if post_weight is not None and post_weight.dtype != weight.dtype:  # one type for both: neither loses bits or range
        weight, post_weight = weight.float(), post_weight.float()
    weight = weight.contiguous()
    post_weight = None if post_weight is None else post_weight.contiguous()
    r_out = torch.empty(x.shape, dtype=rdt, device=x.device)
    out = codes = row_scale = None
    if quantize is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
        row_scale = None if static else torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    if rows:
        _lib.call("lq_residual_rmsnorm", x.device, x=_lib.ptr(x2), x_stride=x2.stride(0), dtype=_CODES[x.dtype],
                  residual=_lib.ptr(r2), residual_stride=0 if r2 is None else r2.stride(0), residual_dtype=_CODES[rdt],
                  gate=_lib.ptr(gate), gate_stride=gate_stride, gate_rows=gate_rows, post_weight=_lib.ptr(post_weight),
                  weight=_lib.ptr(weight), weight_dtype=_CODES[weight.dtype], scale=float(scale), eps=float(eps),
                  residual_out=_lib.ptr(r_out), residual_out_stride=dim, out=_lib.ptr(out), out_stride=dim, codes=_lib.ptr(codes),
                  codes_stride=dim, code_scale=_lib.ptr(quantize) if static else None, row_scale=_lib.ptr(row_scale), rows=rows,
                  dim=dim)
    if quantize is None:
        return out, r_out
    return codes, quantize if static else row_scale, r_out


_ACTIVATIONS = {None: 0, "silu": 1, "swish": 1, "sigmoid": 2}


def groupnorm_gated(x, z=None, weight=None, bias=None, *, num_groups, eps=1e-5, activation="silu"):
    """Group norm of each row, channels last, such as the heads of a linear attention's output, with a gate; in fp32 with one rounding::

        y = (x - mean) * rsqrt(var + eps) * weight + bias        # over each of num_groups groups of adjacent channels of a row
        out = y * act(z)                                         # without z: act(y)

    ``x`` (..., dim) fp16 or bf16, ``z`` like x or None; ``weight``, ``bias`` (dim,) or None, fp16, bf16 or fp32; ``activation`` "silu", "sigmoid"
    or None; dim a multiple of num_groups, up to 16384 channels to a group.  No gradients.  Returns the shape and type of x, dense."""
    act = _ACTIVATIONS.get(activation)
    out = _lib.native().groupnorm_gated(x, z, weight, bias, num_groups, eps, act)
    if out is not None:
        return out
    assert x.dtype in (torch.float16, torch.bfloat16) and x.dim() >= 1
    dim = x.shape[-1]
    assert num_groups >= 1 and dim >= 1 and dim % num_groups == 0 and dim // num_groups <= 16384, f"{dim} channels in {num_groups} groups"
    assert z is None or (z.shape == x.shape and z.dtype == x.dtype), "z: the shape and type of x"
    assert all(t is None or (t.shape == (dim,) and t.dtype in _CODES) for t in (weight, bias)), "weight, bias: (dim,)"
    assert act is not None, f"activation {activation!r}"
    _lib.same_device(x, z, weight, bias)
    rows = x.numel() // dim
    _lib.below_2_31(rows, dim)
    x2 = _row_view(x, dim)
    z2 = None if z is None else _row_view(z, dim)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:  # one type for both: neither loses bits or range
        weight, bias = weight.float(), bias.float()
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    wdt = next((_CODES[t.dtype] for t in (weight, bias) if t is not None), 0)
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if rows:
        _lib.call("lq_groupnorm_gated", x.device, x=_lib.ptr(x2), x_stride=x2.stride(0), z=_lib.ptr(z2), z_stride=0 if z2 is None else z2.stride(0),
                  dtype=_CODES[x.dtype], weight=_lib.ptr(weight), bias=_lib.ptr(bias), weight_dtype=wdt, out=_lib.ptr(out), eps=float(eps), rows=rows,
                  dim=dim, num_groups=num_groups, act=act)
    return out


class RMSNormGated(nn.Module):
    """Module form with the constructor of the norm the mixer receives (hidden_size, eps, group_size;
    norm_before_gate must be False, the only mode the Mamba-2 mixer uses)."""

    def __init__(self, hidden_size, eps=1e-5, group_size=None, norm_before_gate=False, device=None, dtype=None):
        super().__init__()
        assert not norm_before_gate, "only norm_before_gate=False is built"
        self.eps = eps
        self.group_size = hidden_size if group_size is None else group_size
        self.weight = nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype or torch.float16))

    def forward(self, x, z=None):
        return rmsnorm_gated(x, z, self.weight, self.eps, self.group_size)
