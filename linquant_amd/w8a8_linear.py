"""INT8 projections (HIP): activations with one scale for each row (quantized here) or for the tensor, weights with one scale for
each output channel, the product on the INT8 matrix cores.  ``W8A8Linear`` has the ``input_scale`` / ``forward_int8`` surface of
the reference's W4A8B16O16Linear (linquant/w4a8_linear.py), so it takes the place of the fp16 stand-in of quantized_mamba2.py."""

from __future__ import annotations

import torch
import torch.nn as nn

from linquant_amd import _lib
from linquant_amd.w4a8_linear import _fused_fp16_to_int8

_CODES = {torch.float16: _lib.LQ_DT_F16, torch.bfloat16: _lib.LQ_DT_BF16, torch.float32: _lib.LQ_DT_F32}
_K = 16  # the product's contraction length is a multiple of this


def _padded(n):
    return -(-n // _K) * _K


def _quantize(x):
    """Codes in rows of whole 16-byte pieces, (rows, padded), the surplus undefined; scales (rows,)."""
    out = _lib.native().quantize_rows(x, _K)
    if out is not None:
        return out
    assert x.dtype in _CODES and x.dim() >= 1 and 1 <= x.shape[-1] <= 16384
    K = x.shape[-1]
    x2 = x.reshape(-1, K)
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    M = x2.shape[0]
    _lib.below_2_31(M)
    codes = torch.empty(M, _padded(K), dtype=torch.int8, device=x.device)
    scale = torch.empty(M, dtype=torch.float32, device=x.device)
    if M:
        _lib.call("lq_quantize_rows", x.device, x=_lib.ptr(x2), x_stride=x2.stride(0), dtype=_CODES[x.dtype], codes=_lib.ptr(codes),
                  codes_stride=codes.stride(0), scale=_lib.ptr(scale), rows=M, cols=K)
    return codes, scale


def quantize_rows(x):
    """``x`` (..., K) fp16, bf16 or fp32, K up to 16384 -> (codes int8 (..., K), scale fp32 (...)): scale = max |x| / 127 of each row,
    codes = rint(x / scale).  A row of zeros has scale 0 and codes 0; one with an infinity or a NaN has scale NaN and codes 0."""
    codes, scale = _quantize(x)
    K = x.shape[-1]
    codes = codes if codes.shape[1] == K else codes[:, :K]
    if x.dim() == 1:
        return codes[0], scale[0]
    return (codes, scale) if x.dim() == 2 else (codes.unflatten(0, x.shape[:-1]), scale.view(x.shape[:-1]))


def _scale(s, n, device, what):
    if not isinstance(s, torch.Tensor):
        return torch.full((1,), float(s), dtype=torch.float32, device=device), 0
    assert s.numel() in (1, n), f"{what}: one scale or {n}, got {tuple(s.shape)}"
    return _lib.f32(s).reshape(-1).contiguous(), int(s.numel() != 1)


def _matmul(a, b, a_scale, b_scale, bias, out):
    """a (M, K), b (N, K) in rows of whole 16-byte pieces; out (M, N) with unit column stride."""
    (M, K), N = a.shape, b.shape[0]
    a, b = (t if t.stride(0) < 1 << 23 else t.contiguous() for t in (a, b))
    a_scale, per_row = _scale(a_scale, M, a.device, "a_scale")
    b_scale, per_col = _scale(b_scale, N, a.device, "b_scale")
    bias = None if bias is None else bias.contiguous()
    _lib.same_device(a, b, a_scale, b_scale, bias, out)
    if M and N:
        _lib.call("lq_int8_matmul", a.device, a=_lib.ptr(a), a_stride=a.stride(0), b=_lib.ptr(b), b_stride=b.stride(0),
                  a_scale=_lib.ptr(a_scale), b_scale=_lib.ptr(b_scale), a_scale_rows=per_row, b_scale_cols=per_col, bias=_lib.ptr(bias),
                  bias_dtype=0 if bias is None else _CODES[bias.dtype], out=_lib.ptr(out), out_stride=out.stride(0),
                  out_dtype=_CODES[out.dtype], rows=M, cols=N, inner=K)
    return out


def int8_matmul(a, b, a_scale, b_scale, bias=None, out_dtype=torch.float16, out=None):
    """out[..., n] = (sum_k a[..., k] b[n, k]) * a_scale[...] * b_scale[n] + bias[n].  ``a`` int8 (..., K), ``b`` int8 (N, K), K up to
    131056, the sum exact; ``a_scale`` a number, one entry or one for each row of a, ``b_scale`` a number, one entry or (N,);
    ``bias`` (N,) or None and ``out_dtype`` fp16, bf16 or fp32.  ``out``: a (M, N) view of that type with unit column stride to
    write into, for ``a`` of two dimensions.  Rows of K bytes that are not whole 16-byte pieces are copied first."""
    if out is None:
        res = _lib.native().int8_matmul(a, b, a_scale, b_scale, bias, out_dtype)
        if res is not None:
            return res
    assert a.dtype == torch.int8 and b.dtype == torch.int8 and b.dim() == 2 and a.dim() >= 1
    K, N = a.shape[-1], b.shape[0]
    assert b.shape[1] == K and 1 <= K <= 131056, f"contraction lengths {K} and {b.shape[1]}"
    _lib.below_2_31(a.numel() // K, N)
    assert out_dtype in _CODES and (bias is None or (bias.dtype in _CODES and bias.shape == (N,)))
    a2 = a.reshape(-1, K)
    if out is None:
        res = torch.empty(a2.shape[0], N, dtype=out_dtype, device=a.device)
    else:
        assert a.dim() == 2 and out.dtype == out_dtype and out.shape == (a.shape[0], N) and out.stride(1) == 1
        res = out
    if K % _K:
        a2, b = (nn.functional.pad(t, (0, _padded(K) - K)) for t in (a2, b))
    _matmul(_lib.rows16(a2), _lib.rows16(b), a_scale, b_scale, bias, res)
    return res if out is not None or a.dim() == 2 else res.view(*a.shape[:-1], N)


class W8A8Linear(nn.Module):
    """INT8 weight (N, K) with a scale for each output channel.  ``input_scale`` None: activations are quantized with a scale for
    each row; a 0-dim tensor: with that scale (clamp(rint(x / s), -128, 127)).  The output has the activations' 16-bit type."""

    def __init__(self, weight_i8, weight_scale, input_scale=None, bias=None):
        super().__init__()
        assert weight_i8.dtype == torch.int8 and weight_i8.dim() == 2 and weight_scale.shape == (weight_i8.shape[0],)
        self.in_features, self.out_features = weight_i8.shape[1], weight_i8.shape[0]
        # laid out once: rows of whole 16-byte pieces, the surplus zero (so the activations' surplus does not matter)
        self.register_buffer("weight", nn.functional.pad(weight_i8, (0, _padded(self.in_features) - self.in_features)).contiguous())
        self.register_buffer("weight_scale", weight_scale.detach().float().contiguous())
        self.register_buffer("input_scale", None if input_scale is None else torch.as_tensor(input_scale, dtype=torch.float32).reshape(()).clone())
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    @classmethod
    def from_fp16(cls, linear: nn.Linear, input_scale=None):
        """Weights quantized with a scale for each output channel: max |w| / 127, rint."""
        w = linear.weight.detach().float()
        s = w.abs().amax(1) / 127.0
        codes = torch.round(w / torch.where(s > 0, s, 1.0)[:, None]).to(torch.int8)
        return cls(codes, s, input_scale, linear.bias)

    def forward_int8(self, x_i8, scale, out_dtype=torch.float16):
        """Codes (..., in_features) on ``scale`` (a number, one entry, or one for each row)."""
        assert x_i8.dtype == torch.int8 and x_i8.shape[-1] == self.in_features
        a = x_i8.reshape(-1, self.in_features)
        if self.in_features % _K:
            a = nn.functional.pad(a, (0, _padded(self.in_features) - self.in_features))
        return int8_matmul(a, self.weight, scale, self.weight_scale, self.bias, out_dtype).view(*x_i8.shape[:-1], self.out_features)

    def forward(self, x):
        assert x.shape[-1] == self.in_features and x.dtype in (torch.float16, torch.bfloat16)
        if self.input_scale is not None and x.dtype == torch.float16 and self.in_features % 8 == 0:
            q = _fused_fp16_to_int8(_lib.rows16(x.reshape(-1, self.in_features)), self.input_scale, clamp_min=-128.0, reciprocal=False)
            return self.forward_int8(q.view(x.shape), self.input_scale, x.dtype)
        assert self.input_scale is None, "a static input scale takes fp16 activations and in_features a multiple of 8"
        q, s = _quantize(x)
        return int8_matmul(q, self.weight, s, self.weight_scale, self.bias, x.dtype).view(*x.shape[:-1], self.out_features)
