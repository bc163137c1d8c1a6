"""What the serving operators refuse, on the host and before any launch (CPU)."""

import ctypes

import pytest
import torch

from linquant_amd import _lib
from linquant_amd.kernels.mamba2.conv1d_state import conv1d_prompt, conv1d_step
from linquant_amd.kernels.mamba2.ssm import ssm_prompt, ssm_step
from linquant_amd.norm import residual_rmsnorm
from linquant_amd.w8a8_linear import W8A8Linear, int8_matmul, quantize_rows

F16, BF16, F32, I8, I32 = torch.float16, torch.bfloat16, torch.float32, torch.int8, torch.int32


def z(*shape, dtype=F16):
    return torch.zeros(*shape, dtype=dtype)


def refuses(f, *args, **kw):
    with pytest.raises((AssertionError, ValueError)):
        f(*args, **kw)


def test_host_tensors_do_not_reach_a_kernel():
    for call in (lambda: quantize_rows(z(4, 32)), lambda: int8_matmul(z(4, 32, dtype=I8), z(8, 32, dtype=I8), 1.0, 1.0),
                 lambda: residual_rmsnorm(z(4, 32), z(32)), lambda: conv1d_step(z(2, 8), z(2, 3, 8), z(8, 4)),
                 lambda: conv1d_prompt(z(2, 5, 8), z(8, 4)),
                 lambda: ssm_step(z(2, 4, 8, 8, dtype=F32), z(2, 4, 8), z(2, 4), z(4), z(2, 1, 8), z(2, 1, 8)),
                 lambda: ssm_prompt(z(2, 5, 4, 8), z(2, 5, 4), z(4), z(2, 5, 1, 8), z(2, 5, 1, 8))):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_linear_refusals():
    a, b = z(4, 32, dtype=I8), z(8, 32, dtype=I8)
    refuses(int8_matmul, z(4, 32), b, 1.0, 1.0)                               # not codes
    refuses(int8_matmul, a, z(8, 48, dtype=I8), 1.0, 1.0)                     # other contraction length
    refuses(int8_matmul, a, b, torch.ones(3), 1.0)                            # neither one scale nor one a row
    refuses(int8_matmul, a, b, 1.0, torch.ones(4))
    refuses(int8_matmul, a, b, 1.0, 1.0, bias=z(4))
    refuses(int8_matmul, a, b, 1.0, 1.0, out_dtype=torch.float64)
    refuses(int8_matmul, a, b, 1.0, 1.0, out=z(4, 8, dtype=F32))              # another type than out_dtype
    refuses(int8_matmul, a, b, 1.0, 1.0, out=z(8, 4).t())                     # columns not adjacent
    refuses(int8_matmul, z(1, 131072, dtype=I8), z(1, 131072, dtype=I8), 1.0, 1.0)
    refuses(quantize_rows, z(4, 16385))
    refuses(quantize_rows, z(4, 0))
    refuses(quantize_rows, z(4, 8, dtype=torch.float64))
    refuses(W8A8Linear, z(8, 32), torch.ones(8))
    refuses(W8A8Linear, b, torch.ones(4))
    lin = W8A8Linear(b, torch.ones(8), input_scale=0.1)
    refuses(lin, z(2, 32, dtype=BF16))                                        # a static scale takes fp16
    refuses(lin, z(2, 40))


def test_norm_refusals():
    x, w = z(2, 3, 32), z(32)
    refuses(residual_rmsnorm, z(2, 32, dtype=F32), w)
    refuses(residual_rmsnorm, x, z(16))
    refuses(residual_rmsnorm, x, w, z(2, 3, 32, dtype=BF16))                  # neither x's type nor fp32
    refuses(residual_rmsnorm, x, w, z(3, 32))
    refuses(residual_rmsnorm, x, w, gate=z(32, dtype=BF16))
    refuses(residual_rmsnorm, x, w, gate=z(3, 32))
    refuses(residual_rmsnorm, x, w, post_weight=z(16))
    refuses(residual_rmsnorm, x, w, quantize="tensor")
    refuses(residual_rmsnorm, x, w, quantize=torch.ones(2))
    refuses(residual_rmsnorm, x, w, x, residual_dtype=F32)                    # the residual says
    refuses(residual_rmsnorm, z(2, 16385), z(16385))


def test_conv_refusals():
    x, st, w = z(2, 16), z(4, 3, 16), z(16, 4)
    refuses(conv1d_step, z(2, 12), z(4, 3, 12), z(12, 4))                     # channels in whole 16-byte pieces
    refuses(conv1d_step, x, st, z(16, 5))
    refuses(conv1d_step, x, z(4, 2, 16), w)                                   # a state of another width
    refuses(conv1d_step, x, z(4, 3, 16, dtype=BF16), w)
    refuses(conv1d_step, x, z(1, 3, 16), w)                                   # fewer slots than sequences
    refuses(conv1d_step, x, st, w, slots=torch.zeros(2, dtype=torch.int64))
    refuses(conv1d_step, x, st, w, slots=torch.zeros(3, dtype=I32))
    refuses(conv1d_step, x, st, w, activation="relu")
    refuses(conv1d_prompt, x, w)                                              # two dimensions without starts
    refuses(conv1d_prompt, z(1, 2, 16), w, seq_starts=torch.zeros(2, dtype=I32))
    refuses(conv1d_prompt, x, w, seq_starts=torch.zeros(2, dtype=torch.int64))


def test_ssm_refusals():
    ok = dict(x=z(2, 4, 8), dt=z(2, 4), A=z(4, dtype=F32), B=z(2, 2, 16), C=z(2, 2, 16))
    st = z(3, 4, 8, 16, dtype=F32)
    for bad in (dict(x=z(2, 4, 12)), dict(x=z(2, 4, 8, dtype=F32)), dict(B=z(2, 3, 16)), dict(B=z(2, 2, 16, dtype=BF16)), dict(dt=z(2, 3)),
                dict(A=z(3, dtype=F32)), dict(B=z(2, 2, 12), C=z(2, 2, 12)), dict(B=z(2, 2, 264), C=z(2, 2, 264)), dict(D=z(5)),
                dict(dt_bias=z(2)), dict(slots=torch.zeros(2, dtype=torch.int64))):
        refuses(ssm_step, st, **{**ok, **bad})
    refuses(ssm_step, st.half(), **ok)                                        # the state is fp32
    refuses(ssm_step, z(1, 4, 8, 16, dtype=F32), **ok)
    refuses(ssm_step, z(3, 4, 16, 8, dtype=F32).transpose(2, 3), **ok)
    refuses(ssm_prompt, **ok)                                                 # two token dimensions without starts
    refuses(ssm_prompt, **ok, state=st, seq_starts=torch.zeros(2, dtype=torch.int64))
    refuses(ssm_prompt, **ok, state=z(0, 4, 8, 16, dtype=F32), seq_starts=torch.zeros(2, dtype=I32))


@pytest.mark.parametrize("fn,good,bad", [
    ("lq_quantize_rows", dict(x=1, codes=1, scale=1, rows=2, cols=32, x_stride=32, codes_stride=32),
     [dict(cols=0), dict(cols=16385), dict(rows=0), dict(dtype=2), dict(rows=1 << 24, cols=7), dict(rows=1 << 26)]),
    ("lq_int8_matmul", dict(a=1, b=1, a_scale=1, b_scale=1, out=1, rows=2, cols=8, inner=32, a_stride=32, b_stride=32, out_stride=8),
     [dict(inner=24), dict(inner=131072), dict(a_stride=40), dict(b_stride=8), dict(out_dtype=2), dict(rows=0), dict(cols=-1), dict(cols=(1 << 27) + 1),
      dict(rows=(1 << 31) - 1, cols=(1 << 31) - 1)]),
    ("lq_residual_rmsnorm", dict(x=1, weight=1, out=1, rows=2, dim=32),
     [dict(codes=1, row_scale=1), dict(dtype=1), dict(weight_dtype=2), dict(dim=16385), dict(gate=1, gate_rows=0),
      dict(residual=1, residual_dtype=3)]),
    ("lq_conv1d_prompt", dict(x=1, weight=1, out=1, nseq=1, seqlen=4, dim=16, width=4, x_stride_l=16),
     [dict(dim=12), dict(width=5), dict(width=1), dict(x_stride_l=12), dict(seqlen=0), dict(nseq=0), dict(state=1, num_slots=0), dict(dtype=1),
      dict(seq_starts=1, tokens=0), dict(seqlen=1 << 28), dict(nseq=1 << 20, seqlen=1 << 20)]),
    ("lq_conv1d_step", dict(x=1, weight=1, out=1, state=1, num_slots=1, batch=1, dim=16, width=4, x_stride=16),
     [dict(dim=12), dict(width=5), dict(x_stride=12), dict(batch=0), dict(num_slots=0), dict(state_stride_w=4), dict(batch=1 << 26)]),
    ("lq_ssm_prompt", dict(x=1, dt=1, A=1, B=1, C=1, out=1, nseq=1, seqlen=4, nheads=2, headdim=8, ngroups=1, dstate=16, workspace=1,
                           workspace_bytes=1 << 40),
     [dict(headdim=12), dict(dstate=264), dict(dstate=12), dict(ngroups=4), dict(seqlen=0), dict(B_stride_l=4), dict(x_stride_l=1 << 24), dict(workspace_bytes=0),
      dict(state=1, num_slots=0), dict(dtype=1), dict(dt_dtype=2), dict(seqlen=1 << 30), dict(nseq=1 << 26, seqlen=1)]),
    ("lq_ssm_step", dict(x=1, dt=1, A=1, B=1, C=1, out=1, state=1, num_slots=1, batch=1, nheads=2, headdim=8, ngroups=1, dstate=16),
     [dict(headdim=12), dict(dstate=264), dict(ngroups=4), dict(batch=0), dict(batch=65536), dict(state_stride_s=2), dict(num_slots=0)]),
])
def test_entry_points_refuse_before_a_launch(fn, good, bad):
    """Every pointer is host memory: a call that passed the checks would launch, so only refusals are made."""
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    pointers = {n for n, t in _lib.STRUCTS[fn + "_args"]._fields_ if t is ctypes.c_void_p}

    def rc(**kw):
        return getattr(_lib.load(), fn)(ctypes.byref(_lib.fill(fn + "_args", **{k: at if k in pointers and v else v for k, v in kw.items()})), None)

    for kw in bad:
        assert rc(**{**good, **kw}) == -22, kw
    for name in (n for n in good if n in pointers and n != "workspace"):
        assert rc(**{**good, name: None}) == -14, name


def _mixer(**kw):
    from linquant_amd.norm import RMSNormGated
    from linquant_amd.quantized_mamba2 import Int8InputLinear, QuantizedMamba2

    lin = lambda n, k: Int8InputLinear(torch.zeros(n, k), 1.0)  # noqa: E731
    m = QuantizedMamba2(d_model=64, d_ssm=128, nheads=2, headdim=64, d_state=16, ngroups=1, d_conv=4, chunk_size=64,
                        in_proj=lin(2 * 128 + 32 + 2, 64), out_proj=lin(64, 128), conv1d=torch.nn.Conv1d(160, 160, 4, groups=160),
                        norm=RMSNormGated(128), A_log=torch.full((2,), 50, dtype=I8), D=torch.full((2,), 100, dtype=I8), dt_bias=torch.zeros(2), **kw)
    m.register_buffer("A_log_scale", torch.tensor(0.02))
    m.register_buffer("D_scale", torch.tensor(0.01))
    return m


def test_mixer_serving_refusals():
    m = _mixer()
    x = z(1, 64)
    with pytest.raises(RuntimeError, match="prepare_serving"):
        m.step(x, None)
    st = m.allocate_state(3)
    assert st.conv.shape == (3, 3, 160) and st.conv.dtype == F16 and st.ssm.shape == (3, 2, 64, 16) and st.ssm.dtype == F32
    assert torch.allclose(m._serving["A"], torch.full((2,), -2.718281828)) and torch.allclose(m._serving["D"], torch.ones(2))
    for undo in (lambda: m.to("cpu"), lambda: m.load_state_dict(m.state_dict())):       # moved or loaded: what was laid out is gone
        m.prepare_serving()
        undo()
        with pytest.raises(RuntimeError, match="prepare_serving"):
            m.prefill(x[None], st)
    with pytest.raises(NotImplementedError, match="prefill-only"):
        m(x[None], past_key_values=object())
    m.prepare_serving()
    refuses(m.step, (z(1, 1, 64, dtype=I8), 1.0), st)                                   # codes of other dimensions
    refuses(m.prefill, (z(4, 64, dtype=I8), 1.0), st)
    refuses(m.prefill, (z(1, 4, 64, dtype=I8), 1.0), st, None, z(2, dtype=I32))


def test_int8_input_linear_takes_a_scale_for_each_row():
    from linquant_amd.quantized_mamba2 import Int8InputLinear

    w = torch.arange(12.0).view(3, 4) / 8
    lin = Int8InputLinear(w, 1.0)
    codes, scale = torch.arange(-8, 8).to(I8).view(4, 4), torch.tensor([0.5, 1.0, 2.0, 0.25])   # as many rows as columns
    want = torch.cat([lin.forward_int8(codes[i:i + 1], scale[i]) for i in range(4)])
    assert torch.equal(lin.forward_int8(codes, scale), want)
    assert torch.equal(lin.forward_int8(codes.view(2, 2, 4), scale.view(2, 2)), want.view(2, 2, 3))
