"""What the operators of a linear attention block refuse, on the host and before any launch (CPU)."""

import ctypes

import pytest
import torch

from linquant_amd import _lib
from linquant_amd.kernels.zoo.linear_attention import linear_attention_prompt, linear_attention_step, prompt_workspace_bytes
from linquant_amd.norm import groupnorm_gated
from linquant_amd.slots import copy_slots
from linquant_amd.w8a8_linear import LowRankAdapters, W8A8Linear

F16, BF16, F32, I8, I32 = torch.float16, torch.bfloat16, torch.float32, torch.int8, torch.int32


def z(*shape, dtype=F16):
    return torch.zeros(*shape, dtype=dtype)


def refuses(f, *args, **kw):
    with pytest.raises((AssertionError, ValueError)):
        f(*args, **kw)


def _linear():
    return W8A8Linear(z(8, 32, dtype=I8), torch.ones(8)), LowRankAdapters(z(2, 4, 32), z(2, 8, 4))


def test_host_tensors_do_not_reach_a_kernel():
    lin, ad = _linear()
    for call in (lambda: linear_attention_prompt(z(1, 5, 2, 8), z(1, 5, 2, 8), z(1, 5, 2, 8)),
                 lambda: linear_attention_step(z(2, 2, 8, 8, dtype=F32), z(2, 2, 8), z(2, 2, 8), z(2, 2, 8)),
                 lambda: groupnorm_gated(z(4, 32), num_groups=2), lambda: copy_slots(z(3, 8), z(2, dtype=I32), z(2, dtype=I32)),
                 lambda: lin.forward_int8(z(3, 32, dtype=I8), 1.0, adapters=ad, ids=z(3, dtype=I32)), lambda: ad._down(z(3, 32), None, z(3, dtype=I32))):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_attention_refusals():
    q, v, s = z(1, 5, 2, 8), z(1, 5, 2, 16), z(3, 2, 8, 16, dtype=F32)
    refuses(linear_attention_prompt, q.float(), q.float(), v.float())
    refuses(linear_attention_prompt, q, q.bfloat16(), v)
    refuses(linear_attention_prompt, q, z(1, 5, 2, 16), v)                       # q and k of two widths
    refuses(linear_attention_prompt, z(1, 5, 3, 8), z(1, 5, 3, 8), v)            # heads
    refuses(linear_attention_prompt, z(1, 4, 2, 8), z(1, 4, 2, 8), v)            # tokens
    refuses(linear_attention_prompt, z(1, 5, 2, 12), z(1, 5, 2, 12), v)
    refuses(linear_attention_prompt, z(1, 5, 2, 264), z(1, 5, 2, 264), v)
    refuses(linear_attention_prompt, q, q, z(1, 5, 2, 12))
    refuses(linear_attention_prompt, q, q, v, z(3, dtype=F32))
    refuses(linear_attention_prompt, q, q, v, z(1, 5, 2, 8, dtype=F32))          # a decay of each channel
    refuses(linear_attention_prompt, q, q, v, z(2, dtype=torch.float64))
    refuses(linear_attention_prompt, q[0], q[0], v[0])                           # packed without seq_starts
    refuses(linear_attention_prompt, q, q, v, seq_starts=z(2, dtype=I32))
    refuses(linear_attention_prompt, q[0], q[0], v[0], seq_starts=z(2, dtype=torch.int64))
    refuses(linear_attention_prompt, q[0], q[0], v[0], seq_starts=z(0, dtype=I32))
    refuses(linear_attention_prompt, q, q, v, state=s.half())
    refuses(linear_attention_prompt, q, q, v, state=s.transpose(2, 3))
    refuses(linear_attention_prompt, q, q, v, state=z(3, 2, 16, 16, dtype=F32))
    refuses(linear_attention_prompt, q, q, v, state=s, slots=z(2, dtype=I32))
    refuses(linear_attention_prompt, q, q, v, state=s, slots=z(1, dtype=torch.int64))
    refuses(linear_attention_prompt, *(t.expand(4, *t.shape[1:]) for t in (q, q, v)), state=s)   # more prompts than slots
    step = lambda *a, **kw: linear_attention_step(s, *a, **kw)  # noqa: E731
    q, v = q[:, 0], v[:, 0]
    refuses(step, q[0], q[0], v[0])
    refuses(step, q, q, z(2, 2, 16))
    refuses(step, q, q, v, z(2, 2, dtype=F32))
    refuses(step, q, q, v, slots=z(2, dtype=I32))
    refuses(linear_attention_step, s[:, :1], q, q, v)
    refuses(linear_attention_step, s[:, :, :, ::2], q, q, v)
    with pytest.raises(_lib.LinQuantHipError):
        prompt_workspace_bytes(0, 5, 0, False, 2, 8, 8, 0)
    with pytest.raises(_lib.LinQuantHipError):
        prompt_workspace_bytes(1, 5, 0, False, 2, 264, 8, 0)


def test_norm_refusals():
    x = z(4, 32)
    refuses(groupnorm_gated, x.float(), num_groups=2)
    refuses(groupnorm_gated, x, num_groups=3)
    refuses(groupnorm_gated, x, num_groups=0)
    refuses(groupnorm_gated, x, z(4, 16), num_groups=2)
    refuses(groupnorm_gated, x, x.bfloat16(), num_groups=2)
    refuses(groupnorm_gated, x, None, z(16), num_groups=2)
    refuses(groupnorm_gated, x, None, None, z(32, dtype=torch.float64), num_groups=2)
    refuses(groupnorm_gated, x, num_groups=2, activation="gelu")
    refuses(groupnorm_gated, z(1, 16385), num_groups=1)


def test_adapter_refusals():
    refuses(LowRankAdapters, z(2, 4, 32), z(3, 8, 4))
    refuses(LowRankAdapters, z(2, 4, 32), z(2, 8, 5))
    refuses(LowRankAdapters, z(2, 4, 32), z(2, 8, 4, dtype=BF16))
    refuses(LowRankAdapters, z(2, 4, 32, dtype=F32), z(2, 8, 4, dtype=F32))
    refuses(LowRankAdapters, z(2, 129, 32), z(2, 8, 129))
    refuses(LowRankAdapters, z(0, 4, 32), z(0, 8, 4))
    refuses(LowRankAdapters, z(2, 4, 32), z(2, 8, 4), torch.ones(3))
    lin, ad = _linear()
    x, codes = z(3, 32), z(3, 32, dtype=I8)
    refuses(lin.forward_int8, codes, 1.0, adapters=ad)                                          # no ids
    refuses(lin.forward_int8, codes, 1.0, adapters=ad, ids=z(2, dtype=I32))
    refuses(lin.forward_int8, codes, 1.0, adapters=ad, ids=z(3, dtype=torch.int64))
    refuses(lin.forward_int8, codes, 1.0, adapters=LowRankAdapters(z(2, 4, 16), z(2, 8, 4)), ids=z(3, dtype=I32))
    refuses(lin.forward_int8, codes, 1.0, adapters=LowRankAdapters(z(2, 4, 32), z(2, 16, 4)), ids=z(3, dtype=I32))
    refuses(lin.forward_int8, codes, 1.0, torch.float64, adapters=ad, ids=z(3, dtype=I32))
    refuses(ad._down, x.bfloat16(), None, z(3, dtype=I32))                                      # another type than the adapters'
    half = LowRankAdapters(z(2, 4, 32), z(2, 8, 4), torch.full((2,), 0.1)).to(BF16)
    assert half.scaling.dtype == F32 and half.down.dtype == BF16 and half.rank == 4 and half.down.shape == (2, 16, 32)


def test_slot_refusals():
    t, i = z(3, 8), z(2, dtype=I32)
    refuses(copy_slots, t, i.long(), i)
    refuses(copy_slots, t, i, z(3, dtype=I32))
    refuses(copy_slots, t, z(8193, dtype=I32), z(8193, dtype=I32))
    refuses(copy_slots, [t, z(4, 8)], i, i)                                                     # another number of slots
    refuses(copy_slots, z(3, 8, 4).transpose(1, 2), i, i)                                       # slots that are not dense
    refuses(copy_slots, z(1, 8).expand(3, 8), i, i)                                             # slots that are one
    refuses(copy_slots, [t, t], i, i)                                                           # a tensor twice
    refuses(copy_slots, [t, t[:, 4:]], i, i)
    refuses(copy_slots, z(()), i, i)


def test_entry_points_refuse():
    lib = _lib.load()
    rc = lambda fn, **kw: getattr(lib, fn)(ctypes.byref(_lib.fill(fn + "_args", **kw)), None)  # noqa: E731
    step = dict(q=16, k=16, v=16, out=16, state=16, dtype=0, batch=1, nheads=1, num_slots=1, kdim=8, vdim=8)
    for bad in (dict(kdim=257), dict(vdim=6), dict(batch=65536), dict(dtype=1), dict(state=8), dict(v=2), dict(num_slots=0), dict(state_stride_s=3)):
        assert rc("lq_linear_attention_step", **{**step, **bad}) == -22, bad
    prompt = dict(q=16, k=16, v=16, out=16, dtype=0, nseq=1, seqlen=5, nheads=1, kdim=8, vdim=8)
    for bad in (dict(kdim=264), dict(kdim=12), dict(vdim=12), dict(nheads=70000), dict(nheads=2, vdim=1 << 23), dict(q=8), dict(q_stride_l=1 << 24), dict(v_stride_h=4), dict(seqlen=0),
                dict(state=16, num_slots=0), dict(g=18), dict(g=16, g_stride_l=-1)):
        assert rc("lq_linear_attention_prompt", **{**prompt, **bad}) == -22, bad
    norm = dict(x=16, out=16, dtype=0, rows=1, dim=8, num_groups=1)
    for bad in (dict(num_groups=3), dict(dim=16385), dict(act=3), dict(dtype=1), dict(weight=16, weight_dtype=2), dict(rows=0)):
        assert rc("lq_groupnorm_gated", **{**norm, **bad}) == -22, bad
    down = dict(x=16, x_dtype=0, down=16, dtype=0, scaling=16, ids=16, h=16, rows=1, inner=16, inner_padded=16, rank=16, count=1)
    for bad in (dict(rank=8), dict(rank=144), dict(inner_padded=8), dict(inner=17), dict(x_dtype=3), dict(x_stride=4), dict(count=0), dict(down=8)):
        assert rc("lq_adapter_down", **{**down, **bad}) == -22, bad
    assert rc("lq_adapter_down", **{**down, "x_dtype": 2}) == -14                                # codes without a scale
    mm = dict(a=16, b=16, a_scale=16, b_scale=16, out=16, rows=1, cols=1, inner=16, adapter_h=16, adapter_ids=16, adapter_up=16, adapter_rank=16, adapter_count=1)
    for bad in (dict(adapter_rank=8), dict(adapter_rank=144), dict(adapter_dtype=1), dict(adapter_count=0), dict(adapter_up=8)):
        assert rc("lq_int8_matmul", **{**mm, **bad}) == -22, bad
    assert rc("lq_int8_matmul", **{**mm, "adapter_ids": None}) == -14
    table = (ctypes.c_int64 * 3)(4096, 64, 64)
    slots = dict(tensors=ctypes.addressof(table), num_tensors=1, num_slots=2, src=16, dst=16, entries=1)
    assert rc("lq_copy_slots", **{**slots, "entries": 8193}) == -22 and rc("lq_copy_slots", **{**slots, "num_slots": 0}) == -22
    table[1] = 32                                                                                # slots that overlap
    assert rc("lq_copy_slots", **slots) == -22
    table[0] = 0
    assert rc("lq_copy_slots", **slots) == -14


def test_adapters_keep_their_factors_when_a_module_changes_its_type():
    f = torch.tensor([0.1, 3.0001])
    ad = LowRankAdapters(z(2, 4, 32), z(2, 8, 4), f)
    for other in (ad.bfloat16(), ad.half(), ad.to("cpu", F16)):
        assert other is ad and torch.equal(ad.scaling, f) and ad.scaling.dtype == F32
    assert ad.down.dtype == F16 and torch.equal(LowRankAdapters(z(2, 4, 32), z(2, 8, 4), f).double().scaling, f)
