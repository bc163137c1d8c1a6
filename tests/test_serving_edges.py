"""The serving operators at the edges of what they take, as far as the host decides it (CPU)."""

import copy
import ctypes
import io

import pytest
import torch

from linquant_amd import _lib
from linquant_amd.kernels.mamba2.conv1d_state import conv1d_prompt, conv1d_step
from linquant_amd.kernels.mamba2.ssm import ssm_prompt, ssm_step
from linquant_amd.norm import residual_rmsnorm
from linquant_amd.w8a8_linear import int8_matmul, quantize_rows
from tests.test_serving_refusals import _mixer

F16, BF16, F32, I8, I32 = torch.float16, torch.bfloat16, torch.float32, torch.int8, torch.int32


# what makes a prepared mixer's copies stale
STALE = {
    "another out_proj": lambda m: setattr(m, "out_proj", copy.deepcopy(m.out_proj)),
    "another scale": lambda m: setattr(m.out_proj, "input_scale", torch.tensor(0.25)),
    "a scale written to": lambda m: m.out_proj.input_scale.fill_(0.25),
    "out_proj loaded": lambda m: m.out_proj.load_state_dict(m.out_proj.state_dict()),
    "out_proj moved": lambda m: m.out_proj.double(),
    "another conv1d": lambda m: setattr(m, "conv1d", copy.deepcopy(m.conv1d)),
    "conv1d moved": lambda m: m.conv1d.half(),
    "taps written to": lambda m: m.conv1d.weight.detach().add_(1),
    "another dt_bias": lambda m: setattr(m, "dt_bias", torch.ones(2)),
    "D written to": lambda m: m.D.zero_(),
}


@pytest.mark.parametrize("how", list(STALE))
def test_serving_notices_what_changed_after_it_was_prepared(how):
    m = _mixer()
    st = m.allocate_state(2)
    call = lambda: m.step((torch.zeros(1, 64, dtype=I8), 1.0), st)  # noqa: E731
    with pytest.raises(ValueError, match="GPU"):     # prepared: host tensors get as far as the first kernel
        call()
    STALE[how](m)
    with pytest.raises(RuntimeError, match="prepare_serving"):
        call()
    m.allocate_state(1)                              # prepares where it has to
    with pytest.raises(ValueError, match="GPU"):
        call()


def test_a_prepared_mixer_can_be_copied_and_saved():
    m = _mixer()
    st = m.allocate_state(2)
    m.D.zero_()
    m.prepare_serving()
    buf = io.BytesIO()
    torch.save(m, buf)
    buf.seek(0)
    for other in (copy.deepcopy(m), torch.load(buf, weights_only=False)):
        with pytest.raises(ValueError, match="GPU"):
            other.step((torch.zeros(1, 64, dtype=I8), 1.0), st)
        other.out_proj.input_scale.fill_(0.5)
        with pytest.raises(RuntimeError, match="prepare_serving"):
            other.step((torch.zeros(1, 64, dtype=I8), 1.0), st)
    with pytest.raises(ValueError, match="GPU"):
        m.step((torch.zeros(1, 64, dtype=I8), 1.0), st)


# ------------------------------------------------------------------------------------------------------- sizes past 32 bits
def _meta(*shape, dtype=F16):
    return torch.empty(*shape, dtype=dtype, device="meta")


BIG = (1 << 32) + 5   # 5 in 32 bits
PAST = {
    "quantize_rows": lambda: quantize_rows(_meta(BIG, 8)),
    "int8_matmul rows": lambda: int8_matmul(_meta(BIG, 16, dtype=I8), _meta(8, 16, dtype=I8), 1.0, 1.0),
    "int8_matmul columns": lambda: int8_matmul(_meta(8, 16, dtype=I8), _meta(BIG, 16, dtype=I8), 1.0, 1.0),
    "residual_rmsnorm": lambda: residual_rmsnorm(_meta(5, BIG // 5 * 5, 1), _meta(1)),
    "conv1d_prompt": lambda: conv1d_prompt(_meta(BIG, 8), _meta(8, 4), seq_starts=_meta(3, dtype=I32)),
    "conv1d_prompt of a batch": lambda: conv1d_prompt(_meta(1, BIG, 8), _meta(8, 4)),
    "conv1d_step": lambda: conv1d_step(_meta(BIG, 8), _meta(8, 3, 8), _meta(8, 4), slots=_meta(BIG, dtype=I32)),
    "ssm_prompt": lambda: ssm_prompt(_meta(BIG, 1, 8), _meta(BIG, 1), _meta(1), _meta(BIG, 1, 8), _meta(BIG, 1, 8), seq_starts=_meta(3, dtype=I32)),
    "ssm_step": lambda: ssm_step(_meta(8, 1, 8, 8, dtype=F32), _meta(BIG, 1, 8), _meta(BIG, 1), _meta(1), _meta(BIG, 1, 8), _meta(BIG, 1, 8),
                                 slots=_meta(BIG, dtype=I32)),
}


@pytest.mark.parametrize("what", list(PAST))
def test_sizes_past_32_bits_are_refused(what, monkeypatch):
    """Not cut off to what their lowest 32 bits say."""
    monkeypatch.setattr(_lib, "launch", lambda fn, device, st: pytest.fail(f"{fn} with {[(n, getattr(st, n)) for n, _ in st._fields_]}"))
    with pytest.raises(ValueError, match=r"2\*\*31"):
        PAST[what]()


@pytest.mark.parametrize("fn,sizes", [("lq_conv1d_prompt", dict(seqlen=(1 << 31) - 1)), ("lq_conv1d_prompt", dict(dim=(1 << 31) - 8)), ("lq_conv1d_step", dict(dim=(1 << 31) - 8))])
def test_sizes_near_the_last_of_32_bits_are_refused(fn, sizes):
    """Rounding them up to whole units must not wrap: a grid of that would be no refusal but a launch that fails (host memory here)."""
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    args = {n: at for n, t in _lib.STRUCTS[fn + "_args"]._fields_ if t is ctypes.c_void_p and n not in ("seq_starts", "slots", "bias")}
    args.update(nseq=1, seqlen=4, x_stride_l=16) if fn.endswith("prompt") else args.update(batch=1, x_stride=16)
    args.update({**dict(dim=16, width=4, num_slots=1), **sizes})
    assert getattr(_lib.load(), fn)(ctypes.byref(_lib.fill(fn + "_args", **args)), None) == -22


# ------------------------------------------------------------------------------------------------------- one row of a wide tensor
@pytest.mark.parametrize("shape,strides", [((1, 32), (77, 1)), ((1, 32), (1 << 24, 1)), ((1, 1, 32), (5, 3, 1)), ((1, 4, 32), (7, 40, 1)), ((4, 1, 32), (40, 9, 1)),
                                           ((1, 4, 32), (7, 33, 1)), ((1, 1, 4, 32), (3, 3, 33, 1)), ((3, 32), (33, 1)), ((3, 32), (48, 1))])
@pytest.mark.parametrize("dtype", [F16, I8])
def test_rows_of_whole_pieces(shape, strides, dtype):
    """Whatever the strides of dimensions of length one say; a copy only where there are several rows off the grid."""
    n = 16 // torch.empty(0, dtype=dtype).element_size()
    base = torch.arange(4096).to(dtype)
    assert base.data_ptr() % 16 == 0
    t = base.as_strided(shape, strides)
    r = _lib.rows16(t)
    assert torch.equal(r, t) and r.stride(-1) == 1 and r.data_ptr() % 16 == 0 and all(s % n == 0 and s < 1 << 23 for s in r.stride()[:-1])
    off = any(s % n for m, s in zip(shape[:-1], strides) if m > 1)
    assert (r.data_ptr() == t.data_ptr()) == (not off)


# ------------------------------------------------------------------------------------------------------- how prompts are cut
def test_cuts_that_the_gpu_tests_mean():
    """A change of the plan must not leave the forms that they are there for without a test; the prefill of the benchmark takes 3 segments of two pieces."""
    from tests.test_serving_edges_gpu import CUT, _plan

    for dtype in (F16, BF16):
        for dims, lens, packed, cut in CUT:
            assert _plan(lens, packed, *dims, dtype) == cut
    assert {(packed, pieces) for _, _, packed, (chunks, pieces) in CUT if chunks > 1} == {(False, 1), (False, 2), (True, 1), (True, 2)}
    assert _plan([8192] * 4, False, 80, 64, 1, 128, F16) == [44, 2]
    assert _plan([384], False, 80, 64, 1, 128, F16) == [6, 0]          # one segment, not cut
    out = (ctypes.c_int64 * 3)()
    bad = _lib.fill("lq_ssm_prompt_args", nseq=1, seqlen=64, nheads=3, headdim=64, ngroups=2, dstate=16)
    assert _lib.load().lq_ssm_prompt_plan(ctypes.byref(bad), ctypes.byref(out)) == -22 and _lib.load().lq_ssm_prompt_plan(None, ctypes.byref(out)) == -14
