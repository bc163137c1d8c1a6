"""Further refusals of a linear attention block's operators: widths behind the padding, adapters' ids without adapters, states whose slots overlap (CPU)."""

import ctypes

import pytest
import torch

from linquant_amd import _lib
from linquant_amd.kernels.zoo.linear_attention import linear_attention_prompt, linear_attention_step, prompt_workspace_bytes
from linquant_amd.w8a8_linear import LowRankAdapters, W8A8Linear

F16, F32, I8, I32 = torch.float16, torch.float32, torch.int8, torch.int32


def z(*shape, dtype=F16):
    return torch.zeros(*shape, dtype=dtype)


class _Native:
    """In the place of the native calls: takes every call with adapters, none of the others."""

    def __init__(self):
        self.taken = 0

    def adapted(self, *args):
        self.taken += 1
        return "taken"

    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture
def native(monkeypatch):
    n = _Native()
    monkeypatch.setattr(_lib, "native", lambda: n)
    return n


def test_native_calls_with_adapters_keep_the_widths_apart(native):
    """250 and 256 features lie in rows of the same length, and are not the same."""
    ids = z(3, dtype=I32)
    narrow, wide = (W8A8Linear(z(8, k, dtype=I8), torch.ones(8)) for k in (250, 256))
    a250, a256 = (LowRankAdapters(z(2, 4, k), z(2, 8, 4)) for k in (250, 256))
    for lin, ad, k in ((narrow, a250, 256), (narrow, a256, 250), (narrow, a256, 256), (wide, a250, 256), (wide, a250, 250), (wide, a256, 250)):
        with pytest.raises(AssertionError):
            lin(z(3, k), adapters=ad, ids=ids)
        with pytest.raises(AssertionError):
            lin.forward_int8(z(3, k, dtype=I8), torch.ones(3), adapters=ad, ids=ids)
    with pytest.raises(AssertionError, match="another projection"):
        wide(z(3, 256), adapters=LowRankAdapters(z(2, 4, 256), z(2, 16, 4)), ids=ids)
    assert native.taken == 0
    assert wide(z(3, 256), adapters=a256, ids=ids) == "taken" and wide.forward_int8(z(3, 256, dtype=I8), torch.ones(3), adapters=a256, ids=ids) == "taken"


def test_ids_without_adapters_are_refused():
    lin, ids = W8A8Linear(z(8, 32, dtype=I8), torch.ones(8)), z(3, dtype=I32)
    static = W8A8Linear(z(8, 32, dtype=I8), torch.ones(8), input_scale=0.5)
    for call in (lambda: lin(z(3, 32), ids=ids), lambda: static(z(3, 32), ids=ids), lambda: lin.forward_int8(z(3, 32, dtype=I8), 1.0, ids=ids)):
        with pytest.raises(AssertionError, match="ids without adapters"):
            call()


def test_states_whose_slots_overlap_are_refused():
    """Two sequences would write to one place."""
    one = z(1, 2, 8, 16, dtype=F32)
    near = torch.as_strided(z(4 * 256, dtype=F32), (3, 2, 8, 16), (128, 128, 16, 1))
    for s in (one.expand(3, 2, 8, 16), near):
        with pytest.raises(AssertionError, match="overlap"):
            linear_attention_step(s, z(2, 2, 8), z(2, 2, 8), z(2, 2, 16))
        with pytest.raises(AssertionError, match="overlap"):
            linear_attention_prompt(z(1, 5, 2, 8), z(1, 5, 2, 8), z(1, 5, 2, 16), state=s)
    lib = _lib.load()
    rc = lambda fn, **kw: getattr(lib, fn)(ctypes.byref(_lib.fill(fn + "_args", **kw)), None)  # noqa: E731
    both = dict(q=16, k=16, v=16, out=16, state=16, dtype=0, nheads=2, num_slots=3, kdim=8, vdim=16, state_stride_s=252)
    assert rc("lq_linear_attention_step", batch=1, **both) == -22 and rc("lq_linear_attention_prompt", nseq=1, seqlen=5, **both) == -22


@pytest.mark.parametrize("nseq,tokens", [(256, 256), (1024, 4096), (4096, 16384), (10, 6949), (61, 2060), (1, 500), (1, 40000), (65535, 65535)])
@pytest.mark.parametrize("H,K,V", [(32, 128, 128), (1, 64, 64), (8, 256, 72)])
def test_workspace_of_packed_prompts_goes_by_their_tokens(nseq, tokens, H, K, V):
    """However many prompts there are: a place for each 64 tokens, and one for each prompt that can be longer."""
    most = (tokens - 1) // 64 + min(nseq, tokens // 65)
    assert prompt_workspace_bytes(nseq, 0, tokens, True, H, K, V, 0) <= most * H * (K * V + 1) * 4 + 512
