"""A linear attention block's operators at the limits of what they take: sizes and magnitudes where a variant, a unit or a workspace changes."""

import pytest
import torch

from linquant_amd.w8a8_linear import LowRankAdapters, W8A8Linear

pytestmark = pytest.mark.gpu

F16, BF16, F32, I8, I32 = torch.float16, torch.bfloat16, torch.float32, torch.int8, torch.int32


def test_widths_behind_the_padding_are_told_apart(cuda):
    """250 features lie in rows of 256 bytes, as 256 do."""
    lin = {k: W8A8Linear(torch.ones(8, k, dtype=I8), torch.ones(8)).to(cuda) for k in (250, 256)}
    ad = {k: LowRankAdapters(torch.ones(2, 4, k).half(), torch.ones(2, 8, 4).half()).to(cuda) for k in (250, 256)}
    ids = torch.zeros(3, dtype=I32, device=cuda)
    for w in (250, 256):
        for a in (250, 256):
            for k in (250, 256):
                x, codes = torch.ones(3, k, device=cuda).half(), torch.ones(3, k, dtype=I8, device=cuda)
                for call in (lambda: lin[w](x, adapters=ad[a], ids=ids), lambda: lin[w].forward_int8(codes, torch.ones(3, device=cuda), adapters=ad[a], ids=ids)):
                    if w == a == k:
                        assert call().shape == (3, 8)
                    else:
                        with pytest.raises(AssertionError):
                            call()
