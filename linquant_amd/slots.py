"""Slots of serving states (``Mamba2State``, a linear attention's state) copied, forked, exchanged, compacted and freed on the GPU (HIP)."""

from __future__ import annotations

import ctypes

import torch

from linquant_amd import _lib

_MAX_ENTRIES = 8192


def _flatten(states, out):
    if isinstance(states, torch.Tensor):
        out.append(states)
    else:
        for s in states:
            _flatten(s, out)
    return out


def _apart(a, b, slots):
    """Whether two tensors (address, bytes from slot to slot, bytes of a slot) have no byte in common."""
    (at_a, step_a, n_a), (at_b, step_b, n_b) = sorted((a, b))
    if at_a + (slots - 1) * step_a + n_a <= at_b:
        return True
    d = (at_b - at_a) % step_a
    return step_a == step_b and n_a <= d and d + n_b <= step_a  # slots that lie between the other's


def copy_slots(states, src, dst):
    """new[dst[i]] = old[src[i]] in every tensor of ``states``: a tensor, or (nested) lists or tuples of them, such as the ``Mamba2State`` of
    every layer, all with the same number of slots as their first dimension and dense slots.  ``src``, ``dst`` (n,) int32 on the GPU,
    n up to 8192, not read on the host.

    Every source is read before anything is written, so slots can be forked (one source, several destinations), exchanged, put in
    another order or moved together.  A negative source clears the slot (a sequence without tokens); one beyond the slots fills it with NaN
    (all bits one).  Entries whose destination is negative or beyond the slots do nothing; of several with one destination the last counts.
    In place; returns None.  Capturable into a graph."""
    if _lib.native().copy_slots(states, src, dst):
        return
    tensors = _flatten(states, [])
    assert src.dtype == torch.int32 and dst.dtype == torch.int32 and src.dim() == 1 and src.shape == dst.shape, "src, dst: (n,) int32"
    n = src.numel()
    assert n <= _MAX_ENTRIES, f"up to {_MAX_ENTRIES} entries, got {n}"
    if not tensors:
        return
    _lib.same_device(tensors[0], src, dst, *tensors)
    slots = tensors[0].shape[0] if tensors[0].dim() else None
    spans = []
    for t in tensors:
        assert t.dim() >= 1 and t.shape[0] == slots, "states: tensors (slots, ...) with the same number of slots"
        size = t.element_size()
        if t.numel() == 0:
            continue
        assert t[0].is_contiguous() and (slots == 1 or t.stride(0) >= t[0].numel()), "states: dense slots"
        nbytes = t[0].numel() * size
        spans.append((t.data_ptr(), t.stride(0) * size if slots > 1 else nbytes, nbytes))
    assert all(_apart(a, b, slots) for i, a in enumerate(spans) for b in spans[:i]), "states: tensors that do not overlap"
    if not spans or n == 0:
        return
    _lib.below_2_31(slots)
    src, dst = src.contiguous(), dst.contiguous()
    table = (ctypes.c_int64 * (3 * len(spans)))(*(x for span in spans for x in span))
    _lib.call("lq_copy_slots", tensors[0].device, tensors=ctypes.addressof(table), num_tensors=len(spans), num_slots=slots, src=_lib.ptr(src),
              dst=_lib.ptr(dst), entries=n)
