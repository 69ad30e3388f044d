"""The gated linear recurrence over whole stories (``leo_b200_gated_scan``).

The per-byte step decays every neuron's state and every synapse's trace a tick
at a time.  These operators advance such states over all the tokens of a packed
story batch in one call,

    h[t] = decay[t] * h[t - 1] + drive[t]     (per channel, from ``initial`` at a story's first token),

with their gradients for training (:func:`gated_scan_backward`) and the
one-token form for serving (:func:`gated_step`).  Packed tensors hold the
stories' tokens back to back, ``[tokens, channels]``, as
:func:`leo_b200.synthetic.pack_stories` packs their bytes; a
:class:`StoryLayout` made once from the offsets says where they begin.

Types: float32, bfloat16 or float16 drives; gates of the same type or float32
(slow decays such as 0.999 are 1 in bfloat16); states between tokens, initial
and final states are float32.  The calls run asynchronously on the current
stream of the tensors' device, or on ``stream``, and can be captured into a
CUDA graph.  PyTorch only owns the memory; no gradient is recorded for autograd,
and a tensor that asks for one, or carries a forward-mode tangent, is refused.
"""

from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Sequence

import numpy as np
import torch
from torch.autograd.graph import increment_version

from . import native
from .ctypes_types import LeoB200StoryTables
from .device_tensors import (
    check_contiguous,
    check_tensor,
    current_stream,
    device_of,
    dtype_code,
    on_stream,
    pointer,
    row_stride,
)


class StoryLayout:
    """Where the stories of a packed batch begin, checked once on the host and
    laid out on ``device`` for the scans.  ``story_offsets``: ``stories + 1``
    host integers; empty stories are allowed.  The layout may be used by any
    number of calls, streams and graphs, and must outlive the graphs that captured it."""

    def __init__(self, story_offsets: Sequence[int], device: torch.device | str | int):
        offsets = np.asarray(story_offsets)
        if offsets.ndim != 1 or offsets.size < 2 or offsets.dtype.kind not in "iu":
            raise ValueError("story_offsets must be stories + 1 integers, for one story or more")
        if offsets.dtype.kind == "i" and int(offsets.min()) < 0:
            raise ValueError("story_offsets must not be negative")
        offsets = np.ascontiguousarray(offsets.astype(np.uint64))
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if device.type != "cuda":
            raise ValueError("a story layout lives on a CUDA device")
        stories = offsets.size - 1
        L = native.lib()
        size = L.leo_b200_story_table_bytes(offsets.ctypes.data, stories)
        native.check(0 if size else -1)
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        self.index = device.index
        self.stories = stories
        self.tokens = int(offsets[-1])
        host = torch.empty(size, dtype=torch.uint8)
        self._table = torch.empty(size, dtype=torch.uint8, device=device)
        self._c = LeoB200StoryTables()
        self._ref = C.byref(self._c)
        native.check(L.leo_b200_story_table(offsets.ctypes.data, stories, host.data_ptr(), size,
                                            self._table.data_ptr(), self._ref))
        self._table.copy_(host)  # waits for the copy
        self._home = current_stream(device.index)
        # (scratch bytes, carries) by channels: what every call asks for
        self._sizes: dict[int, tuple[int, int]] = {}

    def _used_on(self, raw: int, stream) -> None:
        """Keeps the table from other uses of its memory until a call on a
        stream other than its own has read it."""
        if raw != self._home:
            self._table.record_stream(stream or torch.cuda.current_stream(self.device))

    def _needs(self, channels: int) -> tuple[int, int]:
        needs = self._sizes.get(channels)
        if needs is None:
            L = native.lib()
            needs = (L.leo_b200_gated_scan_workspace(self._ref, channels),
                     L.leo_b200_gated_scan_carry_count(self._ref, channels))
            self._sizes[channels] = needs
        return needs


class GatedScan(NamedTuple):
    """``states`` [tokens, channels] of the drive's type, ``final`` [stories,
    channels] float32, and what the backward pass needs (``None`` unless kept)."""

    states: torch.Tensor
    final: torch.Tensor
    carries: torch.Tensor | None


class GatedScanGradients(NamedTuple):
    """Gradients in the types and shapes of ``drive`` and ``decay``;
    ``initial`` is ``None`` where the scan had no initial state."""

    drive: torch.Tensor
    decay: torch.Tensor
    initial: torch.Tensor | None


def _check_decay(decay, drive, device: int) -> tuple[int, int, int]:
    """(type code, row stride, one row for all tokens or lanes)."""
    check_tensor("decay", decay, device)
    code = dtype_code("decay", decay)
    if decay.dtype != torch.float32 and decay.dtype != drive.dtype:
        raise ValueError(f"decay must be of the drive's type or float32, not {decay.dtype}")
    if decay.dim() == 1:
        if decay.shape[0] != drive.shape[1] or (decay.shape[0] > 1 and decay.stride(0) != 1):
            raise ValueError("a decay of one row must be one adjacent element a channel")
        return code, 0, 1
    if decay.shape != drive.shape:
        raise ValueError(f"decay must have shape {tuple(drive.shape)} or {tuple(drive.shape[1:])}, "
                         f"not {tuple(decay.shape)}")
    return code, row_stride("decay", decay), 0


def _check_scan(drive, decay, layout, initial):
    """(device, type code and row stride of the drive, the decay's)."""
    device = device_of("drive", drive)
    code, stride = dtype_code("drive", drive), row_stride("drive", drive)
    if layout.index != device:
        raise ValueError(f"the layout is on {layout.device}, not on {drive.device}")
    tokens, channels = drive.shape
    if tokens != layout.tokens or channels == 0:
        raise ValueError(f"drive must have {layout.tokens} tokens of at least one channel, not {tuple(drive.shape)}")
    if initial is not None:
        check_tensor("initial", initial, device, torch.float32, (layout.stories, channels))
        check_contiguous("initial", initial)
    return device, code, stride, _check_decay(decay, drive, device)


def gated_scan(drive, decay, layout: StoryLayout, initial=None, keep_carries: bool = False,
               stream=None) -> GatedScan:
    """The states of every token of a packed batch.

    ``drive``: [tokens, channels]; ``decay``: the same shape, or [channels] for
    one fixed decay a channel (the elements of a row adjacent, rows at any
    distance, so a slice of a wider projection will do).  Gates are meant to lie
    in [-1, 1]; larger ones do as long as the product of those of any span of a
    story stays finite (float32).  An infinite state stays infinite, but may be
    NaN after eight gates in a row whose product is 0 in float32, as after a gate
    of 0.  ``initial``: float32 [stories, channels], zero if ``None``.
    ``keep_carries``: keep what :func:`gated_scan_backward` needs."""
    device, code, stride, (decay_code, decay_stride, shared) = _check_scan(drive, decay, layout, initial)
    tokens, channels = drive.shape
    L = native.lib()
    size, kept = layout._needs(channels)
    with on_stream(device, stream, (drive, decay, initial)) as raw:
        states = drive.new_empty((tokens, channels))
        final = drive.new_empty((layout.stories, channels), dtype=torch.float32)
        carries = drive.new_empty(kept, dtype=torch.float32) if keep_carries else None
        scratch = drive.new_empty(size, dtype=torch.uint8) if size else None
        native.check(L.leo_b200_gated_scan(
            device, layout._ref, channels, code, drive.data_ptr(), stride, decay_code, decay.data_ptr(), decay_stride,
            shared, pointer(initial), states.data_ptr(), final.data_ptr(), pointer(carries), pointer(scratch), size,
            raw))
        layout._used_on(raw, stream)
    return GatedScan(states, final, carries)


def gated_scan_backward(grad_states, drive, decay, layout: StoryLayout, carries, initial=None, grad_final=None,
                        stream=None) -> GatedScanGradients:
    """The gradients of :func:`gated_scan` for the same ``drive``, ``decay``,
    ``layout`` and ``initial``, with the ``carries`` that it kept.
    ``grad_states``: of the drive's shape and type; ``grad_final``: float32
    [stories, channels], zero if ``None``.  The gradient of a [channels] decay
    is summed over all tokens in a fixed order."""
    device, code, stride, (decay_code, decay_stride, shared) = _check_scan(drive, decay, layout, initial)
    tokens, channels = drive.shape
    check_tensor("grad_states", grad_states, device, drive.dtype, drive.shape)
    grad_stride = row_stride("grad_states", grad_states)
    if grad_final is not None:
        check_tensor("grad_final", grad_final, device, torch.float32, (layout.stories, channels))
        check_contiguous("grad_final", grad_final)
    L = native.lib()
    if carries is None:
        raise ValueError("the backward pass needs the carries of gated_scan(..., keep_carries=True)")
    size, kept = layout._needs(channels)
    check_tensor("carries", carries, device, torch.float32, (kept,))
    check_contiguous("carries", carries)
    with on_stream(device, stream, (grad_states, drive, decay, carries, initial, grad_final)) as raw:
        grad_drive = drive.new_empty((tokens, channels))
        grad_decay = decay.new_empty(decay.shape)
        grad_initial = None
        if initial is not None:
            grad_initial = initial.new_empty((layout.stories, channels))
        scratch = drive.new_empty(size, dtype=torch.uint8) if size else None
        native.check(L.leo_b200_gated_scan_backward(
            device, layout._ref, channels, code, grad_states.data_ptr(), grad_stride, drive.data_ptr(), stride,
            decay_code, decay.data_ptr(), decay_stride, shared, pointer(initial), pointer(grad_final),
            carries.data_ptr(), grad_drive.data_ptr(), grad_decay.data_ptr(), pointer(grad_initial),
            pointer(scratch), size, raw))
        layout._used_on(raw, stream)
    return GatedScanGradients(grad_drive, grad_decay, grad_initial)


def gated_scan_gave_up(device: int = 0) -> bool:
    """Whether a wait inside a scan on ``device`` ever gave up, which it should
    never do; that scan's results are not to be used.  Waits for the device."""
    flag = C.c_uint32()
    native.check(native.lib().leo_b200_gated_scan_status(device, C.byref(flag)))
    return bool(flag.value)


def gated_step(drive, decay, state, stream=None):
    """One token for each lane: ``state`` (float32 [lanes, channels]) becomes
    ``decay * state + drive`` in place (for autograd too: a backward pass that
    saved ``state`` before fails); returns it in the drive's type.
    ``drive``: [lanes, channels]; ``decay``: the same shape, or [channels]."""
    device = device_of("drive", drive)
    code, stride = dtype_code("drive", drive), row_stride("drive", drive)
    lanes, channels = drive.shape
    if channels == 0:
        raise ValueError("drive must have at least one channel")
    decay_code, decay_stride, shared = _check_decay(decay, drive, device)
    check_tensor("state", state, device, torch.float32, drive.shape)
    state_stride = row_stride("state", state)
    if state_stride < channels and lanes > 1:
        raise ValueError("the rows of state overlap")
    with on_stream(device, stream, (drive, decay, state)) as raw:
        output = drive.new_empty((lanes, channels))
        native.check(native.lib().leo_b200_gated_step(
            device, lanes, channels, code, drive.data_ptr(), stride, decay_code, decay.data_ptr(), decay_stride, shared,
            state.data_ptr(), state_stride, output.data_ptr(), raw))
    increment_version(state)  # a backward pass that saved it fails instead of using the new values
    return output
