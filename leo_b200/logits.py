"""Operators on rows of logits: penalties, biases and grammar masks
(:func:`adjust_logits`), the next symbol (:func:`pick_symbols`), and the cross
entropy over the allowed symbols with its gradient
(:func:`masked_cross_entropy`).

The per-byte step ends in a softmax over 257 classes, a loss and the errors
``p - onehot``; these act on any rows of logits, of that width or another.
Logits are float32, bfloat16 or float16 CUDA tensors ``[rows, vocabulary]``
whose rows may lie at any distance (a padded or sliced tensor will do).

A grammar mask is a table ``allowed`` of bits, one row of int32 words a
grammar state (:func:`pack_allowed` makes it), and the ``state`` of each row:
-1 masks nothing.  What a masked place holds, NaN and infinities included,
never matters.  The calls run asynchronously on the current stream of the
logits' device, or on ``stream``, and can be captured into a CUDA graph;
``repetition``, ``presence``, ``frequency`` and ``temperature`` are numbers or
float32 CUDA tensors ``[rows]`` (whose values are then not checked).
"""

from __future__ import annotations

import ctypes as C
import struct

import torch
from torch.autograd.graph import increment_version

from . import native
from .ctypes_types import LeoB200LogitRules
from .device_tensors import check_contiguous, check_tensor, device_of, dtype_code, on_stream, pointer, row_stride


def pack_allowed(allowed) -> torch.Tensor:
    """The mask table of a bool tensor ``[states, vocabulary]`` (True: allowed):
    int32 words, bit ``v % 32`` of word ``v // 32`` for symbol ``v``."""
    if allowed.dim() != 2 or allowed.dtype != torch.bool:
        raise ValueError("allowed must be a bool tensor [states, vocabulary]")
    states, vocabulary = allowed.shape
    words = (vocabulary + 31) // 32
    padded = torch.zeros((states, words * 32), dtype=torch.int64, device=allowed.device)
    padded[:, :vocabulary] = allowed
    bits = (padded.view(states, words, 32) << torch.arange(32, device=allowed.device)).sum(2)
    return torch.where(bits >= 2**31, bits - 2**32, bits).to(torch.int32)


def _check_logits(logits):
    """(device, type code, row stride)."""
    device = device_of("logits", logits)
    stride = row_stride("logits", logits)
    if logits.shape[1] == 0:
        raise ValueError("logits must have at least one symbol")
    return device, dtype_code("logits", logits), stride


def _check_mask(logits, device, allowed, state):
    """(row stride, states) of the mask table."""
    rows, vocabulary = logits.shape
    if allowed is None:
        if state is not None:
            raise ValueError("state needs a mask table in allowed")
        return 0, 0
    check_tensor("allowed", allowed, device, torch.int32)
    stride = row_stride("allowed", allowed)
    states, words = allowed.shape
    if words < (vocabulary + 31) // 32:
        raise ValueError(f"allowed must have {(vocabulary + 31) // 32} words a state, not {words}")
    if states == 0:
        raise ValueError("allowed must have at least one state")
    if state is not None:
        check_tensor("state", state, device, torch.int32, (rows,))
        check_contiguous("state", state)
    elif states not in (1, rows):
        raise ValueError(f"without state, allowed must have 1 or {rows} rows, not {states}")
    return stride, states


def _scalar_or_rows(name: str, value, logits, device):
    """(tensor or None, number)."""
    if isinstance(value, torch.Tensor):
        check_tensor(name, value, device, torch.float32, (logits.shape[0],))
        check_contiguous(name, value)
        return value, 0.0
    return None, float(value)


# LeoB200LogitRules as bytes, which are made faster than a structure of ctypes.
_RULES = struct.Struct("@PqIPPPPfffPqPqIP")
assert _RULES.size == C.sizeof(LeoB200LogitRules)


class _Rules:
    """The checked rules of a call, and the tensors that they point at."""

    __slots__ = ("tensors", "packed")

    def __init__(self, logits, device, history, lengths, repetition, presence, frequency, bias, allowed, state):
        rows, vocabulary = logits.shape
        history_stride = capacity = bias_stride = 0
        if history is not None:
            check_tensor("history", history, device, torch.int32)
            history_stride = row_stride("history", history)
            if history.shape[0] != rows:
                raise ValueError(f"history must have {rows} rows, not {history.shape[0]}")
            capacity = history.shape[1]
            if lengths is not None:
                check_tensor("lengths", lengths, device, torch.int32, (rows,))
                check_contiguous("lengths", lengths)
        elif lengths is not None:
            raise ValueError("lengths needs a history")
        repetition_rows, repetition = _scalar_or_rows("repetition", repetition, logits, device)
        presence_rows, presence = _scalar_or_rows("presence", presence, logits, device)
        frequency_rows, frequency = _scalar_or_rows("frequency", frequency, logits, device)
        if repetition_rows is not None:
            repetition = 1.0
        if bias is not None:
            check_tensor("bias", bias, device, torch.float32)
            if bias.dim() == 1:
                if bias.shape[0] != vocabulary or (vocabulary > 1 and bias.stride(0) != 1):
                    raise ValueError(f"a bias of one row must be {vocabulary} adjacent elements")
            else:
                if bias.shape != logits.shape:
                    raise ValueError(f"bias must have shape {tuple(logits.shape)} or ({vocabulary},), "
                                     f"not {tuple(bias.shape)}")
                bias_stride = row_stride("bias", bias)
        allowed_stride, states = _check_mask(logits, device, allowed, state)
        self.tensors = (logits, history, lengths, repetition_rows, presence_rows, frequency_rows, bias, allowed, state)
        address = [0 if x is None else x.data_ptr() for x in self.tensors]
        self.packed = _RULES.pack(address[1], history_stride, capacity, address[2], address[3], address[4], address[5],
                                  repetition, presence, frequency, address[6], bias_stride, address[7],
                                  allowed_stride, states, address[8])


def adjust_logits(logits, *, history=None, lengths=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None,
                  allowed=None, state=None, out=None, stream=None):
    """The logits after penalties, bias and mask, in their own type.

    For a symbol that occurs ``c > 0`` times among the first ``lengths[row]``
    symbols of ``history[row]`` (int32 ``[rows, capacity]``, entries outside
    the vocabulary passed over): a positive logit is divided by ``repetition``
    and another one multiplied by it, then ``presence + frequency * c`` is
    taken off.  ``bias`` (float32 ``[vocabulary]`` or ``[rows, vocabulary]``)
    is added, and what the mask forbids becomes -inf.  ``out`` may be
    ``logits`` itself; another one must not overlap it.  (A backward pass that
    saved ``out`` before fails, as after any operation in place.)"""
    device, code, stride = _check_logits(logits)
    rules = _Rules(logits, device, history, lengths, repetition, presence, frequency, bias, allowed, state)
    rows, vocabulary = logits.shape
    if out is not None:
        check_tensor("out", out, device, logits.dtype, logits.shape)
        if row_stride("out", out) < vocabulary and rows > 1:
            raise ValueError("the rows of out overlap")
    given = out
    with on_stream(device, stream, rules.tensors + (out,)) as raw:
        if out is None:
            out = logits.new_empty((rows, vocabulary))
        native.check(native.lib().leo_b200_adjust_logits(
            device, code, logits.data_ptr(), stride, rows, vocabulary, rules.packed, out.data_ptr(),
            out.stride(0), raw))
    if given is not None:
        increment_version(given)  # a backward pass that saved it fails instead of using the new values
    return out


def pick_symbols(logits, *, temperature=0.0, uniforms=None, history=None, lengths=None, repetition=1.0, presence=0.0,
                 frequency=0.0, bias=None, allowed=None, state=None, stream=None):
    """The next symbol of each row under the rules of :func:`adjust_logits`:
    ``(symbols, log_probability)``, int32 and float32 ``[rows]``.

    Rows of ``temperature`` 0 take the largest adjusted logit, the lowest
    symbol of equal ones.  Others take the first symbol at which the running
    sum of the softmax of ``adjusted / temperature`` passes ``uniforms[row]``
    (float64, in [0, 1); it may be ``None`` only if ``temperature`` is the number 0).
    ``log_probability`` is that of the symbol, at
    temperature 1 for a greedy row.  A row with nothing left gives symbol -1
    and -inf; one with a NaN that is not masked (or a temperature that is
    negative or NaN) -1 and NaN.  Everything is computed in 64 bits from the
    inputs as they are, weights below e^-708 of the largest counting as 0; up to
    8,388,600 symbols."""
    device, code, stride = _check_logits(logits)
    rules = _Rules(logits, device, history, lengths, repetition, presence, frequency, bias, allowed, state)
    rows, vocabulary = logits.shape
    temperature_rows, temperature = _scalar_or_rows("temperature", temperature, logits, device)
    if uniforms is not None:
        check_tensor("uniforms", uniforms, device, torch.float64, (rows,))
        check_contiguous("uniforms", uniforms)
    with on_stream(device, stream, rules.tensors + (temperature_rows, uniforms)) as raw:
        symbols = logits.new_empty(rows, dtype=torch.int32)
        log_probability = logits.new_empty(rows, dtype=torch.float32)
        native.check(native.lib().leo_b200_pick_symbols(
            device, code, logits.data_ptr(), stride, rows, vocabulary, rules.packed,
            pointer(temperature_rows), temperature, pointer(uniforms), symbols.data_ptr(),
            log_probability.data_ptr(), raw))
    return symbols, log_probability


def masked_cross_entropy(logits, targets, *, allowed=None, state=None, weights=None, stream=None):
    """Loss and gradient of each row's target among the symbols that its mask
    allows: ``(losses, gradient)``, float32 ``[rows]`` and the logits' shape
    and type.

    ``losses[r] = log(sum over allowed v of exp l[v]) - l[target]``, not
    weighted; ``gradient[r] = weights[r] * (softmax - onehot)``, 0 where masked
    (``weights``: float32 ``[rows]``, 1 if ``None``).  ``targets``: int32
    ``[rows]``; a negative one marks a row without a target (loss and gradient
    0), one of ``vocabulary`` or more gives loss NaN and gradient 0.  A
    masked target, or a row with nothing left, has loss +inf; the gradient
    stays finite."""
    device, code, stride = _check_logits(logits)
    rows, vocabulary = logits.shape
    check_tensor("targets", targets, device, torch.int32, (rows,))
    check_contiguous("targets", targets)
    allowed_stride, states = _check_mask(logits, device, allowed, state)
    if weights is not None:
        check_tensor("weights", weights, device, torch.float32, (rows,))
        check_contiguous("weights", weights)
    with on_stream(device, stream, (logits, targets, allowed, state, weights)) as raw:
        losses = logits.new_empty(rows, dtype=torch.float32)
        gradient = logits.new_empty((rows, vocabulary))
        native.check(native.lib().leo_b200_masked_cross_entropy(
            device, code, logits.data_ptr(), stride, rows, vocabulary, targets.data_ptr(),
            pointer(allowed), allowed_stride, states, pointer(state), pointer(weights), losses.data_ptr(),
            gradient.data_ptr(), vocabulary, raw))
    return losses, gradient
