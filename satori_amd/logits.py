"""What stands between the logits of a batch and its tokens (satori_hip_logit_rules_*): penalties for tokens that a row has had,
biases, grammar masks, and the best token of each row."""
from __future__ import annotations

import ctypes

import numpy as np

from . import ArgumentException, HipContext, _check, _ffi
from .cache import _address, _array, _at

# A row's parameters, as they lie on the device (satori_hip_logit_row).
LOGIT_ROW = np.dtype([("repetition", "<f4"), ("presence", "<f4"), ("frequency", "<f4"), ("history", "<i4"), ("parent", "<i4"),
                      ("token", "<i4"), ("biases", "<i4"), ("mask", "<i4")])


class LogitBatch(ctypes.Structure):
    """A call's arrays: device pointers, strides in elements (satori_hip_logit_batch). Made once and passed while they stay."""
    _fields_ = [("rows", ctypes.c_void_p), ("logits", ctypes.c_void_p), ("output", ctypes.c_void_p), ("best", ctypes.c_void_p),
                ("history", ctypes.c_void_p), ("lengths", ctypes.c_void_p), ("masks", ctypes.c_void_p),
                ("logits_stride", ctypes.c_int64), ("output_stride", ctypes.c_int64), ("history_stride", ctypes.c_int64),
                ("mask_stride", ctypes.c_int64), ("count", ctypes.c_int), ("histories", ctypes.c_int),
                ("mask_count", ctypes.c_int)]


class LogitRules:
    """The bias sets of a vocabulary, at most `bias_entries` tokens each, and the workspace of the calls."""

    def __init__(self, context: HipContext, vocabulary: int, bias_sets: int = 0, bias_entries: int = 0):
        handle = ctypes.c_void_p()
        _check(_ffi.lib().satori_hip_logit_rules_create(context.handle, vocabulary, bias_sets, bias_entries,
                                                        ctypes.byref(handle)))
        self.context, self.vocabulary, self._handle = context, vocabulary, handle

    def set_biases(self, index: int, tokens, values, stream: int = 0) -> None:
        """Set `index`'s tokens, each once, and their values."""
        listed, added = _array(tokens), np.ascontiguousarray(values, np.float32).reshape(-1)
        if len(listed) != added.size:
            raise ArgumentException("Lengths differ.")
        _check(_ffi.lib().satori_hip_logit_rules_set_biases(self._handle, index, _address(listed), _at(added),
                                                            len(listed), stream))

    def apply(self, batch: LogitBatch, stream: int = 0) -> None:
        _check(_ffi.lib().satori_hip_logit_rules_apply(self._handle, ctypes.byref(batch), stream))

    def dispose(self) -> None:
        _check(_ffi.lib().satori_hip_logit_rules_destroy(self._handle))
