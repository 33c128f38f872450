"""Dtypes of the path (reference dtype.py:1-73).

The reference maps ``bfloat16`` to NumPy float32 (reference dtype.py:31),
i.e. it has no 16-bit brain-float storage.  Here ``bfloat16`` is real 2-byte
device storage (``_cuda_ops.BFLOAT16``); host views of it are float32.
"""
from __future__ import annotations

import enum

import numpy as np

from . import _cuda_ops as _cuops


_F32 = np.dtype(np.float32)
_F16 = np.dtype(np.float16)
_I32 = np.dtype(np.int32)
_U8 = np.dtype(np.uint8)


class dtype(enum.Enum):
    float16 = "float16"
    float32 = "float32"
    bfloat16 = "bfloat16"
    # storage only (indices, packed 4-bit weights): no operator computes in them
    int32 = "int32"
    uint8 = "uint8"

    def to_numpy(self) -> np.dtype:
        """Host dtype of this dtype's values (reference dtype.py:25-39)."""
        if self is dtype.int32 or self is dtype.uint8:
            return np.dtype(self.value)
        return np.dtype(np.float16) if self is dtype.float16 else np.dtype(np.float32)

    def device_storage(self) -> np.dtype:
        """Storage dtype of a device tensor of this dtype."""
        if self is dtype.bfloat16:
            return _cuops.BFLOAT16
        return np.dtype(self.value)

    def of_host(self, arr: np.ndarray) -> np.ndarray:
        """`arr` in this dtype's host type.  The integer types take whole
        numbers of their range only: an index or a packed byte that was
        truncated or wrapped would be another one."""
        to = self.to_numpy()
        if to.kind in "iu" and arr.dtype != to and arr.size:
            info = np.iinfo(to)
            if arr.dtype.kind not in "biu" or arr.min() < info.min or arr.max() > info.max:
                raise TypeError("%s values do not convert to %s" % (arr.dtype, to))
        return arr.astype(to, copy=False)

    @staticmethod
    def from_any(d) -> "dtype":
        # The storage dtypes' own objects first: this runs once per operator
        # result, and comparing NumPy dtypes costs a few 100 ns.
        if d is _F32:
            return dtype.float32
        if d is _cuops.BFLOAT16:
            return dtype.bfloat16
        if d is _F16:
            return dtype.float16
        if d is _I32:
            return dtype.int32
        if d is _U8:
            return dtype.uint8
        if isinstance(d, dtype):
            return d
        if isinstance(d, str):
            return dtype(d)
        nd = np.dtype(d)
        if nd == _cuops.BFLOAT16:
            return dtype.bfloat16
        if nd == np.float16:
            return dtype.float16
        if nd in (np.float32, np.float64):
            return dtype.float32
        if nd == _I32:
            return dtype.int32
        if nd == _U8:
            return dtype.uint8
        raise TypeError("unsupported dtype %r" % (d,))

    @property
    def itemsize(self) -> int:
        if self is dtype.uint8:
            return 1
        return 4 if self is dtype.float32 or self is dtype.int32 else 2

    def __repr__(self) -> str:
        return "scaffolding_amd." + self.value


float16 = dtype.float16
float32 = dtype.float32
bfloat16 = dtype.bfloat16
int32 = dtype.int32
uint8 = dtype.uint8
