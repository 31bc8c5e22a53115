"""A stand-in for a device tensor, for calls that are refused before any memory is touched."""

import math


class FakeTensor:
    """Looks like a device tensor; its memory is never touched, since the calls are refused."""

    def __init__(self, shape, stride=None, dtype="float32", ptr=1 << 20):
        self.shape, self.dtype, self._p = tuple(shape), "torch." + dtype, ptr
        if stride is None:
            stride, n = [], 1
            for s in reversed(self.shape):
                stride.insert(0, n)
                n *= s
        self._s = tuple(stride)

    def get_device(self):
        return 0

    def element_size(self):
        return {"float64": 8, "float32": 4, "int32": 4, "int64": 8, "uint8": 1}.get(self.dtype[6:], 2)

    def data_ptr(self):
        return self._p

    def stride(self):
        return self._s

    def numel(self):
        return math.prod(self.shape)

    def is_contiguous(self):
        n = 1
        for s, t in zip(reversed(self.shape), reversed(self._s)):
            if s > 1 and t != n:
                return False
            n *= s
        return True
