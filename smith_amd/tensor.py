"""Minimal device tensor -- the part of src/tensor.js the path needs.

The reference's T.create (src/tensor.js:55-74) returns a pooled SHARED Metal
buffer with a typed-array view (zero copy).  On MI355X the buffer is device
memory: `.data` downloads a host copy and `set_data` uploads, both explicit.
Row-major and contiguous only (the reference's matmulQ4 also passes
a.buffer with no offset or strides, src/ops/quantize.js:83).
"""
import numpy as np

from . import device, prng

# bf16: the upper halves of f32 words on the host, a uint16 array; numbers of any
# other type are rounded to them
_DTYPES = {"f32": np.float32, "i32": np.int32, "u8": np.uint8, "f16": np.float16, "bf16": np.uint16}


def _host(values, dtype):
    """values as the host array of a tensor of dtype."""
    a = np.asarray(values)
    if dtype == "bf16" and a.dtype.kind == "f":  # to nearest, ties to even
        u = np.ascontiguousarray(a, dtype=np.float32).view(np.uint32)
        return np.where((u & 0x7FFFFFFF) > 0x7F800000, u >> 16 | 0x40,
                        (u + (0x7FFF + (u >> 16 & 1))) >> 16).astype(np.uint16).reshape(a.shape)
    return np.asarray(a, dtype=_DTYPES[dtype], order="C")  # a scalar stays one


def _values(values, dtype):
    """The same of a user's values: whole numbers are numbers, and a bf16 tensor's
    bits only as uint16, which is what .data gives."""
    a = np.asarray(values)
    if dtype == "bf16" and a.dtype != np.uint16:
        a = a.astype(np.float32)
    return _host(a, dtype)


class Tensor:
    __slots__ = ("shape", "dtype", "buffer", "size", "strides", "offset", "_owner")

    def __init__(self, shape, dtype="f32", buffer=None):
        self.shape = [int(s) for s in shape]
        self.dtype = dtype
        self.size = int(np.prod(self.shape)) if self.shape else 1
        st, acc = [], 1
        for s in reversed(self.shape):
            st.append(acc)
            acc *= s
        self.strides = list(reversed(st))
        self.offset = 0
        self._owner = buffer is None
        self.buffer = buffer if buffer is not None else device.alloc(self.nbytes)

    @property
    def nbytes(self):
        return self.size * np.dtype(_DTYPES[self.dtype]).itemsize

    @property
    def data(self):
        """Host copy of the contents (device -> host, waits for the stream)."""
        return device.download(self.buffer, self.nbytes, _DTYPES[self.dtype]).reshape(self.shape)

    def set_data(self, arr):
        a = _values(arr, self.dtype)
        if a.size != self.size:
            raise ValueError("set_data: %d elements for a tensor of %d" % (a.size, self.size))
        device.upload(self.buffer, a)
        return self

    def release(self):
        if self._owner and self.buffer:
            device.release_buffer(self.buffer)
        self.buffer = None

    def __repr__(self):
        return "Tensor(shape=%s, dtype=%s)" % (self.shape, self.dtype)


def create(shape, dtype="f32"):
    return Tensor(shape, dtype)


def tensor(data, shape=None, dtype="f32"):
    a = _values(data, dtype)
    t = Tensor(list(a.shape) if shape is None else shape, dtype)
    return t.set_data(a)


def zeros(shape, dtype="f32"):
    return tensor(np.zeros(shape, dtype=_DTYPES[dtype]), dtype=dtype)


def ones(shape, dtype="f32"):
    return tensor(np.ones(shape), dtype=dtype)


def randn(shape, seed=0, std=1.0, mean=0.0):
    """Seeded N(mean, std) -- src/tensor.js:127-146 with a reproducible source."""
    return tensor(prng.randn(shape, seed, std=std, mean=mean))


def to_array(t):
    """toArray: nested host values of a tensor."""
    return t.data.tolist()
